// The loss that keeps codes in even use, C sum_c f_c P_c with f_c = n_c / sum n and
// P_c the mean of softmax(z)_c over the rows that have a code, and its gradient.
//
// sum_c f_c P_c is the mean over the rows of d = sum_c p_c f_c, so no sums over
// columns are needed: with the counts at hand each row is one weighted softmax sum
// (code_rows.cuh), read once. The sums of d over rows are 64-bit, in a fixed order.
//
// Forward and backward, of these the pass over the rows: 2^20 x 256 bf16 335 to 342 and
// 139 us (3.9 TB/s), 16,384 x 16,383 fp16 468 and 190, 65,536 x 1,000 fp32 forward alone 64
// and 55 (4.8 TB/s). What holds the pass over the rows is latency: 46 to 58 % of the issue
// slots with the 22 to 35 % of the warps that its registers leave.
#include "code_tiles.cuh"

namespace gsb {
namespace {

constexpr int kGroupThreads = 256;
constexpr int kCountBlocks = 2 * 148;
constexpr int kCountSharedCodes = 8192;  // counts that a block keeps in shared memory
constexpr int kCountFew = 8192;          // slots that one block counts alone
// Blocks an SM. Short rows wait for memory (65,536 x 1,000 fp32: 62 us with 6, 70 with
// 4); long ones want registers (16,384 x 16,383 fp16, with the backward: 583 and 550 us).
constexpr int kBalanceBlocksShort = 6;
constexpr int kBalanceBlocksLong = 4;
constexpr int kBalanceSums = 32 * 148;   // sums over rows, at most
constexpr int kStateHead = 8;  // floats before the counts in `state`; [0]: C / (rows with a code x codes counted)

__host__ __device__ inline int64_t padded(int64_t codes) { return (codes + 7) / 8 * 8; }

// Where the counts are as floats: `state` behind its head, in the two layouts of Counts.
__host__ __device__ inline Counts counts_of(const float* state, int64_t codes) {
  return Counts{state + kStateHead, state + kStateHead + padded(codes), padded(codes) / 8};
}
// From 2^24 uses of one code on its count is rounded to fp32, by 2^-24 of it at most, and so
// are differences of such counts, whatever their own size. A 64-bit count would cost a value
// twice the bytes and its half of a packed operation.
__device__ __forceinline__ void put_count(float* state, int64_t codes, int64_t c, float n) {
  state[kStateHead + c] = n;
  state[kStateHead + padded(codes) + (c & 7) * (padded(codes) / 8) + (c >> 3)] = n;
}

struct CountParts {  // of each block of the counting kernel: codes counted, rows with one
  uint32_t* codes = nullptr;
  uint32_t* rows = nullptr;
};

// Sum over the threads of a block, in thread 0.
template <typename V>
__device__ __forceinline__ V block_total(V v, V* s_warp) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  if (threadIdx.x % 32 == 0) s_warp[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0;
  if (threadIdx.x == 0)
    for (int w = 0; w < (int)blockDim.x / 32; ++w) v += s_warp[w];
  return v;
}

// How often each code occurs. A block counts in shared memory where the codebook
// fits there (a few hot codes would serialise atomics on L2), and adds what is not
// zero. kAlone: the only block; it writes every count, and their floats, itself. 2^20 x 2
// codes: 9 us.
template <bool kShared, bool kAlone>
__global__ void __launch_bounds__(512)
    k_code_counts(int64_t rows, int bag, int C, Codes codes, int32_t* __restrict__ counts,
                  float* __restrict__ state, CountParts parts, uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ int s_count[];
  __shared__ uint32_t s_warp[2][16];
  if constexpr (kShared) {
    for (int c = threadIdx.x; c < C; c += blockDim.x) s_count[c] = 0;
    __syncthreads();
  }
  uint32_t sum = 0, valid = 0;
  for (int64_t g = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; g < rows; g += (int64_t)gridDim.x * blockDim.x) {
    uint32_t some = 0;
    for (int j = 0; j < bag; ++j) {
      const int64_t c = codes.at(g * bag + j);
      if (c >= C) bad_code(status, kSiteCode);
      if (c >= 0 && c < C) {
        if constexpr (kShared) atomicAdd(&s_count[c], 1);
        else atomicAdd(&counts[c], 1);
        ++some;
      }
    }
    sum += some;
    valid += some != 0;
  }
  sum = block_total(sum, s_warp[0]);
  valid = block_total(valid, s_warp[1]);  // its barrier ends the counting too
  if (threadIdx.x == 0) {
    parts.codes[blockIdx.x] = sum;
    parts.rows[blockIdx.x] = valid;
  }
  if constexpr (kShared) {
    for (int c = threadIdx.x; c < C; c += blockDim.x) {
      const int v = s_count[c];
      if constexpr (kAlone) counts[c] = v, put_count(state, C, c, (float)v);
      else if (v) atomicAdd(&counts[c], v);
    }
    if constexpr (kAlone)
      for (int c = C + threadIdx.x; c < (int)padded(C); c += blockDim.x) put_count(state, C, c, 0.0f);
  }
}

__global__ void __launch_bounds__(256)
    k_counts_f32(int64_t C, const int32_t* __restrict__ counts, float* __restrict__ state) {
  pdl_wait();
  pdl_trigger();
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c < padded(C)) put_count(state, C, c, c < C ? (float)counts[c] : 0.0f);
}

// Whether a row has a code; `width` lanes look.
template <int WIDTH>
__device__ __forceinline__ bool any_code(const Codes& codes, int64_t row, int bag, int64_t C, int lane) {
  int some = 0;
  for (int j = lane; j < bag; j += WIDTH) {
    const int64_t c = codes.at(row * bag + j);
    some |= c >= 0 && c < C;
  }
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) some |= __shfl_xor_sync(kFullMask, some, o, WIDTH);
  return some;
}

// d = sum_c p_c n_c of a row, and what its gradient needs: m, 1 / (1 + s') (0 for a
// row that takes no part), dr = d - n_a, n_a.
__device__ __forceinline__ float finish(RowStat r, bool valid, float4* stats) {
  if (r.m == __int_as_float(0x7f800000)) r.s = quiet_nan();
  const bool out = !valid || (r.m == neg_inf() && r.s == r.s);
  const float inv = out ? 0.0f : 1.0f / (1.0f + r.s);
  const float dr = out ? 0.0f : r.w * inv;
  if (stats) *stats = make_float4(r.m, inv, dr, r.n);
  return out ? 0.0f : r.n + dr;
}

// parts > 1: a part's sums go to `stat` and `stat_a` for k_balance_join.
template <typename T, int L>
__global__ void __launch_bounds__(kTileWarps * 32, L < 32 ? kBalanceBlocksShort : kBalanceBlocksLong)
    k_balance(TileRows<T> t, int bag, Codes codes, Counts counts, float4* __restrict__ stats,
              float4* __restrict__ stat, uint32_t* __restrict__ stat_a, double* __restrict__ sums) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ uint4 s_buf[];
  const int warp = threadIdx.x / 32, lane32 = threadIdx.x % 32, lane = lane32 % L;
  int64_t code = -1;  // one of the row's; a lane takes more only where there are more than lanes
  RowStat row;
  double sum = 0.0;
  walk_tiles<T, L>(
      t, s_buf + warp * kTilePieces * 32, lane32, false,
      [&](const TilePlace<T, L>& place) { code = lane < bag ? codes.at(place.row * bag + lane) : -1; },
      [&](const TilePlace<T, L>& now, int slice, const Slice<T, L>& at, const LaneBuf& buf, auto&& refill) {
        float second;
        RowStat r = lane_sums<true>(buf, at, counts.from(now.c0), second, [](int, float) {}, refill);
        if (L == 32 && r.a != 0xffffffffu) r.a += (uint32_t)now.c0;
        row = slice == 0 ? r : join<true>(row, r);
      },
      [&](const TilePlace<T, L>& now, const Slice<T, L>&, const LaneBuf&) {
        const RowStat r = join_lanes<true, L>(row);
        int valid = code >= 0 && code < t.codes;
        for (int j = lane + L; j < bag; j += L) {
          const int64_t c = codes.at(now.row * bag + j);
          valid |= c >= 0 && c < t.codes;
        }
#pragma unroll
        for (int d = L / 2; d > 0; d >>= 1) valid |= __shfl_xor_sync(kFullMask, valid, d, L);
        if (lane == 0) {
          if (L < 32 || t.parts == 1) {
            if (now.on) sum += (double)finish(r, valid, stats ? stats + now.row : nullptr);
          } else {
            stat[now.item] = make_float4(r.m, r.s, r.w, r.n);
            stat_a[now.item] = r.a;
          }
        }
      });
  if (t.parts == 1) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFullMask, sum, d);
    if (lane32 == 0) sums[blockIdx.x * kTileWarps + warp] = sum;
  }
}
TilePlan balance_plan(int64_t rows, int64_t codes, int size, bool shifted) {
  return tile_plan(rows, codes, size, shifted, 1 << 20, kBalanceBlocksLong, kBalanceBlocksShort);
}

// A warp per row joins its parts' sums. Latency alone: 4 to 6 us.
__global__ void __launch_bounds__(128)
    k_balance_join(int64_t rows, int64_t C, int bag, int parts, Codes codes, const float4* __restrict__ stat,
                   const uint32_t* __restrict__ stat_a, float4* __restrict__ stats, double* __restrict__ sums) {
  pdl_wait();
  pdl_trigger();
  __shared__ double s_warp[4];
  const int lane = threadIdx.x % 32;
  double sum = 0.0;
  for (int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 32; row < rows; row += (int64_t)gridDim.x * 4) {
    // A lane without a part adds nothing: -inf at an index behind all.
    RowStat r{neg_inf(), 0.0f, 0.0f, 0.0f, 0xffffffffu};
    for (int i = lane; i < parts; i += 32) {
      const float4 v = stat[row * parts + i];
      r = join<true>(r, RowStat{v.x, v.y, v.z, v.w, stat_a[row * parts + i]});
    }
    r = join_lanes<true, 32>(r);
    const bool valid = any_code<32>(codes, row, bag, C, lane);
    if (lane == 0) sum += (double)finish(r, valid, stats ? stats + row : nullptr);
  }
  sum = block_total(sum, s_warp);
  if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// The loss from the sums over rows, in one block: 4 to 6 us of latency.
__global__ void __launch_bounds__(256)
    k_balance_loss(int blocks, int64_t C, const double* __restrict__ sums, int count_blocks, CountParts parts,
                   float* __restrict__ loss, float* __restrict__ state) {
  pdl_wait();
  pdl_trigger();
  __shared__ double s_warp[3][8];
  double d = 0.0, codes = 0.0, rows = 0.0;
  for (int i = threadIdx.x; i < blocks; i += 256) d += sums[i];
  for (int i = threadIdx.x; i < count_blocks; i += 256) codes += parts.codes[i], rows += parts.rows[i];
  d = block_total(d, s_warp[0]);
  codes = block_total(codes, s_warp[1]);
  rows = block_total(rows, s_warp[2]);
  if (threadIdx.x == 0) {
    const double k = rows > 0.0 ? (double)C / (codes * rows) : 0.0;
    *loss = (float)(k * d);
    state[0] = (float)k;
  }
}

// dz_c = g coef p_c ((n_c - n_a) - dr); bound by the logits' and the gradient's bytes where
// both are read in whole pieces: 16,384 x 4,096 fp32 79 us (its last writes still
// in L2), 2^20 x 64 bf16 55 (5.1 TB/s). Between 16-byte boundaries, where a count is a load
// of its own and registers spill, 69 % of the issue slots: 2,047 x 50,001 fp16 102 us
// (4.0 TB/s). `at` deals out the result's values (SAME: the logits' lie alike), p and dz are
// their place 0, that of code -shift.
template <bool SAME, typename T, Mode M>
__device__ __forceinline__ void balance_grad(float k, float4 st, const Deal<T, M>& at, int shift, bool on,
                                             const T* __restrict__ p, const Counts& counts, T* __restrict__ dz) {
  float z[kRowElems];
  if constexpr (SAME) load_row(p, at, z);
  else load_row_single(p, at, z);
  const Counts::Offsets off(counts, shift);
  const Base base(st.x);
  if (__any_sync(kFullMask, base.far)) {
    const float f = k * st.y;
#pragma unroll
    for (int i = 0; i < kRowElems; i += 4) {
      if (at.place(i) - at.lane * Deal<T, M>::VEC >= at.hi) continue;  // no lane has any
      float n[4];
      counts.four(at, shift, off, i, n);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = ex2_approx((z[i + j] - st.x) * kLog2e);
        z[i + j] = f * e * ((n[j] - st.w) - st.z);
      }
    }
  } else {
    const F2 l2 = f2(kLog2e), neg_M = f2(base.neg_M), neg_n = f2(-st.w), neg_dr = f2(-st.z),
             f = f2(k * st.y * base.undo);
#pragma unroll
    for (int i = 0; i < kRowElems; i += 4) {
      if (at.place(i) - at.lane * Deal<T, M>::VEC >= at.hi) continue;  // no lane has any
      float n[4];
      counts.four(at, shift, off, i, n);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        float y0, y1;
        split(fma2(f2(z[i + j], z[i + j + 1]), l2, neg_M), y0, y1);
        const F2 e = mul2(f2(ex2_approx(y0), ex2_approx(y1)), f);
        split(mul2(e, add2(add2(f2(n[j], n[j + 1]), neg_n), neg_dr)), z[i + j], z[i + j + 1]);
      }
    }
  }
  if (st.y == 0.0f) {  // takes no part, whatever it holds
#pragma unroll
    for (int i = 0; i < kRowElems; ++i) z[i] = 0.0f;
  }
  if (on) store_row(dz, at, z);
}

template <typename T, Mode M, bool SAME, int L>
__global__ void __launch_bounds__(kGroupThreads, kRowThreadsSM / kGroupThreads)
    k_balance_bwd_group(int64_t rows, int C, const T* __restrict__ logits, int64_t stride,
                        const float4* __restrict__ stats, const float* __restrict__ state,
                        const float* __restrict__ g_loss, T* __restrict__ g_logits) {
  pdl_wait();
  pdl_trigger();
  const float k = *g_loss * state[0];
  const int64_t mine = ((int64_t)blockIdx.x * kGroupThreads + threadIdx.x) / L;
  const bool on = mine < rows;
  const int64_t row = on ? mine : rows - 1;
  T* dz = g_logits + row * C;
  const int shift = shift_of<T, M>(dz);
  balance_grad<SAME>(k, stats[row], Deal<T, M>(shift, C + shift, L, threadIdx.x % L), shift, on,
                     logits + row * stride - shift, counts_of(state, C), dz - shift);
}

template <typename T, Mode M, bool SAME, int W>
__global__ void __launch_bounds__(W * 32, kRowThreadsSM / (W * 32))
    k_balance_bwd_block(int64_t items, int64_t C, int parts, int part_len, const T* __restrict__ logits,
                        int64_t stride, const float4* __restrict__ stats, const float* __restrict__ state,
                        const float* __restrict__ g_loss, T* __restrict__ g_logits) {
  pdl_wait();
  pdl_trigger();
  const float k = *g_loss * state[0];
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = parts == 1 ? item : item / parts;
    T* dz = g_logits + row * C;
    const int shift = shift_of<T, M>(dz), part = (int)(item - row * parts);
    const int c0 = part * part_len;  // of place 0, but for the shift
    const int hi = (int)min((int64_t)part_len, C + shift - c0), lo = part == 0 ? shift : 0;
    balance_grad<SAME>(k, stats[row], Deal<T, M>(lo, hi, W * 32, threadIdx.x), shift, true,
                       logits + row * stride + c0 - shift, counts_of(state, C).from(c0), dz + c0 - shift);
  }
}

struct BalanceScratch {
  CountParts count;
  double* sums = nullptr;
  float4* stat = nullptr;
  uint32_t* stat_a = nullptr;
};
BalanceScratch carve(Carver& ws, int64_t rows, const TilePlan& plan) {
  BalanceScratch b;
  b.count.codes = ws.take<uint32_t>(kCountBlocks);
  b.count.rows = ws.take<uint32_t>(kCountBlocks);
  b.sums = ws.take<double>(kBalanceSums);
  if (plan.parts > 1) {
    b.stat = ws.take<float4>((size_t)rows * plan.parts);
    b.stat_a = ws.take<uint32_t>((size_t)rows * plan.parts);
  }
  return b;
}

}  // namespace
}  // namespace gsb

using namespace gsb;

extern "C" int64_t gsb_code_balance_state_floats(int64_t codebook_rows) {
  return codebook_rows <= 0 ? 0 : kStateHead + 2 * padded(codebook_rows);
}

extern "C" size_t gsb_code_balance_workspace_size(int64_t rows, int64_t codebook_rows) {
  if (check_rows(GSB_DTYPE_F32, rows, codebook_rows, 0, 4) != GSB_OK) return 0;
  size_t need = 0;
  for (int size = 2; size <= 4; size += 2) {
    for (int shifted = 0; shifted < 2; ++shifted) {
      Carver c(nullptr);
      carve(c, rows, balance_plan(rows, codebook_rows, size, shifted));
      need = std::max(need, c.off);
    }
  }
  return need;
}

extern "C" int gsb_code_balance_forward(int32_t dtype, int64_t rows, int64_t codebook_rows, int32_t bag,
                                        const void* logits, int64_t logits_stride, const void* codes,
                                        int32_t code_bytes, float* loss, int32_t* counts, float* stats, float* state,
                                        uint32_t* status, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_rows(dtype, rows, codebook_rows, logits_stride, code_bytes);
  if (rc != GSB_OK) return rc;
  if (bag <= 0) return GSB_ERR_INVALID_ARGUMENT;
  if (rows >= (int64_t(1) << 31) / bag) return GSB_ERR_CAPACITY;
  if (reinterpret_cast<uintptr_t>(stats) % 16 != 0 || reinterpret_cast<uintptr_t>(state) % 16 != 0)
    return GSB_ERR_INVALID_ARGUMENT;
  if (!loss || !counts || !state || !status || (rows > 0 && (!logits || !codes))) return GSB_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < gsb_code_balance_workspace_size(rows, codebook_rows)) return GSB_ERR_WORKSPACE;
  if (rows == 1) logits_stride = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const TilePlan plan = balance_plan(rows, codebook_rows, dtype_bytes(dtype),
                                     rows_shifted(dtype_bytes(dtype), logits, logits_stride));
  Carver ws(workspace);
  const BalanceScratch b = carve(ws, rows, plan);
  const Codes cd{codes, code_bytes == 8};
  const Counts counts_f32 = counts_of(state, codebook_rows);
  // The counts.
  const bool shared = codebook_rows <= kCountSharedCodes;
  const int64_t slots = rows * bag;
  unsigned count_blocks = 1;
  if (shared && slots <= kCountFew) {
    launch_pdl(k_code_counts<true, true>, 1, 512, sizeof(int) * (size_t)codebook_rows, s, rows, bag,
               (int)codebook_rows, cd, counts, state, b.count, status);
    note_launches(1);
  } else {
    if (cudaMemsetAsync(counts, 0, sizeof(int32_t) * (size_t)codebook_rows, s) != cudaSuccess) return GSB_ERR_CUDA;
    count_blocks = (unsigned)std::min<int64_t>(kCountBlocks, grid1d(rows, 512));
    if (shared)
      launch_pdl(k_code_counts<true, false>, count_blocks, 512, sizeof(int) * (size_t)codebook_rows, s, rows, bag,
                 (int)codebook_rows, cd, counts, state, b.count, status);
    else
      launch_pdl(k_code_counts<false, false>, count_blocks, 512, 0, s, rows, bag, (int)codebook_rows, cd, counts,
                 state, b.count, status);
    launch_pdl(k_counts_f32, grid1d(padded(codebook_rows), 256), 256, 0, s, codebook_rows, (const int32_t*)counts,
               state);
    note_launches(2);
  }
  // The rows.
  int n_sums = 0;
  if (rows > 0) {
    with_dtype(dtype, [&](auto tag) {
      using T = decltype(tag);
      const int64_t items = plan.items(rows);
      const TileRows<T> t{(const T*)logits, logits_stride, rows, codebook_rows, plan.part_len, items, plan.parts};
      const int blocks = plan.blocks(rows);
      n_sums = blocks * kTileWarps;
      with_tile_lanes(plan.lanes, [&](auto l) {
        launch_pdl(k_balance<T, decltype(l)::value>, blocks, kTileWarps * 32,
                   kTileWarps * kTilePieces * 32 * sizeof(uint4), s, t, bag, cd, counts_f32,
                   (float4*)stats, b.stat, b.stat_a, b.sums);
      });
    });
    note_launches(1);
    if (plan.parts > 1) {
      n_sums = std::min(kBalanceSums, grid1d(rows, 4));
      launch_pdl(k_balance_join, n_sums, 128, 0, s, rows, codebook_rows, bag, plan.parts, cd, (const float4*)b.stat,
                 (const uint32_t*)b.stat_a, (float4*)stats, b.sums);
      note_launches(1);
    }
  }
  launch_pdl(k_balance_loss, 1, 256, 0, s, n_sums, codebook_rows, (const double*)b.sums, (int)count_blocks, b.count,
             loss, state);
  note_launches(1);
  return cuda_status(cudaGetLastError());
}

extern "C" int gsb_code_balance_backward(int32_t dtype, int64_t rows, int64_t codebook_rows, const void* logits,
                                         int64_t logits_stride, const float* stats, const float* state,
                                         const float* g_loss, void* g_logits, void* stream) {
  const int rc = check_rows(dtype, rows, codebook_rows, logits_stride, 4);
  if (rc != GSB_OK) return rc;
  if (rows == 0) return GSB_OK;
  if (!logits || !stats || !state || !g_loss || !g_logits) return GSB_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(stats) % 16 != 0 || reinterpret_cast<uintptr_t>(state) % 16 != 0)
    return GSB_ERR_INVALID_ARGUMENT;
  if (rows == 1) logits_stride = codebook_rows;  // as the result's
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  with_row_pairs(dtype, logits, logits_stride, g_logits, codebook_rows, [&](auto t, auto m, auto same) {
    using T = decltype(t);
    constexpr Mode M = decltype(m)::value;
    constexpr bool SAME = decltype(same)::value;
    const RowPlan plan = row_plan(rows, codebook_rows, M == Mode::kShifted, Deal<T, M>::VEC);
    if (plan.lanes > 0) {
      with_lanes(plan.lanes, [&](auto l) {
        constexpr int L = decltype(l)::value;
        launch_pdl(k_balance_bwd_group<T, M, SAME, L>, grid1d(rows * L, kGroupThreads), kGroupThreads, 0, s, rows,
                   (int)codebook_rows, (const T*)logits, logits_stride, (const float4*)stats, state, g_loss,
                   (T*)g_logits);
      });
    } else {
      with_warps(plan.warps, [&](auto w) {
        constexpr int W = decltype(w)::value;
        launch_pdl(k_balance_bwd_block<T, M, SAME, W>, item_grid(rows * plan.parts), W * 32, 0, s,
                   rows * plan.parts, codebook_rows, plan.parts, plan.part_len, (const T*)logits, logits_stride,
                   (const float4*)stats, state, g_loss, (T*)g_logits);
      });
    }
  });
  note_launches(1);
  return cuda_status(cudaGetLastError());
}
