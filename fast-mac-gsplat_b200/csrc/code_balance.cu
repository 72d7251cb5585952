// The loss that keeps codes in even use, C sum_c f_c P_c with f_c = n_c / sum n and
// P_c the mean of softmax(z)_c over the rows that have a code, and its gradient.
//
// sum_c f_c P_c is the mean over the rows of d = sum_c p_c f_c, so no sums over
// columns are needed: with the counts at hand each row is one weighted softmax sum
// (code_rows.cuh), read once. The sums of d over rows are 64-bit, in a fixed order.
#include "code_rows.cuh"

namespace gsb {
namespace {

constexpr int kGroupThreads = 256;
constexpr int kCountBlocks = 2 * 148;
constexpr int kCountSharedCodes = 8192;  // counts that a block keeps in shared memory
constexpr int kCountFew = 8192;          // slots that one block counts alone
constexpr int kBalanceBlocks = 16 * 148;
constexpr int kStateHead = 8;  // floats before the counts in `state`; [0]: C / (rows with a code x codes counted)

__host__ __device__ inline int64_t padded(int64_t codes) { return (codes + 7) / 8 * 8; }

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
// zero. kAlone: the only block; it writes every count, and their floats, itself.
template <bool kShared, bool kAlone>
__global__ void __launch_bounds__(512)
    k_code_counts(int64_t rows, int bag, int C, Codes codes, int32_t* __restrict__ counts,
                  float* __restrict__ counts_f32, CountParts parts, uint32_t* status) {
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
      if constexpr (kAlone) counts[c] = v, counts_f32[c] = (float)v;
      else if (v) atomicAdd(&counts[c], v);
    }
    if constexpr (kAlone)
      for (int c = C + threadIdx.x; c < (int)padded(C); c += blockDim.x) counts_f32[c] = 0.0f;
  }
}

__global__ void __launch_bounds__(256)
    k_counts_f32(int64_t C, const int32_t* __restrict__ counts, float* __restrict__ counts_f32) {
  pdl_wait();
  pdl_trigger();
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c < padded(C)) counts_f32[c] = c < C ? (float)counts[c] : 0.0f;
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

// Rows of up to 512 codes: L lanes each.
template <typename T, int VEC, int L>
__global__ void __launch_bounds__(kGroupThreads)
    k_balance_group(int64_t rows, int C, int bag, const T* __restrict__ logits, int64_t stride, Codes codes,
                    const float* __restrict__ counts, float4* __restrict__ stats, double* __restrict__ sums) {
  pdl_wait();
  pdl_trigger();
  __shared__ double s_warp[kGroupThreads / 32];
  constexpr int kRows = kGroupThreads / L;
  const int lane = threadIdx.x % L;
  double sum = 0.0;
  for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < rows; row0 += (int64_t)gridDim.x * kRows) {
    const int64_t mine = row0 + threadIdx.x / L;
    const bool on = mine < rows;
    const int64_t row = on ? mine : rows - 1;  // lanes without a row keep a warp's exchanges whole
    float z[kRowElems];
    load_row<VEC>(logits + row * stride, C, L, lane, z);
    const bool valid = any_code<L>(codes, row, bag, C, lane);
    const RowStat r = row_stat<VEC, L, true>(z, C, L, lane, counts, [&](int c) { return counts[c]; });
    if (on && lane == 0) sum += (double)finish(r, valid, stats ? stats + row : nullptr);
  }
  sum = block_total(sum, s_warp);
  if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// One block of W warps per stretch; parts > 1: its sums go to `stat` for k_balance_join.
template <typename T, int VEC, int W>
__global__ void __launch_bounds__(W * 32)
    k_balance_block(int64_t items, int64_t C, int bag, int parts, int part_len, const T* __restrict__ logits,
                    int64_t stride, Codes codes, const float* __restrict__ counts, float4* __restrict__ stats,
                    float4* __restrict__ stat, uint32_t* __restrict__ stat_a, double* __restrict__ sums) {
  pdl_wait();
  pdl_trigger();
  __shared__ RowStat s_stat[2][W];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  double sum = 0.0;
  int turn = 0;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x, turn ^= 1) {
    const int64_t row = parts == 1 ? item : item / parts;
    const int c0 = (int)(item - row * parts) * part_len;
    const int len = (int)min((int64_t)part_len, C - c0);
    float z[kRowElems];
    load_row<VEC>(logits + row * stride + c0, len, W * 32, tid, z);
    const bool valid = warp == 0 && parts == 1 && any_code<32>(codes, row, bag, C, lane);
    const float* n = counts + c0;
    RowStat r = row_stat<VEC, 32, true>(z, len, W * 32, tid, n, [&](int c) { return n[c]; });
    r.a += (uint32_t)c0;
    if (W > 1) {
      // Two buffers: a warp writes the next stretch's while warp 0 may still read this one's.
      if (lane == 0) s_stat[turn][warp] = r;
      __syncthreads();
      if (warp == 0) {
        r = s_stat[turn][lane % W];
#pragma unroll
        for (int d = W / 2; d > 0; d >>= 1) r = shuffle_join<true>(r, d, W);
      }
    }
    if (tid == 0) {
      if (parts == 1) {
        sum += (double)finish(r, valid, stats ? stats + row : nullptr);
      } else {
        stat[item] = make_float4(r.m, r.s, r.w, r.n);
        stat_a[item] = r.a;
      }
    }
  }
  if (parts == 1 && tid == 0) sums[blockIdx.x] = sum;
}

// A warp per row joins its stretches' sums.
__global__ void __launch_bounds__(128)
    k_balance_join(int64_t rows, int64_t C, int bag, int parts, Codes codes, const float4* __restrict__ stat,
                   const uint32_t* __restrict__ stat_a, float4* __restrict__ stats, double* __restrict__ sums) {
  pdl_wait();
  pdl_trigger();
  __shared__ double s_warp[4];
  const int lane = threadIdx.x % 32;
  double sum = 0.0;
  for (int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 32; row < rows; row += (int64_t)gridDim.x * 4) {
    // A lane without a stretch adds nothing: -inf at an index behind all.
    RowStat r{neg_inf(), 0.0f, 0.0f, 0.0f, 0xffffffffu};
    for (int i = lane; i < parts; i += 32) {
      const float4 v = stat[row * parts + i];
      r = join<true>(r, RowStat{v.x, v.y, v.z, v.w, stat_a[row * parts + i]});
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) r = shuffle_join<true>(r, d, 32);
    const bool valid = any_code<32>(codes, row, bag, C, lane);
    if (lane == 0) sum += (double)finish(r, valid, stats ? stats + row : nullptr);
  }
  sum = block_total(sum, s_warp);
  if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

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

// dz_c = g coef p_c ((n_c - n_a) - dr)
template <typename T, int VEC>
__device__ __forceinline__ void balance_grad(float k, float4 st, int len, int lanes, int lane, bool on,
                                             const T* __restrict__ p, const float* __restrict__ counts,
                                             T* __restrict__ dz) {
  float z[kRowElems];
  load_row<VEC>(p, len, lanes, lane, z);
  const float f = k * st.y;
  constexpr int P = VEC == 1 ? 1 : 4;  // counts that one load brings
#pragma unroll
  for (int k0 = 0; k0 < kRowElems; k0 += P) {
    float n[P];
    const int c = row_index<VEC>(lanes, lane, k0);
    if constexpr (P == 4) {
      const float4 q = c < len ? *reinterpret_cast<const float4*>(counts + c) : make_float4(0.f, 0.f, 0.f, 0.f);
      n[0] = q.x, n[1] = q.y, n[2] = q.z, n[3] = q.w;
    } else {
      n[0] = c < len ? counts[c] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float e = ex2_approx((z[k0 + i] - st.x) * kLog2e);
      z[k0 + i] = f * e * ((n[i] - st.w) - st.z);
    }
  }
  if (st.y == 0.0f) {  // takes no part (m may be -inf)
#pragma unroll
    for (int i = 0; i < kRowElems; ++i) z[i] = 0.0f;
  }
  if (on) store_row<VEC>(dz, len, lanes, lane, z);
}

template <typename T, int VEC, int L>
__global__ void __launch_bounds__(kGroupThreads)
    k_balance_bwd_group(int64_t rows, int C, const T* __restrict__ logits, int64_t stride,
                        const float4* __restrict__ stats, const float* __restrict__ state,
                        const float* __restrict__ g_loss, T* __restrict__ g_logits) {
  pdl_wait();
  pdl_trigger();
  const float k = *g_loss * state[0];
  const int64_t mine = ((int64_t)blockIdx.x * kGroupThreads + threadIdx.x) / L;
  const bool on = mine < rows;
  const int64_t row = on ? mine : rows - 1;
  balance_grad<T, VEC>(k, stats[row], C, L, threadIdx.x % L, on, logits + row * stride, state + kStateHead,
                       g_logits + row * C);
}

template <typename T, int VEC, int W>
__global__ void __launch_bounds__(W * 32)
    k_balance_bwd_block(int64_t items, int64_t C, int parts, int part_len, const T* __restrict__ logits,
                        int64_t stride, const float4* __restrict__ stats, const float* __restrict__ state,
                        const float* __restrict__ g_loss, T* __restrict__ g_logits) {
  pdl_wait();
  pdl_trigger();
  const float k = *g_loss * state[0];
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = parts == 1 ? item : item / parts;
    const int c0 = (int)(item - row * parts) * part_len;
    const int len = (int)min((int64_t)part_len, C - c0);
    balance_grad<T, VEC>(k, stats[row], len, W * 32, threadIdx.x, true, logits + row * stride + c0,
                         state + kStateHead + c0, g_logits + row * C + c0);
  }
}

struct BalanceScratch {
  CountParts count;
  double* sums = nullptr;
  float4* stat = nullptr;
  uint32_t* stat_a = nullptr;
};
BalanceScratch carve(Carver& ws, int64_t rows, const RowPlan& plan) {
  BalanceScratch b;
  b.count.codes = ws.take<uint32_t>(kCountBlocks);
  b.count.rows = ws.take<uint32_t>(kCountBlocks);
  b.sums = ws.take<double>(kBalanceBlocks);
  if (plan.lanes == 0 && plan.parts > 1) {
    b.stat = ws.take<float4>((size_t)rows * plan.parts);
    b.stat_a = ws.take<uint32_t>((size_t)rows * plan.parts);
  }
  return b;
}

}  // namespace
}  // namespace gsb

using namespace gsb;

extern "C" int64_t gsb_code_balance_state_floats(int64_t codebook_rows) {
  return codebook_rows <= 0 ? 0 : kStateHead + padded(codebook_rows);
}

extern "C" size_t gsb_code_balance_workspace_size(int64_t rows, int64_t codebook_rows) {
  if (check_rows(GSB_DTYPE_F32, rows, codebook_rows, 0, 4) != GSB_OK) return 0;
  Carver c(nullptr);
  carve(c, rows, row_plan(std::max<int64_t>(rows, 1), codebook_rows));
  return c.off;
}

extern "C" int gsb_code_balance_forward(int32_t dtype, int64_t rows, int64_t codebook_rows, int32_t bag,
                                        const void* logits, int64_t logits_stride, const void* codes,
                                        int32_t code_bytes, float* loss, int32_t* counts, float* stats, float* state,
                                        uint32_t* status, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_rows(dtype, rows, codebook_rows, logits_stride, code_bytes);
  if (rc != GSB_OK) return rc;
  if (bag <= 0) return GSB_ERR_INVALID_ARGUMENT;
  if (rows >= (int64_t(1) << 31) / bag) return GSB_ERR_CAPACITY;
  if (!loss || !counts || !state || !status || (rows > 0 && (!logits || !codes))) return GSB_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < gsb_code_balance_workspace_size(rows, codebook_rows)) return GSB_ERR_WORKSPACE;
  if (rows == 1) logits_stride = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const RowPlan plan = row_plan(std::max<int64_t>(rows, 1), codebook_rows);
  Carver ws(workspace);
  const BalanceScratch b = carve(ws, rows, plan);
  const Codes cd{codes, code_bytes == 8};
  float* counts_f32 = state + kStateHead;
  // The counts.
  const bool shared = codebook_rows <= kCountSharedCodes;
  const int64_t slots = rows * bag;
  unsigned count_blocks = 1;
  if (shared && slots <= kCountFew) {
    launch_pdl(k_code_counts<true, true>, 1, 512, sizeof(int) * (size_t)codebook_rows, s, rows, bag,
               (int)codebook_rows, cd, counts, counts_f32, b.count, status);
    note_launches(1);
  } else {
    if (cudaMemsetAsync(counts, 0, sizeof(int32_t) * (size_t)codebook_rows, s) != cudaSuccess) return GSB_ERR_CUDA;
    count_blocks = (unsigned)std::min<int64_t>(kCountBlocks, grid1d(rows, 512));
    if (shared)
      launch_pdl(k_code_counts<true, false>, count_blocks, 512, sizeof(int) * (size_t)codebook_rows, s, rows, bag,
                 (int)codebook_rows, cd, counts, counts_f32, b.count, status);
    else
      launch_pdl(k_code_counts<false, false>, count_blocks, 512, 0, s, rows, bag, (int)codebook_rows, cd, counts,
                 counts_f32, b.count, status);
    launch_pdl(k_counts_f32, grid1d(padded(codebook_rows), 256), 256, 0, s, codebook_rows, (const int32_t*)counts,
               counts_f32);
    note_launches(2);
  }
  // The rows.
  int blocks = 0;
  if (rows > 0) {
    with_rows(dtype, rows_wide(dtype, logits, logits_stride), [&](auto t, auto vec) {
      using T = decltype(t);
      constexpr int VEC = decltype(vec)::value;
      const T* z = (const T*)logits;
      if (plan.lanes > 0) {
        with_lanes(plan.lanes, [&](auto l) {
          constexpr int L = decltype(l)::value;
          blocks = std::min(kBalanceBlocks, grid1d(rows * L, kGroupThreads));
          launch_pdl(k_balance_group<T, VEC, L>, blocks, kGroupThreads, 0, s, rows, (int)codebook_rows, bag, z,
                     logits_stride, cd, (const float*)counts_f32, (float4*)stats, b.sums);
        });
      } else {
        with_warps(plan.warps, [&](auto w) {
          constexpr int W = decltype(w)::value;
          const int64_t items = rows * plan.parts;
          blocks = (int)std::min<int64_t>(plan.parts == 1 ? kBalanceBlocks : (int64_t(1) << 31) - 1, items);
          launch_pdl(k_balance_block<T, VEC, W>, blocks, W * 32, 0, s, items, codebook_rows, bag, plan.parts,
                     plan.part_len, z, logits_stride, cd, (const float*)counts_f32, (float4*)stats, b.stat, b.stat_a,
                     b.sums);
        });
        if (plan.parts > 1) {
          blocks = std::min(kBalanceBlocks, grid1d(rows, 4));
          launch_pdl(k_balance_join, blocks, 128, 0, s, rows, codebook_rows, bag, plan.parts, cd,
                     (const float4*)b.stat, (const uint32_t*)b.stat_a, (float4*)stats, b.sums);
          note_launches(1);
        }
      }
    });
    note_launches(1);
  }
  launch_pdl(k_balance_loss, 1, 256, 0, s, blocks, codebook_rows, (const double*)b.sums, (int)count_blocks, b.count,
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
  if (rows == 1) logits_stride = 0;
  const RowPlan plan = row_plan(rows, codebook_rows);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Wide pieces where both the logits' and the gradient's rows are whole ones.
  const bool wide = rows_wide(dtype, logits, logits_stride) && rows_wide(dtype, g_logits, codebook_rows);
  with_rows(dtype, wide, [&](auto t, auto vec) {
    using T = decltype(t);
    constexpr int VEC = decltype(vec)::value;
    if (plan.lanes > 0) {
      with_lanes(plan.lanes, [&](auto l) {
        constexpr int L = decltype(l)::value;
        launch_pdl(k_balance_bwd_group<T, VEC, L>, grid1d(rows * L, kGroupThreads), kGroupThreads, 0, s, rows,
                   (int)codebook_rows, (const T*)logits, logits_stride, (const float4*)stats, state, g_loss,
                   (T*)g_logits);
      });
    } else {
      with_warps(plan.warps, [&](auto w) {
        constexpr int W = decltype(w)::value;
        launch_pdl(k_balance_bwd_block<T, VEC, W>, item_grid(rows * plan.parts), W * 32, 0, s, rows * plan.parts,
                   codebook_rows, plan.parts, plan.part_len, (const T*)logits, logits_stride, (const float4*)stats,
                   state, g_loss, (T*)g_logits);
      });
    }
  });
  note_launches(1);
  return cuda_status(cudaGetLastError());
}
