// Log probability of a given code, entropy and largest alternatives of each row of
// assignment logits, and their gradient. The sums are those of code_rows.cuh.
//
// A -inf logit has probability 0. In a row of -inf only log p is -inf, H and the
// gradient are 0. NaN or +inf make a row's results NaN.
#include "code_rows.cuh"

namespace gsb {
namespace {

constexpr int kGroupThreads = 256;
constexpr int kTopList = 256;  // candidates for the alternatives that a block can rank

struct LogProbsOut {
  float *log_probs, *entropy, *top_log_probs;
  int32_t* top_codes;
  float4* stats;  // m, s', mu, unused
};

struct RowResult {
  float m, ls;  // log p_c = (z_c - m) - ls
  bool empty;
  __device__ __forceinline__ float log_p(float z) const { return empty ? neg_inf() : (z - m) - ls; }
};
__device__ __forceinline__ RowResult finish(RowStat& r) {
  if (r.m == __int_as_float(0x7f800000)) r.s = quiet_nan();
  return RowResult{r.m, log1pf(r.s), r.m == neg_inf() && r.s == r.s};
}
// The row's results but for the alternatives; z: the given code's logit.
__device__ __forceinline__ void write_row(const LogProbsOut& o, int64_t row, const RowStat& r, const RowResult& q,
                                          int64_t code, bool given, float z) {
  const float mu = r.w / (1.0f + r.s);
  o.entropy[row] = q.empty ? 0.0f : q.ls - mu;
  if (o.stats) o.stats[row] = make_float4(r.m, r.s, mu, 0.0f);
  if (o.log_probs) o.log_probs[row] = given ? q.log_p(z) : 0.0f;
}
// The given code of a row, -1 where there is none.
__device__ __forceinline__ int64_t given_code(const LogProbsOut& o, const Codes& codes, int64_t row, int64_t C,
                                              bool report, uint32_t* status) {
  if (!o.log_probs) return -1;
  const int64_t c = codes.at(row);
  if (c >= C && report) bad_code(status, kSiteCode);
  return c < C ? c : -1;
}

// Rows of up to 512 codes: L lanes each. The alternatives come one by one: the
// largest of what is left, taken out of its lane's registers (NaN, which loses
// against any number).
template <typename T, int VEC, int L>
__global__ void __launch_bounds__(kGroupThreads)
    k_log_probs_group(int64_t rows, int C, const T* __restrict__ logits, int64_t stride, Codes codes, int top_k,
                      LogProbsOut o, uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % L;
  const int64_t mine = ((int64_t)blockIdx.x * kGroupThreads + threadIdx.x) / L;
  const bool on = mine < rows;
  const int64_t row = on ? mine : rows - 1;  // lanes without a row keep a warp's exchanges whole
  const T* p = logits + row * stride;
  float z[kRowElems];
  load_row<VEC>(p, C, L, lane, z);
  const int64_t code = given_code(o, codes, row, C, on && lane == 0, status);
  const float zc = code >= 0 ? to_f32(p[code]) : 0.0f;
  RowStat r = row_stat<VEC, L, false>(z, C, L, lane, nullptr, [](int) { return 0.0f; });
  const RowResult q = finish(r);
  if (on && lane == 0) write_row(o, row, r, q, code, code >= 0, zc);
  if (top_k == 0) return;
  uint32_t a = r.a, taken = 0;  // taken: a bit for each of the lane's values
  float best = r.m, top = 0.0f;
  int at = 0;  // the lane's own largest, and where it is
  for (int j = 0;; ++j) {
    if (on && lane == 0) {
      o.top_codes[row * top_k + j] = (int32_t)a;
      o.top_log_probs[row * top_k + j] = q.log_p(best);
    }
    if (j + 1 == top_k) break;
    if (j == 0) {  // places behind the row's end are never taken
#pragma unroll
      for (int k = 0; k < kRowElems; ++k)
        if (row_index<VEC>(L, lane, k) >= C) z[k] = quiet_nan(), taken |= 1u << k;
    }
    const bool owner = (int)(a / VEC) % L == lane;
    if (owner || j == 0) {
      const int out = owner ? (int)(a / (VEC * L)) * VEC + (int)a % VEC : kRowElems;
      if (owner) taken |= 1u << out;
#pragma unroll
      for (int k = 0; k < kRowElems; ++k)
        if (k == out) z[k] = quiet_nan();
      top = lane_max(z);
      at = kRowElems;
#pragma unroll
      for (int k = kRowElems - 1; k >= 0; --k)
        if (z[k] == top) at = k;
    }
    best = top;
#pragma unroll
    for (int d = L / 2; d > 0; d >>= 1) best = fmaxf(best, __shfl_xor_sync(kFullMask, best, d, L));
    // NaN: nothing but NaN is left, taken from the lowest index on.
    const int pick = best != best ? __ffs(~taken) - 1 : (top == best ? at : -1);
    a = pick >= 0 && pick < kRowElems ? (uint32_t)row_index<VEC>(L, lane, pick) : 0x7fffffffu;
#pragma unroll
    for (int d = L / 2; d > 0; d >>= 1) a = min(a, __shfl_xor_sync(kFullMask, a, d, L));
  }
}

// Block-wide largest key below `limit` among the registers' values.
template <int VEC, int W>
__device__ __forceinline__ uint64_t block_best(const float (&z)[kRowElems], int len, int c0, uint64_t limit,
                                               uint64_t* s_key) {
  uint64_t best = 0;
#pragma unroll
  for (int k = 0; k < kRowElems; ++k) {
    const int c = row_index<VEC>(W * 32, threadIdx.x, k);
    const uint64_t key = order_key(z[k], (uint32_t)(c0 + c));
    if (c < len && key < limit && key > best) best = key;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const uint64_t u = __shfl_xor_sync(kFullMask, best, d);
    best = u > best ? u : best;
  }
  if (W > 1) {
    __syncthreads();
    if (threadIdx.x % 32 == 0) s_key[threadIdx.x / 32] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) best = s_key[w] > best ? s_key[w] : best;
  }
  return best;
}

// One block of W warps per stretch. The alternatives: k lanes hold a value of at
// least the k-th largest of a warp's lane maxima, so none of the k largest is below
// the largest of those bounds over the warps; the few values that are not (k and a
// handful) are listed and ranked against one another. Many equal values can overrun
// the list: then the alternatives are found one by one. parts > 1: the stretch's
// sums and keys go to `stat` and `keys` for k_log_probs_join.
template <typename T, int VEC, int W>
__global__ void __launch_bounds__(W * 32)
    k_log_probs_block(int64_t items, int64_t C, int parts, int part_len, const T* __restrict__ logits, int64_t stride,
                      Codes codes, int top_k, LogProbsOut o, float4* __restrict__ stat, uint64_t* __restrict__ keys,
                      uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  __shared__ RowStat s_stat[W];
  __shared__ uint32_t s_bound[W];
  __shared__ uint64_t s_list[kTopList];
  __shared__ uint64_t s_key[W];
  __shared__ RowResult s_result;
  __shared__ int s_count;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = parts == 1 ? item : item / parts;
    const int part = (int)(item - row * parts);
    const int c0 = part * part_len;
    const int len = (int)min((int64_t)part_len, C - c0);
    const T* p = logits + row * stride;
    float z[kRowElems];
    load_row<VEC>(p + c0, len, W * 32, tid, z);
    int64_t code = -1;
    float zc = 0.0f;
    if (parts == 1 && warp == 0) {
      code = given_code(o, codes, row, C, lane == 0, status);
      zc = code >= 0 ? to_f32(p[code]) : 0.0f;
    }
    RowStat r = row_stat<VEC, 32, false>(z, len, W * 32, tid, nullptr, [](int) { return 0.0f; });
    r.a += (uint32_t)c0;
    const int k = min(top_k, len);
    if (k > 1) {
      uint32_t left = order_bits(lane_max(z)), bound = 0;
      for (int j = 0; j < k; ++j) {
        bound = __reduce_max_sync(kFullMask, left);
        const uint32_t who = __ballot_sync(kFullMask, left == bound);
        if (lane == __ffs(who) - 1) left = 0;
      }
      if (lane == 0) s_bound[warp] = bound;
    }
    if (tid == 0) s_count = 0;
    if (lane == 0) s_stat[warp] = r;
    __syncthreads();
    RowResult q;
    if (warp == 0) {
      if (W > 1) {
        r = s_stat[lane % W];
#pragma unroll
        for (int d = W / 2; d > 0; d >>= 1) r = shuffle_join<false>(r, d, W);
      }
      if (parts == 1) {
        q = finish(r);
        if (lane == 0) {
          write_row(o, row, r, q, code, code >= 0, zc);
          s_result = q;
          if (k == 1) {
            o.top_codes[row] = (int32_t)r.a;
            o.top_log_probs[row] = q.log_p(r.m);
          }
        }
      } else if (lane == 0) {
        stat[item] = make_float4(r.m, r.s, r.w, __uint_as_float(r.a));
        if (k == 1 && top_k == 1) keys[item] = order_key(r.m, r.a);
      }
    }
    if (top_k > 1) {
      uint32_t bound = 0;
      if (k > 1) {
#pragma unroll
        for (int w = 0; w < W; ++w) bound = max(bound, s_bound[w]);
      }
      const float least = key_value((uint64_t)bound << 32);
#pragma unroll
      for (int i = 0; i < kRowElems; ++i) {
        if (z[i] >= least) {
          const int c = row_index<VEC>(W * 32, tid, i);
          if (c < len) {
            const int at = atomicAdd(&s_count, 1);
            if (at < kTopList) s_list[at] = order_key(z[i], (uint32_t)(c0 + c));
          }
        }
      }
      __syncthreads();
      const int count = s_count;
      auto put = [&](int j, uint64_t key) {
        if (parts == 1) {
          const RowResult f = s_result;
          o.top_codes[row * top_k + j] = (int32_t)key_index(key);
          o.top_log_probs[row * top_k + j] = f.log_p(key_value(key));
        } else {
          keys[item * top_k + j] = key;
        }
      };
      if (count >= k && count <= kTopList) {
        for (int i = tid; i < count; i += W * 32) {
          const uint64_t key = s_list[i];
          int rank = 0;
          for (int j = 0; j < count; ++j) rank += s_list[j] > key;
          if (rank < k) put(rank, key);
        }
      } else {
        uint64_t limit = ~uint64_t(0);
        for (int j = 0; j < k; ++j) {
          limit = block_best<VEC, W>(z, len, c0, limit, s_key);
          if (tid == 0) put(j, limit);
        }
      }
      if (parts > 1)
        for (int j = k + tid; j < top_k; j += W * 32) keys[item * top_k + j] = 0;  // a short last stretch
    }
    __syncthreads();
  }
}

// One warp per row joins its stretches' sums and picks the largest keys.
template <typename T>
__global__ void __launch_bounds__(128)
    k_log_probs_join(int64_t rows, int64_t C, int parts, const T* __restrict__ logits, int64_t stride, Codes codes,
                     int top_k, const float4* __restrict__ stat, const uint64_t* __restrict__ keys, LogProbsOut o,
                     uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % 32;
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  if (row >= rows) return;
  const int64_t code = given_code(o, codes, row, C, lane == 0, status);
  const float zc = code >= 0 ? to_f32(logits[row * stride + code]) : 0.0f;
  const float4* st = stat + row * parts;
  auto stat_at = [&](int i) {
    const float4 v = st[i];
    return RowStat{v.x, v.y, v.z, 0.0f, __float_as_uint(v.w)};
  };
  // A lane without a stretch adds nothing: -inf at an index behind all.
  RowStat r{neg_inf(), 0.0f, 0.0f, 0.0f, 0xffffffffu};
  for (int i = lane; i < parts; i += 32) r = join<false>(r, stat_at(i));
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) r = shuffle_join<false>(r, d, 32);
  const RowResult q = finish(r);
  if (lane == 0) write_row(o, row, r, q, code, code >= 0, zc);
  const uint64_t* ks = keys + row * parts * top_k;
  const int n = parts * top_k;
  uint64_t limit = ~uint64_t(0);
  for (int j = 0; j < top_k; ++j) {
    uint64_t best = 0;
    for (int i = lane; i < n; i += 32) {
      const uint64_t key = ks[i];
      if (key < limit && key > best) best = key;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      const uint64_t u = __shfl_xor_sync(kFullMask, best, d);
      best = u > best ? u : best;
    }
    limit = best;
    if (lane == 0) {
      o.top_codes[row * top_k + j] = (int32_t)key_index(best);
      o.top_log_probs[row * top_k + j] = q.log_p(key_value(best));
    }
  }
}

struct LogProbsIn {
  Codes codes;
  int top_k;  // 0 where the alternatives have no gradient
  const int32_t* top_codes;
  const float4* stats;
  const float *g_log_probs, *g_entropy, *g_top;
};

// dz_c = p_c (-lead - gH (z_c - m - mu)) + sum_i g_i [c = c_i], lead = sum_i g_i over the
// given code and the alternatives. At the c_i, which are written a second time, the sum
// is (sum of their g_i) (1 - p_c) - (sum of the other g_i) p_c.
// `lane` of `lanes` takes its values of a stretch at c0; sync() orders the two writes.
template <typename T, int VEC, typename Sync>
__device__ __forceinline__ void log_probs_grad(int64_t row, int64_t C, int c0, int len, int lanes, int lane, bool on,
                                               const T* __restrict__ p, T* __restrict__ dz, const LogProbsIn& in,
                                               Sync&& sync) {
  float z[kRowElems];
  load_row<VEC>(p + c0, len, lanes, lane, z);
  const float4 st = in.stats[row];
  const bool empty = st.x == neg_inf() && st.y == st.y;
  const float inv = 1.0f / (1.0f + st.y);
  int64_t code = in.g_log_probs ? in.codes.at(row) : -1;
  if (code >= C) code = -1;
  const float gl = code >= 0 ? in.g_log_probs[row] : 0.0f;
  const float gh = in.g_entropy ? in.g_entropy[row] : 0.0f;
  const int k = in.top_k;
  const int32_t* tc = in.top_codes + row * k;
  const float* gt = in.g_top + row * k;
  float lead = gl;
  for (int j = 0; j < k; ++j) lead += gt[j];
  // p (-lead - gH (x - mu)) = e (alpha + beta x)
  const float beta = -gh * inv, alpha = (gh * st.z - lead) * inv;
#pragma unroll
  for (int i = 0; i < kRowElems; ++i) {
    const float x = max_nan(z[i] - st.x, -200.0f);  // -inf: e is 0, and beta x finite
    z[i] = ex2_approx(x * kLog2e) * fmaf(beta, x, alpha);
  }
  if (empty) {
#pragma unroll
    for (int i = 0; i < kRowElems; ++i) z[i] = 0.0f;
  }
  if (on) store_row<VEC>(dz + c0, len, lanes, lane, z);
  sync();
  if (!on || empty) return;
  for (int j = lane; j <= k; j += lanes) {
    const int64_t c = j < k ? (int64_t)tc[j] : code;
    bool own_place = c >= c0 && c < c0 + len;
    if (j == k)  // the given code, where it is none of the alternatives
      for (int i = 0; i < k; ++i) own_place = own_place && (int64_t)tc[i] != code;
    if (!own_place) continue;
    float own = c == code ? gl : 0.0f, others = c == code ? 0.0f : gl;
    for (int i = 0; i < k; ++i) {
      if (i == j) own += gt[i];
      else others += gt[i];
    }
    const float x = to_f32(p[c]) - st.x;
    const float pr = ex2_approx(x * kLog2e) * inv;
    const float not_p = x == 0.0f ? st.y * inv : 1.0f - pr;
    const float h = pr == 0.0f ? 0.0f : gh * pr * (x - st.z);
    dz[c] = from_f32<T>(own * not_p - others * pr - h);
  }
}

template <typename T, int VEC, int L>
__global__ void __launch_bounds__(kGroupThreads)
    k_log_probs_bwd_group(int64_t rows, int C, const T* __restrict__ logits, int64_t stride, LogProbsIn in,
                          T* __restrict__ g_logits) {
  pdl_wait();
  pdl_trigger();
  const int64_t mine = ((int64_t)blockIdx.x * kGroupThreads + threadIdx.x) / L;
  const bool on = mine < rows;
  const int64_t row = on ? mine : rows - 1;
  log_probs_grad<T, VEC>(row, C, 0, C, L, threadIdx.x % L, on, logits + row * stride, g_logits + row * C, in,
                         [] { __syncwarp(); });
}

template <typename T, int VEC, int W>
__global__ void __launch_bounds__(W * 32)
    k_log_probs_bwd_block(int64_t items, int64_t C, int parts, int part_len, const T* __restrict__ logits,
                          int64_t stride, LogProbsIn in, T* __restrict__ g_logits) {
  pdl_wait();
  pdl_trigger();
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = parts == 1 ? item : item / parts;
    const int c0 = (int)(item - row * parts) * part_len;
    const int len = (int)min((int64_t)part_len, C - c0);
    log_probs_grad<T, VEC>(row, C, c0, len, W * 32, threadIdx.x, true, logits + row * stride, g_logits + row * C, in,
                           [] { __syncthreads(); });
  }
}

struct LogProbsScratch {
  float4* stat = nullptr;
  uint64_t* keys = nullptr;
};
LogProbsScratch carve(Carver& ws, int64_t rows, const RowPlan& plan, int top_k) {
  LogProbsScratch b;
  if (plan.lanes == 0 && plan.parts > 1) {
    b.stat = ws.take<float4>((size_t)rows * plan.parts);
    b.keys = ws.take<uint64_t>((size_t)rows * plan.parts * top_k);
  }
  return b;
}

int check_log_probs(int32_t dtype, int64_t rows, int64_t codes, int64_t stride, int32_t code_bytes, int32_t top_k) {
  const int rc = check_rows(dtype, rows, codes, stride, code_bytes);
  if (rc != GSB_OK) return rc;
  return top_k < 0 || top_k > GSB_CODE_MAX_TOP || top_k > codes ? GSB_ERR_INVALID_ARGUMENT : GSB_OK;
}

}  // namespace
}  // namespace gsb

using namespace gsb;

extern "C" size_t gsb_code_log_probs_workspace_size(int64_t rows, int64_t codebook_rows, int32_t top_k) {
  if (check_log_probs(GSB_DTYPE_F32, rows, codebook_rows, 0, 4, top_k) != GSB_OK || rows == 0) return 0;
  Carver c(nullptr);
  carve(c, rows, row_plan(rows, codebook_rows), top_k);
  return c.off;
}

extern "C" int gsb_code_log_probs_forward(int32_t dtype, int64_t rows, int64_t codebook_rows, const void* logits,
                                          int64_t logits_stride, const void* codes, int32_t code_bytes, int32_t top_k,
                                          float* log_probs, float* entropy, float* top_log_probs, int32_t* top_codes,
                                          float* stats, uint32_t* status, void* workspace, size_t workspace_bytes,
                                          void* stream) {
  const int rc = check_log_probs(dtype, rows, codebook_rows, logits_stride, code_bytes, top_k);
  if (rc != GSB_OK) return rc;
  if (rows == 0) return GSB_OK;
  if (!logits || !entropy || !status || (log_probs != nullptr) != (codes != nullptr) ||
      (top_k > 0 && (!top_log_probs || !top_codes)))
    return GSB_ERR_INVALID_ARGUMENT;
  const size_t need = gsb_code_log_probs_workspace_size(rows, codebook_rows, top_k);
  if (need > 0 && (!workspace || workspace_bytes < need)) return GSB_ERR_WORKSPACE;
  if (rows == 1) logits_stride = 0;
  const RowPlan plan = row_plan(rows, codebook_rows);
  Carver ws(workspace);
  const LogProbsScratch b = carve(ws, rows, plan, top_k);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Codes cd{codes, code_bytes == 8};
  const LogProbsOut o{log_probs, entropy, top_log_probs, top_codes, (float4*)stats};
  with_rows(dtype, rows_wide(dtype, logits, logits_stride), [&](auto t, auto vec) {
    using T = decltype(t);
    constexpr int VEC = decltype(vec)::value;
    const T* z = (const T*)logits;
    if (plan.lanes > 0) {
      with_lanes(plan.lanes, [&](auto l) {
        constexpr int L = decltype(l)::value;
        launch_pdl(k_log_probs_group<T, VEC, L>, grid1d(rows * L, kGroupThreads), kGroupThreads, 0, s, rows,
                   (int)codebook_rows, z, logits_stride, cd, top_k, o, status);
      });
    } else {
      with_warps(plan.warps, [&](auto w) {
        constexpr int W = decltype(w)::value;
        launch_pdl(k_log_probs_block<T, VEC, W>, item_grid(rows * plan.parts), W * 32, 0, s, rows * plan.parts,
                   codebook_rows, plan.parts, plan.part_len, z, logits_stride, cd, top_k, o, b.stat, b.keys, status);
      });
      if (plan.parts > 1) {
        launch_pdl(k_log_probs_join<T>, grid1d(rows * 32, 128), 128, 0, s, rows, codebook_rows, plan.parts, z,
                   logits_stride, cd, top_k, (const float4*)b.stat, (const uint64_t*)b.keys, o, status);
        note_launches(1);
      }
    }
  });
  note_launches(1);
  return cuda_status(cudaGetLastError());
}

extern "C" int gsb_code_log_probs_backward(int32_t dtype, int64_t rows, int64_t codebook_rows, const void* logits,
                                           int64_t logits_stride, const void* codes, int32_t code_bytes, int32_t top_k,
                                           const int32_t* top_codes, const float* stats, const float* g_log_probs,
                                           const float* g_entropy, const float* g_top_log_probs, void* g_logits,
                                           void* stream) {
  const int rc = check_log_probs(dtype, rows, codebook_rows, logits_stride, code_bytes, top_k);
  if (rc != GSB_OK) return rc;
  if (rows == 0) return GSB_OK;
  if (!logits || !stats || !g_logits || (g_log_probs && !codes) || (g_top_log_probs && top_k > 0 && !top_codes))
    return GSB_ERR_INVALID_ARGUMENT;
  if (rows == 1) logits_stride = 0;
  const RowPlan plan = row_plan(rows, codebook_rows);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const LogProbsIn in{Codes{codes, code_bytes == 8}, g_top_log_probs ? top_k : 0, top_codes, (const float4*)stats,
                      g_log_probs, g_entropy, g_top_log_probs};
  // Wide pieces where both the logits' and the gradient's rows are whole ones.
  const bool wide = rows_wide(dtype, logits, logits_stride) && rows_wide(dtype, g_logits, codebook_rows);
  with_rows(dtype, wide, [&](auto t, auto vec) {
    using T = decltype(t);
    constexpr int VEC = decltype(vec)::value;
    if (plan.lanes > 0) {
      with_lanes(plan.lanes, [&](auto l) {
        constexpr int L = decltype(l)::value;
        launch_pdl(k_log_probs_bwd_group<T, VEC, L>, grid1d(rows * L, kGroupThreads), kGroupThreads, 0, s, rows,
                   (int)codebook_rows, (const T*)logits, logits_stride, in, (T*)g_logits);
      });
    } else {
      with_warps(plan.warps, [&](auto w) {
        constexpr int W = decltype(w)::value;
        launch_pdl(k_log_probs_bwd_block<T, VEC, W>, item_grid(rows * plan.parts), W * 32, 0, s, rows * plan.parts,
                   codebook_rows, plan.parts, plan.part_len, (const T*)logits, logits_stride, in, (T*)g_logits);
      });
    }
  });
  note_launches(1);
  return cuda_status(cudaGetLastError());
}
