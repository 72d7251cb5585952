// Row-wise operators on assignment logits z [G, C]: the log probability of a
// given code with the row's entropy and largest alternatives, and the loss that
// keeps the codes in even use, each with its gradient.
//
// Both are sums over a row of e_c = exp(z_c - m), m = max z. The largest value
// (the first one, at a) contributes exactly 1 and is left out of the sums:
//   s' = sum_{c != a} e_c         p_c = e_c / (1 + s')
//   log p_c = (z_c - m) - log1p(s')
//   mu = sum_{c != a} e_c (z_c - m) / (1 + s')     H = log1p(s') - mu
//   dr = sum_{c != a} e_c (n_c - n_a) / (1 + s')   sum_c p_c n_c = n_a + dr
// so that log p, 1 - p, H and n_c - sum p n keep their relative accuracy when
// one probability is close to 1. fp32 throughout; one rounding at the end.
//
// A -inf logit has probability 0. In a row of -inf only log p is -inf, H and the
// gradients are 0. NaN or +inf make a row's values NaN.
#include "code_types.cuh"

namespace gsb {
namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7fc00000); }
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Order of the alternatives as one unsigned number: larger values first, then
// lower indices; -0 equals +0 and NaN comes last. Never 0.
__device__ __forceinline__ uint64_t order_key(float z, uint32_t c) {
  uint32_t u = __float_as_uint(z);
  if ((u & 0x7fffffffu) == 0u) u = 0u;
  uint32_t k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  if ((u & 0x7fffffffu) > 0x7f800000u) k = 0u;
  return ((uint64_t)k << 32) | (uint32_t)~c;
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return ~(uint32_t)key; }

__device__ __forceinline__ uint64_t block_max(uint64_t v, uint64_t* s_warp) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t u = __shfl_xor_sync(kFullMask, v, o);
    v = u > v ? u : v;
  }
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s_warp[0];
#pragma unroll
  for (int w = 1; w < kRowWarps; ++w) v = s_warp[w] > v ? s_warp[w] : v;
  __syncthreads();
  return v;
}
__device__ __forceinline__ float block_sum(float v, float* s_warp) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) v += s_warp[w];
  __syncthreads();
  return v;
}

struct RowSmem {
  uint64_t key[kRowWarps];
  float sum[kRowWarps];
};

// Largest key of the row below `limit`, and whether the row holds a NaN or +inf.
template <typename T>
__device__ __forceinline__ uint64_t row_best(const T* __restrict__ z, int64_t C, uint64_t limit, RowSmem& sm) {
  uint64_t best = 0;
  for (int64_t c = threadIdx.x; c < C; c += kRowThreads) {
    const uint64_t k = order_key(to_f32(z[c]), (uint32_t)c);
    if (k < limit && k > best) best = k;
  }
  return block_max(best, sm.key);
}

// One block per row. stats [rows, 4]: m, s', mu, unused.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
    k_log_probs(int64_t rows, int64_t C, const T* __restrict__ logits, int64_t stride, Codes codes, int top_k,
                float* __restrict__ log_probs, float* __restrict__ entropy, float* __restrict__ top_log_probs,
                int32_t* __restrict__ top_codes, float4* __restrict__ stats, uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  __shared__ RowSmem sm;
  for (int64_t g = blockIdx.x; g < rows; g += gridDim.x) {
    const T* z = logits + g * stride;
    const uint64_t first = row_best(z, C, ~uint64_t(0), sm);
    const uint32_t a = key_index(first);
    const float m = to_f32(z[a]);
    const bool empty = m == neg_inf();
    float s = 0.0f, t = 0.0f;
    for (int64_t c = threadIdx.x; c < C; c += kRowThreads) {
      if (c == a) continue;
      const float x = to_f32(z[c]) - m;
      if (x == neg_inf()) continue;
      const float e = ex2(x * kLog2e);
      s += e;
      t = fmaf(e, x, t);
    }
    s = block_sum(s, sm.sum);
    t = block_sum(t, sm.sum);
    if (!(fabsf(m) <= 3.402823466e38f)) s = quiet_nan();
    const float mu = t / (1.0f + s);
    const float ls = log1pf(s);
    if (threadIdx.x == 0) {
      entropy[g] = empty ? 0.0f : ls - mu;
      if (stats) stats[g] = make_float4(m, s, mu, 0.0f);
      if (log_probs) {
        const int64_t c = codes.at(g);
        if (c >= C) bad_code(status, kSiteCode);
        log_probs[g] = (c < 0 || c >= C) ? 0.0f : empty ? neg_inf() : (to_f32(z[c]) - m) - ls;
      }
    }
    uint64_t limit = ~uint64_t(0);
    for (int j = 0; j < top_k; ++j) {
      limit = j == 0 ? first : row_best(z, C, limit, sm);
      if (threadIdx.x == 0) {
        const uint32_t c = key_index(limit);
        top_codes[g * top_k + j] = (int32_t)c;
        top_log_probs[g * top_k + j] = empty ? neg_inf() : (to_f32(z[c]) - m) - ls;
      }
    }
  }
}

// dz_c = p_c (-lead - gH (z_c - m - mu)) + sum_i g_i [c = c_i], lead = sum_i g_i over the
// given code and the alternatives. At the c_i the sum is taken as
// (sum of their g_i) (1 - p_c) - (sum of the other g_i) p_c.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
    k_log_probs_bwd(int64_t rows, int64_t C, const T* __restrict__ logits, int64_t stride, Codes codes, int top_k,
                    const int32_t* __restrict__ top_codes, const float4* __restrict__ stats,
                    const float* __restrict__ g_log_probs, const float* __restrict__ g_entropy,
                    const float* __restrict__ g_top, T* __restrict__ g_logits) {
  pdl_wait();
  pdl_trigger();
  for (int64_t g = blockIdx.x; g < rows; g += gridDim.x) {
    const T* z = logits + g * stride;
    T* dz = g_logits + g * C;
    const float4 st = stats[g];
    const bool empty = st.x == neg_inf();
    const float inv = 1.0f / (1.0f + st.y);
    const int64_t code = g_log_probs ? codes.at(g) : -1;
    const float gl = code >= 0 && code < C ? g_log_probs[g] : 0.0f;
    const float gh = g_entropy ? g_entropy[g] : 0.0f;
    float lead = gl;
    for (int j = 0; j < top_k; ++j) lead += g_top ? g_top[g * top_k + j] : 0.0f;
    auto value = [&](float zc) {
      const float x = zc - st.x;
      const float e = ex2(x * kLog2e);
      return e == 0.0f || empty ? 0.0f : e * inv * (-lead - gh * (x - st.z));
    };
    for (int64_t c = threadIdx.x; c < C; c += kRowThreads) dz[c] = from_f32<T>(value(to_f32(z[c])));
    __syncthreads();
    // The given code and the alternatives: thread j takes alternative j, thread
    // top_k the code where it is none of them.
    if (threadIdx.x <= top_k && !empty) {
      const int j = threadIdx.x;
      bool mine = j < top_k ? g_top != nullptr : (code >= 0 && code < C);
      const int64_t c = j < top_k ? (mine ? top_codes[g * top_k + j] : -1) : code;
      if (j == top_k && g_top)
        for (int i = 0; i < top_k; ++i) mine = mine && top_codes[g * top_k + i] != code;
      if (mine) {
        float own = c == code ? gl : 0.0f, others = c == code ? 0.0f : gl;
        if (g_top)
          for (int i = 0; i < top_k; ++i) {
            if (i == j) own += g_top[g * top_k + i];
            else others += g_top[g * top_k + i];
          }
        const float x = to_f32(z[c]) - st.x;
        const float e = ex2(x * kLog2e);
        const float p = e * inv;
        const float q = x == 0.0f ? st.y * inv : 1.0f - p;  // 1 - p
        const float h = p == 0.0f ? 0.0f : gh * p * (x - st.z);
        dz[c] = from_f32<T>(own * q - others * p - h);
      }
    }
  }
}

// totals: codes counted, rows with at least one.
__global__ void __launch_bounds__(256)
    k_code_counts(int64_t rows, int bag, int64_t C, Codes codes, int32_t* __restrict__ counts,
                  uint32_t* __restrict__ totals, uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  const int64_t g = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  uint32_t some = 0;
  if (g < rows)
    for (int j = 0; j < bag; ++j) {
      const int64_t c = codes.at(g * bag + j);
      if (c >= C) bad_code(status, kSiteCode);
      if (c >= 0 && c < C) {
        atomicAdd(&counts[c], 1);
        ++some;
      }
    }
  const uint32_t sum = __reduce_add_sync(kFullMask, some);
  const uint32_t valid = __popc(__ballot_sync(kFullMask, some != 0));
  if ((threadIdx.x & 31) == 0 && sum) {
    atomicAdd(&totals[0], sum);
    atomicAdd(&totals[1], valid);
  }
}

__device__ __forceinline__ bool any_code(const Codes& codes, int64_t g, int bag, int64_t C) {
  bool some = false;
  for (int j = 0; j < bag; ++j) {
    const int64_t c = codes.at(g * bag + j);
    some = some || (c >= 0 && c < C);
  }
  return some;
}

// One block per row. stats [rows, 4]: m, 1 / (1 + s') (0 for a row without a
// code or with nothing left), dr, n_a; d[g] = sum_c p_c n_c.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
    k_balance(int64_t rows, int64_t C, int bag, const T* __restrict__ logits, int64_t stride, Codes codes,
              const int32_t* __restrict__ counts, float* __restrict__ d, float4* __restrict__ stats) {
  pdl_wait();
  pdl_trigger();
  __shared__ RowSmem sm;
  for (int64_t g = blockIdx.x; g < rows; g += gridDim.x) {
    const T* z = logits + g * stride;
    const uint64_t first = row_best(z, C, ~uint64_t(0), sm);
    const uint32_t a = key_index(first);
    const float m = to_f32(z[a]);
    const int32_t na = counts[a];
    float s = 0.0f, u = 0.0f;
    for (int64_t c = threadIdx.x; c < C; c += kRowThreads) {
      if (c == a) continue;
      const float e = ex2((to_f32(z[c]) - m) * kLog2e);
      s += e;
      u = fmaf(e, (float)(counts[c] - na), u);
    }
    s = block_sum(s, sm.sum);
    u = block_sum(u, sm.sum);
    if (!(fabsf(m) <= 3.402823466e38f)) s = quiet_nan();
    if (threadIdx.x == 0) {
      const bool out = m == neg_inf() || !any_code(codes, g, bag, C);
      const float inv = out ? 0.0f : 1.0f / (1.0f + s);
      const float dr = out ? 0.0f : u * inv;
      d[g] = out ? 0.0f : (float)na + dr;
      if (stats) stats[g] = make_float4(m, inv, dr, (float)na);
    }
  }
}

// coef = C / (valid rows x codes counted); loss = coef sum_g d[g], in 64 bits.
__global__ void __launch_bounds__(1024)
    k_balance_loss(int64_t rows, int64_t C, const float* __restrict__ d, const uint32_t* __restrict__ totals,
                   float* __restrict__ loss, float* __restrict__ coef) {
  pdl_wait();
  pdl_trigger();
  __shared__ double s_sum[1024];
  double v = 0.0;
  for (int64_t g = threadIdx.x; g < rows; g += 1024) v += (double)d[g];
  s_sum[threadIdx.x] = v;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if (threadIdx.x < o) s_sum[threadIdx.x] += s_sum[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const double k = totals[1] ? (double)C / ((double)totals[0] * (double)totals[1]) : 0.0;
    *loss = (float)(k * s_sum[0]);
    *coef = (float)k;
  }
}

// dz_c = g coef p_c ((n_c - n_a) - dr).
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
    k_balance_bwd(int64_t rows, int64_t C, const T* __restrict__ logits, int64_t stride,
                  const int32_t* __restrict__ counts, const float4* __restrict__ stats,
                  const float* __restrict__ coef, const float* __restrict__ g_loss, T* __restrict__ g_logits) {
  pdl_wait();
  pdl_trigger();
  const float k = *g_loss * *coef;
  for (int64_t g = blockIdx.x; g < rows; g += gridDim.x) {
    const T* z = logits + g * stride;
    const float4 st = stats[g];
    for (int64_t c = threadIdx.x; c < C; c += kRowThreads) {
      const float e = ex2((to_f32(z[c]) - st.x) * kLog2e);
      const float v = k * st.y * e * (((float)counts[c] - st.w) - st.z);
      g_logits[g * C + c] = from_f32<T>(st.y == 0.0f || e == 0.0f ? 0.0f : v);
    }
  }
}

int check_rows(int32_t dtype, int64_t rows, int64_t codes, int64_t stride, int32_t code_bytes) {
  if (!dtype_ok(dtype)) return GSB_ERR_UNSUPPORTED;
  if (rows < 0 || codes <= 0 || stride < 0 || (code_bytes != 4 && code_bytes != 8)) return GSB_ERR_INVALID_ARGUMENT;
  if (codes >= (int64_t(1) << 31) - 1 || rows >= (int64_t(1) << 31)) return GSB_ERR_CAPACITY;
  return GSB_OK;
}

unsigned row_grid(int64_t rows) { return (unsigned)std::min<int64_t>(rows, 1 << 20); }

struct BalanceScratch {
  uint32_t* totals = nullptr;
  float* d = nullptr;
};
BalanceScratch carve(Carver& ws, int64_t rows) {
  BalanceScratch b;
  b.totals = ws.take<uint32_t>(2);
  b.d = ws.take<float>((size_t)rows);
  return b;
}

}  // namespace
}  // namespace gsb

using namespace gsb;

extern "C" int gsb_code_log_probs_forward(int32_t dtype, int64_t rows, int64_t codebook_rows, const void* logits,
                                          int64_t logits_stride, const void* codes, int32_t code_bytes, int32_t top_k,
                                          float* log_probs, float* entropy, float* top_log_probs, int32_t* top_codes,
                                          float* stats, uint32_t* status, void* stream) {
  const int rc = check_rows(dtype, rows, codebook_rows, logits_stride, code_bytes);
  if (rc != GSB_OK) return rc;
  if (top_k < 0 || top_k > GSB_CODE_MAX_TOP || top_k > codebook_rows) return GSB_ERR_INVALID_ARGUMENT;
  if (rows == 0) return GSB_OK;
  if (!logits || !entropy || !status || (log_probs != nullptr) != (codes != nullptr) ||
      (top_k > 0 && (!top_log_probs || !top_codes)))
    return GSB_ERR_INVALID_ARGUMENT;
  const Codes cd{codes, code_bytes == 8};
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    launch_pdl(k_log_probs<T>, row_grid(rows), kRowThreads, 0, static_cast<cudaStream_t>(stream), rows, codebook_rows,
               (const T*)logits, logits_stride, cd, top_k, log_probs, entropy, top_log_probs, top_codes,
               (float4*)stats, status);
  });
  note_launches(1);
  return cuda_status(cudaGetLastError());
}

extern "C" int gsb_code_log_probs_backward(int32_t dtype, int64_t rows, int64_t codebook_rows, const void* logits,
                                           int64_t logits_stride, const void* codes, int32_t code_bytes, int32_t top_k,
                                           const int32_t* top_codes, const float* stats, const float* g_log_probs,
                                           const float* g_entropy, const float* g_top_log_probs, void* g_logits,
                                           void* stream) {
  const int rc = check_rows(dtype, rows, codebook_rows, logits_stride, code_bytes);
  if (rc != GSB_OK) return rc;
  if (top_k < 0 || top_k > GSB_CODE_MAX_TOP || top_k > codebook_rows) return GSB_ERR_INVALID_ARGUMENT;
  if (rows == 0) return GSB_OK;
  if (!logits || !stats || !g_logits || (g_log_probs && !codes) || (g_top_log_probs && top_k > 0 && !top_codes))
    return GSB_ERR_INVALID_ARGUMENT;
  const Codes cd{codes, code_bytes == 8};
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    launch_pdl(k_log_probs_bwd<T>, row_grid(rows), kRowThreads, 0, static_cast<cudaStream_t>(stream), rows,
               codebook_rows, (const T*)logits, logits_stride, cd, g_top_log_probs ? top_k : 0, top_codes,
               (const float4*)stats, g_log_probs, g_entropy, g_top_log_probs, (T*)g_logits);
  });
  note_launches(1);
  return cuda_status(cudaGetLastError());
}

extern "C" size_t gsb_code_balance_workspace_size(int64_t rows, int64_t codebook_rows) {
  if (check_rows(GSB_DTYPE_F32, rows, codebook_rows, 0, 4) != GSB_OK) return 0;
  Carver c(nullptr);
  carve(c, rows);
  return c.off + 256;
}

extern "C" int gsb_code_balance_forward(int32_t dtype, int64_t rows, int64_t codebook_rows, int32_t bag,
                                        const void* logits, int64_t logits_stride, const void* codes,
                                        int32_t code_bytes, float* loss, int32_t* counts, float* stats, float* coef,
                                        uint32_t* status, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_rows(dtype, rows, codebook_rows, logits_stride, code_bytes);
  if (rc != GSB_OK) return rc;
  if (bag <= 0) return GSB_ERR_INVALID_ARGUMENT;
  if (rows >= (int64_t(1) << 31) / bag) return GSB_ERR_CAPACITY;
  if (!loss || !counts || !coef || !status || (rows > 0 && (!logits || !codes))) return GSB_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < gsb_code_balance_workspace_size(rows, codebook_rows)) return GSB_ERR_WORKSPACE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Carver ws(workspace);
  const BalanceScratch b = carve(ws, rows);
  const Codes cd{codes, code_bytes == 8};
  if (cudaMemsetAsync(counts, 0, sizeof(int32_t) * (size_t)codebook_rows, s) != cudaSuccess ||
      cudaMemsetAsync(b.totals, 0, 2 * sizeof(uint32_t), s) != cudaSuccess)
    return GSB_ERR_CUDA;
  if (rows > 0) {
    launch_pdl(k_code_counts, grid1d(rows, 256), 256, 0, s, rows, bag, codebook_rows, cd, counts, b.totals, status);
    with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      launch_pdl(k_balance<T>, row_grid(rows), kRowThreads, 0, s, rows, codebook_rows, bag, (const T*)logits,
                 logits_stride, cd, (const int32_t*)counts, b.d, (float4*)stats);
    });
    note_launches(2);
  }
  launch_pdl(k_balance_loss, 1, 1024, 0, s, rows, codebook_rows, (const float*)b.d, (const uint32_t*)b.totals, loss,
             coef);
  note_launches(1);
  return cuda_status(cudaGetLastError());
}

extern "C" int gsb_code_balance_backward(int32_t dtype, int64_t rows, int64_t codebook_rows, const void* logits,
                                         int64_t logits_stride, const int32_t* counts, const float* stats,
                                         const float* coef, const float* g_loss, void* g_logits, void* stream) {
  const int rc = check_rows(dtype, rows, codebook_rows, logits_stride, 4);
  if (rc != GSB_OK) return rc;
  if (rows == 0) return GSB_OK;
  if (!logits || !counts || !stats || !coef || !g_loss || !g_logits) return GSB_ERR_INVALID_ARGUMENT;
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    launch_pdl(k_balance_bwd<T>, row_grid(rows), kRowThreads, 0, static_cast<cudaStream_t>(stream), rows,
               codebook_rows, (const T*)logits, logits_stride, counts, (const float4*)stats, coef, g_loss,
               (T*)g_logits);
  });
  note_launches(1);
  return cuda_status(cudaGetLastError());
}
