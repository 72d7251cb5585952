// Lookup of codebook rows and its gradients.
//
//   out[n, :] = scale * sum_j w[n, j] * table[code[n, j], :]
//   g_table[c, :] = scale * sum over (n, j) with code c of w[n, j] * g[n, :]
//   g_w[n, j] = scale * <g[n, :], table[code[n, j], :]>
//
// Sums are fp32, rounded once to the result's type. The table gradient sorts
// the codes (stable radix sort), so each row is a sum in a fixed order: the
// result does not depend on the timing of the blocks.
#include "code_types.cuh"
#include "radix_sort.cuh"

namespace gsb {
namespace {

// One thread per output value.
template <typename T, typename O>
__global__ void __launch_bounds__(256)
    k_lookup(int64_t total, int bag, int64_t C, int dim, const T* __restrict__ table, int64_t stride, Codes codes,
             const float* __restrict__ weights, float scale, O* __restrict__ out, uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const int64_t n = i / dim;
  const int d = (int)(i - n * dim);
  float acc = 0.0f;
  for (int j = 0; j < bag; ++j) {
    const int64_t c = codes.at(n * bag + j);
    if (c < 0) continue;
    if (c >= C) {
      bad_code(status, kSiteCode);
      continue;
    }
    acc = fmaf(weights ? weights[n * bag + j] : 1.0f, to_f32(table[c * stride + d]), acc);
  }
  out[i] = from_f32<O>(acc * scale);
}

// Sort keys: the code, or C for an empty slot (sorted behind every code).
__global__ void __launch_bounds__(256)
    k_code_keys(int64_t n, int64_t C, Codes codes, uint32_t* __restrict__ keys, uint32_t* __restrict__ vals,
                uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t c = codes.at(i);
  if (c >= C) bad_code(status, kSiteCode);
  keys[i] = (c < 0 || c >= C) ? (uint32_t)C : (uint32_t)c;
  vals[i] = (uint32_t)i;
}

// One warp per codebook row: its entries are found by bisection.
template <typename T, typename O>
__global__ void __launch_bounds__(256)
    k_table_grad(int64_t n, int bag, int64_t C, int dim, const uint32_t* __restrict__ keys,
                 const uint32_t* __restrict__ vals, const float* __restrict__ weights, float scale,
                 const O* __restrict__ g, T* __restrict__ g_table) {
  pdl_wait();
  pdl_trigger();
  const int64_t c = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (c >= C) return;
  auto first = [&](uint32_t key) {
    int64_t lo = 0, hi = n;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (keys[mid] < key) lo = mid + 1;
      else hi = mid;
    }
    return lo;
  };
  const int64_t lo = first((uint32_t)c), hi = first((uint32_t)c + 1u);
  for (int d = lane; d < dim; d += 32) {
    float acc = 0.0f;
    for (int64_t k = lo; k < hi; ++k) {
      const uint32_t v = vals[k];
      acc = fmaf(weights ? weights[v] : 1.0f, to_f32(g[(int64_t)(v / (uint32_t)bag) * dim + d]), acc);
    }
    g_table[c * dim + d] = from_f32<T>(acc * scale);
  }
}

// One warp per slot.
template <typename T, typename O>
__global__ void __launch_bounds__(256)
    k_weight_grad(int64_t slots, int bag, int64_t C, int dim, const T* __restrict__ table, int64_t stride, Codes codes,
                  float scale, const O* __restrict__ g, float* __restrict__ g_weights, uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (i >= slots) return;
  const int64_t c = codes.at(i);
  float acc = 0.0f;
  if (c >= C) {
    if (lane == 0) bad_code(status, kSiteCode);
  } else if (c >= 0) {
    const int64_t n = i / bag;
    for (int d = lane; d < dim; d += 32) acc = fmaf(to_f32(g[n * dim + d]), to_f32(table[c * stride + d]), acc);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(kFullMask, acc, o);
  if (lane == 0) g_weights[i] = acc * scale;
}

struct BackwardScratch {
  uint32_t *keys = nullptr, *vals = nullptr, *keys_s = nullptr, *vals_s = nullptr;
};
BackwardScratch carve(Carver& ws, int64_t slots) {
  BackwardScratch b;
  b.keys = ws.take<uint32_t>((size_t)slots);
  b.vals = ws.take<uint32_t>((size_t)slots);
  b.keys_s = ws.take<uint32_t>((size_t)slots);
  b.vals_s = ws.take<uint32_t>((size_t)slots);
  return b;
}

// Sizes common to both directions; the blocks of a launch have to fit the grid.
int check_sizes(int32_t table_dtype, int32_t out_dtype, int64_t rows, int32_t bag, int64_t codebook_rows, int32_t dim,
                int64_t stride, int32_t code_bytes) {
  if (!dtype_ok(table_dtype) || !dtype_ok(out_dtype)) return GSB_ERR_UNSUPPORTED;
  if (rows < 0 || bag <= 0 || codebook_rows <= 0 || dim <= 0 || stride < 0 || (code_bytes != 4 && code_bytes != 8))
    return GSB_ERR_INVALID_ARGUMENT;
  if (codebook_rows >= (int64_t(1) << 31) - 1 || rows > kSortMaxN / bag || dim > (1 << 20)) return GSB_ERR_CAPACITY;
  return GSB_OK;
}

}  // namespace
}  // namespace gsb

using namespace gsb;

extern "C" int gsb_codebook_forward(int32_t table_dtype, int32_t out_dtype, int64_t rows, int32_t bag,
                                    int64_t codebook_rows, int32_t dim, const void* table, int64_t table_stride,
                                    const void* codes, int32_t code_bytes, const float* weights, float scale,
                                    void* out, uint32_t* status, void* stream) {
  const int rc = check_sizes(table_dtype, out_dtype, rows, bag, codebook_rows, dim, table_stride, code_bytes);
  if (rc != GSB_OK) return rc;
  if (rows == 0) return GSB_OK;
  if (!table || !codes || !out || !status) return GSB_ERR_INVALID_ARGUMENT;
  const int64_t total = rows * dim;
  if ((total + 255) / 256 >= (int64_t(1) << 31)) return GSB_ERR_CAPACITY;
  const Codes cd{codes, code_bytes == 8};
  with_dtype(table_dtype, [&](auto t) {
    with_dtype(out_dtype, [&](auto o) {
      using T = decltype(t);
      using O = decltype(o);
      launch_pdl(k_lookup<T, O>, grid1d(total, 256), 256, 0, static_cast<cudaStream_t>(stream), total, bag,
                 codebook_rows, dim, (const T*)table, table_stride, cd, weights, scale, (O*)out, status);
    });
  });
  note_launches(1);
  return cuda_status(cudaGetLastError());
}

extern "C" size_t gsb_codebook_backward_workspace_size(int64_t rows, int32_t bag, int64_t codebook_rows, int32_t dim) {
  if (check_sizes(GSB_DTYPE_F32, GSB_DTYPE_F32, rows, bag, codebook_rows, dim, 0, 4) != GSB_OK) return 0;
  const int64_t slots = rows * bag;
  Carver c(nullptr);
  carve(c, slots);
  radix_sort_pairs(c, (const uint32_t*)nullptr, nullptr, nullptr, nullptr, slots, 0, bits_for(codebook_rows), nullptr,
                   0, false);
  return c.off + 256;
}

extern "C" int gsb_codebook_backward(int32_t table_dtype, int32_t out_dtype, int64_t rows, int32_t bag,
                                     int64_t codebook_rows, int32_t dim, const void* table, int64_t table_stride,
                                     const void* codes, int32_t code_bytes, const float* weights, float scale,
                                     const void* grad_out, void* g_table, float* g_weights, uint32_t* status,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_sizes(table_dtype, out_dtype, rows, bag, codebook_rows, dim, table_stride, code_bytes);
  if (rc != GSB_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t slots = rows * bag;
  if (slots == 0) {
    if (g_table && cudaMemsetAsync(g_table, 0, (size_t)codebook_rows * dim * dtype_bytes(table_dtype), s) != cudaSuccess)
      return GSB_ERR_CUDA;
    return GSB_OK;
  }
  if (!codes || !grad_out || !status || (g_weights && !table)) return GSB_ERR_INVALID_ARGUMENT;
  const Codes cd{codes, code_bytes == 8};
  cudaError_t e = cudaSuccess;
  if (g_table) {
    if (!workspace || workspace_bytes < gsb_codebook_backward_workspace_size(rows, bag, codebook_rows, dim))
      return GSB_ERR_WORKSPACE;
    Carver ws(workspace);
    const BackwardScratch b = carve(ws, slots);
    launch_pdl(k_code_keys, grid1d(slots, 256), 256, 0, s, slots, codebook_rows, cd, b.keys, b.vals, status);
    e = radix_sort_pairs(ws, b.keys, b.vals, b.keys_s, b.vals_s, slots, 0, bits_for(codebook_rows), status, s, false);
    if (e != cudaSuccess) return GSB_ERR_CUDA;
    with_dtype(table_dtype, [&](auto t) {
      with_dtype(out_dtype, [&](auto o) {
        using T = decltype(t);
        using O = decltype(o);
        launch_pdl(k_table_grad<T, O>, grid1d(codebook_rows * 32, 256), 256, 0, s, slots, bag, codebook_rows, dim,
                   (const uint32_t*)b.keys_s, (const uint32_t*)b.vals_s, weights, scale, (const O*)grad_out,
                   (T*)g_table);
      });
    });
    note_launches(2);
  }
  if (g_weights) {
    with_dtype(table_dtype, [&](auto t) {
      with_dtype(out_dtype, [&](auto o) {
        using T = decltype(t);
        using O = decltype(o);
        launch_pdl(k_weight_grad<T, O>, grid1d(slots * 32, 256), 256, 0, s, slots, bag, codebook_rows, dim,
                   (const T*)table, table_stride, cd, scale, (const O*)grad_out, g_weights, status);
      });
    });
    note_launches(1);
  }
  return cuda_status(cudaGetLastError());
}
