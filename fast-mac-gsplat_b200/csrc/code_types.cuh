// Element types and index types of the codebook kernels (codebook.cu, code_log_probs.cu,
// code_balance.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gsb_common.cuh"
#include "gsb_host.cuh"

namespace gsb {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
// The one rounding of a result to its type (to nearest, ties to even).
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// The values of 16 bytes, on such a boundary wherever they live.
template <typename T>
struct Piece {
  alignas(16) T v[16 / sizeof(T)];
  __device__ __forceinline__ T& operator[](int i) { return v[i]; }
  __device__ __forceinline__ uint4 bits() const { return *reinterpret_cast<const uint4*>(v); }
};
static_assert(alignof(Piece<float>) == 16 && sizeof(Piece<float>) == 16, "read as one uint4");
static_assert(alignof(Piece<__half>) == 16 && sizeof(Piece<__half>) == 16, "read as one uint4");

// Codes are int32 or int64 values; a negative one is an empty slot.
struct Codes {
  const void* p;
  int wide;  // 1: int64
  __device__ __forceinline__ int64_t at(int64_t i) const {
    return wide ? static_cast<const long long*>(p)[i] : (int64_t) static_cast<const int*>(p)[i];
  }
};

// An error of these kernels. The status block may be mapped host memory, so these are
// plain (posted) stores: a million bad codes cost no round trips.
__device__ __forceinline__ void put_error(uint32_t* status, uint32_t flag, uint32_t site) {
  if (status == nullptr) return;
  st_volatile_u32(&status[GSB_STATUS_ERROR_SITE], site);
  st_volatile_u32(&status[GSB_STATUS_ERROR], flag);
}
// A code of at least n: recorded, and treated as an empty slot.
__device__ __forceinline__ void bad_code(uint32_t* status, uint32_t site) {
  put_error(status, GSB_DEVERR_BOUNDS, site);
}

inline bool dtype_ok(int32_t d) { return d == GSB_DTYPE_F32 || d == GSB_DTYPE_BF16 || d == GSB_DTYPE_F16; }
inline int dtype_bytes(int32_t d) { return d == GSB_DTYPE_F32 ? 4 : 2; }

// Calls fn(T{}) with the element type of a GSB_DTYPE_* value.
template <typename Fn>
inline void with_dtype(int32_t d, Fn&& fn) {
  if (d == GSB_DTYPE_F32) fn(float{});
  else if (d == GSB_DTYPE_BF16) fn(__nv_bfloat16{});
  else fn(__half{});
}

}  // namespace gsb
