// What the row-wise operators on assignment logits z [rows, C] share
// (code_log_probs.cu, code_balance.cu): reading a stretch of a row into
// registers, and its softmax sums.
//
// Sums over a row are taken over e_c = exp(z_c - m), m = max z. The values equal
// to m contribute exactly 1 each and are counted, not added:
//   s' = sum_{z_c < m} e_c + (number of z_c = m) - 1,     p_c = e_c / (1 + s')
//   log p_c = (z_c - m) - log1p(s')
//   t  = sum e_c (z_c - m),  mu = t / (1 + s'),  H = log1p(s') - mu
//   u  = sum e_c (n_c - n_a), a the first c with z_c = m:  sum p_c n_c = n_a + u / (1 + s')
// so that log p, 1 - p, H and n_c - sum p n keep their relative accuracy where
// one probability is close to 1 (s' far below 1). All sums are fp32.
//
// A row is read once. kRowElems values a lane stay in registers between the
// maximum and the sums (a second pass over registers costs less than rescaling
// running sums at every new maximum). Lanes that share a row:
//   - 2 to 16 for rows of up to 512 values (several rows a warp),
//   - 1 to 8 warps for rows, or stretches of rows, of up to 8,192 values. Each
//     warp takes its own maximum and sums; only their results meet.
// Stretches of a longer row, or of a few rows that would leave the GPU idle, are
// joined by a second kernel with the same rule (join).
#pragma once

#include <algorithm>
#include <type_traits>

#include "code_types.cuh"

namespace gsb {

constexpr int kRowElems = 32;          // values a lane
constexpr int kGroupMaxLanes = 16;     // lanes a row, several rows a warp
constexpr int kGroupMaxCodes = kGroupMaxLanes * kRowElems;
constexpr int kBlockMaxWarps = 8;
constexpr int kBlockMaxCodes = kBlockMaxWarps * 32 * kRowElems;

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7fc00000); }
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Order of the alternatives as one unsigned number: larger values first, then
// lower indices; -0 equals +0 and NaN comes last.
__device__ __forceinline__ uint32_t order_bits(float z) {
  const uint32_t u = __float_as_uint(z);
  if ((u & 0x7fffffffu) == 0u) return 0x80000000u;
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(float z, uint32_t c) {
  return ((uint64_t)order_bits(z) << 32) | (uint32_t)~c;
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return ~(uint32_t)key; }
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}

// Values a 16-byte load brings.
template <typename T>
constexpr int wide_of() { return 16 / (int)sizeof(T); }

template <typename T>
__device__ __forceinline__ uint32_t neg_inf_bits();  // -inf in every element of a word
template <>
__device__ __forceinline__ uint32_t neg_inf_bits<float>() { return 0xff800000u; }
template <>
__device__ __forceinline__ uint32_t neg_inf_bits<__nv_bfloat16>() { return 0xff80ff80u; }
template <>
__device__ __forceinline__ uint32_t neg_inf_bits<__half>() { return 0xfc00fc00u; }

// Reads values (v lanes + lane) VEC + i of a stretch of len values, v < kRowElems
// / VEC, i < VEC, into z[v VEC + i]; -inf behind its end. VEC is 1, or a 16-byte
// load's worth where the stretch begins on a 16-byte boundary.
template <int VEC>
__device__ __forceinline__ int row_index(int lanes, int lane, int k) {
  return ((k / VEC) * lanes + lane) * VEC + k % VEC;
}
template <int VEC, typename T>
__device__ __forceinline__ void load_row(const T* __restrict__ p, int len, int lanes, int lane,
                                         float (&z)[kRowElems]) {
  if constexpr (VEC == 1) {
    T q[kRowElems];
#pragma unroll
    for (int k = 0; k < kRowElems; ++k) {
      q[k] = from_f32<T>(neg_inf());
      const int c = k * lanes + lane;
      if (c < len) q[k] = p[c];
    }
#pragma unroll
    for (int k = 0; k < kRowElems; ++k) z[k] = to_f32(q[k]);
  } else {
    constexpr int NV = kRowElems / VEC;
    uint4 q[NV];
    const uint32_t low = neg_inf_bits<T>();
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * lanes + lane) * VEC;
      q[v] = make_uint4(low, low, low, low);
      if (c + VEC <= len) q[v] = *reinterpret_cast<const uint4*>(p + c);
    }
    if (len % VEC != 0) {  // the piece that the end falls into
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = (v * lanes + lane) * VEC;
        if (c < len && c + VEC > len) {
          T e[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            e[i] = from_f32<T>(neg_inf());
            if (c + i < len) e[i] = p[c + i];
          }
          q[v] = *reinterpret_cast<const uint4*>(e);
        }
      }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const T* e = reinterpret_cast<const T*>(&q[v]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) z[v * VEC + i] = to_f32(e[i]);
    }
  }
}

// Writes d[] to the same places, rounded once. The stretch begins on a 16-byte
// boundary and its rows are whole pieces where VEC > 1.
template <int VEC, typename T>
__device__ __forceinline__ void store_row(T* __restrict__ p, int len, int lanes, int lane,
                                          const float (&d)[kRowElems]) {
  if constexpr (VEC == 1) {
#pragma unroll
    for (int k = 0; k < kRowElems; ++k) {
      const int c = k * lanes + lane;
      if (c < len) p[c] = from_f32<T>(d[k]);
    }
  } else {
#pragma unroll
    for (int v = 0; v < kRowElems / VEC; ++v) {
      const int c = (v * lanes + lane) * VEC;
      uint4 q;
      T* e = reinterpret_cast<T*>(&q);
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(d[v * VEC + i]);
      if (c < len) *reinterpret_cast<uint4*>(p + c) = q;
    }
  }
}

// m: largest value (NaN aside), a: its first index, s: s' (NaN if the stretch
// holds a NaN), w: t or u, n: n_a (u alone).
struct RowStat {
  float m, s, w, n;
  uint32_t a;
};

// Of two parts of a row. The part with the larger value, or the lower index of
// equal ones, keeps its base; the other's sums move to it, its own largest value
// with them.
template <bool kCounts>
__device__ __forceinline__ RowStat join(RowStat x, RowStat y) {
  const bool first = x.m > y.m || (x.m == y.m && x.a < y.a);
  const RowStat& hi = first ? x : y;
  const RowStat& lo = first ? y : x;
  RowStat r = hi;
  const float d = lo.m - hi.m;  // NaN where both are -inf: nothing to move then
  const float e = lo.m == neg_inf() ? 0.0f : ex2_approx(d * kLog2e);
  const float one = 1.0f + lo.s;
  r.s = hi.s + (e == 0.0f ? 0.0f * lo.s : e * one);  // 0 * NaN: a NaN stays
  if (e > 0.0f) r.w = hi.w + e * fmaf(kCounts ? lo.n - hi.n : d, one, lo.w);
  return r;
}
template <bool kCounts>
__device__ __forceinline__ RowStat shuffle_join(RowStat x, int offset, int width) {
  RowStat y;
  y.m = __shfl_xor_sync(kFullMask, x.m, offset, width);
  y.s = __shfl_xor_sync(kFullMask, x.s, offset, width);
  y.w = __shfl_xor_sync(kFullMask, x.w, offset, width);
  y.n = kCounts ? __shfl_xor_sync(kFullMask, x.n, offset, width) : 0.0f;
  y.a = __shfl_xor_sync(kFullMask, x.a, offset, width);
  return join<kCounts>(x, y);
}

// Largest of a lane's values; NaN loses against any number.
__device__ __forceinline__ float lane_max(const float (&z)[kRowElems]) {
  float m[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) m[k] = fmaxf(fmaxf(z[k], z[k + 8]), fmaxf(z[k + 16], z[k + 24]));
  return fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), fmaxf(fmaxf(m[4], m[5]), fmaxf(m[6], m[7])));
}

// Softmax sums of the values that WIDTH lanes hold (a stretch of len values, dealt
// out to `lanes` lanes by load_row; the other lanes of the row, if any, make their
// own). kCounts: n[] are the counts of a lane's own values, count_of(c) any one's.
// The index in the result is the stretch's.
template <int VEC, int WIDTH, bool kCounts, typename CountOf>
__device__ __forceinline__ RowStat row_stat(const float (&z)[kRowElems], int len, int lanes, int lane,
                                            const float* __restrict__ counts, CountOf&& count_of) {
  RowStat r;
  const float mine = lane_max(z);
  r.m = mine;
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) r.m = fmaxf(r.m, __shfl_xor_sync(kFullMask, r.m, o, WIDTH));
  int at = kRowElems, same = 0;  // where the largest value is, how often
  if (mine == r.m) {
#pragma unroll
    for (int k = kRowElems - 1; k >= 0; --k)
      if (z[k] == r.m) at = k, ++same;
  }
  const uint32_t own = at < kRowElems ? (uint32_t)row_index<VEC>(lanes, lane, at) : 0x7fffffffu;
  uint32_t a = own;
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) a = min(a, __shfl_xor_sync(kFullMask, a, o, WIDTH));
  r.a = min(a, (uint32_t)(len - 1));  // NaN alone: any
  r.n = kCounts ? count_of((int)r.a) : 0.0f;
  // The 1 of a itself is never added: it would swallow what s' is in a row with one certain code.
  float s = (float)(own == a && at < kRowElems ? same - 1 : same), w = 0.0f;
  constexpr int P = VEC == 1 ? 1 : 4;  // counts that one load brings
#pragma unroll
  for (int k0 = 0; k0 < kRowElems; k0 += P) {
    float n[P];
    if constexpr (kCounts) {
      const int c = row_index<VEC>(lanes, lane, k0);
      if constexpr (P == 4) {
        const float4 q = c < len ? *reinterpret_cast<const float4*>(counts + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        n[0] = q.x, n[1] = q.y, n[2] = q.z, n[3] = q.w;
      } else {
        n[0] = c < len ? counts[c] : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float zk = z[k0 + i];
      const float x = zk - r.m;
      const float e = ex2_approx(x * kLog2e);
      if (!(zk >= r.m)) s += e;  // a NaN is added
      if constexpr (kCounts) {
        w = fmaf(e, n[i] - r.n, w);  // 0 at a itself; its equals count in full
      } else {
        // x = -inf: e is 0, and so is its term (the bound is far below the range of exp).
        const float t = max_nan(x, -200.0f);
        if (!(zk >= r.m)) w = fmaf(e, t, w);
      }
    }
  }
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) {
    s += __shfl_xor_sync(kFullMask, s, o, WIDTH);
    w += __shfl_xor_sync(kFullMask, w, o, WIDTH);
  }
  r.s = s;
  r.w = w;
  return r;
}

// How the rows of a call are taken: `lanes` a row (kGroupMaxLanes or fewer: rows
// side by side in a warp), else warps per stretch and stretches per row.
struct RowPlan {
  int lanes = 0;  // 0: blocks
  int warps = 1, parts = 1, part_len = 0;
};
// Stretches: as few as 8,192 values allow, more where that leaves fewer than two
// blocks an SM, but none below 1,024 values (a warp's).
inline RowPlan row_plan(int64_t rows, int64_t codes) {
  RowPlan p;
  if (codes <= kGroupMaxCodes) {
    p.lanes = 2;
    while ((int64_t)p.lanes * kRowElems < codes) p.lanes *= 2;
    return p;
  }
  constexpr int64_t kFill = 2 * 148;
  int64_t parts = (codes + kBlockMaxCodes - 1) / kBlockMaxCodes;
  if (rows * parts < kFill) parts = std::max(parts, std::min((codes + 1023) / 1024, (kFill + rows - 1) / rows));
  const int64_t len = ((codes + parts - 1) / parts + 7) / 8 * 8;  // 16-byte boundaries of every type
  p.part_len = (int)len;
  p.parts = (int)((codes + len - 1) / len);
  while (p.warps * 32 * kRowElems < len) p.warps *= 2;
  return p;
}

// Calls fn(integral constant).
template <typename Fn>
inline void with_lanes(int lanes, Fn&& fn) {
  if (lanes == 2) fn(std::integral_constant<int, 2>{});
  else if (lanes == 4) fn(std::integral_constant<int, 4>{});
  else if (lanes == 8) fn(std::integral_constant<int, 8>{});
  else fn(std::integral_constant<int, 16>{});
}
template <typename Fn>
inline void with_warps(int warps, Fn&& fn) {
  if (warps == 1) fn(std::integral_constant<int, 1>{});
  else if (warps == 2) fn(std::integral_constant<int, 2>{});
  else if (warps == 4) fn(std::integral_constant<int, 4>{});
  else fn(std::integral_constant<int, 8>{});
}
// Calls fn(T{}, integral constant VEC).
template <typename Fn>
inline void with_rows(int32_t dtype, bool wide, Fn&& fn) {
  with_dtype(dtype, [&](auto t) {
    if (wide) fn(t, std::integral_constant<int, wide_of<decltype(t)>()>{});
    else fn(t, std::integral_constant<int, 1>{});
  });
}
inline bool rows_wide(int32_t dtype, const void* p, int64_t stride) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * dtype_bytes(dtype) % 16 == 0;
}

inline int check_rows(int32_t dtype, int64_t rows, int64_t codes, int64_t stride, int32_t code_bytes) {
  if (!dtype_ok(dtype)) return GSB_ERR_UNSUPPORTED;
  if (rows < 0 || codes <= 0 || stride < 0 || (code_bytes != 4 && code_bytes != 8)) return GSB_ERR_INVALID_ARGUMENT;
  if (codes >= (int64_t(1) << 31) - kBlockMaxCodes || rows >= (int64_t(1) << 31)) return GSB_ERR_CAPACITY;
  return GSB_OK;
}

// Blocks of a launch whose blocks loop over `items`.
inline unsigned item_grid(int64_t items) { return (unsigned)std::min<int64_t>(items, (int64_t(1) << 31) - 1); }

}  // namespace gsb
