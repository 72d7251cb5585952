// What the row-wise operators on assignment logits z [rows, C] share
// (code_log_probs.cu, code_balance.cu): the rule of their softmax sums, the order of
// alternatives, and the backward's way of reading and writing rows (the forward's is
// in code_tiles.cuh).
//
// Sums over a row are taken over e_c = exp(z_c - m), m = max z. The value at a, the
// first c with z_c = m, contributes exactly 1 and is left out:
//   s' = sum_{c != a} e_c,     p_c = e_c / (1 + s')
//   log p_c = (z_c - m) - log1p(s')
//   t  = sum_{c != a} e_c (z_c - m),  mu = t / (1 + s'),  H = log1p(s') - mu
//   u  = sum_{c != a} e_c (n_c - n_a),     sum_c p_c n_c = n_a + u / (1 + s')
// so that log p, 1 - p, H and n_c - sum p n keep their relative accuracy where
// one probability is close to 1 (s' far below 1). All sums are fp32. Sums of two
// parts of a row meet by the same rule (join).
//
// The backward is elementwise: kRowElems values a lane in registers, 2 to 16 lanes a
// row for rows of up to 512 values and 1 to 8 warps for stretches of longer ones; 64
// registers a thread, which keeps enough loads under way (with 80 it took 3 to 9 %
// longer). That was measured where next to nothing spills: rows on 16-byte boundaries.
// Elsewhere 64 is one rule for kernels that want more: of 16-bit types in shifted pieces
// the balance gradient spills 272 to 276 bytes a thread in rows of up to 512 values and 44
// to 96 in longer ones, the log probabilities' 12 to 44 (28 to 88 with one warp a stretch,
// in any mode); fp32 taken one by one spills up to 84. 2^20 x 100 bf16 takes 163 us (balance)
// and 156 us (log probabilities) where 104 values, on boundaries, take 87 and 117.
#pragma once

#include <algorithm>
#include <type_traits>

#include "code_types.cuh"

namespace gsb {

constexpr int kRowElems = 32;          // values a lane
constexpr int kGroupMaxLanes = 16;     // lanes a row, several rows a warp
constexpr int kGroupMaxCodes = kGroupMaxLanes * kRowElems;
constexpr int kBlockMaxWarps = 8;
constexpr int kRowThreadsSM = 1024;     // threads an SM that registers are kept for (64 each)

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

// How a stretch of a row is dealt out to `lanes` lanes: lane l's value k has the
// place (k / VEC lanes + l) VEC + k % VEC. VEC is 1, or the values of a 16-byte piece.
// Where rows begin between 16-byte boundaries (Mode::kShifted) places count from the
// boundary before the row's first value, `shift` values before it, so that pieces lie
// on boundaries whatever the row's length. Places lo .. hi - 1 hold values; `full`:
// the first nv pieces of every lane are whole and the others empty, and nothing else is
// checked.
enum class Mode { kSingle, kWide, kShifted };
template <typename T, Mode M>
struct Deal {
  static constexpr int VEC = M == Mode::kSingle ? 1 : wide_of<T>();
  int lo, hi, lanes, lane, nv;
  bool full;
  __device__ __forceinline__ Deal(int lo_, int hi_, int lanes_, int lane_)
      : lo(lo_), hi(hi_), lanes(lanes_), lane(lane_), nv(hi_ / (lanes_ * VEC)) {
    full = lo == 0 && hi == nv * lanes * VEC;
  }
  __device__ __forceinline__ int place(int k) const { return ((k / VEC) * lanes + lane) * VEC + k % VEC; }
  __device__ __forceinline__ bool has(int c) const { return (M != Mode::kShifted || c >= lo) && c < hi; }
  __device__ __forceinline__ bool whole(int c) const { return (M != Mode::kShifted || c >= lo) && c + VEC <= hi; }
  __device__ __forceinline__ bool ragged(int c) const { return c + VEC > lo && c < hi && !whole(c); }
};
// Values between the 16-byte boundary before p and p.
template <typename T, Mode M>
__device__ __forceinline__ int shift_of(const T* p) {
  return M == Mode::kShifted ? (int)(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T)) : 0;
}

// Reads a lane's values (p: place 0); 0 where there is none.
template <typename T, Mode M>
__device__ __forceinline__ void load_row(const T* __restrict__ p, const Deal<T, M>& at, float (&z)[kRowElems]) {
  constexpr int VEC = Deal<T, M>::VEC;
  if constexpr (VEC == 1) {
    static_assert(sizeof(T) == 4, "values of two bytes are read in pieces");
#pragma unroll
    for (int k = 0; k < kRowElems; ++k) {
      const int c = at.place(k);
      z[k] = 0.0f;
      if (c < at.hi) z[k] = p[c];
    }
  } else {
    constexpr int NV = kRowElems / VEC;
    uint4 q[NV];
    if (at.full) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        q[v] = make_uint4(0u, 0u, 0u, 0u);
        if (v < at.nv) q[v] = *reinterpret_cast<const uint4*>(p + at.place(v * VEC));
      }
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = at.place(v * VEC);
        q[v] = make_uint4(0u, 0u, 0u, 0u);
        if (at.whole(c)) {
          q[v] = *reinterpret_cast<const uint4*>(p + c);
        } else if (M == Mode::kShifted && at.ragged(c)) {
          Piece<T> e;
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            e[i] = from_f32<T>(0.0f);
            if (at.has(c + i)) e[i] = p[c + i];
          }
          q[v] = e.bits();
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

// The same values one by one, for rows that lie differently to the 16-byte
// boundaries than the result that `at` deals out.
template <typename T, Mode M>
__device__ __forceinline__ void load_row_single(const T* __restrict__ p, const Deal<T, M>& at,
                                                float (&z)[kRowElems]) {
  constexpr int VEC = Deal<T, M>::VEC;
  T q[kRowElems];
  if (at.full) {
#pragma unroll
    for (int k = 0; k < kRowElems; ++k) {
      q[k] = from_f32<T>(0.0f);
      if (k / VEC < at.nv) q[k] = p[at.place(k)];
    }
  } else {
#pragma unroll
    for (int k = 0; k < kRowElems; ++k) {
      const int c = at.place(k);
      q[k] = from_f32<T>(0.0f);
      if (at.has(c)) q[k] = p[c];
    }
  }
#pragma unroll
  for (int k = 0; k < kRowElems; ++k) z[k] = to_f32(q[k]);
}

// Writes d[] to the places of a lane's values, rounded once.
template <typename T, Mode M>
__device__ __forceinline__ void store_row(T* __restrict__ p, const Deal<T, M>& at, const float (&d)[kRowElems]) {
  constexpr int VEC = Deal<T, M>::VEC;
  if constexpr (VEC == 1) {
#pragma unroll
    for (int k = 0; k < kRowElems; ++k) {
      const int c = at.place(k);
      if (c < at.hi) p[c] = from_f32<T>(d[k]);
    }
  } else {
    auto piece = [&](int v) {
      Piece<T> e;
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(d[v * VEC + i]);
      return e.bits();
    };
    if (at.full) {
#pragma unroll
      for (int v = 0; v < kRowElems / VEC; ++v)
        if (v < at.nv) *reinterpret_cast<uint4*>(p + at.place(v * VEC)) = piece(v);
    } else {
#pragma unroll
      for (int v = 0; v < kRowElems / VEC; ++v) {
        const int c = at.place(v * VEC);
        if (at.whole(c)) {
          *reinterpret_cast<uint4*>(p + c) = piece(v);
        } else if (M == Mode::kShifted && at.ragged(c)) {
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (at.has(c + i)) p[c + i] = from_f32<T>(d[v * VEC + i]);
        }
      }
    }
  }
}

// Counts of codes as floats, in two layouts: by code, and by code modulo 8 (values
// that lie `lanes` pieces of 8 apart then lie side by side, at any shift).
// `codes` is the codebook's size; both are padded to a multiple of 8.
struct Counts {
  const float* by_code;
  const float* by_eight;
  int64_t eights;  // codes / 8, rounded up
  // Of the codes from c0 on, a multiple of 8.
  __device__ __forceinline__ Counts from(int64_t c0) const { return Counts{by_code + c0, by_eight + c0 / 8, eights}; }
  // Where the count of value j of a piece is in by_eight, relative to that of the first
  // 8-aligned code of the piece: code 8 q + j - shift has the same residue modulo 8 for
  // every q.
  struct Offsets {
    int of[8];
    __device__ __forceinline__ Offsets(const Counts& counts, int shift) {
#pragma unroll
      for (int j = 0; j < 8; ++j) of[j] = ((j - shift) & 7) * (int)counts.eights - (j < shift ? 1 : 0);
    }
  };
  // Those of a lane's values k .. k + 3 (of which some lane has one), place 0 being code
  // -shift; 0 where the lane has none.
  template <typename T, Mode M>
  __device__ __forceinline__ void four(const Deal<T, M>& at, int shift, const Offsets& off, int k,
                                       float (&n)[4]) const {
    const int c = at.place(k);
    if constexpr (M == Mode::kWide) {
      const float4 q = at.full || c < at.hi ? *reinterpret_cast<const float4*>(by_code + c)
                                            : make_float4(0.f, 0.f, 0.f, 0.f);
      n[0] = q.x, n[1] = q.y, n[2] = q.z, n[3] = q.w;
    } else if constexpr (M == Mode::kShifted) {
      static_assert(Deal<T, M>::VEC == 8, "values of two bytes");
      const int first = c - k % 8;  // the piece's
      const float* p = by_eight + first / 8;
      if (at.full) {
#pragma unroll
        for (int i = 0; i < 4; ++i) n[i] = p[off.of[k % 8 + i]];
      } else {
        const bool whole = at.whole(first);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          n[i] = 0.0f;
          if (whole) n[i] = p[off.of[k % 8 + i]];
        }
        if (at.ragged(first)) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (at.has(c + i)) n[i] = by_code[c + i - shift];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ci = at.place(k + i);
        n[i] = ci < at.hi ? by_code[ci] : 0.0f;
      }
    }
  }
};

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
// Of the parts that WIDTH lanes hold: the same rule, with the largest value found
// first, so that every part moves once.
template <bool kCounts, int WIDTH>
__device__ __forceinline__ RowStat join_lanes(const RowStat& x) {
  RowStat r;
  r.m = x.m;
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) r.m = fmaxf(r.m, __shfl_xor_sync(kFullMask, r.m, o, WIDTH));
  r.a = x.m == r.m ? x.a : 0xffffffffu;
  if (WIDTH == 32) {
    r.a = __reduce_min_sync(kFullMask, r.a);
  } else {
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1) r.a = min(r.a, __shfl_xor_sync(kFullMask, r.a, o, WIDTH));
  }
  const bool winner = x.m == r.m && x.a == r.a;
  r.n = 0.0f;
  if (kCounts) {
    r.n = winner ? x.n : neg_inf();
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1) r.n = fmaxf(r.n, __shfl_xor_sync(kFullMask, r.n, o, WIDTH));
  }
  const float d = x.m - r.m;  // NaN where both are -inf: nothing to move then
  const float e = x.m == neg_inf() ? 0.0f : ex2_approx(d * kLog2e);
  const float one = 1.0f + x.s;
  r.s = e == 0.0f ? 0.0f * x.s : e * one;  // 0 * NaN: a NaN stays
  r.w = e > 0.0f ? e * fmaf(kCounts ? x.n - r.n : d, one, x.w) : 0.0f;
  if (winner) r.s = x.s, r.w = x.w;
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) {
    r.s += __shfl_xor_sync(kFullMask, r.s, o, WIDTH);
    r.w += __shfl_xor_sync(kFullMask, r.w, o, WIDTH);
  }
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN loses against any number
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Smallest of a lane's values (NaN loses).
__device__ __forceinline__ float lane_min(const float (&z)[kRowElems]) {
  float m = min3(z[0], z[1], z[2]);
#pragma unroll
  for (int k = 3; k + 1 < kRowElems; k += 2) m = min3(m, z[k], z[k + 1]);
  return fminf(m, z[kRowElems - 1]);
}

// exp of values relative to a row's m, as 2^y with y = z log2 e - M in one rounding,
// M = m log2 e rounded. What that rounding left, d = m log2 e - M, is the same
// factor 2^d on every value; it is taken out of the sums (`undo` = 2^-d). Where m is
// far from 0 that factor leaves its range: `far` rows take z - m first.
struct Base {
  float m, neg_M, d, undo;
  bool far;
  __device__ __forceinline__ explicit Base(float m_) : m(m_) {
    far = !(fabsf(m) <= 1024.0f);  // -inf and NaN too
    neg_M = -__fmul_rn(m, kLog2e);
    d = fmaf(m, kLog2e, neg_M);
    undo = ex2_approx(-d);
  }
};
constexpr float kLn2 = 0.6931471805599453f;
// Below this z log2 e may be -inf, and its product with e = 0 NaN.
constexpr float kLowest = -1e38f;

// How the backward takes the rows of a call: `lanes` a row (kGroupMaxLanes or fewer:
// rows side by side in a warp), else `warps` per stretch of part_len places (whole
// pieces of all their lanes), `parts` stretches per row. Stretches are of up to 8,192
// places, shorter where that leaves fewer than two blocks an SM. shifted: a row may need
// up to 7 places more than it has values.
struct RowPlan {
  int lanes = 0;  // 0: blocks
  int warps = 1, parts = 1, part_len = 0;
};
inline RowPlan row_plan(int64_t rows, int64_t codes, bool shifted, int vec) {
  RowPlan p;
  const int64_t places = codes + (shifted ? 7 : 0);
  if (places <= kGroupMaxCodes) {
    p.lanes = 2;
    while ((int64_t)p.lanes * kRowElems < places) p.lanes *= 2;
    return p;
  }
  p.warps = kBlockMaxWarps;
  while (p.warps > 1 && (p.warps / 2 * 32 * kRowElems >= places ||
                         rows * ((places + p.warps * 32 * kRowElems - 1) / (p.warps * 32 * kRowElems)) < 2 * 148))
    p.warps /= 2;
  const int64_t most = p.warps * 32 * kRowElems, unit = p.warps * 32 * vec;
  const int64_t parts = (places + most - 1) / most;
  p.part_len = (int)(((places + parts - 1) / parts + unit - 1) / unit * unit);
  p.parts = (int)((places + p.part_len - 1) / p.part_len);
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
template <Mode M>
using ModeOf = std::integral_constant<Mode, M>;
// How the rows at p lie: pieces of 16 bytes where all begin on such a boundary;
// values of two bytes in shifted pieces elsewhere, of four one by one (a warp's 128
// bytes a load already).
inline Mode row_mode(int32_t dtype, const void* p, int64_t stride) {
  if (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * dtype_bytes(dtype) % 16 == 0) return Mode::kWide;
  return dtype == GSB_DTYPE_F32 ? Mode::kSingle : Mode::kShifted;
}
// Calls fn(T{}, ModeOf<>{}).
template <typename Fn>
inline void with_rows(int32_t dtype, Mode mode, Fn&& fn) {
  with_dtype(dtype, [&](auto t) {
    if (mode == Mode::kWide) fn(t, ModeOf<Mode::kWide>{});
    else if constexpr (sizeof(t) == 4) fn(t, ModeOf<Mode::kSingle>{});
    else fn(t, ModeOf<Mode::kShifted>{});
  });
}
// The backward's, by the result's rows; the third argument says whether the logits'
// rows lie as the result's do.
template <typename Fn>
inline void with_row_pairs(int32_t dtype, const void* in, int64_t in_stride, const void* out, int64_t out_stride,
                           Fn&& fn) {
  const int64_t size = dtype_bytes(dtype);
  const bool same = (reinterpret_cast<uintptr_t>(in) - reinterpret_cast<uintptr_t>(out)) % 16 == 0 &&
                    (in_stride - out_stride) * size % 16 == 0;
  Mode mode = row_mode(dtype, out, out_stride);
  if (!same) mode = dtype == GSB_DTYPE_F32 ? Mode::kSingle : Mode::kShifted;
  with_rows(dtype, mode, [&](auto t, auto m) {
    if constexpr (decltype(m)::value == Mode::kShifted) {
      if (same) fn(t, m, std::true_type{});
      else fn(t, m, std::false_type{});
    } else {
      fn(t, m, std::true_type{});
    }
  });
}

inline int check_rows(int32_t dtype, int64_t rows, int64_t codes, int64_t stride, int32_t code_bytes) {
  if (!dtype_ok(dtype)) return GSB_ERR_UNSUPPORTED;
  if (rows < 0 || codes <= 0 || stride < 0 || (code_bytes != 4 && code_bytes != 8)) return GSB_ERR_INVALID_ARGUMENT;
  if (codes >= (int64_t(1) << 31) - 65536 || rows >= (int64_t(1) << 31)) return GSB_ERR_CAPACITY;
  return GSB_OK;
}

// Blocks of a launch whose blocks loop over `items`.
inline unsigned item_grid(int64_t items) { return (unsigned)std::min<int64_t>(items, (int64_t(1) << 31) - 1); }

}  // namespace gsb
