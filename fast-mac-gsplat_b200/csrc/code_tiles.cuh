// The forward half of the row-wise operators on assignment logits: softmax sums of
// rows that stream through shared memory.
//
// A warp owns its rows from the first load to the result: no block-wide barrier.
//   - L = 2 .. 16 lanes a row, 32 / L rows at once, for rows that fit 8 pieces of
//     16 bytes a lane;
//   - L = 32 for longer rows (or parts of a row), which pass in slices of 8 pieces a
//     lane; every lane keeps its own maximum and sums over the slices, so that lanes
//     exchange values once a row.
// Slices are copied asynchronously, one ahead of the one in work, and each lane reads only what it copied itself, which needs no barrier either. Shared
// memory also gives a lane's values an index: the largest one is found by piece and
// taken out of the sums by one store, where values in registers cost a comparison
// and a selection each.
//
// Bound by the logits' bytes while a value costs no more than a few instructions: a
// maximum (two values at a time for 16-bit types), a conversion, and half of each of
// an FMA, an addition and an FMA on pairs around one ex2.
#pragma once

#include "code_rows.cuh"

namespace gsb {

constexpr int kTilePieces = 8;  // of 16 bytes, a lane
constexpr int kTileStages = 2;  // one in work, one on its way
constexpr int kTileWarps = 4;   // a block
constexpr int kTileSlices = 8;  // a part, at most

template <typename T>
constexpr int tile_elems() { return kTilePieces * wide_of<T>(); }  // values a lane

// Where a lane's values of a slice lie: piece v's value i has the index at(v) + i in
// its part (or row) of len values. shift: values between the 16-byte boundary before
// the part and its start. Pieces w0 .. w1 - 1 are whole for every lane of the row; of
// the n that any lane has, those beside them are ragged: at most the first and the last.
template <typename T, int L>
struct Slice {
  static constexpr int VEC = wide_of<T>();
  int len, shift, first;  // first: index of the lane's piece 0
  int w0, w1, n;
  __device__ __forceinline__ Slice(int len_, int shift_, int slice, int lane) : len(len_), shift(shift_) {
    const int begin = slice * (L * kTilePieces * VEC) - shift;  // index of lane 0's piece 0
    const int left = len - begin;
    first = begin + lane * VEC;
    w0 = begin < 0 ? 1 : 0;
    w1 = min(left / (L * VEC), kTilePieces);
    n = min((left + L * VEC - 1) / (L * VEC), kTilePieces);
  }
  __device__ __forceinline__ int at(int v) const { return first + v * L * VEC; }
  __device__ __forceinline__ bool has(int c) const { return c >= 0 && c < len; }
  __device__ __forceinline__ bool ragged() const { return w0 > 0 || w1 < n; }
  // Calls fn(v) for the ragged pieces.
  template <typename Fn>
  __device__ __forceinline__ void each_ragged(Fn&& fn) const {
    for (int v = w0 > 0 ? 0 : w1; v < n; v = v < w1 ? w1 : n) fn(v);
  }
};

__device__ __forceinline__ void cp_async16_part(void* smem, const void* gmem, int bytes) {  // the rest is zeros
  const unsigned s = (unsigned)__cvta_generic_to_shared(smem);
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(s), "l"(gmem), "r"(bytes) : "memory");
}

// Begins the copy of a lane's pieces of a slice. A piece may reach in front of its
// row, into the row before (its values are not used), but not in front of `base`,
// the logits' first value: the few values of such a piece are copied one by one.
template <typename T, int L>
__device__ __forceinline__ void issue_slice(uint4* buf, const T* __restrict__ p, const T* __restrict__ base,
                                            const Slice<T, L>& at) {
  constexpr int VEC = wide_of<T>();
  const T* from = p + at.first;
#pragma unroll
  for (int v = 0; v < kTilePieces; ++v)
    if (v >= at.w0 && v < at.w1) cp_async16(buf + v * 32, from + v * L * VEC);
  if (at.ragged()) {
    at.each_ragged([&](int v) {
      const int c = at.at(v);
      uint4* to = buf + v * 32;
      if (c >= at.len || c + VEC <= 0) return;
      if (c < 0 && p + c < base) {
        for (int i = 0; i < VEC; ++i)
          if (at.has(c + i)) reinterpret_cast<T*>(to)[i] = p[c + i];
      } else {
        cp_async16_part(to, p + c, min(VEC, at.len - c) * (int)sizeof(T));
      }
    });
  }
}
// Puts `value` in the places of ragged pieces that hold none of the part's values.
template <typename T, int L>
__device__ __forceinline__ void fill_ragged(uint4* buf, const Slice<T, L>& at, float value) {
  const T e = from_f32<T>(value);
  at.each_ragged([&](int v) {
    for (int i = 0; i < wide_of<T>(); ++i)
      if (!at.has(at.at(v) + i)) reinterpret_cast<T*>(buf + v * 32)[i] = e;
  });
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& q, float (&f)[wide_of<T>()]) {
  const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
  for (int i = 0; i < wide_of<T>(); ++i) f[i] = to_f32(e[i]);
}
// Largest and smallest value of a piece (NaN loses against any).
__device__ __forceinline__ void piece_range(const uint4& q, float, float& hi, float& lo) {
  const float a = __uint_as_float(q.x), b = __uint_as_float(q.y), c = __uint_as_float(q.z), d = __uint_as_float(q.w);
  hi = fmaxf(max3(a, b, c), d);
  lo = fminf(min3(a, b, c), d);
}
__device__ __forceinline__ void piece_range(const uint4& q, __nv_bfloat16, float& hi, float& lo) {
  const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&q);
  const __nv_bfloat162 h = __hmax2(__hmax2(e[0], e[1]), __hmax2(e[2], e[3]));
  const __nv_bfloat162 l = __hmin2(__hmin2(e[0], e[1]), __hmin2(e[2], e[3]));
  hi = fmaxf(__low2float(h), __high2float(h));
  lo = fminf(__low2float(l), __high2float(l));
}
__device__ __forceinline__ void piece_range(const uint4& q, __half, float& hi, float& lo) {
  const __half2* e = reinterpret_cast<const __half2*>(&q);
  const __half2 h = __hmax2(__hmax2(e[0], e[1]), __hmax2(e[2], e[3]));
  const __half2 l = __hmin2(__hmin2(e[0], e[1]), __hmin2(e[2], e[3]));
  hi = fmaxf(__low2float(h), __high2float(h));
  lo = fminf(__low2float(l), __high2float(l));
}

// Counts of a piece's values; 0 where the part has none.
template <typename T, int L>
__device__ __forceinline__ void piece_counts(const Counts& counts, const Slice<T, L>& at, int v,
                                             float (&n)[wide_of<T>()]) {
  constexpr int VEC = wide_of<T>();
  const int c = at.at(v);
  if (at.shift == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      // Padded to a multiple of 8 codes: a piece that the part has any of is all there.
      const float4 q = c < at.len ? *reinterpret_cast<const float4*>(counts.by_code + c + i)
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
      n[i] = q.x, n[i + 1] = q.y, n[i + 2] = q.z, n[i + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      n[i] = 0.0f;
      if (at.has(c + i))
        n[i] = VEC == 8 ? counts.by_eight[((i - at.shift) & 7) * counts.eights + ((c + i) >> 3)]
                        : counts.by_code[c + i];
    }
  }
}

// The sums of a lane's pieces about base.m (r.n: the count that others are taken
// relative to). kClamp: some value is -inf, or so low that its multiple with log2 e
// is; e = 0 times that would be NaN.
template <bool kCounts, bool kClamp, typename T, int L>
__device__ __forceinline__ void piece_sums(const uint4* buf, const Slice<T, L>& at, const Counts& counts,
                                           const Base& base, RowStat& r) {
  constexpr int VEC = wide_of<T>();
  const F2 l2 = f2(kLog2e), neg_M = f2(base.neg_M), neg_n = f2(-r.n);
  F2 s2 = f2(0.0f), w2 = f2(0.0f);
#pragma unroll
  for (int v = 0; v < kTilePieces; ++v) {
    if (v < at.n) {
      float f[VEC], n[VEC];
      if constexpr (kCounts) piece_counts(counts, at, v, n);
      unpack<T>(buf[v * 32], f);
#pragma unroll
      for (int i = 0; i < VEC; i += 2) {
        F2 y = fma2(f2(f[i], f[i + 1]), l2, neg_M);
        float y0, y1;
        split(y, y0, y1);
        if constexpr (kClamp) {
          y0 = max_nan(y0, -300.0f), y1 = max_nan(y1, -300.0f);
          y = f2(y0, y1);
        }
        const F2 e = f2(ex2_approx(y0), ex2_approx(y1));
        s2 = add2(s2, e);
        w2 = fma2(e, kCounts ? add2(f2(n[i], n[i + 1]), neg_n) : y, w2);
      }
    }
  }
  float s0, s1, w0, w1;
  split(s2, s0, s1);
  split(w2, w0, w1);
  r.s = s0 + s1;
  r.w = w0 + w1;
  // Out with the base's rounding; t from log2 to log.
  r.w = kCounts ? r.w * base.undo : (r.w - base.d * r.s) * (base.undo * kLn2);
  r.s *= base.undo;
}

// The softmax sums of one lane's values of a slice (buf: its pieces, 32 apart),
// without its largest (its first largest, which leaves `buf` too). The index in the
// result is the part's.
template <bool kCounts, typename T, int L>
__device__ __forceinline__ RowStat lane_sums(uint4* buf, const Slice<T, L>& at, const Counts& counts) {
  constexpr int VEC = wide_of<T>();
  if (at.ragged()) fill_ragged(buf, at, quiet_nan());
  float top[kTilePieces], low = 0.0f;
#pragma unroll
  for (int v = 0; v < kTilePieces; ++v) {
    top[v] = quiet_nan();
    if (v < at.n) {
      float lo;
      piece_range(buf[v * 32], T{}, top[v], lo);
      low = fminf(low, lo);
    }
  }
  RowStat r;
  const float m = max3(max3(top[0], top[1], top[2]), max3(top[3], top[4], top[5]), fmaxf(top[6], top[7]));
  const bool some = m == m;                   // else: no value, or NaN alone
  const Base base(m > neg_inf() ? m : 0.0f);  // with m = -inf all is 0 (or NaN) relative to 0 too
  const float none = base.far ? neg_inf() : base.m - 200.0f;  // adds nothing
  r.a = 0xffffffffu;
  if (some) {
    int v0 = 0;
#pragma unroll
    for (int v = kTilePieces - 1; v >= 0; --v)
      if (top[v] == m) v0 = v;
    float f[VEC];
    unpack<T>(buf[v0 * 32], f);
    int i0 = 0;
#pragma unroll
    for (int i = VEC - 1; i >= 0; --i)
      if (f[i] == m) i0 = i;
    reinterpret_cast<T*>(buf + v0 * 32)[i0] = from_f32<T>(none);
    r.a = (uint32_t)(at.at(v0) + i0);
  }
  if (at.ragged()) fill_ragged(buf, at, none);
  r.n = kCounts && some ? counts.by_code[r.a] : 0.0f;
  if (__any_sync(kFullMask, base.far)) {
    r.s = r.w = 0.0f;
    for (int v = 0; v < at.n; ++v) {
      float f[VEC], n[VEC];
      unpack<T>(buf[v * 32], f);
      if constexpr (kCounts) piece_counts(counts, at, v, n);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float x = max_nan(f[i] - base.m, -200.0f);
        const float e = ex2_approx(x * kLog2e);
        r.s += e;
        r.w = fmaf(e, kCounts ? n[i] - r.n : x, r.w);
      }
    }
  } else if (!kCounts && __any_sync(kFullMask, low < kLowest)) {
    piece_sums<kCounts, !kCounts>(buf, at, counts, base, r);
  } else {
    piece_sums<kCounts, false>(buf, at, counts, base, r);
  }
  const bool lane_any = at.first < at.len && at.first + (kTilePieces - 1) * L * VEC + VEC > 0;
  r.m = some ? m : neg_inf();
  if (!some) {
    r.w = 0.0f;
    if (!lane_any) r.s = 0.0f;
  }
  return r;
}

// How a call's rows are dealt to warps.
struct TilePlan {
  int lanes = 32;
  int parts = 1;
  int64_t part_len = 0;
  int64_t items(int64_t rows) const { return lanes < 32 ? (rows + 32 / lanes - 1) / (32 / lanes) : rows * parts; }
};
// Rows that fit 16 lanes share a warp. Longer ones take a warp a part; parts of
// kTileSlices slices at most, or shorter ones where there are too few rows for two
// rounds of the warps that are resident, but none below a slice.
// shifted: rows may begin between 16-byte boundaries.
inline TilePlan tile_plan(int64_t rows, int64_t codes, int size, bool shifted) {
  TilePlan p;
  const int vec = 16 / size, elems = kTilePieces * vec;
  p.part_len = codes;
  for (int l = 2; l <= 16; l *= 2) {
    if (codes + (shifted ? vec - 1 : 0) <= l * elems) {
      p.lanes = l;
      return p;
    }
  }
  const int64_t slice = 32 * elems, most = kTileSlices * slice - 8;
  int64_t parts = (codes + most - 1) / most;
  constexpr int64_t kFill = 2 * 148 * 16;
  if (rows * parts < kFill) parts = std::max(parts, std::min((codes + slice - 1) / slice, (kFill + rows - 1) / rows));
  p.part_len = ((codes + parts - 1) / parts + 7) / 8 * 8;
  p.parts = (int)((codes + p.part_len - 1) / p.part_len);
  return p;
}
template <typename Fn>
inline void with_tile_lanes(int lanes, Fn&& fn) {
  if (lanes == 2) fn(std::integral_constant<int, 2>{});
  else if (lanes == 4) fn(std::integral_constant<int, 4>{});
  else if (lanes == 8) fn(std::integral_constant<int, 8>{});
  else if (lanes == 16) fn(std::integral_constant<int, 16>{});
  else fn(std::integral_constant<int, 32>{});
}

inline bool rows_shifted(int size, const void* p, int64_t stride) {
  return reinterpret_cast<uintptr_t>(p) % 16 != 0 || stride * size % 16 != 0;
}
inline int tile_blocks(int64_t items) {
  constexpr int kResident = 148 * 5;  // by shared memory
  return (int)std::min<int64_t>(kResident, (items + kTileWarps - 1) / kTileWarps);
}

// The rows of a call, and where a warp is in them.
template <typename T>
struct TileRows {
  const T* logits;
  int64_t stride, rows, codes, part_len, items;
  int parts;
};
template <typename T, int L>
struct TilePlace {
  int64_t item, row, c0;
  const T* p;  // the part's first value
  int slice, slices, len, shift;
  bool on;
  __device__ __forceinline__ TilePlace(const TileRows<T>& t, int64_t item_, int lane32) : item(item_), slice(0) {
    if (L < 32) {
      const int64_t mine = item * (32 / L) + lane32 / L;
      on = mine < t.rows;
      row = on ? mine : t.rows - 1;  // lanes without a row keep a warp's exchanges whole
      c0 = 0;
      len = (int)t.codes;
    } else {
      on = true;
      row = t.parts == 1 ? item : item / t.parts;
      c0 = (item - row * t.parts) * t.part_len;
      len = (int)min(t.part_len, t.codes - c0);
    }
    p = t.logits + row * t.stride + c0;
    shift = (int)(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
    constexpr int kSlice = L * tile_elems<T>();
    slices = L < 32 ? 1 : (len + shift + kSlice - 1) / kSlice;
  }
  __device__ __forceinline__ Slice<T, L> values(int lane32) const { return Slice<T, L>(len, shift, slice, lane32 % L); }
};

// Takes a warp through its items, slice by slice: work(place, buffer) once a slice is
// there (buffer: the lane's pieces); ahead(place) a slice's work before an item's first one (for loads that the
// item will want), turn() between the last slice of an item and the next item.
template <typename T, int L, typename Ahead, typename Turn, typename Work>
__device__ __forceinline__ void walk_tiles(const TileRows<T>& t, uint4* warp_buf, int lane32, Ahead&& ahead, Turn&& turn,
                                           Work&& work) {
  constexpr int kStage = kTilePieces * 32;
  uint4* buf = warp_buf + lane32;  // a lane's pieces lie 32 apart
  const int64_t step = (int64_t)gridDim.x * kTileWarps;
  const int64_t first = (int64_t)blockIdx.x * kTileWarps + threadIdx.x / 32;
  if (first >= t.items) return;
  TilePlace<T, L> now(t, first, lane32);
  ahead(now);
  turn();
  issue_slice<T, L>(buf, now.p, t.logits, now.values(lane32));
  cp_async_commit();
  int stage = 0;
  for (bool more = true; more;) {
    TilePlace<T, L> next = now;
    if (++next.slice == now.slices) {
      more = now.item + step < t.items;
      if (more) next = TilePlace<T, L>(t, now.item + step, lane32);
    }
    // The lane's accesses to the buffer that the copy goes to come before it.
    __syncwarp();
    if (more) issue_slice<T, L>(buf + (stage ^ 1) * kStage, next.p, t.logits, next.values(lane32));
    cp_async_commit();
    const bool new_item = more && next.slice == 0;
    if (new_item) ahead(next);
    cp_async_wait<1>();
    __syncwarp();
    work(now, buf + stage * kStage);
    if (new_item) turn();
    now = next;
    stage ^= 1;
  }
}

}  // namespace gsb
