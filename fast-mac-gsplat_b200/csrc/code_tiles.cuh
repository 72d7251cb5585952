// The forward half of the row-wise operators on assignment logits: softmax sums of
// rows that stream through shared memory.
//
// A warp owns its rows from the first load to the result: no block-wide barrier.
//   - L = 1 .. 16 lanes a row, 32 / L rows at once, for rows that fit 16 pieces of 16
//     bytes a lane (what a row costs besides its values is paid once for all of them);
//   - L = 32 for longer rows (or parts of a row), which pass in slices of 16 pieces a
//     lane; every lane keeps its own maximum and sums over the slices, so that lanes
//     exchange values once a row.
// Pieces are copied asynchronously and each lane reads only what it copied itself,
// which needs no barrier either. A warp's buffer is refilled from the next slice four
// pieces at a time as the sums pass over it. Shared memory also gives a lane's values
// an index: the largest one is found by piece and taken out of the sums by one store,
// where values in registers cost a comparison and a selection each.
//
// Bound by the logits' bytes while a value costs no more than a few instructions: a
// maximum and a minimum (of two values at a time for 16-bit types), a conversion, and
// half of each of an FMA, an addition and an FMA on pairs around one ex2. What is reached
// is below both bounds: half of the issue slots and 55 to 60 % of nominal DRAM rate
// with fp32, 27 to 33 % with 16-bit types, 4 or 6 blocks an SM (registers) hiding latency.
#pragma once

#include "code_rows.cuh"

namespace gsb {

constexpr int kTileWarps = 4;    // a block
constexpr int kTilePieces = 16;  // of a lane
// Pieces that are worked on and refilled together. With 8, 0 to 30 % longer (2^20 x 256
// bf16, balance loss and gradient: 437 us against 337), with 2, 0 to 8 %.
constexpr int kTileGroup = 4;

// Where a lane's values of a slice lie: piece v's value i has the index at(v) + i in
// its part (or row) of len values. shift: values between the 16-byte boundary before
// the part and its start. Pieces w0 .. w1 - 1 are whole for every lane of the row; of
// the n (a multiple of kTileGroup) in work, the others are ragged or empty.
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
    constexpr int kGroupValues = L * VEC * kTileGroup;
    n = min((left + kGroupValues - 1) / kGroupValues * kTileGroup, kTilePieces);
    if (L < 32) n = __reduce_max_sync(kFullMask, n);  // rows may lie differently; a warp goes through as many pieces
  }
  __device__ __forceinline__ int at(int v) const { return first + v * L * VEC; }
  __device__ __forceinline__ bool has(int c) const { return c >= 0 && c < len; }
  __device__ __forceinline__ bool ragged() const { return w0 > 0 || w1 < n; }
  // Calls fn(v) for the pieces that are not whole.
  template <typename Fn>
  __device__ __forceinline__ void each_ragged(Fn&& fn) const {
    for (int v = w0 > 0 ? 0 : w1; v < n; v = v + 1 < w1 && v < w1 ? w1 : v + 1) fn(v);
  }
};

__device__ __forceinline__ void cp_async16_part(void* smem, const void* gmem, int bytes) {  // the rest is zeros
  const unsigned s = (unsigned)__cvta_generic_to_shared(smem);
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(s), "l"(gmem), "r"(bytes) : "memory");
}

// A lane's pieces in its warp's buffer; piece v of the lanes lie side by side.
struct LaneBuf {
  uint4* base;
  __device__ __forceinline__ uint4& operator[](int v) const { return base[v * 32]; }
};

// Begins the copy of the whole pieces v0 .. v0 + kTileGroup - 1 of a lane.
template <typename T, int L>
__device__ __forceinline__ void copy_group(const LaneBuf& buf, const T* __restrict__ p, const Slice<T, L>& at, int v0) {
  constexpr int VEC = wide_of<T>();
  const T* from = p + at.first + v0 * L * VEC;
  if (v0 >= at.w0 && v0 + kTileGroup <= at.w1) {
#pragma unroll
    for (int v = 0; v < kTileGroup; ++v) cp_async16(&buf[v0 + v], from + v * L * VEC);
  } else {
    for (int v = v0; v < v0 + kTileGroup; ++v)
      if (v >= at.w0 && v < at.w1) cp_async16(&buf[v], p + at.at(v));
  }
}
// Begins the copy of the ragged pieces. A piece may reach in front of its row, into
// the row before (its values are not used), but not in front of `base`, the logits'
// first value: the few values of such a piece are copied one by one.
template <typename T, int L>
__device__ __forceinline__ void copy_ragged(const LaneBuf& buf, const T* __restrict__ p, const T* __restrict__ base,
                                            const Slice<T, L>& at) {
  constexpr int VEC = wide_of<T>();
  if (!at.ragged()) return;
  at.each_ragged([&](int v) {
    const int c = at.at(v);
    uint4* to = &buf[v];
    if (c >= at.len || c + VEC <= 0) return;
    if (c < 0 && p + c < base) {
      for (int i = 0; i < VEC; ++i)
        if (at.has(c + i)) reinterpret_cast<T*>(to)[i] = p[c + i];
    } else {
      cp_async16_part(to, p + c, min(VEC, at.len - c) * (int)sizeof(T));
    }
  });
}
// Puts `value` in the places of ragged pieces that hold none of the part's values.
template <typename T, int L>
__device__ __forceinline__ void fill_ragged(const LaneBuf& buf, const Slice<T, L>& at, float value) {
  constexpr int VEC = wide_of<T>();
  Piece<T> e;
#pragma unroll
  for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(value);
  at.each_ragged([&](int v) {
    const int c = at.at(v);
    if (c >= at.len || c + VEC <= 0) {
      buf[v] = e.bits();
    } else if (c < 0 || c + VEC > at.len) {
      for (int i = 0; i < VEC; ++i)
        if (!at.has(c + i)) reinterpret_cast<T*>(&buf[v])[i] = e[0];
    }
  });
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& q, float (&f)[wide_of<T>()]) {
  const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
  for (int i = 0; i < wide_of<T>(); ++i) f[i] = to_f32(e[i]);
}

// Largest and smallest value (NaN loses against any) of pieces, 16-bit types two at a
// time.
template <typename T>
struct Range;
template <>
struct Range<float> {
  float hi, lo;
  __device__ __forceinline__ explicit Range(const uint4& q) {
    const float a = __uint_as_float(q.x), b = __uint_as_float(q.y), c = __uint_as_float(q.z),
                d = __uint_as_float(q.w);
    hi = fmaxf(max3(a, b, c), d);
    lo = fminf(min3(a, b, c), d);
  }
  __device__ __forceinline__ void add(const Range& r) { hi = fmaxf(hi, r.hi), lo = fminf(lo, r.lo); }
  __device__ __forceinline__ float top() const { return hi; }
  __device__ __forceinline__ float low() const { return lo; }
};
template <typename P>
struct PairRange {
  P hi, lo;
  __device__ __forceinline__ explicit PairRange(const uint4& q) {
    const P* e = reinterpret_cast<const P*>(&q);
    hi = __hmax2(__hmax2(e[0], e[1]), __hmax2(e[2], e[3]));
    lo = __hmin2(__hmin2(e[0], e[1]), __hmin2(e[2], e[3]));
  }
  __device__ __forceinline__ void add(const PairRange& r) { hi = __hmax2(hi, r.hi), lo = __hmin2(lo, r.lo); }
  __device__ __forceinline__ float top() const { return fmaxf(__low2float(hi), __high2float(hi)); }
  __device__ __forceinline__ float low() const { return fminf(__low2float(lo), __high2float(lo)); }
};
template <>
struct Range<__nv_bfloat16> : PairRange<__nv_bfloat162> {
  using PairRange::PairRange;
};
template <>
struct Range<__half> : PairRange<__half2> {
  using PairRange::PairRange;
};

// Counts of the values of the pieces v0 .. v0 + kTileGroup - 1; 0 where the part has none.
template <typename T, int L>
__device__ __forceinline__ void group_counts(const Counts& counts, const Slice<T, L>& at, const Counts::Offsets& off,
                                             int v0, float (&n)[kTileGroup][wide_of<T>()]) {
  constexpr int VEC = wide_of<T>();
  if (at.shift == 0 && v0 + kTileGroup <= at.w1) {
    const float4* p = reinterpret_cast<const float4*>(counts.by_code + at.at(v0));
#pragma unroll
    for (int v = 0; v < kTileGroup; ++v)
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        const float4 q = p[(v * L * VEC + i) / 4];
        n[v][i] = q.x, n[v][i + 1] = q.y, n[v][i + 2] = q.z, n[v][i + 3] = q.w;
      }
  } else if (v0 >= at.w0 && v0 + kTileGroup <= at.w1) {
    const int c = at.at(v0);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float* p = VEC == 8 ? counts.by_eight + (((c + at.shift) >> 3) + off.of[i % 8]) : counts.by_code + c + i;
#pragma unroll
      for (int v = 0; v < kTileGroup; ++v) n[v][i] = p[VEC == 8 ? v * L : v * L * VEC];
    }
  } else {
#pragma unroll
    for (int v = 0; v < kTileGroup; ++v) {
      const int c = at.at(v0 + v);
      if (VEC == 8 && v0 + v >= at.w0 && v0 + v < at.w1) {
        const float* p = counts.by_eight + ((c + at.shift) >> 3);
#pragma unroll
        for (int i = 0; i < VEC; ++i) n[v][i] = p[off.of[i % 8]];
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) n[v][i] = at.has(c + i) ? counts.by_code[c + i] : 0.0f;
      }
    }
  }
}

// The sums of a lane's pieces about base.m (r.n: the count that others are taken
// relative to). kClamp: some value is -inf, or so low that its multiple with log2 e
// is; e = 0 times that would be NaN. done(v) is called when pieces v .. v +
// kTileGroup - 1 are not needed any more.
template <bool kCounts, bool kClamp, typename T, int L, typename Done>
__device__ __forceinline__ void piece_sums(const LaneBuf& buf, const Slice<T, L>& at, const Counts& counts,
                                           const Base& base, RowStat& r, Done&& done) {
  constexpr int VEC = wide_of<T>();
  const F2 l2 = f2(kLog2e), neg_M = f2(base.neg_M), neg_n = f2(-r.n);
  F2 s2 = f2(0.0f), w2 = f2(0.0f);
  const Counts::Offsets off(counts, at.shift);
  for (int v0 = 0; v0 < at.n; v0 += kTileGroup) {
    float n[kTileGroup][VEC];
    if constexpr (kCounts) group_counts(counts, at, off, v0, n);
#pragma unroll
    for (int v = 0; v < kTileGroup; ++v) {
      float f[VEC];
      unpack<T>(buf[v0 + v], f);
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
        w2 = fma2(e, kCounts ? add2(f2(n[v][i], n[v][i + 1]), neg_n) : y, w2);
      }
    }
    done(v0);
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

// The largest of a lane's pieces: its value (NaN: there is none) and group, the
// largest of the other groups, and the smallest. group_top(v, top) is told each
// group's largest.
struct LaneTop {
  float m, rest, low;
  int group;
};
template <typename T, int L, typename GroupTop>
__device__ __forceinline__ LaneTop lane_top(const LaneBuf& buf, const Slice<T, L>& at, GroupTop&& group_top) {
  LaneTop t{quiet_nan(), quiet_nan(), 0.0f, 0};
  for (int v0 = 0; v0 < at.n; v0 += kTileGroup) {
    Range<T> range(buf[v0]);
#pragma unroll
    for (int v = 1; v < kTileGroup; ++v) range.add(Range<T>(buf[v0 + v]));
    const float top = range.top();
    t.low = fminf(t.low, range.low());
    const bool first = top > t.m || t.m != t.m;  // the first of equal ones
    t.rest = fmaxf(t.rest, first ? t.m : top);
    if (first) t.m = top, t.group = v0;
    group_top(v0, top);
  }
  return t;
}
// The first place of the value m in a group of a lane's pieces, and the largest of
// the group's other values.
template <typename T>
__device__ __forceinline__ void find_value(const LaneBuf& buf, int v0, float m, int* v_out, int* i_out, float* rest) {
  constexpr int VEC = wide_of<T>();
  float top[kTileGroup];
#pragma unroll
  for (int v = 0; v < kTileGroup; ++v) top[v] = Range<T>(buf[v0 + v]).top();
  int v_at = kTileGroup - 1;
#pragma unroll
  for (int v = kTileGroup - 2; v >= 0; --v)
    if (top[v] == m) v_at = v;
  float f[VEC], other = quiet_nan();
#pragma unroll
  for (int v = 0; v < kTileGroup; ++v) other = fmaxf(other, v == v_at ? quiet_nan() : top[v]);
  unpack<T>(buf[v0 + v_at], f);
  int i_at = 0;
#pragma unroll
  for (int i = VEC - 1; i >= 0; --i)
    if (f[i] == m) i_at = i;
#pragma unroll
  for (int i = 0; i < VEC; ++i) other = fmaxf(other, i == i_at ? quiet_nan() : f[i]);
  *v_out = v0 + v_at;
  *i_out = i_at;
  *rest = other;
}

// The softmax sums of one lane's values of a slice, without its largest (its first
// largest, which leaves `buf` too). The index in the result is the part's. second: the
// largest of the others (NaN: none).
template <bool kCounts, typename T, int L, typename GroupTop, typename Done>
__device__ __forceinline__ RowStat lane_sums(const LaneBuf& buf, const Slice<T, L>& at, const Counts& counts,
                                             float& second, GroupTop&& group_top, Done&& done) {
  constexpr int VEC = wide_of<T>();
  if (at.ragged()) fill_ragged(buf, at, quiet_nan());
  const LaneTop top = lane_top(buf, at, group_top);
  RowStat r;
  const bool some = top.m == top.m;                   // else: no value, or NaN alone
  const Base base(top.m > neg_inf() ? top.m : 0.0f);  // with m = -inf all is 0 (or NaN) relative to 0 too
  const float none = base.far ? neg_inf() : base.m - 200.0f;  // adds nothing
  r.a = 0xffffffffu;
  second = quiet_nan();
  if (some) {
    int v, i;
    find_value<T>(buf, top.group, top.m, &v, &i, &second);
    second = fmaxf(second, top.rest);
    reinterpret_cast<T*>(&buf[v])[i] = from_f32<T>(none);
    r.a = (uint32_t)(at.at(v) + i);
  }
  if (at.ragged()) fill_ragged(buf, at, none);
  r.n = kCounts && some ? counts.by_code[r.a] : 0.0f;
  if (__any_sync(kFullMask, base.far)) {
    r.s = r.w = 0.0f;
    const Counts::Offsets off(counts, at.shift);
    for (int v0 = 0; v0 < at.n; v0 += kTileGroup) {
      float n[kTileGroup][VEC];
      if constexpr (kCounts) group_counts(counts, at, off, v0, n);
#pragma unroll
      for (int v = 0; v < kTileGroup; ++v) {
        float f[VEC];
        unpack<T>(buf[v0 + v], f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float x = max_nan(f[i] - base.m, -200.0f);
          const float e = ex2_approx(x * kLog2e);
          r.s += e;
          r.w = fmaf(e, kCounts ? n[v][i] - r.n : x, r.w);
        }
      }
      done(v0);
    }
  } else if (!kCounts && __any_sync(kFullMask, top.low < kLowest)) {
    piece_sums<kCounts, !kCounts>(buf, at, counts, base, r, done);
  } else {
    piece_sums<kCounts, false>(buf, at, counts, base, r, done);
  }
  const bool lane_any = at.first < at.len && at.at(at.n - 1) + VEC > 0;
  r.m = some ? top.m : neg_inf();
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
  int blocks_sm = 1;
  int64_t part_len = 0;
  int blocks(int64_t rows) const {
    return (int)std::min<int64_t>(148 * blocks_sm, (items(rows) + kTileWarps - 1) / kTileWarps);
  }
  int64_t items(int64_t rows) const { return lanes < 32 ? (rows + 32 / lanes - 1) / (32 / lanes) : rows * parts; }
};
// Rows that fit 16 lanes share a warp (shifted: they may begin between 16-byte
// boundaries). Longer ones take a warp a part; there are as many parts as make the
// longest warp's way shortest, a part costing a quarter of a slice besides its
// values. most_slices: of a part; blocks_sm: blocks that an SM holds (of the kernels
// for short rows: blocks_sm_short).
inline TilePlan tile_plan(int64_t rows, int64_t codes, int size, bool shifted, int64_t most_slices, int blocks_sm,
                          int blocks_sm_short) {
  TilePlan p;
  rows = std::max<int64_t>(rows, 1);
  p.blocks_sm = blocks_sm;
  const int64_t resident = 148 * blocks_sm * kTileWarps;
  const int vec = 16 / size;
  p.part_len = codes;
  for (int l = 1; l <= 16; l *= 2) {
    if (codes + (shifted ? vec - 1 : 0) <= l * kTilePieces * vec) {
      p.lanes = l;
      p.blocks_sm = blocks_sm_short;
      return p;
    }
  }
  const int64_t slice = 32 * kTilePieces * vec, most = most_slices * slice - (shifted ? 8 : 0);
  const int64_t least_parts = (codes + most - 1) / most;
  const int64_t most_parts = std::max(least_parts, std::min<int64_t>((codes + slice / 4 - 1) / (slice / 4), 1024));
  int64_t best_cost = INT64_MAX, best = least_parts;
  auto consider = [&](int64_t parts) {
    const int64_t rounds = (rows * parts + resident - 1) / resident;
    const int64_t cost = rounds * ((codes + parts - 1) / parts + slice / 4) + (parts > 1 ? slice / 2 : 0);
    if (cost < best_cost) best_cost = cost, best = parts;
  };
  consider(least_parts);
  // Of the numbers of parts that make as many rounds the largest is best, or a smaller one
  // with parts as long. More than 16 rounds are even enough.
  for (int64_t rounds = (rows * least_parts + resident - 1) / resident; rounds <= 16; ++rounds) {
    const int64_t parts = std::min(most_parts, rounds * resident / rows), len = (codes + parts - 1) / parts;
    if (parts > least_parts) consider(std::max(least_parts, (codes + len - 1) / len));
    if (parts == most_parts) break;
  }
  p.part_len = ((codes + best - 1) / best + 7) / 8 * 8;
  p.parts = (int)((codes + p.part_len - 1) / p.part_len);
  return p;
}
template <typename Fn>
inline void with_tile_lanes(int lanes, Fn&& fn) {
  if (lanes == 1) fn(std::integral_constant<int, 1>{});
  else if (lanes == 2) fn(std::integral_constant<int, 2>{});
  else if (lanes == 4) fn(std::integral_constant<int, 4>{});
  else if (lanes == 8) fn(std::integral_constant<int, 8>{});
  else if (lanes == 16) fn(std::integral_constant<int, 16>{});
  else fn(std::integral_constant<int, 32>{});
}
inline bool rows_shifted(int size, const void* p, int64_t stride) {
  return reinterpret_cast<uintptr_t>(p) % 16 != 0 || stride * size % 16 != 0;
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
  int slices, len, shift;
  bool on;
  __device__ __forceinline__ TilePlace(const TileRows<T>& t, int64_t item_, int lane32) : item(item_) {
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
    constexpr int kSlice = L * kTilePieces * wide_of<T>();
    slices = L < 32 ? 1 : (len + shift + kSlice - 1) / kSlice;
  }
  __device__ __forceinline__ Slice<T, L> values(int slice, int lane32) const {
    return Slice<T, L>(len, shift, slice, lane32 % L);
  }
};

// Takes a warp through its items. For each: ahead(place), once, before the item's
// first copy is waited for (for loads that it will want); then for each slice
// work(place, slice, values, buffer, refill), whose refill is the `done` of lane_sums;
// last turn(place, values, buffer). hold: turn wants the last slice's values still; the
// next item's copy begins after it.
template <typename T, int L, typename Ahead, typename Work, typename Turn>
__device__ __forceinline__ void walk_tiles(const TileRows<T>& t, uint4* warp_buf, int lane32, bool hold, Ahead&& ahead,
                                           Work&& work, Turn&& turn) {
  const LaneBuf buf{warp_buf + lane32};
  const int64_t step = (int64_t)gridDim.x * kTileWarps;
  int64_t item = (int64_t)blockIdx.x * kTileWarps + threadIdx.x / 32;
  if (item >= t.items) return;
  TilePlace<T, L> now(t, item, lane32);
  Slice<T, L> at = now.values(0, lane32);
  // Groups from v0 on, and what is not whole.
  auto copy_rest = [&](const TilePlace<T, L>& place, const Slice<T, L>& values, int v0) {
    for (; v0 < values.n; v0 += kTileGroup) copy_group(buf, place.p, values, v0);
    copy_ragged(buf, place.p, t.logits, values);
    cp_async_commit();
  };
  ahead(now);
  copy_rest(now, at, 0);
  int slice = 0;
  for (bool more = true; more;) {
    cp_async_wait<0>();
    __syncwarp();
    const bool last = L < 32 || slice + 1 == now.slices;
    TilePlace<T, L> next = now;
    int next_slice = slice + 1;
    if (last) {
      item += step;
      more = item < t.items;
      next_slice = 0;
      if (more) next = TilePlace<T, L>(t, item, lane32);
    }
    const Slice<T, L> next_at = next.values(next_slice, lane32);
    const bool refill = more && !(hold && last);
    work(now, slice, at, buf, [&](int v0) {
      __syncwarp();  // what was read comes before the copy that replaces it
      if (refill) copy_group(buf, next.p, next_at, v0);
    });
    __syncwarp();
    if (refill) copy_rest(next, next_at, at.n);
    if (last) {
      turn(now, at, buf);
      __syncwarp();
      if (more && hold) copy_rest(next, next_at, 0);
      if (more) ahead(next);
    }
    now = next;
    at = next_at;
    slice = next_slice;
  }
}

}  // namespace gsb
