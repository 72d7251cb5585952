// Log probability of a given code, entropy and largest alternatives of each row of
// assignment logits, and their gradient. The sums are those of code_rows.cuh.
//
// A -inf logit has probability 0. In a row of -inf only log p is -inf, H and the
// gradient are 0. NaN or +inf make a row's results NaN.
//
// Forward and backward, of these the forward: 65,536 x 4,096 fp32 with 4 alternatives 540
// to 566 and 230 us (4.7 TB/s), 2,047 x 50,001 fp16 157 and 55, 2^20 x 64 bf16 with 2 162
// and 71.
#include "code_tiles.cuh"

namespace gsb {
namespace {

constexpr int kGroupThreads = 256;

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

// The largest of a warp's keys.
__device__ __forceinline__ uint64_t warp_max(uint64_t key) {
  const uint32_t hi = __reduce_max_sync(kFullMask, (uint32_t)(key >> 32));
  const uint32_t lo = __reduce_max_sync(kFullMask, (uint32_t)(key >> 32) == hi ? (uint32_t)key : 0u);
  return (uint64_t)hi << 32 | lo;
}

// Alternatives of a row that L lanes have in `buf` (a slice holds it all), one by
// one: every lane has its own largest, taken out of the buffer; the row's largest of
// those is next, and its lane looks for another, through all its values again: 2^20 x 64
// bf16, forward, with 2, 8, 16 and 32 alternatives 77, 131, 219 and 512 us.
template <typename T, int L>
__device__ __forceinline__ void pick_alternatives(const LaneBuf& buf, int lane, const TilePlace<T, L>& now,
                                                  const Slice<T, L>& at, const RowStat& own, const RowResult& q,
                                                  const LogProbsOut& o, int top_k) {
  constexpr int VEC = wide_of<T>();
  uint64_t best = own.a == 0xffffffffu ? 0 : order_key(own.m, own.a);
  int nan_from = 0;
  // What is out is NaN from here on.
  if (at.ragged()) fill_ragged(buf, at, quiet_nan());
  if (best != 0) {
    const int k = (int)own.a - at.first;  // pieces lie L VEC apart
    reinterpret_cast<T*>(&buf[k / (L * VEC)])[k % (L * VEC)] = from_f32<T>(quiet_nan());
  }
  for (int j = 0;; ++j) {
    uint64_t row_best = best;
#pragma unroll
    for (int d = L / 2; d > 0; d >>= 1) {
      const uint64_t u = __shfl_xor_sync(kFullMask, row_best, d, L);
      row_best = u > row_best ? u : row_best;
    }
    if (now.on && lane == 0) {
      uint32_t c = key_index(row_best);
      float z = key_value(row_best);
      if (row_best == 0) {  // NaN alone is left, from the lowest index on
        while (nan_from < at.len - 1 && to_f32(now.p[nan_from]) == to_f32(now.p[nan_from])) ++nan_from;
        c = (uint32_t)nan_from++;
        z = quiet_nan();
      }
      o.top_codes[now.row * top_k + j] = (int32_t)c;
      o.top_log_probs[now.row * top_k + j] = q.log_p(z);
    }
    if (j + 1 == top_k) break;
    if (best == row_best && best != 0) {
      const LaneTop top = lane_top(buf, at, [](int, float) {});
      best = 0;
      if (top.m == top.m) {
        int v, i;
        float rest;
        find_value<T>(buf, top.group, top.m, &v, &i, &rest);
        best = order_key(top.m, (uint32_t)(at.at(v) + i));
        reinterpret_cast<T*>(&buf[v])[i] = from_f32<T>(quiet_nan());
      }
    }
  }
}

// The k largest keys of a part of a row, to put(rank, key). k lanes hold a value of
// at least the k-th largest of the lanes' maxima, so none of the k largest is below
// that. As a rule (4 alternatives: four rows in five) no lane's second value reaches
// it, and the lanes' maxima are all there is to rank. Else those lanes read the groups
// of pieces that reach it again (they come from L2), and the few values that do are
// listed and ranked against one another. Many equal values can overrun the list: then
// the part is searched once for each key.
constexpr int kTopList = 128;
// 128 registers a thread: with 80, for 6 blocks, the same kernels took 654 / 170 / 185 us
// where these took 615 / 164 / 170 (65,536 x 4,096 fp32, 2,047 x 50,001 fp16 and 2^20 x 64
// bf16, forward and backward, before later steps).
constexpr int kLogProbsBlocksSM = 4;
constexpr int kTopSlices = 2;  // of a part with more than one alternative
constexpr int kTopGroups = kTopSlices * kTilePieces / kTileGroup;
struct TopSmem {
  float top[kTopGroups][32];
  uint64_t list[kTopList];
  int count;
};
template <typename T, typename Put>
__device__ __forceinline__ void list_alternatives(const TilePlace<T, 32>& now, int lane, const RowStat& own,
                                                  float second, int k, TopSmem& sm, Put&& put) {
  constexpr int VEC = wide_of<T>();
  constexpr int kGroups = kTilePieces / kTileGroup;  // of a slice
  uint32_t left = order_bits(own.m), bound = 0;
  for (int j = 0; j < k; ++j) {
    bound = __reduce_max_sync(kFullMask, left);
    const uint32_t who = __ballot_sync(kFullMask, left == bound);
    if (lane == __ffs(who) - 1) left = 0;
  }
  const float least = key_value((uint64_t)bound << 32);
  const bool again = second >= least;
  const uint64_t own_key = order_key(own.m, own.a);
  const bool single = own.m >= least && own.a != 0xffffffffu;  // a lane without a value has m = -inf
  if (!__any_sync(kFullMask, again)) {
    const uint32_t who = __ballot_sync(kFullMask, single);
    if (__popc(who) >= k) {
      int rank = 0;
      for (uint32_t w = who; w != 0; w &= w - 1) rank += __shfl_sync(kFullMask, own_key, __ffs(w) - 1) > own_key;
      if (single && rank < k) put(rank, own_key);
      return;
    }
  }
  if (lane == 0) sm.count = 0;
  __syncwarp();
  uint32_t mine = 0;  // the lane's groups that reach it
  if (again) {
#pragma unroll
    for (int g = 0; g < kTopGroups; ++g)
      if (g < now.slices * kGroups && sm.top[g][lane] >= least) mine |= 1u << g;
  } else if (single) {
    const int to = atomicAdd(&sm.count, 1);
    if (to < kTopList) sm.list[to] = own_key;
  }
  for (; mine != 0; mine &= mine - 1) {
    const int g = __ffs(mine) - 1;
    const Slice<T, 32> at(now.len, now.shift, g / kGroups, lane);
    const int v0 = g % kGroups * kTileGroup;
    uint4 q[kTileGroup];
#pragma unroll
    for (int v = 0; v < kTileGroup; ++v) {
      const int c = at.at(v0 + v);
      Piece<T> e;
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(quiet_nan());
      q[v] = e.bits();
      if (c >= 0 && c + VEC <= at.len) {
        q[v] = *reinterpret_cast<const uint4*>(now.p + c);
      } else if (c < at.len && c + VEC > 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (at.has(c + i)) e[i] = now.p[c + i];
        q[v] = e.bits();
      }
    }
#pragma unroll
    for (int v = 0; v < kTileGroup; ++v) {
      if (Range<T>(q[v]).top() >= least) {
        float f[VEC];
        unpack<T>(q[v], f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          if (f[i] >= least) {
            const int to = atomicAdd(&sm.count, 1);
            if (to < kTopList) sm.list[to] = order_key(f[i], (uint32_t)(now.c0 + at.at(v0 + v) + i));
          }
        }
      }
    }
  }
  __syncwarp();
  const int n = sm.count;
  if (n >= k && n <= kTopList) {
    for (int i = lane; i < n; i += 32) {
      const uint64_t key = sm.list[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += sm.list[j] > key;
      if (rank < k) put(rank, key);
    }
  } else {
    uint64_t limit = ~uint64_t(0);
    for (int j = 0; j < k; ++j) {
      uint64_t best = 0;
      for (int c = lane; c < now.len; c += 32) {
        const uint64_t key = order_key(to_f32(now.p[c]), (uint32_t)(now.c0 + c));
        if (key < limit && key > best) best = key;
      }
      limit = best = warp_max(best);
      if (lane == 0) put(j, best);
    }
  }
  __syncwarp();
}

// parts > 1: a part's sums and keys go to `stat` and `keys` for k_log_probs_join.
template <typename T, int L>
__global__ void __launch_bounds__(kTileWarps * 32, kLogProbsBlocksSM)
    k_log_probs(TileRows<T> t, Codes codes, int top_k, LogProbsOut o, float4* __restrict__ stat,
                uint64_t* __restrict__ keys, uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ uint4 s_buf[];  // the warps' buffers, then (L = 32, top_k > 1) a TopSmem each
  const int warp = threadIdx.x / 32, lane32 = threadIdx.x % 32, lane = lane32 % L;
  TopSmem* tops = reinterpret_cast<TopSmem*>(s_buf + kTileWarps * kTilePieces * 32) + warp;
  int64_t code = -1;
  float zc = 0.0f;
  const bool given = o.log_probs != nullptr && (L < 32 || t.parts == 1);
  RowStat sums;
  float second = 0.0f;
  walk_tiles<T, L>(
      t, s_buf + warp * kTilePieces * 32, lane32, L < 32 && top_k > 1,
      [&](const TilePlace<T, L>& place) {
        if (given) code = codes.at(place.row);
      },
      [&](const TilePlace<T, L>& now, int slice, const Slice<T, L>& at, const LaneBuf& buf, auto&& refill) {
        if (slice == 0) {
          if (code >= t.codes) {
            if (now.on && lane == 0) bad_code(status, kSiteCode);
            code = -1;
          }
          zc = code >= 0 ? to_f32(now.p[code]) : 0.0f;
        }
        float next_best;
        RowStat r = lane_sums<false>(
            buf, at, Counts{}, next_best,
            [&](int v0, float top) {
              if (L == 32 && top_k > 1)
                tops->top[slice * (kTilePieces / kTileGroup) + v0 / kTileGroup][lane32] = top;
            },
            refill);
        if (L == 32 && r.a != 0xffffffffu) r.a += (uint32_t)now.c0;
        second = slice == 0 ? next_best : fmaxf(fmaxf(second, next_best), fminf(sums.m, r.m));
        sums = slice == 0 ? r : join<false>(sums, r);
      },
      [&](const TilePlace<T, L>& now, const Slice<T, L>& at, const LaneBuf& buf) {
        RowStat r = join_lanes<false, L>(sums);
        const bool nan_alone = r.a == 0xffffffffu;
        if (L < 32 || t.parts == 1) {
          const RowResult q = finish(r);
          if (now.on && lane == 0) {
            write_row(o, now.row, r, q, code, code >= 0, zc);
            if (top_k == 1) {
              o.top_codes[now.row] = nan_alone ? 0 : (int32_t)r.a;
              o.top_log_probs[now.row] = q.log_p(r.m);
            }
          }
          if (top_k > 1) {
            if constexpr (L < 32)
              pick_alternatives<T, L>(buf, lane, now, at, sums, q, o, top_k);
            else
              list_alternatives(now, lane32, sums, second, top_k, *tops, [&](int j, uint64_t key) {
                o.top_codes[now.row * top_k + j] = (int32_t)key_index(key);
                o.top_log_probs[now.row * top_k + j] = q.log_p(key_value(key));
              });
          }
        } else if constexpr (L == 32) {
          if (lane32 == 0) stat[now.item] = make_float4(r.m, r.s, r.w, __uint_as_float(r.a));
          uint64_t* to = keys + now.item * top_k;
          if (top_k == 1 && lane32 == 0)
            to[0] = nan_alone ? order_key(quiet_nan(), (uint32_t)now.c0) : order_key(r.m, r.a);
          if (top_k > 1) {
            const int k = min(top_k, now.len);
            list_alternatives(now, lane32, sums, second, k, *tops, [&](int j, uint64_t key) { to[j] = key; });
            for (int j = k + lane32; j < top_k; j += 32) to[j] = 0;  // a short last part
          }
        }
      });
}

// Parts of a call with more than one alternative have kTopSlices slices at most.
TilePlan log_probs_plan(int64_t rows, int64_t codes, int size, bool shifted, int top_k) {
  return tile_plan(rows, codes, size, shifted, top_k > 1 ? kTopSlices : 1 << 20, kLogProbsBlocksSM,
                   kLogProbsBlocksSM);
}

// One warp per row joins its parts' sums and picks the largest of their keys, which it
// keeps in registers where they are few. Latency alone: a call on 1 x 65,536 bf16 with 8
// alternatives, both kernels, takes 9.3 us (12.0 with the keys in shared memory).
constexpr int kJoinKeys = 16;  // a lane
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
  // A lane without a part adds nothing: -inf at an index behind all.
  RowStat r{neg_inf(), 0.0f, 0.0f, 0.0f, 0xffffffffu};
#pragma unroll 4
  for (int i = lane; i < parts; i += 32) r = join<false>(r, stat_at(i));
  r = join_lanes<false, 32>(r);
  const RowResult q = finish(r);
  if (lane == 0) write_row(o, row, r, q, code, code >= 0, zc);
  const uint64_t* ks = keys + row * parts * top_k;
  const int n = parts * top_k;
  const bool few = n <= kJoinKeys * 32;
  uint64_t own[kJoinKeys];
#pragma unroll
  for (int i = 0; i < kJoinKeys; ++i) own[i] = few && lane + 32 * i < n ? ks[lane + 32 * i] : 0;
  uint64_t limit = ~uint64_t(0);
  for (int j = 0; j < top_k; ++j) {
    uint64_t best = 0;
    if (few) {
#pragma unroll
      for (int i = 0; i < kJoinKeys; ++i)
        if (own[i] < limit && own[i] > best) best = own[i];
    } else {
      for (int i = lane; i < n; i += 32) {
        const uint64_t key = ks[i];
        if (key < limit && key > best) best = key;
      }
    }
    limit = best = warp_max(best);
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
// given code and the alternatives. The places c_i are written a second time, with
// (sum of their g_i) (1 - p_c) - (sum of the other g_i) p_c for the sum.
// Bound by the logits' and the gradient's bytes.
struct RowGrad {
  float4 st;
  float inv, gl, gh, lead;
  int64_t code;
  bool empty;
  __device__ __forceinline__ RowGrad(const LogProbsIn& in, int64_t row, int64_t C) {
    st = in.stats[row];
    code = in.g_log_probs ? in.codes.at(row) : -1;
    if (code >= C) code = -1;
    gl = in.g_log_probs ? in.g_log_probs[row] : 0.0f;
    if (code < 0) gl = 0.0f;
    gh = in.g_entropy ? in.g_entropy[row] : 0.0f;
    lead = gl;
    for (int j = 0; j < in.top_k; ++j) lead += in.g_top[row * in.top_k + j];
    empty = st.x == neg_inf() && st.y == st.y;
    inv = 1.0f / (1.0f + st.y);
  }
  // p (-lead - gH (x - mu)) = e (alpha + beta x)
  __device__ __forceinline__ float beta() const { return -gh * inv; }
  __device__ __forceinline__ float alpha() const { return (gh * st.z - lead) * inv; }
};
// The second writing of a place: alternative j, or (j = top_k) the given code where it
// is none of the alternatives. Its loads can be made ahead. Each place adds up the others'
// gradients anew, k^2 loads a row, which shows from 16 alternatives on: 2, 8, 16 and 32
// take 90, 211, 778 and 4,660 us at 2^20 x 64 bf16 (a lane a row), 61, 78, 113 and 385 at
// 65,536 x 512 fp32.
struct Special {
  int64_t c;  // -1: none
  float own, others, z;
  template <typename T>
  __device__ __forceinline__ Special(const LogProbsIn& in, const RowGrad& g, int64_t row, int64_t C, int j,
                                     const T* __restrict__ p) {
    const int k = in.top_k;
    c = -1;
    own = others = z = 0.0f;
    if (j > k || g.empty) return;
    const int32_t* tc = in.top_codes + row * k;
    const float* gt = in.g_top + row * k;
    c = j < k ? (int64_t)tc[j] : g.code;
    if (c >= C) c = -1;
    own = c == g.code ? g.gl : 0.0f;
    others = c == g.code ? 0.0f : g.gl;
    for (int i = 0; i < k; ++i) {
      if (j == k && (int64_t)tc[i] == c) c = -1;
      if (i == j) own += gt[i];
      else others += gt[i];
    }
    z = c >= 0 ? to_f32(p[c]) : 0.0f;
  }
  template <typename T>
  __device__ __forceinline__ void write(const RowGrad& g, T* __restrict__ dz) const {
    const float x = z - g.st.x;
    const float pr = ex2_approx(x * kLog2e) * g.inv;
    const float not_p = x == 0.0f ? g.st.y * g.inv : 1.0f - pr;
    const float h = pr == 0.0f ? 0.0f : g.gh * pr * (x - g.st.z);
    dz[c] = from_f32<T>(own * not_p - others * pr - h);
  }
};

// The factor of y = x log2 e in a row's gradient, b2, up to which the short way of
// row_grad holds: beside it y, at least kLowestGrad log2 e, makes no product beyond fp32
// (1e19 x 1.5e18; a masked place has e = 0, and 0 times infinity is NaN). Larger ones come
// of incoming gradients above 1e19.
constexpr float kLowestGrad = -1e18f;
constexpr float kLargestFactor = 1e19f;

// e (alpha + beta x) of a lane's values, in place (far: Base does not hold, or b2 is too
// large); 0 wherever e is, at -inf and at any value far enough below m.
__device__ __forceinline__ void row_grad(float (&z)[kRowElems], bool far, float m, float alpha, float beta,
                                         float neg_M, float a2, float b2) {
  if (__any_sync(kFullMask, far || lane_min(z) < kLowestGrad)) {
#pragma unroll
    for (int i = 0; i < kRowElems; ++i) {
      const float x = max_nan(z[i] - m, -128.0f);  // e is 0, and beta x finite up to beta = 2.6e36
      z[i] = ex2_approx(x * kLog2e) * fmaf(beta, x, alpha);
    }
  } else {
    const F2 l2 = f2(kLog2e), M2 = f2(neg_M), B = f2(b2), A = f2(a2);
#pragma unroll
    for (int i = 0; i < kRowElems; i += 2) {
      const F2 y = fma2(f2(z[i], z[i + 1]), l2, M2);
      float y0, y1;
      split(y, y0, y1);
      split(mul2(f2(ex2_approx(y0), ex2_approx(y1)), fma2(B, y, A)), z[i], z[i + 1]);
    }
  }
}

// Rows of up to 512 codes, 32 to a warp: what a row costs besides its values is done
// for 32 rows at once, a lane each; then L lanes a row go through the values of 32 / L
// rows at a time. 2^20 x 64 bf16: 86 us for 311 MB (134 twice, 43 of what belongs to the
// rows), 3.6 TB/s; the latency of the loads, with 64 registers a thread.
template <typename T, Mode M, bool SAME, int L>
__global__ void __launch_bounds__(kGroupThreads, kRowThreadsSM / kGroupThreads)
    k_log_probs_bwd_group(int64_t rows, int C, const T* __restrict__ logits, int64_t stride, LogProbsIn in,
                          T* __restrict__ g_logits) {
  pdl_wait();
  pdl_trigger();
  const int lane32 = threadIdx.x % 32, lane = lane32 % L;
  const int64_t row0 = ((int64_t)blockIdx.x * kGroupThreads + threadIdx.x) / 32 * 32;
  if (row0 >= rows) return;
  const int64_t own = min(row0 + lane32, rows - 1);
  const RowGrad g(in, own, C);
  const Base base(g.st.x);
  const float beta = g.beta(), alpha = g.alpha(), beta2 = beta * kLn2;
  const float b2 = beta2 * base.undo, a2 = (alpha - beta2 * base.d) * base.undo;
  const bool far = (base.far || !(fabsf(b2) <= kLargestFactor)) && !g.empty;  // an empty row's values are not used
#pragma unroll 1
  for (int h = 0; h < L; ++h) {
    const int from = h * (32 / L) + lane32 / L;
    if (row0 + h * (32 / L) >= rows) break;
    const int64_t row = min(row0 + from, rows - 1);
    const bool on = row0 + from < rows;
    const T* p = logits + row * stride;
    T* dz = g_logits + row * C;
    const int shift = shift_of<T, M>(dz);
    const Deal<T, M> at(shift, C + shift, L, lane);
    float z[kRowElems];
    if constexpr (SAME) load_row(p - shift, at, z);
    else load_row_single(p - shift, at, z);
    auto of = [&](float v) { return __shfl_sync(kFullMask, v, from); };
    const bool empty = __shfl_sync(kFullMask, g.empty, from);
    row_grad(z, __shfl_sync(kFullMask, far, from), of(g.st.x), of(alpha), of(beta), of(base.neg_M), of(a2), of(b2));
    if (empty) {
#pragma unroll
      for (int i = 0; i < kRowElems; ++i) z[i] = 0.0f;
    }
    if (on) store_row(dz - shift, at, z);
  }
  __syncwarp();  // the second writing comes after the first
  if (row0 + lane32 >= rows) return;
  auto special = [&](int j) { return Special(in, g, own, C, j, logits + own * stride); };
  auto write = [&](const Special& sp) {
    if (sp.c >= 0) sp.write(g, g_logits + own * C);
  };
  for (int j = 0; j <= in.top_k; j += 3) {  // the loads of three places at once
    const Special s0 = special(j), s1 = special(j + 1), s2 = special(j + 2);
    write(s0), write(s1), write(s2);
  }
}

// Longer rows: W warps a stretch of the result (SAME: the logits' rows lie alike).
// 16,384 x 4,096 fp32: 92 us, 5.8 TB/s; 2,047 x 50,001 fp16, rows between 16-byte
// boundaries, 105 us, 3.9 TB/s: half of the issue slots and a quarter of the DRAM rate, so
// the latency of what a thread does in turn (16,384 x 16,383 fp16 342 us, x 16,384 261).
template <typename T, Mode M, bool SAME, int W>
__global__ void __launch_bounds__(W * 32, kRowThreadsSM / (W * 32))
    k_log_probs_bwd_block(int64_t items, int64_t C, int parts, int part_len, const T* __restrict__ logits,
                          int64_t stride, LogProbsIn in, T* __restrict__ g_logits) {
  pdl_wait();
  pdl_trigger();
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = parts == 1 ? item : item / parts;
    const T* p = logits + row * stride;
    T* dz = g_logits + row * C;
    const int shift = shift_of<T, M>(dz), part = (int)(item - row * parts);
    const int c0 = part * part_len - shift;  // the code of place 0
    const int hi = (int)min((int64_t)part_len, C - c0), lo = part == 0 ? shift : 0;
    const Deal<T, M> at(lo, hi, W * 32, threadIdx.x);
    float z[kRowElems];
    if constexpr (SAME) load_row(p + c0, at, z);
    else load_row_single(p + c0, at, z);
    const RowGrad g(in, row, C);
    const Special sp(in, g, row, C, (int)threadIdx.x, p);
    const Base base(g.st.x);
    const float beta = g.beta(), alpha = g.alpha(), beta2 = beta * kLn2;
    const float b2 = beta2 * base.undo, a2 = (alpha - beta2 * base.d) * base.undo;
    const bool far = (base.far || !(fabsf(b2) <= kLargestFactor)) && !g.empty;
    row_grad(z, far, g.st.x, alpha, beta, base.neg_M, a2, b2);
    if (g.empty) {
#pragma unroll
      for (int i = 0; i < kRowElems; ++i) z[i] = 0.0f;
    }
    store_row(dz + c0, at, z);
    __syncthreads();  // the second writing comes after the first
    if (sp.c >= max(c0, 0) && sp.c < c0 + hi) sp.write(g, dz);
    if (W == 1 && in.top_k == 32 && threadIdx.x == 0) {  // one place more than threads
      const Special more(in, g, row, C, 32, p);
      if (more.c >= max(c0, 0) && more.c < c0 + hi) more.write(g, dz);
    }
  }
}

struct LogProbsScratch {
  float4* stat = nullptr;
  uint64_t* keys = nullptr;
};
LogProbsScratch carve(Carver& ws, int64_t rows, const TilePlan& plan, int top_k) {
  LogProbsScratch b;
  if (plan.parts > 1) {
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
  size_t need = 0;
  for (int size = 2; size <= 4; size += 2) {
    for (int shifted = 0; shifted < 2; ++shifted) {
      Carver c(nullptr);
      carve(c, rows, log_probs_plan(rows, codebook_rows, size, shifted, top_k), top_k);
      need = std::max(need, c.off);
    }
  }
  return need;
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
  if (reinterpret_cast<uintptr_t>(stats) % 16 != 0) return GSB_ERR_INVALID_ARGUMENT;
  const size_t need = gsb_code_log_probs_workspace_size(rows, codebook_rows, top_k);
  if (need > 0 && (!workspace || workspace_bytes < need)) return GSB_ERR_WORKSPACE;
  if (rows == 1) logits_stride = 0;
  const TilePlan plan = log_probs_plan(rows, codebook_rows, dtype_bytes(dtype),
                                       rows_shifted(dtype_bytes(dtype), logits, logits_stride), top_k);
  Carver ws(workspace);
  const LogProbsScratch b = carve(ws, rows, plan, top_k);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Codes cd{codes, code_bytes == 8};
  const LogProbsOut o{log_probs, entropy, top_log_probs, top_codes, (float4*)stats};
  with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    const int64_t items = plan.items(rows);
    const TileRows<T> t{(const T*)logits, logits_stride, rows, codebook_rows, plan.part_len, items, plan.parts};
    const size_t smem = kTileWarps * (kTilePieces * 32 * sizeof(uint4) +
                                      (plan.lanes == 32 && top_k > 1 ? sizeof(TopSmem) : 0));
    with_tile_lanes(plan.lanes, [&](auto l) {
      launch_pdl(k_log_probs<T, decltype(l)::value>, plan.blocks(rows), kTileWarps * 32, smem, s, t, cd, top_k, o,
                 b.stat, b.keys, status);
    });
    if (plan.parts > 1) {
      launch_pdl(k_log_probs_join<T>, grid1d(rows * 32, 128), 128, 0, s, rows, codebook_rows, plan.parts,
                 (const T*)logits, logits_stride, cd, top_k, (const float4*)b.stat, (const uint64_t*)b.keys, o,
                 status);
      note_launches(1);
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
  if (reinterpret_cast<uintptr_t>(stats) % 16 != 0) return GSB_ERR_INVALID_ARGUMENT;
  if (!logits || !stats || !g_logits || (g_log_probs && !codes) || (g_top_log_probs && top_k > 0 && !top_codes))
    return GSB_ERR_INVALID_ARGUMENT;
  if (rows == 1) logits_stride = codebook_rows;  // as the result's
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const LogProbsIn in{Codes{codes, code_bytes == 8}, g_top_log_probs ? top_k : 0, top_codes, (const float4*)stats,
                      g_log_probs, g_entropy, g_top_log_probs};
  with_row_pairs(dtype, logits, logits_stride, g_logits, codebook_rows, [&](auto t, auto m, auto same) {
    using T = decltype(t);
    constexpr Mode M = decltype(m)::value;
    constexpr bool SAME = decltype(same)::value;
    const RowPlan plan = row_plan(rows, codebook_rows, M == Mode::kShifted, Deal<T, M>::VEC);
    if (plan.lanes > 0) {
      with_lanes(plan.lanes, [&](auto l) {
        constexpr int L = decltype(l)::value;
        launch_pdl(k_log_probs_bwd_group<T, M, SAME, L>, grid1d(rows, kGroupThreads), kGroupThreads, 0, s, rows,
                   (int)codebook_rows, (const T*)logits, logits_stride, in, (T*)g_logits);
      });
    } else {
      with_warps(plan.warps, [&](auto w) {
        constexpr int W = decltype(w)::value;
        launch_pdl(k_log_probs_bwd_block<T, M, SAME, W>, item_grid(rows * plan.parts), W * 32, 0, s,
                   rows * plan.parts, codebook_rows, plan.parts, plan.part_len, (const T*)logits, logits_stride, in,
                   (T*)g_logits);
      });
    }
  });
  note_launches(1);
  return cuda_status(cudaGetLastError());
}
