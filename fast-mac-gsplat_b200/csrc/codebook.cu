// Lookup of codebook rows and its gradients.
//
//   out[n, :] = scale * sum_j w[n, j] * table[code[n, j], :]
//   g_table[c, :] = scale * sum over (n, j) with code c of w[n, j] * g[n, :]
//   g_w[n, j] = scale * <g[n, :], table[code[n, j], :]>
//
// Sums are fp32, rounded once to the result's type. The table gradient sorts
// the codes (stable radix sort), so each row is a sum in a fixed order: the
// result does not depend on the timing of the blocks.
#include <algorithm>
#include <type_traits>

#include "code_types.cuh"
#include "radix_sort.cuh"

namespace gsb {
namespace {

// V values of a row at once: V = 4 where rows, strides and addresses allow it.
template <int V, typename T>
struct Vec {
  float v[V];
  __device__ __forceinline__ void load(const T* __restrict__ p) {
    if constexpr (V == 4 && sizeof(T) == 4) {
      const float4 q = *reinterpret_cast<const float4*>(p);
      v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
    } else if constexpr (V == 4) {
      const uint2 q = *reinterpret_cast<const uint2*>(p);
      const T* h = reinterpret_cast<const T*>(&q);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = to_f32(h[i]);
    } else {
      v[0] = to_f32(*p);
    }
  }
};
template <int V, typename T>
__device__ __forceinline__ void store_vec(T* __restrict__ p, const float (&v)[V]) {
  if constexpr (V == 4 && sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else if constexpr (V == 4) {
    uint2 q;
    T* h = reinterpret_cast<T*>(&q);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = from_f32<T>(v[i]);
    *reinterpret_cast<uint2*>(p) = q;
  } else {
    *p = from_f32<T>(v[0]);
  }
}

// One thread per V values of the result and kLookupItems such pieces, a block's
// width apart: stores of a warp are contiguous whatever the row's length, and the
// loads of the pieces overlap. A block's codes and weights go through shared memory
// (kStage; they are each wanted by every piece of a row) unless rows are so short that
// there are too many of them. Bound by the stores: the table comes from L2 and L1.
// 2^20 rows of 48, fp16 to fp32: 41 us, 5.0 TB/s (two pieces 47, eight 51; a fill of the
// result alone takes 30). Four of 27 bf16 for 100,003 rows: 13 us, 76 % of the issue slots
// (one load a value).
constexpr int kLookupItems = 4;
constexpr int kLookupPieces = 256 * kLookupItems;  // a block's
constexpr int kLookupSlots = 2048;                 // that are staged, at most
template <typename T, typename O, int V, bool kStage, bool kWeights>
__global__ void __launch_bounds__(256)
    k_lookup(int64_t pieces, int bag, int64_t C, int nvec, FastDiv div_nvec, const T* __restrict__ table,
             int64_t stride, Codes codes, const float* __restrict__ weights, float scale, O* __restrict__ out,
             uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  __shared__ int s_at[kStage ? kLookupSlots : 1];  // the row's first value (-1: no row)
  __shared__ float s_weight[kStage && kWeights ? kLookupSlots : 1];
  const int64_t tile = (int64_t)blockIdx.x * kLookupPieces;
  const int64_t row0 = tile / nvec;
  const int off0 = (int)(tile - row0 * nvec);
  auto row_at = [&](int64_t i) {
    const int64_t c = codes.at(i);
    if (c >= C) bad_code(status, kSiteCode);
    return c < 0 || c >= C ? (int64_t)-1 : c * stride;
  };
  const int count = (int)min((int64_t)kLookupPieces, pieces - tile);
  if (kStage) {
    const int n = (fast_div(off0 + count - 1, div_nvec) + 1) * bag;
    for (int i = threadIdx.x; i < n; i += 256) {
      s_at[i] = (int)row_at(row0 * bag + i);
      if (kWeights) s_weight[i] = weights[row0 * bag + i];
    }
    __syncthreads();
  }
  float acc[kLookupItems][V];
  int r[kLookupItems], d[kLookupItems];
#pragma unroll
  for (int k = 0; k < kLookupItems; ++k) {
    const int local = off0 + min(k * 256 + (int)threadIdx.x, count - 1);
    r[k] = fast_div(local, div_nvec);
    d[k] = (local - r[k] * nvec) * V;
    r[k] *= bag;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[k][i] = 0.0f;
  }
  for (int j = 0; j < bag; ++j) {
    Vec<V, T> t[kLookupItems];
    float w[kLookupItems];
#pragma unroll
    for (int k = 0; k < kLookupItems; ++k) {
#pragma unroll
      for (int i = 0; i < V; ++i) t[k].v[i] = 0.0f;
      w[k] = 0.0f;  // an empty slot adds nothing, whatever its weight is
      if constexpr (kStage) {
        const int at = s_at[r[k] + j];
        if (at >= 0) {
          t[k].load(table + (at + d[k]));
          w[k] = kWeights ? s_weight[r[k] + j] : 1.0f;
        }
      } else {
        const int64_t slot = row0 * bag + r[k] + j, at = row_at(slot);
        if (at >= 0) {
          t[k].load(table + (at + d[k]));
          w[k] = kWeights ? weights[slot] : 1.0f;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kLookupItems; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[k][i] = kWeights ? fmaf(w[k], t[k].v[i], acc[k][i]) : acc[k][i] + t[k].v[i];
  }
  O* to = out + tile * V;
#pragma unroll
  for (int k = 0; k < kLookupItems; ++k) {
    const int piece = k * 256 + (int)threadIdx.x;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[k][i] *= scale;
    if (piece < count) store_vec<V>(to + piece * V, acc[k]);
  }
}

// Sort key of slot i: its code, or C for an empty one (sorted behind every code).
__device__ __forceinline__ uint32_t code_key(const Codes& codes, int64_t i, int64_t C, uint32_t* status) {
  const int64_t c = codes.at(i);
  if (c >= C) bad_code(status, kSiteCode);
  return (c < 0 || c >= C) ? (uint32_t)C : (uint32_t)c;
}
// Zeroes the bytes of the table's gradient (rows that no code names stay 0).
__device__ __forceinline__ void zero_words(uint32_t* to, int64_t bytes) {
  const int64_t words = bytes / 4, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < words; i += step) to[i] = 0u;
  if (bytes % 4 != 0 && blockIdx.x == 0 && threadIdx.x == 0) reinterpret_cast<uint16_t*>(to)[words * 2] = 0;
}

// Keys and slots for the sort, and the counts of the keys' 8-bit digits that it needs: one
// pass over the codes, counted in shared memory. 2^20 codes, with 1.6 MB of gradient
// zeroed, 12 us.
constexpr int kKeyItems = 8;
__global__ void __launch_bounds__(256)
    k_code_keys(int64_t n, int64_t C, int passes, Codes codes, uint32_t* __restrict__ keys,
                uint32_t* __restrict__ vals, uint32_t* __restrict__ digits, uint32_t* __restrict__ zero,
                int64_t zero_bytes, uint32_t* __restrict__ sort_status, uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t s_digits[4][kRadix];
  for (int i = threadIdx.x; i < passes * kRadix; i += 256) (&s_digits[0][0])[i] = 0;
  __syncthreads();
  for (int64_t i0 = (int64_t)blockIdx.x * 256 * kKeyItems; i0 < n; i0 += (int64_t)gridDim.x * 256 * kKeyItems) {
#pragma unroll
    for (int k = 0; k < kKeyItems; ++k) {
      const int64_t i = i0 + k * 256 + threadIdx.x;
      if (i >= n) break;
      const uint32_t key = code_key(codes, i, C, status);
      keys[i] = key;
      vals[i] = (uint32_t)i;
      for (int p = 0; p < passes; ++p) atomicAdd(&s_digits[p][(key >> (8 * p)) & (kRadix - 1)], 1u);
    }
  }
  zero_words(zero, zero_bytes);
  if (blockIdx.x == 0 && threadIdx.x < GSB_STATUS_WORDS) sort_status[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < passes * kRadix; i += 256) {
    const uint32_t v = (&s_digits[0][0])[i];
    if (v) atomicAdd(&digits[i], v);
  }
}

// Few slots: every slot's place is the number of smaller ones, counted by a warp for four
// slots at a time over all the keys in shared memory; one launch instead of four or five.
// n^2 comparisons, so the whole gradient (48 columns) takes 10.4 us at 512 slots, 18.5 at
// 4,096 and 29.6 at 8,192 where it takes 16.8, 21.7 and 23.4 with the radix sort.
constexpr int kFewSlots = 4096;
constexpr int kRankWarp = 4;                 // slots a warp
constexpr int kRankBlock = 8 * kRankWarp;    // and a block: 32, one of each lane's keys
__global__ void __launch_bounds__(256)
    k_rank_few(int n, int64_t C, Codes codes, uint32_t* __restrict__ keys, uint32_t* __restrict__ vals,
               uint32_t* __restrict__ zero, int64_t zero_bytes, uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  static_assert(kRankBlock == 32, "the block's own slots are one turn of the loops below");
  __shared__ uint32_t s_key[kFewSlots];
  zero_words(zero, zero_bytes);
  const int own = (int)blockIdx.x * kRankBlock;
  if (own >= n) return;
  const int lane = threadIdx.x % 32, first = own + threadIdx.x / 32 * kRankWarp;
  const int turns = (n + 31) / 32 * 32;
  for (int i = threadIdx.x; i < turns; i += 256)
    s_key[i] = i < n ? code_key(codes, i, C, i / kRankBlock == (int)blockIdx.x ? status : nullptr) : 0xffffffffu;
  __syncthreads();
  uint32_t key[kRankWarp];
  int rank[kRankWarp];
#pragma unroll
  for (int u = 0; u < kRankWarp; ++u) {
    key[u] = s_key[first + u];
    const uint32_t k = s_key[own + lane];
    rank[u] = k < key[u] || (k == key[u] && own + lane < first + u);
  }
  // Of equal keys those in front come first.
#pragma unroll 4
  for (int i = lane; i < own; i += 32) {
    const uint32_t k = s_key[i];
#pragma unroll
    for (int u = 0; u < kRankWarp; ++u) rank[u] += k <= key[u];
  }
#pragma unroll 4
  for (int i = own + 32 + lane; i < turns; i += 32) {
    const uint32_t k = s_key[i];
#pragma unroll
    for (int u = 0; u < kRankWarp; ++u) rank[u] += k < key[u];
  }
#pragma unroll
  for (int u = 0; u < kRankWarp; ++u) {
    const int to = __reduce_add_sync(kFullMask, rank[u]);
    if (lane == 0 && first + u < n) keys[to] = key[u], vals[to] = (uint32_t)(first + u);
  }
}

// Sums of the sorted entries, run by run (a run: the entries of one code).
//
// A group of GL lanes adds up kRunEntries consecutive entries, each lane R
// pieces of V columns; a block of 256 threads takes 256 / GL such stretches. A
// run inside a stretch is written at once. A run that crosses stretches leaves
// its parts in shared memory, where the group it starts in adds them up, and one
// that crosses blocks leaves at most two parts per block (head: of a run begun
// in an earlier block; tail: of one that goes on) for k_run_parts. So every row
// is a sum in one order, however uneven the codes are, and a code that all
// entries share costs no more than an even use.
//
// Bound by the gather of g: rows in code order, one load of the whole row per
// entry. With WGRAD the same loads give g_w (GL lanes share a dot product); that
// takes the row in one tile of columns. 2^20 x 48 fp32 of 8,192 codes: 50 us, 4.8 TB/s
// read. Four of 27 bf16 for 100,003 rows, with g_w: 30 us; rows of 54 bytes come a value
// at a time, out of L2.
//
// sort_status (NULL: nothing waited): the words of the sort that made the order, its own
// because it gives up waiting when they hold an error, which the call's may from earlier
// calls and other streams. An order that was given up is no permutation and not followed.
constexpr int kRunEntries = 16;
constexpr int kRunBlockEntries = 2048;  // at most, per block
template <int GL>
constexpr int run_entries() {
  return kRunBlockEntries / (256 / GL) < kRunEntries ? kRunBlockEntries / (256 / GL) : kRunEntries;
}
template <int GL>
constexpr int run_block_entries() { return run_entries<GL>() * (256 / GL); }

template <typename T, typename O, int V, int GL, int R, bool WGRAD>
__global__ void __launch_bounds__(256, WGRAD ? 1 : 4)
    k_run_sums(int n, int bag, FastDiv div_bag, int C, int dim, const uint32_t* __restrict__ keys,
               const uint32_t* __restrict__ vals, const float* __restrict__ weights, float scale,
               const O* __restrict__ g, const T* __restrict__ table, int64_t stride, T* __restrict__ g_table,
               float* __restrict__ g_weights, float* __restrict__ parts, const uint32_t* __restrict__ sort_status,
               uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  constexpr int NG = 256 / GL, E = run_entries<GL>(), L = run_block_entries<GL>(), W = GL * V * R;
  // Entries whose loads are in flight together. Two of them and four blocks an SM took 56
  // us where four and two took 61 (2^20 x 48 fp32); with WGRAD registers come first.
  constexpr int U = 2;
  __shared__ uint32_t s_key[L + 2];  // the entries' keys, with the neighbours' on either side
  __shared__ uint32_t s_val[L];
  __shared__ __align__(16) float s_part[2][NG][W];
  const int tid = threadIdx.x, lane = tid % GL, grp = tid / GL;
  const int64_t b0 = (int64_t)blockIdx.x * L;
  const int cnt = (int)min((int64_t)L, n - b0);
  const uint32_t kNone = 0xffffffffu;  // no entry: differs from every key
  const bool given_up = sort_status != nullptr && sort_status[GSB_STATUS_ERROR] != 0;
  for (int i = tid; i < L + 2; i += 256) {
    const int64_t k = b0 + i - 1;
    s_key[i] = k >= 0 && k < n ? keys[k] : kNone;
    if (i >= 1 && i <= L) s_val[i - 1] = i <= cnt ? vals[k] : 0u;
  }
  if (given_up) {
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0)
      put_error(status, GSB_DEVERR_LOOKBACK_TIMEOUT, kSiteSortLookback);
    return;
  }
  __syncthreads();
  const int col0 = (int)blockIdx.y * W + lane * V;
  const int s = grp * E, e = min(s + E, cnt);
  float acc[R][V];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < V; ++i) acc[r][i] = 0.0f;
  bool head = s < e && s_key[s] == s_key[s + 1];  // the run in hand began before this stretch
  auto put = [&](float* to) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < V; ++i) to[(r * GL + lane) * V + i] = acc[r][i];
  };
  auto write_row = [&](uint32_t key) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int d = col0 + r * GL * V;
      if (d < dim) {
        float v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = acc[r][i] * scale;
        store_vec<V>(g_table + (int64_t)key * dim + d, v);
      }
    }
  };
  // As many turns for every group of a warp: the dot products exchange lanes.
  for (int k0 = s; k0 < s + E; k0 += U) {
    float w[U];
    Vec<V, O> x[U][R];
    Vec<V, T> t[WGRAD ? U : 1][R];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u;
      const uint32_t key = k < e ? s_key[k + 1] : (uint32_t)C;
      const uint32_t v = k < e ? s_val[k] : 0u;
      const bool on = key < (uint32_t)C;
      w[u] = on ? (weights ? weights[v] : 1.0f) : 0.0f;
      const int64_t row = fast_div((int)v, div_bag);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int d = col0 + r * GL * V;
#pragma unroll
        for (int i = 0; i < V; ++i) x[u][r].v[i] = 0.0f;
        if (on && d < dim) x[u][r].load(g + row * dim + d);
        if constexpr (WGRAD) {
#pragma unroll
          for (int i = 0; i < V; ++i) t[u][r].v[i] = 0.0f;
          if (on && d < dim) t[u][r].load(table + (int64_t)key * stride + d);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u;
      if constexpr (WGRAD) {
        float dot = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < V; ++i) dot = fmaf(x[u][r].v[i], t[u][r].v[i], dot);
#pragma unroll
        for (int o = GL / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(kFullMask, dot, o, GL);
        if (lane == 0 && k < e) g_weights[s_val[k]] = dot * scale;
      }
      if (k < e) {
        const uint32_t key = s_key[k + 1];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < V; ++i) acc[r][i] = fmaf(w[u], x[u][r].v[i], acc[r][i]);
        const bool ends = s_key[k + 2] != key;
        if ((ends || k == e - 1) && key < (uint32_t)C) {
          if (head) put(s_part[0][grp]);
          else if (ends) write_row(key);
          else put(s_part[1][grp]);
        }
        if (ends) {
          head = false;
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < V; ++i) acc[r][i] = 0.0f;
        }
      }
    }
  }
  __syncthreads();
  if (s >= e) return;
  // The runs that cross stretches: the group a run starts in takes its tail and
  // the heads after it; group 0 also takes a run from before the block.
  // Adds the heads of stretches from, from + 1, ...; true if the run goes on behind the block.
  auto chain = [&](int from) {
    for (int j = from; j < NG; ++j) {
      const float* h = s_part[0][j];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[r][i] += h[(r * GL + lane) * V + i];
      const int je = min((j + 1) * E, cnt);
      // One run from the stretch's first entry to its last, and on.
      if (s_key[j * E + 1] != s_key[je] || s_key[je + 1] != s_key[je]) return false;
      if (je == cnt) return true;
    }
    return true;
  };
  auto put_block = [&](int which) {
    float* to = parts + ((int64_t)blockIdx.x * 2 + which) * dim;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int d = col0 + r * GL * V;
      if (d < dim)
#pragma unroll
        for (int i = 0; i < V; ++i) to[d + i] = acc[r][i];
    }
  };
  auto clear = [&]() {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[r][i] = 0.0f;
  };
  if (grp == 0 && s_key[0] == s_key[1] && s_key[1] < (uint32_t)C) {
    clear();
    chain(0);
    put_block(0);
  }
  const uint32_t last = s_key[e];
  const bool goes_on = s_key[e + 1] == last && last < (uint32_t)C;
  const bool began_here = s_key[s] != s_key[s + 1] || s_key[s + 1] != last;  // the last run starts in this stretch
  if (goes_on && began_here) {
    const float* h = s_part[1][grp];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[r][i] = h[(r * GL + lane) * V + i];
    if (e == cnt || chain(grp + 1)) put_block(1);
    else write_row(last);
  }
}

// The runs that cross blocks of k_run_sums: the block a run starts in adds its
// tail and the heads of the blocks after it, 256 / columns of them at a time. Latency
// alone: 8 us for the 1,024 blocks of 2^20 entries.
template <typename T>
__global__ void __launch_bounds__(256)
    k_run_parts(int n, int C, int dim, int block_entries, const uint32_t* __restrict__ keys, float scale,
                const float* __restrict__ parts, T* __restrict__ g_table) {
  pdl_wait();
  pdl_trigger();
  __shared__ float s_sum[256];
  const int64_t b0 = (int64_t)blockIdx.x * block_entries, end = b0 + block_entries;
  if (end >= n) return;
  const uint32_t key = keys[end - 1];
  if (key >= (uint32_t)C || keys[end] != key || (b0 > 0 && keys[b0 - 1] == key)) return;
  // The blocks after this one that begin with the same code, 256 looked at at a time.
  __shared__ int s_heads;
  int64_t heads = 0;
  for (bool more = true; more;) {
    if (threadIdx.x == 0) s_heads = 256;
    __syncthreads();
    const int64_t at = end + (heads + threadIdx.x) * block_entries;
    if (at >= n || keys[at] != key) atomicMin(&s_heads, (int)threadIdx.x);
    __syncthreads();
    heads += s_heads;
    more = s_heads == 256;
    __syncthreads();
  }
  const int cols = min(dim, 256), ways = 256 / cols;
  const int way = threadIdx.x / cols, col = threadIdx.x - way * cols;
  for (int d0 = 0; d0 < dim; d0 += cols) {
    const int d = d0 + col;
    float acc = 0.0f;
    if (way < ways && d < dim) {
      const float* p = parts + (int64_t)blockIdx.x * 2 * dim + d;
      if (way == 0) acc = p[dim];
#pragma unroll 4
      for (int64_t h = 1 + way; h <= heads; h += ways) acc += p[h * 2 * dim];
    }
    s_sum[threadIdx.x] = acc;
    __syncthreads();
    if (way == 0 && d < dim) {
      for (int i = 1; i < ways; ++i) acc += s_sum[i * cols + col];
      g_table[(int64_t)key * dim + d] = from_f32<T>(acc * scale);
    }
    __syncthreads();
  }
}

// One warp per slot: where rows are too long for one tile of k_run_sums, and where the
// codebook has no gradient (a frozen one). Bound by the two rows it reads, from L2 as a rule:
// 2 of 1,200 fp32 for 20,000 rows 38 us, 10 TB/s. Rows shorter than a warp leave lanes idle:
// 4 of bf16 for 100,003 rows take 76 us with 27 values, 86 with 48, 139 with 400.
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

// How the columns of a row are dealt out: V values a piece, GL lanes a row, R pieces a
// lane (2 or 3 of four values, 2 or 4 single ones), whichever leaves fewer lanes idle,
// of equals the larger; more columns take more tiles.
struct RunShape {
  int V, GL, R;
  int block_entries() const {
    const int ng = 256 / GL;
    return ng * std::min(kRunEntries, kRunBlockEntries / ng);
  }
  int tiles(int dim) const { return (dim + V * GL * R - 1) / (V * GL * R); }
};
RunShape run_shape(int dim, int V) {
  const int nvec = (dim + V - 1) / V;
  const int most = V == 4 ? 3 : 4;
  RunShape best{V, 32, most};
  int waste = 1 << 30;
  for (int R : {most, 2}) {
    int GL = 1;
    while (GL < 32 && GL * R < nvec) GL *= 2;
    if (GL * R < nvec) continue;
    if (GL * R - nvec < waste) {
      waste = GL * R - nvec;
      best = RunShape{V, GL, R};
    }
  }
  return best;
}

struct BackwardScratch {
  uint32_t *keys = nullptr, *vals = nullptr, *keys_s = nullptr, *vals_s = nullptr;
  uint32_t* sort_status = nullptr;
  float* parts = nullptr;
};
BackwardScratch carve(Carver& ws, int64_t slots, int dim) {
  BackwardScratch b;
  b.keys = ws.take<uint32_t>((size_t)slots);
  b.vals = ws.take<uint32_t>((size_t)slots);
  b.keys_s = ws.take<uint32_t>((size_t)slots);
  b.vals_s = ws.take<uint32_t>((size_t)slots);
  b.sort_status = ws.take<uint32_t>(GSB_STATUS_WORDS);
  const int64_t least = std::min(run_shape(dim, 1).block_entries(), run_shape(dim, 4).block_entries());
  b.parts = ws.take<float>((size_t)((slots + least - 1) / least) * 2 * (size_t)dim);
  return b;
}

inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Calls fn(T{}, O{}) for the element types of table and result.
template <typename Fn>
void with_dtypes(int32_t table_dtype, int32_t out_dtype, Fn&& fn) {
  with_dtype(table_dtype, [&](auto t) {
    if (out_dtype == GSB_DTYPE_F32) fn(t, float{});
    else fn(t, t);
  });
}

// Calls fn(integral constants V, GL, R).
template <typename Fn>
void with_shape(const RunShape& s, Fn&& fn) {
  auto lanes = [&](auto v, auto r) {
    switch (s.GL) {
      case 1: fn(v, std::integral_constant<int, 1>{}, r); break;
      case 2: fn(v, std::integral_constant<int, 2>{}, r); break;
      case 4: fn(v, std::integral_constant<int, 4>{}, r); break;
      case 8: fn(v, std::integral_constant<int, 8>{}, r); break;
      case 16: fn(v, std::integral_constant<int, 16>{}, r); break;
      default: fn(v, std::integral_constant<int, 32>{}, r); break;
    }
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  using Three = std::integral_constant<int, 3>;
  using Four = std::integral_constant<int, 4>;
  if (s.V == 4 && s.R == 2) lanes(Four{}, Two{});
  else if (s.V == 4) lanes(Four{}, Three{});
  else if (s.R == 2) lanes(One{}, Two{});
  else lanes(One{}, Four{});
}

// Sizes common to both directions; the blocks of a launch have to fit the grid.
int check_sizes(int32_t table_dtype, int32_t out_dtype, int64_t rows, int32_t bag, int64_t codebook_rows, int32_t dim,
                int64_t stride, int32_t code_bytes) {
  if (!dtype_ok(table_dtype) || (out_dtype != table_dtype && out_dtype != GSB_DTYPE_F32)) return GSB_ERR_UNSUPPORTED;
  if (rows < 0 || bag <= 0 || codebook_rows <= 0 || dim <= 0 || stride < 0 || (code_bytes != 4 && code_bytes != 8))
    return GSB_ERR_INVALID_ARGUMENT;
  // Column tiles of the gradient are at least 64 wide and fit the grid's 65,535.
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
  const Codes cd{codes, code_bytes == 8};
  const int so = dtype_bytes(out_dtype), st = dtype_bytes(table_dtype);
  const int V = dim % 4 == 0 && table_stride % 4 == 0 && aligned_to(table, 4 * st) && aligned_to(out, 4 * so) ? 4 : 1;
  const int64_t pieces = rows * (dim / V);
  const int64_t blocks = (pieces + kLookupPieces - 1) / kLookupPieces;
  if (blocks >= (int64_t(1) << 31)) return GSB_ERR_CAPACITY;
  with_dtypes(table_dtype, out_dtype, [&](auto t, auto o) {
      using T = decltype(t);
      using O = decltype(o);
      const bool stage = (int64_t)(kLookupPieces / (dim / V) + 2) * bag <= kLookupSlots &&
                         codebook_rows * std::max<int64_t>(table_stride, dim) < (int64_t(1) << 31);
      auto pick = [&](auto v, auto w) {
        constexpr int W = decltype(v)::value;
        constexpr bool kWeights = decltype(w)::value;
        return stage ? k_lookup<T, O, W, true, kWeights> : k_lookup<T, O, W, false, kWeights>;
      };
      using One = std::integral_constant<int, 1>;
      using Four = std::integral_constant<int, 4>;
      auto kernel = V == 4 ? (weights ? pick(Four{}, std::true_type{}) : pick(Four{}, std::false_type{}))
                           : (weights ? pick(One{}, std::true_type{}) : pick(One{}, std::false_type{}));
      launch_pdl(kernel, (unsigned)blocks, 256, 0, static_cast<cudaStream_t>(stream), pieces, bag,
                 codebook_rows, dim / V, make_fast_div((uint32_t)(dim / V)),
                 (const T*)table, table_stride, cd, weights, scale, (O*)out, status);
  });
  note_launches(1);
  return cuda_status(cudaGetLastError());
}

extern "C" size_t gsb_codebook_backward_workspace_size(int64_t rows, int32_t bag, int64_t codebook_rows, int32_t dim) {
  if (check_sizes(GSB_DTYPE_F32, GSB_DTYPE_F32, rows, bag, codebook_rows, dim, 0, 4) != GSB_OK) return 0;
  const int64_t slots = rows * bag;
  Carver c(nullptr);
  carve(c, slots, dim);
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
    const size_t bytes = (size_t)codebook_rows * dim * dtype_bytes(table_dtype);
    if (g_table && cudaMemsetAsync(g_table, 0, bytes, s) != cudaSuccess) return GSB_ERR_CUDA;
    return GSB_OK;
  }
  if (!codes || !grad_out || !status || (g_weights && !table) || !aligned_to(g_table, 4))
    return GSB_ERR_INVALID_ARGUMENT;
  const Codes cd{codes, code_bytes == 8};
  cudaError_t e = cudaSuccess;
  if (g_table) {
    if (!workspace || workspace_bytes < gsb_codebook_backward_workspace_size(rows, bag, codebook_rows, dim))
      return GSB_ERR_WORKSPACE;
    Carver ws(workspace);
    const BackwardScratch b = carve(ws, slots, dim);
    const int64_t table_bytes = codebook_rows * dim * dtype_bytes(table_dtype);
    const int zero_blocks = (int)std::min<int64_t>(148 * 8, (table_bytes + (1 << 14) - 1) >> 14);
    const bool few = slots <= kFewSlots;
    if (few) {
      const int blocks = std::max(zero_blocks, ((int)slots + kRankBlock - 1) / kRankBlock);
      launch_pdl(k_rank_few, blocks, 256, 0, s, (int)slots, codebook_rows, cd, b.keys_s, b.vals_s,
                 (uint32_t*)g_table, table_bytes, status);
      note_launches(1);
    } else {
      const int bits = bits_for(codebook_rows);
      const ZeroRegion zero = radix_sort_zero_region(ws, slots, 0, bits, true);  // begins with the digits' counts
      if (cudaMemsetAsync(zero.ptr, 0, zero.words * sizeof(uint32_t), s) != cudaSuccess) return GSB_ERR_CUDA;
      const int blocks = std::max(zero_blocks, (int)std::min<int64_t>(148 * 8, grid1d(slots, 256 * kKeyItems)));
      launch_pdl(k_code_keys, blocks, 256, 0, s, slots, codebook_rows, sort_passes(0, bits), cd, b.keys, b.vals,
                 zero.ptr, (uint32_t*)g_table, table_bytes, b.sort_status, status);
      note_launches(1);
      e = radix_sort_pairs(ws, b.keys, b.vals, b.keys_s, b.vals_s, slots, 0, bits, b.sort_status, s, true, zero.ptr);
      if (e != cudaSuccess) return GSB_ERR_CUDA;
    }
    const int so = dtype_bytes(out_dtype), st = dtype_bytes(table_dtype);
    const bool vec = dim % 4 == 0 && aligned_to(grad_out, 4 * so) && aligned_to(g_table, 4 * st) &&
                     (!g_weights || (table_stride % 4 == 0 && aligned_to(table, 4 * st)));
    const RunShape shape = run_shape(dim, vec ? 4 : 1);
    const int block_entries = shape.block_entries();
    const dim3 grid((unsigned)((slots + block_entries - 1) / block_entries), (unsigned)shape.tiles(dim));
    const bool fused = g_weights && shape.tiles(dim) == 1;
    with_dtypes(table_dtype, out_dtype, [&](auto t, auto o) {
        using T = decltype(t);
        using O = decltype(o);
        with_shape(shape, [&](auto v, auto gl, auto r) {
          constexpr int W = decltype(v)::value, GL = decltype(gl)::value, R = decltype(r)::value;
          auto kernel = fused ? k_run_sums<T, O, W, GL, R, true> : k_run_sums<T, O, W, GL, R, false>;
          launch_pdl(kernel, grid, 256, 0, s, (int)slots, bag, make_fast_div((uint32_t)bag), (int)codebook_rows, dim,
                     (const uint32_t*)b.keys_s, (const uint32_t*)b.vals_s, weights, scale, (const O*)grad_out,
                     (const T*)table, table_stride, (T*)g_table, g_weights, b.parts,
                     few ? (const uint32_t*)nullptr : (const uint32_t*)b.sort_status, status);
        });
        if (grid.x > 1)
          launch_pdl(k_run_parts<T>, grid.x - 1, 256, 0, s, (int)slots, (int)codebook_rows, dim, block_entries,
                     (const uint32_t*)b.keys_s, scale, (const float*)b.parts, (T*)g_table);
    });
    note_launches(grid.x > 1 ? 2 : 1);
    if (fused) g_weights = nullptr;  // done
  }
  if (g_weights) {
    with_dtypes(table_dtype, out_dtype, [&](auto t, auto o) {
        using T = decltype(t);
        using O = decltype(o);
        launch_pdl(k_weight_grad<T, O>, grid1d(slots * 32, 256), 256, 0, s, slots, bag, codebook_rows, dim,
                   (const T*)table, table_stride, cd, scale, (const O*)grad_out, g_weights, status);
    });
    note_launches(1);
  }
  return cuda_status(cudaGetLastError());
}
