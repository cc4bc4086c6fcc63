// Token embedding of the features in front of the sparse layer.
//
//   y[t] = s table[ids[t]],        dtable[v] = s sum over the tokens t with ids[t] = v of dy[t], zeros where there is none
//
// Forward: memory alone; a thread moves 16 bytes at a time.
// Backward: tokens are sorted by id (stable, so that a row's sum always runs in the order of its tokens), and then rows and tokens are one list of things
// to do, "read the gradient of a token" and "write a row": every block takes the same number of them, whether these are a thousand tokens of one
// frequent word or a thousand rows that no token asked for.  What a block has summed of a row that another one writes goes through scratch memory, and a last launch
// adds such parts, again in a fixed order.  Sums are fp32.
#include "common.cuh"
#include "launchers.h"
#include "runtime.h"
#include "sm100.cuh"

#include <cooperative_groups.h>

#include <atomic>

namespace haste {
namespace {

// ---------------------------------------------------------------- ids
struct Ids {
  const void* p;
  int wide;                        // int64, else int32
  __device__ __forceinline__ int64_t operator[](int64_t i) const {
    return wide ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
  }
};

template <class T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
    const uint32_t r[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(r[i] << 16); v[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u); }
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = rn_bf16_bits(v[2 * i]) | static_cast<uint32_t>(rn_bf16_bits(v[2 * i + 1])) << 16;
    return make_uint4(r[0], r[1], r[2], r[3]);
  }
  static __device__ __forceinline__ float get(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[4]) {
    v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[4]) { return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])); }
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};

// ---------------------------------------------------------------- forward
// An id that is no row of the table makes a row of NaN.  A thread has AHEAD pieces of 16 bytes of the output, all of whose ids and then rows are on their way at once.
// Bound: memory, most of it the output's stores (frequent rows come from L2).  65536 tokens of 1024 bf16 out of 32000 rows: 34.5 us, 72 % of what the bytes take at a plain copy's rate, 36.9 with 2 pieces
// a thread, 38.9 with 8; one piece each took 43.  9 tokens of 768: 3 us, a launch and two dependent reads.
constexpr int FORWARD_THREADS = 256;
template <class T, bool WHOLE, int AHEAD>
__global__ void __launch_bounds__(FORWARD_THREADS) embedding_kernel(const Ids ids, const T* __restrict__ table, T* __restrict__ y, int64_t tokens, int64_t D, int64_t V, int64_t ld,
                                                                    float scale) {
  constexpr int N = Vec<T>::N;
  const int64_t n = tokens * D, pieces = (n + N - 1) / N, first = static_cast<int64_t>(blockIdx.x) * (FORWARD_THREADS * AHEAD) + threadIdx.x;
  const bool narrow = n <= 0x7FFFFFFF;
  if (WHOLE) {                                     // a piece lies in one row, on 16 bytes on both sides
    int64_t id[AHEAD], c[AHEAD];
    uint4 q[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int64_t i = first + k * FORWARD_THREADS;
      id[k] = -1;
      if (i < pieces) {
        const int64_t t = narrow ? static_cast<uint32_t>(i * N) / static_cast<uint32_t>(D) : i * N / D;
        c[k] = i * N - t * D;
        id[k] = ids[t];
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (static_cast<uint64_t>(id[k]) < static_cast<uint64_t>(V)) q[k] = __ldg(reinterpret_cast<const uint4*>(table + id[k] * ld + c[k]));
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int64_t i = first + k * FORWARD_THREADS;
      if (i >= pieces) break;
      float v[N];
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = __int_as_float(0x7FFFFFFF);
      if (static_cast<uint64_t>(id[k]) < static_cast<uint64_t>(V)) {
        Vec<T>::unpack(q[k], v);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] *= scale;
      }
      *reinterpret_cast<uint4*>(y + i * N) = Vec<T>::pack(v);
    }
  } else {
    // neighbouring elements by neighbouring threads
    const int64_t from = static_cast<int64_t>(blockIdx.x) * (FORWARD_THREADS * AHEAD * N) + threadIdx.x;
    int64_t id[AHEAD * N], c[AHEAD * N];
    T x[AHEAD * N];
#pragma unroll
    for (int k = 0; k < AHEAD * N; ++k) {
      const int64_t i = from + k * FORWARD_THREADS;
      id[k] = -1;
      if (i < n) {
        const int64_t t = narrow ? static_cast<uint32_t>(i) / static_cast<uint32_t>(D) : i / D;
        c[k] = i - t * D;
        id[k] = ids[t];
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD * N; ++k)
      if (static_cast<uint64_t>(id[k]) < static_cast<uint64_t>(V)) x[k] = table[id[k] * ld + c[k]];
#pragma unroll
    for (int k = 0; k < AHEAD * N; ++k) {
      const int64_t i = from + k * FORWARD_THREADS;
      if (i < n) y[i] = Vec<T>::put(static_cast<uint64_t>(id[k]) < static_cast<uint64_t>(V) ? Vec<T>::get(x[k]) * scale : __int_as_float(0x7FFFFFFF));
    }
  }
}

// ---------------------------------------------------------------- sorting tokens by id
constexpr int SORT_THREADS = 256, SORT_ITEMS = 16, SORT_TILE = SORT_THREADS * SORT_ITEMS, DIGITS = 256;

// The lanes whose digit (up to DIGITS) is this lane's: nine votes, which take less time than one match
__device__ __forceinline__ unsigned lanes_alike(int digit) {
  unsigned same = 0xffffffffu;
#pragma unroll
  for (int bit = 0; bit < 9; ++bit) {
    const bool set = (digit >> bit) & 1;
    const unsigned votes = __ballot_sync(0xffffffffu, set);
    same &= set ? votes : ~votes;
  }
  return same;
}

struct SortPass {
  const int2* in;                  // key and token; NULL in the first pass: from the ids
  int2* out;
  int32_t* counts;                 // [DIGITS][blocks]
  int64_t n;
  int shift, blocks;
};
// The id, or V where the token has no row or the row is the padding's
__device__ __forceinline__ int2 first_item(const Ids& ids, int64_t i, int64_t V, int64_t padding) {
  const int64_t id = ids[i];
  return make_int2(static_cast<uint64_t>(id) < static_cast<uint64_t>(V) && id != padding ? static_cast<int32_t>(id) : static_cast<int32_t>(V), static_cast<int32_t>(i));
}
__device__ __forceinline__ int2 item_of(const SortPass& s, const Ids& ids, int64_t i, int64_t V, int64_t padding) {
  return s.in != nullptr ? s.in[i] : first_item(ids, i, V, padding);
}
__global__ void __launch_bounds__(SORT_THREADS) sort_count_kernel(const SortPass s, const Ids ids, int64_t V, int64_t padding) {
  __shared__ int32_t count[DIGITS];
  count[threadIdx.x] = 0;
  sm100::grid_dependency_wait();
  __syncthreads();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * SORT_TILE;
  for (int k = 0; k < SORT_ITEMS; ++k) {
    const int64_t i = first + k * SORT_THREADS + threadIdx.x;
    if (i < s.n) atomicAdd(&count[(item_of(s, ids, i, V, padding).x >> s.shift) & (DIGITS - 1)], 1);
  }
  __syncthreads();
  s.counts[static_cast<int64_t>(threadIdx.x) * s.blocks + blockIdx.x] = count[threadIdx.x];
}
// Exclusive sums over all counts, by one block
__global__ void __launch_bounds__(1024) sort_scan_kernel(int32_t* counts, int64_t n) {
  __shared__ int32_t warps[32];
  __shared__ int32_t carry;
  if (threadIdx.x == 0) carry = 0;
  sm100::grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t at = 0; at < n; at += 4096) {
    int32_t v[4], sum = 0;
    const int64_t i = at + 4 * threadIdx.x;
#pragma unroll
    for (int k = 0; k < 4; ++k) { v[k] = i + k < n ? counts[i + k] : 0; sum += v[k]; }
    int32_t up = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int32_t x = __shfl_up_sync(0xffffffffu, up, o); if (lane >= o) up += x; }
    if (lane == 31) warps[warp] = up;
    __syncthreads();
    if (warp == 0) {
      int32_t w = warps[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int32_t x = __shfl_up_sync(0xffffffffu, w, o); if (lane >= o) w += x; }
      warps[lane] = w;
    }
    __syncthreads();
    int32_t before = carry + (warp ? warps[warp - 1] : 0) + up - sum;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i + k < n) counts[i + k] = before;
      before += v[k];
    }
    __syncthreads();
    if (threadIdx.x == 0) carry += warps[31];
    __syncthreads();
  }
}
// A warp has 512 neighbours, 32 at a time: a token's place is that of its digit, plus the same digits in the block's warps before this one, plus those in this warp
// before it.
__global__ void __launch_bounds__(SORT_THREADS) sort_place_kernel(const SortPass s, const Ids ids, int64_t V, int64_t padding) {
  constexpr int WARPS = SORT_THREADS / 32;
  __shared__ int32_t count[WARPS][DIGITS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) count[w][threadIdx.x] = 0;
  sm100::grid_dependency_wait();
  __syncthreads();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * SORT_TILE + warp * (32 * SORT_ITEMS) + lane;
  int2 item[SORT_ITEMS];
  int32_t rank[SORT_ITEMS];
#pragma unroll
  for (int k = 0; k < SORT_ITEMS; ++k) {
    const int64_t i = first + 32 * k;
    item[k] = i < s.n ? item_of(s, ids, i, V, padding) : make_int2(0, 0);
  }
#pragma unroll
  for (int k = 0; k < SORT_ITEMS; ++k) {
    const bool live = first + 32 * k < s.n;
    const int digit = live ? (item[k].x >> s.shift) & (DIGITS - 1) : DIGITS;
    const unsigned same = lanes_alike(digit);
    const int before = __popc(same & ((1u << lane) - 1));
    int32_t base = 0;
    if (live) base = count[warp][digit];
    __syncwarp();
    if (live && before == 0) count[warp][digit] = base + __popc(same);
    __syncwarp();
    rank[k] = base + before;
  }
  __syncthreads();
  int32_t sum = s.counts[static_cast<int64_t>(threadIdx.x) * s.blocks + blockIdx.x];
#pragma unroll
  for (int w = 0; w < WARPS; ++w) { const int32_t x = count[w][threadIdx.x]; count[w][threadIdx.x] = sum; sum += x; }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < SORT_ITEMS; ++k) {
    const int64_t i = first + 32 * k;
    if (i < s.n) {
      s.out[count[warp][(item[k].x >> s.shift) & (DIGITS - 1)] + rank[k]] = item[k];
    }
  }
}

// Up to CLUSTER_MOST tokens (what the registers and shared memory of 16 blocks hold), where the device can place it: one launch of one cluster, whose blocks keep the tokens in registers and shared memory.  In each pass every block places its tokens as above;
// how many tokens of each digit the other blocks have comes through their shared memory, and so do the tokens themselves on their way to the block of their new place.
// Bound: a pass's chain of latencies, some 8 us: 65536 tokens in two passes 18 us, 4099 in 8.  Whole backward calls of 128 columns, this way and through the launches above: 1000 tokens 16.0 and 28.1
// us, 16384: 21.0 and 39.1, 65536: 32.9 and 45.8, 131072: 58.8 and 64.6.  Clusters of 8 blocks (which any device must have) took 32 us for the sort of 65536.
constexpr int CLUSTER_THREADS = 1024, CLUSTER_BLOCKS = 16, CLUSTER_MOST = CLUSTER_BLOCKS * CLUSTER_THREADS * 8;
template <int ITEMS>
constexpr int cluster_smem() { return CLUSTER_THREADS * ITEMS * 8 + 32 * DIGITS * 2 + CLUSTER_BLOCKS * DIGITS * 4 + DIGITS * 4 + 64; }

template <int ITEMS>
__global__ void __launch_bounds__(CLUSTER_THREADS) sort_cluster_kernel(const Ids ids, int64_t n, int64_t V, int64_t padding, int passes, int2* __restrict__ out) {
  constexpr int CHUNK = CLUSTER_THREADS * ITEMS;
  extern __shared__ __align__(16) uint8_t raw[];
  int2* items = reinterpret_cast<int2*>(raw);                                     // key, token
  uint16_t* count = reinterpret_cast<uint16_t*>(raw + CHUNK * 8);                 // [32 warps][DIGITS]
  int32_t* totals = reinterpret_cast<int32_t*>(raw + CHUNK * 8 + 32 * DIGITS * 2);        // [blocks][DIGITS]
  int32_t* base = totals + CLUSTER_BLOCKS * DIGITS;
  int32_t* sums = base + DIGITS;                                                  // [8]
  cluster_started_arrive();
  auto cluster = cooperative_groups::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), blocks = static_cast<int>(cluster.num_blocks()), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = warp * (32 * ITEMS) + lane;
  const int live = static_cast<int>(min(static_cast<int64_t>(CHUNK), max(n - static_cast<int64_t>(rank) * CHUNK, static_cast<int64_t>(0))));
  int2 item[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int at = first + 32 * k;
    item[k] = make_int2(0, 0);
    if (at < live) {
      item[k] = first_item(ids, static_cast<int64_t>(rank) * CHUNK + at, V, padding);
    }
  }
  cluster_started_wait();
  for (int p = 0; p < passes; ++p) {
    const int shift = 8 * p;
    for (int i = threadIdx.x; i < 32 * DIGITS / 2; i += CLUSTER_THREADS) reinterpret_cast<uint32_t*>(count)[i] = 0;
    __syncthreads();
    uint16_t place[ITEMS];
    uint16_t* mine = count + warp * DIGITS;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const bool there = first + 32 * k < live;
      const int digit = there ? (item[k].x >> shift) & (DIGITS - 1) : DIGITS;
      const unsigned same = lanes_alike(digit);
      const int before = __popc(same & ((1u << lane) - 1));
      int at = 0;
      if (there) at = mine[digit];
      __syncwarp();
      if (there && before == 0) mine[digit] = static_cast<uint16_t>(at + __popc(same));
      __syncwarp();
      place[k] = static_cast<uint16_t>(at + before);
    }
    __syncthreads();
    if (threadIdx.x < DIGITS) {
      int sum = 0;
#pragma unroll 8
      for (int w = 0; w < 32; ++w) {
        const int x = count[w * DIGITS + threadIdx.x];
        count[w * DIGITS + threadIdx.x] = static_cast<uint16_t>(sum);
        sum += x;
      }
      for (int b = 0; b < blocks; ++b) *cluster.map_shared_rank(&totals[rank * DIGITS + threadIdx.x], b) = sum;
    }
    cluster.sync();
    if (threadIdx.x < DIGITS) {
      int all = 0, before = 0;
      for (int b = 0; b < blocks; ++b) {
        const int x = totals[b * DIGITS + threadIdx.x];
        if (b < rank) before += x;
        all += x;
      }
      int up = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, up, o); if (lane >= o) up += x; }
      if (lane == 31) sums[warp] = up;
      base[threadIdx.x] = up - all + before;
    }
    __syncthreads();
    if (threadIdx.x < DIGITS) {
      int lower = 0;
      for (int w = 0; w < warp; ++w) lower += sums[w];
      base[threadIdx.x] += lower;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
      if (first + 32 * k < live) {
        const int digit = (item[k].x >> shift) & (DIGITS - 1), to = base[digit] + mine[digit] + place[k];
        if (p + 1 == passes) {
          out[to] = item[k];
        } else {
          *cluster.map_shared_rank(&items[to % CHUNK], to / CHUNK) = item[k];
        }
      }
    if (p + 1 == passes) break;
    cluster.sync();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
      if (first + 32 * k < live) item[k] = items[first + 32 * k];
  }
}

// ---------------------------------------------------------------- sums
constexpr int UNITS = 128;         // rows and tokens of a block, at most
constexpr int SUM_THREADS = 128;

// The list of things to do, at place d: v rows are written and i tokens read before it.  A row is written when its last token has been read.
// By a warp: 32 places are looked at together, so that the search takes 4 reads after each other among 65536 tokens and not 16.
__device__ __forceinline__ int32_t rows_before(const int2* __restrict__ sorted, int64_t n, int64_t V, int64_t d) {
  int64_t lo = d > V ? d - V : 0, hi = d < n ? d : n;              // the number of tokens among the first d
  while (lo < hi) {
    const int64_t step = (hi - lo + 31) / 32, i = lo + (threadIdx.x & 31) * step;
    // is token i among them?  It is before the end of its row, at place i + key.
    const int c = __popc(__ballot_sync(0xffffffffu, i < hi && sorted[i].x <= d - 1 - i));
    if (c == 0) break;
    hi = min(hi, lo + c * step);
    lo += (c - 1) * step + 1;
  }
  return static_cast<int32_t>(d - lo);
}

struct SumArgs {
  const int2* sorted;              // key and token
  int32_t* starts;                 // of each block: the row that is worked on there
  int32_t* joins;                  // of each block: that row, if others began it and this one ends it, else -1
  float *head, *tail;              // [blocks][D]: parts of a block's first row, begun before it, and of the row after its last one
  int64_t n, V, D, lddy;
  float scale;
  int blocks, units;               // units: of a block
};

// Bound: memory, and the wait for each block's first gradients: 65536 tokens of 1024 bf16 into 32000 rows 33 us (200 MB: 31 at a plain copy's rate).  With equal shares no word, however frequent, holds a
// block up (a block for each row took 151 us a call, of now 60).  64 units a block instead of 128: 71 us a call.
// WHOLE: pieces of 16 bytes on both sides; else a thread has every SUM_THREADS-th element
template <class G, class T, bool WHOLE>
__global__ void __launch_bounds__(SUM_THREADS) embedding_sum_kernel(const SumArgs a, const G* __restrict__ dy, T* __restrict__ out) {
  constexpr int N = WHOLE ? Vec<G>::N : 4;
  constexpr int AHEAD = 8;
  __shared__ int32_t todo[UNITS + AHEAD];          // a token, or ~row at its end
  __shared__ int32_t bounds[2];
  sm100::grid_dependency_wait();
  const int64_t d0 = static_cast<int64_t>(blockIdx.x) * a.units, all = a.V + a.n, d1 = d0 + a.units < all ? d0 + a.units : all;
  if (threadIdx.x < 64) {
    const int which = threadIdx.x >> 5;
    const int32_t v = rows_before(a.sorted, a.n, a.V, which ? d1 : d0);
    if ((threadIdx.x & 31) == 0) {
      bounds[which] = v;
      if (blockIdx.y == 0 && which == 0) a.starts[blockIdx.x] = v;
    }
  }
  for (int i = threadIdx.x; i < UNITS + AHEAD; i += SUM_THREADS) todo[i] = INT32_MIN;
  __syncthreads();
  const int32_t v0 = bounds[0], v1 = bounds[1];
  const int64_t i0 = d0 - v0, i1 = d1 - v1;
  // tokens at their places, which those of their rows precede; the places left are rows' ends
  for (int64_t i = i0 + threadIdx.x; i < i1; i += SUM_THREADS) {
    const int2 it = a.sorted[i];
    if (it.x < a.V) todo[i + it.x - d0] = it.y;
  }
  __syncthreads();
  const int units = static_cast<int>(d1 - d0);
  if (threadIdx.x < 32) {                          // the k-th place without a token is the end of row v0 + k
    int32_t v = v0;
    for (int k = threadIdx.x; k - static_cast<int>(threadIdx.x) < units; k += 32) {
      const bool end = k < units && todo[k] == INT32_MIN;
      const unsigned mask = __ballot_sync(0xffffffffu, end);
      const int32_t row = v + __popc(mask & ((1u << threadIdx.x) - 1));
      if (end && row < a.V) todo[k] = ~row;
      v += __popc(mask);
    }
  }
  __syncthreads();
  const bool begun = i0 > 0 && v0 < a.V && a.sorted[i0 - 1].x == v0;                   // the first row has tokens before this block
  if (blockIdx.y == 0 && threadIdx.x == 0 && a.n > 0) a.joins[blockIdx.x] = begun && v1 > v0 ? v0 : -1;
  const int64_t column = (static_cast<int64_t>(blockIdx.y) * SUM_THREADS + threadIdx.x) * N;
  const int64_t first = WHOLE ? column : static_cast<int64_t>(blockIdx.y) * SUM_THREADS * N + threadIdx.x;
  if (first >= a.D) return;
  float sum[N];
#pragma unroll
  for (int k = 0; k < N; ++k) sum[k] = 0.f;
  int32_t open = v0;                               // the row that is summed
  for (int u = 0; u < units; u += AHEAD) {
    float v[AHEAD][N];
    uint4 q[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int32_t what = todo[u + k];
      if (what >= 0) {
        const G* row = dy + static_cast<int64_t>(what) * a.lddy;
        if (WHOLE) {
          q[k] = __ldg(reinterpret_cast<const uint4*>(row + first));
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) v[k][e] = first + e * SUM_THREADS < a.D ? Vec<G>::get(row[first + e * SUM_THREADS]) : 0.f;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int32_t what = todo[u + k];
      if (what >= 0) {
        if constexpr (WHOLE) Vec<G>::unpack(q[k], v[k]);
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += v[k][e];
      } else if (what != INT32_MIN) {
        const int32_t row = ~what;
        if (row == v0 && begun) {                  // the others' parts are added by the last launch
          float* h = a.head + static_cast<int64_t>(blockIdx.x) * a.D;
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (WHOLE || first + e * SUM_THREADS < a.D) h[WHOLE ? first + e : first + e * SUM_THREADS] = sum[e];
        } else {
          T* o = out + static_cast<int64_t>(row) * a.D;
          if constexpr (WHOLE && Vec<T>::N == N) {
            float s[N];
#pragma unroll
            for (int e = 0; e < N; ++e) s[e] = sum[e] * a.scale;
            *reinterpret_cast<uint4*>(o + first) = Vec<T>::pack(s);
          } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
              if (WHOLE || first + e * SUM_THREADS < a.D) o[WHOLE ? first + e : first + e * SUM_THREADS] = Vec<T>::put(sum[e] * a.scale);
          }
        }
        open = row + 1;
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = 0.f;
      }
    }
  }
  if (open < a.V && i1 > 0 && a.sorted[i1 - 1].x == open) {          // some of its tokens are read: here, or before
    float* h = a.tail + static_cast<int64_t>(blockIdx.x) * a.D;
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (WHOLE || first + e * SUM_THREADS < a.D) h[WHOLE ? first + e : first + e * SUM_THREADS] = sum[e];
  }
}

// A block whose first row was begun before it, and ends in it: the parts of the blocks before, in order, and its own.  11 us after 65536 tokens, 8 after 4099: the chain of the most frequent word's parts,
// eight of which are on their way at once (sixteen: a call 1.5 us longer).
constexpr int JOIN_THREADS = 256;
template <class T>
__global__ void __launch_bounds__(JOIN_THREADS) embedding_join_kernel(const SumArgs a, T* __restrict__ out) {
  sm100::grid_dependency_wait();
  const int b = blockIdx.x;
  const int32_t row = a.joins[b], last = a.starts[b > 0 ? b - 1 : 0];
  if (row < 0) return;
  // the first block whose tail is of this row: the last that started in an earlier row (or with this row's first token)
  int lo = 0, hi = b - 1;
  if (last < row) lo = hi;                         // nearly always the one before
  while (lo < hi) {                                // by a warp, 32 at a time
    const int step = (hi - lo + 31) / 32, c = lo + ((threadIdx.x & 31) + 1) * step;
    bool before = false;
    if (c <= hi) {
      const int32_t at = a.starts[c];
      const int64_t i = static_cast<int64_t>(c) * a.units - at;
      before = at < row || i == 0 || a.sorted[i - 1].x != row;
    }
    const int n = __popc(__ballot_sync(0xffffffffu, before));
    hi = min(hi, lo + (n + 1) * step - 1);
    lo += n * step;
  }
  const float *t = a.tail + static_cast<int64_t>(lo) * a.D, *h = a.head + static_cast<int64_t>(b) * a.D;
  T* o = out + static_cast<int64_t>(row) * a.D;
  if (a.D % 4 == 0) {
    for (int64_t col = (static_cast<int64_t>(blockIdx.y) * JOIN_THREADS + threadIdx.x) * 4; col < a.D; col += static_cast<int64_t>(gridDim.y) * JOIN_THREADS * 4) {
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int c = 0; c < b - lo; ++c) {
        const float4 x = *reinterpret_cast<const float4*>(t + static_cast<int64_t>(c) * a.D + col);
        s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
      }
      const float4 x = *reinterpret_cast<const float4*>(h + col);
      o[col] = Vec<T>::put((s.x + x.x) * a.scale); o[col + 1] = Vec<T>::put((s.y + x.y) * a.scale);
      o[col + 2] = Vec<T>::put((s.z + x.z) * a.scale); o[col + 3] = Vec<T>::put((s.w + x.w) * a.scale);
    }
  } else {
    for (int64_t col = static_cast<int64_t>(blockIdx.y) * JOIN_THREADS + threadIdx.x; col < a.D; col += static_cast<int64_t>(gridDim.y) * JOIN_THREADS) {
      float s = 0.f;
#pragma unroll 8
      for (int c = 0; c < b - lo; ++c) s += t[static_cast<int64_t>(c) * a.D + col];
      o[col] = Vec<T>::put((s + h[col]) * a.scale);
    }
  }
}

int64_t up256(int64_t n) { return (n + 255) & ~int64_t(255); }
int passes_of(int64_t V) {         // over the digits of keys 0 .. V
  int n = 1;
  while (n < 4 && (V >> (8 * n)) > 0) ++n;
  return n;
}
int sort_blocks(int64_t tokens) { return static_cast<int>((tokens + SORT_TILE - 1) / SORT_TILE); }
// Rows and tokens of a block: as many as make one round of all SMs, 7 blocks each
int units_of(int64_t tokens, int64_t V, int64_t D) {
  const int64_t pieces = (D + 511) / 512, rounds = static_cast<int64_t>(sm_count()) * 7;
  const int64_t units = ((tokens + V) * pieces + rounds - 1) / rounds;
  return static_cast<int>(units < 8 ? 8 : units > UNITS ? UNITS : units);
}

template <class G, class T>
int sums(const SumArgs& a, const void* dy, void* out, cudaStream_t st) {
  constexpr int E = sizeof(G) > sizeof(T) ? sizeof(T) : sizeof(G);
  const bool whole = a.D % Vec<G>::N == 0 && (a.lddy * sizeof(G)) % 16 == 0 && aligned16(dy) && aligned16(out) && (a.D * E) % 16 == 0;
  const int64_t per = SUM_THREADS * (whole ? Vec<G>::N : 4);
  const dim3 grid(static_cast<unsigned>(a.blocks), static_cast<unsigned>((a.D + per - 1) / per));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(SUM_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = a.n > 0 ? 1 : 0;                  // without tokens no kernel of this call comes before
  const G* g = static_cast<const G*>(dy);
  T* o = static_cast<T*>(out);
  cudaError_t e = whole ? cudaLaunchKernelEx(&cfg, embedding_sum_kernel<G, T, true>, a, g, o) : cudaLaunchKernelEx(&cfg, embedding_sum_kernel<G, T, false>, a, g, o);
  if (e == cudaSuccess && a.n > 0) {
    const int64_t columns = JOIN_THREADS * (a.D % 4 == 0 ? 4 : 1);
    cfg.gridDim = dim3(grid.x, static_cast<unsigned>(imin64((a.D + columns - 1) / columns, 16)));
    cfg.blockDim = dim3(JOIN_THREADS);
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, embedding_join_kernel<T>, a, o);
  }
  if (e != cudaSuccess) return fail(HASTE_ERR_LAUNCH, "cudaLaunchKernelEx: %s", cudaGetErrorString(e));
  return HASTE_OK;
}

}  // namespace

template <class T>
static int forward_typed(const Ids& ids, const void* table, void* y, int64_t tokens, int64_t D, int64_t V, int64_t ld, float scale, cudaStream_t st) {
  constexpr int N = Vec<T>::N;
  const bool whole = D % N == 0 && ld % N == 0 && aligned16(table) && aligned16(y);
  const int64_t pieces = (tokens * D + N - 1) / N, most = static_cast<int64_t>(sm_count()) * 8 * FORWARD_THREADS;
  const T* from = static_cast<const T*>(table);
  T* to = static_cast<T*>(y);
  const bool few = pieces <= most;                 // as many threads as run at once have one piece each
  const int64_t per = FORWARD_THREADS * (few || !whole ? 1 : 4);
  const unsigned grid = static_cast<unsigned>((pieces + per - 1) / per);
  if (!whole) embedding_kernel<T, false, 1><<<grid, FORWARD_THREADS, 0, st>>>(ids, from, to, tokens, D, V, ld, scale);
  else if (few) embedding_kernel<T, true, 1><<<grid, FORWARD_THREADS, 0, st>>>(ids, from, to, tokens, D, V, ld, scale);
  else embedding_kernel<T, true, 4><<<grid, FORWARD_THREADS, 0, st>>>(ids, from, to, tokens, D, V, ld, scale);
  return check_launch("embedding_kernel");
}

int launch_embedding_forward(const void* ids, int wide, const void* table, void* y, int64_t tokens, int64_t D, int64_t V, int64_t ld, float scale, int type, cudaStream_t st) {
  if (tokens == 0) return HASTE_OK;
  const Ids i = {ids, wide};
  return type == HASTE_BF16 ? forward_typed<__nv_bfloat16>(i, table, y, tokens, D, V, ld, scale, st) : forward_typed<float>(i, table, y, tokens, D, V, ld, scale, st);
}

int64_t embedding_backward_scratch(int64_t tokens, int64_t D, int64_t V) {
  const int64_t blocks = (tokens + V + units_of(tokens, V, D) - 1) / units_of(tokens, V, D);
  const int64_t starts = 2 * up256(blocks * 4);
  if (tokens == 0) return starts;
  const int64_t sorting = 2 * up256(tokens * 8) + up256(static_cast<int64_t>(sort_blocks(tokens)) * DIGITS * 4);      // what sorting in several launches takes
  return sorting + starts + 2 * up256(blocks * D * 4);
}

// Whether the current device can place a cluster of so many blocks, which it is asked once.  It need not: more than 8 are beyond what every device has, and a part of one has fewer SMs side by side.
template <int ITEMS>
static bool cluster_fits(cudaLaunchConfig_t& cfg, unsigned blocks) {
  static std::atomic<int> known[64][CLUSTER_BLOCKS + 1];             // by device: 1 it can, -1 it cannot, 0 not asked yet
  if (blocks > static_cast<unsigned>(cluster_limit())) return false;
  auto kernel = sort_cluster_kernel<ITEMS>;
  int dev = 0;
  cudaGetDevice(&dev);
  const bool keep = dev >= 0 && dev < 64;
  if (keep)
    if (const int can = known[dev][blocks].load(std::memory_order_acquire)) return can > 0;
  int clusters = 0;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, cluster_smem<ITEMS>());
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg);
  const bool can = e == cudaSuccess && clusters > 0;
  if (e != cudaSuccess) cudaGetLastError();                          // no answer: it is asked again
  else if (keep) known[dev][blocks].store(can ? 1 : -1, std::memory_order_release);
  return can;
}

// *sorted stays false where the cluster cannot be placed
template <int ITEMS>
static int sort_in_cluster(const Ids& ids, int64_t tokens, int64_t V, int64_t padding, int2* out, bool* sorted, cudaStream_t st) {
  unsigned blocks = 1;
  while (static_cast<int64_t>(blocks) * CLUSTER_THREADS * ITEMS < tokens) blocks *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(CLUSTER_THREADS);
  cfg.dynamicSmemBytes = cluster_smem<ITEMS>();
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (!cluster_fits<ITEMS>(cfg, blocks)) return HASTE_OK;
  cfg.stream = st;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sort_cluster_kernel<ITEMS>, ids, tokens, V, padding, passes_of(V), out);
  if (e != cudaSuccess) return fail(HASTE_ERR_LAUNCH, "cudaLaunchKernelEx: %s", cudaGetErrorString(e));
  *sorted = true;
  return HASTE_OK;
}

int launch_embedding_backward(const void* ids, int wide, const void* dy, void* dtable, void* scratch, int64_t tokens, int64_t D, int64_t V, int64_t lddy, float scale, int64_t padding,
                              int dy_type, int out_type, cudaStream_t st) {
  char* mem = static_cast<char*>(scratch);
  auto take = [&](int64_t bytes) { char* p = mem; mem += up256(bytes); return p; };
  const Ids i = {ids, wide};
  int2* pairs[2] = {};
  int cur = 0;
  bool sorted = false;
  if (tokens > 0) pairs[0] = reinterpret_cast<int2*>(take(tokens * 8));
  if (tokens > 0 && tokens <= CLUSTER_MOST) {
    int rc = 0;
    if (tokens <= CLUSTER_MOST / 8) rc = sort_in_cluster<1>(i, tokens, V, padding, pairs[0], &sorted, st);
    else if (tokens <= CLUSTER_MOST / 2) rc = sort_in_cluster<4>(i, tokens, V, padding, pairs[0], &sorted, st);
    else rc = sort_in_cluster<8>(i, tokens, V, padding, pairs[0], &sorted, st);
    if (rc) return rc;
  }
  if (tokens > 0 && !sorted) {
    pairs[1] = reinterpret_cast<int2*>(take(tokens * 8));
    SortPass s = {};
    s.n = tokens; s.blocks = sort_blocks(tokens);
    s.counts = reinterpret_cast<int32_t*>(take(static_cast<int64_t>(s.blocks) * DIGITS * 4));
    const int passes = passes_of(V);
    for (int p = 0; p < passes; ++p, cur ^= 1) {
      s.shift = 8 * p;
      s.in = p ? pairs[cur ^ 1] : nullptr;
      s.out = pairs[cur];
      if (p == 0) {
        sort_count_kernel<<<s.blocks, SORT_THREADS, 0, st>>>(s, i, V, padding);
        if (int rc = check_launch("sort_count_kernel")) return rc;
      } else if (int rc = launch_behind(sort_count_kernel, s.blocks, SORT_THREADS, st, s, i, V, padding)) {
        return rc;
      }
      if (int rc = launch_behind(sort_scan_kernel, 1, 1024, st, s.counts, static_cast<int64_t>(s.blocks) * DIGITS)) return rc;
      if (int rc = launch_behind(sort_place_kernel, s.blocks, SORT_THREADS, st, s, i, V, padding)) return rc;
    }
    cur ^= 1;
  }
  SumArgs a = {};
  a.sorted = pairs[cur];
  a.n = tokens; a.V = V; a.D = D; a.lddy = lddy; a.scale = scale;
  a.units = units_of(tokens, V, D);
  a.blocks = static_cast<int>((tokens + V + a.units - 1) / a.units);
  a.starts = reinterpret_cast<int32_t*>(take(a.blocks * static_cast<int64_t>(4)));
  a.joins = reinterpret_cast<int32_t*>(take(a.blocks * static_cast<int64_t>(4)));
  if (tokens > 0) {
    a.head = reinterpret_cast<float*>(take(a.blocks * D * 4));
    a.tail = reinterpret_cast<float*>(take(a.blocks * D * 4));
  }
  using B = __nv_bfloat16;
  if (dy_type == HASTE_BF16) return out_type == HASTE_BF16 ? sums<B, B>(a, dy, dtable, st) : sums<B, float>(a, dy, dtable, st);
  return out_type == HASTE_BF16 ? sums<float, B>(a, dy, dtable, st) : sums<float, float>(a, dy, dtable, st);
}

}  // namespace haste
