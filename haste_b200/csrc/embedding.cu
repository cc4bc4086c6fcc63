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
#include "sm100.cuh"

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
// An id that is no row of the table makes a row of NaN.
template <class T, bool WHOLE>
__global__ void __launch_bounds__(256) embedding_kernel(const Ids ids, const T* __restrict__ table, T* __restrict__ y, int64_t tokens, int64_t D, int64_t V, int64_t ld, float scale) {
  constexpr int N = Vec<T>::N;
  const int64_t n = tokens * D, pieces = (n + N - 1) / N, stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < pieces; i += stride) {
    float v[N];
    int64_t t = n <= 0x7FFFFFFF ? static_cast<uint32_t>(i * N) / static_cast<uint32_t>(D) : i * N / D, c = i * N - t * D;
    if (WHOLE) {                                   // the piece lies in one row, on 16 bytes on both sides
      const int64_t id = ids[t];
      if (static_cast<uint64_t>(id) < static_cast<uint64_t>(V)) {
        Vec<T>::unpack(__ldg(reinterpret_cast<const uint4*>(table + id * ld + c)), v);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] *= scale;
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = __int_as_float(0x7FFFFFFF);
      }
      *reinterpret_cast<uint4*>(y + i * N) = Vec<T>::pack(v);
    } else {
      int64_t id = ids[t];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if (c == D) { c = 0; if (++t < tokens) id = ids[t]; }
        if (t < tokens) y[i * N + k] = Vec<T>::put(static_cast<uint64_t>(id) < static_cast<uint64_t>(V) ? Vec<T>::get(table[id * ld + c]) * scale : __int_as_float(0x7FFFFFFF));
        ++c;
      }
    }
  }
}

// ---------------------------------------------------------------- sorting tokens by id
constexpr int SORT_THREADS = 256, SORT_ITEMS = 16, SORT_TILE = SORT_THREADS * SORT_ITEMS, DIGITS = 256;

struct SortPass {
  const int32_t *keys, *tokens;    // NULL in the first pass: from the ids
  int32_t *keys_out, *tokens_out;
  int32_t* counts;                 // [DIGITS][blocks]
  int64_t n;
  int shift, blocks;
};
// The id, or V where the token has no row or the row is the padding's
__device__ __forceinline__ int32_t key_of(const SortPass& s, const Ids& ids, int64_t i, int64_t V, int64_t padding) {
  if (s.keys != nullptr) return s.keys[i];
  const int64_t id = ids[i];
  return static_cast<uint64_t>(id) < static_cast<uint64_t>(V) && id != padding ? static_cast<int32_t>(id) : static_cast<int32_t>(V);
}
__global__ void __launch_bounds__(SORT_THREADS) sort_count_kernel(const SortPass s, const Ids ids, int64_t V, int64_t padding) {
  __shared__ int32_t count[DIGITS];
  count[threadIdx.x] = 0;
  sm100::grid_dependency_wait();
  __syncthreads();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * SORT_TILE;
  for (int k = 0; k < SORT_ITEMS; ++k) {
    const int64_t i = first + k * SORT_THREADS + threadIdx.x;
    if (i < s.n) atomicAdd(&count[(key_of(s, ids, i, V, padding) >> s.shift) & (DIGITS - 1)], 1);
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
  int32_t key[SORT_ITEMS], rank[SORT_ITEMS];
#pragma unroll
  for (int k = 0; k < SORT_ITEMS; ++k) {
    const int64_t i = first + 32 * k;
    key[k] = i < s.n ? key_of(s, ids, i, V, padding) : 0;
  }
#pragma unroll
  for (int k = 0; k < SORT_ITEMS; ++k) {
    const bool live = first + 32 * k < s.n;
    const int digit = live ? (key[k] >> s.shift) & (DIGITS - 1) : DIGITS;
    const unsigned same = __match_any_sync(0xffffffffu, digit);
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
      const int32_t to = count[warp][(key[k] >> s.shift) & (DIGITS - 1)] + rank[k];
      s.keys_out[to] = key[k];
      s.tokens_out[to] = s.tokens != nullptr ? s.tokens[i] : static_cast<int32_t>(i);
    }
  }
}

// ---------------------------------------------------------------- sums
constexpr int UNITS = 64;          // rows and tokens of a block
constexpr int SUM_THREADS = 128;

// The list of things to do, at place d: v rows are written and i tokens read before it.  A row is written when its last token has been read.
__device__ __forceinline__ int32_t rows_before(const int32_t* __restrict__ keys, int64_t n, int64_t V, int64_t d) {
  int64_t lo = d > V ? d - V : 0, hi = d < n ? d : n;              // the number of tokens among the first d
  while (lo < hi) {
    const int64_t i = (lo + hi) >> 1;                              // is token i among them?  It is before the end of row keys[i], at place i + keys[i].
    if (keys[i] <= d - 1 - i) lo = i + 1;
    else hi = i;
  }
  return static_cast<int32_t>(d - lo);
}

struct SumArgs {
  const int32_t *keys, *tokens;    // sorted
  int32_t* starts;                 // of each block and the end: the row that is worked on there
  float *head, *tail;              // [blocks][D]: parts of a block's first row, begun before it, and of the row after its last one
  int64_t n, V, D, lddy;
  float scale;
  int blocks;
};

// WHOLE: pieces of 16 bytes on both sides; else a thread has every SUM_THREADS-th element
template <class G, class T, bool WHOLE>
__global__ void __launch_bounds__(SUM_THREADS) embedding_sum_kernel(const SumArgs a, const G* __restrict__ dy, T* __restrict__ out) {
  constexpr int N = WHOLE ? Vec<G>::N : 4;
  constexpr int AHEAD = 8;
  __shared__ int32_t todo[UNITS + AHEAD];          // a token, or ~row at its end
  __shared__ int32_t bounds[2];
  sm100::grid_dependency_wait();
  const int64_t d0 = static_cast<int64_t>(blockIdx.x) * UNITS, all = a.V + a.n, d1 = d0 + UNITS < all ? d0 + UNITS : all;
  if (threadIdx.x < 2) {
    const int32_t v = rows_before(a.keys, a.n, a.V, threadIdx.x ? d1 : d0);
    bounds[threadIdx.x] = v;
    if (blockIdx.y == 0 && (threadIdx.x == 0 || d1 == all)) a.starts[blockIdx.x + threadIdx.x] = v;
  }
  if (threadIdx.x < UNITS + AHEAD) todo[threadIdx.x] = INT32_MIN;
  __syncthreads();
  const int32_t v0 = bounds[0], v1 = bounds[1];
  const int64_t i0 = d0 - v0, i1 = d1 - v1;
  // tokens at their places, which those of their rows precede; the places left are rows' ends
  for (int64_t i = i0 + threadIdx.x; i < i1; i += SUM_THREADS) {
    const int32_t key = a.keys[i];
    if (key < a.V) todo[i + key - d0] = a.tokens[i];
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
  const bool begun = i0 > 0 && v0 < a.V && a.keys[i0 - 1] == v0;                   // the first row has tokens before this block
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
  if (open < a.V && i1 > 0 && a.keys[i1 - 1] == open) {          // some of its tokens are read: here, or before
    float* h = a.tail + static_cast<int64_t>(blockIdx.x) * a.D;
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (WHOLE || first + e * SUM_THREADS < a.D) h[WHOLE ? first + e : first + e * SUM_THREADS] = sum[e];
  }
}

// A block whose first row was begun before it, and ends in it: the parts of the blocks before, in order, and its own
constexpr int JOIN_COLUMNS = 32, JOIN_GROUPS = 8;
template <class T>
__global__ void __launch_bounds__(JOIN_COLUMNS * JOIN_GROUPS) embedding_join_kernel(const SumArgs a, T* __restrict__ out) {
  __shared__ float part[JOIN_GROUPS][JOIN_COLUMNS];
  sm100::grid_dependency_wait();
  const int b = blockIdx.x;
  const int32_t row = a.starts[b];
  const int64_t i0 = static_cast<int64_t>(b) * UNITS - row;
  if (b == 0 || row >= a.V || a.starts[b + 1] <= row || i0 == 0 || a.keys[i0 - 1] != row) return;
  // the first block whose tail is of this row: the last that started in an earlier row (or with this row's first token)
  int lo = 0, hi = b - 1;
  while (lo < hi) {
    const int c = (lo + hi + 1) >> 1;
    const int32_t at = a.starts[c];
    const int64_t i = static_cast<int64_t>(c) * UNITS - at;
    if (at < row || i == 0 || a.keys[i - 1] != row) lo = c;
    else hi = c - 1;
  }
  const int group = threadIdx.x / JOIN_COLUMNS, x = threadIdx.x % JOIN_COLUMNS;
  for (int64_t c0 = static_cast<int64_t>(blockIdx.y) * JOIN_COLUMNS; c0 < a.D; c0 += static_cast<int64_t>(gridDim.y) * JOIN_COLUMNS) {
    const int64_t col = c0 + x;
    float s = 0.f;
    if (col < a.D) {
#pragma unroll 4
      for (int c = lo + group; c < b; c += JOIN_GROUPS) s += a.tail[static_cast<int64_t>(c) * a.D + col];
    }
    part[group][x] = s;
    __syncthreads();
    if (group == 0 && col < a.D) {
      for (int g = 1; g < JOIN_GROUPS; ++g) s += part[g][x];
      s += a.head[static_cast<int64_t>(b) * a.D + col];
      out[static_cast<int64_t>(row) * a.D + col] = Vec<T>::put(s * a.scale);
    }
    __syncthreads();
  }
}

int64_t up256(int64_t n) { return (n + 255) & ~int64_t(255); }
int passes_of(int64_t V) {         // over the digits of keys 0 .. V
  int n = 1;
  while (n < 4 && (V >> (8 * n)) > 0) ++n;
  return n;
}
int sort_blocks(int64_t tokens) { return static_cast<int>((tokens + SORT_TILE - 1) / SORT_TILE); }
int64_t sum_blocks(int64_t tokens, int64_t V) { return (tokens + V + UNITS - 1) / UNITS; }

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
    cfg.gridDim = dim3(grid.x, static_cast<unsigned>(imin64((a.D + JOIN_COLUMNS - 1) / JOIN_COLUMNS, 32)));
    cfg.blockDim = dim3(JOIN_COLUMNS * JOIN_GROUPS);
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, embedding_join_kernel<T>, a, o);
  }
  if (e != cudaSuccess) return fail(HASTE_ERR_LAUNCH, "cudaLaunchKernelEx: %s", cudaGetErrorString(e));
  return HASTE_OK;
}

}  // namespace

int launch_embedding_forward(const void* ids, int wide, const void* table, void* y, int64_t tokens, int64_t D, int64_t V, int64_t ld, float scale, int type, cudaStream_t st) {
  if (tokens == 0) return HASTE_OK;
  const int n = type == HASTE_BF16 ? 8 : 4;
  const bool whole = D % n == 0 && ld % n == 0 && aligned16(table) && aligned16(y);
  const int64_t pieces = (tokens * D + n - 1) / n;
  const unsigned grid = static_cast<unsigned>(imin64((pieces + 255) / 256, static_cast<int64_t>(sm_count()) * 64));
  const Ids i = {ids, wide};
  if (type == HASTE_BF16) {
    using B = __nv_bfloat16;
    if (whole) embedding_kernel<B, true><<<grid, 256, 0, st>>>(i, static_cast<const B*>(table), static_cast<B*>(y), tokens, D, V, ld, scale);
    else embedding_kernel<B, false><<<grid, 256, 0, st>>>(i, static_cast<const B*>(table), static_cast<B*>(y), tokens, D, V, ld, scale);
  } else if (whole) {
    embedding_kernel<float, true><<<grid, 256, 0, st>>>(i, static_cast<const float*>(table), static_cast<float*>(y), tokens, D, V, ld, scale);
  } else {
    embedding_kernel<float, false><<<grid, 256, 0, st>>>(i, static_cast<const float*>(table), static_cast<float*>(y), tokens, D, V, ld, scale);
  }
  return check_launch("embedding_kernel");
}

int64_t embedding_backward_scratch(int64_t tokens, int64_t D, int64_t V) {
  if (tokens == 0) return 256 + up256((sum_blocks(0, V) + 1) * 4);
  return 4 * up256(tokens * 4) + up256(static_cast<int64_t>(sort_blocks(tokens)) * DIGITS * 4) + up256((sum_blocks(tokens, V) + 1) * 4) + 2 * up256(sum_blocks(tokens, V) * D * 4);
}

int launch_embedding_backward(const void* ids, int wide, const void* dy, void* dtable, void* scratch, int64_t tokens, int64_t D, int64_t V, int64_t lddy, float scale, int64_t padding,
                              int dy_type, int out_type, cudaStream_t st) {
  char* mem = static_cast<char*>(scratch);
  auto take = [&](int64_t bytes) { char* p = mem; mem += up256(bytes); return p; };
  const Ids i = {ids, wide};
  int32_t *keys[2], *toks[2];
  for (int k = 0; k < 2; ++k) { keys[k] = reinterpret_cast<int32_t*>(take(tokens * 4)); toks[k] = reinterpret_cast<int32_t*>(take(tokens * 4)); }
  SortPass s = {};
  s.n = tokens; s.blocks = sort_blocks(tokens);
  s.counts = reinterpret_cast<int32_t*>(take(static_cast<int64_t>(s.blocks) * DIGITS * 4));
  int cur = 0;
  if (tokens > 0) {
    const int passes = passes_of(V);
    for (int p = 0; p < passes; ++p, cur ^= 1) {
      s.shift = 8 * p;
      s.keys = p ? keys[cur ^ 1] : nullptr; s.tokens = p ? toks[cur ^ 1] : nullptr;
      s.keys_out = keys[cur]; s.tokens_out = toks[cur];
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
  a.keys = keys[cur]; a.tokens = toks[cur];
  a.n = tokens; a.V = V; a.D = D; a.lddy = lddy; a.scale = scale;
  a.blocks = static_cast<int>(sum_blocks(tokens, V));
  a.starts = reinterpret_cast<int32_t*>(take((a.blocks + 1) * static_cast<int64_t>(4)));
  if (tokens > 0) {
    a.head = reinterpret_cast<float*>(take(a.blocks * D * 4));
    a.tail = reinterpret_cast<float*>(take(a.blocks * D * 4));
  }
  using B = __nv_bfloat16;
  if (dy_type == HASTE_BF16) return out_type == HASTE_BF16 ? sums<B, B>(a, dy, dtable, st) : sums<B, float>(a, dy, dtable, st);
  return out_type == HASTE_BF16 ? sums<float, B>(a, dy, dtable, st) : sums<float, float>(a, dy, dtable, st);
}

}  // namespace haste
