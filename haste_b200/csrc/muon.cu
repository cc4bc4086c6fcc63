// Muon: the update of a matrix is its momentum, made orthogonal by Newton-Schulz steps.
//
//   m = mu m + (1 - mu) g,   u = mu m + (1 - mu) g (Nesterov) or m,   X = u / max(|u|, eps)        (X has the smaller side as rows)
//   steps times:  A = X X^T,  B = a I + b A + c A A,  X <- B X
//   w = w (1 - lr weight_decay) - lr rate X
//
// For a list of matrices at once: one launch for the norms, one that writes the momentum and X (rows and columns padded with zeros to multiples of 64, which stay
// zeros: so matrices of nearly one size are one batch), one for all steps (newton_schulz.cuh), one that updates the weights.  Matrices with a side of 32 or less take three others, in 64 bits ("few rows"
// below).
//
// Rounding.  The products take fp16: X times 2^8 (its entries are at most 1, later 1.3 or so; the factor keeps small ones out of the subnormals), A and
// B = a I + b A + c A A.  By the term a I small singular values grow 3.4 times a step, and so does what rounding X adds to them: up to the last but two steps a X takes X as a sum of two fp16 values,
// hi + lo 2^-11, 22 bits, while hi goes through B; in the last two steps X has hi's 11 bits.  Without lo an update of low rank with noise is off by 1.3e-2 after five steps (2-norm of the difference
// over that of the result), with it in the first three by 2.2e-3 at most and a Gaussian one by 1.2e-3 to 1.7e-3 (of 300 x 40: 2.9e-3); with lo in all steps and a outside B 5e-4, with bf16 in place of
// fp16 1e-1 and 1e-2.  The result's own rounding to bf16 is 1.7e-3.  A and A A are symmetric: tiles on and below the diagonal are computed, the others are their mirror.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <vector>

#include "newton_schulz.cuh"

namespace haste {
namespace {

using newton_schulz::LO_SCALE;
using newton_schulz::X_SCALE;

// ---------------------------------------------------------------- elementwise
constexpr int NORM_THREADS = 256;
constexpr int NORM_PARTS = 64;                     // of a matrix, at most
constexpr int NORM_ELEMENTS = 8192;                // of a block, at least
constexpr int FEW = 8, MANY = 192;                 // matrices of one launch
constexpr int SIDE = 64;                           // of an elementwise tile
constexpr int ROWS = SIDE / 16;                    // of a thread: 16 of a block's threads have a row, 4 elements each

struct Matrix {
  const void* g;
  void* w;                         // the parameter, or the result
  float* m;                        // momentum, NULL without
  uint16_t *hi, *lo;               // X's parts, rows of ld elements
  double* parts;                   // sums of squares, by block
  unsigned long long *done, need;  // the steps' counter, and what it shows when they are complete
  int64_t at;                      // place in the momentum, for the random bits
  int rows, cols, ld, nparts;      // ld: X's columns, padded
  float rate;
};
template <int N>
struct Matrices {
  int first_part[N + 1], first_tile[N + 1];        // of each matrix, and the ends
  int n;
  Matrix a[N];
};
struct Coefficients {
  float mu, one_mu, decay, eps;
  int nesterov, sr;
  uint32_t seed, step, stream;
  unsigned long long* drawn;       // the steps' numbers
};
// The last matrix that begins at `block` or before (a walk over all of them took longer than the work: every step a miss in the constants' cache)
__device__ __forceinline__ int matrix_of(const int* first, int n, int block) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= block) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Four neighbouring elements as they lie in memory: looked into only when all loads are on their way
template <class T>
struct Raw;
template <>
struct Raw<__nv_bfloat16> {
  uint2 q;
  __device__ __forceinline__ void zero() { q = make_uint2(0, 0); }
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { q = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int n) {
    const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? u[i] : 0;
    q = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
  }
  __device__ __forceinline__ void get(float (&v)[4]) const {
    const float2 a = gemm::unpack_bf16(q.x), b = gemm::unpack_bf16(q.y);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  }
};
template <>
struct Raw<float> {
  float4 q;
  __device__ __forceinline__ void zero() { q = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load(const float* p) { q = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void load(const float* p, int n) { q = make_float4(n > 0 ? p[0] : 0.f, n > 1 ? p[1] : 0.f, n > 2 ? p[2] : 0.f, n > 3 ? p[3] : 0.f); }
  __device__ __forceinline__ void get(float (&v)[4]) const { v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w; }
};
template <class T>
__device__ __forceinline__ bool on_four(const T* p) { return (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(T) - 1)) == 0; }
__device__ __forceinline__ void store4(float* p, int n, bool vec, const float (&v)[4]) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = v[i];
  }
}
template <class T>
__device__ __forceinline__ bool vec4(const T* p, int n) { return n == 4 && (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(T) - 1)) == 0; }

// The momentum after this step and what is made orthogonal
__device__ __forceinline__ float direction(const Coefficients& c, float g, float& m, bool momentum) {
  if (!momentum) return g;
  m = fmaf(c.mu, m, c.one_mu * g);
  return c.nesterov ? fmaf(c.mu, m, c.one_mu * g) : m;
}

// Bound: memory; 101 M elements, bf16 gradients and fp32 momentum (6 bytes each): 94 us, 98 % of a plain copy's rate.
// Sum of squares of each matrix's direction, in 64 bits (a square of fp32 has a place there whatever its size), in an order that the sizes alone decide
template <class G, int N>
__global__ void __launch_bounds__(NORM_THREADS) muon_squares_kernel(const __grid_constant__ Matrices<N> t, const Coefficients c) {
  constexpr int AT_ONCE = 4;
  __shared__ double warps[NORM_THREADS / 32];
  const int k = matrix_of(t.first_part, t.n, blockIdx.x), part = blockIdx.x - t.first_part[k];
  const Matrix& a = t.a[k];
  const int64_t n = static_cast<int64_t>(a.rows) * a.cols, groups = (n + 3) / 4;
  const G* g = static_cast<const G*>(a.g);
  const float* m = a.m;
  const bool vec = on_four(g);
  const int64_t stride = static_cast<int64_t>(a.nparts) * NORM_THREADS;
  double sum = 0;
  for (int64_t i0 = static_cast<int64_t>(part) * NORM_THREADS + threadIdx.x; i0 < groups; i0 += stride * AT_ONCE) {
    Raw<G> gr[AT_ONCE];
    Raw<float> mr[AT_ONCE];
    if (vec && 4 * (i0 + (AT_ONCE - 1) * stride) + 4 <= n) {
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) gr[j].load(g + 4 * (i0 + j * stride));
      if (m != nullptr) {
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) mr[j].load(m + 4 * (i0 + j * stride));
      }
    } else {                                       // zeros beyond the matrix
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const int64_t i = i0 + j * stride;
        const int have = static_cast<int>(imin64(4, n - 4 * i));
        gr[j].load(g + 4 * i, have);
        if (m != nullptr) mr[j].load(m + 4 * i, have);
      }
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      float gv[4], mv[4] = {0.f, 0.f, 0.f, 0.f};
      gr[j].get(gv);
      if (m != nullptr) mr[j].get(mv);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const double u = direction(c, gv[x], mv[x], m != nullptr);
        sum = fma(u, u, sum);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < NORM_THREADS / 32; ++i) sum += warps[i];
    a.parts[part] = sum;
  }
}

// 1 / max(norm, eps), NaN or 0 where the norm is NaN or inf; by every warp for itself, so the root is taken in 32 bits: of the sum times an even power of two
__device__ __forceinline__ float inverse_norm(const Matrix& a, float eps) {
  const int lane = threadIdx.x & 31;
  double s = (lane < a.nparts ? a.parts[lane] : 0.0) + (lane + 32 < a.nparts ? a.parts[lane + 32] : 0.0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (!(s < INFINITY)) return static_cast<float>(s) - static_cast<float>(s);       // NaN
  const int high = __double2hiint(s), k = ((high >> 20) - 1023) >> 1;              // s = m 4^k, 1 <= m < 4
  const float m = __double2float_rn(s == 0.0 ? 0.0 : __hiloint2double(high - (k << 21), __double2loint(s)));
  const float root = sqrtf(m);
  // |u| = root 2^k against eps, and its inverse
  const float norm = ldexpf(root, k);
  return norm < eps ? 1.f / eps : ldexpf(1.f / root, -k);
}
__device__ __forceinline__ bool usable(float inverse) { return inverse > 0.f && inverse < INFINITY; }
// Whether the steps' launch has done all of them: a wait may have run out in it, and then X's buffer holds something else
__device__ __forceinline__ bool complete(const Matrix& a) { return __ldcg(a.done) == a.need; }

// A block's share of all tiles of 64 x 64, one after the other: what a matrix needs is looked up once
template <int N>
struct Walk {
  const Matrices<N>& t;
  int at, end, k, across, row0, col0;
  __device__ __forceinline__ explicit Walk(const Matrices<N>& m) : t(m) {
    const int tiles = t.first_tile[t.n];
    at = static_cast<int>(static_cast<int64_t>(tiles) * blockIdx.x / gridDim.x);
    end = static_cast<int>(static_cast<int64_t>(tiles) * (blockIdx.x + 1) / gridDim.x);
    k = matrix_of(t.first_tile, t.n, at);
    across = (t.a[k].cols + SIDE - 1) / SIDE;
    const int i = at - t.first_tile[k];
    row0 = i / across * SIDE;
    col0 = (i - i / across * across) * SIDE;
  }
  __device__ __forceinline__ bool more() const { return at < end; }
  // whether the next tile is of another matrix
  __device__ __forceinline__ bool next() {
    ++at;
    col0 += SIDE;
    if (col0 >= across * SIDE) {
      col0 = 0;
      row0 += SIDE;
    }
    if (at < end && at >= t.first_tile[k + 1]) {
      ++k;
      across = (t.a[k].cols + SIDE - 1) / SIDE;
      row0 = col0 = 0;
      return true;
    }
    return false;
  }
};
__device__ __forceinline__ void store_x(const Matrix& a, int row, int col, const float (&x)[4]) {
  const uint32_t h0 = gemm::pack_f16(x[0], x[1]), h1 = gemm::pack_f16(x[2], x[3]);
  const float2 a0 = gemm::unpack_f16(h0), a1 = gemm::unpack_f16(h1);
  const int64_t to = static_cast<int64_t>(row) * a.ld + col;
  *reinterpret_cast<uint2*>(a.hi + to) = make_uint2(h0, h1);
  *reinterpret_cast<uint2*>(a.lo + to) = make_uint2(gemm::pack_f16((x[0] - a0.x) * LO_SCALE, (x[1] - a0.y) * LO_SCALE), gemm::pack_f16((x[2] - a1.x) * LO_SCALE, (x[3] - a1.y) * LO_SCALE));
}

// Bound: memory; 101 M elements (14 bytes each): 277 us, 78 % of a plain copy's rate.  (A look into bf16 pairs right behind each load, or a walk over the tables at each tile, kept the loads from being on their
// way together: they are raw until all are asked for, and a block walks neighbouring tiles.)
// Momentum and X, zeros in its padding.  A matrix whose norm is not finite keeps its momentum.
template <class G, int N>
__global__ void __launch_bounds__(256) muon_start_kernel(const __grid_constant__ Matrices<N> t, const Coefficients c) {
  __shared__ float turned[SIDE][SIDE + 1];
  Walk<N> walk(t);
  const int cg = (threadIdx.x & 15) * 4, r0 = threadIdx.x / 16;
  sm100::grid_dependency_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0) *c.drawn = 0;
  float inv = walk.more() ? inverse_norm(t.a[walk.k], c.eps) : 0.f;
  while (walk.more()) {
    const Matrix& a = t.a[walk.k];
    const int row0 = walk.row0, col0 = walk.col0;
    const bool tall = a.rows > a.cols, momentum = a.m != nullptr, write = momentum && usable(inv);
    const float factor = inv * X_SCALE;
    const int col = col0 + cg, have = min(4, a.cols - col);
    const G* g = static_cast<const G*>(a.g);
    Raw<G> gr[ROWS];
    Raw<float> mr[ROWS];
    // a tile within the matrix, whose rows all start on four elements
    const bool whole = row0 + SIDE <= a.rows && col0 + SIDE <= a.cols && a.cols % 4 == 0 && on_four(g);
    const int64_t from = static_cast<int64_t>(row0 + r0) * a.cols + col, step = static_cast<int64_t>(16) * a.cols;
    if (whole) {
#pragma unroll
      for (int k = 0; k < ROWS; ++k) gr[k].load(g + from + k * step);
      if (momentum) {
#pragma unroll
        for (int k = 0; k < ROWS; ++k) mr[k].load(a.m + from + k * step);
      }
    } else {
#pragma unroll
      for (int k = 0; k < ROWS; ++k) {
        const int n = row0 + r0 + 16 * k < a.rows ? have : 0;
        gr[k].load(g + from + k * step, n);
        if (momentum) mr[k].load(a.m + from + k * step, n);
      }
    }
    if (row0 == 0 && col0 == 0 && threadIdx.x == 0) *a.done = 0;
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const int r = r0 + 16 * k, row = row0 + r;
      const int64_t i = static_cast<int64_t>(row) * a.cols + col;
      const bool there = row < a.rows;
      float x[4], gv[4], mv[4] = {0.f, 0.f, 0.f, 0.f};
      gr[k].get(gv);
      if (momentum) mr[k].get(mv);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = direction(c, gv[e], mv[e], momentum) * factor;
        if (!there || e >= have) x[e] = 0.f;
      }
      if (write && there && have > 0) store4(a.m + i, have, vec4(a.m + i, have), mv);
      if (tall) {
#pragma unroll
        for (int e = 0; e < 4; ++e) turned[cg + e][r] = x[e];
      } else {
        store_x(a, row, col, x);
      }
    }
    if (tall) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < ROWS; ++k) {
        const int r = r0 + 16 * k;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = turned[r][cg + e];
        store_x(a, col0 + r, row0 + cg, x);
      }
      __syncthreads();
    }
    if (walk.next()) inv = inverse_norm(t.a[walk.k], c.eps);
  }
}

// Philox4x32 with 7 rounds, key (seed, step), counter (i, i >> 32, stream, 2): one word for each of the elements 4 i .. 4 i + 3
__device__ __forceinline__ uint4 random_words(const Coefficients& c, int64_t i) {
  uint32_t c0 = static_cast<uint32_t>(i), c1 = static_cast<uint32_t>(static_cast<uint64_t>(i) >> 32), c2 = c.stream, c3 = 2, k0 = c.seed, k1 = c.step;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(0xD2511F53u) * c0, p1 = static_cast<uint64_t>(0xCD9E8D57u) * c2;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0; c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
    c1 = static_cast<uint32_t>(p1); c3 = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}
__device__ __forceinline__ uint32_t word(const uint4& r, int i) { return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w; }

__device__ __forceinline__ void store_weights(float* p, int have, const float (&v)[4], const Coefficients&, int64_t) { store4(p, have, vec4(p, have), v); }
// No random bits for a NaN: it is 0x7FFFFFFF here, and adding any would run over into the sign and leave -0.  A sum that is no NaN has none among its terms: nearly always one test is all
// that it takes.
__device__ __forceinline__ void spare_nans(uint32_t (&random)[4], const float (&v)[4]) {
  const float any = (v[0] + v[1]) + (v[2] + v[3]);
  if (any != any) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (v[e] != v[e]) random[e] = 0;
  }
}

__device__ __forceinline__ void store_weights(__nv_bfloat16* p, int have, const float (&v)[4], const Coefficients& c, int64_t i) {
  uint32_t b[4];
  if (c.sr) {
    const uint4 first = random_words(c, i >> 2);
    if ((i & 3) == 0) {
      b[0] = first.x; b[1] = first.y; b[2] = first.z; b[3] = first.w;
    } else {
      const int skip = static_cast<int>(i & 3);
      const uint4 second = random_words(c, (i >> 2) + 1);
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = word(e + skip < 4 ? first : second, (e + skip) & 3);
    }
    spare_nans(b, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = sr_bf16_bits(v[e], b[e] & 0xFFFFu);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = rn_bf16_bits(v[e]);
  }
  if (vec4(p, have)) {
    *reinterpret_cast<uint2*>(p) = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < have) p[e] = __ushort_as_bfloat16(static_cast<uint16_t>(b[e]));
  }
}

// Four elements whose place in memory and in the momentum is a multiple of four
__device__ __forceinline__ void store_whole(float* p, const float (&v)[4], const Coefficients&, int64_t) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store_whole(__nv_bfloat16* p, const float (&v)[4], const Coefficients& c, int64_t i) {
  if (c.sr) {
    const uint4 r = random_words(c, i >> 2);
    uint32_t b[4] = {r.x, r.y, r.z, r.w};
    spare_nans(b, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(v[e]) + (b[e] & 0xFFFFu);          // the upper halves are what sr_bf16_bits() gives
    *reinterpret_cast<uint2*>(p) = make_uint2(__byte_perm(b[0], b[1], 0x7632), __byte_perm(b[2], b[3], 0x7632));
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(gemm::pack_bf16(v[0], v[1]), gemm::pack_bf16(v[2], v[3]));
  }
}

// Bound: instruction issue (random words and rounding), then memory: 101 M bf16 weights rounded stochastically 164 us, 56 % of a plain copy's rate for 6 bytes an element; 11 more with whole tiles stored as
// the ragged ones are and random words from separate halves of products.  50 M elements of X alone, 4 bytes each: 47 us, 65 %.
// UPDATE: the weights, left alone where the norm is not finite or the steps are not complete; else X itself, in bf16, NaN where they are not
template <class W, bool UPDATE, int N>
__global__ void __launch_bounds__(256) muon_finish_kernel(const __grid_constant__ Matrices<N> t, const Coefficients c) {
  __shared__ float turned[SIDE][SIDE + 1];
  Walk<N> walk(t);
  const int cg = (threadIdx.x & 15) * 4, r0 = threadIdx.x / 16;
  sm100::grid_dependency_wait();
  float inv = UPDATE && walk.more() ? inverse_norm(t.a[walk.k], c.eps) : 1.f;
  bool done = walk.more() && complete(t.a[walk.k]);
  while (walk.more()) {
    const Matrix& a = t.a[walk.k];
    const int row0 = walk.row0, col0 = walk.col0, col = col0 + cg, have = min(4, a.cols - col);
    const bool tall = a.rows > a.cols;
    W* w = static_cast<W*>(a.w);
    if (!UPDATE || (done && usable(inv))) {     // the same for all of the block
      const float unit = done ? 1.f / X_SCALE : __int_as_float(0x7FFFFFFF);
      Raw<W> wr[ROWS];
      uint2 q[ROWS];
      float x[ROWS][4];
      const int64_t from = static_cast<int64_t>(row0 + r0) * a.cols + col, step = static_cast<int64_t>(16) * a.cols;
      const uint16_t* hi = a.hi + static_cast<int64_t>((tall ? col0 : row0) + r0) * a.ld + (tall ? row0 : col0) + cg;
      const bool whole = row0 + SIDE <= a.rows && col0 + SIDE <= a.cols && a.cols % 4 == 0 && on_four(w);
      if (UPDATE) {
        if (whole) {
#pragma unroll
          for (int k = 0; k < ROWS; ++k) wr[k].load(w + from + k * step);
        } else {
#pragma unroll
          for (int k = 0; k < ROWS; ++k) wr[k].load(w + from + k * step, row0 + r0 + 16 * k < a.rows ? have : 0);
        }
      }
#pragma unroll
      for (int k = 0; k < ROWS; ++k) q[k] = *reinterpret_cast<const uint2*>(hi + static_cast<int64_t>(16 * k) * a.ld);
#pragma unroll
      for (int k = 0; k < ROWS; ++k) {
        const float2 x0 = gemm::unpack_f16(q[k].x), x1 = gemm::unpack_f16(q[k].y);
        x[k][0] = x0.x; x[k][1] = x0.y; x[k][2] = x1.x; x[k][3] = x1.y;
      }
      if (tall) {
#pragma unroll
        for (int k = 0; k < ROWS; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) turned[cg + e][r0 + 16 * k] = x[k][e];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ROWS; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[k][e] = turned[r0 + 16 * k][cg + e];
        __syncthreads();
      }
#pragma unroll
      for (int k = 0; k < ROWS; ++k) {
        const int row = row0 + r0 + 16 * k;
        if (row < a.rows && have > 0) {
          const int64_t i = static_cast<int64_t>(row) * a.cols + col;
          float v[4];
          if (UPDATE) wr[k].get(v);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = UPDATE ? fmaf(-a.rate * (1.f / X_SCALE), x[k][e], v[e] * c.decay) : x[k][e] * unit;
          if (whole) store_whole(w + i, v, c, a.at + i);
          else store_weights(w + i, have, v, c, a.at + i);
        }
      }
    }
    if (walk.next()) {
      if (UPDATE) inv = inverse_norm(t.a[walk.k], c.eps);
      done = complete(t.a[walk.k]);
    }
  }
}

// ---------------------------------------------------------------- few rows
// X of at most FEW_ROWS rows.  A few roundings of A and B to fp16 do not average out: steps with the products above are off by up to 1.2e-2 for 2 x 3 and 6.9e-3 for 2 x 300 (worst of 400), 4.3e-3 for
// 8 x 30, 3.1e-3 for 24 x 300, 2.4e-3 for 32 x 300; from 33 rows on by 2.3e-3, where rounding the result alone gives 1.7e-3.  All X_k are polynomials of G = u u^T times u, and G is p x p:
//   X_k = F_k u,   A_k = F_k G F_k,   M = a I + b A_k + c A_k A_k,   F_{k+1} = M F_k,   A_{k+1} = M (M A_k)        (symmetric matrices that commute)
// All of that is in 64 bits: F grows 3.4 times a step where singular values are small, and what G is rounded to with its square, so that 32 bits would leave 1e-3.  One launch for G, in parts along the
// longer side, one that adds them and takes the steps, one for F u and what is done with it.  Nothing is rounded to fewer than 32 bits but the result.
//
// Bound: the 64-bit products (16 a clock and SM) of the one block that takes a matrix's steps, 5 us for 16 rows and 20 for 32, and three launches' latency; long ones by those of G and F u.  A call, in
// brackets with the products above: 8 x 8 15 us (66), 32 x 32 31 (66), 32 x 768 41 (85), 16 x 4096 25 (158), 30 x 40000 80 (1020), 32 x 1000000 859 (23410), 40 of 20 x 300 50 (109), 200 of 32 x 512
// 213 (301).  Beside larger matrices the three launches come first: 512 x 768 and 20 of 16 x 1000 147 (182), 512 x 768 and 8 of 32 x 32 150 (129).
constexpr int FEW_ROWS = 32, FEW_THREADS = 256;
constexpr int FEW_SLOTS = 2048;                    // elements that a block has at a time: 8 a thread
constexpr int GRAM_LOOPS = 4, GRAM_PARTS = 128;    // times so many for a part of G at least, and its parts at most
static_assert(FEW_SLOTS == 8 * FEW_THREADS, "");

__host__ __device__ __forceinline__ int log_rows(int p) { return p <= 4 ? 2 : p <= 8 ? 3 : p <= 16 ? 4 : 5; }        // of X's rows in a block, a power of two
// G's tiles of 4 x 4 on and below the diagonal, all of one part after the other's
__host__ __device__ __forceinline__ int gram_tiles(int p) { const int n = (p + 3) >> 2; return n * (n + 1) / 2; }
__host__ __device__ __forceinline__ int gram_size(int p) { return 16 * gram_tiles(p); }

// A thread's 8 elements of the direction from place j0 along the longer side on, zeros beyond it: all loads are on their way before one is looked at (looked at one by one they took 4 us of 5)
template <class G>
struct Eight {
  G g[8];
  float m[8];
  int64_t at[8];                   // in the matrix, -1 where there is none
  int to[8];                       // row * rows' stride + place, or the other way round
  // by_row: whether a row's places are neighbours in shared memory
  __device__ __forceinline__ void load(const Matrix& a, bool by_row, int p, int lp, int ld, int64_t j0, int n) {
    const bool tall = a.rows > a.cols;
    const int lj = 11 - lp, rows = 1 << lp, places = 1 << lj;
    const int64_t longer = max(a.rows, a.cols);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int e = threadIdx.x + FEW_THREADS * x, i = tall ? e & (rows - 1) : e >> lj, j = tall ? e >> lp : e & (places - 1);
      to[x] = by_row ? i * ld + j : j * ld + i;
      at[x] = i >= p || j >= n ? -1 : tall ? (j0 + j) * p + i : i * longer + j0 + j;
    }
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (at[x] >= 0) g[x] = static_cast<const G*>(a.g)[at[x]];
    if (a.m != nullptr) {
#pragma unroll
      for (int x = 0; x < 8; ++x)
        if (at[x] >= 0) m[x] = a.m[at[x]];
    }
  }
  // The direction, and the momentum after this step in m
  __device__ __forceinline__ float direction_of(int x, const Coefficients& c, bool momentum) { return at[x] < 0 ? 0.f : direction(c, static_cast<float>(g[x]), m[x], momentum); }
};

template <class G, int N>
__global__ void __launch_bounds__(FEW_THREADS) muon_gram_kernel(const __grid_constant__ Matrices<N> t, const Coefficients c) {
  __shared__ __align__(16) double mem[16 * FEW_THREADS];            // u, [places][rows + 2]; at last the threads' sums
  const int k = matrix_of(t.first_part, t.n, blockIdx.x), part = blockIdx.x - t.first_part[k];
  const Matrix& a = t.a[k];
  const int p = min(a.rows, a.cols), lp = log_rows(p), places = FEW_SLOTS >> lp, ld = (1 << lp) + 2;
  const int64_t longer = max(a.rows, a.cols), begin = longer * part / a.nparts, end = longer * (part + 1) / a.nparts;
  const int tiles = gram_tiles(p), slices = FEW_THREADS / tiles, slice = threadIdx.x / tiles, tile = threadIdx.x - slice * tiles;
  int ti = 0;
  while ((ti + 1) * (ti + 2) / 2 <= tile) ++ti;
  const int tj = tile - ti * (ti + 1) / 2;
  double acc[4][4] = {};
  for (int64_t j0 = begin; j0 < end; j0 += places) {
    const int n = static_cast<int>(imin64(places, end - j0));
    Eight<G> u;
    u.load(a, false, p, lp, ld, j0, n);
#pragma unroll
    for (int x = 0; x < 8; ++x) mem[u.to[x]] = u.direction_of(x, c, a.m != nullptr);
    __syncthreads();
    if (slice < slices)
      for (int j = slice; j < n; j += slices) {
        const double2 *x = reinterpret_cast<const double2*>(mem + j * ld + 4 * ti), *y = reinterpret_cast<const double2*>(mem + j * ld + 4 * tj);
        const double2 x0 = x[0], x1 = x[1], y0 = y[0], y1 = y[1];
        const double xs[4] = {x0.x, x0.y, x1.x, x1.y}, ys[4] = {y0.x, y0.y, y1.x, y1.y};
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[r][q] = fma(xs[r], ys[q], acc[r][q]);
      }
    __syncthreads();
  }
  if (slice < slices) {
#pragma unroll
    for (int e = 0; e < 16; ++e) mem[(slice * tiles + tile) * 16 + e] = acc[e >> 2][e & 3];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * tiles; e += FEW_THREADS) {
    double sum = 0;
    for (int s = 0; s < slices; ++s) sum += mem[s * tiles * 16 + e];
    a.parts[static_cast<int64_t>(part) * 16 * tiles + e] = sum;
  }
}

// Rows of the matrices in shared memory.  What stands on the left of a product is symmetric, so that two neighbours of its column are two of its row: 16 bytes at a time (8 at a time, and a product for each of the two of M below,
// the second launch took 30 us for 32 rows).
constexpr int FEW_LD = FEW_ROWS + 2;
struct Square {
  double2 at[FEW_ROWS][FEW_LD / 2];
  __device__ __forceinline__ double& operator()(int i, int j) { return reinterpret_cast<double*>(at[i])[j]; }
};
// 2 x 2 of x y, at (i, j), for matrices of p rows
__device__ __forceinline__ void times(const Square& x, const Square& y, int p, int i, int j, double (&out)[2][2]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e >> 1][e & 1] = 0;
#pragma unroll 4
  for (int k = 0; k < p; ++k) {
    const double2 l = x.at[k][i >> 1], r = y.at[k][j >> 1];
    out[0][0] = fma(l.x, r.x, out[0][0]); out[0][1] = fma(l.x, r.y, out[0][1]);
    out[1][0] = fma(l.y, r.x, out[1][0]); out[1][1] = fma(l.y, r.y, out[1][1]);
  }
}
__device__ __forceinline__ void times(const Square& x, const Square& y, const Square& z, int p, int i, int j, double (&out)[2][2], double (&other)[2][2]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e >> 1][e & 1] = other[e >> 1][e & 1] = 0;
#pragma unroll 4
  for (int k = 0; k < p; ++k) {
    const double2 l = x.at[k][i >> 1], r = y.at[k][j >> 1], q = z.at[k][j >> 1];
    out[0][0] = fma(l.x, r.x, out[0][0]); out[0][1] = fma(l.x, r.y, out[0][1]);
    out[1][0] = fma(l.y, r.x, out[1][0]); out[1][1] = fma(l.y, r.y, out[1][1]);
    other[0][0] = fma(l.x, q.x, other[0][0]); other[0][1] = fma(l.x, q.y, other[0][1]);
    other[1][0] = fma(l.y, q.x, other[1][0]); other[1][1] = fma(l.y, q.y, other[1][1]);
  }
}
__device__ __forceinline__ void put(Square& to, int i, int j, const double (&v)[2][2]) {
  to.at[i][j >> 1] = make_double2(v[0][0], v[0][1]);
  to.at[i + 1][j >> 1] = make_double2(v[1][0], v[1][1]);
}
// Where a matrix's F / |u| [p][p] lies, behind G's parts, and behind it whether the norm is finite (1 or 0)
__device__ __forceinline__ double* factor_of(const Matrix& a, int p) { return a.parts + static_cast<int64_t>(a.nparts) * gram_size(p); }

// A block for each matrix
template <int N>
__global__ void __launch_bounds__(FEW_THREADS) muon_few_steps_kernel(const __grid_constant__ Matrices<N> t, const Coefficients c, int steps, double ca, double cb, double cc) {
  __shared__ Square A, M, F, T;
  const Matrix& a = t.a[blockIdx.x];
  const int p = min(a.rows, a.cols), size = gram_size(p), i = 2 * (threadIdx.x >> 4), j = 2 * (threadIdx.x & 15);
  sm100::grid_dependency_wait();
  for (int e = threadIdx.x; e < FEW_ROWS * FEW_ROWS; e += FEW_THREADS) {
    const int r = e / FEW_ROWS, q = e % FEW_ROWS, hi = max(r, q), lo = min(r, q);
    double sum = 0;
    if (hi < p) {
      const double* from = a.parts + 16 * ((hi >> 2) * ((hi >> 2) + 1) / 2 + (lo >> 2)) + 4 * (hi & 3) + (lo & 3);
#pragma unroll 8
      for (int k = 0; k < a.nparts; ++k) sum += from[static_cast<int64_t>(k) * size];
    }
    A(r, q) = sum;
  }
  __syncthreads();
  double squares = 0;
  for (int k = 0; k < p; ++k) squares += A(k, k);
  const bool finite = squares < INFINITY;          // (not NaN either)
  const double norm = sqrt(squares), inv = 1.0 / (norm < c.eps ? static_cast<double>(c.eps) : norm);
  __syncthreads();
  for (int e = threadIdx.x; e < FEW_ROWS * FEW_ROWS; e += FEW_THREADS) A(e / FEW_ROWS, e % FEW_ROWS) *= inv * inv;
  __syncthreads();
  const bool mine = i < p && j < p;
  for (int s = 0; s < steps; ++s) {
    const bool more = s + 1 < steps;
    double v[2][2], w[2][2];
    if (mine) {
      times(A, A, p, i, j, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = i + (e >> 1), q = j + (e & 1);
        v[e >> 1][e & 1] = fma(cc, v[e >> 1][e & 1], fma(cb, A(r, q), r == q ? ca : 0.0));
      }
      put(M, i, j, v);
      if (s == 0) put(F, i, j, v);
    }
    __syncthreads();
    if (mine) {
      if (s == 0) {
        if (more) times(M, A, p, i, j, w);
      } else if (more) {
        times(M, F, A, p, i, j, v, w);
      } else {
        times(M, F, p, i, j, v);
      }
    }
    __syncthreads();
    if (mine) {
      if (s > 0) put(F, i, j, v);
      if (more) put(T, i, j, w);
    }
    __syncthreads();
    if (mine && more && i >= j) {
      // A is kept symmetric to the last bit, and M with it: what it were not would grow by 4 times a step and more (2e-9 of the result after 9 steps, 1e-2 after 15)
      times(M, T, p, i, j, v);
      if (i == j) v[0][1] = v[1][0];
      put(A, i, j, v);
      if (i > j) {
        const double turned[2][2] = {{v[0][0], v[1][0]}, {v[0][1], v[1][1]}};
        put(A, j, i, turned);
      }
    }
    __syncthreads();
  }
  double* to = factor_of(a, p);
  for (int e = threadIdx.x; e < p * p; e += FEW_THREADS) to[e] = F(e / p, e % p) * inv;
  if (threadIdx.x == 0) to[p * p] = finite ? 1.0 : 0.0;
}

// UPDATE: momentum and weights, left alone where the norm is not finite; else X itself, NaN there
template <class G, class W, bool UPDATE, int N>
__global__ void __launch_bounds__(FEW_THREADS) muon_few_finish_kernel(const __grid_constant__ Matrices<N> t, const Coefficients c) {
  __shared__ double F[FEW_ROWS][FEW_ROWS], u[FEW_SLOTS + FEW_ROWS];           // u, and X: [rows][places + 1]
  __shared__ float x[FEW_SLOTS + FEW_ROWS];
  sm100::grid_dependency_wait();
  const int all = t.first_tile[t.n];
  int at = static_cast<int>(static_cast<int64_t>(all) * blockIdx.x / gridDim.x);
  const int end = static_cast<int>(static_cast<int64_t>(all) * (blockIdx.x + 1) / gridDim.x);
  int k = matrix_of(t.first_tile, t.n, at);
  bool fresh = true, finite = false;
  for (; at < end; ++at) {
    if (at >= t.first_tile[k + 1]) { ++k; fresh = true; }
    const Matrix& a = t.a[k];
    const bool tall = a.rows > a.cols;
    const int p = min(a.rows, a.cols), lp = log_rows(p), rows = 1 << lp, places = FEW_SLOTS >> lp, ld = places + 1;
    const int64_t longer = max(a.rows, a.cols), j0 = static_cast<int64_t>(at - t.first_tile[k]) * places;
    const int n = static_cast<int>(imin64(places, longer - j0));
    if (fresh) {
      const double* from = factor_of(a, p);
      for (int e = threadIdx.x; e < FEW_ROWS * FEW_ROWS; e += FEW_THREADS) {
        const int r = e / FEW_ROWS, q = e % FEW_ROWS;
        F[r][q] = r < p && q < p ? from[r * p + q] : 0.0;
      }
      finite = from[p * p] == 1.0;
      fresh = false;
    }
    if (!UPDATE || finite) {                       // the same for all of the block
      Eight<G> v;
      v.load(a, true, p, lp, ld, j0, n);
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        u[v.to[s]] = v.direction_of(s, c, a.m != nullptr);
        if (UPDATE && v.at[s] >= 0) a.m[v.at[s]] = v.m[s];
      }
      __syncthreads();
      // 8 rows of X a thread (4, where there are no more)
      const int groups = rows >> 3 ? rows >> 3 : 1, i0 = 8 * (threadIdx.x % groups);
      for (int j = threadIdx.x / groups; j < n; j += FEW_THREADS / groups) {
        double sum[8] = {};
        for (int r = 0; r < p; ++r) {
          const double y = u[r * ld + j];
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[e] = fma(F[r][i0 + e], y, sum[e]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i0 + e < p) x[(i0 + e) * ld + j] = finite ? static_cast<float>(sum[e]) : __int_as_float(0x7FFFFFFF);
      }
      __syncthreads();
      // four neighbours in memory at a time
      W* w = static_cast<W*>(a.w);
      const int across = tall ? (p + 3) >> 2 : (n + 3) >> 2, lines = tall ? n : p;
      for (int e = threadIdx.x; e < across * lines; e += FEW_THREADS) {
        const int line = e / across, first = 4 * (e - line * across), have = min(4, (tall ? p : n) - first);
        const int64_t i = tall ? (j0 + line) * p + first : line * longer + j0 + first;
        float y[4], z[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) y[q] = q < have ? (tall ? x[(first + q) * ld + line] : x[line * ld + first + q]) : 0.f;
        if (UPDATE) {
          Raw<W> old;
          old.load(w + i, have);
          old.get(z);
#pragma unroll
          for (int q = 0; q < 4; ++q) y[q] = fmaf(-a.rate, y[q], z[q] * c.decay);
        }
        store_weights(w + i, have, y, c, a.at + i);
      }
      __syncthreads();
    } else {
      __syncthreads();                             // F is read by all before it is another one's
    }
  }
}

// ---------------------------------------------------------------- host side
constexpr int64_t ROUND_BYTES = int64_t(1) << 30;      // of scratch memory, unless one matrix needs more: a round of so much keeps the GPU busy for a millisecond

int64_t up64(int64_t n) { return (n + 63) & ~int64_t(63); }
int64_t up256(int64_t n) { return (n + 255) & ~int64_t(255); }
struct Sizes {
  int64_t p, q;                    // rows and columns of X, padded
  int64_t x() const { return p * q; }
  int64_t a() const { return p * p; }
  int64_t bytes() const { return 2 * (3 * x() + a()) + 4 * 256 + 8 * NORM_PARTS + 8; }
};
Sizes sizes_of(int64_t rows, int64_t cols) { return {up64(std::min(rows, cols)), up64(std::max(rows, cols))}; }
bool few_rows(int64_t rows, int64_t cols) { return std::min(rows, cols) <= FEW_ROWS; }
int gram_parts(int64_t rows, int64_t cols) {
  const int64_t each = static_cast<int64_t>(GRAM_LOOPS) * (FEW_SLOTS >> log_rows(static_cast<int>(std::min(rows, cols))));
  return static_cast<int>(std::min<int64_t>(GRAM_PARTS, (std::max(rows, cols) + each - 1) / each));
}
int64_t few_bytes(int64_t rows, int64_t cols) {              // of G's parts and F
  const int p = static_cast<int>(std::min(rows, cols));
  return up256(8 * (static_cast<int64_t>(gram_parts(rows, cols)) * gram_size(p) + p * p + 1));
}
int64_t bytes_of(int64_t rows, int64_t cols) { return few_rows(rows, cols) ? few_bytes(rows, cols) : sizes_of(rows, cols).bytes(); }

// The matrices by shape, cut into rounds.  Rounds are those of the whole list, whichever of it have a gradient: fewer of them in a round need less, but other rounds could need more than the
// scratch memory that was asked for.
struct Plan {
  std::vector<int64_t> order;
  std::vector<size_t> rounds;      // where in `order` each begins, and the end
  int64_t bytes = 0;
};
Plan plan_of(const int64_t* rows, const int64_t* cols, int64_t count) {
  Plan p;
  for (int64_t i = 0; i < count; ++i)
    if (rows[i] > 0 && cols[i] > 0) p.order.push_back(i);
  auto key = [&](int64_t i) { const Sizes s = sizes_of(rows[i], cols[i]); return std::make_pair(s.p, s.q); };
  std::stable_sort(p.order.begin(), p.order.end(), [&](int64_t i, int64_t j) { return key(i) > key(j); });
  int64_t used = 0;
  for (size_t k = 0; k < p.order.size(); ++k) {
    const int64_t need = bytes_of(rows[p.order[k]], cols[p.order[k]]);
    if (k == 0 || used + need > ROUND_BYTES) {
      p.rounds.push_back(k);
      used = 0;
    }
    used += need;
    p.bytes = std::max(p.bytes, used + 512);
  }
  p.rounds.push_back(p.order.size());
  return p;
}

// f(table, blocks of squares, elementwise tiles) for the matrices, as many at a time as a launch's parameters hold
template <bool FEW_OF_X, int N, class F>
int with_table(const std::vector<Matrix>& all, size_t from, F&& f) {
  static thread_local Matrices<N> t;
  t.n = static_cast<int>(std::min<size_t>(N, all.size() - from));
  int64_t parts = 0, tiles = 0;
  for (int k = 0; k < t.n; ++k) {
    const Matrix& a = t.a[k] = all[from + k];
    t.first_part[k] = static_cast<int>(parts);
    t.first_tile[k] = static_cast<int>(tiles);
    parts += a.nparts;
    if (FEW_OF_X) tiles += (std::max(a.rows, a.cols) + (FEW_SLOTS >> log_rows(std::min(a.rows, a.cols))) - 1) / (FEW_SLOTS >> log_rows(std::min(a.rows, a.cols)));
    else tiles += static_cast<int64_t>((a.rows + SIDE - 1) / SIDE) * ((a.cols + SIDE - 1) / SIDE);
    if (tiles > 0x7FFFFFFF) return fail(HASTE_ERR_TOO_LARGE, "matrices of too many elements for one call");
  }
  t.first_part[t.n] = static_cast<int>(parts); t.first_tile[t.n] = static_cast<int>(tiles);
  // the elementwise launches' blocks share the tiles: as many as run at once
  return f(t, std::integral_constant<int, N>(), static_cast<unsigned>(parts), static_cast<unsigned>(imin64(tiles, static_cast<int64_t>(sm_count()) * 6)));
}
template <bool FEW_OF_X, class F>
int for_each_table(const std::vector<Matrix>& all, F&& f) {
  for (size_t i = 0; i < all.size(); i += MANY) {
    const int rc = all.size() - i <= FEW ? with_table<FEW_OF_X, FEW>(all, i, f) : with_table<FEW_OF_X, MANY>(all, i, f);
    if (rc) return rc;
  }
  return HASTE_OK;
}

// Everything for matrices of few rows
int launch_few_rows(const std::vector<Matrix>& all, const MuonCall& c, const Coefficients& k, cudaStream_t st) {
  const bool gb = c.g_type == HASTE_BF16;
  return for_each_table<true>(all, [&](const auto& t, auto size, unsigned parts, unsigned tiles) -> int {
    constexpr int N = decltype(size)::value;
    using B = __nv_bfloat16;
    if (gb) muon_gram_kernel<B, N><<<parts, FEW_THREADS, 0, st>>>(t, k);
    else muon_gram_kernel<float, N><<<parts, FEW_THREADS, 0, st>>>(t, k);
    if (int e = check_launch("muon_gram_kernel")) return e;
    if (int e = launch_behind(muon_few_steps_kernel<N>, static_cast<unsigned>(t.n), FEW_THREADS, st, t, k, c.steps, c.a, c.b, c.c)) return e;
    auto finish = [&](auto kernel) { return launch_behind(kernel, tiles, FEW_THREADS, st, t, k); };
    if (!c.update) return gb ? finish(muon_few_finish_kernel<B, B, false, N>) : finish(muon_few_finish_kernel<float, B, false, N>);
    if (c.p_type == HASTE_BF16) return gb ? finish(muon_few_finish_kernel<B, B, true, N>) : finish(muon_few_finish_kernel<float, B, true, N>);
    return gb ? finish(muon_few_finish_kernel<B, float, true, N>) : finish(muon_few_finish_kernel<float, float, true, N>);
  });
}

}  // namespace

int64_t muon_scratch(const int64_t* rows, const int64_t* cols, int64_t count) { return plan_of(rows, cols, count).bytes; }

int launch_muon(const MuonCall& c, cudaStream_t st) {
  if (int rc = report_pending_status(c.who)) return rc;
  const Plan plan = plan_of(c.rows, c.cols, c.count);
  std::vector<int64_t> at(c.count);
  int64_t total = 0;
  for (int64_t i = 0; i < c.count; ++i) {
    at[i] = total;
    total += (c.rows[i] * c.cols[i] + 255) / 256 * 256;
  }
  Coefficients k;
  k.mu = static_cast<float>(c.mu); k.one_mu = static_cast<float>(1.0 - c.mu);
  k.decay = static_cast<float>(1.0 - c.lr * c.weight_decay);
  k.eps = static_cast<float>(c.eps);
  k.nesterov = c.nesterov; k.sr = (c.flags & HASTE_F_SR) ? 1 : 0;
  k.seed = static_cast<uint32_t>(c.seed); k.step = static_cast<uint32_t>(c.step); k.stream = c.stream;
  for (size_t r = 0; r + 1 < plan.rounds.size(); ++r) {
    char* mem = static_cast<char*>(c.scratch);
    auto take = [&](int64_t bytes) { char* p = mem; mem += up256(bytes); return p; };
    std::vector<int64_t> some, few;    // those with a gradient
    for (size_t i = plan.rounds[r]; i < plan.rounds[r + 1]; ++i) {
      const int64_t o = plan.order[i];
      if (c.grads[o] != nullptr) (few_rows(c.rows[o], c.cols[o]) ? few : some).push_back(o);
    }
    const bool gb = c.g_type == HASTE_BF16;
    auto matrix = [&](int64_t o) {
      Matrix m = {};
      m.g = c.grads[o]; m.w = c.params[o];
      m.m = c.momentum ? c.momentum + at[o] : nullptr;
      m.at = at[o];
      m.rows = static_cast<int>(c.rows[o]); m.cols = static_cast<int>(c.cols[o]);
      m.rate = static_cast<float>(c.lr * (c.adjust == HASTE_MUON_MATCH_RMS ? 0.2 * std::sqrt(static_cast<double>(std::max(c.rows[o], c.cols[o])))
                                                                            : std::sqrt(std::max(1.0, static_cast<double>(c.rows[o]) / static_cast<double>(c.cols[o])))));
      return m;
    };
    if (!few.empty()) {
      std::vector<Matrix> all;
      for (int64_t o : few) {
        Matrix m = matrix(o);
        m.nparts = gram_parts(c.rows[o], c.cols[o]);
        m.parts = reinterpret_cast<double*>(take(few_bytes(c.rows[o], c.cols[o])));
        all.push_back(m);
      }
      if (int rc = launch_few_rows(all, c, k, st)) return rc;
    }
    if (some.empty()) continue;
    const int64_t n = static_cast<int64_t>(some.size());
    auto* done = reinterpret_cast<unsigned long long*>(take(8 * (n + 1)));
    k.drawn = done + n;
    auto* parts = reinterpret_cast<double*>(take(8 * NORM_PARTS * n));
    int64_t elements = 0;
    for (int64_t o : some) elements += c.rows[o] * c.cols[o];
    // blocks of squares: 8 for every SM, shared by size
    const int64_t each = std::max<int64_t>(NORM_ELEMENTS, elements / (static_cast<int64_t>(sm_count()) * 8));
    std::vector<Matrix> all;
    std::vector<newton_schulz::Batch> batches;
    for (size_t i = 0; i < some.size();) {
      const Sizes s = sizes_of(c.rows[some[i]], c.cols[some[i]]);
      size_t end = i;
      while (end < some.size() && sizes_of(c.rows[some[end]], c.cols[some[end]]).p == s.p && sizes_of(c.rows[some[end]], c.cols[some[end]]).q == s.q) ++end;
      newton_schulz::Batch h;
      h.p = s.p; h.q = s.q; h.count = static_cast<int64_t>(end - i);
      for (uint16_t** x : {&h.hi[0], &h.hi[1], &h.lo}) *x = reinterpret_cast<uint16_t*>(take(2 * h.count * s.x()));
      h.B = reinterpret_cast<uint16_t*>(take(2 * h.count * s.a()));
      for (size_t j = i; j < end; ++j) {
        const int64_t o = some[j], x = static_cast<int64_t>(j - i) * s.x(), size = c.rows[o] * c.cols[o];
        Matrix m = matrix(o);
        m.hi = h.hi[0] + x; m.lo = h.lo + x;
        m.ld = static_cast<int>(s.q);
        m.nparts = static_cast<int>(std::min<int64_t>(NORM_PARTS, (size + each - 1) / each));
        m.parts = parts + NORM_PARTS * all.size();
        m.done = done + all.size();
        all.push_back(m);
      }
      batches.push_back(h);
      i = end;
    }
    const bool narrow = newton_schulz::take_narrow(batches);
    int rc = for_each_table<false>(all, [&](const auto& t, auto size, unsigned parts, unsigned tiles) -> int {
      constexpr int N = decltype(size)::value;
      if (gb) muon_squares_kernel<__nv_bfloat16, N><<<parts, NORM_THREADS, 0, st>>>(t, k);
      else muon_squares_kernel<float, N><<<parts, NORM_THREADS, 0, st>>>(t, k);
      if (int e = check_launch("muon_squares_kernel")) return e;
      return gb ? launch_behind(muon_start_kernel<__nv_bfloat16, N>, tiles, 256, st, t, k) : launch_behind(muon_start_kernel<float, N>, tiles, 256, st, t, k);
    });
    if (rc) return rc;
    rc = newton_schulz::run(batches, narrow, done, k.drawn, c.steps, c.a, c.b, c.c, st);
    if (rc) return rc;
    size_t at_matrix = 0;
    for (const newton_schulz::Batch& h : batches) {
      const unsigned long long need = newton_schulz::count_of(h, narrow, c.steps);
      for (int64_t j = 0; j < h.count; ++j, ++at_matrix) {
        all[at_matrix].need = need;
        if (c.steps & 1) all[at_matrix].hi = h.hi[1] + j * h.p * h.q;          // X is in the other buffer
      }
    }
    rc = for_each_table<false>(all, [&](const auto& t, auto size, unsigned, unsigned tiles) -> int {
      constexpr int N = decltype(size)::value;
      if (!c.update) return launch_behind(muon_finish_kernel<__nv_bfloat16, false, N>, tiles, 256, st, t, k);
      return c.p_type == HASTE_BF16 ? launch_behind(muon_finish_kernel<__nv_bfloat16, true, N>, tiles, 256, st, t, k) : launch_behind(muon_finish_kernel<float, true, N>, tiles, 256, st, t, k);
    });
    if (rc) return rc;
  }
  return HASTE_OK;
}

}  // namespace haste
