// Muon: the update of a matrix is its momentum, made orthogonal by Newton-Schulz steps.
//
//   m = mu m + (1 - mu) g,   u = mu m + (1 - mu) g (Nesterov) or m,   X = u / max(|u|, eps)        (X has the smaller side as rows)
//   steps times:  A = X X^T,  B = a I + b A + c A A,  X <- B X
//   w = w (1 - lr weight_decay) - lr rate X
//
// For a list of matrices at once: one launch for the norms, one that writes the momentum and X (rows and columns padded with zeros to multiples of 64, which stay
// zeros: so matrices of nearly one size are one batch), one for all steps (newton_schulz.cuh), one that updates the weights.
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
    const int64_t need = sizes_of(rows[p.order[k]], cols[p.order[k]]).bytes();
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
template <int N, class F>
int with_table(const std::vector<Matrix>& all, size_t from, F&& f) {
  static thread_local Matrices<N> t;
  t.n = static_cast<int>(std::min<size_t>(N, all.size() - from));
  int64_t parts = 0, tiles = 0;
  for (int k = 0; k < t.n; ++k) {
    const Matrix& a = t.a[k] = all[from + k];
    t.first_part[k] = static_cast<int>(parts);
    t.first_tile[k] = static_cast<int>(tiles);
    parts += a.nparts;
    tiles += static_cast<int64_t>((a.rows + SIDE - 1) / SIDE) * ((a.cols + SIDE - 1) / SIDE);
    if (tiles > 0x7FFFFFFF) return fail(HASTE_ERR_TOO_LARGE, "matrices of too many elements for one call");
  }
  t.first_part[t.n] = static_cast<int>(parts); t.first_tile[t.n] = static_cast<int>(tiles);
  // the elementwise launches' blocks share the tiles: as many as run at once
  return f(t, std::integral_constant<int, N>(), static_cast<unsigned>(parts), static_cast<unsigned>(imin64(tiles, static_cast<int64_t>(sm_count()) * 6)));
}
template <class F>
int for_each_table(const std::vector<Matrix>& all, F&& f) {
  for (size_t i = 0; i < all.size(); i += MANY) {
    const int rc = all.size() - i <= FEW ? with_table<FEW>(all, i, f) : with_table<MANY>(all, i, f);
    if (rc) return rc;
  }
  return HASTE_OK;
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
    std::vector<int64_t> some;         // those with a gradient
    for (size_t i = plan.rounds[r]; i < plan.rounds[r + 1]; ++i)
      if (c.grads[plan.order[i]] != nullptr) some.push_back(plan.order[i]);
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
        Matrix m = {};
        m.g = c.grads[o]; m.w = c.params[o];
        m.m = c.momentum ? c.momentum + at[o] : nullptr;
        m.hi = h.hi[0] + x; m.lo = h.lo + x;
        m.at = at[o];
        m.rows = static_cast<int>(c.rows[o]); m.cols = static_cast<int>(c.cols[o]); m.ld = static_cast<int>(s.q);
        m.nparts = static_cast<int>(std::min<int64_t>(NORM_PARTS, (size + each - 1) / each));
        m.parts = parts + NORM_PARTS * all.size();
        m.done = done + all.size();
        m.rate = static_cast<float>(c.lr * (c.adjust == HASTE_MUON_MATCH_RMS ? 0.2 * std::sqrt(static_cast<double>(std::max(c.rows[o], c.cols[o])))
                                                                              : std::sqrt(std::max(1.0, static_cast<double>(c.rows[o]) / static_cast<double>(c.cols[o])))));
        all.push_back(m);
      }
      batches.push_back(h);
      i = end;
    }
    const bool gb = c.g_type == HASTE_BF16, narrow = newton_schulz::take_narrow(batches);
    int rc = for_each_table(all, [&](const auto& t, auto size, unsigned parts, unsigned tiles) -> int {
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
    rc = for_each_table(all, [&](const auto& t, auto size, unsigned, unsigned tiles) -> int {
      constexpr int N = decltype(size)::value;
      if (!c.update) return launch_behind(muon_finish_kernel<__nv_bfloat16, false, N>, tiles, 256, st, t, k);
      return c.p_type == HASTE_BF16 ? launch_behind(muon_finish_kernel<__nv_bfloat16, true, N>, tiles, 256, st, t, k) : launch_behind(muon_finish_kernel<float, true, N>, tiles, 256, st, t, k);
    });
    if (rc) return rc;
  }
  return HASTE_OK;
}

}  // namespace haste
