// Muon: the update of a matrix is its momentum, made orthogonal by Newton-Schulz steps.
//
//   m = mu m + (1 - mu) g,   u = mu m + (1 - mu) g (Nesterov) or m,   X = u / max(|u|, eps)        (X has the smaller side as rows)
//   steps times:  A = X X^T,  X <- a X + (b A + c A A) X
//   w = w (1 - lr weight_decay) - lr rate X
//
// For a list of matrices at once: one launch for the norms, one that writes the momentum and X, three products a step over all matrices (those of one shape
// are a batch, shapes are problems of one launch, gemm_sm100.cuh), one that updates the weights.
//
// Rounding.  The products take fp16: X times 2^8 (its entries are at most 1, later 1.3 or so; the factor keeps small ones out of the subnormals), A and
// B = b A + c A A.  The term a X, by which small singular values grow 3.4 times a step, takes X as a sum of two fp16 values, hi + lo 2^-11: 22 bits.  Without lo
// an update of low rank with noise is off by 1.3e-2 after five steps (2-norm of the difference over that of the result), with it by 1e-3, a Gaussian one by 1.4e-3;
// with bf16 in place of fp16 1e-1 and 1e-2.  A and A A are symmetric: tiles on and below the diagonal are computed, the others are their mirror.
#include "gemm_sm100.cuh"

#include <algorithm>
#include <cmath>
#include <vector>

namespace haste {
namespace {

using gemm::Problem;
using gemm::Tile;
using gemm::Work;

constexpr float X_SCALE = 256.f;
constexpr float LO_SCALE = 2048.f;

// ---------------------------------------------------------------- products
template <class S>
__device__ __forceinline__ void put_symmetric(const Problem& p, const Tile& t, int row0, int col, bool diagonal, const uint32_t (&packed)[16], S& st, int lane) {
  const bool inside = row0 < p.M && col < p.N;
  uint32_t box = st.get();
  gemm::box_row(box, lane, packed);
  st.put(&p.out[0], box, col, row0, t.batch, inside);
  if (!diagonal) {
    box = st.get();
    gemm::box_column(box, lane, packed);
    st.put(&p.out[0], box, row0, col, t.batch, inside);
  }
}

// A = scale0 X X^T
struct Gram {
  static constexpr bool A_MN = false, B_MN = false, F16 = true, PAIRED_B = false;
  static constexpr int INPUTS = 0;
  template <class W, class I, class S>
  static __device__ __forceinline__ void chunk(const W& w, const Problem& p, const Tile& t, int row0, int col, bool diagonal, uint32_t tmem, I&, S& st, int lane) {
    uint32_t v[32], packed[16];
    sm100::tmem_ld32(tmem, v);
    sm100::tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) packed[i] = gemm::pack_f16(__uint_as_float(v[2 * i]) * w.scale0, __uint_as_float(v[2 * i + 1]) * w.scale0);
    put_symmetric(p, t, row0, col, diagonal, packed, st, lane);
  }
};

// B = scale0 A + scale1 A A^T; in[0] = A
struct Polynomial {
  static constexpr bool A_MN = false, B_MN = false, F16 = true, PAIRED_B = false;
  static constexpr int INPUTS = 1;
  template <class W, class I, class S>
  static __device__ __forceinline__ void chunk(const W& w, const Problem& p, const Tile& t, int row0, int col, bool diagonal, uint32_t tmem, I& in, S& st, int lane) {
    uint32_t v[32], packed[16];
    sm100::tmem_ld32(tmem, v);
    in.get(0, packed);
    in.release();
    sm100::tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 a = gemm::unpack_f16(packed[i]);
      packed[i] = gemm::pack_f16(fmaf(w.scale1, __uint_as_float(v[2 * i]), w.scale0 * a.x), fmaf(w.scale1, __uint_as_float(v[2 * i + 1]), w.scale0 * a.y));
    }
    put_symmetric(p, t, row0, col, diagonal, packed, st, lane);
  }
};

// X' = scale0 X + B X; in[0] = X's upper part, in[1] its lower one, if it has one (LOWER: 2 and 1); out[0] and out[1] those of X', the lower one with LOWER = 2 alone.  (in[1] and
// out[1] are one place: a tile reads what it writes.)
template <int LOWER>
struct Apply {
  static constexpr bool A_MN = false, B_MN = true, F16 = true, PAIRED_B = false;
  static constexpr int INPUTS = LOWER ? 2 : 1;
  template <class W, class I, class S>
  static __device__ __forceinline__ void chunk(const W& w, const Problem& p, const Tile& t, int row0, int col, bool, uint32_t tmem, I& in, S& st, int lane) {
    const bool inside = row0 < p.M && col < p.N;
    uint32_t v[32], hi[16], lo[16];
    sm100::tmem_ld32(tmem, v);
    in.get(0, hi);
    if (LOWER) in.get(1, lo);
    in.release();
    sm100::tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float2 h = gemm::unpack_f16(hi[i]);
      if (LOWER) {
        const float2 l = gemm::unpack_f16(lo[i]);
        h.x = fmaf(l.x, 1.f / LO_SCALE, h.x);
        h.y = fmaf(l.y, 1.f / LO_SCALE, h.y);
      }
      const float x = fmaf(w.scale0, h.x, __uint_as_float(v[2 * i])), y = fmaf(w.scale0, h.y, __uint_as_float(v[2 * i + 1]));
      hi[i] = gemm::pack_f16(x, y);
      if (LOWER == 2) {
        const float2 r = gemm::unpack_f16(hi[i]);
        lo[i] = gemm::pack_f16((x - r.x) * LO_SCALE, (y - r.y) * LO_SCALE);
      }
    }
    uint32_t box = st.get();
    gemm::box_row(box, lane, hi);
    st.put(&p.out[0], box, col, row0, t.batch, inside);
    if (LOWER == 2) {
      box = st.get();
      gemm::box_row(box, lane, lo);
      st.put(&p.out[1], box, col, row0, t.batch, inside);
    }
  }
};

// ---------------------------------------------------------------- elementwise
constexpr int NORM_THREADS = 256;
constexpr int NORM_PARTS = 256;                    // of a matrix, at most
constexpr int NORM_ELEMENTS = 8192;                // of a block, at least
constexpr int TABLE = 192;                         // matrices of one launch
constexpr int SIDE = 64;                           // of an elementwise tile

struct Matrix {
  const void* g;
  void* w;                         // the parameter, or the result
  float* m;                        // momentum, NULL without
  uint16_t *hi, *lo;               // X's parts, rows of ld elements
  double* parts;                   // sums of squares, by block
  int64_t at;                      // place in the momentum, for the random bits
  int rows, cols, ld;
  int nparts, first_part, first_tile;
  float rate;
};
struct Matrices {
  Matrix a[TABLE];
  int n, parts, tiles;
};
struct Coefficients {
  float mu, one_mu, decay, eps;
  int nesterov, sr;
  uint32_t seed, step, stream;
};

__device__ __forceinline__ void load4(const __nv_bfloat16* p, int n, bool vec, float (&v)[4]) {
  if (vec) {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    const float2 a = gemm::unpack_bf16(q.x), b = gemm::unpack_bf16(q.y);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? __bfloat162float(p[i]) : 0.f;
  }
}
__device__ __forceinline__ void load4(const float* p, int n, bool vec, float (&v)[4]) {
  if (vec) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : 0.f;
  }
}
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

// Sum of squares of each matrix's direction, in 64 bits (a square of fp32 has a place there whatever its size), in an order that the sizes alone decide
template <class G>
__global__ void __launch_bounds__(NORM_THREADS) muon_squares_kernel(const __grid_constant__ Matrices t, const Coefficients c) {
  __shared__ double warps[NORM_THREADS / 32];
  int k = 0;
  while (k + 1 < t.n && static_cast<int>(blockIdx.x) >= t.a[k + 1].first_part) ++k;
  const Matrix& a = t.a[k];
  const int part = blockIdx.x - a.first_part;
  const int64_t n = static_cast<int64_t>(a.rows) * a.cols, groups = (n + 3) / 4;
  const G* g = static_cast<const G*>(a.g);
  double sum = 0;
  for (int64_t i = static_cast<int64_t>(part) * NORM_THREADS + threadIdx.x; i < groups; i += static_cast<int64_t>(a.nparts) * NORM_THREADS) {
    const int have = static_cast<int>(imin64(4, n - 4 * i));
    float gv[4], mv[4] = {0, 0, 0, 0};
    load4(g + 4 * i, have, vec4(g + 4 * i, have), gv);
    if (a.m != nullptr) load4(a.m + 4 * i, have, have == 4, mv);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const double u = direction(c, gv[x], mv[x], a.m != nullptr);
      if (x < have) sum += u * u;
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

// 1 / max(norm, eps), NaN or 0 where the norm is NaN or inf; by all threads of a block
__device__ __forceinline__ float inverse_norm(const Matrix& a, float eps, double* shared) {
  double s = threadIdx.x < a.nparts ? a.parts[threadIdx.x] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0;
  for (int i = 0; i < NORM_THREADS / 32; ++i) s += shared[i];
  const double norm = sqrt(s);
  return static_cast<float>(1.0 / (norm < eps ? static_cast<double>(eps) : norm));
}
__device__ __forceinline__ bool usable(float inverse) { return inverse > 0.f && inverse < INFINITY; }

__device__ __forceinline__ const Matrix& tile_of(const Matrices& t, int block, int& row0, int& col0) {
  int k = 0;
  while (k + 1 < t.n && block >= t.a[k + 1].first_tile) ++k;
  const Matrix& a = t.a[k];
  const int across = (a.cols + SIDE - 1) / SIDE, i = block - a.first_tile;
  row0 = i / across * SIDE;
  col0 = (i - i / across * across) * SIDE;
  return a;
}

// Momentum and X.  A matrix whose norm is not finite keeps its momentum.
template <class G>
__global__ void __launch_bounds__(256) muon_start_kernel(const __grid_constant__ Matrices t, const Coefficients c) {
  __shared__ double sums[NORM_THREADS / 32];
  __shared__ float turned[SIDE][SIDE + 1];
  int row0, col0;
  const Matrix& a = tile_of(t, blockIdx.x, row0, col0);
  sm100::grid_dependency_wait();
  const float inv = inverse_norm(a, c.eps, sums), factor = inv * X_SCALE;
  const bool tall = a.rows > a.cols, momentum = a.m != nullptr, write = momentum && usable(inv);
  const int cg = (threadIdx.x & 15) * 4, col = col0 + cg, have = min(4, a.cols - col);
#pragma unroll
  for (int k = 0; k < SIDE / 16; ++k) {
    const int r = threadIdx.x / 16 + 16 * k, row = row0 + r;
    if (row < a.rows && have > 0) {
      const int64_t i = static_cast<int64_t>(row) * a.cols + col;
      const G* g = static_cast<const G*>(a.g) + i;
      float gv[4], mv[4] = {0, 0, 0, 0}, x[4];
      load4(g, have, vec4(g, have), gv);
      if (momentum) load4(a.m + i, have, vec4(a.m + i, have), mv);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = direction(c, gv[e], mv[e], momentum) * factor;
      if (write) store4(a.m + i, have, vec4(a.m + i, have), mv);
      if (tall) {
#pragma unroll
        for (int e = 0; e < 4; ++e) turned[cg + e][r] = x[e];
      } else {
        const uint32_t h0 = gemm::pack_f16(x[0], x[1]), h1 = gemm::pack_f16(x[2], x[3]);
        const float2 a0 = gemm::unpack_f16(h0), a1 = gemm::unpack_f16(h1);
        const int64_t to = static_cast<int64_t>(row) * a.ld + col;
        *reinterpret_cast<uint2*>(a.hi + to) = make_uint2(h0, h1);           // rows are padded to a multiple of 8
        *reinterpret_cast<uint2*>(a.lo + to) = make_uint2(gemm::pack_f16((x[0] - a0.x) * LO_SCALE, (x[1] - a0.y) * LO_SCALE), gemm::pack_f16((x[2] - a1.x) * LO_SCALE, (x[3] - a1.y) * LO_SCALE));
      }
    }
  }
  if (!tall) return;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < SIDE / 16; ++k) {
    const int r = threadIdx.x / 16 + 16 * k, row = col0 + r, at = row0 + cg;       // of X
    if (row < a.cols && at < a.rows) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = at + e < a.rows ? turned[r][cg + e] : 0.f;
      const uint32_t h0 = gemm::pack_f16(x[0], x[1]), h1 = gemm::pack_f16(x[2], x[3]);
      const float2 a0 = gemm::unpack_f16(h0), a1 = gemm::unpack_f16(h1);
      const int64_t to = static_cast<int64_t>(row) * a.ld + at;
      *reinterpret_cast<uint2*>(a.hi + to) = make_uint2(h0, h1);
      *reinterpret_cast<uint2*>(a.lo + to) = make_uint2(gemm::pack_f16((x[0] - a0.x) * LO_SCALE, (x[1] - a0.y) * LO_SCALE), gemm::pack_f16((x[2] - a1.x) * LO_SCALE, (x[3] - a1.y) * LO_SCALE));
    }
  }
}

// Philox4x32 with 7 rounds, key (seed, step), counter (i, i >> 32, stream, 2): one word for each of the elements 4 i .. 4 i + 3
__device__ __forceinline__ uint4 random_words(const Coefficients& c, int64_t i) {
  uint32_t c0 = static_cast<uint32_t>(i), c1 = static_cast<uint32_t>(static_cast<uint64_t>(i) >> 32), c2 = c.stream, c3 = 2, k0 = c.seed, k1 = c.step;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint32_t hi0 = __umulhi(0xD2511F53u, c0), lo0 = 0xD2511F53u * c0, hi1 = __umulhi(0xCD9E8D57u, c2), lo1 = 0xCD9E8D57u * c2;
    c0 = hi1 ^ c1 ^ k0; c2 = hi0 ^ c3 ^ k1; c1 = lo1; c3 = lo0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}
__device__ __forceinline__ uint32_t word(const uint4& r, int i) { return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w; }

__device__ __forceinline__ void store_weights(float* p, int have, const float (&v)[4], const Coefficients&, int64_t) { store4(p, have, vec4(p, have), v); }
__device__ __forceinline__ void store_weights(__nv_bfloat16* p, int have, const float (&v)[4], const Coefficients& c, int64_t i) {
  uint32_t b[4];
  if (c.sr) {
    const uint4 first = random_words(c, i >> 2);
    const int skip = static_cast<int>(i & 3);
    const uint4 second = skip ? random_words(c, (i >> 2) + 1) : first;
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = sr_bf16_bits(v[e], word(e + skip < 4 ? first : second, (e + skip) & 3) & 0xFFFFu);
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

// UPDATE: the weights; else X itself, in bf16
template <class W, bool UPDATE>
__global__ void __launch_bounds__(256) muon_finish_kernel(const __grid_constant__ Matrices t, const Coefficients c) {
  __shared__ double sums[NORM_THREADS / 32];
  __shared__ float turned[SIDE][SIDE + 1];
  int row0, col0;
  const Matrix& a = tile_of(t, blockIdx.x, row0, col0);
  sm100::grid_dependency_wait();
  if (UPDATE && !usable(inverse_norm(a, c.eps, sums))) return;       // the same for all of the block
  const bool tall = a.rows > a.cols;
  const int cg = (threadIdx.x & 15) * 4;
  if (tall) {
#pragma unroll
    for (int k = 0; k < SIDE / 16; ++k) {
      const int r = threadIdx.x / 16 + 16 * k, row = col0 + r, at = row0 + cg;
      if (row < a.cols && at < a.rows) {
        const uint2 q = *reinterpret_cast<const uint2*>(a.hi + static_cast<int64_t>(row) * a.ld + at);
        const float2 x0 = gemm::unpack_f16(q.x), x1 = gemm::unpack_f16(q.y);
        turned[cg][r] = x0.x; turned[cg + 1][r] = x0.y; turned[cg + 2][r] = x1.x; turned[cg + 3][r] = x1.y;
      }
    }
    __syncthreads();
  }
  const int col = col0 + cg, have = min(4, a.cols - col);
  if (have <= 0) return;
#pragma unroll
  for (int k = 0; k < SIDE / 16; ++k) {
    const int r = threadIdx.x / 16 + 16 * k, row = row0 + r;
    if (row >= a.rows) break;
    float x[4];
    if (tall) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = turned[r][cg + e];
    } else {
      const uint2 q = *reinterpret_cast<const uint2*>(a.hi + static_cast<int64_t>(row) * a.ld + col);
      const float2 x0 = gemm::unpack_f16(q.x), x1 = gemm::unpack_f16(q.y);
      x[0] = x0.x; x[1] = x0.y; x[2] = x1.x; x[3] = x1.y;
    }
    const int64_t i = static_cast<int64_t>(row) * a.cols + col;
    W* to = static_cast<W*>(a.w) + i;
    float v[4];
    if (UPDATE) {
      load4(to, have, vec4(to, have), v);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(-a.rate * (1.f / X_SCALE), x[e], v[e] * c.decay);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = x[e] * (1.f / X_SCALE);
    }
    store_weights(to, have, v, c, a.at + i);
  }
}

// ---------------------------------------------------------------- host side
constexpr int64_t ROUND_BYTES = int64_t(1) << 30;      // of scratch memory, unless one matrix needs more: a round of so much keeps the GPU busy for a millisecond

int64_t up8(int64_t n) { return (n + 7) & ~int64_t(7); }
int64_t up256(int64_t n) { return (n + 255) & ~int64_t(255); }
struct Sizes {
  int64_t p, q;                    // rows and columns of X
  int64_t x() const { return p * up8(q); }
  int64_t a() const { return p * up8(p); }
  int64_t bytes() const { return 2 * (3 * up256(x()) + 2 * up256(a())) + 8 * NORM_PARTS; }
};
Sizes sizes_of(int64_t rows, int64_t cols) { return {std::min(rows, cols), std::max(rows, cols)}; }

// The matrices with a gradient, by shape, cut into rounds
struct Plan {
  std::vector<int64_t> order;
  std::vector<size_t> rounds;      // where in `order` each begins, and the end
  int64_t bytes = 0;
};
Plan plan_of(const void* const* grads, const int64_t* rows, const int64_t* cols, int64_t count) {
  Plan p;
  for (int64_t i = 0; i < count; ++i)
    if ((grads == nullptr || grads[i] != nullptr) && rows[i] > 0 && cols[i] > 0) p.order.push_back(i);
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
    p.bytes = std::max(p.bytes, used);
  }
  p.rounds.push_back(p.order.size());
  return p;
}

// A batch of matrices of one shape in the scratch memory
struct Shape {
  int64_t p, q, batch;
  uint16_t *hi[2], *lo, *A, *B;
};

// One product of all shapes.  phase 0: A = X X^T, 1: B = b A + c A A, 2: X
template <class Policy, int TN, int P>
int run_product(const std::vector<Shape>& shapes, size_t from, size_t to, int phase, int cur, double scale0, double scale1, cudaStream_t st) {
  static thread_local Work<P> w;
  w.problems = static_cast<int>(to - from);
  w.scale0 = static_cast<float>(scale0); w.scale1 = static_cast<float>(scale1);
  for (size_t i = from; i < to; ++i) {
    const Shape& h = shapes[i];
    Problem& p = w.p[i - from];
    const gemm::Operand x = {h.hi[cur], up8(h.q), h.p * up8(h.q)}, low = {h.lo, x.ld, x.batch_stride}, next = {h.hi[cur ^ 1], x.ld, x.batch_stride}, A = {h.A, up8(h.p), h.p * up8(h.p)},
                        B = {h.B, A.ld, A.batch_stride};
    const int64_t k = phase == 0 ? h.q : h.p, N = phase == 2 ? h.q : h.p;
    p.partial = nullptr;
    p.M = static_cast<int>(h.p); p.N = static_cast<int>(N);
    p.symmetric = phase < 2;
    p.batch = static_cast<int>(h.batch);
    p.splits = 1;
    p.steps0 = p.steps = static_cast<int>(gemm::steps_of(k));
    int rc = gemm::map_a<Policy, TN>(&p.a[0], phase == 0 ? x : phase == 1 ? A : B, h.p, k, h.batch);
    rc = rc ? rc : gemm::map_b<Policy, TN>(&p.b[0], phase == 1 ? A : x, N, k, h.batch);
    rc = rc ? rc : gemm::map_result<Policy>(&p.out[0], phase == 0 ? A : phase == 1 ? B : next, h.p, N, h.batch);
    if (phase == 1) rc = rc ? rc : gemm::map_result<Policy>(&p.in[0], A, h.p, N, h.batch);
    if (phase == 2) {
      rc = rc ? rc : gemm::map_result<Policy>(&p.in[0], x, h.p, N, h.batch);
      rc = rc ? rc : gemm::map_result<Policy>(&p.in[1], low, h.p, N, h.batch);
      p.out[1] = p.in[1];
    }
    if (rc) return rc;
  }
  return gemm::launch<Policy, TN>(w, true, st);
}

// What X is rounded to after the last but two steps is amplified by two steps at most (12 times), which leaves 2^-12 of its values where the products' own roundings
// are: its lower part is kept up to there.
constexpr int STEPS_WITHOUT_LOWER = 2;

template <int P>
int run_steps(const std::vector<Shape>& shapes, size_t from, size_t to, int steps, double a, double b, double c, cudaStream_t st) {
  double wide[2] = {}, narrow[2] = {};               // of the symmetric products and of the last one
  int64_t tiles[2][2] = {}, work[2] = {};
  for (size_t i = from; i < to; ++i)
    for (int k = 0; k < 2; ++k) {
      const Shape& h = shapes[i];
      const int64_t N = k ? h.q : h.p;
      for (int n = 0; n < 2; ++n) tiles[k][n] += h.batch * gemm::tiles_for(h.p, N, n ? 64 : 256);
      work[k] += h.batch * gemm::tiles_for(h.p, N, 256) * gemm::steps_of(h.p);
    }
  for (int k = 0; k < 2; ++k) {
    const int64_t per = (work[k] + tiles[k][0] - 1) / tiles[k][0];          // steps of a tile, on average
    wide[k] = gemm::cost_of(k ? tiles[k][0] : (tiles[k][0] + 1) / 2, per, false);
    narrow[k] = gemm::cost_of(k ? tiles[k][1] : (tiles[k][1] + 1) / 2, per, true);
  }
  const bool n0 = narrow[0] < wide[0], n1 = narrow[1] < wide[1];
  for (int s = 0; s < steps; ++s) {
    const int cur = s & 1;
    const double gram = 1.0 / (X_SCALE * X_SCALE);
    int rc = n0 ? run_product<Gram, 64, P>(shapes, from, to, 0, cur, gram, 0, st) : run_product<Gram, 256, P>(shapes, from, to, 0, cur, gram, 0, st);
    if (rc) return rc;
    rc = n0 ? run_product<Polynomial, 64, P>(shapes, from, to, 1, cur, b, c, st) : run_product<Polynomial, 256, P>(shapes, from, to, 1, cur, b, c, st);
    if (rc) return rc;
    const int left = steps - STEPS_WITHOUT_LOWER - s;
    if (left > 1) rc = n1 ? run_product<Apply<2>, 64, P>(shapes, from, to, 2, cur, a, 0, st) : run_product<Apply<2>, 256, P>(shapes, from, to, 2, cur, a, 0, st);
    else if (left == 1 || s == 0) rc = n1 ? run_product<Apply<1>, 64, P>(shapes, from, to, 2, cur, a, 0, st) : run_product<Apply<1>, 256, P>(shapes, from, to, 2, cur, a, 0, st);
    else rc = n1 ? run_product<Apply<0>, 64, P>(shapes, from, to, 2, cur, a, 0, st) : run_product<Apply<0>, 256, P>(shapes, from, to, 2, cur, a, 0, st);
    if (rc) return rc;
  }
  return HASTE_OK;
}

template <class F>
int for_each_table(const std::vector<Matrix>& all, F&& f) {
  for (size_t i = 0; i < all.size(); i += TABLE) {
    static thread_local Matrices t;
    t.n = static_cast<int>(std::min<size_t>(TABLE, all.size() - i));
    int64_t parts = 0, tiles = 0;
    for (int k = 0; k < t.n; ++k) {
      t.a[k] = all[i + k];
      t.a[k].first_part = static_cast<int>(parts);
      t.a[k].first_tile = static_cast<int>(tiles);
      parts += t.a[k].nparts;
      tiles += static_cast<int64_t>((t.a[k].rows + SIDE - 1) / SIDE) * ((t.a[k].cols + SIDE - 1) / SIDE);
      if (tiles > 0x7FFFFFFF) return fail(HASTE_ERR_TOO_LARGE, "matrices of too many elements for one call");
    }
    t.parts = static_cast<int>(parts); t.tiles = static_cast<int>(tiles);
    if (int rc = f(t)) return rc;
  }
  return HASTE_OK;
}

constexpr int FEW_SHAPES = 4, MANY_SHAPES = 24;

}  // namespace

int64_t muon_scratch(const int64_t* rows, const int64_t* cols, int64_t count) { return plan_of(nullptr, rows, cols, count).bytes; }

int launch_muon(const MuonCall& c, cudaStream_t st) {
  if (int rc = report_pending_status(c.who)) return rc;
  const Plan plan = plan_of(c.grads, c.rows, c.cols, c.count);
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
    std::vector<Matrix> all;
    std::vector<Shape> shapes;
    for (size_t i = plan.rounds[r]; i < plan.rounds[r + 1];) {
      const Sizes s = sizes_of(c.rows[plan.order[i]], c.cols[plan.order[i]]);
      size_t end = i;
      while (end < plan.rounds[r + 1] && sizes_of(c.rows[plan.order[end]], c.cols[plan.order[end]]).p == s.p && sizes_of(c.rows[plan.order[end]], c.cols[plan.order[end]]).q == s.q) ++end;
      Shape h;
      h.p = s.p; h.q = s.q; h.batch = static_cast<int64_t>(end - i);
      for (uint16_t** x : {&h.hi[0], &h.hi[1], &h.lo}) *x = reinterpret_cast<uint16_t*>(take(2 * h.batch * s.x()));
      for (uint16_t** x : {&h.A, &h.B}) *x = reinterpret_cast<uint16_t*>(take(2 * h.batch * s.a()));
      for (size_t j = i; j < end; ++j) {
        const int64_t o = plan.order[j], x = static_cast<int64_t>(j - i) * s.x();
        Matrix m = {};
        m.g = c.grads[o]; m.w = c.params[o];
        m.m = c.momentum ? c.momentum + at[o] : nullptr;
        m.hi = h.hi[0] + x; m.lo = h.lo + x;
        m.at = at[o];
        m.rows = static_cast<int>(c.rows[o]); m.cols = static_cast<int>(c.cols[o]); m.ld = static_cast<int>(up8(s.q));
        m.nparts = static_cast<int>(std::min<int64_t>(NORM_PARTS, (s.p * s.q + NORM_ELEMENTS - 1) / NORM_ELEMENTS));
        m.parts = reinterpret_cast<double*>(take(8 * NORM_PARTS));
        m.rate = static_cast<float>(c.lr * (c.adjust == HASTE_MUON_MATCH_RMS ? 0.2 * std::sqrt(static_cast<double>(s.q))
                                                                              : std::sqrt(std::max(1.0, static_cast<double>(c.rows[o]) / static_cast<double>(c.cols[o])))));
        all.push_back(m);
      }
      shapes.push_back(h);
      i = end;
    }
    const bool gb = c.g_type == HASTE_BF16;
    int rc = for_each_table(all, [&](const Matrices& t) -> int {
      if (gb) muon_squares_kernel<__nv_bfloat16><<<t.parts, NORM_THREADS, 0, st>>>(t, k);
      else muon_squares_kernel<float><<<t.parts, NORM_THREADS, 0, st>>>(t, k);
      if (int e = check_launch("muon_squares_kernel")) return e;
      return gb ? launch_behind(muon_start_kernel<__nv_bfloat16>, t.tiles, 256, st, t, k) : launch_behind(muon_start_kernel<float>, t.tiles, 256, st, t, k);
    });
    if (rc) return rc;
    for (size_t from = 0; from < shapes.size(); from += MANY_SHAPES) {
      const size_t to = std::min(shapes.size(), from + MANY_SHAPES);
      rc = to - from <= FEW_SHAPES ? run_steps<FEW_SHAPES>(shapes, from, to, c.steps, c.a, c.b, c.c, st) : run_steps<MANY_SHAPES>(shapes, from, to, c.steps, c.a, c.b, c.c, st);
      if (rc) return rc;
    }
    if (c.steps & 1)                   // X is in the other buffer
      for (Matrix& m : all)
        for (const Shape& h : shapes)
          if (m.hi >= h.hi[0] && m.hi < h.hi[0] + h.batch * h.p * up8(h.q)) { m.hi = h.hi[1] + (m.hi - h.hi[0]); break; }
    rc = for_each_table(all, [&](const Matrices& t) -> int {
      if (!c.update) return launch_behind(muon_finish_kernel<__nv_bfloat16, false>, t.tiles, 256, st, t, k);
      return c.p_type == HASTE_BF16 ? launch_behind(muon_finish_kernel<__nv_bfloat16, true>, t.tiles, 256, st, t, k) : launch_behind(muon_finish_kernel<float, true>, t.tiles, 256, st, t, k);
    });
    if (rc) return rc;
  }
  return HASTE_OK;
}

}  // namespace haste
