// One AdamW step over many tensors at once, the 2-norm of their gradients, and moments held in 8 bits.
//
//   g  = grad * scale,  scale = grad_scale * min(1, max_norm / (norm + 1e-6))
//   m' = b1 m + (1 - b1) g          v' = b2 v + (1 - b2) g^2
//   w' = w (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Arithmetic is fp32.  bf16 weights are rounded stochastically (there is no fp32 copy of them: rounded to nearest, a step below half a
// bf16 ulp would be lost every time) or to nearest.
//
// The moments of all tensors lie in one buffer, each tensor's at a multiple of ADAM_BLOCK elements, so that a block of the buffer
// belongs to one tensor: a warp takes a block, a lane 8 consecutive elements of it.
//
// Moments in 8 bits: a block of 256 values has one fp32 scale, max |value| / 1.875, and a code per value: 3 bits of mantissa and as
// many octaves as the remaining codes give, without subnormals, so that encoding is integer arithmetic on the fp32 pattern.
//   first moment   sign, 127 codes: 1.125 * 2^-15 .. 1.875, smaller values become 0
//   second moment  255 codes: 1.125 * 2^-31 .. 1.875 (the same range for its root), smaller ones become the lowest code: a zero would
//                  leave eps alone in the denominator
// Both are rounded stochastically.  With b2 = 0.999 a second moment moves by a thousandth of itself a step, an eighth to a
// sixteenth is between codes: rounded to nearest it stays where it is until one gradient exceeds it thirtyfold (simulated over 6000 steps
// with gradients that change their scale: the spread of log sqrt(v) against fp32 is 0.6 to 1.2 with nearest, 0.12 to 0.16 so).
//
// Random bits: Philox4x32 with 7 rounds (the fewest that its authors found to pass their statistical tests), key (seed, step), counter
// (i, i >> 32, stream, 1) for elements 4i .. 4i+3 of the buffer, a word each: bits 0-15 round the weight, 16-23 the first moment,
// 24-31 the second.
#include "common.cuh"

#include <math.h>
#include "launchers.h"

namespace haste {

constexpr int ADAM_BLOCK = 256;        // elements that share a scale; the place of a tensor in the moments is a multiple of it
constexpr int ADAM_THREADS = 256;
constexpr float CODE_TOP = 1.875f;
constexpr float CODE_TINY = 0x1p-120f; // a block whose largest value is below holds zeros (1.875 / it is finite)

// The tensors of one launch, as a kernel parameter.  first[i]: first block of tensor i among the launch's blocks.
template <int N>
struct TensorTable {
  void* p[N];              // the norm's kernel has no weights: type of g[i] (HASTE_BF16 / HASTE_F32) as a number
  const void* g[N];
  int64_t n[N];
  int32_t first[N + 1];
  int32_t count;
};

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
}
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// 8 elements of a lane; left: how many exist (the others read as 0).  vec: all 8 are there and the address is on 16 bytes.
template <class T>
__device__ __forceinline__ void load_lane(const T* p, bool vec, int64_t left, float (&v)[8]) {
  if (vec) { load8(p, v); return; }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < left ? load1(p + i) : 0.f;
}

// The fp32 patterns in u become weights: stored as they are, or their upper halves.
__device__ __forceinline__ void store_lane(float* p, bool vec, int64_t left, const uint32_t (&u)[8]) {
  if (vec) {
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    *reinterpret_cast<uint4*>(p + 4) = make_uint4(u[4], u[5], u[6], u[7]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) if (i < left) p[i] = __uint_as_float(u[i]);
}
__device__ __forceinline__ void store_lane(__nv_bfloat16* p, bool vec, int64_t left, const uint32_t (&u)[8]) {
  if (vec) {
    *reinterpret_cast<uint4*>(p) = make_uint4(__byte_perm(u[0], u[1], 0x7632), __byte_perm(u[2], u[3], 0x7632), __byte_perm(u[4], u[5], 0x7632),
                                              __byte_perm(u[6], u[7], 0x7632));
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) if (i < left) p[i] = __ushort_as_bfloat16(static_cast<uint16_t>(u[i] >> 16));
}

__device__ __forceinline__ uint4 philox4x32_7(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint32_t hi0 = __umulhi(0xD2511F53u, c0), lo0 = 0xD2511F53u * c0;
    const uint32_t hi1 = __umulhi(0xCD9E8D57u, c2), lo1 = 0xCD9E8D57u * c2;
    c0 = hi1 ^ c1 ^ k0;
    c2 = hi0 ^ c3 ^ k1;
    c1 = lo1;
    c3 = lo0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Root and quotient of the update to a few units in the last place: the update is a small part of the weight, whose own rounding hides
// them, and neither enters the moments.  (133 M bf16 weights with 32-bit moments: 663 us with correctly rounded ones, 460 so; 56 M with
// 8-bit moments 386 and 244.)
__device__ __forceinline__ float root_of(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// ---------------------------------------------------------------- 8-bit codes
// Code c of a value y in (0, 1.875]: the upper 12 bits of its fp32 pattern less BASE.
constexpr uint32_t M_BASE = 0x380u, V_BASE = 0x300u;      // pattern of 1.875 is 0x3FF.....: 0x3FF - 127 and 0x3FF - 255

__device__ __forceinline__ float decode_m(uint32_t c) {
  const uint32_t mag = c & 0x7Fu;
  const float y = mag ? __uint_as_float((mag + M_BASE) << 20) : 0.f;
  return c & 0x80u ? -y : y;
}
__device__ __forceinline__ float decode_v(uint32_t c) { return c ? __uint_as_float((c + V_BASE) << 20) : 0.f; }

// r8: 8 random bits.  Half of the last random place is added, so that the sum's truncation is right on average.
__device__ __forceinline__ uint32_t encode_m(float y, uint32_t r8) {
  const uint32_t bits = __float_as_uint(y), u = (bits & 0x7FFFFFFFu) + (r8 << 12) + 0x800u;
  const int c = min(max(static_cast<int>(u >> 20) - static_cast<int>(M_BASE), 0), 127);
  return c ? (static_cast<uint32_t>(c) | ((bits >> 24) & 0x80u)) : 0u;
}
__device__ __forceinline__ uint32_t encode_v(float y, uint32_t r8) {
  const uint32_t u = __float_as_uint(y) + (r8 << 12) + 0x800u;
  const int c = min(max(static_cast<int>(u >> 20) - static_cast<int>(V_BASE), 1), 255);
  return y > 0.f ? static_cast<uint32_t>(c) : 0u;
}
// Scale of a block and what its values are multiplied with.  Where a value is inf or NaN the scale is NaN, and the block reads as NaN.
__device__ __forceinline__ float block_scale(float top, float& inv) {
  if (!(top < __uint_as_float(0x7F800000u))) { inv = 0.f; return __uint_as_float(0x7FC00000u); }
  const bool fine = top >= CODE_TINY;
  inv = fine ? CODE_TOP / top : 0.f;
  return fine ? top * (1.0f / CODE_TOP) : 0.f;
}
// Largest pattern over a warp; patterns of non-negative floats compare as the floats do, inf and NaN above all.
__device__ __forceinline__ float warp_top(const float (&x)[8]) {
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  return __uint_as_float(__reduce_max_sync(0xffffffffu, top));
}

struct AdamArgs {
  float b1, c1, b2, c2;        // c = 1 - b
  float decay, rate, root, eps; // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  float grad_scale, max_norm;
  const float* norm;           // of the gradients times grad_scale; NULL: not clipped
  uint32_t seed, step, stream;
  int sr;
};

// BITS: 32, 8.  m, v: fp32 moments or codes; ms, vs: scales; all of the launch's first block.  block0: index of that block in the
// whole buffer, for the random counters.
template <class P, class G, int BITS, int N>
__global__ void __launch_bounds__(ADAM_THREADS) adamw_kernel(const __grid_constant__ TensorTable<N> tab, void* __restrict__ m_all, float* __restrict__ ms,
                                                             void* __restrict__ v_all, float* __restrict__ vs, int64_t block0, const __grid_constant__ AdamArgs a) {
  float scale = a.grad_scale;
  if (a.norm != nullptr) {
    const float norm = *a.norm;
    if (!(norm < __uint_as_float(0x7F800000u))) return;       // a gradient is not finite: nothing is changed
    scale *= fminf(1.f, a.max_norm / (norm + 1e-6f));
  }
  const int lane = threadIdx.x & 31, blocks = tab.first[tab.count];
  const int warps = gridDim.x * (ADAM_THREADS / 32);
  int t = 0;
  for (int b = blockIdx.x * (ADAM_THREADS / 32) + (threadIdx.x >> 5); b < blocks; b += warps) {
    while (tab.first[t + 1] <= b) ++t;
    if (tab.g[t] == nullptr) continue;
    const int64_t at = static_cast<int64_t>(b - tab.first[t]) * ADAM_BLOCK + lane * 8, left = tab.n[t] - at;
    P* p = static_cast<P*>(tab.p[t]) + at;
    const G* gp = static_cast<const G*>(tab.g[t]) + at;
    const bool vec_p = left >= 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0, vec_g = left >= 8 && (reinterpret_cast<uintptr_t>(gp) & 15) == 0;
    const int64_t e = static_cast<int64_t>(b) * ADAM_BLOCK + lane * 8;
    float w[8], g[8], m[8], v[8];
    load_lane(p, vec_p, left, w);
    load_lane(gp, vec_g, left, g);
    if (BITS == 32) {
      load8(static_cast<const float*>(m_all) + e, m);
      load8(static_cast<const float*>(v_all) + e, v);
    } else {
      const uint2 mc = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(m_all) + e), vc = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(v_all) + e);
      const float sm = ms[b], sv = vs[b];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        m[i] = decode_m(((i < 4 ? mc.x : mc.y) >> (8 * (i & 3))) & 0xFFu) * sm;
        v[i] = decode_v(((i < 4 ? vc.x : vc.y) >> (8 * (i & 3))) & 0xFFu) * sv;
      }
    }
    if (left < 8) {                       // what pads a tensor's last block counts for nothing, whatever the buffer held
#pragma unroll
      for (int i = 0; i < 8; ++i) if (i >= left) m[i] = v[i] = 0.f;
    }
    uint32_t rnd[8], out[8];
    const bool sr = sizeof(P) == 2 && a.sr;
    if (BITS == 8 || sr) {
      const uint64_t i = (static_cast<uint64_t>(block0 + b) * ADAM_BLOCK + lane * 8) / 4;      // even
      const uint4 r0 = philox4x32_7(static_cast<uint32_t>(i), static_cast<uint32_t>(i >> 32), a.stream, 1u, a.seed, a.step);
      const uint4 r1 = philox4x32_7(static_cast<uint32_t>(i) + 1u, static_cast<uint32_t>(i >> 32), a.stream, 1u, a.seed, a.step);
      rnd[0] = r0.x; rnd[1] = r0.y; rnd[2] = r0.z; rnd[3] = r0.w; rnd[4] = r1.x; rnd[5] = r1.y; rnd[6] = r1.z; rnd[7] = r1.w;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float gi = g[i] * scale;
      m[i] = fmaf(a.b1, m[i], a.c1 * gi);
      v[i] = fmaf(a.b2, v[i], a.c2 * gi * gi);
      const float wn = fmaf(-a.rate, __fdividef(m[i], fmaf(root_of(v[i]), a.root, a.eps)), w[i] * a.decay);
      if (sizeof(P) == 4) out[i] = __float_as_uint(wn);
      // (a NaN's pattern is 0x7FFFFFFF: with bits added it would read as -0)
      else out[i] = sr ? __float_as_uint(wn) + (wn == wn ? rnd[i] & 0xFFFFu : 0u) : static_cast<uint32_t>(rn_bf16_bits(wn)) << 16;
    }
    store_lane(p, vec_p, left, out);
    if (BITS == 32) {
      float* mp = static_cast<float*>(m_all) + e;
      float* vp = static_cast<float*>(v_all) + e;
      *reinterpret_cast<float4*>(mp) = make_float4(m[0], m[1], m[2], m[3]);
      *reinterpret_cast<float4*>(mp + 4) = make_float4(m[4], m[5], m[6], m[7]);
      *reinterpret_cast<float4*>(vp) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(vp + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      float im, iv;
      const float sm = block_scale(warp_top(m), im), sv = block_scale(warp_top(v), iv);
      uint32_t mc[2] = {0u, 0u}, vc[2] = {0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        mc[i >> 2] |= encode_m(m[i] * im, (rnd[i] >> 16) & 0xFFu) << (8 * (i & 3));
        vc[i >> 2] |= encode_v(v[i] * iv, rnd[i] >> 24) << (8 * (i & 3));
      }
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(m_all) + e) = make_uint2(mc[0], mc[1]);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(v_all) + e) = make_uint2(vc[0], vc[1]);
      if (lane == 0) { ms[b] = sm; vs[b] = sv; }
    }
  }
}

// ---------------------------------------------------------------- 2-norm of the gradients
// Sums of squares of the launch's blocks, one per thread block, into partial[part0 + blockIdx.x].
template <int N>
__global__ void __launch_bounds__(ADAM_THREADS) grad_squares_kernel(const __grid_constant__ TensorTable<N> tab, float* __restrict__ partial, int part0) {
  __shared__ float sums[ADAM_THREADS / 32];
  const int lane = threadIdx.x & 31, blocks = tab.first[tab.count];
  const int warps = gridDim.x * (ADAM_THREADS / 32);
  float s = 0.f;
  int t = 0;
  for (int b = blockIdx.x * (ADAM_THREADS / 32) + (threadIdx.x >> 5); b < blocks; b += warps) {
    while (tab.first[t + 1] <= b) ++t;
    const int64_t at = static_cast<int64_t>(b - tab.first[t]) * ADAM_BLOCK + lane * 8, left = tab.n[t] - at;
    float g[8];
    const char* gp = static_cast<const char*>(tab.g[t]);
    if (reinterpret_cast<uintptr_t>(tab.p[t]) == HASTE_BF16) {
      gp += 2 * at;
      load_lane(reinterpret_cast<const __nv_bfloat16*>(gp), left >= 8 && (reinterpret_cast<uintptr_t>(gp) & 15) == 0, left, g);
    } else {
      gp += 4 * at;
      load_lane(reinterpret_cast<const float*>(gp), left >= 8 && (reinterpret_cast<uintptr_t>(gp) & 15) == 0, left, g);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(g[i], g[i], s);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < ADAM_THREADS / 32; ++i) s += sums[i];
    partial[part0 + blockIdx.x] = s;
  }
}

// sqrt of the sum of the partial sums (in 64 bits: one block adds a few hundred), in an order that depends on their number alone.
__global__ void __launch_bounds__(ADAM_THREADS) grad_norm_finish_kernel(const float* __restrict__ partial, int parts, float grad_scale, float* __restrict__ norm) {
  __shared__ double sums[ADAM_THREADS / 32];
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += ADAM_THREADS) s += partial[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < ADAM_THREADS / 32; ++i) s += sums[i];
    *norm = static_cast<float>(sqrt(s) * fabsf(grad_scale));
  }
}

// ---------------------------------------------------------------- values -> codes (nearest), codes -> values
template <bool SIGNED>
__global__ void __launch_bounds__(ADAM_THREADS) quantize_kernel(const float* __restrict__ x, uint8_t* __restrict__ codes, float* __restrict__ scales, int64_t blocks) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (ADAM_THREADS / 32);
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * (ADAM_THREADS / 32) + (threadIdx.x >> 5); b < blocks; b += warps) {
    const int64_t e = b * ADAM_BLOCK + lane * 8;
    float v[8], inv;
    load8(x + e, v);
    const float s = block_scale(warp_top(v), inv);
    uint32_t c[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i >> 2] |= (SIGNED ? encode_m(v[i] * inv, 127u) : encode_v(v[i] * inv, 127u)) << (8 * (i & 3));
    *reinterpret_cast<uint2*>(codes + e) = make_uint2(c[0], c[1]);
    if (lane == 0) scales[b] = s;
  }
}

template <class O, bool SIGNED>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales, O* __restrict__ out, int64_t n8) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n8; i += stride) {
    const uint2 c = *reinterpret_cast<const uint2*>(codes + i * 8);
    const float s = scales[i / (ADAM_BLOCK / 8)];
    uint32_t u[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t code = ((k < 4 ? c.x : c.y) >> (8 * (k & 3))) & 0xFFu;
      const float x = (SIGNED ? decode_m(code) : decode_v(code)) * s;
      u[k] = sizeof(O) == 4 ? __float_as_uint(x) : static_cast<uint32_t>(rn_bf16_bits(x)) << 16;
    }
    store_lane(out + i * 8, true, 8, u);
  }
}

// ================================================================ launchers
static int adam_grid(int64_t blocks) {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t want = (blocks + ADAM_THREADS / 32 - 1) / (ADAM_THREADS / 32);
  return static_cast<int>(want < sms * 4 ? want : sms * 4);
}

constexpr int TABLE_SMALL = 112, TABLE_LARGE = 1024;      // 3.2 KB and 28.7 KB of kernel parameters (32,764 bytes at most)
constexpr int64_t MAX_BLOCKS = (int64_t(1) << 31) - 1 - 65536;

// Calls f(table, first block of the part) for consecutive parts of the tensors; a tensor with more than 2^31 blocks is refused before.
template <class F>
static int for_each_table(void* const* params, const int32_t* types, const void* const* grads, const int64_t* sizes, int64_t count, F&& f) {
  int64_t i = 0, block0 = 0;
  while (i < count) {
    TensorTable<TABLE_LARGE> tab;
    int k = 0;
    int64_t blocks = 0;
    tab.first[0] = 0;
    for (; i < count && k < TABLE_LARGE; ++i) {
      const int64_t nb = (sizes[i] + ADAM_BLOCK - 1) / ADAM_BLOCK;
      if (blocks + nb > MAX_BLOCKS) break;
      tab.p[k] = params ? params[i] : reinterpret_cast<void*>(static_cast<intptr_t>(types[i]));
      tab.g[k] = grads[i];
      tab.n[k] = sizes[i];
      blocks += nb;
      tab.first[++k] = static_cast<int32_t>(blocks);
    }
    tab.count = k;
    if (blocks > 0)
      if (int rc = f(tab, block0, blocks)) return rc;
    block0 += blocks;
  }
  return HASTE_OK;
}

static TensorTable<TABLE_SMALL> small_table(const TensorTable<TABLE_LARGE>& tab) {
  TensorTable<TABLE_SMALL> s;
  s.count = tab.count;
  s.first[0] = 0;
  for (int i = 0; i < tab.count; ++i) { s.p[i] = tab.p[i]; s.g[i] = tab.g[i]; s.n[i] = tab.n[i]; s.first[i + 1] = tab.first[i + 1]; }
  return s;
}

template <class P, class G, int BITS>
static int adamw_typed(const AdamWCall& c, const AdamArgs& a, cudaStream_t st) {
  return for_each_table(c.params, nullptr, c.grads, c.sizes, c.count, [&](const TensorTable<TABLE_LARGE>& tab, int64_t block0, int64_t blocks) {
    char* m = static_cast<char*>(c.exp_avg) + block0 * ADAM_BLOCK * (BITS / 8);
    char* v = static_cast<char*>(c.exp_avg_sq) + block0 * ADAM_BLOCK * (BITS / 8);
    float* ms = BITS == 8 ? c.avg_scale + block0 : nullptr;
    float* vs = BITS == 8 ? c.sq_scale + block0 : nullptr;
    const int grid = adam_grid(blocks);
    if (tab.count <= TABLE_SMALL) adamw_kernel<P, G, BITS, TABLE_SMALL><<<grid, ADAM_THREADS, 0, st>>>(small_table(tab), m, ms, v, vs, block0, a);
    else adamw_kernel<P, G, BITS, TABLE_LARGE><<<grid, ADAM_THREADS, 0, st>>>(tab, m, ms, v, vs, block0, a);
    return check_launch("adamw_kernel");
  });
}

int launch_adamw(const AdamWCall& c, cudaStream_t st) {
  AdamArgs a;
  a.b1 = static_cast<float>(c.beta1); a.c1 = static_cast<float>(1.0 - c.beta1);
  a.b2 = static_cast<float>(c.beta2); a.c2 = static_cast<float>(1.0 - c.beta2);
  a.decay = static_cast<float>(1.0 - c.lr * c.weight_decay);
  a.rate = static_cast<float>(c.lr / (1.0 - pow(c.beta1, static_cast<double>(c.step))));
  a.root = static_cast<float>(1.0 / sqrt(1.0 - pow(c.beta2, static_cast<double>(c.step))));
  a.eps = static_cast<float>(c.eps);
  a.grad_scale = c.grad_scale; a.max_norm = c.max_norm; a.norm = c.norm;
  a.seed = static_cast<uint32_t>(c.seed); a.step = static_cast<uint32_t>(c.step); a.stream = c.stream;
  a.sr = (c.flags & HASTE_F_SR) ? 1 : 0;
  using B = __nv_bfloat16;
  using F = float;
  const bool pb = c.p_type == HASTE_BF16, gb = c.g_type == HASTE_BF16;
  if (c.bits == 8) {
    if (pb) return gb ? adamw_typed<B, B, 8>(c, a, st) : adamw_typed<B, F, 8>(c, a, st);
    return gb ? adamw_typed<F, B, 8>(c, a, st) : adamw_typed<F, F, 8>(c, a, st);
  }
  if (pb) return gb ? adamw_typed<B, B, 32>(c, a, st) : adamw_typed<B, F, 32>(c, a, st);
  return gb ? adamw_typed<F, B, 32>(c, a, st) : adamw_typed<F, F, 32>(c, a, st);
}

int launch_grad_norm(const void* const* grads, const int32_t* types, const int64_t* sizes, int64_t count, float grad_scale, float* partial, float* norm,
                     cudaStream_t st) {
  const int64_t tables = count / TABLE_LARGE + 1;           // or one more for every 2^31 blocks, whose grids are as large as they get
  const int64_t cap = HASTE_GRAD_NORM_PARTIALS / 2 / tables;
  int parts = 0;
  const int rc = for_each_table(nullptr, types, grads, sizes, count, [&](const TensorTable<TABLE_LARGE>& tab, int64_t, int64_t blocks) {
    const int grid = static_cast<int>(imin64(adam_grid(blocks), cap));
    if (grid < 1 || parts + grid > HASTE_GRAD_NORM_PARTIALS) return fail(HASTE_ERR_TOO_LARGE, "haste_grad_norm: too many tensors for one call");
    if (tab.count <= TABLE_SMALL) grad_squares_kernel<TABLE_SMALL><<<grid, ADAM_THREADS, 0, st>>>(small_table(tab), partial, parts);
    else grad_squares_kernel<TABLE_LARGE><<<grid, ADAM_THREADS, 0, st>>>(tab, partial, parts);
    parts += grid;
    return check_launch("grad_squares_kernel");
  });
  if (rc != HASTE_OK) return rc;
  grad_norm_finish_kernel<<<1, ADAM_THREADS, 0, st>>>(partial, parts, grad_scale, norm);
  return check_launch("grad_norm_finish_kernel");
}

int launch_quantize(const float* x, uint8_t* codes, float* scales, int64_t n, int is_signed, cudaStream_t st) {
  if (n == 0) return HASTE_OK;
  const int grid = adam_grid(n / ADAM_BLOCK);
  if (is_signed) quantize_kernel<true><<<grid, ADAM_THREADS, 0, st>>>(x, codes, scales, n / ADAM_BLOCK);
  else quantize_kernel<false><<<grid, ADAM_THREADS, 0, st>>>(x, codes, scales, n / ADAM_BLOCK);
  return check_launch("quantize_kernel");
}

int launch_dequantize(const uint8_t* codes, const float* scales, void* out, int64_t n, int is_signed, int type, cudaStream_t st) {
  if (n == 0) return HASTE_OK;
  const int64_t n8 = n / 8, want = (n8 + 255) / 256;
  const unsigned grid = static_cast<unsigned>(want < 148 * 16 ? want : 148 * 16);
  if (type == HASTE_BF16) {
    if (is_signed) dequantize_kernel<__nv_bfloat16, true><<<grid, 256, 0, st>>>(codes, scales, (__nv_bfloat16*)out, n8);
    else dequantize_kernel<__nv_bfloat16, false><<<grid, 256, 0, st>>>(codes, scales, (__nv_bfloat16*)out, n8);
  } else if (is_signed) dequantize_kernel<float, true><<<grid, 256, 0, st>>>(codes, scales, (float*)out, n8);
  else dequantize_kernel<float, false><<<grid, 256, 0, st>>>(codes, scales, (float*)out, n8);
  return check_launch("dequantize_kernel");
}

}  // namespace haste
