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

#include <cooperative_groups.h>
#include <math.h>
#include "launchers.h"

namespace haste {

constexpr int ADAM_BLOCK = 256;        // elements that share a scale; the place of a tensor in the moments is a multiple of it
constexpr int ADAM_THREADS = 256, ADAM_WARPS = ADAM_THREADS / 32;
constexpr int AHEAD = 4;               // blocks of gradients that a warp of the norm has on their way
constexpr float CODE_TOP = 1.875f;
constexpr float CODE_TINY = 0x1p-120f; // a block whose largest value is below holds zeros (1.875 / it is finite)

// 0.7, 7 and 28.7 KB of kernel parameters (32,764 bytes at most); the larger ones cost the host more (launching a step
// over 150 tensors 9.6 us with the largest, 7.5 with the middle one).
constexpr int TABLE_SMALL = 24, TABLE_MIDDLE = 256, TABLE_LARGE = 1024;

// The tensors of one launch, as a kernel parameter.  first[i]: first block of tensor i among the launch's blocks.
template <int N>
struct TensorTable {
  void* p[N];              // the norm's kernel has no weights: type of g[i] (HASTE_BF16 / HASTE_F32) as a number
  const void* g[N];
  int64_t n[N];
  int32_t first[N + 1];
  int32_t count;
};

// The tensor that block b of the launch belongs to.
template <int N>
__device__ __forceinline__ int tensor_of(const TensorTable<N>& tab, int b) {
  int lo = 0, hi = tab.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (tab.first[mid + 1] <= b) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// 8 elements of a lane as they lie in memory.  Loading does not look at them: a load that is unpacked in its own branch is waited for
// there, before the next one starts (56 M gradients: norm 35 us so unpacked).
template <class T>
struct Lane8 {
  static constexpr int WORDS = static_cast<int>(sizeof(T)) / 2;       // of 16 bytes
  uint4 q[WORDS];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) q[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  // the first `left` elements one by one, then zeros
  __device__ __forceinline__ void load_part(const T* p, int64_t left) {
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 4) u[i] = i < left ? __float_as_uint(p[i]) : 0u;
      else u[i] = i < left ? reinterpret_cast<const uint16_t*>(p)[i] : 0u;
    }
    if constexpr (sizeof(T) == 4) { q[0] = make_uint4(u[0], u[1], u[2], u[3]); q[1] = make_uint4(u[4], u[5], u[6], u[7]); }
    else q[0] = make_uint4(u[0] | (u[1] << 16), u[2] | (u[3] << 16), u[4] | (u[5] << 16), u[6] | (u[7] << 16));
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) q[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void get(float2 (&v)[4]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v[2 * i] = make_float2(__uint_as_float(q[i].x), __uint_as_float(q[i].y));
        v[2 * i + 1] = make_float2(__uint_as_float(q[i].z), __uint_as_float(q[i].w));
      }
    } else {
      const uint32_t u[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xFFFF0000u));
    }
  }
};
__device__ __forceinline__ bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

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

// (products of 64 bits: 2 % of the 8-bit step faster than high and low halves apart)
__device__ __forceinline__ uint4 philox4x32_7(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(0xD2511F53u) * c0, p1 = static_cast<uint64_t>(0xCD9E8D57u) * c2;
    const uint32_t hi0 = static_cast<uint32_t>(p0 >> 32), lo0 = static_cast<uint32_t>(p0), hi1 = static_cast<uint32_t>(p1 >> 32), lo1 = static_cast<uint32_t>(p1);
    c0 = hi1 ^ c1 ^ k0;
    c2 = hi0 ^ c3 ^ k1;
    c1 = lo1;
    c3 = lo0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Two fp32 numbers as one operand: one instruction for both.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)),
      "l"(reinterpret_cast<const uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Root and quotient of the update to 2^-23 each (133 M bf16 weights with 32-bit moments: 663 us with correctly rounded ones, 460 so; 56 M with 8-bit
// moments 386 and 244).  They are 2 to 3 ulp of the step, not of the weight, and a weight that starts at zero has them in its first values.
// The moments in 32 bits do not depend on them; the scale by which values of 8 bits are encoded does, so that one within an ulp of a
// boundary may take the next code.
// Second moments in 32 bits may be subnormal: with an eps that is smaller still, a root of 0 would leave eps alone under the first moment.  In
// 8 bits they count as 0 here (one instruction instead of several), as a block of less than CODE_TINY holds zeros anyway.
template <int BITS>
__device__ __forceinline__ float root_of(float v) {
  float r;
  if constexpr (BITS == 32) asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  else asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float inverse_of(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// ---------------------------------------------------------------- 8-bit codes
// The code of a value y in (0, 1.875] is the upper 12 bits of its fp32 pattern less a base: 0x300 for the second moment (0x3FF, the pattern
// of 1.875, becomes 255), 0x380 for the first one's magnitude (0x3FF becomes 127).  Integer instructions that are not products have half the
// rate of the others and were what bounded the 8-bit step, so codes are taken apart two at a time, as bf16 (whose pattern is the upper
// half of fp32's), and put together by byte selection: 56 M bf16 weights 244 us one at a time, 154 so (143 with what came after).
// Copying the next block ahead of time, which takes 15 registers, changed nothing (151 to 155 us).
constexpr uint32_t M_LEAST = 0x38000000u, V_LEAST = 0x30100000u;      // patterns of the first moment's (unused) code 0 and the second's code 1

__device__ __forceinline__ float2 halves(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)); }
// u holds two bf16; those not above `least` become 0
__device__ __forceinline__ uint32_t drop_least(uint32_t u, uint32_t least) {
  const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&u), l = *reinterpret_cast<const __nv_bfloat162*>(&least);
  const __nv_bfloat162 r = __hmul2(v, __hgt2(v, l));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Codes 0, 1 (PAIR 0) or 2, 3 (PAIR 1) of a word
template <int PAIR>
__device__ __forceinline__ float2 decode_m(uint32_t codes) {
  const uint32_t c = __byte_perm(codes, 0u, PAIR ? 0x4342 : 0x4140);                  // one code in each half
  const uint32_t mag = drop_least((c & 0x007F007Fu) * 16u + 0x38003800u, 0x38003800u);
  return halves(mag | ((c * 256u) & 0x80008000u));
}
template <int PAIR>
__device__ __forceinline__ float2 decode_v(uint32_t codes) {
  return halves(drop_least(__byte_perm(codes, 0u, PAIR ? 0x4342 : 0x4140) * 16u + 0x30003000u, 0x30003000u));
}
template <bool SIGNED>
__device__ __forceinline__ void decode8(uint2 codes, float2 (&x)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t c = i < 2 ? codes.x : codes.y;
    if (SIGNED) x[i] = i & 1 ? decode_m<1>(c) : decode_m<0>(c); else x[i] = i & 1 ? decode_v<1>(c) : decode_v<0>(c);
  }
}
template <bool SIGNED>
__device__ __forceinline__ void decode8(uint2 codes, float scale, float2 (&x)[4]) {
  decode8<SIGNED>(codes, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = mul2(x[i], both(scale));
}

// The highest bytes of four words
__device__ __forceinline__ uint32_t high_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}
// With 8 random bits r, code = floor((pattern + r 2^12 + 2^11) / 2^20) - base: half of the last random place is added, so that cutting is right
// on average.  All of it is taken times 16, which puts the code into the highest byte; nothing rounds up beyond the highest code, the
// pattern of which is 0xFF7FF short of the next one's.  rnd: bits 16-23 for the first, 24-31 for the second moment.
__device__ __forceinline__ uint32_t encode4_m(const float (&x)[4], float inv, const uint32_t (&rnd)[4]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = max(__float_as_uint(fabsf(x[i]) * inv), M_LEAST) * 16u + __byte_perm(rnd[i], 0x00008000u, 0x6254);
  const uint32_t mag = high_bytes(u[0], u[1], u[2], u[3]) & 0x7F7F7F7Fu;              // (the base leaves 0x80 in each)
  const uint32_t sign = high_bytes(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  return mag | ((mag + 0x7F7F7F7Fu) & sign & 0x80808080u);                            // no sign for code 0
}
__device__ __forceinline__ uint32_t encode4_v(const float (&x)[4], float inv, const uint32_t (&rnd)[4]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)      // less 1, which makes 0 the largest number: it stays 0 where the other small ones become code 1
    u[i] = __viaddmax_u32(__float_as_uint(x[i] * inv), 0xFFFFFFFFu, V_LEAST - 1u) * 16u + __byte_perm(rnd[i], 0x00008010u, 0x6354);
  return high_bytes(u[0], u[1], u[2], u[3]);
}
template <bool SIGNED>
__device__ __forceinline__ uint2 encode8(const float (&x)[8], float inv, const uint32_t (&rnd)[8]) {
  const float a[4] = {x[0], x[1], x[2], x[3]}, b[4] = {x[4], x[5], x[6], x[7]};
  const uint32_t r[4] = {rnd[0], rnd[1], rnd[2], rnd[3]}, q[4] = {rnd[4], rnd[5], rnd[6], rnd[7]};
  return SIGNED ? make_uint2(encode4_m(a, inv, r), encode4_m(b, inv, q)) : make_uint2(encode4_v(a, inv, r), encode4_v(b, inv, q));
}
// Scale of a block and what its values are multiplied with.  Where a value is inf or NaN the scale is NaN, and the block reads as NaN.
__device__ __forceinline__ float block_scale(float top, float& inv) {
  if (!(top < __uint_as_float(0x7F800000u))) { inv = 0.f; return __uint_as_float(0x7FC00000u); }
  const bool fine = top >= CODE_TINY;
  inv = fine ? inverse_of(top * 0.0625f) * (CODE_TOP * 0.0625f) : 0.f;      // (2^-4: the inverse of the largest numbers would be subnormal)
  return fine ? top * (1.0f / CODE_TOP) : 0.f;
}
// Largest magnitude over a warp; NaN where one is NaN.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float warp_top(const float (&x)[8]) {
  const float t = max3_abs(max3_abs(x[0], x[1], x[2]), max3_abs(x[3], x[4], x[5]), max3_abs(x[6], x[7], x[7]));
  float r;
  asm volatile("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(t));
  return r;
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
  const int lane = threadIdx.x & 31;
  const int blocks = tab.first[tab.count], step = gridDim.x * ADAM_WARPS;
  int b = blockIdx.x * ADAM_WARPS + (threadIdx.x >> 5), t = tensor_of(tab, b);
  for (; b < blocks; b += step) {
    while (tab.first[t + 1] <= b) ++t;
    if (tab.g[t] == nullptr) continue;
    const int64_t at = static_cast<int64_t>(b - tab.first[t]) * ADAM_BLOCK, size = tab.n[t], left = size - at - lane * 8;
    P* p = static_cast<P*>(tab.p[t]) + at + lane * 8;
    const G* gp = static_cast<const G*>(tab.g[t]) + at + lane * 8;
    const bool whole = size - at >= ADAM_BLOCK && on16(tab.p[t]) && on16(tab.g[t]);        // for the warp: 16 bytes at a time
    const int64_t e = static_cast<int64_t>(b) * ADAM_BLOCK + lane * 8;
    Lane8<P> wl;
    Lane8<G> gl;
    Lane8<float> ml, vl;
    uint2 mc, vc;
    float sm, sv;
    if (BITS == 32) {
      ml.load(static_cast<const float*>(m_all) + e);
      vl.load(static_cast<const float*>(v_all) + e);
    } else {
      mc = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(m_all) + e);
      vc = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(v_all) + e);
      sm = ms[b];
      sv = vs[b];
    }
    if (whole) { wl.load(p); gl.load(gp); } else { wl.load_part(p, left); gl.load_part(gp, left); }
    uint32_t rnd[8], out[8];
    const bool sr = sizeof(P) == 2 && a.sr;
    if (BITS == 8 || sr) {                // while the loads are on their way
      const uint64_t i = (static_cast<uint64_t>(block0 + b) * ADAM_BLOCK + lane * 8) / 4;      // even
      const uint4 r0 = philox4x32_7(static_cast<uint32_t>(i), static_cast<uint32_t>(i >> 32), a.stream, 1u, a.seed, a.step);
      const uint4 r1 = philox4x32_7(static_cast<uint32_t>(i) + 1u, static_cast<uint32_t>(i >> 32), a.stream, 1u, a.seed, a.step);
      rnd[0] = r0.x; rnd[1] = r0.y; rnd[2] = r0.z; rnd[3] = r0.w; rnd[4] = r1.x; rnd[5] = r1.y; rnd[6] = r1.z; rnd[7] = r1.w;
    }
    float2 w[4], g[4], m2[4], v2[4];
    if (BITS == 32) { ml.get(m2); vl.get(v2); } else { decode8<true>(mc, m2); decode8<false>(vc, v2); }
    if (left < 8) {                       // what pads a tensor's last block counts for nothing, whatever the buffer held
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (2 * i >= left) m2[i].x = v2[i].x = 0.f;
        if (2 * i + 1 >= left) m2[i].y = v2[i].y = 0.f;
      }
    }
    wl.get(w);
    gl.get(g);
    // (a block's scale goes into the factors that follow)
    const float b1 = BITS == 8 ? a.b1 * sm : a.b1, b2 = BITS == 8 ? a.b2 * sv : a.b2;
    float m[8], v[8];
    float2 bad = both(0.f);               // becomes NaN with any weight that is inf or NaN
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 gi = mul2(g[i], both(scale));
      const float2 mi = fma2(both(b1), m2[i], mul2(both(a.c1), gi)), vi = fma2(both(b2), v2[i], mul2(mul2(both(a.c2), gi), gi));
      const float2 den = fma2(make_float2(root_of<BITS>(vi.x), root_of<BITS>(vi.y)), both(a.root), both(a.eps));
      const float2 q = mul2(mi, make_float2(inverse_of(den.x), inverse_of(den.y)));
      const float2 wn = fma2(both(-a.rate), q, mul2(w[i], both(a.decay)));
      m[2 * i] = mi.x; m[2 * i + 1] = mi.y; v[2 * i] = vi.x; v[2 * i + 1] = vi.y;
      out[2 * i] = __float_as_uint(wn.x); out[2 * i + 1] = __float_as_uint(wn.y);
      if (sizeof(P) == 2) bad = fma2(wn, both(0.f), bad);
    }
    if (sizeof(P) == 2) {
      if (sr) {
        // a NaN is 0x7FFFFFFF here: it must not run over into the sign
        if (bad.x + bad.y != 0.f) {
#pragma unroll
          for (int i = 0; i < 8; ++i) rnd[i] = (out[i] & 0x7FFFFFFFu) > 0x7F800000u ? rnd[i] & 0xFFFF0000u : rnd[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] += rnd[i] & 0xFFFFu;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = static_cast<uint32_t>(rn_bf16_bits(__uint_as_float(out[i]))) << 16;
      }
    }
    store_lane(p, whole, left, out);
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
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(m_all) + e) = encode8<true>(m, im, rnd);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(v_all) + e) = encode8<false>(v, iv, rnd);
      if (lane == 0) { ms[b] = sm; vs[b] = sv; }
    }
  }
}

// ---------------------------------------------------------------- 2-norm of the gradients
// Sum of squares of blocks lo .. hi - 1 of the launch over THREADS threads, in thread 0.  A warp has the loads of 4 blocks on their way at
// once (56 M bf16 gradients 35 us with one, 27 with 4), and stays with a tensor, which it looks up once (30 us where each block was looked up).
// Sums of 64 squares go on in 64 bits: an fp32 sum over a tensor of billions would lose what comes after a large value.
template <int THREADS, int N>
__device__ __forceinline__ float sum_of_squares(const TensorTable<N>& tab, int lo, int hi) {
  constexpr int WARPS = THREADS / 32;
  __shared__ float sums[WARPS];
  const int lane = threadIdx.x & 31;
  float2 acc[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) acc[k] = both(0.f);
  double total = 0.0;
  int t = tensor_of(tab, lo) - 1, next = 0, first = 0, type = HASTE_BF16, turns = 0;
  int64_t size = 0;
  const char* from = nullptr;
  for (int b0 = lo + (threadIdx.x >> 5); b0 < hi; b0 += WARPS * AHEAD) {
    Lane8<float> g[AHEAD];            // fp32, or in the first word bf16
    bool half[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int b = b0 + k * WARPS;
      g[k].clear();
      half[k] = false;
      if (b >= hi) continue;
      if (b >= next) {
        do ++t; while (tab.first[t + 1] <= b);
        first = tab.first[t]; next = tab.first[t + 1]; size = tab.n[t]; from = static_cast<const char*>(tab.g[t]);
        type = static_cast<int>(reinterpret_cast<uintptr_t>(tab.p[t]));
      }
      const int64_t at = static_cast<int64_t>(b - first) * ADAM_BLOCK;
      const bool whole = size - at >= ADAM_BLOCK && on16(from);
      half[k] = type == HASTE_BF16;
      if (half[k]) {
        const __nv_bfloat16* gp = reinterpret_cast<const __nv_bfloat16*>(from) + at + lane * 8;
        Lane8<__nv_bfloat16> h;
        if (whole) h.load(gp); else h.load_part(gp, size - at - lane * 8);
        g[k].q[0] = h.q[0];
      } else {
        const float* gp = reinterpret_cast<const float*>(from) + at + lane * 8;
        if (whole) g[k].load(gp); else g[k].load_part(gp, size - at - lane * 8);
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      float2 f[4];
      if (half[k]) { Lane8<__nv_bfloat16> h; h.q[0] = g[k].q[0]; h.get(f); } else g[k].get(f);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[k] = fma2(f[i], f[i], acc[k]);
    }
    if (++turns == 16) {
      turns = 0;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) { total += static_cast<double>(acc[k].x) + acc[k].y; acc[k] = both(0.f); }
    }
  }
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) s += acc[k].x + acc[k].y;
  s = static_cast<float>(total + s);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int i = 1; i < WARPS; ++i) s += sums[i];
  return s;
}

// One sum per thread block, each of which has a share of the blocks of its own, into partial[part0 + blockIdx.x].
template <int N>
__global__ void __launch_bounds__(ADAM_THREADS) grad_squares_kernel(const __grid_constant__ TensorTable<N> tab, float* __restrict__ partial, int part0) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t blocks = tab.first[tab.count];
  const float s = sum_of_squares<ADAM_THREADS>(tab, static_cast<int>(blocks * blockIdx.x / gridDim.x), static_cast<int>(blocks * (blockIdx.x + 1) / gridDim.x));
  if (threadIdx.x == 0) partial[part0 + blockIdx.x] = s;
}

// Up to 2^20 elements: one cluster, whose blocks hand their sums to the first one, and no second launch (0.4 M elements, calls back to back:
// 12.0 us instead of 14.2; the launch costs more than the other SMs would bring).
constexpr int NORM_CLUSTER = 8, NORM_THREADS = 1024;
constexpr int64_t NORM_SMALL_BLOCKS = 4096;
template <int N>
__global__ void __cluster_dims__(NORM_CLUSTER, 1, 1) __launch_bounds__(NORM_THREADS) grad_norm_small_kernel(const __grid_constant__ TensorTable<N> tab,
                                                                                                           float grad_scale, float* __restrict__ norm) {
  __shared__ float sums[NORM_CLUSTER];
  cluster_started_arrive();
  auto cluster = cooperative_groups::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), blocks = tab.first[tab.count];
  const float s = sum_of_squares<NORM_THREADS>(tab, blocks * rank / NORM_CLUSTER, blocks * (rank + 1) / NORM_CLUSTER);
  cluster_started_wait();
  if (threadIdx.x == 0) *cluster.map_shared_rank(&sums[rank], 0) = s;
  cluster.sync();
  if (rank == 0 && threadIdx.x == 0) {
    double total = 0.0;
    for (int i = 0; i < NORM_CLUSTER; ++i) total += sums[i];
    *norm = static_cast<float>(sqrt(total) * fabsf(grad_scale));
  }
}

// sqrt of the sum of the partial sums (in 64 bits: one block adds a few hundred), in an order that depends on their number alone.
__global__ void __launch_bounds__(ADAM_THREADS) grad_norm_finish_kernel(const float* __restrict__ partial, int parts, float grad_scale, float* __restrict__ norm) {
  __shared__ double sums[ADAM_THREADS / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
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
    Lane8<float> l;
    float2 f[4];
    l.load(x + e);
    l.get(f);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = f[i].x; v[2 * i + 1] = f[i].y; }
    const float s = block_scale(warp_top(v), inv);
    constexpr uint32_t half = 0x7F7F0000u;
    const uint32_t rnd[8] = {half, half, half, half, half, half, half, half};
    *reinterpret_cast<uint2*>(codes + e) = encode8<SIGNED>(v, inv, rnd);
    if (lane == 0) scales[b] = s;
  }
}

// A lane takes 8 codes at a time, so that a warp stores whole lines, and 4 such pieces of them at once.
template <class O, bool SIGNED>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales, O* __restrict__ out, int64_t n8) {
  constexpr int PIECES = 4;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * 256 * PIECES + threadIdx.x; base < n8; base += static_cast<int64_t>(gridDim.x) * 256 * PIECES) {
    uint2 c[PIECES];
    float s[PIECES];
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const int64_t i = base + k * 256;
      c[k] = i < n8 ? __ldcs(reinterpret_cast<const uint2*>(codes + i * 8)) : make_uint2(0u, 0u);
      s[k] = i < n8 ? __ldg(scales + i / (ADAM_BLOCK / 8)) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const int64_t i = base + k * 256;
      float2 x[4];
      decode8<SIGNED>(c[k], s[k], x);
      uint32_t u[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        u[2 * q] = sizeof(O) == 4 ? __float_as_uint(x[q].x) : static_cast<uint32_t>(rn_bf16_bits(x[q].x)) << 16;
        u[2 * q + 1] = sizeof(O) == 4 ? __float_as_uint(x[q].y) : static_cast<uint32_t>(rn_bf16_bits(x[q].y)) << 16;
      }
      if (i < n8) store_lane(out + i * 8, true, 8, u);
    }
  }
}

// ================================================================ launchers
// Thread blocks for a number of blocks of elements: one for 8 of them, at most `per_sm` times the SMs.
static int adam_grid(int64_t blocks, int per_sm) {
  const int64_t want = (blocks + ADAM_WARPS - 1) / ADAM_WARPS, most = static_cast<int64_t>(sm_count()) * per_sm;
  return static_cast<int>(want < most ? want : most);
}

// The 32-bit step is bound by memory, which is fastest when all of the GPU works on one short stretch of the buffers at a time: many
// thread blocks that take a few blocks of elements each and are started in order (56 M weights, fp32: 272 us with 4 a SM, 228 with 64;
// bf16: 214 and 180).  The 8-bit step is bound by its instructions and pays for starting up: 151 us with 4, 191 with 64.
constexpr int ADAM_PER_SM_32 = 64, ADAM_PER_SM_8 = 4;

constexpr int64_t MAX_BLOCKS = int64_t(1) << 30;          // of a launch: a block's number and one more round of all warps fit 32 bits

// Calls f(table, first block of the part, its blocks) for consecutive parts of the tensors; a tensor of more than 2^30 blocks is refused before.
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

template <int N>
static TensorTable<N> cut_table(const TensorTable<TABLE_LARGE>& tab) {
  TensorTable<N> s;
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
    const int grid = adam_grid(blocks, BITS == 32 ? ADAM_PER_SM_32 : ADAM_PER_SM_8);
    if (tab.count <= TABLE_SMALL) adamw_kernel<P, G, BITS, TABLE_SMALL><<<grid, ADAM_THREADS, 0, st>>>(cut_table<TABLE_SMALL>(tab), m, ms, v, vs, block0, a);
    else if (tab.count <= TABLE_MIDDLE) adamw_kernel<P, G, BITS, TABLE_MIDDLE><<<grid, ADAM_THREADS, 0, st>>>(cut_table<TABLE_MIDDLE>(tab), m, ms, v, vs, block0, a);
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
  const int64_t tables = count / TABLE_LARGE + 1;           // or one more for every 2^30 blocks, whose grids are as large as they get
  const int64_t cap = HASTE_GRAD_NORM_PARTIALS / 2 / tables;
  int parts = 0;
  bool done = false;
  const int rc = for_each_table(nullptr, types, grads, sizes, count, [&](const TensorTable<TABLE_LARGE>& tab, int64_t, int64_t blocks) {
    if (tab.count == count && count <= TABLE_MIDDLE && blocks <= NORM_SMALL_BLOCKS) {          // all of them, not what is left behind 2^30 blocks
      if (count <= TABLE_SMALL) grad_norm_small_kernel<<<NORM_CLUSTER, NORM_THREADS, 0, st>>>(cut_table<TABLE_SMALL>(tab), grad_scale, norm);
      else grad_norm_small_kernel<<<NORM_CLUSTER, NORM_THREADS, 0, st>>>(cut_table<TABLE_MIDDLE>(tab), grad_scale, norm);
      done = true;
      return check_launch("grad_norm_small_kernel");
    }
    const int grid = static_cast<int>(imin64(adam_grid(blocks, 4), cap));
    if (grid < 1 || parts + grid > HASTE_GRAD_NORM_PARTIALS) return fail(HASTE_ERR_TOO_LARGE, "haste_grad_norm: too many tensors for one call");
    if (tab.count <= TABLE_MIDDLE) grad_squares_kernel<TABLE_MIDDLE><<<grid, ADAM_THREADS, 0, st>>>(cut_table<TABLE_MIDDLE>(tab), partial, parts);
    else grad_squares_kernel<TABLE_LARGE><<<grid, ADAM_THREADS, 0, st>>>(tab, partial, parts);
    parts += grid;
    return check_launch("grad_squares_kernel");
  });
  if (rc != HASTE_OK || done) return rc;
  if (parts > 0) return launch_behind(grad_norm_finish_kernel, 1, ADAM_THREADS, st, static_cast<const float*>(partial), parts, grad_scale, norm);
  grad_norm_finish_kernel<<<1, ADAM_THREADS, 0, st>>>(partial, parts, grad_scale, norm);           // no elements: no kernel of this call comes before
  return check_launch("grad_norm_finish_kernel");
}

int launch_quantize(const float* x, uint8_t* codes, float* scales, int64_t n, int is_signed, cudaStream_t st) {
  if (n == 0) return HASTE_OK;
  const int grid = adam_grid(n / ADAM_BLOCK, 4);
  if (is_signed) quantize_kernel<true><<<grid, ADAM_THREADS, 0, st>>>(x, codes, scales, n / ADAM_BLOCK);
  else quantize_kernel<false><<<grid, ADAM_THREADS, 0, st>>>(x, codes, scales, n / ADAM_BLOCK);
  return check_launch("quantize_kernel");
}

int launch_dequantize(const uint8_t* codes, const float* scales, void* out, int64_t n, int is_signed, int type, cudaStream_t st) {
  if (n == 0) return HASTE_OK;
  const int64_t n8 = n / 8, want = (n8 + 1023) / 1024;
  const unsigned grid = static_cast<unsigned>(imin64(want, static_cast<int64_t>(sm_count()) * 16));
  if (type == HASTE_BF16) {
    if (is_signed) dequantize_kernel<__nv_bfloat16, true><<<grid, 256, 0, st>>>(codes, scales, (__nv_bfloat16*)out, n8);
    else dequantize_kernel<__nv_bfloat16, false><<<grid, 256, 0, st>>>(codes, scales, (__nv_bfloat16*)out, n8);
  } else if (is_signed) dequantize_kernel<float, true><<<grid, 256, 0, st>>>(codes, scales, (float*)out, n8);
  else dequantize_kernel<float, false><<<grid, 256, 0, st>>>(codes, scales, (float*)out, n8);
  return check_launch("dequantize_kernel");
}

}  // namespace haste
