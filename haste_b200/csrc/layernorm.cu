// Layer norm over the last dimension, forward and backward.
//
//   mean = sum(x) / D     var = sum((x - mean)^2) / D     r = 1 / sqrt(var + eps)     z = (x - mean) r
//   y  = z w + b
//   h  = dy w             dx = r (h - mean(h) - z mean(h z))     dw = sum_rows dy z     db = sum_rows dy
//
// All sums are fp32; the variance is taken around the mean, not from the sum of squares, which cancels for rows whose mean is large
// against their spread.  x is added up times a power of two below 1 / D, so that a row of the largest numbers has a mean, which is not beyond them.
// Inputs and outputs are bf16 or fp32, rounded once (nearest even) when stored.
//
// Memory bounds all of it: x in and y out, or dy and x in and dx out.  A row is read once and stays on the chip: 1 to 32 lanes of a
// warp have it, or a thread block where it is wider, each thread up to 4 vectors of 16 bytes.  These groups walk over the rows with the
// next rows on their way, so that in the backward pass a thread owns its columns for good and sums dw and db in registers; the blocks'
// sums go to memory and are added in a second, small launch.  Rows of more than 8192 elements (16384 bf16 in the forward pass) are
// read again for each pass.
#include "common.cuh"

#include <cooperative_groups.h>
#include <atomic>
#include "launchers.h"

namespace haste {

__device__ __forceinline__ float ld_f(const float* p) { return *p; }
__device__ __forceinline__ float ld_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st_f(float* p, float v) { *p = v; }
__device__ __forceinline__ void st_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum over the block, the same value in every thread.  `buf`: one float per warp; the caller may use it again at once.
__device__ __forceinline__ float block_sum(float v, float* buf) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < (blockDim.x >> 5); ++i) s += buf[i];
  return s;
}

// Half the largest power of two that is not above 1 / D: a sum of so much of D finite numbers is finite, whatever its roundings.
__device__ __forceinline__ float power_below(int64_t D) { return __int_as_float((126 - (64 - __clzll(D - 1))) << 23); }
// A mean that was made from that sum: it may have been rounded beyond the largest number, where the mean of finite numbers is not.
__device__ __forceinline__ float in_range(float mean, float sum) {
  const float most = __int_as_float(0x7F7FFFFF);
  return fabsf(sum) <= most ? fminf(fmaxf(mean, -most), most) : mean;
}

constexpr int LN_THREADS = 256;

// ---------------------------------------------------------------- rows of any width: one block a row, the row read again for each pass
template <class X, class W>
__global__ void __launch_bounds__(LN_THREADS) ln_fwd_wide_kernel(const X* __restrict__ x, const W* __restrict__ w, const W* __restrict__ b, X* __restrict__ y,
                                                                 float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows, int64_t D,
                                                                 int64_t ldx, float eps) {
  __shared__ float buf[LN_THREADS / 32];
  const float part = power_below(D);
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const X* xr = x + r * ldx;
    float s = 0.f;
    for (int64_t j = threadIdx.x; j < D; j += LN_THREADS) s = fmaf(ld_f(xr + j), part, s);
    const float sum = block_sum(s, buf), mean = in_range(sum / (static_cast<float>(D) * part), sum);
    s = 0.f;
    for (int64_t j = threadIdx.x; j < D; j += LN_THREADS) { const float d = ld_f(xr + j) - mean; s += d * d; }
    const float rstd = 1.f / sqrtf(block_sum(s, buf) / static_cast<float>(D) + eps);
    for (int64_t j = threadIdx.x; j < D; j += LN_THREADS) {
      const float z = (ld_f(xr + j) - mean) * rstd;
      st_f(y + r * D + j, fmaf(z, w ? ld_f(w + j) : 1.f, b ? ld_f(b + j) : 0.f));
    }
    if (threadIdx.x == 0 && mean_out) { mean_out[r] = mean; rstd_out[r] = rstd; }
  }
}

template <class X, class G, class W>
__global__ void __launch_bounds__(LN_THREADS) ln_bwd_dx_wide_kernel(const G* __restrict__ dy, const X* __restrict__ x, const W* __restrict__ w,
                                                                    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, X* __restrict__ dx,
                                                                    int64_t rows, int64_t D, int64_t lddy, int64_t ldx) {
  __shared__ float buf[LN_THREADS / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const X* xr = x + r * ldx;
    const G* gr = dy + r * lddy;
    const float mean = mean_in[r], rstd = rstd_in[r];
    float sh = 0.f, shz = 0.f;
    for (int64_t j = threadIdx.x; j < D; j += LN_THREADS) {
      const float h = ld_f(gr + j) * (w ? ld_f(w + j) : 1.f);
      sh += h;
      shz = fmaf(h, (ld_f(xr + j) - mean) * rstd, shz);
    }
    const float mh = block_sum(sh, buf) / static_cast<float>(D), mhz = block_sum(shz, buf) / static_cast<float>(D);
    for (int64_t j = threadIdx.x; j < D; j += LN_THREADS) {
      const float h = ld_f(gr + j) * (w ? ld_f(w + j) : 1.f), z = (ld_f(xr + j) - mean) * rstd;
      st_f(dx + r * D + j, rstd * (h - mh - z * mhz));
    }
  }
}

// Column sums of dy z and dy over the rows of one of `parts` row ranges: part p goes to partial[p][0][.] and partial[p][1][.].
template <class X, class G>
__global__ void __launch_bounds__(LN_THREADS) ln_bwd_columns_kernel(const G* __restrict__ dy, const X* __restrict__ x, const float* __restrict__ mean_in,
                                                                    const float* __restrict__ rstd_in, float* __restrict__ partial, int64_t rows, int64_t D,
                                                                    int64_t lddy, int64_t ldx) {
  __shared__ float sw[8][32], sb[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t part = blockIdx.y, parts = gridDim.y, r0 = rows * part / parts, r1 = rows * (part + 1) / parts;
  for (int64_t c0 = static_cast<int64_t>(blockIdx.x) * 32; c0 < D; c0 += static_cast<int64_t>(gridDim.x) * 32) {
    const int64_t c = c0 + tx;
    float aw = 0.f, ab = 0.f;
    if (c < D)
      for (int64_t r = r0 + ty; r < r1; r += 8) {
        const float g = ld_f(dy + r * lddy + c);
        aw = fmaf(g, (ld_f(x + r * ldx + c) - mean_in[r]) * rstd_in[r], aw);
        ab += g;
      }
    sw[ty][tx] = aw; sb[ty][tx] = ab;
    __syncthreads();
    if (ty == 0 && c < D) {
#pragma unroll
      for (int i = 1; i < 8; ++i) { aw += sw[i][tx]; ab += sb[i][tx]; }
      partial[(2 * part) * D + c] = aw;
      partial[(2 * part + 1) * D + c] = ab;
    }
    __syncthreads();
  }
}

// The parts of dw and db as they lie in the scratch: part p is [2][width], column j of dw at j + (p step & mask), db's behind them.
// (A block whose rows start s elements behind a 16-byte boundary leaves its sums s places further on, so that it
// stores whole vectors: 4099 x 1021 backward 19.1 us a call, 23.3 with an element at a time; 32768 x 4096 161 and 168.)
struct Parts {
  int count;
  int64_t width;
  unsigned step, mask;
};

// dw and db from the partial sums, in an order that depends on their number alone: the same bits every time.  A block adds 32 columns over
// 16 shares of the parts; with many parts CLUSTER blocks do, and hand their sums to the first of them.
constexpr int LN_FINISH_THREADS = 512, LN_FINISH_CLUSTER = 4;
template <class W, int CLUSTER>
__device__ __forceinline__ void finish_columns(const float* __restrict__ partial, const Parts& parts, int64_t D, W* __restrict__ dw, W* __restrict__ db) {
  constexpr int SPLIT = LN_FINISH_THREADS / 32;
  __shared__ float buf[SPLIT][33];
  __shared__ float shares[CLUSTER][32];
  if constexpr (CLUSTER > 1) cluster_started_arrive();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, rank = blockIdx.x % CLUSTER;
  const int64_t c = static_cast<int64_t>(blockIdx.x / CLUSTER) * 32 + tx;      // column of dw, or D more: of db
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float s = 0.f;
  if (c < 2 * D) {
    const float* from = partial + (c < D ? c : c - D + parts.width);
#pragma unroll 8
    for (int p = rank * SPLIT + ty; p < parts.count; p += SPLIT * CLUSTER) s += from[p * 2 * parts.width + (p * parts.step & parts.mask)];
  }
  buf[ty][tx] = s;
  __syncthreads();
  if constexpr (CLUSTER > 1) cluster_started_wait();
  if (ty == 0) {
#pragma unroll
    for (int i = 1; i < SPLIT; ++i) s += buf[i][tx];
    if constexpr (CLUSTER > 1) *cooperative_groups::this_cluster().map_shared_rank(&shares[rank][tx], 0) = s;
  }
  if constexpr (CLUSTER > 1) {
    cooperative_groups::this_cluster().sync();
    if (rank != 0) return;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < CLUSTER; ++i) s += shares[i][tx];
  }
  if (ty == 0 && c < 2 * D) {
    if (c < D) { if (dw) st_f(dw + c, s); }
    else if (db) st_f(db + (c - D), s);
  }
}
template <class W>
__global__ void __launch_bounds__(LN_FINISH_THREADS) ln_bwd_finish_kernel(const float* __restrict__ partial, const Parts parts, int64_t D, W* __restrict__ dw,
                                                                         W* __restrict__ db) {
  finish_columns<W, 1>(partial, parts, D, dw, db);
}
template <class W>
__global__ void __cluster_dims__(LN_FINISH_CLUSTER, 1, 1) __launch_bounds__(LN_FINISH_THREADS)
    ln_bwd_finish_many_kernel(const float* __restrict__ partial, const Parts parts, int64_t D, W* __restrict__ dw, W* __restrict__ db) {
  finish_columns<W, LN_FINISH_CLUSTER>(partial, parts, D, dw, db);
}

// ---------------------------------------------------------------- rows that stay on the chip
// A row is cut at the 16-byte boundaries of the (contiguous, aligned) output, so that vector q of a row holds its columns
// q VEC - s .. q VEC - s + VEC - 1, s being the row's distance from the boundary before it; of the first and the last vector a part may
// belong to the neighbouring rows.  Groups of threads take rows at distances that are multiples of VEC: s stays the same, and a thread
// its columns.  An input whose rows have the same s (contiguous ones do) is copied in vectors as well, any other element by element.
//
// Each thread copies its own vectors of the row after next into its own slots of shared memory (cp.async: no registers, no barrier) while
// it works on the row that has arrived.  What lies outside the row or the rows reads as zero, so that most sums need no masks: the copies
// fill up with zeros, and of a row's first vector the part before the row is dropped when it is read.
__device__ __forceinline__ uint32_t smem_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Vectors that a row may touch.
__host__ __device__ constexpr int64_t row_units(int64_t D, int vec) { return D % vec == 0 ? D / vec : (D + 2 * vec - 2) / vec; }

constexpr int LN_STAGES = 3;              // rows on their way or at work, per group
constexpr int LN_WARP_THREADS = 128;      // block of the variant whose groups are within a warp

// Two fp32 numbers as one operand: one instruction for both.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)),
      "l"(reinterpret_cast<const uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// VEC elements of type T in a slot: WORDS accesses of 16 bytes (one of 8 for 4 bf16), `step` bytes apart, so that the lanes of a
// warp touch consecutive 16 bytes each time.  Addresses `dst` are shared memory's.
template <class T, int VEC> struct Slot {
  static constexpr int BYTES = VEC * static_cast<int>(sizeof(T)), WORDS = (BYTES + 15) / 16, UNIT = BYTES < 16 ? BYTES : 16, PER = UNIT / static_cast<int>(sizeof(T));
  static __device__ __forceinline__ void copy_unit(uint32_t dst, const void* src, int bytes) {       // of which `bytes` are read, the rest becomes zeros
    if (UNIT == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
  }
  static __device__ __forceinline__ void copy(uint32_t dst, int step, const T* src) {
#pragma unroll
    for (int k = 0; k < WORDS; ++k) {
      if (UNIT == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + k * step), "l"(src + k * PER) : "memory");
      else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst + k * step), "l"(src + k * PER) : "memory");
    }
  }
  static __device__ __forceinline__ void copy_part(uint32_t dst, int step, const T* src, int n) {    // the first n > 0 elements, then zeros
#pragma unroll
    for (int k = 0; k < WORDS; ++k) {
      const int bytes = min(max((n - k * PER) * static_cast<int>(sizeof(T)), 0), UNIT);
      copy_unit(dst + k * step, bytes > 0 ? src + k * PER : src, bytes);
    }
  }
  static __device__ void copy_single(char* dst, int step, const T* src, int first, int n) {          // elements first .. n-1, zeros elsewhere
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      T v;
      st_f(&v, 0.f);
      if (e >= first && e < n) v = src[e];
      reinterpret_cast<T*>(dst + e / PER * step)[e % PER] = v;
    }
  }
  static __device__ __forceinline__ void clear(char* dst, int step) {
#pragma unroll
    for (int k = 0; k < WORDS; ++k) {
      if (UNIT == 16) *reinterpret_cast<uint4*>(dst + k * step) = make_uint4(0u, 0u, 0u, 0u);
      else *reinterpret_cast<uint2*>(dst + k * step) = make_uint2(0u, 0u);
    }
  }
  // Masks of the words that hold elements `first` and following: what lies before belongs to another row and reads as 0.
  static constexpr int REGS = BYTES / 4;
  static __device__ __forceinline__ void head_masks(int first, uint32_t (&m)[REGS]) {
#pragma unroll
    for (int e = 0; e < REGS; ++e) {
      if constexpr (sizeof(T) == 4) m[e] = e < first ? 0u : 0xFFFFFFFFu;
      else m[e] = (2 * e < first ? 0u : 0x0000FFFFu) | (2 * e + 1 < first ? 0u : 0xFFFF0000u);
    }
  }
  template <bool MASK>
  static __device__ __forceinline__ void get(const char* src, int step, float2 (&f)[VEC / 2], const uint32_t (&m)[REGS]) {
    uint32_t u[REGS];
#pragma unroll
    for (int k = 0; k < WORDS; ++k) {
      if constexpr (UNIT == 16) { const uint4 v = *reinterpret_cast<const uint4*>(src + k * step); u[4 * k] = v.x; u[4 * k + 1] = v.y; u[4 * k + 2] = v.z; u[4 * k + 3] = v.w; }
      else { const uint2 v = *reinterpret_cast<const uint2*>(src + k * step); u[0] = v.x; u[1] = v.y; }
    }
#pragma unroll
    for (int e = 0; e < REGS; ++e) if (MASK) u[e] &= m[e];
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
      if constexpr (sizeof(T) == 4) f[e] = make_float2(__uint_as_float(u[2 * e]), __uint_as_float(u[2 * e + 1]));
      else f[e] = make_float2(__uint_as_float(u[e] << 16), __uint_as_float(u[e] & 0xFFFF0000u));
    }
  }
};

__device__ __forceinline__ void pack(const float2 (&f)[4], uint32_t (&w)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[i].x, f[i].y);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
}
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float2 (&f)[4]) {
  uint32_t w[4];
  pack(f, w);
  __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
}
__device__ __forceinline__ void store_vec(float* p, const float2 (&f)[2]) { __stcs(reinterpret_cast<float4*>(p), make_float4(f[0].x, f[0].y, f[1].x, f[1].y)); }
// A row's end of one of its vectors, elements first .. VEC - 1 or 0 .. n - 1, in powers of two: three stores instead of up to seven (the
// warp waits for the lane that has them).
__device__ __forceinline__ void store_head(__nv_bfloat16* p, int first, const float2 (&f)[4]) {
  uint32_t w[4];
  pack(f, w);
  if (first <= 4) *reinterpret_cast<uint2*>(p + 4) = make_uint2(w[2], w[3]);
  if ((first + 1) & 2) *reinterpret_cast<uint32_t*>(p + (first <= 2 ? 2 : 6)) = first <= 2 ? w[1] : w[3];
  if (first & 1) *reinterpret_cast<uint16_t*>(p + first) = static_cast<uint16_t>((first < 4 ? (first < 2 ? w[0] : w[1]) : (first < 6 ? w[2] : w[3])) >> 16);
}
__device__ __forceinline__ void store_tail(__nv_bfloat16* p, int n, const float2 (&f)[4]) {
  uint32_t w[4];
  pack(f, w);
  if (n & 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  if (n & 2) *reinterpret_cast<uint32_t*>(p + (n & 4)) = n & 4 ? w[2] : w[0];
  if (n & 1) *reinterpret_cast<uint16_t*>(p + n - 1) = static_cast<uint16_t>(n & 4 ? (n & 2 ? w[3] : w[2]) : (n & 2 ? w[1] : w[0]));
}
__device__ __forceinline__ void store_head(float* p, int first, const float2 (&f)[2]) {
  if (first <= 2) *reinterpret_cast<float2*>(p + 2) = f[1];
  if (first & 1) p[first] = first < 2 ? f[0].y : f[1].y;
}
__device__ __forceinline__ void store_tail(float* p, int n, const float2 (&f)[2]) {
  if (n & 2) *reinterpret_cast<float2*>(p) = f[0];
  if (n & 1) p[n - 1] = n & 2 ? f[1].x : f[0].x;
}
// Columns j0 .. of a row, p the first one's place: the whole vector, or those of its elements that belong to the row.  HEAD, TAIL: whether
// the row may begin, end in it.
template <int VEC, bool HEAD, bool TAIL, class T>
__device__ __forceinline__ void store_part(T* p, int j0, int D, const float2 (&f)[VEC / 2]) {
  if ((!HEAD || j0 >= 0) && (!TAIL || j0 + VEC <= D)) store_vec(p, f);
  else if (HEAD && j0 < 0 && j0 + VEC <= D) store_head(p, -j0, f);
  else if (TAIL && j0 >= 0) store_tail(p, D - j0, f);
  else {
    if constexpr (HEAD && TAIL) {                                      // both: D < VEC
#pragma unroll
      for (int k = 0; k < VEC; ++k) if (static_cast<unsigned>(j0 + k) < static_cast<unsigned>(D)) st_f(p + k, k & 1 ? f[k / 2].y : f[k / 2].x);
    }
  }
}

// Weights of a thread's columns, once per kernel; 0 outside the row.  vec: whole vectors only, on 16 bytes.
template <int VEC>
__device__ __forceinline__ void load_weights(const void* w, int w_type, bool vec, int j0, int D, float fill, float2 (&out)[VEC / 2]) {
  float f[VEC];
  if (w == nullptr) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[k] = static_cast<unsigned>(j0 + k) < static_cast<unsigned>(D) ? fill : 0.f;
  } else if (w_type == HASTE_BF16) {
    const uint16_t* p = static_cast<const uint16_t*>(w) + j0;
    uint32_t u[VEC];
    if (vec) {
      if constexpr (VEC == 8) {
        const uint4 v = j0 < D ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0u, 0u, 0u, 0u);
        u[0] = v.x << 16; u[1] = v.x & 0xFFFF0000u; u[2] = v.y << 16; u[3] = v.y & 0xFFFF0000u;
        u[4] = v.z << 16; u[5] = v.z & 0xFFFF0000u; u[6] = v.w << 16; u[7] = v.w & 0xFFFF0000u;
      } else {
        const uint2 v = j0 < D ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0u, 0u);
        u[0] = v.x << 16; u[1] = v.x & 0xFFFF0000u; u[2] = v.y << 16; u[3] = v.y & 0xFFFF0000u;
      }
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) u[k] = static_cast<unsigned>(j0 + k) < static_cast<unsigned>(D) ? static_cast<uint32_t>(__ldg(p + k)) << 16 : 0u;
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[k] = __uint_as_float(u[k]);
  } else {
    const float* p = static_cast<const float*>(w) + j0;
    if (vec) {
#pragma unroll
      for (int k = 0; k < VEC; k += 4) {
        const float4 v = j0 < D ? __ldg(reinterpret_cast<const float4*>(p + k)) : make_float4(0.f, 0.f, 0.f, 0.f);
        f[k] = v.x; f[k + 1] = v.y; f[k + 2] = v.z; f[k + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] = static_cast<unsigned>(j0 + k) < static_cast<unsigned>(D) ? __ldg(p + k) : 0.f;
    }
  }
#pragma unroll
  for (int k = 0; k < VEC / 2; ++k) out[k] = make_float2(f[2 * k], f[2 * k + 1]);
}

// The threads that share a row: T lanes of a warp (a power of two), or the block.  Thread c of a warp's group has vectors c, c + T, c + 2 T ..
// of the row; warp v of a block has its vectors 32 NV v and following in the same way, so that from one vector of a thread to its next it
// is 32 vectors, a constant, wherever T >= 32 (FULL).
enum RowMode { SUB, FULL, BLOCK };       // groups of up to 32 lanes, of 32, blocks
template <int MODE, int NV>
struct RowGroup {
  int T, c;              // threads of a warp's group; first vector of this thread
  int slot = 0;          // buffer of the next sum over a block: a buffer is written again two sums (two barriers) later
  __device__ explicit RowGroup(int t) : T(MODE == SUB ? t : 32), c(MODE == SUB ? static_cast<int>(threadIdx.x) & (t - 1) : MODE == FULL ? static_cast<int>(threadIdx.x & 31) : static_cast<int>((threadIdx.x >> 5) * 32 * NV + (threadIdx.x & 31))) {}
  // rows of a warp (of a block) are neighbours; first: that of its first group
  __device__ int64_t first_row() const { return MODE == BLOCK ? blockIdx.x : (static_cast<int64_t>(blockIdx.x) * blockDim.x + (threadIdx.x & ~31u)) / T; }
  __device__ int64_t stride() const { return MODE == BLOCK ? gridDim.x : static_cast<int64_t>(gridDim.x) * blockDim.x / T; }
  __device__ int64_t own() const { return MODE == SUB ? static_cast<int64_t>((threadIdx.x & 31u) / T) : 0; }
  __device__ __forceinline__ void sum_warps(float& v, float* buf) {        // buf: of the slot
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < (static_cast<int>(blockDim.x) + 127) >> 7; ++i) {  // slots of warps that the block has not got hold zeros
      const float4 q = reinterpret_cast<const float4*>(buf)[i];
      v += (q.x + q.y) + (q.z + q.w);
    }
  }
  __device__ __forceinline__ float sum(float v, float (*buf)[2][16]) {
    if (MODE == SUB) {
      for (int o = T >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      return v;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (MODE == BLOCK) { sum_warps(v, buf[slot][0]); slot ^= 1; }
    return v;
  }
  // Two sums for little more than one: after the first exchange the lower half of a warp adds up a, the upper half b.
  __device__ __forceinline__ void sum2_lanes(float& a, float& b) {
    if (MODE == SUB) {
      for (int o = T >> 1; o > 0; o >>= 1) { a += __shfl_xor_sync(0xffffffffu, a, o); b += __shfl_xor_sync(0xffffffffu, b, o); }
      return;
    }
    const bool upper = threadIdx.x & 16;
    const float other = __shfl_xor_sync(0xffffffffu, upper ? a : b, 16);
    float v = (upper ? b : a) + other;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (MODE == BLOCK) { a = v; return; }                                  // sum2_warps takes it from lanes 0 and 16
    a = __shfl_sync(0xffffffffu, v, 0);
    b = __shfl_sync(0xffffffffu, v, 16);
  }
  __device__ __forceinline__ void sum2_warps(float& a, float& b, float (*buf)[2][16]) {
    if (MODE != BLOCK) return;
    if ((threadIdx.x & 15) == 0) buf[slot][(threadIdx.x >> 4) & 1][threadIdx.x >> 5] = a;
    __syncthreads();
    a = b = 0.f;
    for (int i = 0; i < (static_cast<int>(blockDim.x) + 127) >> 7; ++i) {
      const float4 q = reinterpret_cast<const float4*>(buf[slot][0])[i], p = reinterpret_cast<const float4*>(buf[slot][1])[i];
      a += (q.x + q.y) + (q.z + q.w);
      b += (p.x + p.y) + (p.z + p.w);
    }
    slot ^= 1;
  }
  // Zeros for the warps that the block has not got; a barrier follows before the first sum is read.
  __device__ __forceinline__ void clear(float (*buf)[2][16]) {
    if (MODE == BLOCK && threadIdx.x < 64) (&buf[0][0][0])[threadIdx.x] = 0.f;
    if (MODE == BLOCK) __syncthreads();
  }
};

// A row group's walk over an input: the copies of its next row.  A warp's slots lie together, 32 units for each word of a vector.
template <class T, int VEC, int NV, int MODE, bool EDGE>
struct Feed {
  using S = Slot<T, VEC>;
  static constexpr int STEP = 32 * S::UNIT, WARP_BYTES = NV * S::WORDS * STEP;      // between the words of a slot; of a warp and stage
  const T* next;           // column j0 of the row to be copied next
  int64_t row_step;        // elements from a row of the group to its next one
  int t_step;              // elements from a vector of the thread to its next one (SUB)
  int j0, D;
  bool vec;
  char* slots;             // the thread's own, of the first stage
  uint32_t to;
  uint32_t masks[S::REGS]; // of the thread's first vector
  __device__ __forceinline__ Feed(const T* p, int64_t ld, int64_t row, int64_t stride, int j0_, int D_, int T_, bool vec_, char* area)
      : next(p + row * ld + j0_), row_step(stride * ld), t_step(T_ * VEC), j0(j0_), D(D_), vec(vec_),
        slots(area + (threadIdx.x >> 5) * WARP_BYTES + (threadIdx.x & 31) * S::UNIT), to(smem_address(slots)) { S::head_masks(-j0_, masks); }
  __device__ __forceinline__ int vec_step() const { return MODE == SUB ? t_step : 32 * VEC; }
  static __device__ __forceinline__ int bytes() { return WARP_BYTES * static_cast<int>(blockDim.x >> 5); }
  // Slots that no copy reaches (vectors right of the row) hold zeros for good.
  __device__ __forceinline__ void clear(int stages, int stage_bytes) const {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (j0 + i * vec_step() >= D)
        for (int k = 0; k < stages; ++k) S::clear(slots + k * stage_bytes + i * S::WORDS * STEP, STEP);
  }
  __device__ __forceinline__ void fetch(int at, bool there) {
    if (there) {
      if (vec) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int j = j0 + i * vec_step();
          if (j < D) {
            if (!EDGE || !may_end(i)) S::copy(to + at + i * S::WORDS * STEP, STEP, next + i * vec_step());
            else S::copy_part(to + at + i * S::WORDS * STEP, STEP, next + i * vec_step(), min(D - j, VEC));
          }
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < NV; ++i) {
          const int j = j0 + i * vec_step();
          if (j < D) S::copy_single(slots + at + i * S::WORDS * STEP, STEP, next + i * vec_step(), -j, D - j);
        }
      }
    }
    next += row_step;
  }
  // Whether the row may end in a thread's vector i: one of the last two, or any (a block may have whole warps beyond the row).
  static __device__ __forceinline__ constexpr bool may_end(int i) { return MODE == BLOCK || i >= NV - 2; }
  __device__ __forceinline__ void get(int at, int i, float2 (&f)[VEC / 2]) const {
    if (i == 0) S::template get<EDGE>(slots + at, STEP, f, masks);
    else S::template get<false>(slots + at + i * S::WORDS * STEP, STEP, f, masks);
  }
};

// Factors 1 and 0 of a vector's elements that belong to the row and that do not, in shared memory: entry n <= VEC has the first n,
// entry VEC + s the elements s and following, entry 2 VEC + s elements s .. s + D - 1 (a row within a vector).
template <int VEC>
struct EdgeTable {
  static constexpr int ENTRIES = 3 * VEC;
  float4 q[ENTRIES][VEC / 4];
  __device__ __forceinline__ void fill(int D) {
    for (int i = threadIdx.x; i < ENTRIES * VEC; i += blockDim.x) {
      const int e = i / VEC, k = i % VEC, s = e % VEC;
      reinterpret_cast<float*>(q)[i] = (e <= VEC ? k < e : e < 2 * VEC ? k >= s : k >= s && k < s + D) ? 1.f : 0.f;
    }
  }
  static __device__ __forceinline__ int entry(int j, int D) {             // of the vector that begins at column j, in bytes
    const int n = min(max(D - j, 0), VEC);
    return (j >= 0 ? n : D - j >= VEC ? VEC - j : 2 * VEC - j) * VEC * 4;
  }
  __device__ __forceinline__ const float4& get(int at, int k) const { return *reinterpret_cast<const float4*>(reinterpret_cast<const char*>(q) + at + 16 * k); }
};

template <int VEC, class FEED, class T>
__device__ __forceinline__ void store_at(T* p, int i, int j, int D, const float2 (&f)[VEC / 2]) {
  if (i == 0) { if (FEED::may_end(0)) store_part<VEC, true, true>(p, j, D, f); else store_part<VEC, true, false>(p, j, D, f); }
  else { if (FEED::may_end(i)) store_part<VEC, false, true>(p, j, D, f); else store_vec(p, f); }
}

// Blocks of at most LN_WARP_THREADS: 4 on a SM, but 3 with 4 vectors of 8 elements where rows are cut (67041 x 1001 68 us with 4, for which the registers
// do not suffice, 49 with 3; with 3 vectors a thread 68 and 74).
// The factors of cut rows (EdgeTable) are read where a vector has 8 elements: 130816 x 513 bf16 68 us, 94 with comparisons; with 4 elements these cost
// less (332222 x 101 fp32 51 and 49).
// EDGE: D is no multiple of VEC, rows have first and last vectors that are theirs in part.
template <class X, int VEC, int NV, int MODE, bool EDGE>
__global__ void __launch_bounds__(MODE == BLOCK ? 512 : LN_WARP_THREADS, MODE == BLOCK ? 1 : EDGE && VEC * NV > 24 ? 3 : 4)
    ln_fwd_kernel(const X* __restrict__ x, const void* __restrict__ w, const void* __restrict__ b, int w_type, X* __restrict__ y, float* __restrict__ mean_out,
                  float* __restrict__ rstd_out, int64_t rows, int D, int64_t ldx, float eps, int t, bool x_vec, bool w_vec) {
  __shared__ __align__(16) float buf[2][2][16];
  extern __shared__ __align__(16) char slots[];
  constexpr bool TABLE = EDGE && VEC == 8;
  __shared__ EdgeTable<VEC> edges;
  if (TABLE) { edges.fill(D); __syncthreads(); }
  RowGroup<MODE, NV> grp(t);
  grp.clear(buf);
  const float inv_d = 1.f / static_cast<float>(D), part = power_below(D), inv_dp = 1.f / (static_cast<float>(D) * part);
  const int64_t stride = grp.stride();
  int64_t r = grp.first_row() + grp.own(), left = rows - grp.first_row();       // left: rows from the warp's (block's) first one on
  const int s = EDGE ? static_cast<int>(r * D % VEC) : 0, first = grp.c == 0 ? s : 0, j0 = grp.c * VEC - s;
  Feed<X, VEC, NV, MODE, EDGE> in(x, ldx, r, stride, j0, D, grp.T, x_vec, slots);
  const int stage_bytes = in.bytes(), all = LN_STAGES * stage_bytes;
  in.clear(LN_STAGES, stage_bytes);
#pragma unroll
  for (int k = 0; k < LN_STAGES - 1; ++k) { in.fetch(k * stage_bytes, r + k * stride < rows); copies_commit(); }
  float2 wf[NV][VEC / 2], bf[NV][VEC / 2];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_weights<VEC>(w, w_type, !EDGE && w_vec, j0 + i * in.vec_step(), D, 1.f, wf[i]);
    load_weights<VEC>(b, w_type, !EDGE && w_vec, j0 + i * in.vec_step(), D, 0.f, bf[i]);
  }
  int edge_at[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) edge_at[i] = TABLE ? EdgeTable<VEC>::entry(j0 + i * in.vec_step(), D) : 0;
  X* out = y + r * D + j0;
  for (int at = 0, next_at = all - stage_bytes; left > 0; left -= stride, r += stride, out += stride * D) {
    copies_wait<LN_STAGES - 2>();
    in.fetch(next_at, r + (LN_STAGES - 1) * stride < rows);          // to where the last row was
    copies_commit();
    float2 f[NV][VEC / 2], s1 = both(0.f), s2 = both(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      in.get(at, i, f[i]);
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) { if (k & 1) s2 = fma2(f[i][k], both(part), s2); else s1 = fma2(f[i][k], both(part), s1); }
    }
    s1 = add2(s1, s2);
    const float sum = grp.sum(s1.x + s1.y, buf), mean = in_range(sum * inv_dp, sum);
    s1 = s2 = both(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = j0 + i * in.vec_step();
      // what is not the row's counts for nothing
      if (TABLE && (i == 0 || in.may_end(i))) {
#pragma unroll
        for (int q = 0; q < VEC / 4; ++q) {
          const float4 ours = edges.get(edge_at[i], q);
          f[i][2 * q] = fma2(make_float2(ours.x, ours.y), both(-mean), f[i][2 * q]);
          f[i][2 * q + 1] = fma2(make_float2(ours.z, ours.w), both(-mean), f[i][2 * q + 1]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) f[i][k] = add2(f[i][k], both(-mean));
        if (EDGE && i == 0) {
#pragma unroll
          for (int k = 0; k < VEC / 2; ++k) { f[i][k].x = 2 * k < first ? 0.f : f[i][k].x; f[i][k].y = 2 * k + 1 < first ? 0.f : f[i][k].y; }
        }
        if (EDGE && in.may_end(i)) {
#pragma unroll
          for (int k = 0; k < VEC / 2; ++k) { f[i][k].x = j + 2 * k < D ? f[i][k].x : 0.f; f[i][k].y = j + 2 * k + 1 < D ? f[i][k].y : 0.f; }
        }
      }
      if (EDGE || j < D) {
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) { if (k & 1) s2 = fma2(f[i][k], f[i][k], s2); else s1 = fma2(f[i][k], f[i][k], s1); }
      }
    }
    s1 = add2(s1, s2);
    const float rstd = 1.f / sqrtf(fmaf(grp.sum(s1.x + s1.y, buf), inv_d, eps));
    if (r < rows) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = j0 + i * in.vec_step();
        if (j < D) {
#pragma unroll
          for (int k = 0; k < VEC / 2; ++k) f[i][k] = fma2(mul2(f[i][k], both(rstd)), wf[i][k], bf[i][k]);
          if (EDGE) store_at<VEC, decltype(in)>(out + i * in.vec_step(), i, j, D, f[i]); else store_vec(out + i * in.vec_step(), f[i]);
        }
      }
      if (grp.c == 0 && mean_out != nullptr) { mean_out[r] = mean; rstd_out[r] = rstd; }
    }
    next_at = at;
    at = at + stage_bytes < all ? at + stage_bytes : 0;
  }
  copies_wait<0>();
}

// dx, and the block's part of dw and db: partial[block][0][.] and [1][.] (NULL: only dx is wanted).
// A row's sums are on their way through the warps while the next row's are taken, so two rows have arrived and the others (two of STAGES = 4,
// one of 3) are being copied.
template <class X, class G, int VEC, int NV, int MODE, bool EDGE, int STAGES>
__global__ void __launch_bounds__(MODE == BLOCK ? (VEC * NV > 16 ? 256 : 512) : LN_WARP_THREADS) __maxnreg__(VEC * NV > 16 ? 168 : 128)
    ln_bwd_kernel(const G* __restrict__ dy, const X* __restrict__ x, const void* __restrict__ w, int w_type, const float* __restrict__ mean_in,
                  const float* __restrict__ rstd_in, X* __restrict__ dx, float* __restrict__ partial, int64_t rows, int D, int64_t lddy, int64_t ldx, int t,
                  bool x_vec, bool dy_vec, bool w_vec) {
  __shared__ __align__(16) float buf[2][2][16];
  extern __shared__ __align__(16) char slots[];
  RowGroup<MODE, NV> grp(t);
  grp.clear(buf);
  const float inv_d = 1.f / static_cast<float>(D);
  const int64_t stride = grp.stride();
  int64_t r = grp.first_row() + grp.own(), left = rows - grp.first_row();
  const int s = EDGE ? static_cast<int>(r * D % VEC) : 0, j0 = grp.c * VEC - s;
  Feed<X, VEC, NV, MODE, EDGE> xin(x, ldx, r, stride, j0, D, grp.T, x_vec, slots);
  Feed<G, VEC, NV, MODE, EDGE> gin(dy, lddy, r, stride, j0, D, grp.T, dy_vec, slots + xin.bytes());
  const int stage_bytes = xin.bytes() + gin.bytes(), all = STAGES * stage_bytes;
  xin.clear(STAGES, stage_bytes);
  gin.clear(STAGES, stage_bytes);
#pragma unroll
  for (int k = 0; k < STAGES - 1; ++k) {
    xin.fetch(k * stage_bytes, r + k * stride < rows);
    gin.fetch(k * stage_bytes, r + k * stride < rows);
    copies_commit();
  }
  float2 wf[NV][VEC / 2], aw[NV][VEC / 2], ab[NV][VEC / 2];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_weights<VEC>(w, w_type, !EDGE && w_vec, j0 + i * xin.vec_step(), D, 1.f, wf[i]);
#pragma unroll
    for (int k = 0; k < VEC / 2; ++k) aw[i][k] = ab[i][k] = both(0.f);
  }
  // Sums of h and h z over a thread's columns of the row at `at`.  Outside the row g and x are 0, and x - mean is finite where z might not be
  // (a row of the largest numbers): z is not formed, its factor r goes to dy and to the sum.
  auto row_sums = [&](int at, float mean, float rstd, float& a, float& b) {
    float2 sh = both(0.f), shz = both(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float2 f[VEC / 2], g[VEC / 2];
      xin.get(at, i, f);
      gin.get(at, i, g);
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) {
        const float2 c = add2(f[k], both(-mean)), h = mul2(g[k], wf[i][k]);
        aw[i][k] = fma2(mul2(g[k], both(rstd)), c, aw[i][k]);
        ab[i][k] = add2(ab[i][k], g[k]);
        sh = add2(sh, h);
        shz = fma2(h, c, shz);
      }
    }
    a = sh.x + sh.y;
    b = (shz.x + shz.y) * rstd;
  };
  const float *mean_at = mean_in + r, *rstd_at = rstd_in + r;
  float mean = 0.f, rstd = 0.f, next_mean = 0.f, next_rstd = 0.f, a = 0.f, b = 0.f;
  if (r < rows) { mean = __ldg(mean_at); rstd = __ldg(rstd_at); }
  if (r + stride < rows) { next_mean = __ldg(mean_at + stride); next_rstd = __ldg(rstd_at + stride); }
  copies_wait<STAGES - 2>();
  if (r < rows) row_sums(0, mean, rstd, a, b);
  X* out = dx + r * D + j0;
  for (int at = 0, free_at = all - stage_bytes; left > 0; left -= stride, r += stride, out += stride * D) {
    const int next_at = at + stage_bytes < all ? at + stage_bytes : 0;
    copies_wait<STAGES - 3>();
    xin.fetch(free_at, r + (STAGES - 1) * stride < rows);     // to where the last row was
    gin.fetch(free_at, r + (STAGES - 1) * stride < rows);
    copies_commit();
    mean_at += stride;
    rstd_at += stride;
    float after_mean = 0.f, after_rstd = 0.f, next_a = 0.f, next_b = 0.f;
    if (r + 2 * stride < rows) { after_mean = __ldg(mean_at + stride); after_rstd = __ldg(rstd_at + stride); }
    grp.sum2_lanes(a, b);
    if (r + stride < rows) row_sums(next_at, next_mean, next_rstd, next_a, next_b);
    grp.sum2_warps(a, b, buf);
    if (r < rows) {
      // dx = r (h - mean(h) - z mean(h z)) = r h + ((x - mean) A + B)
      const float A = -rstd * rstd * (b * inv_d), B = -rstd * (a * inv_d);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = j0 + i * xin.vec_step();
        if (j < D) {
          float2 f[VEC / 2], g[VEC / 2];
          xin.get(at, i, f);
          gin.get(at, i, g);
#pragma unroll
          for (int k = 0; k < VEC / 2; ++k) f[k] = fma2(mul2(g[k], wf[i][k]), both(rstd), fma2(add2(f[k], both(-mean)), both(A), both(B)));
          if (EDGE) store_at<VEC, decltype(xin)>(out + i * xin.vec_step(), i, j, D, f); else store_vec(out + i * xin.vec_step(), f);
        }
      }
    }
    mean = next_mean; rstd = next_rstd; next_mean = after_mean; next_rstd = after_rstd; a = next_a; b = next_b;
    free_at = at;
    at = next_at;
  }
  copies_wait<0>();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (partial == nullptr) return;
  const int width = static_cast<int>(row_units(D, VEC)) * VEC, vec_step = xin.vec_step();
  float* const part = partial + static_cast<int64_t>(blockIdx.x) * 2 * width;
  if (MODE == BLOCK) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (j0 + i * vec_step < D) {
        float4* const at = reinterpret_cast<float4*>(part + (grp.c * VEC + i * vec_step));
#pragma unroll
        for (int k = 0; k < VEC / 4; ++k) {
          at[k] = make_float4(aw[i][2 * k].x, aw[i][2 * k].y, aw[i][2 * k + 1].x, aw[i][2 * k + 1].y);
          at[width / 4 + k] = make_float4(ab[i][2 * k].x, ab[i][2 * k].y, ab[i][2 * k + 1].x, ab[i][2 * k + 1].y);
        }
      }
    return;
  }
  // The groups of a block have rows of different s where D is no multiple of VEC, so their sums meet by column: the groups of a warp one
  // after the other in shared memory (by shuffles where s is the same for all), the four warps in the end.
  constexpr int WARPS = LN_WARP_THREADS / 32;
  float* const cols = reinterpret_cast<float*>(slots);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr bool same = !EDGE;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
    if (!same) {
      for (int j = lane; j < D; j += 32) cols[warp * D + j] = 0.f;
      __syncwarp();
    }
    for (int g = 0; g < (same ? 1 : 32 / grp.T); ++g) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float2 pair = which ? ab[i][k / 2] : aw[i][k / 2];
          float a = k & 1 ? pair.y : pair.x;
          const int j = j0 + i * vec_step + k;
          if (same) {
            for (int o = 16; o >= grp.T; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
            if (lane < grp.T && j < D) cols[warp * D + j] = a;
          } else if (lane / grp.T == g && j >= 0 && j < D) {
            cols[warp * D + j] += a;
          }
        }
      __syncwarp();
    }
    __syncthreads();
    for (int j = threadIdx.x; j < D; j += LN_WARP_THREADS) {
      float a = cols[j];
#pragma unroll
      for (int k = 1; k < WARPS; ++k) a += cols[k * D + j];
      part[which * width + j] = a;
    }
  }
}

// ================================================================ launchers
static unsigned capped(int64_t want, int64_t cap) { return static_cast<unsigned>(want < cap ? want : cap); }

// How a row of D elements is held: nv vectors of `vec` elements a thread, T threads (lanes of a warp, or a block), or `wide`.  Few threads with
// many vectors: sums over threads and barriers cost more than warps that wait (32768 x 4096 bf16 backward 175 us with 4 vectors a thread, 214 with
// 3, 211 with 2, before the last changes); a fifth vector does not fit the registers (65536 x 1280 backward 152 us instead of 116).
struct RowPlan {
  bool wide = false, block = false;
  int nv = 1, T = 32;
};
// most: threads of a block that a row may take; few: no 3 vectors in part of a warp.
// Within a warp: as few lanes as 4 vectors each allow, which leaves the others to more rows.  Whole vectors want twice the lanes with
// half of them each (bf16 rows of 64 elements, 134 MB: forward 45 us and 60, backward 79 and 95; 256 elements 46 and 48, the same), rows that are
// cut do not (101 elements fp32: 63 us and 49, 89 and 78).  3 vectors stay 3 (384 elements bf16: 49 us in 16 lanes, 62 with 2 vectors in 32; backward
// 75 and 100), but in the forward pass over whole vectors of fp32 (96 elements: 51 us, 47 with 2).
static RowPlan plan_rows(int64_t D, int vec, int most, bool few) {
  RowPlan p;
  const int64_t units = row_units(D, vec);
  if (units <= 32 * 4) {
    p.T = 1;
    while (p.T < 32 && p.T * 4 < units) p.T *= 2;
    p.nv = static_cast<int>((units + p.T - 1) / p.T);
    if (p.T < 32 && (p.nv == 3 ? few : p.nv > 1 && D % vec == 0)) { p.T *= 2; p.nv = p.nv / 2 + (p.nv & 1); }
    return p;
  }
  p.block = true;
  const int64_t by3 = (units + 95) / 96 * 32, by4 = (units + 127) / 128 * 32;
  p.nv = by3 * 3 <= by4 * 4 && by3 <= most ? 3 : 4;                              // what leaves fewer of the threads without work
  const int64_t T = p.nv == 3 ? by3 : by4;
  p.wide = T > most;
  p.T = static_cast<int>(T);
  return p;
}

// Blocks of the row kernels: as many as stay resident (in the backward pass more are slower: 65536 x 1024 bf16 72 us with these, 80 with
// twice and 90 with four times as many).  Where rows do not all start on a 16-byte boundary, a group's rows have to be a multiple of 8 apart.
static unsigned row_blocks(const RowPlan& p, int64_t rows, int64_t D, int vec, int per_sm, int turns) {
  const int64_t groups = p.block ? 1 : LN_WARP_THREADS / p.T, want = (rows + groups - 1) / groups;
  int64_t most = static_cast<int64_t>(per_sm) * sm_count();
  if (turns > 1) most *= want / (4 * most) < 1 ? 1 : imin64(want / (4 * most), turns);
  if (want <= most) return static_cast<unsigned>(want);
  return static_cast<unsigned>(D % vec == 0 ? most : most < 8 ? 8 : most / 8 * 8);
}
// Whether the rows of an input can be copied in vectors: the same distances from a boundary as the output's.
static bool in_vectors(const void* p, int64_t ld, int64_t D, int vec, int64_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (ld - D) % vec == 0;
}

// A kernel on the devices it was used on: its dynamic shared memory is allowed once on each.
struct KernelState {
  std::atomic<uint64_t> allowed{0};
  std::atomic<int> regs{0}, smem{0};      // of a thread; of a block, static
};
template <class K>
static int allow_slots(K kernel, KernelState& state) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (dev < 64 && (state.allowed.load(std::memory_order_acquire) & bit)) return HASTE_OK;
  if (int rc = allow_dynamic_smem(kernel)) return rc;
  cudaFuncAttributes attr;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, kernel);
  if (e != cudaSuccess) return fail(HASTE_ERR_LAUNCH, "layer norm: attributes of a kernel: %s", cudaGetErrorString(e));
  state.regs.store(attr.numRegs, std::memory_order_relaxed);
  state.smem.store(static_cast<int>(attr.sharedSizeBytes), std::memory_order_relaxed);
  if (dev < 64) state.allowed.fetch_or(bit, std::memory_order_release);
  return HASTE_OK;
}
// Blocks that stay resident on a SM: a quarter of its 64 K registers to each scheduler, in units of 8 a thread; 228 KB of shared memory, of
// which a block takes 1 KB more than its own.  One block more has a turn to itself: 131072 x 512 bf16 forward 48 us with the 5 that fit, 65
// with 6; 32768 x 1024 fp32 backward 62 and 74.
static int resident_blocks(const KernelState& state, int threads, int smem) {
  const int regs = (state.regs.load(std::memory_order_relaxed) + 7) / 8 * 8, warps = 16384 / (32 * (regs > 0 ? regs : 8)) * 4;
  const int by_regs = (warps < 64 ? warps : 64) / (threads / 32), by_smem = 228 * 1024 / (smem + state.smem.load(std::memory_order_relaxed) + 1024);
  return by_regs < 1 ? 1 : by_regs < by_smem ? by_regs : by_smem < 1 ? 1 : by_smem;
}

template <class X, class W>
static int ln_fwd_wide(const X* x, const W* w, const W* b, X* y, float* mean, float* rstd, int64_t rows, int64_t D, int64_t ldx, float eps, cudaStream_t st) {
  ln_fwd_wide_kernel<X, W><<<capped(rows, sm_count() * 8), LN_THREADS, 0, st>>>(x, w, b, y, mean, rstd, rows, D, ldx, eps);
  return check_launch("layer_norm_forward");
}

struct FwdCall {
  const void *x, *w, *b;
  void* y;
  float *mean, *rstd;
  int64_t rows, D, ldx;
  float eps;
  int w_type;
  cudaStream_t st;
};

template <class X, int VEC, int NV, int MODE, bool EDGE>
static int ln_fwd_rows(const FwdCall& c, const RowPlan& p) {
  static KernelState state;
  const int threads = MODE == BLOCK ? p.T : LN_WARP_THREADS, smem = LN_STAGES * NV * threads * VEC * static_cast<int>(sizeof(X));
  if (int rc = allow_slots(ln_fwd_kernel<X, VEC, NV, MODE, EDGE>, state)) return rc;
  // Where D is a multiple of VEC and a thread has 3 vectors or more, up to 4 times (fp32: 8 times) as many blocks as stay resident, each with
  // at least 4 rows to a group: started in order they stay closer together in memory than blocks that walk over all of it (65536 x 1024
  // bf16 51 -> 47 us, fp32 99 -> 81).  With fewer vectors, or weights to be loaded one by one, starting up costs more than that.
  const int turns = !EDGE && NV >= 3 ? (sizeof(X) == 2 ? 4 : 8) : 1;
  const unsigned blocks = row_blocks(p, c.rows, c.D, VEC, resident_blocks(state, threads, smem), turns);
  ln_fwd_kernel<X, VEC, NV, MODE, EDGE><<<blocks, threads, smem, c.st>>>((const X*)c.x, c.w, c.b, c.w_type, (X*)c.y, c.mean, c.rstd, c.rows, static_cast<int>(c.D), c.ldx,
                                                                    c.eps, p.T, in_vectors(c.x, c.ldx, c.D, VEC, 16), aligned16(c.w) && aligned16(c.b));
  return check_launch("layer_norm_forward");
}

template <class X, int VEC, bool EDGE>
static int ln_fwd_plan(const FwdCall& c, const RowPlan& p) {
  if (p.block) return p.nv == 3 ? ln_fwd_rows<X, VEC, 3, BLOCK, EDGE>(c, p) : ln_fwd_rows<X, VEC, 4, BLOCK, EDGE>(c, p);
  if (p.nv == 1) return ln_fwd_rows<X, VEC, 1, SUB, EDGE>(c, p);
  if (p.nv == 2) return ln_fwd_rows<X, VEC, 2, SUB, EDGE>(c, p);
  if (p.T < 32) {                       // (whole vectors: 3 only of 8 elements, and never 4)
    if constexpr (EDGE) return p.nv == 3 ? ln_fwd_rows<X, VEC, 3, SUB, EDGE>(c, p) : ln_fwd_rows<X, VEC, 4, SUB, EDGE>(c, p);
    else if constexpr (VEC == 8) return ln_fwd_rows<X, VEC, 3, SUB, EDGE>(c, p);
  }
  if (p.nv == 3) return ln_fwd_rows<X, VEC, 3, FULL, EDGE>(c, p);
  return ln_fwd_rows<X, VEC, 4, FULL, EDGE>(c, p);
}

template <class X>
static int ln_fwd(const FwdCall& c) {
  if (c.rows == 0) return HASTE_OK;
  constexpr int VEC = 16 / sizeof(X);
  RowPlan p = plan_rows(c.D, VEC, 512, VEC == 4 && c.D % VEC == 0);
  if (!aligned16(c.y)) p.wide = true;
  if (p.wide) {
    using B = __nv_bfloat16;
    if (c.w_type == HASTE_BF16) return ln_fwd_wide((const X*)c.x, (const B*)c.w, (const B*)c.b, (X*)c.y, c.mean, c.rstd, c.rows, c.D, c.ldx, c.eps, c.st);
    return ln_fwd_wide((const X*)c.x, (const float*)c.w, (const float*)c.b, (X*)c.y, c.mean, c.rstd, c.rows, c.D, c.ldx, c.eps, c.st);
  }
  return c.D % VEC ? ln_fwd_plan<X, VEC, true>(c, p) : ln_fwd_plan<X, VEC, false>(c, p);
}

int launch_layer_norm_forward(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows, int64_t D, int64_t ldx,
                              float eps, int x_type, int w_type, cudaStream_t st) {
  const FwdCall c{x, w, b, y, mean, rstd, rows, D, ldx, eps, w_type, st};
  return x_type == HASTE_BF16 ? ln_fwd<__nv_bfloat16>(c) : ln_fwd<float>(c);
}

// Blocks a SM of the backward pass, each of which leaves a part of dw and db in the scratch, with `per_thread` elements to a thread: at most
// this many, whatever registers and shared memory would allow.
static int bwd_most_blocks(const RowPlan& p, int per_thread) {
  const int threads = p.block ? p.T : LN_WARP_THREADS, most = (per_thread > 16 ? 384 : per_thread > 8 ? 512 : 1024) / threads;
  return most < 1 ? 1 : most < 8 ? most : 8;
}
// Threads of a block that a row may take there: with 8 elements a vector, more would leave too few registers.
constexpr int bwd_most(int vec) { return vec == 8 ? 256 : 512; }

// Parts of dw and db: as many as blocks; of the wide rows' kernel, as many as it makes ranges of rows.
static int64_t wide_parts(int64_t rows) { return rows < 16 * 64 ? (rows + 63) / 64 : 16; }

int64_t layer_norm_backward_scratch(int64_t rows, int64_t D) {
  int64_t most = wide_parts(rows) * D;
  for (int vec = 4; vec <= 8; vec += 4) {              // fp32 and bf16 rows
    const RowPlan p = plan_rows(D, vec, bwd_most(vec), false);
    if (!p.wide && rows > 0) {
      const int64_t n = row_blocks(p, rows, D, vec, bwd_most_blocks(p, vec * p.nv), 1);
      const int64_t elements = n * row_units(D, vec) * vec;
      if (elements > most) most = elements;
    }
  }
  return most * 2;
}

template <class X, class G, class W>
static int ln_bwd_wide(const G* dy, const X* x, const W* w, const float* mean, const float* rstd, X* dx, float* partial, int64_t rows, int64_t D, int64_t lddy,
                       int64_t ldx, cudaStream_t st) {
  ln_bwd_dx_wide_kernel<X, G, W><<<capped(rows, sm_count() * 8), LN_THREADS, 0, st>>>(dy, x, w, mean, rstd, dx, rows, D, lddy, ldx);
  if (partial != nullptr) {
    const dim3 grid(capped((D + 31) / 32, 65535), static_cast<unsigned>(wide_parts(rows)));
    ln_bwd_columns_kernel<X, G><<<grid, LN_THREADS, 0, st>>>(dy, x, mean, rstd, partial, rows, D, lddy, ldx);
  }
  return check_launch("layer_norm_backward");
}

struct BwdCall {
  const void *dy, *x, *w;
  const float *mean, *rstd;
  void *dx, *dw, *db;
  float* scratch;
  int64_t rows, D, lddy, ldx;
  int w_type;
  cudaStream_t st;
};

template <class X, class G, int VEC, int NV, int MODE, bool EDGE, int STAGES = 4>
static int ln_bwd_rows(const BwdCall& c, const RowPlan& p, float* partial, Parts& parts) {
  static KernelState state;
  const int threads = MODE == BLOCK ? p.T : LN_WARP_THREADS;
  if constexpr (MODE == BLOCK && STAGES == 4 && VEC * sizeof(G) == 16)          // fp32 rows of more than 6144 elements: 4 stages do not fit
    if (STAGES * NV * threads * VEC * static_cast<int>(sizeof(X) + sizeof(G)) > DYN_SMEM_MAX) return ln_bwd_rows<X, G, VEC, NV, MODE, EDGE, 3>(c, p, partial, parts);
  const int slots = STAGES * NV * threads * VEC * static_cast<int>(sizeof(X) + sizeof(G));
  const int cols = MODE == BLOCK ? 0 : LN_WARP_THREADS / 32 * static_cast<int>(c.D) * 4, smem = slots > cols ? slots : cols;
  if (int rc = allow_slots(ln_bwd_kernel<X, G, VEC, NV, MODE, EDGE, STAGES>, state)) return rc;
  const int per_sm = resident_blocks(state, threads, smem), most = bwd_most_blocks(p, VEC * NV);
  const unsigned blocks = row_blocks(p, c.rows, c.D, VEC, per_sm < most ? per_sm : most, 1);
  parts = Parts{static_cast<int>(blocks), row_units(c.D, VEC) * VEC, static_cast<unsigned>(c.D), MODE == BLOCK && EDGE ? VEC - 1 : 0u};
  const int64_t g_bytes = VEC * sizeof(G) < 16 ? 8 : 16;
  ln_bwd_kernel<X, G, VEC, NV, MODE, EDGE, STAGES><<<blocks, threads, smem, c.st>>>((const G*)c.dy, (const X*)c.x, c.w, c.w_type, c.mean, c.rstd, (X*)c.dx, partial, c.rows,
                                                                      static_cast<int>(c.D), c.lddy, c.ldx, p.T, in_vectors(c.x, c.ldx, c.D, VEC, 16),
                                                                      in_vectors(c.dy, c.lddy, c.D, VEC, g_bytes), aligned16(c.w));
  return check_launch("layer_norm_backward");
}

template <class X, class G, int VEC, bool EDGE>
static int ln_bwd_plan(const BwdCall& c, const RowPlan& p, float* partial, Parts& parts) {
  if (p.block) return p.nv == 3 ? ln_bwd_rows<X, G, VEC, 3, BLOCK, EDGE>(c, p, partial, parts) : ln_bwd_rows<X, G, VEC, 4, BLOCK, EDGE>(c, p, partial, parts);
  if (p.nv == 1) return ln_bwd_rows<X, G, VEC, 1, SUB, EDGE>(c, p, partial, parts);
  if (p.nv == 2) return ln_bwd_rows<X, G, VEC, 2, SUB, EDGE>(c, p, partial, parts);
  if (p.T < 32) {                       // (whole vectors: never 4)
    if constexpr (EDGE) return p.nv == 3 ? ln_bwd_rows<X, G, VEC, 3, SUB, EDGE>(c, p, partial, parts) : ln_bwd_rows<X, G, VEC, 4, SUB, EDGE>(c, p, partial, parts);
    else return ln_bwd_rows<X, G, VEC, 3, SUB, EDGE>(c, p, partial, parts);
  }
  if (p.nv == 3) return ln_bwd_rows<X, G, VEC, 3, FULL, EDGE>(c, p, partial, parts);
  return ln_bwd_rows<X, G, VEC, 4, FULL, EDGE>(c, p, partial, parts);
}

// Four blocks to 32 columns where there are many parts and few columns: 888 parts of 1021 columns 6.3 us by one, 4.7 by four; 444 of 4096
// 5.3 and 9.0.
template <class W>
static int ln_finish(const BwdCall& c, const Parts& parts, W* dw, W* db) {
  const unsigned grid = static_cast<unsigned>((2 * c.D + 31) / 32);
  if (parts.count >= 256 && grid <= 128)
    return launch_behind(ln_bwd_finish_many_kernel<W>, grid * LN_FINISH_CLUSTER, LN_FINISH_THREADS, c.st, static_cast<const float*>(c.scratch), parts, c.D, dw, db);
  if (c.rows == 0) {                    // no kernel of this call comes before
    ln_bwd_finish_kernel<W><<<grid, LN_FINISH_THREADS, 0, c.st>>>(c.scratch, parts, c.D, dw, db);
    return check_launch("layer_norm_backward");
  }
  return launch_behind(ln_bwd_finish_kernel<W>, grid, LN_FINISH_THREADS, c.st, static_cast<const float*>(c.scratch), parts, c.D, dw, db);
}

template <class X, class G>
static int ln_bwd(const BwdCall& c) {
  constexpr int VEC = 16 / sizeof(X);
  using B = __nv_bfloat16;
  const bool want = c.dw != nullptr || c.db != nullptr;
  float* partial = want ? c.scratch : nullptr;
  Parts parts{0, c.D, 0u, 0u};
  if (c.rows > 0) {
    RowPlan p = plan_rows(c.D, VEC, bwd_most(VEC), false);
    if (!aligned16(c.dx)) p.wide = true;
    int rc = HASTE_OK;
    if (p.wide) {
      parts.count = static_cast<int>(wide_parts(c.rows));
      rc = c.w_type == HASTE_BF16 ? ln_bwd_wide((const G*)c.dy, (const X*)c.x, (const B*)c.w, c.mean, c.rstd, (X*)c.dx, partial, c.rows, c.D, c.lddy, c.ldx, c.st)
                                  : ln_bwd_wide((const G*)c.dy, (const X*)c.x, (const float*)c.w, c.mean, c.rstd, (X*)c.dx, partial, c.rows, c.D, c.lddy, c.ldx, c.st);
    } else {
      rc = c.D % VEC ? ln_bwd_plan<X, G, VEC, true>(c, p, partial, parts) : ln_bwd_plan<X, G, VEC, false>(c, p, partial, parts);
    }
    if (rc != HASTE_OK) return rc;
  }
  if (want) {
    return c.w_type == HASTE_BF16 ? ln_finish(c, parts, (B*)c.dw, (B*)c.db) : ln_finish(c, parts, (float*)c.dw, (float*)c.db);
  }
  return check_launch("layer_norm_backward");
}

int launch_layer_norm_backward(const void* dy, const void* x, const void* w, const float* mean, const float* rstd, void* dx, void* dw, void* db,
                               float* scratch, int64_t rows, int64_t D, int64_t lddy, int64_t ldx, int x_type, int dy_type, int w_type, cudaStream_t st) {
  using B = __nv_bfloat16;
  const BwdCall c{dy, x, w, mean, rstd, dx, dw, db, scratch, rows, D, lddy, ldx, w_type, st};
  if (x_type == HASTE_BF16) return dy_type == HASTE_BF16 ? ln_bwd<B, B>(c) : ln_bwd<B, float>(c);
  return dy_type == HASTE_BF16 ? ln_bwd<float, B>(c) : ln_bwd<float, float>(c);
}

}  // namespace haste
