// Layer norm over the last dimension, forward and backward.
//
//   mean = sum(x) / D     var = sum((x - mean)^2) / D     r = 1 / sqrt(var + eps)     z = (x - mean) r
//   y  = z w + b
//   h  = dy w             dx = r (h - mean(h) - z mean(h z))     dw = sum_rows dy z     db = sum_rows dy
//
// All sums are fp32; the variance is taken around the mean, not from the sum of squares, which cancels for rows whose mean is large
// against their spread.  Inputs and outputs are bf16 or fp32, rounded once (nearest even) when stored.
//
// Memory bounds all of it: x in and y out, or dy and x in and dx out.  A row is read once and stays in registers: a group of 1 to 32
// lanes of a warp has it, or a thread block where it is wider, each thread up to 4 vectors of 16 bytes (16 single elements where rows
// do not start on 16 bytes).  Groups walk over the rows with the next row's loads in flight, so that in the backward pass a thread owns
// its columns for good and sums dw and db in registers; the blocks' sums go to memory and are added in a second, small launch.
#include "common.cuh"

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

constexpr int LN_THREADS = 256;

// ---------------------------------------------------------------- rows of any width: one block a row, the row read again for each pass
template <class X, class W>
__global__ void __launch_bounds__(LN_THREADS) ln_fwd_wide_kernel(const X* __restrict__ x, const W* __restrict__ w, const W* __restrict__ b, X* __restrict__ y,
                                                                 float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows, int64_t D,
                                                                 int64_t ldx, float eps) {
  __shared__ float buf[LN_THREADS / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const X* xr = x + r * ldx;
    float s = 0.f;
    for (int64_t j = threadIdx.x; j < D; j += LN_THREADS) s += ld_f(xr + j);
    const float mean = block_sum(s, buf) / static_cast<float>(D);
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

// dw and db from the partial sums, added in the order of the parts: the same bits every time.
constexpr int LN_FINISH_THREADS = 512;
template <class W>
__global__ void __launch_bounds__(LN_FINISH_THREADS) ln_bwd_finish_kernel(const float* __restrict__ partial, int parts, int64_t D, W* __restrict__ dw,
                                                                         W* __restrict__ db) {
  constexpr int SPLIT = LN_FINISH_THREADS / 32;
  __shared__ float buf[SPLIT][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + tx;      // column of the [2 D] row of one part
  float s = 0.f;
  if (c < 2 * D) {
#pragma unroll 8
    for (int p = ty; p < parts; p += SPLIT) s += partial[static_cast<int64_t>(p) * 2 * D + c];
  }
  buf[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < 2 * D) {
#pragma unroll
    for (int i = 1; i < SPLIT; ++i) s += buf[i][tx];
    if (c < D) { if (dw) st_f(dw + c, s); }
    else if (db) st_f(db + (c - D), s);
  }
}

// ---------------------------------------------------------------- rows that stay in registers
// VEC elements of type T as they lie in memory (a single element: as fp32).
template <class T, int VEC> struct Raw;
template <> struct Raw<__nv_bfloat16, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void clear() { v = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
  }
};
template <> struct Raw<__nv_bfloat16, 4> {
  uint2 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __ldcs(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ void clear() { v = make_uint2(0u, 0u); }
  __device__ __forceinline__ void get(float (&f)[4]) const {
    f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xFFFF0000u); f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xFFFF0000u);
  }
};
template <int VEC> struct Raw<float, VEC> {
  float4 v[VEC / 4];
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) v[i] = __ldcs(reinterpret_cast<const float4*>(p) + i);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void get(float (&f)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) { f[4 * i] = v[i].x; f[4 * i + 1] = v[i].y; f[4 * i + 2] = v[i].z; f[4 * i + 3] = v[i].w; }
  }
};
template <> struct Raw<float, 1> {
  float v;
  __device__ __forceinline__ void load(const float* p) { v = __ldcs(p); }
  __device__ __forceinline__ void clear() { v = 0.f; }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = v; }
};
template <> struct Raw<__nv_bfloat16, 1> {
  float v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __bfloat162float(__ldcs(p)); }
  __device__ __forceinline__ void clear() { v = 0.f; }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = v; }
};

__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
}
__device__ __forceinline__ void store_vec(float* p, const float (&f)[4]) { __stcs(reinterpret_cast<float4*>(p), make_float4(f[0], f[1], f[2], f[3])); }
template <class T>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[1]) { st_f(p, f[0]); }

// Weights j .. j+VEC-1: hot in L1 (x and dy go past it), so they are read for every row rather than held in registers.
template <int VEC>
__device__ __forceinline__ void load_weights(const void* w, int w_type, int64_t j, float fill, float (&f)[VEC]) {
  if (w == nullptr) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = fill;
  } else if (w_type == HASTE_BF16) {
    const uint16_t* p = static_cast<const uint16_t*>(w) + j;
    if constexpr (VEC == 8) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(u[i] << 16); f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u); }
    } else if constexpr (VEC == 4) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
      f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xFFFF0000u); f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xFFFF0000u);
    } else {
      f[0] = bf16_bits_to_float(__ldg(p));
    }
  } else {
    const float* p = static_cast<const float*>(w) + j;
    if constexpr (VEC >= 4) {
#pragma unroll
      for (int i = 0; i < VEC / 4; ++i) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p) + i);
        f[4 * i] = v.x; f[4 * i + 1] = v.y; f[4 * i + 2] = v.z; f[4 * i + 3] = v.w;
      }
    } else {
      f[0] = __ldg(p);
    }
  }
}

// The threads that share a row: T lanes of a warp (a power of two), or the block.
template <bool BLOCK>
struct RowGroup {
  int T, c;              // threads of the group, this thread's place among them
  int slot = 0;          // buffer of the next sum over a block: a buffer is written again two sums (two barriers) later
  __device__ explicit RowGroup(int t) : T(BLOCK ? static_cast<int>(blockDim.x) : t), c(static_cast<int>(threadIdx.x) & (BLOCK ? 0x7FFFFFFF : t - 1)) {}
  // rows of a warp (of a block) are neighbours; first: that of its first group
  __device__ int64_t first_row() const { return BLOCK ? blockIdx.x : (static_cast<int64_t>(blockIdx.x) * blockDim.x + (threadIdx.x & ~31u)) / T; }
  __device__ int64_t stride() const { return BLOCK ? gridDim.x : static_cast<int64_t>(gridDim.x) * blockDim.x / T; }
  __device__ int64_t own() const { return BLOCK ? 0 : static_cast<int64_t>((threadIdx.x & 31u) / T); }
  template <int N>
  __device__ __forceinline__ void sum(float (&v)[N], float (*buf)[N][16]) {
    if (BLOCK) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
      if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int k = 0; k < N; ++k) buf[slot][k][threadIdx.x >> 5] = v[k];
      __syncthreads();
      const int warps = blockDim.x >> 5;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        v[k] = buf[slot][k][0];
        for (int i = 1; i < warps; ++i) v[k] += buf[slot][k][i];
      }
      slot ^= 1;
    } else {
      for (int o = T >> 1; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    }
  }
};

constexpr int LN_WARP_THREADS = 128;      // block of the variant whose groups are within a warp

template <class X, int VEC, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : LN_WARP_THREADS) ln_fwd_kernel(const X* __restrict__ x, const void* __restrict__ w, const void* __restrict__ b,
                                                                              int w_type, X* __restrict__ y, float* __restrict__ mean_out,
                                                                              float* __restrict__ rstd_out, int64_t rows, int D, int64_t ldx, float eps, int t) {
  __shared__ float buf[2][1][16];
  RowGroup<BLOCK> grp(t);
  const float inv_d = 1.f / static_cast<float>(D);
  Raw<X, VEC> cur[NV], nxt[NV];
  auto fetch = [&](int64_t r, Raw<X, VEC> (&v)[NV]) {
    const X* xr = x + r * ldx;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (grp.c + i * grp.T) * VEC;
      if (r < rows && j < D) v[i].load(xr + j); else v[i].clear();
    }
  };
  int64_t r0 = grp.first_row();
  fetch(r0 + grp.own(), cur);
  for (; r0 < rows; r0 += grp.stride()) {
    const int64_t r = r0 + grp.own();
    fetch(r + grp.stride(), nxt);
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[VEC];
      cur[i].get(f);
#pragma unroll
      for (int k = 0; k < VEC; ++k) s[0] += f[k];
    }
    grp.sum(s, buf);
    const float mean = s[0] * inv_d;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[VEC];
      cur[i].get(f);
      const bool in = (grp.c + i * grp.T) * VEC < D;
#pragma unroll
      for (int k = 0; k < VEC; ++k) { const float d = f[k] - mean; if (in) s[0] = fmaf(d, d, s[0]); }
    }
    grp.sum(s, buf);
    const float rstd = 1.f / sqrtf(fmaf(s[0], inv_d, eps));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (grp.c + i * grp.T) * VEC;
      if (r < rows && j < D) {
        float f[VEC], wf[VEC], bf[VEC];
        cur[i].get(f);
        load_weights<VEC>(w, w_type, j, 1.f, wf);
        load_weights<VEC>(b, w_type, j, 0.f, bf);
#pragma unroll
        for (int k = 0; k < VEC; ++k) f[k] = fmaf((f[k] - mean) * rstd, wf[k], bf[k]);
        store_vec(y + r * D + j, f);
      }
    }
    if (grp.c == 0 && r < rows && mean_out != nullptr) { mean_out[r] = mean; rstd_out[r] = rstd; }
#pragma unroll
    for (int i = 0; i < NV; ++i) cur[i] = nxt[i];
  }
}

// dx, and the block's part of dw and db: partial[block][0][.] and [1][.] (NULL: only dx is wanted).
template <class X, class G, int VEC, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? (VEC * NV > 16 ? 256 : 512) : LN_WARP_THREADS)
    ln_bwd_kernel(const G* __restrict__ dy, const X* __restrict__ x, const void* __restrict__ w, int w_type, const float* __restrict__ mean_in,
                  const float* __restrict__ rstd_in, X* __restrict__ dx, float* __restrict__ partial, int64_t rows, int D, int64_t lddy, int64_t ldx, int t) {
  __shared__ float buf[2][2][16];
  RowGroup<BLOCK> grp(t);
  const float inv_d = 1.f / static_cast<float>(D);
  float aw[NV][VEC], ab[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < VEC; ++k) aw[i][k] = ab[i][k] = 0.f;
  Raw<X, VEC> cx[NV], nx[NV];
  Raw<G, VEC> cg[NV], ng[NV];
  float cmean, crstd, nmean, nrstd;
  auto fetch = [&](int64_t r, Raw<X, VEC> (&xv)[NV], Raw<G, VEC> (&gv)[NV], float& mean, float& rstd) {
    const X* xr = x + r * ldx;
    const G* gr = dy + r * lddy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (grp.c + i * grp.T) * VEC;
      if (r < rows && j < D) { xv[i].load(xr + j); gv[i].load(gr + j); } else { xv[i].clear(); gv[i].clear(); }
    }
    mean = r < rows ? __ldg(mean_in + r) : 0.f;
    rstd = r < rows ? __ldg(rstd_in + r) : 0.f;
  };
  int64_t r0 = grp.first_row();
  fetch(r0 + grp.own(), cx, cg, cmean, crstd);
  for (; r0 < rows; r0 += grp.stride()) {
    const int64_t r = r0 + grp.own();
    fetch(r + grp.stride(), nx, ng, nmean, nrstd);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (grp.c + i * grp.T) * VEC;
      if (j < D) {
        float f[VEC], g[VEC], wf[VEC];
        cx[i].get(f);
        cg[i].get(g);
        load_weights<VEC>(w, w_type, j, 1.f, wf);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float z = (f[k] - cmean) * crstd, h = g[k] * wf[k];
          aw[i][k] = fmaf(g[k], z, aw[i][k]);
          ab[i][k] += g[k];
          s[0] += h;
          s[1] = fmaf(h, z, s[1]);
        }
      }
    }
    grp.sum(s, buf);
    const float mh = s[0] * inv_d, mhz = s[1] * inv_d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (grp.c + i * grp.T) * VEC;
      if (r < rows && j < D) {
        float f[VEC], g[VEC], wf[VEC];
        cx[i].get(f);
        cg[i].get(g);
        load_weights<VEC>(w, w_type, j, 1.f, wf);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float z = (f[k] - cmean) * crstd;
          f[k] = crstd * (fmaf(g[k], wf[k], -mh) - z * mhz);
        }
        store_vec(dx + r * D + j, f);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) { cx[i] = nx[i]; cg[i] = ng[i]; }
    cmean = nmean; crstd = nrstd;
  }
  if (partial == nullptr) return;
  float* out = partial + static_cast<int64_t>(blockIdx.x) * 2 * D;
  if (BLOCK) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (grp.c + i * grp.T) * VEC;
      if (j < D)
#pragma unroll
        for (int k = 0; k < VEC; ++k) { out[j + k] = aw[i][k]; out[D + j + k] = ab[i][k]; }
    }
    return;
  }
  // the groups of a warp by shuffles, its four warps through shared memory
  constexpr int WARPS = LN_WARP_THREADS / 32;
  __shared__ float cols[WARPS][32 * NV * VEC];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        float a = which ? ab[i][k] : aw[i][k];
        for (int o = 16; o >= grp.T; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        const int j = (grp.c + i * grp.T) * VEC + k;
        if ((threadIdx.x & 31) < grp.T && j < D) cols[threadIdx.x >> 5][j] = a;
      }
    __syncthreads();
    for (int j = threadIdx.x; j < D; j += LN_WARP_THREADS) {
      float a = cols[0][j];
#pragma unroll
      for (int k = 1; k < WARPS; ++k) a += cols[k][j];
      out[which * D + j] = a;
    }
    __syncthreads();
  }
}

// ================================================================ launchers
static int sm_count() {
  static std::atomic<int> cached[64];              // of each device, 0 = not asked yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int sms = cached[dev].load(std::memory_order_relaxed);
  if (sms == 0) {
    sms = 148;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    cached[dev].store(sms, std::memory_order_relaxed);
  }
  return sms;
}
static unsigned capped(int64_t want, int64_t cap) { return static_cast<unsigned>(want < cap ? want : cap); }

// How a row of D elements is held: vec elements a vector, nv vectors a thread, T threads (within a warp, or a block), or `wide`.
struct RowPlan {
  bool wide = false, block = false;
  int vec = 1, nv = 1, T = 32;
};
// most: threads of a block that a row may take
static RowPlan plan_rows(int64_t D, int vec, bool aligned, int most_vec, int most_single) {
  RowPlan p;
  p.vec = aligned ? vec : 1;
  const int64_t units = (D + p.vec - 1) / p.vec;      // vectors of a row
  const int per_thread = aligned ? 4 : 16;
  if (units <= 32 * per_thread) {
    // the fewest threads: a group of few lanes leaves the others to more rows
    p.T = 1;
    while (p.T < 32 && p.T * (aligned ? 2 : 4) < units) p.T *= 2;
    const int64_t need = (units + p.T - 1) / p.T;
    p.nv = aligned ? static_cast<int>(need) : need <= 1 ? 1 : need <= 4 ? 4 : 16;
    return p;
  }
  p.block = true;
  p.nv = per_thread;
  const int64_t T = (units + 32 * per_thread - 1) / (32 * per_thread) * 32;
  if (T > (aligned ? most_vec : most_single)) p.wide = true;
  p.T = static_cast<int>(T);
  return p;
}
static bool on(const void* p, int64_t ld_bytes, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld_bytes % bytes == 0; }

// Blocks of the row kernels: as many as stay resident (registers allow about 3 to 4 blocks of 128 threads with 24 to 32 elements a
// thread and twice that with fewer), since each of them leaves a part of dw and db.
static unsigned row_blocks(const RowPlan& p, int64_t rows, int resident_threads) {
  const int64_t groups = p.block ? 1 : LN_WARP_THREADS / p.T, threads = p.block ? p.T : LN_WARP_THREADS;
  const int64_t want = (rows + groups - 1) / groups, per_sm = resident_threads / threads < 1 ? 1 : resident_threads / threads;
  return capped(want < 1 ? 1 : want, per_sm * sm_count());
}

template <class X, class W>
static int ln_fwd_wide(const X* x, const W* w, const W* b, X* y, float* mean, float* rstd, int64_t rows, int64_t D, int64_t ldx, float eps, cudaStream_t st) {
  ln_fwd_wide_kernel<X, W><<<capped(rows, sm_count() * 8), LN_THREADS, 0, st>>>(x, w, b, y, mean, rstd, rows, D, ldx, eps);
  return check_launch("layer_norm_forward");
}

template <class X>
static int ln_fwd(const X* x, const void* w, const void* b, X* y, float* mean, float* rstd, int64_t rows, int64_t D, int64_t ldx, float eps, int w_type,
                  cudaStream_t st) {
  if (rows == 0) return HASTE_OK;
  constexpr int VEC = 16 / sizeof(X);
  const int64_t w_bytes = w_type == HASTE_BF16 && VEC == 4 ? 8 : 16;
  const bool aligned = D % VEC == 0 && on(x, ldx * sizeof(X), 16) && on(y, 0, 16) && on(w, 0, w_bytes) && on(b, 0, w_bytes);
  const RowPlan p = plan_rows(D, VEC, aligned, 512, 512);
  if (p.wide) {
    if (w_type == HASTE_BF16) return ln_fwd_wide(x, (const __nv_bfloat16*)w, (const __nv_bfloat16*)b, y, mean, rstd, rows, D, ldx, eps, st);
    return ln_fwd_wide(x, (const float*)w, (const float*)b, y, mean, rstd, rows, D, ldx, eps, st);
  }
  const unsigned blocks = row_blocks(p, rows, 1024), threads = p.block ? p.T : LN_WARP_THREADS;
#define HASTE_LN_FWD(V, NV, BLOCK) \
  ln_fwd_kernel<X, V, NV, BLOCK><<<blocks, threads, 0, st>>>(x, w, b, w_type, y, mean, rstd, rows, static_cast<int>(D), ldx, eps, p.T)
  if (aligned) {
    if (p.block) HASTE_LN_FWD(VEC, 4, true);
    else if (p.nv == 1) HASTE_LN_FWD(VEC, 1, false);
    else if (p.nv == 2) HASTE_LN_FWD(VEC, 2, false);
    else if (p.nv == 3) HASTE_LN_FWD(VEC, 3, false);
    else HASTE_LN_FWD(VEC, 4, false);
  } else {
    if (p.block) HASTE_LN_FWD(1, 16, true);
    else if (p.nv == 1) HASTE_LN_FWD(1, 1, false);
    else if (p.nv == 4) HASTE_LN_FWD(1, 4, false);
    else HASTE_LN_FWD(1, 16, false);
  }
#undef HASTE_LN_FWD
  return check_launch("layer_norm_forward");
}

int launch_layer_norm_forward(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows, int64_t D, int64_t ldx,
                              float eps, int x_type, int w_type, cudaStream_t st) {
  using B = __nv_bfloat16;
  if (x_type == HASTE_BF16) return ln_fwd((const B*)x, w, b, (B*)y, mean, rstd, rows, D, ldx, eps, w_type, st);
  return ln_fwd((const float*)x, w, b, (float*)y, mean, rstd, rows, D, ldx, eps, w_type, st);
}

// Parts of dw and db that the wide rows' kernel makes; the others make at most MAX_PARTS (one per block).
static int64_t wide_parts(int64_t rows) { return rows < 16 * 64 ? (rows + 63) / 64 : 16; }
static int64_t max_parts() { return static_cast<int64_t>(sm_count()) * 8; }

int64_t layer_norm_backward_scratch(int64_t rows, int64_t D) {
  const int64_t parts = rows < max_parts() ? rows : max_parts();
  return (D > 8192 ? wide_parts(rows) : parts) * 2 * D;
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

template <class X, class G>
static int ln_bwd(const G* dy, const X* x, const void* w, const float* mean, const float* rstd, X* dx, void* dw, void* db, float* scratch, int64_t rows,
                  int64_t D, int64_t lddy, int64_t ldx, int w_type, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(X);
  const bool want = dw != nullptr || db != nullptr;
  float* partial = want ? scratch : nullptr;
  unsigned parts = 0;
  if (rows > 0) {
    const int64_t w_bytes = w_type == HASTE_BF16 && VEC == 4 ? 8 : 16, g_bytes = VEC * sizeof(G) < 16 ? 8 : 16;
    const bool aligned = D % VEC == 0 && on(x, ldx * sizeof(X), 16) && on(dx, 0, 16) && on(dy, lddy * sizeof(G), g_bytes) && on(w, 0, w_bytes);
    const RowPlan p = plan_rows(D, VEC, aligned, VEC == 8 ? 256 : 512, 512);
    if (p.wide) {
      parts = static_cast<unsigned>(wide_parts(rows));
      const int rc = w_type == HASTE_BF16 ? ln_bwd_wide(dy, x, (const __nv_bfloat16*)w, mean, rstd, dx, partial, rows, D, lddy, ldx, st)
                                          : ln_bwd_wide(dy, x, (const float*)w, mean, rstd, dx, partial, rows, D, lddy, ldx, st);
      if (rc != HASTE_OK) return rc;
    } else {
      parts = row_blocks(p, rows, p.vec * p.nv > 16 ? 384 : p.vec * p.nv > 8 ? 512 : 1024);
      const unsigned threads = p.block ? p.T : LN_WARP_THREADS;
#define HASTE_LN_BWD(V, NV, BLOCK) \
  ln_bwd_kernel<X, G, V, NV, BLOCK><<<parts, threads, 0, st>>>(dy, x, w, w_type, mean, rstd, dx, partial, rows, static_cast<int>(D), lddy, ldx, p.T)
      if (aligned) {
        if (p.block) HASTE_LN_BWD(VEC, 4, true);
        else if (p.nv == 1) HASTE_LN_BWD(VEC, 1, false);
        else if (p.nv == 2) HASTE_LN_BWD(VEC, 2, false);
        else if (p.nv == 3) HASTE_LN_BWD(VEC, 3, false);
        else HASTE_LN_BWD(VEC, 4, false);
      } else {
        if (p.block) HASTE_LN_BWD(1, 16, true);
        else if (p.nv == 1) HASTE_LN_BWD(1, 1, false);
        else if (p.nv == 4) HASTE_LN_BWD(1, 4, false);
        else HASTE_LN_BWD(1, 16, false);
      }
#undef HASTE_LN_BWD
    }
  }
  if (want) {
    const unsigned grid = static_cast<unsigned>((2 * D + 31) / 32);
    if (w_type == HASTE_BF16) ln_bwd_finish_kernel<<<grid, LN_FINISH_THREADS, 0, st>>>(scratch, static_cast<int>(parts), D, (__nv_bfloat16*)dw, (__nv_bfloat16*)db);
    else ln_bwd_finish_kernel<<<grid, LN_FINISH_THREADS, 0, st>>>(scratch, static_cast<int>(parts), D, (float*)dw, (float*)db);
  }
  return check_launch("layer_norm_backward");
}

int launch_layer_norm_backward(const void* dy, const void* x, const void* w, const float* mean, const float* rstd, void* dx, void* dw, void* db,
                               float* scratch, int64_t rows, int64_t D, int64_t lddy, int64_t ldx, int x_type, int dy_type, int w_type, cudaStream_t st) {
  using B = __nv_bfloat16;
  using F = float;
  if (x_type == HASTE_BF16) {
    if (dy_type == HASTE_BF16) return ln_bwd((const B*)dy, (const B*)x, w, mean, rstd, (B*)dx, dw, db, scratch, rows, D, lddy, ldx, w_type, st);
    return ln_bwd((const F*)dy, (const B*)x, w, mean, rstd, (B*)dx, dw, db, scratch, rows, D, lddy, ldx, w_type, st);
  }
  if (dy_type == HASTE_BF16) return ln_bwd((const B*)dy, (const F*)x, w, mean, rstd, (F*)dx, dw, db, scratch, rows, D, lddy, ldx, w_type, st);
  return ln_bwd((const F*)dy, (const F*)x, w, mean, rstd, (F*)dx, dw, db, scratch, rows, D, lddy, ldx, w_type, st);
}

}  // namespace haste
