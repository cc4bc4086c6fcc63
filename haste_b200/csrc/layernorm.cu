// Layer norm over the last dimension, forward and backward.
//
//   mean = sum(x) / D     var = sum((x - mean)^2) / D     r = 1 / sqrt(var + eps)     z = (x - mean) r
//   y  = z w + b
//   h  = dy w             dx = r (h - mean(h) - z mean(h z))     dw = sum_rows dy z     db = sum_rows dy
//
// All sums are fp32; the variance is taken around the mean, not from the sum of squares, which cancels for rows whose mean is large
// against their spread.  Inputs and outputs are bf16 or fp32, rounded once (nearest even) when stored.
#include "common.cuh"
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
template <class W>
__global__ void __launch_bounds__(LN_THREADS) ln_bwd_finish_kernel(const float* __restrict__ partial, int parts, int64_t D, W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float buf[8][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + tx;      // column of the [2 D] row of one part
  float s = 0.f;
  if (c < 2 * D)
    for (int p = ty; p < parts; p += 8) s += partial[static_cast<int64_t>(p) * 2 * D + c];
  buf[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < 2 * D) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += buf[i][tx];
    if (c < D) { if (dw) st_f(dw + c, s); }
    else if (db) st_f(db + (c - D), s);
  }
}

// ================================================================ launchers
static int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}
static unsigned capped(int64_t want, int64_t cap) { return static_cast<unsigned>(want < cap ? want : cap); }

template <class X, class W>
static int ln_fwd(const X* x, const W* w, const W* b, X* y, float* mean, float* rstd, int64_t rows, int64_t D, int64_t ldx, float eps, cudaStream_t st) {
  if (rows == 0) return HASTE_OK;
  ln_fwd_wide_kernel<X, W><<<capped(rows, sm_count() * 8), LN_THREADS, 0, st>>>(x, w, b, y, mean, rstd, rows, D, ldx, eps);
  return check_launch("layer_norm_forward");
}

int launch_layer_norm_forward(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows, int64_t D, int64_t ldx,
                              float eps, int x_type, int w_type, cudaStream_t st) {
  using B = __nv_bfloat16;
  if (x_type == HASTE_BF16) {
    if (w_type == HASTE_BF16) return ln_fwd((const B*)x, (const B*)w, (const B*)b, (B*)y, mean, rstd, rows, D, ldx, eps, st);
    return ln_fwd((const B*)x, (const float*)w, (const float*)b, (B*)y, mean, rstd, rows, D, ldx, eps, st);
  }
  if (w_type == HASTE_BF16) return ln_fwd((const float*)x, (const B*)w, (const B*)b, (float*)y, mean, rstd, rows, D, ldx, eps, st);
  return ln_fwd((const float*)x, (const float*)w, (const float*)b, (float*)y, mean, rstd, rows, D, ldx, eps, st);
}

static int64_t ln_bwd_parts(int64_t rows) { return rows < 16 * 64 ? (rows + 63) / 64 : 16; }

int64_t layer_norm_backward_scratch(int64_t rows, int64_t D) { return ln_bwd_parts(rows) * 2 * D; }

template <class X, class G, class W>
static int ln_bwd(const G* dy, const X* x, const W* w, const float* mean, const float* rstd, X* dx, W* dw, W* db, float* scratch, int64_t rows, int64_t D,
                  int64_t lddy, int64_t ldx, cudaStream_t st) {
  const int parts = static_cast<int>(ln_bwd_parts(rows));
  if (rows > 0) {
    ln_bwd_dx_wide_kernel<X, G, W><<<capped(rows, sm_count() * 8), LN_THREADS, 0, st>>>(dy, x, w, mean, rstd, dx, rows, D, lddy, ldx);
    if (dw || db) {
      const dim3 grid(capped((D + 31) / 32, 65535), parts);
      ln_bwd_columns_kernel<X, G><<<grid, LN_THREADS, 0, st>>>(dy, x, mean, rstd, scratch, rows, D, lddy, ldx);
    }
  }
  if (dw || db) ln_bwd_finish_kernel<W><<<static_cast<unsigned>((2 * D + 31) / 32), LN_THREADS, 0, st>>>(scratch, parts, D, dw, db);
  return check_launch("layer_norm_backward");
}

int launch_layer_norm_backward(const void* dy, const void* x, const void* w, const float* mean, const float* rstd, void* dx, void* dw, void* db,
                               float* scratch, int64_t rows, int64_t D, int64_t lddy, int64_t ldx, int x_type, int dy_type, int w_type, cudaStream_t st) {
  using B = __nv_bfloat16;
  using F = float;
#define HASTE_LN_BWD(X, G, W) \
  return ln_bwd<X, G, W>((const G*)dy, (const X*)x, (const W*)w, mean, rstd, (X*)dx, (W*)dw, (W*)db, scratch, rows, D, lddy, ldx, st)
  if (x_type == HASTE_BF16) {
    if (dy_type == HASTE_BF16) { if (w_type == HASTE_BF16) HASTE_LN_BWD(B, B, B); HASTE_LN_BWD(B, B, F); }
    if (w_type == HASTE_BF16) HASTE_LN_BWD(B, F, B);
    HASTE_LN_BWD(B, F, F);
  }
  if (dy_type == HASTE_BF16) { if (w_type == HASTE_BF16) HASTE_LN_BWD(F, B, B); HASTE_LN_BWD(F, B, F); }
  if (w_type == HASTE_BF16) HASTE_LN_BWD(F, F, B);
  HASTE_LN_BWD(F, F, F);
#undef HASTE_LN_BWD
}

}  // namespace haste
