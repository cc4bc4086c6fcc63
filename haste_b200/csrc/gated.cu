// Gated feed-forward block of the features in front of the sparse layer, forward and backward:
//
//   gate = x Wg^T,  up = x Wu^T,  h = act(gate) * up,  y = h Wd^T            x [T, D], Wg, Wu [F, D], Wd [O, F]
//   dh = dy Wd,  dgate = dh * up * act'(gate),  dup = dh * act(gate),  dx = dgate Wg + dup Wu,  dWg = dgate^T x,  dWu = dup^T x,  dWd = dy^T h
//
// Forward: one launch for both projections, the activation and the product (a pair of CTAs sums 128 columns of gate and of up side by side), one for y.
// Backward: one for dh whose epilogue makes dgate, dup and h from the kept projections, one for dx (k runs over dgate and then over dup), one for the three weight
// gradients.  Operands are bf16, sums fp32.  gate, up, h, dgate and dup are rounded to bf16 where they leave the chip: they are operands of the
// next product or what training keeps, and 2^-8 of each value adds in squares to the result's own rounding.  Up to FEW_ROWS rows the weights are streamed through registers instead.
//
// Measured (bf16): forward with gate and up kept, T = 65536, D = O = 1024, F = 2048: 404 us for the first launch (1361 TFLOP/s), 171 for the second (1608); backward,
// T = 16384, D = F = O = 4096: 397 us for dh (1385), 701 for dx (1568), 1149 for the weights' (1435).  That is each launch alone; call after call the power limit bounds all of them (gemm_sm100.cuh), and
// the first launch of either direction the three matrices that its epilogue writes besides.
#include "gemm_sm100.cuh"

#include <type_traits>

namespace haste {
namespace {

using gemm::Operand;
using gemm::steps_of;
using gemm::Tile;
using gemm::Work;

enum { SILU = HASTE_ACT_SILU, GELU = HASTE_ACT_GELU, GELU_TANH = HASTE_ACT_GELU_TANH, RELU = HASTE_ACT_RELU };

__device__ __forceinline__ float sigmoid(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }

// act(g) and act'(g)
template <int ACT>
__device__ __forceinline__ void activation(float g, float& a, float& slope) {
  if (ACT == SILU) {
    const float s = sigmoid(g);
    a = g * s;
    slope = s + a * (1.f - s);
  } else if (ACT == RELU) {
    a = g > 0.f ? g : (g != g ? g : 0.f);
    slope = g > 0.f ? 1.f : 0.f;
  } else if (ACT == GELU) {
    const float cdf = 0.5f * erfcf(-0.70710678f * g);
    a = g * cdf;
    slope = cdf + g * 0.39894228f * __expf(-0.5f * g * g);
  } else {
    // 1 + tanh(u) = 2 sigmoid(2 u)
    const float s = sigmoid(1.59576912f * (g + 0.044715f * g * g * g));
    a = g * s;
    slope = s + a * (1.f - s) * 1.59576912f * (1.f + 0.134145f * g * g);
  }
}
template <int ACT>
__device__ __forceinline__ float activate(float g) {
  float a, slope;
  activation<ACT>(g, a, slope);
  return a;
}

// ---------------------------------------------------------------- tensor-core policies
// out[0] = gate, out[1] = up (kept for training where scale0 is set), out[2] = h
template <int ACT>
struct GatedForward {
  static constexpr bool A_MN = false, B_MN = false, PAIRED_B = true;
  static constexpr int PARTS = 1, OUTPUTS = 3, INPUTS = 0;
  template <int TN, class W, class I>
  static __device__ __forceinline__ void chunk(const W& w, const gemm::Problem<GatedForward>& p, const Tile&, int row, int col, uint32_t tmem, I&) {
    uint32_t g[32], u[32], packed[16];
    sm100::tmem_ld32(tmem, g);
    sm100::tmem_ld32(tmem + TN / 2, u);              // up's accumulator stands behind gate's
    sm100::tmem_ld_wait();
    if (row >= p.M) return;
    if (w.scale0 != 0.f) {
#pragma unroll
      for (int i = 0; i < 16; ++i) packed[i] = gemm::pack_bf16(__uint_as_float(g[2 * i]), __uint_as_float(g[2 * i + 1]));
      gemm::store_row(p.out[0], row, col, packed);
#pragma unroll
      for (int i = 0; i < 16; ++i) packed[i] = gemm::pack_bf16(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
      gemm::store_row(p.out[1], row, col, packed);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      packed[i] = gemm::pack_bf16(activate<ACT>(__uint_as_float(g[2 * i])) * __uint_as_float(u[2 * i]),
                                  activate<ACT>(__uint_as_float(g[2 * i + 1])) * __uint_as_float(u[2 * i + 1]));
    gemm::store_row(p.out[2], row, col, packed);
  }
};

// The accumulator is dh; in[0] = gate, in[1] = up; out[0] = dgate, out[1] = dup, out[2] = h.  (The loop holds a row's piece of six matrices.  With erf in the narrow form and tanh in the wide one that is
// more than 168 registers, and 76 and 32 bytes a thread go through local memory.  12 warps leave no more registers.)
template <int ACT>
struct GatedBackward {
  static constexpr bool A_MN = false, B_MN = true, PAIRED_B = false;
  static constexpr int PARTS = 1, OUTPUTS = 3, INPUTS = 2;
  template <int TN, class W, class I>
  static __device__ __forceinline__ void chunk(const W&, const gemm::Problem<GatedBackward>& p, const Tile&, int row, int col, uint32_t tmem, I& in) {
    uint32_t d[32], dup[16], h[16];
    sm100::tmem_ld32(tmem, d);
    sm100::tmem_ld_wait();
    if (row >= p.M) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 gg = gemm::unpack_bf16(in[0][i]), uu = gemm::unpack_bf16(in[1][i]);
      const float d0 = __uint_as_float(d[2 * i]), d1 = __uint_as_float(d[2 * i + 1]);
      float a0, s0, a1, s1;
      activation<ACT>(gg.x, a0, s0);
      activation<ACT>(gg.y, a1, s1);
      in[0][i] = gemm::pack_bf16(d0 * uu.x * s0, d1 * uu.y * s1);
      dup[i] = gemm::pack_bf16(d0 * a0, d1 * a1);
      h[i] = gemm::pack_bf16(a0 * uu.x, a1 * uu.y);
    }
    gemm::store_row(p.out[0], row, col, in[0]);
    gemm::store_row(p.out[1], row, col, dup);
    gemm::store_row(p.out[2], row, col, h);
  }
};

// Rows of fp32 parts: whole sectors, stored at once (in halves the weights' gradients of 333 rows, 509 x 1021, took 14.4 us, now 12)
__host__ __device__ constexpr int64_t parts_ld(int64_t N) { return (N + 7) & ~int64_t(7); }
// out[0] = the product in bf16, or fp32 parts in `partial` [splits][M][parts_ld(N)]
template <bool A, bool B, int K_PARTS = 1>
struct Plain {
  static constexpr bool A_MN = A, B_MN = B, PAIRED_B = false;
  static constexpr int PARTS = K_PARTS, OUTPUTS = 1, INPUTS = 0;
  template <int TN, class W, class I>
  static __device__ __forceinline__ void chunk(const W&, const gemm::Problem<Plain>& p, const Tile& t, int row, int col, uint32_t tmem, I&) {
    uint32_t v[32];
    sm100::tmem_ld32(tmem, v);
    sm100::tmem_ld_wait();
    if (row >= p.M) return;
    if (p.partial != nullptr) {
      const int64_t ld = parts_ld(p.N);
      float* to = p.partial + (static_cast<int64_t>(t.split) * p.M + row) * ld;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (col + 8 * i < ld) gemm::store_32_bytes(to + col + 8 * i, v + 8 * i);
    } else {
      uint32_t packed[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) packed[i] = gemm::pack_bf16(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
      gemm::store_row(p.out[0], row, col, packed);
    }
  }
};

// ---------------------------------------------------------------- helpers around the products
// Rows whose stride or base is not a multiple of 16 bytes are copied to where they are: tensor maps need it.  Memory alone: x, dy and the three weights of 333 rows, 509 x 1021, in 5 us,
// most of it the launch's.
constexpr int MAX_JOBS = 8;
struct Copies {
  const uint16_t* src[MAX_JOBS];
  uint16_t* dst[MAX_JOBS];
  int64_t ld_src[MAX_JOBS], ld_dst[MAX_JOBS], cols[MAX_JOBS], first[MAX_JOBS + 1];      // first: 16-byte pieces before a job's
  int n;
};
__global__ void align_rows_kernel(const __grid_constant__ Copies c) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < c.first[c.n]; i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    int k = 0;
    while (i >= c.first[k + 1]) ++k;
    const int64_t per = c.ld_dst[k] >> 3, j = i - c.first[k], row = j / per, col = (j - row * per) * 8;
    const uint16_t* s = c.src[k] + row * c.ld_src[k] + col;
    uint32_t v[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) v[x] = col + x < c.cols[k] ? s[x] : 0;
    *reinterpret_cast<uint4*>(c.dst[k] + row * c.ld_dst[k] + col) = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
  }
}

// Sums of the parts of up to four products, in order, rounded to bf16.  Memory alone; one launch for all of a call (333 rows, 509 x 1021: 6 us for 6 MB, which L2 has; a
// second launch for dx cost 2 us more).
struct Sums {
  const float* part[4];
  __nv_bfloat16* out[4];
  int64_t rows[4], cols[4], ld_out[4], first[5];
  int splits[4], n;
};
__global__ void sum_parts_kernel(const __grid_constant__ Sums s) {
  sm100::grid_dependency_wait();
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < s.first[s.n]; i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    int k = 0;
    while (i >= s.first[k + 1]) ++k;
    const int64_t ld = parts_ld(s.cols[k]), j = (i - s.first[k]) * 4, row = j / ld, col = j - row * ld, each = s.rows[k] * ld;
    float4 v = *reinterpret_cast<const float4*>(s.part[k] + j);
    for (int p = 1; p < s.splits[k]; ++p) {
      const float4 q = *reinterpret_cast<const float4*>(s.part[k] + p * each + j);
      v.x += q.x; v.y += q.y; v.z += q.z; v.w += q.w;
    }
    __nv_bfloat16* o = s.out[k] + row * s.ld_out[k] + col;
    const float a[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (col + x < s.cols[k]) o[x] = __float2bfloat16_rn(a[x]);
  }
}

// ---------------------------------------------------------------- one row
// One row's sums in CUDA cores, which have neither sums of warps to collect nor operands to shape: 3.3, 5.5, 8.6, 11.4 and 24.4 us a call at the sizes of the table below, in the
// form for few rows 4.3, 7.0, 11.0, 11.9 and 25.4.  (A call of 768 x 2048 was 8.2 us before the second launch fetched its weights early.)
constexpr int ONE_THREADS = 256;

template <bool VEC>
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int64_t i, int64_t n, float (&v)[8]) {
  if (VEC) {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p + i));
    const uint32_t r[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) { const float2 f = gemm::unpack_bf16(r[k]); v[2 * k] = f.x; v[2 * k + 1] = f.y; }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = i + k < n ? __bfloat162float(p[i + k]) : 0.f;
  }
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// h[f], one warp for each f
template <int ACT, bool VEC>
__global__ void __launch_bounds__(ONE_THREADS) gated_one_kernel(const __nv_bfloat16* __restrict__ x, const __nv_bfloat16* __restrict__ wg, const __nv_bfloat16* __restrict__ wu,
                                                                __nv_bfloat16* __restrict__ gate, __nv_bfloat16* __restrict__ up, float* __restrict__ h, int64_t D, int64_t F) {
  const int lane = threadIdx.x & 31;
  const int64_t f = static_cast<int64_t>(blockIdx.x) * (ONE_THREADS / 32) + (threadIdx.x >> 5);
  sm100::grid_launch_dependents();                 // the next launch fetches its weights meanwhile
  if (f >= F) return;
  float g = 0.f, u = 0.f;
#pragma unroll 2
  for (int64_t i = lane * 8; i < D; i += 256) {
    float a[8], b[8], v[8];
    load8<VEC>(wg + f * D, i, D, a);
    load8<VEC>(wu + f * D, i, D, b);
    load8<VEC>(x, i, D, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) { g = fmaf(a[k], v[k], g); u = fmaf(b[k], v[k], u); }
  }
  g = warp_sum(g);
  u = warp_sum(u);
  if (lane == 0) {
    h[f] = activate<ACT>(g) * u;
    if (gate != nullptr) {
      gate[f] = __float2bfloat16_rn(g);
      up[f] = __float2bfloat16_rn(u);
    }
  }
}

// y[o] = sum_f h[f] Wd[o, f]: `warps` warps for each o.  A lane's first EARLY pieces of the weights are on their way before h is there.
template <bool VEC>
__global__ void __launch_bounds__(ONE_THREADS) down_one_kernel(const float* h, const __nv_bfloat16* __restrict__ wd, __nv_bfloat16* __restrict__ y, int64_t F, int64_t O, int warps) {
  constexpr int EARLY = 2;
  __shared__ float part[ONE_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = warp % warps;
  const int64_t o = static_cast<int64_t>(blockIdx.x) * (ONE_THREADS / 32 / warps) + warp / warps, step = warps * 256, first = (mine * 32 + lane) * 8;
  const __nv_bfloat16* row = wd + o * F;
  float s = 0.f, early[EARLY][8];
#pragma unroll
  for (int k = 0; k < EARLY; ++k)
    if (o < O && first + k * step < F) load8<VEC>(row, first + k * step, F, early[k]);
  sm100::grid_dependency_wait();
  auto add = [&](const float (&a)[8], int64_t i) {
    if (VEC) {
      const float4 p = *reinterpret_cast<const float4*>(h + i), q = *reinterpret_cast<const float4*>(h + i + 4);
      s = fmaf(a[0], p.x, fmaf(a[1], p.y, fmaf(a[2], p.z, fmaf(a[3], p.w, s))));
      s = fmaf(a[4], q.x, fmaf(a[5], q.y, fmaf(a[6], q.z, fmaf(a[7], q.w, s))));
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i + k < F) s = fmaf(a[k], h[i + k], s);
    }
  };
  if (o < O) {
#pragma unroll
    for (int k = 0; k < EARLY; ++k)
      if (first + k * step < F) add(early[k], first + k * step);
#pragma unroll 2
    for (int64_t i = first + EARLY * step; i < F; i += step) {
      float a[8];
      load8<VEC>(row, i, F, a);
      add(a, i);
    }
  }
  s = warp_sum(s);
  if (lane == 0) part[warp] = s;
  __syncthreads();
  if (mine == 0 && o < O && lane == 0) {
    float v = 0.f;
    for (int k = 0; k < warps; ++k) v += part[warp + k];
    y[o] = __float2bfloat16_rn(v);
  }
}
template <int ACT, bool VEC>
int one_row(const GatedCall& c, float* h, cudaStream_t st) {
  using B = __nv_bfloat16;
  constexpr int WARPS = ONE_THREADS / 32;
  gated_one_kernel<ACT, VEC><<<static_cast<unsigned>((c.F + WARPS - 1) / WARPS), ONE_THREADS, 0, st>>>(
      static_cast<const B*>(c.x), static_cast<const B*>(c.wg), static_cast<const B*>(c.wu), static_cast<B*>(c.gate), static_cast<B*>(c.up), h, c.D, c.F);
  if (int rc = check_launch("gated_one_kernel")) return rc;
  int warps = 1;
  while (warps < WARPS && c.O * warps < static_cast<int64_t>(sm_count()) * 16 && c.F > warps * 256) warps *= 2;
  return launch_behind(down_one_kernel<VEC>, static_cast<unsigned>((c.O * warps + WARPS - 1) / WARPS), ONE_THREADS, st, static_cast<const float*>(h), static_cast<const B*>(c.wd),
                       static_cast<B*>(c.y), c.F, c.O, warps);
}

// ---------------------------------------------------------------- few rows
// Up to FEW_ROWS rows the weights' bytes are what it takes: every weight is read once, straight into the registers of a product of 16 of a matrix's rows with 8 of x (a warp's
// tensor-core instruction, which keeps up with memory; the sums in CUDA cores do not).  A block has 16 rows, its warps share k, and their sums meet in shared memory.
// us a call, weights from L2 (the first) or memory (the last):     D x F = O x F 512 x 1024   768 x 2048   1024 x 4096   2048 x 2560   4096 x 4096
//   8 rows, here                                                          4.6          7.6          11.6          12.5          25.8
//   8 rows, in CUDA cores                                                 9.0         15.8          24.2          34.5         104.8
//   32 rows, here                                                         5.7          9.8          14.4          16.1          33.3
//   32 rows, in tiles                                                     14.5         18.4          22.2          23.5          35.7
// The weights take 0.5, 1.4, 3.8, 4.8 and 15.4 us at the rate of memory: what is left is two launches, each with the latency of its first loads.
// With more weights than memory's latency hides, tiles catch up where 17 rows or more make a block read x as often as weights: 17 to 32 rows of 8192 x 8192 104 to 108 us here, 83 to 84 in
// tiles, of 2048 x 16384 56 to 60 and 52 to 57; of 16384 x 2048 72 to 77 and 79 to 82, where this rule by the number of weights alone takes the slower form.  8 and 16 rows of 8192 x 8192 90 and 78,
// 82 and 83 in tiles, of 16384 x 2048 48 and 45, 80.
constexpr int FEW_ROWS = 32, FEW_ROWS_ALWAYS = 16;
constexpr int64_t FEW_WEIGHTS = int64_t(1) << 26;      // elements of the three matrices
constexpr int EXACT_ROWS = 8;      // h stays in 32 bits up to these, and is bf16 beyond, as in the tiled form
constexpr int FEW_LINE = 64;       // k of a warp at a time: 128 bytes of each of its rows

bool takes_few(const GatedCall& c) { return c.T <= FEW_ROWS_ALWAYS || (c.T <= FEW_ROWS && (2 * c.D + c.O) * c.F <= FEW_WEIGHTS); }

template <int NT>
constexpr int few_warps() { return NT == 4 ? 8 : 16; }       // of a block, at most: what their sums' place in shared memory allows

// Elements i .. i + 7 of a row of n, zeros where there are none
template <bool VEC>
__device__ __forceinline__ uint4 piece(const __nv_bfloat16* row, int i, int n, bool there) {
  if (VEC) return there && i < n ? *reinterpret_cast<const uint4*>(row + i) : make_uint4(0, 0, 0, 0);
  const uint16_t* s = reinterpret_cast<const uint16_t*>(row) + i;
  uint32_t v[8];
#pragma unroll
  for (int x = 0; x < 8; ++x) v[x] = there && i + x < n ? s[x] : 0;
  return make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
}
__device__ __forceinline__ void mma_16x8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 32 of k: a lane has 8 neighbours of each operand, which the instruction takes for its own order of them, the same for both
__device__ __forceinline__ void add_products(float (&d)[4], const uint4& low, const uint4& high, const uint4& b) {
  mma_16x8(d, low.x, high.x, low.y, high.y, b.x, b.y);
  mma_16x8(d, low.z, high.z, low.w, high.w, b.z, b.w);
}
// A warp's sums [16 rows of the matrix][8 NT of x] to where the block adds them
template <int NT>
__device__ __forceinline__ void put_sums(float (*to)[20], const float (&d)[NT][4], int lane) {
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) to[8 * t + 2 * (lane & 3) + (e & 1)][(lane >> 2) + 8 * (e >> 1)] = d[t][e];
}

// h[t, f], 16 of f a block
template <int ACT, int NT, bool VEC>
__global__ void __launch_bounds__(few_warps<NT>() * 32, 1) gated_few_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, const __nv_bfloat16* __restrict__ wg,
                                                                         const __nv_bfloat16* __restrict__ wu, __nv_bfloat16* __restrict__ gate, __nv_bfloat16* __restrict__ up,
                                                                         int64_t ldh, __nv_bfloat16* __restrict__ h, int T, int D, int F) {
  __shared__ float part[few_warps<NT>()][2][8 * NT][20];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int f0 = blockIdx.x * 16, low = f0 + (lane >> 2), high = low + 8;
  const __nv_bfloat16 *g_low = wg + static_cast<int64_t>(low) * D, *g_high = g_low + static_cast<int64_t>(8) * D, *u_low = wu + (g_low - wg), *u_high = wu + (g_high - wg);
  sm100::grid_launch_dependents();                 // the next launch fetches its weights meanwhile
  float g[NT][4] = {}, u[NT][4] = {};
#pragma unroll 1                                   // (unrolled twice it is slower at every size: 512 x 1024 6.0 us a call instead of 4.5)
  for (int k0 = warp * FEW_LINE; k0 < D; k0 += warps * FEW_LINE) {
    uint4 gl[2], gh[2], ul[2], uh[2], xs[2][NT];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int k = k0 + c * 32 + (lane & 3) * 8;
      gl[c] = piece<VEC>(g_low, k, D, low < F); gh[c] = piece<VEC>(g_high, k, D, high < F);
      ul[c] = piece<VEC>(u_low, k, D, low < F); uh[c] = piece<VEC>(u_high, k, D, high < F);
#pragma unroll
      for (int t = 0; t < NT; ++t) xs[c][t] = piece<VEC>(x + (8 * t + (lane >> 2)) * ldx, k, D, 8 * t + (lane >> 2) < T);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        add_products(g[t], gl[c], gh[c], xs[c][t]);
        add_products(u[t], ul[c], uh[c], xs[c][t]);
      }
  }
  put_sums<NT>(part[warp][0], g, lane);
  put_sums<NT>(part[warp][1], u, lane);
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * T; i += blockDim.x) {
    const int t = i >> 4, row = i & 15;
    if (f0 + row >= F) continue;
    float gs = 0.f, us = 0.f;
    for (int w = 0; w < warps; ++w) { gs += part[w][0][t][row]; us += part[w][1][t][row]; }
    const float v = activate<ACT>(gs) * us;
    __nv_bfloat16* to = h + static_cast<int64_t>(t) * F + f0 + row;
    if (NT * 8 <= EXACT_ROWS) {
      // the sum of three bf16, without a rounding: 8 bits of it each
      float rest = v;
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const uint32_t top = __float_as_uint(rest) & 0xFFFF0000u;
        to[static_cast<int64_t>(k) * T * F] = __ushort_as_bfloat16(static_cast<uint16_t>(top >> 16));
        rest = (top & 0x7F800000u) == 0x7F800000u ? 0.f : rest - __uint_as_float(top);             // (inf and NaN are in the first alone)
      }
    } else {
      *to = __float2bfloat16_rn(v);
    }
    if (gate != nullptr) {
      gate[t * ldh + f0 + row] = __float2bfloat16_rn(gs);
      up[t * ldh + f0 + row] = __float2bfloat16_rn(us);
    }
  }
}

// y[t, o] = sum_f h[t, f] Wd[o, f], 16 of o a block.  The first pieces of the weights are on their way before h is there.
template <int NT, bool VEC>
__global__ void __launch_bounds__(few_warps<NT>() * 32, 1) down_few_kernel(const __nv_bfloat16* h, const __nv_bfloat16* __restrict__ wd, __nv_bfloat16* __restrict__ y, int T, int F, int O) {
  constexpr int C = NT == 1 ? 2 : 4, PARTS = NT * 8 <= EXACT_ROWS ? 3 : 1;         // C: pieces of each row that are on their way at once
  __shared__ float part[few_warps<NT>()][8 * NT][20];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int o0 = blockIdx.x * 16, low = o0 + (lane >> 2), high = low + 8;
  const __nv_bfloat16 *w_low = wd + static_cast<int64_t>(low) * F, *w_high = w_low + static_cast<int64_t>(8) * F, *h_mine = h + static_cast<int64_t>(lane >> 2) * F;
  auto at = [&](int k0, int c) { return k0 + (c >> 1) * warps * FEW_LINE + (c & 1) * 32 + (lane & 3) * 8; };
  float s[PARTS][NT][4] = {};
  uint4 wl[C], wh[C];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      wl[c] = piece<VEC>(w_low, at(k0, c), F, low < O);
      wh[c] = piece<VEC>(w_high, at(k0, c), F, high < O);
    }
  };
  int k0 = warp * FEW_LINE;
  fetch(k0);
  sm100::grid_dependency_wait();
#pragma unroll 1
  while (k0 < F) {
    uint4 hs[C][NT][PARTS];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < PARTS; ++k) hs[c][t][k] = piece<VEC>(h_mine + (static_cast<int64_t>(k) * T + 8 * t) * F, at(k0, c), F, 8 * t + (lane >> 2) < T);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < PARTS; ++k) add_products(s[k][t], wl[c], wh[c], hs[c][t][k]);
    k0 += warps * FEW_LINE * (C / 2);
    if (k0 < F) fetch(k0);
  }
  // Where the first parts' sum is not finite, infinite weights or h have made it so, and it is the result: the other parts of h, which may be zeros, would make NaN of an infinity.
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float sum = s[0][t][e];
#pragma unroll
      for (int k = 1; k < PARTS; ++k) sum += s[k][t][e];
      if (fabsf(s[0][t][e]) < INFINITY) s[0][t][e] = sum;
    }
  put_sums<NT>(part[warp], s[0], lane);
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * T; i += blockDim.x) {
    const int t = i >> 4, row = i & 15;
    if (o0 + row >= O) continue;
    float v = 0.f;
    for (int w = 0; w < warps; ++w) v += part[w][t][row];
    y[static_cast<int64_t>(t) * O + o0 + row] = __float2bfloat16_rn(v);
  }
}

// Warps of a block: as many as there are lines of k; 8 at most where there are more blocks than SMs (D = 1024, F = 4096: 11.0 us a call, 12.4 with 16), 16 elsewhere
template <int NT>
int warps_for(int64_t k, int64_t blocks) {
  const int64_t most = blocks <= sm_count() ? few_warps<NT>() : 8, lines = (k + FEW_LINE - 1) / FEW_LINE;
  return static_cast<int>(imin64(most, lines));
}
template <int ACT, int NT, bool VEC>
int few_rows(const GatedCall& c, __nv_bfloat16* h, cudaStream_t st) {
  using B = __nv_bfloat16;
  const int D = static_cast<int>(c.D), F = static_cast<int>(c.F), O = static_cast<int>(c.O), T = static_cast<int>(c.T);
  const int64_t up = (c.F + 15) / 16, down = (c.O + 15) / 16;
  gated_few_kernel<ACT, NT, VEC><<<static_cast<unsigned>(up), 32 * warps_for<NT>(c.D, up), 0, st>>>(
      static_cast<const B*>(c.x), c.ldx, static_cast<const B*>(c.wg), static_cast<const B*>(c.wu), static_cast<B*>(c.gate), static_cast<B*>(c.up), c.ldh, h, T, D, F);
  if (int rc = check_launch("gated_few_kernel")) return rc;
  return launch_behind(down_few_kernel<NT, VEC>, static_cast<unsigned>(down), 32 * warps_for<NT>(c.F, down), st, static_cast<const B*>(h), static_cast<const B*>(c.wd),
                       static_cast<B*>(c.y), T, F, O);
}
template <int ACT>
int few_rows_act(const GatedCall& c, void* scratch, bool vec, cudaStream_t st) {
  if (c.T == 1) return vec ? one_row<ACT, true>(c, static_cast<float*>(scratch), st) : one_row<ACT, false>(c, static_cast<float*>(scratch), st);
  __nv_bfloat16* h = static_cast<__nv_bfloat16*>(scratch);
  if (c.T <= 8) return vec ? few_rows<ACT, 1, true>(c, h, st) : few_rows<ACT, 1, false>(c, h, st);
  if (c.T <= 16) return vec ? few_rows<ACT, 2, true>(c, h, st) : few_rows<ACT, 2, false>(c, h, st);
  return vec ? few_rows<ACT, 4, true>(c, h, st) : few_rows<ACT, 4, false>(c, h, st);
}

// ---------------------------------------------------------------- host side
int64_t up8(int64_t n) { return (n + 7) & ~int64_t(7); }

// What a call lays out in its scratch memory, or would: with a NULL base the sizes alone
struct Arena {
  char* base;
  int64_t used = 0;
  void* take(int64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += (bytes + 255) & ~int64_t(255);
    return p;
  }
};

// A matrix as the tensor maps want it
struct Rows {
  const void* p;
  int64_t ld;
};

struct Aligner {
  Copies c = {};
  Arena& arena;
  explicit Aligner(Arena& a) : arena(a) {}
  // always: where sizes are asked for that are enough whatever the addresses will be
  Rows operator()(const void* p, int64_t ld, int64_t rows, int64_t cols, bool always) {
    if (!always && aligned16(p) && ld % 8 == 0) return {p, ld};
    const int64_t to = up8(cols);
    void* dst = arena.take(rows * to * 2);
    const int k = c.n++;
    c.src[k] = static_cast<const uint16_t*>(p); c.dst[k] = static_cast<uint16_t*>(dst);
    c.ld_src[k] = ld; c.ld_dst[k] = to; c.cols[k] = cols;
    c.first[k + 1] = c.first[k] + rows * (to >> 3);
    return {dst, to};
  }
  int run(cudaStream_t st) {
    if (c.n == 0) return HASTE_OK;
    const int64_t blocks = (c.first[c.n] + 255) / 256;
    align_rows_kernel<<<static_cast<unsigned>(imin64(blocks, static_cast<int64_t>(sm_count()) * 32)), 256, 0, st>>>(c);
    return check_launch("align_rows_kernel");
  }
};

// The form of a launch, and into how many parts k is cut where its tiles leave SMs idle: the parts are written and read once at 6 TB/s, the launch that adds
// them takes 2 us.
struct Form {
  bool narrow;
  int splits;
};
Form choose_form(int64_t wide, int64_t narrow, int64_t steps, int64_t elements) {
  const int64_t pairs = sm_count() / 2;
  Form best = {false, 1};
  double cost = 0;
  for (int s = 1; s <= 16 && s <= steps; ++s)
    for (int n = 0; n < 2; ++n) {
      const double c = gemm::cost_of((n ? narrow : wide) * s, (steps + s - 1) / s, n != 0, pairs) + (s > 1 ? 7 + static_cast<double>(elements) * s * 8 / 6e6 / 0.28 : 0);
      if ((s == 1 && n == 0) || c < cost) { best = {n != 0, s}; cost = c; }
    }
  return best;
}
Form form_for(int64_t M, int64_t N, int64_t steps) { return choose_form(gemm::tiles_for(M, N, gemm::TILE), gemm::tiles_for(M, N, 64), steps, M * N); }

// out [M, N] contiguous at any alignment: straight from the tiles, or through fp32 parts
struct Output {
  void* p;
  float* part;
  int splits;
};
Output output_of(Arena& arena, void* p, int64_t M, int64_t N, const Form& f, bool always) {
  Output o = {p, nullptr, f.splits};
  if (always || o.splits > 1 || N % 8 != 0 || !aligned16(p)) o.part = static_cast<float*>(arena.take(o.splits * M * parts_ld(N) * 4));
  return o;
}
void set_sizes(gemm::Sizes& p, int64_t M, int64_t N, int64_t steps0, int64_t steps) {
  p = gemm::Sizes();
  p.M = static_cast<int>(M); p.N = static_cast<int>(N);
  p.splits = 1;
  p.steps0 = static_cast<int>(steps0); p.steps = static_cast<int>(steps);
}
template <class Policy>
void set_output(gemm::Problem<Policy>& p, const Output& o) {
  p.splits = o.splits;
  p.partial = o.part;
  p.out[0] = gemm::result({o.p, p.N}, p.N);
}
void add_sum(Sums& s, const Output& o, int64_t M, int64_t N) {
  if (o.part == nullptr) return;
  const int k = s.n++;
  s.part[k] = o.part; s.out[k] = static_cast<__nv_bfloat16*>(o.p);
  s.rows[k] = M; s.cols[k] = N; s.ld_out[k] = N; s.splits[k] = o.splits;
  s.first[k + 1] = s.first[k] + M * (parts_ld(N) / 4);
}
int run_sums(const Sums& s, cudaStream_t st) {
  if (s.n == 0) return HASTE_OK;
  const int64_t blocks = (s.first[s.n] + 255) / 256;
  return launch_behind(sum_parts_kernel, static_cast<unsigned>(imin64(blocks, static_cast<int64_t>(sm_count()) * 16)), 256, st, s);
}

#define HASTE_TRY(...) \
  if (int rc_ = (__VA_ARGS__)) return rc_

// f(policy of the activation, number of columns of the form) for a launch
template <template <int> class Policy, class F>
int by_activation(int act, bool narrow, F&& f) {
  auto with = [&](auto policy) -> int {
    using K = decltype(policy);
    return narrow ? f(policy, std::integral_constant<int, gemm::narrow<K>()>()) : f(policy, std::integral_constant<int, 256>());
  };
  switch (act) {
    case SILU: return with(Policy<SILU>());
    case GELU: return with(Policy<GELU>());
    case GELU_TANH: return with(Policy<GELU_TANH>());
    default: return with(Policy<RELU>());
  }
}
template <class Policy, class F>
int by_form(bool narrow, F&& f) {
  return narrow ? f(Policy(), std::integral_constant<int, gemm::narrow<Policy>()>()) : f(Policy(), std::integral_constant<int, 256>());
}

// arena.base == NULL: only what it takes, with aligned operands or with any
int forward(Arena& arena, const GatedCall& c, cudaStream_t st) {
  const bool plan = arena.base == nullptr, any = plan && !c.aligned;
  if (takes_few(c)) {
    void* h = arena.take(c.T * c.F * (c.T == 1 ? 4 : c.T <= EXACT_ROWS ? 6 : 2));
    if (plan) return HASTE_OK;
    const bool vec = c.D % 8 == 0 && c.F % 8 == 0 && c.ldx % 8 == 0 && aligned16(c.x) && aligned16(c.wg) && aligned16(c.wu) && aligned16(c.wd);
    switch (c.act) {
      case SILU: return few_rows_act<SILU>(c, h, vec, st);
      case GELU: return few_rows_act<GELU>(c, h, vec, st);
      case GELU_TANH: return few_rows_act<GELU_TANH>(c, h, vec, st);
      default: return few_rows_act<RELU>(c, h, vec, st);
    }
  }
  const int64_t ldF = up8(c.F), sD = steps_of(c.D), sF = steps_of(c.F);
  Aligner align(arena);
  const Rows x = align(c.x, c.ldx, c.T, c.D, any), wg = align(c.wg, c.D, c.F, c.D, any), wu = align(c.wu, c.D, c.F, c.D, any), wd = align(c.wd, c.F, c.O, c.F, any);
  void* h = arena.take(c.T * ldF * 2);
  const Form fy = form_for(c.T, c.O, sF);
  const Output y = output_of(arena, c.y, c.T, c.O, fy, any);
  if (plan) return HASTE_OK;
  HASTE_TRY(align.run(st));
  const int64_t pairs = sm_count() / 2;
  const bool narrow = gemm::cost_of(gemm::tiles_for(c.T, c.F, 64), sD, true, pairs) < gemm::cost_of(gemm::tiles_for(c.T, c.F, 128), sD, false, pairs);
  HASTE_TRY(by_activation<GatedForward>(c.act, narrow, [&](auto policy, auto columns) -> int {
    using K = decltype(policy);
    constexpr int TN = decltype(columns)::value;
    Work<K, 1> w = {};
    w.problems = 1;
    w.scale0 = c.gate != nullptr ? 1.f : 0.f;
    auto& p = w.p[0];
    set_sizes(p, c.T, c.F, sD, sD);
    HASTE_TRY((gemm::map_a<K, TN>(&p.a[0], {x.p, x.ld}, c.T, c.D)));
    HASTE_TRY((gemm::map_b<K, TN>(&p.b[0], {wg.p, wg.ld}, c.F, c.D)));
    HASTE_TRY((gemm::map_b<K, TN>(&p.b[1], {wu.p, wu.ld}, c.F, c.D)));
    if (c.gate != nullptr) {
      p.out[0] = gemm::result({c.gate, c.ldh}, c.F);
      p.out[1] = gemm::result({c.up, c.ldh}, c.F);
    }
    p.out[2] = gemm::result({h, ldF}, c.F);
    return gemm::launch<K, TN>(w, align.c.n > 0, st);
  }));
  HASTE_TRY(by_form<Plain<false, false>>(fy.narrow, [&](auto policy, auto columns) -> int {
    using K = decltype(policy);
    constexpr int TN = decltype(columns)::value;
    Work<K, 1> w = {};
    w.problems = 1;
    auto& p = w.p[0];
    set_sizes(p, c.T, c.O, sF, sF);
    set_output<K>(p, y);
    HASTE_TRY((gemm::map_a<K, TN>(&p.a[0], {h, ldF}, c.T, c.F)));
    HASTE_TRY((gemm::map_b<K, TN>(&p.b[0], {wd.p, wd.ld}, c.O, c.F)));
    return gemm::launch<K, TN>(w, true, st);
  }));
  Sums s = {};
  add_sum(s, y, c.T, c.O);
  return run_sums(s, st);
}

int backward(Arena& arena, const GatedGradCall& c, cudaStream_t st) {
  const bool plan = arena.base == nullptr, any = plan && !c.aligned;
  const int64_t ldF = up8(c.F), sT = steps_of(c.T), sF = steps_of(c.F), sO = steps_of(c.O);
  Aligner align(arena);
  const Rows dy = align(c.dy, c.lddy, c.T, c.O, any), x = align(c.x, c.ldx, c.T, c.D, any), wg = align(c.wg, c.D, c.F, c.D, any), wu = align(c.wu, c.D, c.F, c.D, any),
             wd = align(c.wd, c.F, c.O, c.F, any), gate = align(c.gate, c.ldgate, c.T, c.F, any), up = align(c.up, c.ldup, c.T, c.F, any);
  void *dgate = arena.take(c.T * ldF * 2), *dup = arena.take(c.T * ldF * 2), *h = arena.take(c.T * ldF * 2);
  const Form fx = form_for(c.T, c.D, 2 * sF);
  int64_t tiles[2];                                // of all three, whichever are wanted: a gradient's bits do not depend on that
  for (int n = 0; n < 2; ++n) tiles[n] = 2 * gemm::tiles_for(c.F, c.D, n ? 64 : 256) + gemm::tiles_for(c.O, c.F, n ? 64 : 256);
  const Form fw = choose_form(tiles[0], tiles[1], sT, 2 * c.F * c.D + c.O * c.F);
  const Output dx = output_of(arena, c.dx, c.T, c.D, fx, any), dwg = output_of(arena, c.dwg, c.F, c.D, fw, any), dwu = output_of(arena, c.dwu, c.F, c.D, fw, any),
               dwd = output_of(arena, c.dwd, c.O, c.F, fw, any);
  if (plan) return HASTE_OK;
  HASTE_TRY(align.run(st));
  {
    const int64_t pairs = sm_count() / 2;
    const bool narrow = gemm::cost_of(gemm::tiles_for(c.T, c.F, 64), sO, true, pairs) < gemm::cost_of(gemm::tiles_for(c.T, c.F, 256), sO, false, pairs);
    HASTE_TRY(by_activation<GatedBackward>(c.act, narrow, [&](auto policy, auto columns) -> int {
      using K = decltype(policy);
      constexpr int TN = decltype(columns)::value;
      Work<K, 1> w = {};
      w.problems = 1;
      auto& p = w.p[0];
      set_sizes(p, c.T, c.F, sO, sO);
      HASTE_TRY((gemm::map_a<K, TN>(&p.a[0], {dy.p, dy.ld}, c.T, c.O)));
      HASTE_TRY((gemm::map_b<K, TN>(&p.b[0], {wd.p, wd.ld}, c.F, c.O)));
      p.in[0] = gemm::result({gate.p, gate.ld}, c.F);
      p.in[1] = gemm::result({up.p, up.ld}, c.F);
      void* outs[3] = {dgate, dup, h};
      for (int i = 0; i < 3; ++i) p.out[i] = gemm::result({outs[i], ldF}, c.F);
      return gemm::launch<K, TN>(w, align.c.n > 0, st);
    }));
  }
  Sums s = {};
  if (c.dx != nullptr) {
    HASTE_TRY(by_form<Plain<false, true, 2>>(fx.narrow, [&](auto policy, auto columns) -> int {
      using K = decltype(policy);
      constexpr int TN = decltype(columns)::value;
      Work<K, 1> w = {};
      w.problems = 1;
      auto& p = w.p[0];
      set_sizes(p, c.T, c.D, sF, 2 * sF);
      set_output<K>(p, dx);
      HASTE_TRY((gemm::map_a<K, TN>(&p.a[0], {dgate, ldF}, c.T, c.F)));
      HASTE_TRY((gemm::map_a<K, TN>(&p.a[1], {dup, ldF}, c.T, c.F)));
      HASTE_TRY((gemm::map_b<K, TN>(&p.b[0], {wg.p, wg.ld}, c.D, c.F)));
      HASTE_TRY((gemm::map_b<K, TN>(&p.b[1], {wu.p, wu.ld}, c.D, c.F)));
      return gemm::launch<K, TN>(w, true, st);
    }));
    add_sum(s, dx, c.T, c.D);
  }
  if (c.dwg == nullptr && c.dwu == nullptr && c.dwd == nullptr) return run_sums(s, st);
  HASTE_TRY(by_form<Plain<true, true>>(fw.narrow, [&](auto policy, auto columns) -> int {
    using K = decltype(policy);
    constexpr int TN = decltype(columns)::value;
    Work<K, 3> w = {};
    auto weight = [&](const Output& o, const Operand& a, const Operand& b, int64_t M, int64_t N) -> int {
      if (o.p == nullptr) return HASTE_OK;
      auto& p = w.p[w.problems++];
      set_sizes(p, M, N, sT, sT);
      set_output<K>(p, o);
      HASTE_TRY((gemm::map_a<K, TN>(&p.a[0], a, M, c.T)));
      HASTE_TRY((gemm::map_b<K, TN>(&p.b[0], b, N, c.T)));
      add_sum(s, o, M, N);
      return HASTE_OK;
    };
    HASTE_TRY(weight(dwg, {dgate, ldF}, {x.p, x.ld}, c.F, c.D));
    HASTE_TRY(weight(dwu, {dup, ldF}, {x.p, x.ld}, c.F, c.D));
    HASTE_TRY(weight(dwd, {dy.p, dy.ld}, {h, ldF}, c.O, c.F));
    return gemm::launch<K, TN>(w, true, st);
  }));
  return run_sums(s, st);
}

}  // namespace

int64_t gated_forward_scratch(const GatedCall& c) {
  Arena a = {nullptr};
  forward(a, c, nullptr);
  return a.used;
}
int64_t gated_backward_scratch(const GatedGradCall& c) {
  Arena a = {nullptr};
  backward(a, c, nullptr);
  return a.used;
}
int launch_gated_forward(const GatedCall& c, void* scratch, cudaStream_t st) {
  HASTE_TRY(report_pending_status("haste_gated_forward"));
  Arena a = {static_cast<char*>(scratch)};
  return forward(a, c, st);
}
int launch_gated_backward(const GatedGradCall& c, void* scratch, cudaStream_t st) {
  HASTE_TRY(report_pending_status("haste_gated_backward"));
  Arena a = {static_cast<char*>(scratch)};
  return backward(a, c, st);
}

}  // namespace haste
