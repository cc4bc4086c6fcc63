// Gated feed-forward block of the features in front of the sparse layer, forward and backward:
//
//   gate = x Wg^T,  up = x Wu^T,  h = act(gate) * up,  y = h Wd^T            x [T, D], Wg, Wu [F, D], Wd [O, F]
//   dh = dy Wd,  dgate = dh * up * act'(gate),  dup = dh * act(gate),  dx = dgate Wg + dup Wu,  dWg = dgate^T x,  dWu = dup^T x,  dWd = dy^T h
//
// Forward: one launch for both projections, the activation and the product (a pair of CTAs sums 128 columns of gate and of up side by side), one for y.
// Backward: one for dh whose epilogue makes dgate, dup and h from the kept projections, one for dx (k runs over dgate and then over dup), one for the three weight
// gradients.  Operands are bf16, sums fp32.  gate, up, h, dgate and dup are rounded to bf16 where they leave the chip: they are operands of the
// next product or what training keeps, and 2^-8 of each value adds in squares to the result's own rounding.  Up to GEMV_ROWS rows the weights are streamed through CUDA cores instead.
//
// Measured (bf16): forward with gate and up kept, T = 65536, D = O = 1024, F = 2048: 410 us for the first launch (1341 TFLOP/s), 176 for the second (1562); backward,
// T = 16384, D = F = O = 4096: 402 us for dh (1368), 716 for dx (1535), 1173 for the weights' (1406).  The power limit bounds all of them, and the first launch of either direction
// the three matrices that its epilogue writes besides.
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

// The accumulator is dh; in[0] = gate, in[1] = up; out[0] = dgate, out[1] = dup, out[2] = h
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

// out[0] = the product in bf16, or fp32 parts in `partial` [splits][M][N rounded up to 4]
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
      const int64_t ld = (p.N + 3) & ~3;
      float* to = p.partial + (static_cast<int64_t>(t.split) * p.M + row) * ld;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + 4 * i < ld) *reinterpret_cast<uint4*>(to + col + 4 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
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
    const int64_t ld = (s.cols[k] + 3) & ~int64_t(3), j = (i - s.first[k]) * 4, row = j / ld, col = j - row * ld, each = s.rows[k] * ld;
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

// ---------------------------------------------------------------- few rows
constexpr int GEMV_ROWS = 8;
constexpr int GEMV_THREADS = 256;

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

// h[t, f] for T <= ROWS rows, one warp for each f.  Bound by the weights' bytes: one row, D = 768, F = 2048 (6 MB): 5.0 us, and 4.7 for the second launch, which overlaps
// it: 7.3 in all, 8.2 before its weights were fetched early.  From L2, as the weights are from call to call; with more rows the sums in CUDA cores bind (8 rows: 19 us;
// 9 rows take the tensor cores).
template <int ACT, int ROWS, bool VEC>
__global__ void __launch_bounds__(GEMV_THREADS) gated_few_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, const __nv_bfloat16* __restrict__ wg,
                                                                 const __nv_bfloat16* __restrict__ wu, __nv_bfloat16* __restrict__ gate, __nv_bfloat16* __restrict__ up,
                                                                 int64_t ldh, float* __restrict__ h, int T, int64_t D, int64_t F) {
  const int lane = threadIdx.x & 31;
  const int64_t f = static_cast<int64_t>(blockIdx.x) * (GEMV_THREADS / 32) + (threadIdx.x >> 5);
  sm100::grid_launch_dependents();                 // the next launch fetches its weights meanwhile
  if (f >= F) return;
  float g[ROWS], u[ROWS];
#pragma unroll
  for (int t = 0; t < ROWS; ++t) g[t] = u[t] = 0.f;
#pragma unroll 2
  for (int64_t i = lane * 8; i < D; i += 256) {
    float a[8], b[8], v[8];
    load8<VEC>(wg + f * D, i, D, a);
    load8<VEC>(wu + f * D, i, D, b);
#pragma unroll
    for (int t = 0; t < ROWS; ++t) {
      if (t < T) {
        load8<VEC>(x + t * ldx, i, D, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) { g[t] = fmaf(a[k], v[k], g[t]); u[t] = fmaf(b[k], v[k], u[t]); }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < ROWS; ++t) {
    if (t >= T) break;
    const float gs = warp_sum(g[t]), us = warp_sum(u[t]);
    if (lane == 0) {
      h[t * F + f] = activate<ACT>(gs) * us;
      if (gate != nullptr) {
        gate[t * ldh + f] = __float2bfloat16_rn(gs);
        up[t * ldh + f] = __float2bfloat16_rn(us);
      }
    }
  }
}

// y[t, o] = sum_f h[t, f] Wd[o, f]: `warps` warps for each o.  A lane's first EARLY pieces of the weights are on their way before h is there.
template <int ROWS, bool VEC>
__global__ void __launch_bounds__(GEMV_THREADS) down_few_kernel(const float* __restrict__ h, const __nv_bfloat16* __restrict__ wd, __nv_bfloat16* __restrict__ y, int T, int64_t F,
                                                                int64_t O, int warps) {
  constexpr int EARLY = 2;
  __shared__ float part[GEMV_THREADS / 32][ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t o = static_cast<int64_t>(blockIdx.x) * (GEMV_THREADS / 32 / warps) + warp / warps, step = warps * 256;
  const int mine = warp % warps;
  const int64_t first = (mine * 32 + lane) * 8;
  const __nv_bfloat16* row = wd + o * F;
  float s[ROWS], early[EARLY][8];
#pragma unroll
  for (int t = 0; t < ROWS; ++t) s[t] = 0.f;
#pragma unroll
  for (int k = 0; k < EARLY; ++k)
    if (o < O && first + k * step < F) load8<VEC>(row, first + k * step, F, early[k]);
  sm100::grid_dependency_wait();
  auto add = [&](const float (&a)[8], int64_t i) {
#pragma unroll
    for (int t = 0; t < ROWS; ++t)
      if (t < T) {
        if (VEC) {
          const float4 p = *reinterpret_cast<const float4*>(h + t * F + i), q = *reinterpret_cast<const float4*>(h + t * F + i + 4);
          s[t] = fmaf(a[0], p.x, fmaf(a[1], p.y, fmaf(a[2], p.z, fmaf(a[3], p.w, s[t]))));
          s[t] = fmaf(a[4], q.x, fmaf(a[5], q.y, fmaf(a[6], q.z, fmaf(a[7], q.w, s[t]))));
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (i + k < F) s[t] = fmaf(a[k], h[t * F + i + k], s[t]);
        }
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
#pragma unroll
  for (int t = 0; t < ROWS; ++t) {
    s[t] = warp_sum(s[t]);
    if (lane == 0) part[warp][t] = s[t];
  }
  __syncthreads();
  if (mine == 0 && o < O && lane < T && lane < ROWS) {
    float v = 0.f;
    for (int k = 0; k < warps; ++k) v += part[warp + k][lane];
    y[lane * O + o] = __float2bfloat16_rn(v);
  }
}

template <int ACT, int ROWS, bool VEC>
int few_rows(const void* x, int64_t ldx, const void* wg, const void* wu, const void* wd, void* gate, void* up, int64_t ldh, void* y, float* h, int64_t T, int64_t D, int64_t F,
             int64_t O, cudaStream_t st) {
  using B = __nv_bfloat16;
  constexpr int WARPS = GEMV_THREADS / 32;
  gated_few_kernel<ACT, ROWS, VEC><<<static_cast<unsigned>((F + WARPS - 1) / WARPS), GEMV_THREADS, 0, st>>>(
      static_cast<const B*>(x), ldx, static_cast<const B*>(wg), static_cast<const B*>(wu), static_cast<B*>(gate), static_cast<B*>(up), ldh, h, static_cast<int>(T), D, F);
  if (int rc = check_launch("gated_few_kernel")) return rc;
  int warps = 1;
  while (warps < WARPS && O * warps < static_cast<int64_t>(sm_count()) * 16 && F > warps * 256) warps *= 2;
  return launch_behind(down_few_kernel<ROWS, VEC>, static_cast<unsigned>((O * warps + WARPS - 1) / WARPS), GEMV_THREADS, st, static_cast<const float*>(h), static_cast<const B*>(wd),
                       static_cast<B*>(y), static_cast<int>(T), F, O, warps);
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
  if (always || o.splits > 1 || N % 8 != 0 || !aligned16(p)) o.part = static_cast<float*>(arena.take(o.splits * M * ((N + 3) & ~int64_t(3)) * 4));
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
  s.first[k + 1] = s.first[k] + M * (((N + 3) & ~int64_t(3)) / 4);
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

template <int ACT>
int few_rows_act(bool vec, int64_t T, const void* x, int64_t ldx, const void* wg, const void* wu, const void* wd, void* gate, void* up, int64_t ldh, void* y, float* h, int64_t D, int64_t F,
                 int64_t O, cudaStream_t st) {
#define HASTE_FEW(R) (vec ? few_rows<ACT, R, true>(x, ldx, wg, wu, wd, gate, up, ldh, y, h, T, D, F, O, st) : few_rows<ACT, R, false>(x, ldx, wg, wu, wd, gate, up, ldh, y, h, T, D, F, O, st))
  return T == 1 ? HASTE_FEW(1) : T <= 4 ? HASTE_FEW(4) : HASTE_FEW(8);
#undef HASTE_FEW
}

// arena.base == NULL: only what it takes, with aligned operands or with any
int forward(Arena& arena, const GatedCall& c, cudaStream_t st) {
  const bool plan = arena.base == nullptr, any = plan && !c.aligned;
  if (c.T <= GEMV_ROWS) {
    float* h = static_cast<float*>(arena.take(c.T * c.F * 4));
    if (plan) return HASTE_OK;
    const bool vec = c.D % 8 == 0 && c.F % 8 == 0 && c.ldx % 8 == 0 && aligned16(c.x) && aligned16(c.wg) && aligned16(c.wu) && aligned16(c.wd);
    switch (c.act) {
      case SILU: return few_rows_act<SILU>(vec, c.T, c.x, c.ldx, c.wg, c.wu, c.wd, c.gate, c.up, c.ldh, c.y, h, c.D, c.F, c.O, st);
      case GELU: return few_rows_act<GELU>(vec, c.T, c.x, c.ldx, c.wg, c.wu, c.wd, c.gate, c.up, c.ldh, c.y, h, c.D, c.F, c.O, st);
      case GELU_TANH: return few_rows_act<GELU_TANH>(vec, c.T, c.x, c.ldx, c.wg, c.wu, c.wd, c.gate, c.up, c.ldh, c.y, h, c.D, c.F, c.O, st);
      default: return few_rows_act<RELU>(vec, c.T, c.x, c.ldx, c.wg, c.wu, c.wd, c.gate, c.up, c.ldh, c.y, h, c.D, c.F, c.O, st);
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
