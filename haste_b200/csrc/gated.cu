// Gated feed-forward block of the features in front of the sparse layer, forward and backward:
//
//   gate = x Wg^T,  up = x Wu^T,  h = act(gate) * up,  y = h Wd^T            x [T, D], Wg, Wu [F, D], Wd [O, F]
//   dh = dy Wd,  dgate = dh * up * act'(gate),  dup = dh * act(gate),  dx = dgate Wg + dup Wu,  dWg = dgate^T x,  dWu = dup^T x,  dWd = dy^T h
//
// Forward: one launch for both projections, the activation and the product (a pair of CTAs sums 128 columns of gate and of up side by side), one for y.
// Backward: one for dh whose epilogue makes dgate, dup and h from the kept projections, one for dx (k runs over dgate and then over dup), one for the three weight
// gradients.  Operands are bf16, sums fp32.  gate, up, h, dgate and dup are rounded to bf16 where they leave the chip: they are operands of the
// next product or what training keeps, and 2^-8 of each value adds in squares to the result's own rounding.  Up to GEMV_ROWS rows the weights are streamed through CUDA cores instead.
#include "gemm_sm100.cuh"

namespace haste {
namespace {

using gemm::Problem;
using gemm::Stager;
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
  static constexpr bool A_MN = false, B_MN = false, F16 = false, PAIRED_B = true;
  template <int P>
  static __device__ __forceinline__ void epilogue(const Work<P>& w, const Problem& p, const Tile& t, int row0, int half, uint32_t tmem, Stager& st, int lane) {
    const bool keep = w.scale0 != 0.f;
#pragma unroll 1
    for (int j = 0; j < 2; ++j) {
      const int at = half * 64 + j * 32, col = t.n * 128 + at;
      const bool inside = row0 < p.M && col < p.N;
      uint32_t g[32], u[32], packed[16];
      sm100::tmem_ld32(tmem + at, g);
      sm100::tmem_ld32(tmem + 128 + at, u);
      sm100::tmem_ld_wait();
      if (keep) {
#pragma unroll
        for (int i = 0; i < 16; ++i) packed[i] = gemm::pack_bf16(__uint_as_float(g[2 * i]), __uint_as_float(g[2 * i + 1]));
        uint32_t box = st.get();
        gemm::box_row(box, lane, packed);
        st.put(&p.out[0], box, col, row0, t.batch, inside);
#pragma unroll
        for (int i = 0; i < 16; ++i) packed[i] = gemm::pack_bf16(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
        box = st.get();
        gemm::box_row(box, lane, packed);
        st.put(&p.out[1], box, col, row0, t.batch, inside);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        packed[i] = gemm::pack_bf16(activate<ACT>(__uint_as_float(g[2 * i])) * __uint_as_float(u[2 * i]),
                                    activate<ACT>(__uint_as_float(g[2 * i + 1])) * __uint_as_float(u[2 * i + 1]));
      const uint32_t box = st.get();
      gemm::box_row(box, lane, packed);
      st.put(&p.out[2], box, col, row0, t.batch, inside);
    }
  }
};

// The accumulator is dh; in[0] = gate, in[1] = up; out[0] = dgate, out[1] = dup, out[2] = h
template <int ACT>
struct GatedBackward {
  static constexpr bool A_MN = false, B_MN = true, F16 = false, PAIRED_B = false;
  template <int P>
  static __device__ __forceinline__ void epilogue(const Work<P>&, const Problem& p, const Tile& t, int row0, int half, uint32_t tmem, Stager& st, int lane) {
    const int row = row0 + lane;
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {
      const int at = half * 128 + j * 32, col = t.n * gemm::TILE + at;
      const bool inside = row0 < p.M && col < p.N;
      uint32_t g[16], u[16], d[32];
      gemm::load_row(g, p.in[0] + static_cast<int64_t>(row) * p.ld_in, col, p.ld_in, row < p.M);
      gemm::load_row(u, p.in[1] + static_cast<int64_t>(row) * p.ld_in, col, p.ld_in, row < p.M);
      sm100::tmem_ld32(tmem + at, d);
      sm100::tmem_ld_wait();
      uint32_t dup[16], h[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 gg = gemm::unpack_bf16(g[i]), uu = gemm::unpack_bf16(u[i]);
        const float d0 = __uint_as_float(d[2 * i]), d1 = __uint_as_float(d[2 * i + 1]);
        float a0, s0, a1, s1;
        activation<ACT>(gg.x, a0, s0);
        activation<ACT>(gg.y, a1, s1);
        g[i] = gemm::pack_bf16(d0 * uu.x * s0, d1 * uu.y * s1);
        dup[i] = gemm::pack_bf16(d0 * a0, d1 * a1);
        h[i] = gemm::pack_bf16(a0 * uu.x, a1 * uu.y);
      }
      uint32_t box = st.get();
      gemm::box_row(box, lane, g);
      st.put(&p.out[0], box, col, row0, t.batch, inside);
      box = st.get();
      gemm::box_row(box, lane, dup);
      st.put(&p.out[1], box, col, row0, t.batch, inside);
      box = st.get();
      gemm::box_row(box, lane, h);
      st.put(&p.out[2], box, col, row0, t.batch, inside);
    }
  }
};

// out[0] = the product in bf16, or fp32 parts in `partial` [splits][M][N rounded up to 4]
template <bool A, bool B>
struct Plain {
  static constexpr bool A_MN = A, B_MN = B, F16 = false, PAIRED_B = false;
  template <int P>
  static __device__ __forceinline__ void epilogue(const Work<P>&, const Problem& p, const Tile& t, int row0, int half, uint32_t tmem, Stager& st, int lane) {
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {
      const int at = half * 128 + j * 32, col = t.n * gemm::TILE + at;
      uint32_t v[32];
      sm100::tmem_ld32(tmem + at, v);
      sm100::tmem_ld_wait();
      if (p.partial != nullptr) {
        const int64_t ld = (p.N + 3) & ~3;
        if (row0 + lane < p.M) {
          float* to = p.partial + (static_cast<int64_t>(t.split) * p.M + row0 + lane) * ld;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (col + 4 * i < ld)
              *reinterpret_cast<uint4*>(to + col + 4 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
      } else {
        uint32_t packed[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) packed[i] = gemm::pack_bf16(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
        const uint32_t box = st.get();
        gemm::box_row(box, lane, packed);
        st.put(&p.out[0], box, col, row0, t.batch, row0 < p.M && col < p.N);
      }
    }
  }
};

// ---------------------------------------------------------------- helpers around the products
// Rows whose stride or base is not a multiple of 16 bytes are copied to where they are: tensor maps need it.
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

// Sums of the parts of up to three products, in order, rounded to bf16
struct Sums {
  const float* part[3];
  __nv_bfloat16* out[3];
  int64_t rows[3], cols[3], ld_out[3], first[4];
  int splits[3], n;
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

// h[t, f] for T <= ROWS rows, one warp for each f
template <int ACT, int ROWS, bool VEC>
__global__ void __launch_bounds__(GEMV_THREADS) gated_few_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, const __nv_bfloat16* __restrict__ wg,
                                                                 const __nv_bfloat16* __restrict__ wu, __nv_bfloat16* __restrict__ gate, __nv_bfloat16* __restrict__ up,
                                                                 int64_t ldh, float* __restrict__ h, int T, int64_t D, int64_t F) {
  const int lane = threadIdx.x & 31;
  const int64_t f = static_cast<int64_t>(blockIdx.x) * (GEMV_THREADS / 32) + (threadIdx.x >> 5);
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

// y[t, o] = sum_f h[t, f] Wd[o, f]: WARPS warps for each o
template <int ROWS, bool VEC>
__global__ void __launch_bounds__(GEMV_THREADS) down_few_kernel(const float* __restrict__ h, const __nv_bfloat16* __restrict__ wd, __nv_bfloat16* __restrict__ y, int T, int64_t F,
                                                                int64_t O, int warps) {
  __shared__ float part[GEMV_THREADS / 32][ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t o = static_cast<int64_t>(blockIdx.x) * (GEMV_THREADS / 32 / warps) + warp / warps;
  const int mine = warp % warps;
  float s[ROWS];
#pragma unroll
  for (int t = 0; t < ROWS; ++t) s[t] = 0.f;
  sm100::grid_dependency_wait();
  if (o < O) {
#pragma unroll 2
    for (int64_t i = (mine * 32 + lane) * 8; i < F; i += warps * 256) {
      float a[8];
      load8<VEC>(wd + o * F, i, F, a);
#pragma unroll
      for (int t = 0; t < ROWS; ++t)
        if (t < T) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (VEC || i + k < F) s[t] = fmaf(a[k], h[t * F + i + k], s[t]);
        }
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

// A product M x N over `steps` of k is cut along k where its tiles leave SMs idle.  In units of a step of k of one tile (0.28 us): a tile costs its steps and
// 6 more, the parts are written and read once at 6 TB/s, the launch that adds them takes 2 us.
int choose_splits(int64_t tiles, int64_t steps, int64_t elements) {
  const int64_t pairs = sm_count() / 2;
  int best = 1;
  double cost = 0;
  for (int s = 1; s <= 16 && s <= steps; ++s) {
    const double c = static_cast<double>((tiles * s + pairs - 1) / pairs) * (static_cast<double>((steps + s - 1) / s) + 6) +
                     (s > 1 ? 7 + static_cast<double>(elements) * s * 8 / 6e6 / 0.28 : 0);
    if (s == 1 || c < cost) { best = s; cost = c; }
  }
  return best;
}
int64_t tiles_for(int64_t M, int64_t N) { return ((M + gemm::TILE - 1) / gemm::TILE) * ((N + gemm::TILE - 1) / gemm::TILE); }
int64_t k_steps(int64_t K) { return (K + gemm::KSTEP - 1) / gemm::KSTEP; }

// out [M, N] contiguous at any alignment: straight from the tiles, or through fp32 parts
struct Output {
  void* p;
  float* part;
  int splits;
};
Output output_of(Arena& arena, void* p, int64_t M, int64_t N, int64_t tiles, int64_t steps, bool always) {
  Output o = {p, nullptr, choose_splits(tiles, steps, M * N)};
  if (always || o.splits > 1 || N % 8 != 0 || !aligned16(p))
    o.part = static_cast<float*>(arena.take(o.splits * M * ((N + 3) & ~int64_t(3)) * 4));
  return o;
}
int set_product(Problem& p, const Output& o, int64_t M, int64_t N, int64_t steps0, int64_t steps) {
  p = Problem();
  p.M = static_cast<int>(M); p.N = static_cast<int>(N);
  p.tiles_m = static_cast<int>((M + gemm::TILE - 1) / gemm::TILE); p.tiles_n = static_cast<int>((N + gemm::TILE - 1) / gemm::TILE);
  p.batch = 1; p.splits = o.splits;
  p.steps0 = static_cast<int>(steps0); p.steps = static_cast<int>(steps);
  p.partial = o.part;
  if (o.part == nullptr) return gemm::make_map(&p.out[0], o.p, false, N, M, 1, N, 0, gemm::BOX_STORE);
  return HASTE_OK;
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

template <template <int> class Policy>
int launch_by_activation(int act, Work<1>& w, bool behind, cudaStream_t st) {
  switch (act) {
    case SILU: return gemm::launch<Policy<SILU>>(w, behind, st);
    case GELU: return gemm::launch<Policy<GELU>>(w, behind, st);
    case GELU_TANH: return gemm::launch<Policy<GELU_TANH>>(w, behind, st);
    default: return gemm::launch<Policy<RELU>>(w, behind, st);
  }
}

#define HASTE_TRY(e) \
  if (int rc_ = (e)) return rc_

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
  const int64_t ldF = up8(c.F);
  Aligner align(arena);
  const Rows x = align(c.x, c.ldx, c.T, c.D, any), wg = align(c.wg, c.D, c.F, c.D, any), wu = align(c.wu, c.D, c.F, c.D, any), wd = align(c.wd, c.F, c.O, c.F, any);
  void* h = arena.take(c.T * ldF * 2);
  const Output y = output_of(arena, c.y, c.T, c.O, tiles_for(c.T, c.O), k_steps(c.F), any);
  if (plan) return HASTE_OK;
  HASTE_TRY(align.run(st));
  Work<1> w = {};
  w.problems = 1;
  w.scale0 = c.gate != nullptr ? 1.f : 0.f;
  Problem& p = w.p[0];
  p.M = static_cast<int>(c.T); p.N = static_cast<int>(c.F);
  p.tiles_m = static_cast<int>((c.T + gemm::TILE - 1) / gemm::TILE); p.tiles_n = static_cast<int>((c.F + 127) / 128);
  p.batch = p.splits = 1;
  p.steps0 = p.steps = static_cast<int>(k_steps(c.D));
  HASTE_TRY(gemm::make_map(&p.a[0], x.p, false, c.D, c.T, 1, x.ld, 0, gemm::BOX_K));
  HASTE_TRY(gemm::make_map(&p.b[0], wg.p, false, c.D, c.F, 1, wg.ld, 0, gemm::BOX_K));
  HASTE_TRY(gemm::make_map(&p.b[1], wu.p, false, c.D, c.F, 1, wu.ld, 0, gemm::BOX_K));
  if (c.gate != nullptr) {
    HASTE_TRY(gemm::make_map(&p.out[0], c.gate, false, c.F, c.T, 1, c.ldh, 0, gemm::BOX_STORE));
    HASTE_TRY(gemm::make_map(&p.out[1], c.up, false, c.F, c.T, 1, c.ldh, 0, gemm::BOX_STORE));
  }
  HASTE_TRY(gemm::make_map(&p.out[2], h, false, c.F, c.T, 1, ldF, 0, gemm::BOX_STORE));
  HASTE_TRY(launch_by_activation<GatedForward>(c.act, w, align.c.n > 0, st));
  HASTE_TRY(set_product(p, y, c.T, c.O, k_steps(c.F), k_steps(c.F)));
  HASTE_TRY(gemm::make_map(&p.a[0], h, false, c.F, c.T, 1, ldF, 0, gemm::BOX_K));
  HASTE_TRY(gemm::make_map(&p.b[0], wd.p, false, c.F, c.O, 1, wd.ld, 0, gemm::BOX_K));
  HASTE_TRY((gemm::launch<Plain<false, false>>(w, true, st)));
  Sums s = {};
  add_sum(s, y, c.T, c.O);
  return run_sums(s, st);
}

int backward(Arena& arena, const GatedGradCall& c, cudaStream_t st) {
  const bool plan = arena.base == nullptr, any = plan && !c.aligned;
  const int64_t ldF = up8(c.F);
  Aligner align(arena);
  const Rows dy = align(c.dy, c.lddy, c.T, c.O, any), x = align(c.x, c.ldx, c.T, c.D, any), wg = align(c.wg, c.D, c.F, c.D, any), wu = align(c.wu, c.D, c.F, c.D, any),
             wd = align(c.wd, c.F, c.O, c.F, any);
  Rows gate = align(c.gate, c.ldgate, c.T, c.F, any), up = align(c.up, c.ldup, c.T, c.F, any);
  if (!plan && gate.ld != up.ld) {                     // the epilogue reads both with one stride
    if (gate.p == c.gate) gate = align(c.gate, c.ldgate, c.T, c.F, true);
    if (up.p == c.up) up = align(c.up, c.ldup, c.T, c.F, true);
  }
  void *dgate = arena.take(c.T * ldF * 2), *dup = arena.take(c.T * ldF * 2), *h = arena.take(c.T * ldF * 2);
  const int64_t sT = k_steps(c.T), sF = k_steps(c.F), tw = tiles_for(c.F, c.D), td = tiles_for(c.O, c.F);
  const int64_t all = (c.dwg ? tw : 0) + (c.dwu ? tw : 0) + (c.dwd ? td : 0);
  const Output dx = output_of(arena, c.dx, c.T, c.D, tiles_for(c.T, c.D), 2 * sF, any);
  const Output dwg = output_of(arena, c.dwg, c.F, c.D, all, sT, any), dwu = output_of(arena, c.dwu, c.F, c.D, all, sT, any), dwd = output_of(arena, c.dwd, c.O, c.F, all, sT, any);
  if (plan) return HASTE_OK;
  HASTE_TRY(align.run(st));
  {
    Work<1> w = {};
    w.problems = 1;
    Problem& p = w.p[0];
    HASTE_TRY(set_product(p, {dgate, reinterpret_cast<float*>(dgate), 1}, c.T, c.F, k_steps(c.O), k_steps(c.O)));
    p.partial = nullptr;
    p.in[0] = static_cast<const uint16_t*>(gate.p); p.in[1] = static_cast<const uint16_t*>(up.p);
    p.ld_in = gate.ld;
    HASTE_TRY(gemm::make_map(&p.a[0], dy.p, false, c.O, c.T, 1, dy.ld, 0, gemm::BOX_K));
    HASTE_TRY(gemm::make_map(&p.b[0], wd.p, false, c.F, c.O, 1, wd.ld, 0, gemm::BOX_MN));
    void* outs[3] = {dgate, dup, h};
    for (int i = 0; i < 3; ++i) HASTE_TRY(gemm::make_map(&p.out[i], outs[i], false, c.F, c.T, 1, ldF, 0, gemm::BOX_STORE));
    HASTE_TRY(launch_by_activation<GatedBackward>(c.act, w, align.c.n > 0, st));
  }
  Sums s = {};
  if (c.dx != nullptr) {
    Work<1> w = {};
    w.problems = 1;
    Problem& p = w.p[0];
    HASTE_TRY(set_product(p, dx, c.T, c.D, sF, 2 * sF));
    HASTE_TRY(gemm::make_map(&p.a[0], dgate, false, c.F, c.T, 1, ldF, 0, gemm::BOX_K));
    HASTE_TRY(gemm::make_map(&p.a[1], dup, false, c.F, c.T, 1, ldF, 0, gemm::BOX_K));
    HASTE_TRY(gemm::make_map(&p.b[0], wg.p, false, c.D, c.F, 1, wg.ld, 0, gemm::BOX_MN));
    HASTE_TRY(gemm::make_map(&p.b[1], wu.p, false, c.D, c.F, 1, wu.ld, 0, gemm::BOX_MN));
    HASTE_TRY((gemm::launch<Plain<false, true>>(w, true, st)));
    if (dx.part != nullptr) {
      Sums one = {};
      add_sum(one, dx, c.T, c.D);
      HASTE_TRY(run_sums(one, st));
    }
  }
  Work<3> w = {};
  auto weight = [&](const Output& o, const void* a, int64_t lda, const Rows& b, int64_t M, int64_t N) -> int {
    if (o.p == nullptr) return HASTE_OK;
    Problem& p = w.p[w.problems++];
    HASTE_TRY(set_product(p, o, M, N, sT, sT));
    HASTE_TRY(gemm::make_map(&p.a[0], a, false, M, c.T, 1, lda, 0, gemm::BOX_MN));
    HASTE_TRY(gemm::make_map(&p.b[0], b.p, false, N, c.T, 1, b.ld, 0, gemm::BOX_MN));
    add_sum(s, o, M, N);
    return HASTE_OK;
  };
  HASTE_TRY(weight(dwg, dgate, ldF, x, c.F, c.D));
  HASTE_TRY(weight(dwu, dup, ldF, x, c.F, c.D));
  HASTE_TRY(weight(dwd, dy.p, dy.ld, {h, ldF}, c.O, c.F));
  if (w.problems == 0) return HASTE_OK;
  HASTE_TRY((gemm::launch<Plain<true, true>>(w, true, st)));
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
