// Dense products for the operators in front of the sparse layer: one persistent kernel over the tiles of several products, two SMs to a tile.
//
//   acc[m, n] = sum_k a[m, k] b[n, k]        (a second pair of operands may go on where the first ends)
//
// A cluster of two CTAs has a tile of 256 x TN: each loads its half of both operands by TMA (128 rows of a, TN / 2 of b, 64 along k), the even one
// issues tcgen05.mma.cta_group::2, whose operands are both CTAs' shared memory and whose accumulator is 128 x TN fp32 in each CTA's TMEM (two of
// them, so that one is read while the next is summed).  Either operand lies with k or with its rows (m, n) contiguous.  What happens to an accumulator is
// the policy's: its warps read TMEM, 32 rows x 32 columns at a time, a lane's own row of 64 bytes of up to two 16-bit matrices beside it, loaded a chunk ahead, and
// store a lane's row in whole 32-byte sectors, so that all shared memory is left to the operands' stages.  Staged in shared memory and stored through tensor maps
// instead, with a stage less, a product whose epilogue reads two matrices and writes three took 450 us (16384 x 4096 x 4096; here 398), one that writes one 181 to 186 us
// (65536 x 1024 x 2048; 173), one that writes three beside a longer sum 394 to 413 us (2 x 65536 x 2048 x 1024; 406).
//
// Bound: the tensor cores, and over more than some 100 us the power limit under them.  Alone, the products of the gated block run at 1360 to 1610 TFLOP/s, 83 to 98 % of
// a library product's burst rate here (1640), with the tensor pipe 75 to 81 % busy and L2 at 55 and 37 % of its rate.  Call after call, at the power limit (993 W), clocks fall to 1250 MHz: the block's
// forward pass settles at 1150 TFLOP/s, its backward pass at 1237; a library's two products of the forward pass alone, with nothing applied or kept, at 1238 (1425 MHz), of 8192^3 at 1408 (1335 MHz).
//
// TN = 256 is what keeps the tensor cores fed from L2; where there are fewer such tiles than pairs of SMs a narrow form (TN = 64, or 128 for a paired b) has more
// and shorter ones: cost_of() weighs both.  The gradients of a gated block of 333 rows, 509 x 1021: 57 us with the wide form alone, 43 with both.
//
// Roles (12 warps): warp 0 TMA, warp 1 MMA (in the even CTA), warp 2 TMEM, warps 4-11 epilogue (lane quarter x column half).  Every wait is bounded;
// after one has run out all roles go on without touching global memory, the kernel returns and the status word says so.
#pragma once
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"
#include "launchers.h"
#include "runtime.h"
#include "sm100.cuh"

namespace haste {
namespace gemm {

using namespace sm100;

constexpr int TILE = 256;              // rows of a pair's tile
constexpr int KSTEP = 64;              // one 128-byte swizzle row of 16-bit values
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 12 * 32;
constexpr int GROUP_M = 8;             // tiles of m that are walked before the next of n: what runs at once shares its operands in L2

// The narrow form of a policy
template <class Policy>
constexpr int narrow() { return Policy::PAIRED_B ? 128 : 64; }

template <int TN>
struct Layout {
  static constexpr int A_BYTES = 128 * KSTEP * 2;
  static constexpr int B_BYTES = TN / 2 * KSTEP * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 224 * 1024 / STAGE_BYTES;
  static constexpr int OFF_BAR = STAGES * STAGE_BYTES;
  static constexpr int BARRIERS = 2 * STAGES + 4;
  static constexpr int SMEM_BYTES = OFF_BAR + 8 * BARRIERS + 16 + 1024;      // the last for aligning the first stage
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");
};

// ---------------------------------------------------------------- pairs of CTAs
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Address of the same place in the even CTA's shared memory
__device__ __forceinline__ uint32_t leaders(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void arrive_at_leader(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(leaders(bar)) : "memory");
}
// One box into this CTA's shared memory; its bytes count at `bar`, the even CTA's barrier.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const void* tmap, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void umma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives at the barrier of both CTAs when the products issued so far are done
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t smem_dst, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// ---------------------------------------------------------------- what a launch works on
// One product: its sizes, its operands' tensor maps and what the policy reads and writes.
struct Sizes {
  float* partial;                  // fp32 sums of the parts that k was cut into
  int M, N;                        // of the result
  int tiles_m, tiles_n;            // set by launch()
  int splits;
  int steps0, steps;               // steps of k in the first part, and in both
  int first;                       // number of this problem's first tile; set by launch()
};
// A 16-bit matrix of the result's size that the policy reads or writes: rows of ld elements, of which the first `cols` (the result's columns, rounded up to a multiple of 8)
// are read or written and what is behind them is others'.  on: the bytes that base, rows and cols are multiples of, 32 or 16 (with a third form for any, every lane storing its row's values one by one, the weights' gradients of 333 x 509 x 1021 took 43 us, through fp32 parts 12 and 6)
struct Matrix16 {
  uint16_t* p;
  int64_t ld;
  int cols, on;
};
template <class Policy>
struct Problem : Sizes {
  CUtensorMap a[Policy::PARTS], b[Policy::PAIRED_B ? 2 : Policy::PARTS];      // by the part of k; of a paired b by the CTA
  Matrix16 out[Policy::OUTPUTS], in[Policy::INPUTS > 0 ? Policy::INPUTS : 1];
};
template <class Policy, int P>
struct Work {
  Problem<Policy> p[P];
  int problems, tiles;
  float scale0;                    // the policy's
  int* err;
  long long wait_limit;
};
struct Tile {
  int problem, split, m, n;
};

template <class Policy, int P>
__device__ __forceinline__ Tile tile_at(const Work<Policy, P>& w, int t) {
  Tile r;
  r.problem = 0;
  if (P > 1)
    while (r.problem + 1 < w.problems && t >= w.p[r.problem + 1].first) ++r.problem;
  const Sizes& p = w.p[r.problem];
  t -= p.first;
  const int each = p.tiles_m * p.tiles_n;
  r.split = t / each;
  t -= r.split * each;
  const int band = t / (GROUP_M * p.tiles_n), in_band = t - band * GROUP_M * p.tiles_n;
  const int high = min(GROUP_M, p.tiles_m - band * GROUP_M);
  r.n = in_band / high;
  r.m = band * GROUP_M + in_band - r.n * high;
  return r;
}

// ---------------------------------------------------------------- epilogue helpers
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack_bf16(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); }
__device__ __forceinline__ float2 unpack_f16(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ void store_32_bytes(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// 32 columns of a row, packed in pairs: those that the matrix has
__device__ __forceinline__ void store_row(const Matrix16& m, int row, int col, const uint32_t (&v)[16]) {
  uint16_t* to = m.p + static_cast<int64_t>(row) * m.ld + col;
  if (m.on == 32) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (col + 16 * j < m.cols) store_32_bytes(to + 16 * j, v + 8 * j);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + 8 * j < m.cols) *reinterpret_cast<uint4*>(to + 8 * j) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  }
}
// and zeros beyond it
__device__ __forceinline__ void load_row(const Matrix16& m, int row, int col, bool there, uint32_t (&v)[16]) {
  const uint16_t* from = m.p + static_cast<int64_t>(row) * m.ld + col;
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0;
  if (!there) return;
  if (m.on == 32) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (col + 16 * j < m.cols)
        asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v[8 * j]), "=r"(v[8 * j + 1]), "=r"(v[8 * j + 2]), "=r"(v[8 * j + 3]), "=r"(v[8 * j + 4]), "=r"(v[8 * j + 5]), "=r"(v[8 * j + 6]), "=r"(v[8 * j + 7])
                     : "l"(from + 16 * j));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + 8 * j < m.cols) {
        const uint4 q = __ldg(reinterpret_cast<const uint4*>(from + 8 * j));
        v[4 * j] = q.x; v[4 * j + 1] = q.y; v[4 * j + 2] = q.z; v[4 * j + 3] = q.w;
      }
  }
}

// ---------------------------------------------------------------- the kernel
// Policy: A_MN, B_MN (the operand's rows are contiguous, not k), PAIRED_B (each CTA has an operand b of its own: TN / 2 columns of
// two products side by side), PARTS of k, OUTPUTS, INPUTS, and
//   static void chunk<TN>(w, p, tile, row, col, tmem, inputs)   32 columns of this lane's row of the result, accumulator at tmem
template <class Policy, int P, int TN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1) gemm_sm100_kernel(const __grid_constant__ Work<Policy, P> w) {
  using L = Layout<TN>;
  constexpr int STAGES = L::STAGES, TMEM_COLUMNS = 2 * TN;
  constexpr int COLUMNS = Policy::PAIRED_B ? TN / 2 : TN, CHUNKS = COLUMNS / 64;         // columns of the result in a tile, and a warp's chunks of 32 of them
  constexpr bool B_SMALL = Policy::B_MN && TN == 64;         // an operand b of 32 rows with these contiguous has a swizzle of 64 bytes
  extern __shared__ uint8_t raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = smem_u32(sm);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  auto bar_full = [&](int s) { return base + L::OFF_BAR + 8 * s; };
  auto bar_empty = [&](int s) { return base + L::OFF_BAR + 8 * (STAGES + s); };
  auto bar_done = [&](int s) { return base + L::OFF_BAR + 8 * (2 * STAGES + s); };
  auto bar_free = [&](int s) { return base + L::OFF_BAR + 8 * (2 * STAGES + 2 + s); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + L::OFF_BAR + 8 * L::BARRIERS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + L::OFF_BAR + 8 * L::BARRIERS + 8);
  const long long WL = w.wait_limit;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(bar_full(s), 1); mbar_init(bar_empty(s), 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(bar_done(s), 1); mbar_init(bar_free(s), 2 * EPI_WARPS); }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 2) tmem_alloc_pair(smem_u32(tmem_slot), TMEM_COLUMNS);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                // the other CTA's barriers are there, and it has started
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();

  const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;
  if (warp == 0 && lane == 0) {
    // ---------------- loads
    int it = 0;
    for (int t = first; t < w.tiles && !*abort_flag; t += stride) {
      const Tile tl = tile_at(w, t);
      const Problem<Policy>& p = w.p[tl.problem];
      const int k0 = static_cast<int>(static_cast<int64_t>(p.steps) * tl.split / p.splits), k1 = static_cast<int>(static_cast<int64_t>(p.steps) * (tl.split + 1) / p.splits);
      const int am = tl.m * TILE + static_cast<int>(rank) * 128;
      const int bn = Policy::PAIRED_B ? tl.n * (TN / 2) : tl.n * TN + static_cast<int>(rank) * (TN / 2);
      for (int k = k0; k < k1; ++k, ++it) {
        const int s = it % STAGES;
        if (!mbar_wait(bar_empty(s), ((it / STAGES) & 1) ^ 1, abort_flag, w.err, 301, WL)) break;
        if (rank == 0) mbar_arrive_expect_tx(bar_full(s), 2 * L::STAGE_BYTES);
        const uint32_t bar = leaders(bar_full(s));
        const int part = k >= p.steps0;
        const int kc = (part ? k - p.steps0 : k) * KSTEP;
        const uint32_t as = base + s * L::STAGE_BYTES, bs = as + L::A_BYTES;
        const CUtensorMap* ta = &p.a[part];
        const CUtensorMap* tb = &p.b[Policy::PAIRED_B ? static_cast<int>(rank) : part];
        if (Policy::A_MN) {
          tma_load_pair(as, ta, am, kc, 0, bar);
          tma_load_pair(as + L::A_BYTES / 2, ta, am + 64, kc, 0, bar);
        } else {
          tma_load_pair(as, ta, kc, am, 0, bar);
        }
        if (Policy::B_MN) {
          tma_load_pair(bs, tb, bn, kc, 0, bar);
          if (TN == 256) tma_load_pair(bs + L::B_BYTES / 2, tb, bn + 64, kc, 0, bar);
        } else {
          tma_load_pair(bs, tb, kc, bn, 0, bar);
        }
      }
    }
    // The last arrivals at this CTA's barriers come from the even one's products: they are in before the CTA may go.
    for (int i = it > STAGES ? it - STAGES : 0; i < it; ++i) mbar_wait(bar_empty(i % STAGES), (i / STAGES) & 1, abort_flag, w.err, 302, WL);
  } else if (warp == 1 && rank == 0) {
    // ---------------- products
    constexpr uint32_t FORMAT = (1u << 7) | (1u << 10);          // both operands bf16
    constexpr uint32_t IDESC = (1u << 4) | FORMAT | (static_cast<uint32_t>(Policy::A_MN) << 15) | (static_cast<uint32_t>(Policy::B_MN) << 16) |
                               (static_cast<uint32_t>(TN >> 3) << 17) | (static_cast<uint32_t>(TILE >> 4) << 24);
    const uint64_t da = make_sdesc(base, Policy::A_MN ? L::A_BYTES / 2 : 16, 1024);
    const uint64_t db = B_SMALL ? make_sdesc64(base + L::A_BYTES, 16, 512) : make_sdesc(base + L::A_BYTES, Policy::B_MN ? L::B_BYTES / 2 : 16, 1024);
    constexpr uint64_t KA = Policy::A_MN ? 2048 >> 4 : 32 >> 4, KB = B_SMALL ? 1024 >> 4 : Policy::B_MN ? 2048 >> 4 : 32 >> 4;
    int it = 0, n = 0;
    for (int t = first; t < w.tiles; t += stride, ++n) {
      const Tile tl = tile_at(w, t);
      const Problem<Policy>& p = w.p[tl.problem];
      const int steps = static_cast<int>(static_cast<int64_t>(p.steps) * (tl.split + 1) / p.splits) - static_cast<int>(static_cast<int64_t>(p.steps) * tl.split / p.splits);
      const int buf = n & 1;
      if (!mbar_wait(bar_free(buf), ((n >> 1) & 1) ^ 1, abort_flag, w.err, 303, WL)) break;
      tc_fence_after();
      bool ok = true;
      for (int k = 0; k < steps; ++k, ++it) {
        const int s = it % STAGES;
        ok = mbar_wait(bar_full(s), (it / STAGES) & 1, abort_flag, w.err, 304, WL);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t off = static_cast<uint64_t>((s * L::STAGE_BYTES) >> 4);
#pragma unroll
          for (int j = 0; j < KSTEP / 16; ++j) umma_pair(tmem + buf * TN, da + off + j * KA, db + off + j * KB, IDESC, (k | j) != 0);
          commit_pair(bar_empty(s));
        }
        __syncwarp();
      }
      if (!ok) break;
      if (elect_one()) commit_pair(bar_done(buf));
      __syncwarp();
    }
  } else if (warp >= 4) {
    // ---------------- epilogue
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    constexpr int INPUTS = Policy::INPUTS > 0 ? Policy::INPUTS : 1;
    int n = 0;
    for (int t = first; t < w.tiles; t += stride, ++n) {
      const Tile tl = tile_at(w, t);
      const Problem<Policy>& p = w.p[tl.problem];
      const int buf = n & 1, row = tl.m * TILE + static_cast<int>(rank) * 128 + quarter * 32 + lane, at = half * (COLUMNS / 2), col0 = tl.n * COLUMNS + at;
      uint32_t in[INPUTS][16], ahead[INPUTS][16];
      if (Policy::INPUTS > 0) {
#pragma unroll
        for (int i = 0; i < INPUTS; ++i) load_row(p.in[i], row, col0, row < p.M, ahead[i]);
      }
      bool ok = mbar_wait(bar_done(buf), (n >> 1) & 1, abort_flag, w.err, 305, WL);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
#pragma unroll 1
      for (int j = 0; j < CHUNKS; ++j) {
        if (Policy::INPUTS > 0) {
#pragma unroll
          for (int i = 0; i < INPUTS; ++i) {
#pragma unroll
            for (int e = 0; e < 16; ++e) in[i][e] = ahead[i][e];
            if (j + 1 < CHUNKS) load_row(p.in[i], row, col0 + 32 * (j + 1), row < p.M, ahead[i]);
          }
        }
        __syncwarp();                // TMEM is read by whole warps
        Policy::template chunk<TN>(w, p, tl, row, col0 + 32 * j, tmem + buf * TN + (static_cast<uint32_t>(quarter * 32) << 16) + at + 32 * j, in);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_at_leader(bar_free(buf));
    }
  }

  // ---------------- teardown.  After an abort copies may be on their way into this CTA's shared memory, and products into its TMEM: they have some
  // milliseconds, thousands of times what they need.
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < (1ll << 24)) __nanosleep(1000);
  }
  cluster_sync_all();
  tc_fence_after();
  if (warp == 2) tmem_dealloc_pair(tmem, TMEM_COLUMNS);
}

// ---------------------------------------------------------------- host side
// A batch of 16-bit matrices [outer][inner] as a tensor map; base and strides are multiples of 16 bytes.
inline int make_map(CUtensorMap* out, const void* base, bool f16, int64_t inner, int64_t outer, int64_t batch, int64_t ld, int64_t batch_stride, int box_inner, int box_outer) {
  return make_tmap_16bit_3d(out, base, f16, inner, outer, batch, ld * 2, (batch_stride ? batch_stride : ld * outer) * 2, static_cast<uint32_t>(box_inner), static_cast<uint32_t>(box_outer));
}
// Where a 16-bit matrix lies
struct Operand {
  const void* p;
  int64_t ld;
};
// Operand a of `rows` (the result's M) and b of `rows` (its N), k values each; inputs and outputs of the result's size
template <class Policy, int TN>
int map_a(CUtensorMap* out, const Operand& o, int64_t rows, int64_t k) {
  return Policy::A_MN ? make_map(out, o.p, false, rows, k, 1, o.ld, 0, 64, 64) : make_map(out, o.p, false, k, rows, 1, o.ld, 0, 64, 128);
}
template <class Policy, int TN>
int map_b(CUtensorMap* out, const Operand& o, int64_t rows, int64_t k) {
  return Policy::B_MN ? make_map(out, o.p, false, rows, k, 1, o.ld, 0, TN == 64 ? 32 : 64, 64)
                      : make_map(out, o.p, false, k, rows, 1, o.ld, 0, 64, TN / 2);
}
inline Matrix16 result(const Operand& o, int64_t columns) {
  const int cols = static_cast<int>((columns + 7) & ~int64_t(7));
  return {static_cast<uint16_t*>(const_cast<void*>(o.p)), o.ld, cols, o.ld % 16 == 0 && cols % 16 == 0 && reinterpret_cast<uintptr_t>(o.p) % 32 == 0 ? 32 : 16};
}
inline int64_t steps_of(int64_t k) { return (k + KSTEP - 1) / KSTEP; }

// Pairs of CTAs that may run at once on the current device.  The first call on a device allows the kernel its shared memory there, which its launches need.
template <auto KERNEL>                 // (the address: kernels of one type have their own)
int pairs_resident(int smem, int* pairs) {
  static std::atomic<int> cached[64];
  int dev = 0;
  cudaGetDevice(&dev);
  const bool keep = dev >= 0 && dev < 64;
  if (keep && (*pairs = cached[dev].load(std::memory_order_acquire)) > 0) return HASTE_OK;
  const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return fail(HASTE_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(sm_count() & ~1));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, KERNEL, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    *pairs = sm_count() / 2;
    return HASTE_OK;
  }
  *pairs = n < sm_count() / 2 ? n : sm_count() / 2;
  if (keep) cached[dev].store(*pairs, std::memory_order_release);
  return HASTE_OK;
}

// Time of a launch of `tiles` tiles of `steps` steps of k each, in units of a step of the wide form (0.28 us).  Both forms, us a call (all launches of a call in the form, or as the rule has them):
//                                        rule   wide  narrow                                     rule   wide  narrow
//   forward       40 x  512 x 1024       14.9   17.8    14.9      steps, one   64 x 64            72.2  101.7    72.1
//                 64 x  768 x 2048       16.4   20.0    16.4                  512 x 768          117.7  149.2   117.1
//                333 x 1024 x 2048       21.4   25.2    21.3                 1024 x 1024         178.2  186.7   172.6
//               1024 x  768 x 2048       23.3   26.2    24.4                 2048 x 2048         354.9  338.9   445.2
//               1024 x 4096 x 4096       78.8   79.2   127.0      steps,  4 of 768 x 768         175.9  175.0   174.5
//               2048 x 1024 x 2048       36.9   36.8    43.8               20 of 256 x 512       144.7  144.9   139.9
//               4096 x 1024 x 2048       48.8   47.7    71.9               40 of 256 x 512       173.4  174.2   186.9
//              16384 x 1024 x 2048      158.5  159.0   246.3               40 of 512 x 512       249.2  250.7   434.8
//   gradients     40 x  512 x 1024       23.1   28.3    23.0              100 of  64 x 128       105.7  136.6   105.6
//                 64 x  768 x 2048       24.7   31.5    27.7
//                333 x 1024 x 2048       36.1   42.9    42.0
//               1024 x  768 x 2048       47.0   45.2    56.3
//               4096 x 1024 x 2048      106.2  106.5   212.8
//              16384 x 1024 x 2048      369.9  404.7   825.6
// It is 5 % off where both are close: it does not know of the parts that an epilogue of fp32 stores, nor that narrow tiles of Newton-Schulz wait for fewer others.
inline double cost_of(int64_t tiles, int64_t steps, bool is_narrow, int64_t pairs) {
  return static_cast<double>((tiles + pairs - 1) / pairs) * (is_narrow ? 0.6 * static_cast<double>(steps) + 3.5 : static_cast<double>(steps) + 6.0);
}
inline int64_t tiles_for(int64_t M, int64_t N, int64_t columns) { return ((M + TILE - 1) / TILE) * ((N + columns - 1) / columns); }

// Launches what is in w.p[0 .. problems): tiles are counted here.  behind: the kernel before it in the stream is one of the same call.
template <class Policy, int TN, int P>
int launch(Work<Policy, P>& w, bool behind, cudaStream_t st) {
  using L = Layout<TN>;
  constexpr int COLUMNS = Policy::PAIRED_B ? TN / 2 : TN;
  constexpr auto kernel = &gemm_sm100_kernel<Policy, P, TN>;
  int64_t tiles = 0;
  for (int i = 0; i < w.problems; ++i) {
    Sizes& p = w.p[i];
    p.tiles_m = (p.M + TILE - 1) / TILE;
    p.tiles_n = (p.N + COLUMNS - 1) / COLUMNS;
    if (static_cast<int64_t>(p.tiles_m) * p.tiles_n > 0x3FFFFFFF) return fail(HASTE_ERR_TOO_LARGE, "too many tiles for one launch");
    p.first = static_cast<int>(tiles);
    tiles += static_cast<int64_t>(p.tiles_m) * p.tiles_n * p.splits;
    if (tiles > 0x3FFFFFFF) return fail(HASTE_ERR_TOO_LARGE, "too many tiles for one launch");
  }
  if (tiles == 0) return HASTE_OK;
  w.tiles = static_cast<int>(tiles);
  if (int rc = device_status_word(&w.err)) return rc;
  w.wait_limit = wait_limit_cycles();
  int pairs = 0;
  if (int rc = pairs_resident<kernel>(L::SMEM_BYTES, &pairs)) return rc;
  pairs = static_cast<int>(imin64(pairs, tiles));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = L::SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = behind ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, w);
  if (e != cudaSuccess) return fail(HASTE_ERR_LAUNCH, "cudaLaunchKernelEx: %s", cudaGetErrorString(e));
  return HASTE_OK;
}

}  // namespace gemm
}  // namespace haste
