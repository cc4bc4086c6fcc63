// Dense products for the operators in front of the sparse layer: one persistent kernel over the tiles of several products, two SMs to a tile.
//
//   acc[m, n] = sum_k a[m, k] b[n, k]        (a second pair of operands may go on where the first ends)
//
// A cluster of two CTAs has a tile of 256 x 256: each loads its half of both operands by TMA (128 rows of a, 128 of b, 64 along k), the even one
// issues tcgen05.mma.cta_group::2, whose operands are both CTAs' shared memory and whose accumulator is 128 x 256 fp32 in each CTA's TMEM (two of
// them, so that one is read while the next is summed).  Either operand lies with k or with its rows (m, n) contiguous.  What happens to an accumulator is
// the policy's: its warps read TMEM, 32 rows x 32 columns at a time, and hand 16-bit tiles of that size to tensor-map stores.
//
// Roles (12 warps): warp 0 TMA, warp 1 MMA (in the even CTA), warp 2 TMEM, warps 4-11 epilogue (lane quarter x column half).  Every wait is bounded;
// after one has run out all roles go on without touching global memory, the kernel returns and the status word says so.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "launchers.h"
#include "runtime.h"
#include "sm100.cuh"

namespace haste {
namespace gemm {

using namespace sm100;

constexpr int TILE = 256;              // of the pair, both ways
constexpr int KSTEP = 64;              // one 128-byte swizzle row of 16-bit values
constexpr int HALF_BYTES = 128 * KSTEP * 2;
constexpr int STAGE_BYTES = 2 * HALF_BYTES;
constexpr int STAGES = 5;
constexpr int EPI_WARPS = 8;
constexpr int BOX_BYTES = 32 * 32 * 2; // what a warp stages for one store
constexpr int BOXES = 4;               // per warp, in turn
constexpr int THREADS = 12 * 32;
constexpr int OFF_EPI = STAGES * STAGE_BYTES;
constexpr int OFF_BAR = OFF_EPI + EPI_WARPS * BOXES * BOX_BYTES;
constexpr int SMEM_BYTES = OFF_BAR + 256 + 1024;      // the last for aligning the first stage
constexpr int GROUP_M = 8;             // tiles of m that are walked before the next of n: what runs at once shares its operands in L2

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
__device__ __forceinline__ void tma_store_3d(const void* tmap, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(tmap), "r"(x), "r"(y), "r"(z), "r"(src)
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
// One product, or a batch of products of one shape.
struct Problem {
  CUtensorMap a[2], b[2];          // first and second part of k; a policy with two operands b (one for each CTA) has them in b
  CUtensorMap out[3];
  const uint16_t* in[2];           // 16-bit matrices that the policy reads at the tile's place
  float* partial;                  // fp32 sums of the parts that k was cut into
  int64_t ld_in, batch_in;         // strides of `in` in elements
  int M, N;
  int tiles_m, tiles_n;            // tiles_n < 0: symmetric, only tiles with n <= m
  int batch, splits;
  int steps0, steps;               // steps of k in the first part, and in both
  int first;                       // number of this problem's first tile
};
template <int P>
struct Work {
  Problem p[P];
  int problems, tiles;
  float scale0, scale1;            // the policy's factors
  int* err;
  long long wait_limit;
};
struct Tile {
  int problem, batch, split, m, n;
};

__host__ __device__ inline int tiles_of(const Problem& p) { return p.tiles_n < 0 ? p.tiles_m * (p.tiles_m + 1) / 2 : p.tiles_m * p.tiles_n; }

template <int P>
__device__ __forceinline__ Tile tile_at(const Work<P>& w, int t) {
  Tile r;
  r.problem = 0;
  if (P > 1)
    while (r.problem + 1 < w.problems && t >= w.p[r.problem + 1].first) ++r.problem;
  const Problem& p = w.p[r.problem];
  t -= p.first;
  const int each = tiles_of(p);
  const int bs = t / each;
  t -= bs * each;
  r.batch = bs / p.splits;
  r.split = bs - r.batch * p.splits;
  if (p.tiles_n < 0) {
    int m = static_cast<int>((sqrtf(8.f * static_cast<float>(t) + 1.f) - 1.f) * 0.5f);
    while (m * (m + 1) / 2 > t) --m;
    while ((m + 1) * (m + 2) / 2 <= t) ++m;
    r.m = m;
    r.n = t - m * (m + 1) / 2;
  } else {
    const int band = t / (GROUP_M * p.tiles_n), in_band = t - band * GROUP_M * p.tiles_n;
    const int high = min(GROUP_M, p.tiles_m - band * GROUP_M);
    r.n = in_band / high;
    r.m = band * GROUP_M + in_band - r.n * high;
  }
  return r;
}

// ---------------------------------------------------------------- epilogue helpers
// A warp's boxes of 32 rows x 32 16-bit columns on their way to memory (64-byte swizzle: 16-byte chunk j of row r at j ^ (r / 2 % 4)).
struct Stager {
  uint32_t base;
  int lane, next;
  // The next free box
  __device__ __forceinline__ uint32_t get() {
    if (lane == 0) bulk_wait_read<BOXES - 1>();
    __syncwarp();
    const uint32_t at = base + next * BOX_BYTES;
    next = (next + 1) % BOXES;
    return at;
  }
  __device__ __forceinline__ void put(const void* tmap, uint32_t box, int x, int y, int z, bool inside) {
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) {
      if (inside) tma_store_3d(tmap, box, x, y, z);
      bulk_commit();
    }
  }
};
__device__ __forceinline__ void st_shared_v4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void st_shared_u16(uint32_t at, uint32_t v) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(static_cast<uint16_t>(v)) : "memory");
}
// Row `lane` of a box: 32 values packed in pairs
__device__ __forceinline__ void box_row(uint32_t box, int lane, const uint32_t (&p)[16]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) st_shared_v4(box + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4), p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]);
}
// Column `lane` of a box
__device__ __forceinline__ void box_column(uint32_t box, int lane, const uint32_t (&p)[16]) {
#pragma unroll
  for (int c = 0; c < 32; ++c)
    st_shared_u16(box + c * 64 + (((lane >> 3) ^ ((c >> 1) & 3)) << 4) + (lane & 7) * 2, c & 1 ? p[c >> 1] >> 16 : p[c >> 1] & 0xFFFFu);
}
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
// 32 16-bit values of one row, packed in pairs; zeros beyond the row's `cols`, a multiple of 8 (rows are padded), and where !there
__device__ __forceinline__ void load_row(uint32_t (&v)[16], const uint16_t* row, int col, int64_t cols, bool there) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint4 q = make_uint4(0, 0, 0, 0);
    if (there && col + 8 * j < cols) q = *reinterpret_cast<const uint4*>(row + col + 8 * j);
    v[4 * j] = q.x; v[4 * j + 1] = q.y; v[4 * j + 2] = q.z; v[4 * j + 3] = q.w;
  }
}

// ---------------------------------------------------------------- the kernel
// Policy: A_MN, B_MN (the operand's rows are contiguous, not k), F16 (else bf16), PAIRED_B (each CTA has an operand b of its own: 128 columns of
// two products side by side), and
//   static void epilogue(w, p, tile, row0, col0, column half, tmem, stager, lane)   one warp's part of a tile
template <class Policy, int P>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1) gemm_sm100_kernel(const __grid_constant__ Work<P> w) {
  extern __shared__ uint8_t raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = smem_u32(sm);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  auto bar_full = [&](int s) { return base + OFF_BAR + 8 * s; };
  auto bar_empty = [&](int s) { return base + OFF_BAR + 8 * (STAGES + s); };
  auto bar_done = [&](int s) { return base + OFF_BAR + 8 * (2 * STAGES + s); };
  auto bar_free = [&](int s) { return base + OFF_BAR + 8 * (2 * STAGES + 2 + s); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + OFF_BAR + 8 * (2 * STAGES + 4));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + OFF_BAR + 8 * (2 * STAGES + 4) + 8);
  const long long WL = w.wait_limit;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(bar_full(s), 1); mbar_init(bar_empty(s), 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(bar_done(s), 1); mbar_init(bar_free(s), 2 * EPI_WARPS); }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 2) tmem_alloc_pair(smem_u32(tmem_slot), 512);
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
      const Problem& p = w.p[tl.problem];
      const int k0 = static_cast<int>(static_cast<int64_t>(p.steps) * tl.split / p.splits), k1 = static_cast<int>(static_cast<int64_t>(p.steps) * (tl.split + 1) / p.splits);
      const int am = tl.m * TILE + static_cast<int>(rank) * 128;
      const int bn = Policy::PAIRED_B ? tl.n * 128 : tl.n * TILE + static_cast<int>(rank) * 128;
      for (int k = k0; k < k1; ++k, ++it) {
        const int s = it % STAGES;
        if (!mbar_wait(bar_empty(s), ((it / STAGES) & 1) ^ 1, abort_flag, w.err, 301, WL)) break;
        if (rank == 0) mbar_arrive_expect_tx(bar_full(s), 2 * STAGE_BYTES);
        const uint32_t bar = leaders(bar_full(s));
        const int part = k >= p.steps0;
        const int kc = (part ? k - p.steps0 : k) * KSTEP;
        const uint32_t as = base + s * STAGE_BYTES, bs = as + HALF_BYTES;
        const CUtensorMap* ta = &p.a[part];
        const CUtensorMap* tb = &p.b[Policy::PAIRED_B ? static_cast<int>(rank) : part];
        if (Policy::A_MN) {
          tma_load_pair(as, ta, am, kc, tl.batch, bar);
          tma_load_pair(as + HALF_BYTES / 2, ta, am + 64, kc, tl.batch, bar);
        } else {
          tma_load_pair(as, ta, kc, am, tl.batch, bar);
        }
        if (Policy::B_MN) {
          tma_load_pair(bs, tb, bn, kc, tl.batch, bar);
          tma_load_pair(bs + HALF_BYTES / 2, tb, bn + 64, kc, tl.batch, bar);
        } else {
          tma_load_pair(bs, tb, kc, bn, tl.batch, bar);
        }
      }
    }
    // The last arrivals at this CTA's barriers come from the even one's products: they are in before the CTA may go.
    for (int i = it > STAGES ? it - STAGES : 0; i < it; ++i) mbar_wait(bar_empty(i % STAGES), (i / STAGES) & 1, abort_flag, w.err, 302, WL);
  } else if (warp == 1 && rank == 0) {
    // ---------------- products
    constexpr uint32_t FORMAT = Policy::F16 ? 0u : (1u << 7) | (1u << 10);
    constexpr uint32_t IDESC = (1u << 4) | FORMAT | (static_cast<uint32_t>(Policy::A_MN) << 15) | (static_cast<uint32_t>(Policy::B_MN) << 16) |
                               (static_cast<uint32_t>(TILE >> 3) << 17) | (static_cast<uint32_t>(TILE >> 4) << 24);
    const uint64_t da = make_sdesc(base, Policy::A_MN ? HALF_BYTES / 2 : 16, 1024), db = make_sdesc(base + HALF_BYTES, Policy::B_MN ? HALF_BYTES / 2 : 16, 1024);
    constexpr uint64_t KA = Policy::A_MN ? 2048 >> 4 : 32 >> 4, KB = Policy::B_MN ? 2048 >> 4 : 32 >> 4;
    int it = 0, n = 0;
    for (int t = first; t < w.tiles; t += stride, ++n) {
      const Tile tl = tile_at(w, t);
      const Problem& p = w.p[tl.problem];
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
          const uint64_t off = static_cast<uint64_t>((s * STAGE_BYTES) >> 4);
#pragma unroll
          for (int j = 0; j < KSTEP / 16; ++j) umma_pair(tmem + buf * TILE, da + off + j * KA, db + off + j * KB, IDESC, (k | j) != 0);
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
    Stager st = {base + OFF_EPI + static_cast<uint32_t>(warp - 4) * BOXES * BOX_BYTES, lane, 0};
    int n = 0;
    for (int t = first; t < w.tiles; t += stride, ++n) {
      const Tile tl = tile_at(w, t);
      const int buf = n & 1;
      const bool ok = mbar_wait(bar_done(buf), (n >> 1) & 1, abort_flag, w.err, 305, WL);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      Policy::epilogue(w, w.p[tl.problem], tl, tl.m * TILE + static_cast<int>(rank) * 128 + quarter * 32, half,
                       tmem + buf * TILE + (static_cast<uint32_t>(quarter * 32) << 16), st, lane);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_at_leader(bar_free(buf));
    }
    if (lane == 0) bulk_wait<0>();
    __syncwarp();
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
  if (warp == 2) tmem_dealloc_pair(tmem, 512);
}

// ---------------------------------------------------------------- host side
// A batch of 16-bit matrices [outer][inner] as a tensor map.  An operand with k contiguous: inner = k, box 64 x 128; with its rows contiguous: inner =
// rows, box 64 x 64; stores: box 32 x 32.  Base and strides are multiples of 16 bytes.
enum Box { BOX_K, BOX_MN, BOX_STORE };
inline int make_map(CUtensorMap* out, const void* base, bool f16, int64_t inner, int64_t outer, int64_t batch, int64_t ld, int64_t batch_stride, Box box) {
  return make_tmap_16bit_3d(out, base, f16, inner, outer, batch, ld * 2, (batch_stride ? batch_stride : ld * outer) * 2, box == BOX_STORE ? 32 : 64,
                            box == BOX_STORE ? 32 : box == BOX_K ? 128 : 64);
}

// CTAs that a launch of pairs may have at once on the current device
template <class K>
int pairs_resident(K kernel) {
  static int cached[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && cached[dev] > 0) return cached[dev];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(sm_count() & ~1));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    return sm_count() / 2;
  }
  if (dev >= 0 && dev < 64) cached[dev] = n;
  return n;
}

// Launches what is in w.p[0 .. problems): tiles are counted here.  behind: the kernel before it in the stream is one of the same call.
template <class Policy, int P>
int launch(Work<P>& w, bool behind, cudaStream_t st) {
  auto kernel = gemm_sm100_kernel<Policy, P>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
  if (e != cudaSuccess) return fail(HASTE_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  int64_t tiles = 0;
  for (int i = 0; i < w.problems; ++i) {
    w.p[i].first = static_cast<int>(tiles);
    tiles += static_cast<int64_t>(tiles_of(w.p[i])) * w.p[i].batch * w.p[i].splits;
    if (tiles > 0x3FFFFFFF) return fail(HASTE_ERR_TOO_LARGE, "too many tiles for one launch");
  }
  if (tiles == 0) return HASTE_OK;
  w.tiles = static_cast<int>(tiles);
  if (int rc = device_status_word(&w.err)) return rc;
  w.wait_limit = wait_limit_cycles();
  const int pairs = static_cast<int>(imin64(pairs_resident(kernel), tiles));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = behind ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, kernel, w);
  if (e != cudaSuccess) return fail(HASTE_ERR_LAUNCH, "cudaLaunchKernelEx: %s", cudaGetErrorString(e));
  return HASTE_OK;
}

}  // namespace gemm
}  // namespace haste
