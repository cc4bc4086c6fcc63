// All Newton-Schulz steps over many matrices in one launch:  steps times  A = X X^T,  B = a I + b A + c A A,  X <- B X   (X [p, q], p and q multiples of 64)
//
// The three products of all steps are one list of tiles, which the pairs of CTAs take in turn.  A tile may be worked on when the matrix's product before it is complete:
// every warp that has stored its part of a tile adds one to the matrix's counter, and who needs the result waits for the count.  (A launch for each product left a quarter of
// the SMs without work in the last tiles of 5, and took 3 us and the first loads' latency each time.)
//
// The list walks the matrices in groups: a group's A tiles, its B tiles, its X tiles, the next step, ..., then the next group.  Groups are large enough that what a tile waits for
// was begun a product earlier by others (see GROUP_BYTES).
// Every tile's predecessors stand before it in the list, a pair draws the next tile's number from a counter when it runs, and it works on its tiles in that order: the first unfinished
// tile is with a pair that runs and has nothing before it, so it can always proceed, however many pairs of the launch run at once: it is an ordinary launch, not a cooperative one, which
// a device may refuse.  Waits are bounded as everywhere.
//
// A and B are symmetric: only tiles on and below the diagonal are computed and stored.  Where an operand's block lies above it, the block on the other side is loaded and
// read by the tensor core with its rows and columns exchanged.
//
// Bound, many matrices: 50 M elements in matrices of 768 x 768 and 768 x 2048, 5 steps: 860 us, 830 TFLOP/s, 61 % of what a library's product sustains; 101 M of 1024 x 1024 and 1024 x 2048: 1909 us, 1030.
// Products alone, without inputs and stores, take two thirds of that with these stages: the rest is stores into lines that L2 keeps for both dies, and waits for what they
// count.  Nothing is at its rate meanwhile: tensor pipe 57 % busy, L2 at 53 % (11.4 GB), DRAM at 41 % (2.6 GB).  Bound, one matrix: latency; 512 x 768 110 us, 15 products of 7.3: 1.1 from the count to the first operands, 1.7 until the last of them has come at an SM's share of L2's rate,
// 1 for the epilogue, 1 until its stores have arrived, 1 until the count has and is seen.
//
// Tiles are 256 x TN of a pair, with roles, barriers and an epilogue as in gemm_sm100.cuh; warp 3 looks up what comes next and waits for it, ahead of the others.
#pragma once
#include "gemm_sm100.cuh"

namespace haste {
namespace newton_schulz {

using namespace sm100;
using gemm::EPI_WARPS;
using gemm::KSTEP;
using gemm::THREADS;
using gemm::TILE;

constexpr float X_SCALE = 256.f;       // X is kept times this in fp16
constexpr float LO_SCALE = 2048.f;     // and its lower part times this as well
// What X is rounded to after the last but two steps is amplified by two steps at most (12 times), which leaves 2^-12 of its values where the products' own roundings
// are: its lower part is kept up to there.
constexpr int STEPS_WITHOUT_LOWER = 2;
__host__ __device__ constexpr bool has_lower(int step, int steps) { return step == 0 || step < steps - STEPS_WITHOUT_LOWER; }       // X before this step

// Tensor maps of a batch of matrices of one shape: X's two buffers as operand a and b with k contiguous and as operand b with its rows contiguous, A and B as operand a (A's also b)
// either way, and boxes of 32 x 32 of A, B, X and X's lower part for stores.  In the wide form operands a and b are alike.  A is kept where the next X will be, so there are two of its maps too.
enum Map { X_A, X_N = 2, X_BOX = 4, A_A = 6, A_T = 8, A_BOX = 10, B_A = 12, B_T, B_BOX, LO_BOX, MAPS_WIDE, X_B = 16, A_B = 18, A_TB = 20, MAPS_NARROW = 22 };

struct Info {
  int p, q, tiles_m, tiles_n, tiles_q; // tiles_n: columns' tiles of A and B, tiles_q: of X
  int symmetric, full;                 // tiles of A or B, and of X, in a matrix
  uint16_t *x[2], *low, *b;            // X's buffers (A is in the other one), its lower part, B
};
struct Segment {                       // neighbouring matrices of one shape in a group
  int shape, batch, count, matrix;     // first batch entry, how many, number of the first matrix
  int symmetric0, full0;               // tiles of the group before it
};
struct Group {
  int first;                           // tile number
  int segment, end;                    // its segments
  int symmetric, full;                 // tiles of a product of all of it
};
template <int TN>
struct Steps {
  static constexpr int MAPS = TN == TILE ? static_cast<int>(MAPS_WIDE) : static_cast<int>(MAPS_NARROW);
  static constexpr int SHAPES = TN == TILE ? 14 : 10, SEGMENTS = 64, GROUPS = 32;
  CUtensorMap map[SHAPES][MAPS];
  Info info[SHAPES];
  Segment segment[SEGMENTS];
  Group group[GROUPS];
  int groups, tiles, steps;
  float a, b, c;
  unsigned long long* done;            // by matrix
  unsigned long long* drawn;           // numbers of tiles, from `base` on
  unsigned long long base;
  int* err;
  long long wait_limit;
};

struct Task {
  int shape, batch, matrix, m, n, phase, step;
  unsigned long long need;             // of the matrix's counter
};

template <int TN>
__device__ __forceinline__ Task task_at(const Steps<TN>& w, int t, int& g) {
  constexpr int PER = TILE / TN;
  while (g + 1 < w.groups && t >= w.group[g + 1].first) ++g;
  const Group& gr = w.group[g];
  Task r;
  t -= gr.first;
  const int per = 2 * gr.symmetric + gr.full;
  r.step = t / per;
  t -= r.step * per;
  r.phase = t < gr.symmetric ? 0 : t < 2 * gr.symmetric ? 1 : 2;
  t -= r.phase * gr.symmetric;
  int s = gr.segment;
  while (s + 1 < gr.end && t >= (r.phase < 2 ? w.segment[s + 1].symmetric0 : w.segment[s + 1].full0)) ++s;
  const Segment& sg = w.segment[s];
  const Info& info = w.info[sg.shape];
  t -= r.phase < 2 ? sg.symmetric0 : sg.full0;
  const int each = r.phase < 2 ? info.symmetric : info.full, i = t / each;
  t -= i * each;
  r.shape = sg.shape;
  r.batch = sg.batch + i;
  r.matrix = sg.matrix + i;
  if (r.phase < 2) {
    // rows of tiles grow by PER until they are as wide as the matrix
    int m = static_cast<int>((sqrtf(8.f * static_cast<float>(t / PER) + 1.f) - 1.f) * 0.5f);
    while (m * (m + 1) / 2 * PER > t) --m;
    while ((m + 1) * (m + 2) / 2 * PER <= t) ++m;
    r.m = m;
    r.n = t - m * (m + 1) / 2 * PER;
  } else {
    r.n = t / info.tiles_m;
    r.m = t - r.n * info.tiles_m;
  }
  const unsigned long long whole = 2ull * info.symmetric + info.full;
  r.need = (r.step * whole + static_cast<unsigned long long>(r.phase) * info.symmetric) * (2 * EPI_WARPS);
  return r;
}

// 32 columns of a row of what other SMs may have written
__device__ __forceinline__ void load_row(const uint16_t* p, uint32_t* v) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t* r = v + 8 * j;
    asm volatile("ld.relaxed.gpu.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "l"(p + 16 * j) : "memory");
  }
}
__device__ __forceinline__ void tma_store_3d(const void* tmap, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(tmap), "r"(x), "r"(y), "r"(z), "r"(src)
               : "memory");
}
// A warp's box of 32 rows x 32 columns (64-byte swizzle: 16-byte piece j of row r at j ^ (r / 2 % 4)), and on its way to memory
constexpr int BOX_BYTES = 32 * 32 * 2;
__device__ __forceinline__ void fill_box(uint32_t box, int lane, const uint32_t (&p)[16]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t at = box + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(p[4 * j]), "r"(p[4 * j + 1]), "r"(p[4 * j + 2]), "r"(p[4 * j + 3]) : "memory");
  }
}

// ---------------------------------------------------------------- counters
__device__ __forceinline__ unsigned long long load_acquire(const unsigned long long* p) {
  unsigned long long v;
  asm volatile("ld.acquire.gpu.global.b64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void fence_proxy_async_all() { asm volatile("fence.proxy.async;" ::: "memory"); }
// Until the count is there: what was stored before it may then be read, by copies too
__device__ __noinline__ bool wait_count(const unsigned long long* p, unsigned long long need, volatile int* abort_flag, int* err, int code, long long limit) {
  const long long t0 = clock64();
  while (load_acquire(p) < need) {
    if (*abort_flag) return false;
    if (clock64() - t0 > limit) {
      *abort_flag = 1;
      if (err != nullptr) *reinterpret_cast<volatile int*>(err) = code;
      return false;
    }
    __nanosleep(32);
  }
  fence_proxy_async_all();
  return true;
}
// What this thread's stores (bulk groups) wrote, once it has waited for them, is there for whoever sees the count: the addition releases it, a second fence before it took 50 us of 1230
// for steps over 50 M elements and 5 of 124 for one matrix of 512 x 768
__device__ __forceinline__ void add_count(unsigned long long* p) {
  fence_proxy_async_all();
  asm volatile("red.release.gpu.global.add.u64 [%0], %1;" ::"l"(p), "l"(1ull) : "memory");
}

// The next tile's number
template <int TN>
__device__ __forceinline__ int draw(const Steps<TN>& w) {
  const unsigned long long n = atomicAdd(w.drawn, 1ull) - w.base;
  return n < static_cast<unsigned long long>(w.tiles) ? static_cast<int>(n) : w.tiles;
}
// A number into the odd CTA's shared memory, where its arrival counts at a barrier
__device__ __forceinline__ void send(uint32_t to, int value, uint32_t bar) {
  uint32_t there, bar_there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 1;" : "=r"(there) : "r"(to));
  asm volatile("mapa.shared::cluster.u32 %0, %1, 1;" : "=r"(bar_there) : "r"(bar));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.u32 [%0], %1, [%2];" ::"r"(there), "r"(value), "r"(bar_there) : "memory");
}

// ---------------------------------------------------------------- the kernel
template <int TN>
struct Layout {
  static constexpr int A_BYTES = 128 * KSTEP * 2, B_BYTES = TN / 2 * KSTEP * 2, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int TASKS = 4, CHUNKS = TN / 64, BOXES = 2, EPI_BYTES = EPI_WARPS * BOXES * BOX_BYTES, STAGES = (224 * 1024 - EPI_BYTES) / STAGE_BYTES;
  static constexpr int OFF_EPI = STAGES * STAGE_BYTES;
  static constexpr int OFF_TASK = OFF_EPI + EPI_BYTES;
  static constexpr int OFF_MAIL = OFF_TASK + TASKS * 64;
  static constexpr int OFF_BAR = OFF_MAIL + TASKS * 8;
  static constexpr int BARRIERS = 2 * STAGES + 4 + 4 * TASKS;
  static constexpr int SMEM_BYTES = OFF_BAR + 8 * BARRIERS + 16 + 1024;
  static_assert(SMEM_BYTES <= 227 * 1024 && sizeof(Task) <= 64, "shared memory");
};

template <int TN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1) newton_schulz_kernel(const __grid_constant__ Steps<TN> w) {
  using L = Layout<TN>;
  constexpr int STAGES = L::STAGES, TASKS = L::TASKS;
  constexpr bool WIDE = TN == TILE;
  extern __shared__ uint8_t raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = smem_u32(sm);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = gemm::cta_rank();
  auto bar_full = [&](int s) { return base + L::OFF_BAR + 8 * s; };
  auto bar_empty = [&](int s) { return base + L::OFF_BAR + 8 * (STAGES + s); };
  auto bar_done = [&](int s) { return base + L::OFF_BAR + 8 * (2 * STAGES + s); };
  auto bar_free = [&](int s) { return base + L::OFF_BAR + 8 * (2 * STAGES + 2 + s); };
  auto bar_task = [&](int s) { return base + L::OFF_BAR + 8 * (2 * STAGES + 4 + s); };
  auto bar_slot = [&](int s) { return base + L::OFF_BAR + 8 * (2 * STAGES + 4 + TASKS + s); };
  auto bar_mail = [&](int s) { return base + L::OFF_BAR + 8 * (2 * STAGES + 4 + 2 * TASKS + s); };         // in the odd CTA: a number has come
  auto bar_read = [&](int s) { return base + L::OFF_BAR + 8 * (2 * STAGES + 4 + 3 * TASKS + s); };         // in the even one: it has been read there
  auto slot_of = [&](int n) -> volatile Task& { return *reinterpret_cast<volatile Task*>(sm + L::OFF_TASK + (n % TASKS) * 64); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + L::OFF_BAR + 8 * L::BARRIERS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + L::OFF_BAR + 8 * L::BARRIERS + 8);
  const long long WL = w.wait_limit;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(bar_full(s), 2); mbar_init(bar_empty(s), 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(bar_done(s), 1); mbar_init(bar_free(s), 2 * EPI_WARPS); }
    // read by the warps for loads, products (in the even CTA) and the epilogue
    for (int s = 0; s < TASKS; ++s) { mbar_init(bar_task(s), 1); mbar_init(bar_slot(s), EPI_WARPS + (rank == 0 ? 3 : 2)); mbar_init(bar_mail(s), 1); mbar_init(bar_read(s), 1); }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 2) gemm::tmem_alloc_pair(smem_u32(tmem_slot), 2 * TN);
  tc_fence_before();
  __syncthreads();
  gemm::cluster_sync_all();          // the other CTA's barriers are there, and it has started
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // The n-th tile of this pair, when it may be worked on, by one thread, or by a warp with every = true; false after the last one
  auto take = [&](int n, bool every, Task& k) -> bool {
    bool ok = mbar_wait(bar_task(n % TASKS), (n / TASKS) & 1, abort_flag, w.err, 329, WL);
    if (every) ok = __all_sync(0xffffffffu, ok);
    if (!ok) return false;
    volatile Task& s = slot_of(n);
    k.shape = s.shape;
    if (k.shape < 0) return false;
    k.batch = s.batch; k.matrix = s.matrix; k.m = s.m; k.n = s.n; k.phase = s.phase; k.step = s.step;
    if (every) __syncwarp();
    if (!every || lane == 0) mbar_arrive(bar_slot(n % TASKS));
    return true;
  };
  // Whether block kc of k lies above the diagonal for an operand's rows
  auto above = [](int kc, int row) { return kc / TILE > row / TILE; };

  if (warp == 3 && lane == 0) {
    // ---------------- what comes next
    int g = 0, next = rank == 0 ? draw(w) : 0;
    for (int n = 0;; ++n) {
      const int slot = n % TASKS, parity = (n / TASKS) & 1;
      int t = next;
      if (rank == 0) {                                 // draws for both, one ahead
        if (t < w.tiles) next = draw(w);
        if (!mbar_wait(bar_read(slot), parity ^ 1, abort_flag, w.err, 330, WL)) break;
        send(base + L::OFF_MAIL + 8 * slot, t, bar_mail(slot));
      } else {
        mbar_arrive_expect_tx(bar_mail(slot), 4);
        if (!mbar_wait(bar_mail(slot), parity, abort_flag, w.err, 331, WL)) break;
        t = *reinterpret_cast<volatile int*>(sm + L::OFF_MAIL + 8 * slot);
        gemm::arrive_at_leader(bar_read(slot));
      }
      if (!mbar_wait(bar_slot(slot), parity ^ 1, abort_flag, w.err, 320, WL)) break;
      volatile Task& s = slot_of(n);
      if (t >= w.tiles) {
        s.shape = -1;
        mbar_arrive(bar_task(slot));
        break;
      }
      const Task k = task_at(w, t, g);
      if (!wait_count(w.done + k.matrix, k.need, abort_flag, w.err, 321, WL)) break;
      s.shape = k.shape; s.batch = k.batch; s.matrix = k.matrix; s.m = k.m; s.n = k.n; s.phase = k.phase; s.step = k.step;
      mbar_arrive(bar_task(slot));
    }
  } else if ((warp == 0 || warp == 2) && lane == 0) {
    // ---------------- loads: of operand a by warp 0, of b by warp 2 (one thread's instructions for both took longer than the narrow form's products)
    int it = 0;
    Task k;
    for (int n = 0; take(n, false, k); ++n) {
      fence_proxy_async_all();
      const Info& info = w.info[k.shape];
      const int cur = k.step & 1, next = cur ^ 1, steps = (k.phase == 0 ? info.q : info.p) / KSTEP;
      const CUtensorMap* maps = w.map[k.shape];
      const CUtensorMap *straight, *turned;
      int row, skip;                                   // of the operand; turned from block `skip` of k on
      if (warp == 0) {
        straight = maps + (k.phase == 0 ? X_A + cur : k.phase == 1 ? A_A + next : B_A);
        turned = maps + (k.phase == 1 ? A_T + next : B_T);
        row = k.m * TILE + static_cast<int>(rank) * 128;
        skip = k.phase == 0 ? steps : (row / TILE + 1) * (TILE / KSTEP);
      } else {
        straight = maps + (k.phase == 0 ? (WIDE ? X_A : X_B) + cur : (WIDE ? A_A : A_B) + next);
        turned = maps + (k.phase == 1 ? (WIDE ? A_T : A_TB) + next : X_N + cur);
        row = k.n * TN + static_cast<int>(rank) * (TN / 2);
        skip = k.phase == 0 ? steps : k.phase == 1 ? (row / TILE + 1) * (TILE / KSTEP) : 0;
      }
      const bool two = warp == 0 || WIDE;              // blocks of 64 rows of a turned operand
      for (int i = 0; i < steps; ++i, ++it) {
        const int s = it % STAGES, kc = i * KSTEP;
        if (!mbar_wait(bar_empty(s), ((it / STAGES) & 1) ^ 1, abort_flag, w.err, 322, WL)) break;
        if (rank == 0) mbar_arrive_expect_tx(bar_full(s), 2 * (warp == 0 ? L::A_BYTES : L::B_BYTES));
        const uint32_t bar = gemm::leaders(bar_full(s)), to = base + s * L::STAGE_BYTES + (warp == 0 ? 0 : L::A_BYTES);
        if (i < skip) {
          gemm::tma_load_pair(to, straight, kc, row, k.batch, bar);
        } else {
          gemm::tma_load_pair(to, turned, row, kc, k.batch, bar);
          if (two) gemm::tma_load_pair(to + 64 * KSTEP * 2, turned, row + 64, kc, k.batch, bar);
        }
      }
      if (*abort_flag) break;
    }
    for (int i = it > STAGES ? it - STAGES : 0; i < it; ++i) mbar_wait(bar_empty(i % STAGES), (i / STAGES) & 1, abort_flag, w.err, 323, WL);
  } else if (warp == 1 && rank == 0) {
    // ---------------- products
    constexpr uint32_t IDESC = (1u << 4) | (static_cast<uint32_t>(TN >> 3) << 17) | (static_cast<uint32_t>(TILE >> 4) << 24);
    const uint64_t da = make_sdesc(base, 16, 1024), dat = make_sdesc(base, L::A_BYTES / 2, 1024);
    const uint64_t db = make_sdesc(base + L::A_BYTES, 16, 1024), dbt = WIDE ? make_sdesc(base + L::A_BYTES, L::B_BYTES / 2, 1024) : make_sdesc64(base + L::A_BYTES, 16, 512);
    constexpr uint32_t KBT = WIDE ? 2048 >> 4 : 1024 >> 4;
    int it = 0;
    Task k;
    for (int n = 0; take(n, true, k); ++n) {
      const Info& info = w.info[k.shape];
      const int buf = n & 1, steps = (k.phase == 0 ? info.q : info.p) / KSTEP, am = k.m * TILE, bn = k.n * TN;
      if (!mbar_wait(bar_free(buf), ((n >> 1) & 1) ^ 1, abort_flag, w.err, 324, WL)) break;
      tc_fence_after();
      bool ok = true;
      for (int i = 0; i < steps; ++i, ++it) {
        const int s = it % STAGES;
        ok = mbar_wait(bar_full(s), (it / STAGES) & 1, abort_flag, w.err, 325, WL);
        if (!ok) break;
        tc_fence_after();
        const bool at = k.phase > 0 && above(i * KSTEP, am), bt = k.phase == 2 || (k.phase == 1 && above(i * KSTEP, bn));
        const uint64_t off = static_cast<uint64_t>((s * L::STAGE_BYTES) >> 4), a = (at ? dat : da) + off, b = (bt ? dbt : db) + off;
        const uint32_t ka = at ? 2048 >> 4 : 32 >> 4, kb = bt ? KBT : 32 >> 4, idesc = IDESC | (static_cast<uint32_t>(at) << 15) | (static_cast<uint32_t>(bt) << 16);
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < KSTEP / 16; ++j) gemm::umma_pair(tmem + buf * TN, a + j * ka, b + j * kb, idesc, (i | j) != 0);
          gemm::commit_pair(bar_empty(s));
        }
        __syncwarp();
      }
      if (!ok) break;
      if (elect_one()) gemm::commit_pair(bar_done(buf));
      __syncwarp();
    }
  } else if (warp >= 4) {
    // ---------------- epilogue
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t boxes = base + L::OFF_EPI + static_cast<uint32_t>(warp - 4) * L::BOXES * BOX_BYTES;
    unsigned long long* pending = nullptr;             // counter of the tile before, whose stores may be on their way
    int stores = 0;
    auto tell = [&] {
      if (pending != nullptr && lane == 0) {
        bulk_wait<0>();
        add_count(pending);
      }
      pending = nullptr;
    };
    // 32 x 32 of the result on their way, from the box of the store before the last; one group each
    auto put = [&](const CUtensorMap* map, const uint32_t (&v)[16], int col, int row0, int batch, bool inside) {
      if (lane == 0) bulk_wait_read<L::BOXES - 1>();
      __syncwarp();
      const uint32_t box = boxes + (stores++ % L::BOXES) * BOX_BYTES;
      fill_box(box, lane, v);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        if (inside) tma_store_3d(map, box, col, row0, batch);
        bulk_commit();
      }
    };
    Task k;
    for (int n = 0;; ++n) {
      // nobody may wait for this warp's last tile while it waits itself
      if (!mbar_test(bar_task(n % TASKS), (n / TASKS) & 1)) tell();
      if (!take(n, true, k)) break;
      const Info& info = w.info[k.shape];
      const CUtensorMap* maps = w.map[k.shape];
      const int buf = n & 1, cur = k.step & 1, row0 = k.m * TILE + static_cast<int>(rank) * 128 + quarter * 32, col0 = k.n * TN + half * (TN / 2);
      const int N = k.phase == 2 ? info.q : info.p;
      const bool low = k.phase == 2 && has_lower(k.step, w.steps), more = k.phase == 2 && has_lower(k.step + 1, w.steps), there = row0 < info.p;
      const CUtensorMap* to = maps + (k.phase == 0 ? A_BOX + (cur ^ 1) : k.phase == 1 ? B_BOX : X_BOX + (cur ^ 1));
      // the tile's input, all of it, while it is summed
      uint32_t in[L::CHUNKS][16];
      if (k.phase == 1 || low) {
        const uint16_t* from = (k.phase == 1 ? info.x[cur ^ 1] : info.low) + static_cast<int64_t>(k.batch) * info.p * info.q + static_cast<int64_t>(row0 + lane) * N + col0;
#pragma unroll
        for (int j = 0; j < L::CHUNKS; ++j)
          if (there && col0 + 32 * j < N) load_row(from + 32 * j, in[j]);
      }
      if (!mbar_test(bar_done(buf), (n >> 1) & 1)) tell();
      bool ok = mbar_wait(bar_done(buf), (n >> 1) & 1, abort_flag, w.err, 327, WL);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int j = 0; j < L::CHUNKS; ++j) {
        const int col = col0 + 32 * j;
        uint32_t v[32], hi[16];
        uint32_t(&e)[16] = in[j];
        __syncwarp();                                  // TMEM is read by whole warps
        tmem_ld32(tmem + buf * TN + (static_cast<uint32_t>(quarter * 32) << 16) + half * (TN / 2) + 32 * j, v);
        tmem_ld_wait();
        if (k.phase == 0) {
          constexpr float SCALE = 1.f / (X_SCALE * X_SCALE);
#pragma unroll
          for (int i = 0; i < 16; ++i) hi[i] = gemm::pack_f16(__uint_as_float(v[2 * i]) * SCALE, __uint_as_float(v[2 * i + 1]) * SCALE);
        } else if (k.phase == 1) {
          const int own = row0 + lane - col;           // where the diagonal is in this row
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 a = gemm::unpack_f16(e[i]);
            float x = fmaf(w.c, __uint_as_float(v[2 * i]), w.b * a.x), y = fmaf(w.c, __uint_as_float(v[2 * i + 1]), w.b * a.y);
            if (2 * i == own) x += w.a;
            if (2 * i + 1 == own) y += w.a;
            hi[i] = gemm::pack_f16(x, y);
          }
        } else {
          const float scale = w.a * (1.f / LO_SCALE);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float x = __uint_as_float(v[2 * i]), y = __uint_as_float(v[2 * i + 1]);
            if (low) {
              const float2 l = gemm::unpack_f16(e[i]);
              x = fmaf(scale, l.x, x);
              y = fmaf(scale, l.y, y);
            }
            hi[i] = gemm::pack_f16(x, y);
            if (more) {
              const float2 r = gemm::unpack_f16(hi[i]);
              e[i] = gemm::pack_f16((x - r.x) * LO_SCALE, (y - r.y) * LO_SCALE);
            }
          }
        }
        const bool inside = there && col < N;
        put(to, hi, col, row0, k.batch, inside);
        if (more) put(maps + LO_BOX, e, col, row0, k.batch, inside);       // in the place of what it was made of
        if (j == 0 && pending != nullptr) {
          if (lane == 0) {                             // the tile before: all groups but this chunk's
            if (more) bulk_wait<2>();
            else bulk_wait<1>();
            add_count(pending);
          }
          pending = nullptr;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) gemm::arrive_at_leader(bar_free(buf));
      pending = w.done + k.matrix;
    }
    tell();
    if (lane == 0) bulk_wait<0>();
    __syncwarp();
  }

  // ---------------- teardown, as in gemm_sm100.cuh
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < (1ll << 24)) __nanosleep(1000);
  }
  gemm::cluster_sync_all();
  tc_fence_after();
  if (warp == 2) gemm::tmem_dealloc_pair(tmem, 2 * TN);
}

// ---------------------------------------------------------------- host side
// A batch of matrices of one shape: X [batch][p][q] in two buffers and its lower part, B [batch][p][p]
struct Batch {
  int64_t p, q, count;
  uint16_t *hi[2], *lo, *B;
};
// What a group's matrices have in their two buffers of X and in B.  Fewer fit L2 (126 MB), but too few tiles for a product let pairs wait for each other: Muon step over 101 M elements, groups of
// 80, 160, 250, 400 MB: 3057, 3033, 2927, 2952 us; steps over 50 M 1279, 1198, 1214, 1185.  Two halves of a group whose products alternate, so that others stand between a product and the one
// that needs it, gave nothing there and cost 130 us of 450 with 7 matrices.
constexpr int64_t GROUP_BYTES = int64_t(250) << 20;

inline int64_t bytes_of(const Batch& b) { return 2 * (2 * b.p * b.q + b.p * b.p); }      // of a matrix

// Tiles of a product of one matrix: of A or B, on and below the diagonal, and of X
struct Tiles {
  int symmetric, full;
};
inline Tiles tiles_of(const Batch& b, int columns) {
  const int m = static_cast<int>((b.p + TILE - 1) / TILE), n = static_cast<int>((b.p + columns - 1) / columns);
  Tiles t = {0, static_cast<int>(m * ((b.q + columns - 1) / columns))};
  for (int i = 0; i < m; ++i) t.symmetric += std::min((i + 1) * (TILE / columns), n);
  return t;
}
inline int columns_of(bool narrow) { return narrow ? 64 : TILE; }
// What a matrix's counter shows when all of its steps are complete; less where a wait has run out
inline unsigned long long count_of(const Batch& b, bool narrow, int steps) {
  const Tiles t = tiles_of(b, columns_of(narrow));
  return static_cast<unsigned long long>(steps) * (2ull * t.symmetric + t.full) * (2 * EPI_WARPS);
}

template <int TN>
int set_shape(Steps<TN>& w, int i, const Batch& b) {
  using gemm::make_map;
  Info& f = w.info[i];
  f.p = static_cast<int>(b.p); f.q = static_cast<int>(b.q);
  f.tiles_m = (f.p + TILE - 1) / TILE; f.tiles_n = (f.p + TN - 1) / TN; f.tiles_q = (f.q + TN - 1) / TN;
  const Tiles t = tiles_of(b, TN);
  f.symmetric = t.symmetric;
  f.full = t.full;
  f.x[0] = b.hi[0]; f.x[1] = b.hi[1]; f.low = b.lo; f.b = b.B;
  CUtensorMap* m = w.map[i];
  int rc = 0;
  auto map = [&](int at, const void* base, int64_t inner, int64_t each, int box_inner, int box_outer) {
    if (rc == 0) rc = make_map(&m[at], base, true, inner, b.p, b.count, inner, each, box_inner, box_outer);
  };
  for (int k = 0; k < 2; ++k) {
    map(X_A + k, b.hi[k], b.q, b.p * b.q, 64, 128);
    map(X_N + k, b.hi[k], b.q, b.p * b.q, TN == TILE ? 64 : 32, 64);
    map(X_BOX + k, b.hi[k], b.q, b.p * b.q, 32, 32);
    map(A_BOX + k, b.hi[k], b.p, b.p * b.q, 32, 32);
    map(A_A + k, b.hi[k], b.p, b.p * b.q, 64, 128);
    map(A_T + k, b.hi[k], b.p, b.p * b.q, 64, 64);
    if (TN != TILE) {
      map(X_B + k, b.hi[k], b.q, b.p * b.q, 64, TN / 2);
      map(A_B + k, b.hi[k], b.p, b.p * b.q, 64, TN / 2);
      map(A_TB + k, b.hi[k], b.p, b.p * b.q, 32, 64);
    }
  }
  map(B_A, b.B, b.p, b.p * b.p, 64, 128);
  map(B_T, b.B, b.p, b.p * b.p, 64, 64);
  map(B_BOX, b.B, b.p, b.p * b.p, 32, 32);
  map(LO_BOX, b.lo, b.q, b.p * b.q, 32, 32);
  return rc;
}

// The steps for batches from `from` on (and in that one from matrix `start` on), as many as a launch's parameters hold; both move on, and done and base with them.
template <int TN>
int launch(const std::vector<Batch>& batches, size_t& from, int64_t& start, unsigned long long*& done, unsigned long long* drawn, unsigned long long& base, int steps, double a, double b, double c,
           cudaStream_t st) {
  using S = Steps<TN>;
  static thread_local S w;
  // groups of about one size
  int64_t total = 0;
  for (size_t i = from; i < batches.size(); ++i) total += bytes_of(batches[i]) * (batches[i].count - (i == from ? start : 0));
  const int64_t want = std::max<int64_t>(1, (total + GROUP_BYTES - 1) / GROUP_BYTES), limit = (total + want - 1) / want;
  int shapes = 0, segments = 0, groups = 0, matrices = 0;
  int64_t tiles = 0, used = 0;
  bool full = false;
  while (!full && from < batches.size() && shapes < S::SHAPES) {
    const Batch& x = batches[from];
    if (int rc = set_shape(w, shapes, x)) return rc;
    const Info& f = w.info[shapes];
    while (start < x.count) {
      if (groups == 0 || used + bytes_of(x) / 2 > limit) {                     // the group has what it should: the next one
        if (groups == S::GROUPS || segments == S::SEGMENTS) { full = true; break; }
        w.group[groups++] = {static_cast<int>(tiles), segments, segments, 0, 0};
        used = 0;
      }
      if (segments == S::SEGMENTS) { full = true; break; }
      Group& gr = w.group[groups - 1];
      const int64_t room = std::max<int64_t>(1, (limit - used + bytes_of(x) / 2) / bytes_of(x)), k = std::min(x.count - start, room);
      const int64_t more = static_cast<int64_t>(steps) * k * (2 * f.symmetric + f.full);
      if (tiles + more > 0x3FFFFFFF) {
        if (segments == 0) return fail(HASTE_ERR_TOO_LARGE, "matrices of too many tiles for one launch");
        full = true;
        break;
      }
      tiles += more;
      w.segment[segments++] = {shapes, static_cast<int>(start), static_cast<int>(k), matrices, gr.symmetric, gr.full};
      gr.end = segments;
      gr.symmetric += static_cast<int>(k * f.symmetric);
      gr.full += static_cast<int>(k * f.full);
      used += k * bytes_of(x);
      matrices += static_cast<int>(k);
      start += k;
    }
    ++shapes;
    if (full) break;
    ++from;
    start = 0;
  }
  if (groups > 0 && w.group[groups - 1].end == w.group[groups - 1].segment) --groups;          // an empty last one
  w.groups = groups;
  w.tiles = static_cast<int>(tiles);
  w.steps = steps;
  w.a = static_cast<float>(a); w.b = static_cast<float>(b); w.c = static_cast<float>(c);
  w.done = done;
  w.drawn = drawn;
  w.base = base;
  done += matrices;
  if (tiles == 0) return HASTE_OK;
  if (int rc = device_status_word(&w.err)) return rc;
  w.wait_limit = wait_limit_cycles();
  constexpr auto kernel = &newton_schulz_kernel<TN>;
  int pairs = 0;
  if (int rc = gemm::pairs_resident<kernel>(Layout<TN>::SMEM_BYTES, &pairs)) return rc;
  if (const int n = product_pairs()) pairs = n;
  pairs = static_cast<int>(imin64(pairs, tiles));
  base += static_cast<unsigned long long>(tiles) + pairs;          // every pair draws one number behind the last tile's
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = Layout<TN>::SMEM_BYTES;
  cfg.stream = st;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, w);
  if (e != cudaSuccess) return fail(HASTE_ERR_LAUNCH, "cudaLaunchKernelEx: %s", cudaGetErrorString(e));
  return HASTE_OK;
}

// The wide form, or the narrow one where wide tiles would leave pairs without work: a product's time in either, over the matrices that are worked on together
inline bool take_narrow(const std::vector<Batch>& batches) {
  int64_t total = 0, tiles[2] = {}, work = 0;
  for (const Batch& b : batches) {
    total += bytes_of(b) * b.count;
    for (int n = 0; n < 2; ++n) tiles[n] += b.count * gemm::tiles_for(b.p, b.q, n ? 64 : TILE);
    work += b.count * gemm::tiles_for(b.p, b.q, TILE) * gemm::steps_of(b.p);
  }
  const int64_t groups = std::max<int64_t>(1, (total + GROUP_BYTES - 1) / GROUP_BYTES), per = (work + tiles[0] - 1) / tiles[0], pairs = sm_count() / 2;
  return gemm::cost_of(tiles[1] / groups, per, true, pairs) < gemm::cost_of(tiles[0] / groups, per, false, pairs);
}

// narrow: what take_narrow() says; done: a counter for every matrix; drawn: one more.  All zeros.
inline int run(const std::vector<Batch>& batches, bool narrow, unsigned long long* done, unsigned long long* drawn, int steps, double a, double b, double c, cudaStream_t st) {
  size_t from = 0;
  int64_t start = 0;
  unsigned long long base = 0;
  while (from < batches.size()) {
    if (int rc = narrow ? launch<64>(batches, from, start, done, drawn, base, steps, a, b, c, st) : launch<TILE>(batches, from, start, done, drawn, base, steps, a, b, c, st)) return rc;
  }
  return HASTE_OK;
}

}  // namespace newton_schulz
}  // namespace haste
