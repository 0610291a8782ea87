// Products with one matrix for each group of rows (16-bit storage, fp32 sums), on tcgen05.mma kind::f16.
//
//   nt   Y[t, n] = sum_k X[t, k] W[e, n, k]        t in group e
//   nn   Z[t, k] = sum_n Y[t, n] W[e, n, k]
//   tn   D[e, n, k] = sum_{t in group e} Y[t, n] X[t, k]
//
// All three are D[m, j] = sum_r P[m, r] Q[j, r] (tiles_sm100.cuh), stored at out[j, m]:
//   nt   P = W[e] as it lies (rows along the reduction), Q = X
//   nn   P = W[e]^T, read as it lies: its rows run along m ("mn-major" operand tiles), Q = Y
//   tn   P = X^T, Q = Y^T, both mn-major; the reduction runs over the rows of the group
//
// A persistent CTA, or a pair of them, walks tiles of 128 (256) m x up to 256 j:
//   warp 0     loads operand stages of 64 reduction steps by TMA (128-byte swizzle)
//   warp 1     allocates the tensor memory and issues the products
//   warps 2-9  take the accumulator out of tensor memory and store it; two accumulators alternate, so that this runs under the next tile's
//              products
//   warp 10    of tn: clears what a group's last stage holds of the next group
// Where tiles are few a cluster of CTAs shares a tile's reduction and adds it up through each other's shared memory.
//
// Measured on one B200: nt, 32 groups of together 32768 rows, 4096 x 2048: 463 to 502 us by the chip = 1095 to 1190 TFLOP/s in a stream of calls, at the power cap (cuBLAS, 32 equal
// groups: 439 to 450 us, these here 441 to 452), 385 us = 1430 TFLOP/s for a call after a pause; a trace has 16,280 to 17,000 cycles from tile to tile, nominally 16,384 for its
// products.  nn and tn of 16 groups, 16384 rows, 2048 x 1024: 64 to 69 and 70 to 77 us.  Small calls are bound by latency, 3.4 us for the smallest, or by the weights: 16 rows of 32 groups, 1536 x 1024, read 38 MB in
// 10.9 us where they fall to 12 of these, in 9.2 out of the L2.
#include "tiles_sm100.cuh"

namespace {

using namespace pcl_group;
using namespace pcl_tiles;

__device__ PclStatus g_status;

__global__ void take_kernel(PclStatus* to) { take(&g_status, to); }

constexpr int NT = 0, NN = 1, TN = 2;
constexpr int BR = 64;                         // reduction steps of a stage
constexpr int LANES = 128;
constexpr int P_BYTES = LANES * BR * 2;
constexpr int OPERAND_BYTES = 192 * 1024;
constexpr int MAX_STAGES = 8;
constexpr int EPI_WARPS = 8;
constexpr int FIX_WARP = 2 + EPI_WARPS;
// tn has a warp more: it clears what a group's last stage holds of the next group
constexpr int threads_of(int mode) { return 64 + 32 * EPI_WARPS + (mode == 2 ? 32 : 0); }
// CG: CTAs that work on a tile, one or a pair on neighbouring SMs (tcgen05 cta_group::2); each of a pair holds its 128 m and half the j
// COLS: columns of an accumulator, the most j of a tile
// SPLIT: a cluster shares a tile's reduction (single CTAs of 64 or 128 columns)
template <int CG, int COLS, bool SPLIT>
struct Form {
  static constexpr int Q_BYTES = COLS / CG * BR * 2;
  static constexpr int STAGE_BYTES = P_BYTES + Q_BYTES;
  // A cluster's 128 columns: the parts are sent to where the operands were, behind a barrier of the cluster more; three stages beside them left the loads waiting
  // (one group of 131072 rows, 512 x 512: 135 and 113 us; 114 to 118 with its sums in parts)
  static constexpr bool AFTER = SPLIT && COLS == 128;
  static constexpr int STAGES = (OPERAND_BYTES - (SPLIT && !AFTER ? inbox_bytes(COLS) : 0)) / STAGE_BYTES;
  static_assert(!AFTER || inbox_bytes(COLS) <= OPERAND_BYTES, "room for the parts");
  static constexpr int M = LANES * CG;   // m of a tile
  // Rows of Q that a load brings: all that fit, or a quarter of them, up to three times.  A load takes the warp that issues it 135 cycles, and the products of a
  // stage 512 at most: four or five loads to a stage were what bound a call.
  static constexpr int BOX = COLS / CG, SMALL_BOX = BOX / 4;
  static_assert(STAGES <= MAX_STAGES, "barriers");
  static_assert(COLS % (16 * CG) == 0, "a chunk rounded up to the product's columns fits an accumulator, and none is left empty");
};

struct Args {
  void* out;
  long long ldo;
  Offsets off;
  int mdim;            // extent of m: N (nt), K (nn, tn)
  int jdim;            // tn: extent of j, N
  int red;             // nt, nn: extent of the reduction
  uint32_t type;       // operands: 0 fp16, 1 bf16
  int fill;            // nt, nn: rows of no group become zero
  bool boxed;          // results leave through mapOut
  bool wide;           // tn: the maps have columns in blocks of 64 as their third dimension, so that one load brings all blocks of an operand
};

struct Shared {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES], tail[MAX_STAGES], tfull[2], tempty[2];
  uint32_t tmem;
  int abort_flag;
  Table table;
};

constexpr int SMEM_BYTES = 1024 + OPERAND_BYTES + EPI_WARPS * PIECE_BYTES + (int)sizeof(Shared);

struct Tile {
  int e, m0, j0, n, ncol, r0, r1;   // columns: n of them, ncol with those that the product rounds up to
};

// The tiles of a call, numbered: those that share rows of Q are neighbours.
template <int MODE, int CG, int COLS, bool SPLIT>
struct Walk {
  const Args& a;
  const Table& t;
  int mb, jparts, jsize, chunks;

  __device__ Walk(const Args& a_, const Table& t_) : a(a_), t(t_) {
    mb = (a.mdim + Form<CG, COLS, SPLIT>::M - 1) / Form<CG, COLS, SPLIT>::M;
    jparts = jsize = 0;
    if (MODE == TN) {
      jparts = (a.jdim + COLS - 1) / COLS;
      const int step = (a.wide ? 64 : 16) * CG;
      jsize = ((a.jdim + jparts - 1) / jparts + step - 1) / step * step;
      chunks = a.off.groups * jparts;
    } else {
      chunks = t.chunks[a.off.groups];
    }
  }

  __device__ Counter start(int first, int step) const { return Counter(first, step, mb); }
  __device__ bool has(const Counter& i) const { return i.c < chunks; }

  __device__ Tile at(const Counter& i) const {
    Tile w;
    w.m0 = i.m * Form<CG, COLS, SPLIT>::M;
    if (MODE == TN) {
      w.e = i.c / jparts;
      w.j0 = (i.c - w.e * jparts) * jsize;
      w.n = min(jsize, a.jdim - w.j0);
      w.r0 = t.bounds[w.e];
      w.r1 = t.bounds[w.e + 1];
    } else {
      t.find(a.off.groups, i.c, 16 * CG, w.e, w.j0, w.n);
      w.r0 = 0;
      w.r1 = a.red;
    }
    if (SPLIT) {   // this CTA's stages (none, where a group has fewer than the cluster has CTAs)
      const long long steps = ((long long)w.r1 - w.r0 + BR - 1) / BR;
      const int rank = (int)cluster_ctarank(), parts = (int)cluster_size(), first = w.r0;
      w.r0 = first + (int)(rank * steps / parts) * BR;
      w.r1 = (int)min((long long)w.r1, first + (rank + 1) * steps / parts * BR);
    }
    // (with the wide maps either CTA of a pair begins with a block of 64)
    const int unit = (MODE == TN && a.wide ? 64 : 16) * CG;
    w.ncol = (w.n + unit - 1) / unit * unit;
    return w;
  }
};

template <int MODE, int CG, int COLS, bool SPLIT, class TO>
__global__ void __launch_bounds__(threads_of(MODE), 1)
product_kernel(const __grid_constant__ CUtensorMap mapP, const __grid_constant__ CUtensorMap mapQ,
               const __grid_constant__ CUtensorMap mapQ_small, const __grid_constant__ CUtensorMap mapOut, Args a) {
  using F = Form<CG, COLS, SPLIT>;
  constexpr int Q_BYTES = F::Q_BYTES, STAGE_BYTES = F::STAGE_BYTES, STAGES = F::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* pieces = stages + OPERAND_BYTES;
  Shared& s = *reinterpret_cast<Shared*>(pieces + EPI_WARPS * PIECE_BYTES);
  float* inbox = reinterpret_cast<float*>(stages + (F::AFTER ? 0 : STAGES * STAGE_BYTES));   // SPLIT
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t me = CG == 2 ? cluster_ctarank() : 0;   // 0 leads the pair
  volatile int* abort_flag = &s.abort_flag;

  if (warp == 0) {
    if (lane < STAGES) {
      mbar_init(s.full + lane, MODE == TN ? CG : 1);
      mbar_init(s.empty + lane, 1);
      mbar_init(s.tail + lane, 1);
    }
    if (lane < 2) { mbar_init(s.tfull + lane, 1); mbar_init(s.tempty + lane, CG * EPI_WARPS); }
    if (lane == 0) s.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2 && lane == 0) {
    for (const CUtensorMap* m : {&mapP, &mapQ, &mapQ_small, &mapOut}) asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
  }
  let_next_begin();
  after_previous();
  load_bounds(a.off, s.table.bounds, &g_status);
  __syncthreads();
  if (warp == 0) s.table.build(a.off.groups, COLS, &g_status);
  if (warp == 1) tmem_alloc<CG>(&s.tmem, 2 * COLS);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  sync_cluster_or_block<CG == 2 || SPLIT>();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = s.tmem;
  const int share = SPLIT ? (int)cluster_size() : CG;
  const int group = blockIdx.x / share, groups = gridDim.x / share;
  const Walk<MODE, CG, COLS, SPLIT> walk(a, s.table);
  using Turn = Tiles<Walk<MODE, CG, COLS, SPLIT>, SPLIT>;
  bool ok = true;

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    for (Turn i(walk, group, groups); i.has() && ok; i.next()) {
      const Tile w = i.tile();
      const int steps = (w.r1 - w.r0 + BR - 1) / BR;
      const int mine = w.ncol / CG;
      const int j = w.j0 + (int)me * mine;
      const bool whole = MODE == TN ? a.wide : mine > 3 * F::SMALL_BOX;
      const int boxes = whole ? 1 : MODE == TN ? (mine + 63) / 64 : (mine + F::SMALL_BOX - 1) / F::SMALL_BOX;
      const uint32_t q_bytes = whole ? (uint32_t)Q_BYTES : MODE == TN ? boxes * 8192u : boxes * (uint32_t)(F::SMALL_BOX * BR * 2);
      for (int kb = 0; kb < steps; ++kb) {
        if (!mbar_wait(s.empty + stage, phase ^ 1, abort_flag)) {
          if (lane == 0) post(&g_status, CODE_WAIT, 41, kb, stage);
          abort_all<CG>(abort_flag, me ^ 1u);
          ok = false;
          break;
        }
        uint8_t* st = stages + stage * STAGE_BYTES;
        const uint32_t sp = smem_u32(st), sq = smem_u32(st + P_BYTES);
        const int r = w.r0 + kb * BR;
        // the group's last rows share their stage with the next group's: they are loaded under a barrier of this CTA's own, and the
        // warp that waits for it clears what follows them, in both operands (zero times infinity is not zero)
        const bool tail = MODE == TN && r + BR > w.r1;
        if (elect()) {
          uint32_t bar = smem_u32((tail ? s.tail : s.full) + stage);
          const uint32_t bytes = P_BYTES + q_bytes;
          if (tail) {
            mbar_expect_tx(s.tail + stage, bytes);
          } else {
            if (me == 0) mbar_expect_tx(s.full + stage, CG * bytes);
            if (CG == 2) bar = map_to_cta(bar, 0);
            if (MODE == TN && me != 0) mbar_arrive_cluster(bar);
          }
          const int m = w.m0 + (int)me * LANES;
          if (MODE == NT) {
            tma_load_3d<CG>(sp, &mapP, bar, r, m, w.e);
          } else if (MODE == TN && a.wide) {
            if (tail) {
              tma_load_3d<1>(sp, &mapP, bar, 0, r, m / 64);
              tma_load_3d<1>(sq, &mapQ, bar, 0, r, j / 64);
            } else {
              tma_load_3d<CG>(sp, &mapP, bar, 0, r, m / 64);
              tma_load_3d<CG>(sq, &mapQ, bar, 0, r, j / 64);
            }
          } else {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              if (tail) tma_load_3d<1>(sp + b * 8192, &mapP, bar, m + 64 * b, r, 0);
              else tma_load_3d<CG>(sp + b * 8192, &mapP, bar, m + 64 * b, r, MODE == TN ? 0 : w.e);
            }
          }
          if (MODE == TN) {
            for (int b = 0; b < (a.wide ? 0 : boxes); ++b) {
              if (tail) tma_load_3d<1>(sq + b * 8192, &mapQ, bar, j + 64 * b, r, 0);
              else tma_load_3d<CG>(sq + b * 8192, &mapQ, bar, j + 64 * b, r, 0);
            }
          } else if (whole) {
            tma_load_3d<CG>(sq, &mapQ, bar, r, j, 0);
          } else {
            for (int b = 0; b < boxes; ++b)
              tma_load_3d<CG>(sq + b * F::SMALL_BOX * BR * 2, &mapQ_small, bar, r, j + b * F::SMALL_BOX, 0);
          }
        }
        __syncwarp();
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
    }
    if (!ok)
      for (int i = 0; i < 2048; ++i) __nanosleep(1000);   // copies in flight land before the shared memory goes away
  } else if (warp == 1) {
    if (me == 0) {
      const uint32_t idesc0 = (1u << 4) | (a.type << 7) | (a.type << 10) | ((MODE != NT ? 1u : 0u) << 15) |
                              ((MODE == TN ? 1u : 0u) << 16) | ((uint32_t)(LANES * CG >> 4) << 24);
      // from one 16-step product to the next: 32 bytes along a row, or 16 rows of 128 bytes
      constexpr uint64_t STEP_P = MODE == NT ? 2 : 128, STEP_Q = MODE == TN ? 128 : 2;
      const uint64_t dp0 = MODE == NT ? desc_k_major(smem_u32(stages)) : desc_mn_major(smem_u32(stages));
      const uint64_t dq0 = MODE == TN ? desc_mn_major(smem_u32(stages + P_BYTES)) : desc_k_major(smem_u32(stages + P_BYTES));
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;   // bit i of acc_phase: accumulator i
      bool ready = false;                  // the next stage has arrived
      for (Turn i(walk, group, groups); i.has() && ok; i.next()) {
        const Tile w = i.tile();
        const int len = w.r1 - w.r0, steps = (len + BR - 1) / BR;
        if (len <= 0) continue;
        const uint32_t idesc = idesc0 | ((uint32_t)(w.ncol >> 3) << 17);
        const uint32_t d = tmem + (uint32_t)(acc * COLS);
        // Parts of LONG stages: each waits until the one before it has been added up.  The sum is in the other accumulator, which counts as used from the second part on (the
        // warps that store take it up in turn behind the tile that was there) until it is stored; the next tile does not wait for that, but takes this accumulator.
        for (int begin = 0; begin < steps && ok; begin += LONG) {
          for (int b = acc;; b = acc ^ 1) {
            if (!mbar_wait(s.tempty + b, (acc_phase >> b & 1u) ^ 1u, abort_flag)) {
              if (lane == 0) post(&g_status, CODE_WAIT, 42, b, 0);
              abort_all<CG>(abort_flag, me ^ 1u);
              ok = false;
              break;
            }
            acc_phase ^= 1u << b;
            if (b != acc || begin != LONG) break;
          }
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const int end = min(steps, begin + LONG);
          for (int r = begin; r < end; ++r) {
            if (!ready && !wait_full(s.full + stage, phase, abort_flag)) {
              if (lane == 0) post(&g_status, CODE_WAIT, 43, r, stage);
              abort_all<CG>(abort_flag, me ^ 1u);
              ok = false;
              break;
            }
            const int next = stage + 1 == STAGES ? 0 : stage + 1;
            ready = has_passed(s.full + next, phase ^ (uint32_t)(next == 0));
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect()) {
              const uint64_t dp = dp0 + (uint32_t)(stage * STAGE_BYTES) / 16, dq = dq0 + (uint32_t)(stage * STAGE_BYTES) / 16;
              if (r * BR + BR <= len) {
#pragma unroll
                for (int k = 0; k < BR / 16; ++k) umma_f16<CG>(d, dp + k * STEP_P, dq + k * STEP_Q, idesc, (r > begin || k > 0) ? 1u : 0u);
              } else {
                for (int k = 0; r * BR + 16 * k < len; ++k) umma_f16<CG>(d, dp + k * STEP_P, dq + k * STEP_Q, idesc, (r > begin || k > 0) ? 1u : 0u);
              }
              commit<CG>(smem_u32(s.empty + stage));
              if (r + 1 == end) commit<CG>(smem_u32(s.tfull + acc));
            }
            __syncwarp();
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
          }
        }
        if (steps <= LONG) acc ^= 1;
      }
    }
  } else if (MODE == TN && warp == FIX_WARP) {
    int stage = 0;
    uint32_t phases = 0;   // bit i: parity of the next wait on tail[i]
    long long since = 0;   // stages since the last wait: tiles without a tail are passed over at once, and the next tail comes behind all of theirs
    for (Turn i(walk, group, groups); i.has() && ok; i.next()) {
      const Tile w = i.tile();
      const int len = w.r1 - w.r0, steps = (len + BR - 1) / BR;
      const int last = (stage + steps + STAGES - 1) % STAGES;
      stage = (stage + steps) % STAGES;
      since += steps;
      if (len % BR == 0) continue;
      if (!wait_full(s.tail + last, (phases >> last) & 1u, abort_flag, tile_ns(since))) {
        if (lane == 0) post(&g_status, CODE_WAIT, 45, last, 0);
        abort_all<CG>(abort_flag, me ^ 1u);
        ok = false;
        break;
      }
      phases ^= 1u << last;
      since = 0;
      // the products stop at the next multiple of 16 steps
      uint8_t* st = stages + last * STAGE_BYTES;
      const int left = len % BR, upto = (left + 15) & ~15;
      const int boxes = 2 + (w.ncol / CG + 63) / 64, pieces = (upto - left) * 8;   // 16-byte pieces of a box
      for (int b = 0; b < boxes; ++b)                                                 // Q's boxes lie behind P's
        for (int q = lane; q < pieces; q += 32)
          *reinterpret_cast<uint4*>(st + b * 8192 + left * 128 + q * 16) = make_uint4(0, 0, 0, 0);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive_cluster(CG == 2 ? map_to_cta(smem_u32(s.full + last), 0) : smem_u32(s.full + last));
    }
  } else {
    const int sub = warp & 3;                 // the quarter of the tensor memory's lanes that this warp can read
    const int half = (warp - 2) >> 2;         // two warps share a quarter: 32 columns in turn
    TO* out = static_cast<TO*>(a.out);
    int acc = 0;
    uint32_t acc_phase = 0;                   // bit i: accumulator i
    bool free = false;                        // AFTER: no CTA of the cluster reads its operands any more
    for (Turn i(walk, group, groups); i.has() && ok; i.next()) {
      const Tile w = i.tile();
      const int m = w.m0 + (int)me * LANES + sub * 32;
      TO* dst = out + (MODE == TN ? ((long long)w.e * a.jdim + w.j0) * a.ldo : (long long)w.j0 * a.ldo) + m;
      if (SPLIT && w.r1 <= w.r0) {   // no rows for this part
        if (F::AFTER) cluster_sync_all();
        free = true;
        send_columns(0, sub, half * 32, w.n, inbox, cluster_ctarank(), columns_of_part(w.n, share), true);
        continue;
      }
      if (w.r1 <= w.r0) {   // a group without rows: its matrix of sums is zero
        // the tile's rows have no gaps: every m block takes a part of them all
        zero_part(out + ((long long)w.e * a.jdim + w.j0) * a.ldo, (long long)w.n * a.ldo, w.m0 / LANES + (int)me, walk.mb * CG, (int)threadIdx.x - 64, 32 * EPI_WARPS);
        continue;
      }
      const int steps = (w.r1 - w.r0 + BR - 1) / BR;
      const uint32_t lanes0 = tmem + ((uint32_t)(sub * 32) << 16), part0 = lanes0 + (uint32_t)(acc * COLS), sum0 = lanes0 + (uint32_t)((acc ^ 1) * COLS);
      for (int done = LONG;; done += LONG) {   // stages, parts of them
        if (!wait_full(s.tfull + acc, acc_phase >> acc & 1u, abort_flag, tile_ns(LONG))) {
          if (lane == 0) post(&g_status, CODE_WAIT, 44, acc, 0);
          abort_all<CG>(abort_flag, me ^ 1u);
          ok = false;
          break;
        }
        acc_phase ^= 1u << acc;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (steps <= LONG) break;
        __syncwarp();
        add_part(part0, sum0, half * 32, w.n, done == LONG);
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(CG == 2 ? map_to_cta(smem_u32(s.tempty + acc), 0) : smem_u32(s.tempty + acc));
        if (done >= steps) break;
      }
      if (!ok) break;
      const int from = steps <= LONG ? acc : acc ^ 1;   // accumulator to store
      const uint32_t t0 = steps <= LONG ? part0 : sum0;
      if (SPLIT) {   // the cluster has this one tile
        __syncwarp();
        if (F::AFTER) cluster_sync_all();
        free = true;
        send_columns(t0, sub, half * 32, w.n, inbox, cluster_ctarank(), columns_of_part(w.n, share));
        continue;
      }
      store_columns<TO>(t0, half * 32, w.n, dst, a.ldo, a.mdim - m, a.boxed, pieces + (warp - 2) * PIECE_BYTES, &mapOut, m, w.j0, MODE == TN ? w.e : 0);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(CG == 2 ? map_to_cta(smem_u32(s.tempty + from), 0) : smem_u32(s.tempty + from));
      if (steps <= LONG) acc ^= 1;
    }
    __syncwarp();
    if (F::AFTER && !free) cluster_sync_all();
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // the copy engine has read and written all boxes
    if (MODE != TN && a.fill) {
      const int first = s.table.bounds[0], last = s.table.bounds[a.off.groups];
      const int rows = first + (a.off.rows - last);
      for (long long q = (long long)blockIdx.x * EPI_WARPS + warp - 2; q < rows; q += (long long)gridDim.x * EPI_WARPS) {
        TO* row = out + (q < first ? q : q - first + last) * a.ldo;
        for (int c = lane; c < a.mdim; c += 32) row[c] = to_out<TO>(0.f);
      }
    }
  }

  if (F::AFTER && (warp < 2 || warp == FIX_WARP)) {
    __syncwarp();
    cluster_sync_all();
  }
  // Nobody leaves while the pair still reads this CTA's shared memory or signals its barriers; the parts of a split tile are in their inboxes
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncwarp();
  sync_cluster_or_block<CG == 2 || SPLIT>();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem_free<CG>(tmem, 2 * COLS);
  }
  if (SPLIT && warp >= 2 && warp < FIX_WARP && walk.has(walk.start(group, groups))) {
    const Tile w = walk.at(walk.start(group, groups));
    add_up<TO>(inbox, w.n, columns_of_part(w.n, share), cluster_ctarank(), share, 64, 32 * EPI_WARPS,
               static_cast<TO*>(a.out) + (MODE == TN ? (long long)w.e * a.jdim + w.j0 : (long long)w.j0) * a.ldo + w.m0, a.ldo, a.mdim - w.m0);
  }
}

template <int MODE, int CG, int COLS, bool SPLIT, class TO>
int launch(const CUtensorMap& p, const CUtensorMap& q, const CUtensorMap& qs, const CUtensorMap& o, const Args& a, int parts, cudaStream_t stream) {
  auto kernel = product_kernel<MODE, CG, COLS, SPLIT, TO>;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
  if (e != cudaSuccess) return (int)e;
  const long long mb = (a.mdim + Form<CG, COLS, SPLIT>::M - 1) / Form<CG, COLS, SPLIT>::M;
  const long long chunks = MODE == TN ? (long long)a.off.groups * ((a.jdim + COLS - 1) / COLS)
                                      : most_chunks(a.off.rows, a.off.groups, COLS);
  // a cluster that shares a tile has no other
  const unsigned grid = SPLIT ? (unsigned)(chunks * mb) * parts : (unsigned)min((long long)(sms / CG), chunks * mb) * CG;
  const Launch l(grid, threads_of(MODE), SMEM_BYTES, SPLIT ? parts : CG, stream);
  e = cudaLaunchKernelEx(&l.cfg, kernel, p, q, qs, o, a);
  return e != cudaSuccess ? (int)e : pcl_last_error();
}

template <int MODE, int CG, int COLS, bool SPLIT>
int launch_as(int in_type, int out_type, const CUtensorMap& p, const CUtensorMap& q, const CUtensorMap& qs, const CUtensorMap& o, const Args& a, int parts,
              cudaStream_t stream) {
  if (out_type == TYPE_F32) return launch<MODE, CG, COLS, SPLIT, float>(p, q, qs, o, a, parts, stream);
  if (out_type != in_type) return (int)cudaErrorInvalidValue;
  return in_type == TYPE_BF16 ? launch<MODE, CG, COLS, SPLIT, __nv_bfloat16>(p, q, qs, o, a, parts, stream) : launch<MODE, CG, COLS, SPLIT, __half>(p, q, qs, o, a, parts, stream);
}

// The shapes of a call's tiles: tiles of at most 64, 128 or 256 rows of Q, whichever takes the shortest time; and of 256 by pairs of CTAs, which load a third
// fewer bytes for a tile of 256 x 256 than two CTAs for theirs, where there are two tiles for every SM without (fewer spread better).  Measured, us:
// 1537 rows of 11 groups, nt, 1001 x 776: 15.1 with 64, 13.3 with 128, 16.6 with 256; 16 rows of 32 groups, nt, 1536 x 1024: 9.2 with 64, 10.3 with 256.
enum Shape { FEW, SOME, MANY, PAIR };
constexpr int FEW_COLS = 64, SOME_COLS = 128;
constexpr int SHAPE_COLS[] = {FEW_COLS, SOME_COLS, MAX_COLS, MAX_COLS / 2 /* of each CTA */};

// tn without a cluster takes the last two only: with few rows to a group its tiles have few stages, and 64 columns instead of 256 in each took 11.1 instead of 9.2 us for 1000
// rows of 24 groups, 520 x 264.
bool pairs_pay(long long chunks, int mdim) { return chunks * ((mdim + LANES - 1) / LANES) >= 2 * SMS; }

Shape shape_of(long long rows, int groups, int mdim, int steps) {
  Shape best = FEW;
  long long least = -1, chunks = 0;
  for (const Shape f : {FEW, SOME, MANY}) {
    chunks = likely_chunks(rows, groups, SHAPE_COLS[f]);
    const long long c = tiles_cost(chunks, SHAPE_COLS[f], mdim, steps);
    if (least < 0 || c < least) { least = c; best = f; }
  }
  return best == MANY && pairs_pay(chunks, mdim) ? PAIR : best;
}

template <int MODE>
int launch_shape(Shape shape, int in_type, int out_type, const CUtensorMap& p, const CUtensorMap& q, const CUtensorMap& qs, const CUtensorMap& o,
                 const Args& a, cudaStream_t stream) {
  if (shape == MANY) return launch_as<MODE, 1, MAX_COLS, false>(in_type, out_type, p, q, qs, o, a, 1, stream);
  if (shape == PAIR) return launch_as<MODE, 2, MAX_COLS, false>(in_type, out_type, p, q, qs, o, a, 1, stream);
  if constexpr (MODE != TN) {
    if (shape == SOME) return launch_as<MODE, 1, SOME_COLS, false>(in_type, out_type, p, q, qs, o, a, 1, stream);
    const long long tiles = most_chunks(a.off.rows, a.off.groups, FEW_COLS) * ((a.mdim + LANES - 1) / LANES);
    const int parts = parts_of(tiles, (a.red + BR - 1) / BR);
    return parts > 1 ? launch_as<MODE, 1, FEW_COLS, true>(in_type, out_type, p, q, qs, o, a, parts, stream)
                     : launch_as<MODE, 1, FEW_COLS, false>(in_type, out_type, p, q, qs, o, a, 1, stream);
  }
  return (int)cudaErrorInvalidValue;
}

// How tn is done: by pairs, by single CTAs, or by clusters that share the reduction of a tile of 64 or 128 columns, whichever takes the shortest time where all
// groups have the same rows.  In ns, fitted to the measurements: a stage of a cluster's CTA takes 1.6 for every line of 128 bytes (all SMs load), 1.3 with 128 columns,
// of a single CTA 0.9, or 72 for each of its loads where these are more; to send and add up the parts takes 2600 or 4900.  us without and with clusters: one group of 8192
// rows, 1024 x 1024: 50 and 28.6; of 65536 rows, 256 x 512: 357 and 45; three of 15399 rows, 1144 x 128: 42.5 and 16.4; 8 of 4096 rows, 128 x 256: 7.0 and 8.2, so
// not taken.
struct TnPlan {
  bool pair;
  int parts, cols;   // CTAs of a cluster, columns of a CTA
};

TnPlan tn_plan(long long rows, int groups, int N, int K, bool wide) {
  auto blocks = [&](int cols) { return (N + cols - 1) / cols; };
  if (pairs_pay((long long)groups * blocks(MAX_COLS), K)) return {true, 1, MAX_COLS / 2};
  const long long each = (rows + groups - 1) / groups, steps = (each + BR - 1) / BR;
  auto width = [&](int cols) { return (N + blocks(cols) - 1) / blocks(cols); };   // columns of a tile
  TnPlan plan{false, 1, MAX_COLS};
  const int loads = wide ? 2 : 2 + (width(MAX_COLS) + 63) / 64;
  long long least = steps * max(9 * (LANES + width(MAX_COLS)) / 10, 72 * loads);
  for (const int cols : {FEW_COLS, SOME_COLS}) {
    const int parts = parts_of((long long)groups * blocks(cols) * ((K + LANES - 1) / LANES), (int)steps);
    const long long t = (steps + parts - 1) / parts * (cols == FEW_COLS ? 16 : 13) * (LANES + width(cols)) / 10 + (cols == FEW_COLS ? 2600 : 4900);
    if (parts > 1 && t < least) {
      least = t;
      plan = {false, parts, cols};
    }
  }
  return plan;
}

bool sizes_ok(int in_type, long long rows, int groups, int N, int K) {
  return (in_type == TYPE_BF16 || in_type == TYPE_F16) && rows >= 0 && rows < (1ll << 31) - 512 && groups >= 1 &&
         groups <= MAX_GROUPS && N >= 1 && N < (1 << 30) && K >= 1 && K < (1 << 30);
}

// ---- operands whose rows do not start at multiples of 16 bytes ----
//
// The tensor copies cannot read these, so a call copies them first, both of a product in one launch: rows of any distance to rows of whole 16 bytes, the last one
// filled up with zeros.  Matrices of groups without rows are left out.  A block has some 1024 chunks of 16 bytes, of as many rows as these make or of a part of one;
// a thread has four.  Bound by the launch for small operands, by memory for large ones:
// 16384 x 1023 takes 18 us, 32768 x 2047 57 us, 4.7 TB/s (a general copy of strided rows 39 and 147 us).
constexpr int PAD_THREADS = 256, PAD_EACH = 4, PAD_CHUNKS = PAD_THREADS * PAD_EACH;

struct Pad {
  const uint16_t* src;
  uint4* dst;
  long long step_e, step, rows;
  unsigned per;                          // rows of a matrix
  int cols, in_block, col_blocks;        // rows of a block, blocks of a row
  bool eights;                           // rows begin at multiples of eight bytes
  long long blocks;
};

// 16 bytes from any even address, out of the one or two aligned words of 16 bytes that they lie in (either holds a byte of them, so both can be read); or from a multiple
// of eight
__device__ __forceinline__ uint4 load_chunk(const uint16_t* src, bool eights) {
  if (eights) {
    const uint2 a = reinterpret_cast<const uint2*>(src)[0], b = reinterpret_cast<const uint2*>(src)[1];
    return make_uint4(a.x, a.y, b.x, b.y);
  }
  const uint4* at = reinterpret_cast<const uint4*>((uintptr_t)src & ~(uintptr_t)15);
  const uint32_t off = (uint32_t)(uintptr_t)src & 15u;
  const uint4 lo = at[0], hi = off ? at[1] : lo;
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  if (off & 8)
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  if (off & 4)
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  const uint32_t bits = (off & 2) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                    __funnelshift_r(w[3], w[4], bits));
}

// off: null, or the bounds of the groups that have the matrices of `second`
__global__ void __launch_bounds__(PAD_THREADS) pad_kernel(const __grid_constant__ Pad first, const __grid_constant__ Pad second, const void* off, int off64) {
  after_previous();
  let_next_begin();
  const bool other = blockIdx.x >= first.blocks;
  const Pad& p = other ? second : first;
  const unsigned b = blockIdx.x - (other ? (unsigned)first.blocks : 0u);
  const unsigned row_block = b / (unsigned)p.col_blocks, col_block = b - row_block * p.col_blocks;
  const int chunks = (p.cols + 7) >> 3, c0 = (int)col_block * PAD_CHUNKS, across = min(chunks - c0, PAD_CHUNKS);
  const long long r0 = (long long)row_block * p.in_block;
  const int rows = (int)min((long long)p.in_block, p.rows - r0);
  const long long e0 = p.per == p.rows ? 0 : r0 / p.per;
  const unsigned first_row = (unsigned)(r0 - e0 * p.per);
  const float inverse = 1.f / (float)across;
  uint4 v[PAD_EACH];
  bool there[PAD_EACH];
  long long to[PAD_EACH];
#pragma unroll
  for (int i = 0; i < PAD_EACH; ++i) {
    const int at = (int)threadIdx.x + i * PAD_THREADS;
    const int r = (int)(((float)at + 0.5f) * inverse);   // at / across: below 2^10 a half is further from a whole number than the product is wrong
    const int c = c0 + at - r * across;
    there[i] = r < rows;
    v[i] = make_uint4(0, 0, 0, 0);
    if (!there[i]) continue;
    const unsigned row = first_row + (unsigned)r, more = p.per == p.rows ? 0 : row / p.per;
    const long long e = e0 + more;
    if (other && off != nullptr) {
      const long long begin = off64 ? static_cast<const long long*>(off)[e] : static_cast<const int*>(off)[e];
      const long long end = off64 ? static_cast<const long long*>(off)[e + 1] : static_cast<const int*>(off)[e + 1];
      there[i] = end > begin;   // (a group whose end is moved up has the rows of none)
      if (!there[i]) continue;
    }
    const uint16_t* src = p.src + e * p.step_e + (long long)(row - more * p.per) * p.step + c * 8ll;
    to[i] = (r0 + r) * chunks + c;
    const int left = p.cols - c * 8;
    if (left >= 8) {
      v[i] = load_chunk(src, p.eights);
    } else {
      uint16_t t[8] = {};
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < left) t[j] = src[j];
      memcpy(&v[i], t, 16);
    }
  }
#pragma unroll
  for (int i = 0; i < PAD_EACH; ++i)
    if (there[i]) p.dst[to[i]] = v[i];
}

// matrices [mats, rows, cols] of 16-bit values, the columns contiguous
bool pad_of(Pad* p, const void* src, long long step_e, long long step, long long mats, long long rows, long long cols, void* dst) {
  if (mats < 1 || rows < 1 || rows >= (1ll << 31) - 512 || cols < 1 || cols >= (1 << 30) || ((uintptr_t)src & 1) || ((uintptr_t)dst & 15)) return false;
  *p = Pad{static_cast<const uint16_t*>(src), static_cast<uint4*>(dst), step_e, step, mats * rows, (unsigned)rows, (int)cols, 1, 1, false, 0};
  p->eights = (((uintptr_t)src | (unsigned long long)(mats == 1 ? 0 : step_e) * 2 | (unsigned long long)(rows == 1 ? 0 : step) * 2) & 7) == 0;
  const int chunks = (int)((cols + 7) / 8);
  p->in_block = chunks < PAD_CHUNKS ? PAD_CHUNKS / chunks : 1;
  p->col_blocks = (chunks + PAD_CHUNKS - 1) / PAD_CHUNKS;
  p->blocks = (p->rows + p->in_block - 1) / p->in_block * p->col_blocks;
  return p->blocks < (1ll << 30);
}

}  // namespace

// Copies of one or two operands [mats, rows, cols] of 16-bit values, matrices step_e and rows step values apart, the columns contiguous: dst has
// mats * rows rows of ceil(cols / 8) * 8 values.  first or second may be null; offsets, where given, are the bounds of mats2 groups, and matrices of groups without rows are
// not copied.
PCL_API int pcl_grouped_pad(const void* first, long long step_e, long long step, long long mats, long long rows, int cols, void* dst, const void* second,
                            long long step_e2, long long step2, long long mats2, long long rows2, int cols2, void* dst2, const void* offsets, int off64,
                            cudaStream_t stream) {
  Pad a{}, b{};
  if (first != nullptr && !pad_of(&a, first, step_e, step, mats, rows, cols, dst)) return (int)cudaErrorInvalidValue;
  if (second != nullptr && !pad_of(&b, second, step_e2, step2, mats2, rows2, cols2, dst2)) return (int)cudaErrorInvalidValue;
  if (a.blocks + b.blocks == 0) return (int)cudaErrorInvalidValue;
  Launch l((unsigned)(a.blocks + b.blocks), PAD_THREADS, 0, 1, stream);
  return (int)cudaLaunchKernelEx(&l.cfg, pad_kernel, a, b, offsets, off64);
}

// mode 0: X [rows, K] -> out [rows, N]; mode 1: X [rows, N] -> out [rows, K].  W [groups, N, K] with strides (ws_e, ws_n, 1); rows of X and W
// start at multiples of 16 bytes.  in_type 1 / 2 (bf16 / fp16), out_type the same or 0 (fp32).  fill: rows of no group
// become zero, else they are left.
PCL_API int pcl_grouped_rows(int mode, int in_type, int out_type, const void* X, long long ldx, const void* W,
                             long long ws_e, long long ws_n, const void* offsets, int off64, void* out,
                             long long ldo, long long rows, int groups, int N, int K, int fill,
                             cudaStream_t stream) {
  if (!sizes_ok(in_type, rows, groups, N, K) || (mode != 0 && mode != 1)) return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  const CUtensorMapDataType t = in_type == TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const int red = mode == 0 ? K : N;
  const Shape shape = shape_of(rows, groups, mode == 0 ? N : K, (red + BR - 1) / BR);
  CUtensorMap p, q, qs, o;
  int rc = make_map_3d(&p, t, W, K, N, groups, ws_n * 2, ws_e * 2, 64, mode == 0 ? LANES : BR);
  if (rc == 0) rc = make_map_3d(&q, t, X, red, rows, 1, ldx * 2, ldx * 2, BR, SHAPE_COLS[shape]);
  if (rc == 0) rc = make_map_3d(&qs, t, X, red, rows, 1, ldx * 2, ldx * 2, BR, SHAPE_COLS[shape] / 4);
  if (rc) return rc;
  Args a{out, ldo, Offsets{offsets, off64, groups, (int)rows}, mode == 0 ? N : K, 0, red, in_type == TYPE_BF16 ? 1u : 0u, fill, false, false};
  a.boxed = make_out_map(&o, p, out_type, out, a.mdim, rows, 1, ldo, ldo);
  if (mode == 0) return launch_shape<NT>(shape, in_type, out_type, p, q, qs, o, a, stream);
  return launch_shape<NN>(shape, in_type, out_type, p, q, qs, o, a, stream);
}

// out [groups, N, K] (contiguous): every matrix is written, zeros where a group has no row
PCL_API int pcl_grouped_tn(int in_type, int out_type, const void* Y, long long ldy, const void* X, long long ldx,
                           const void* offsets, int off64, void* out, long long rows, int groups, int N, int K,
                           cudaStream_t stream) {
  if (!sizes_ok(in_type, rows, groups, N, K) || rows == 0) return (int)cudaErrorInvalidValue;
  const CUtensorMapDataType t = in_type == TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  // (a block that is not full would reach into the next row, and behind the last one)
  const bool wide = N % 64 == 0 && K % 64 == 0;
  const TnPlan plan = tn_plan(rows, groups, N, K, wide);
  CUtensorMap p, q, o;
  int rc = 0;
  if (wide) {
    rc = make_map_3d(&p, t, X, 64, rows, K / 64, ldx * 2, 128, 64, BR, CU_TENSOR_MAP_SWIZZLE_128B, LANES / 64);
    if (rc == 0) rc = make_map_3d(&q, t, Y, 64, rows, N / 64, ldy * 2, 128, 64, BR, CU_TENSOR_MAP_SWIZZLE_128B, plan.cols / 64);
  } else {
    rc = make_map_3d(&p, t, X, K, rows, 1, ldx * 2, ldx * 2, 64, BR);
    if (rc == 0) rc = make_map_3d(&q, t, Y, N, rows, 1, ldy * 2, ldy * 2, 64, BR);
  }
  if (rc) return rc;
  Args a{out, K, Offsets{offsets, off64, groups, (int)rows}, K, N, 0, in_type == TYPE_BF16 ? 1u : 0u, 0, false, wide};
  a.boxed = make_out_map(&o, p, out_type, out, K, N, groups, K, (long long)N * K);
  if (plan.parts > 1)
    return plan.cols == FEW_COLS ? launch_as<TN, 1, FEW_COLS, true>(in_type, out_type, p, q, q, o, a, plan.parts, stream)
                                 : launch_as<TN, 1, SOME_COLS, true>(in_type, out_type, p, q, q, o, a, plan.parts, stream);
  return launch_shape<TN>(plan.pair ? PAIR : MANY, in_type, out_type, p, q, q, o, a, stream);
}

// Moves the report that the status block of the grouped products holds, if any, to `to` in the device's memory, behind what the stream has so far.
PCL_API int pcl_grouped_status(PclStatus* to, cudaStream_t stream) {
  take_kernel<<<1, 1, 0, stream>>>(to);
  return pcl_last_error();
}
