// Building blocks of the tcgen05 products over groups of rows: the table that turns a tile's number into its group and rows,
// and the forms of loads, products and commits for one CTA (CG 1) and for a pair (CG 2).
//
// Every product here is D[m, j] = sum_r P[m, r] Q[j, r]: the 128 lanes of a CTA's tensor memory are rows m of P, the accumulator's
// columns rows j of Q.  The matrices of the groups are P and the rows that share them Q, so that a ragged
// group costs its rows rounded up to 16 columns instead of to 128 lanes, and neighbouring lanes store
// neighbouring values of a row of the result.
#pragma once
#include "gemm_sm100.cuh"
#include "grouped.cuh"

namespace pcl_tiles {

using namespace pcl_sm100;

constexpr int MAX_COLS = 256;   // columns of an accumulator
constexpr int SMS = 148;        // that the rules for a call's shape count on

// Rows of a chunk where `rows` are cut into `parts` chunks, as equal as multiples of `step` allow.  (Not (rows + parts - 1) / parts: that leaves 32 bits from 2.11e9 rows on.)
__host__ __device__ constexpr int chunk_size(int rows, int parts, int step) { return ((rows - 1) / parts + 1 + step - 1) / step * step; }

constexpr int MOST_ROWS = (int)((1ll << 31) - 513);   // of a call
__host__ __device__ constexpr int chunks_of(int rows, int most) { return (rows + most - 1) / most; }
constexpr bool cut_right(int rows, int most, int step) {
  const int parts = chunks_of(rows, most), size = chunk_size(rows, parts, step);
  return size > 0 && size <= most && (long long)size * parts >= rows && (long long)size * (parts - 1) < rows;
}
static_assert(cut_right(MOST_ROWS, 64, 16) && cut_right(MOST_ROWS, 128, 16) && cut_right(MOST_ROWS, 208, 16) && cut_right(MOST_ROWS, 256, 32), "as many rows as a call takes");
static_assert(cut_right(MOST_ROWS - 1601, 64, 16) && cut_right(2114537830, 64, 16) && cut_right(1, 64, 16) && cut_right(65, 64, 16) && cut_right(257, 256, 32), "and others");

// The rows of a group are cut into chunks of at most MAX_COLS, as equal as multiples of `step` allow.
struct Table {
  int bounds[pcl_group::MAX_GROUPS + 1];
  int chunks[pcl_group::MAX_GROUPS + 1];   // chunks of the groups before

  // By the first warp, behind load_bounds and a barrier.  Bounds are made ascending (each at least the one before it) whatever the array
  // holds, so that no row is in two groups; the first one that had to be moved goes into the status block.
  __device__ __forceinline__ void build(int groups, int most, PclStatus* st) {
    const int lane = threadIdx.x;
    int top = bounds[0], carry = 0, moved = -1, from = 0;
    for (int i0 = 0; i0 < groups; i0 += 32) {
      const int i = i0 + lane + 1;
      const int own = i <= groups ? bounds[i] : 0;
      int v = max(own, top);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v = max(v, u);
      }
      int before = __shfl_up_sync(0xffffffffu, v, 1);
      if (lane == 0) before = top;
      top = __shfl_sync(0xffffffffu, v, 31);
      if (i <= groups) {
        bounds[i] = v;
        if (v != own && moved < 0) {
          moved = i;
          from = own;
        }
      }
      const int parts = i <= groups ? chunks_of(v - before, most) : 0;
      int sum = parts;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += u;
      }
      if (i <= groups) chunks[i - 1] = carry + sum - parts;
      carry += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) chunks[groups] = carry;
    if (moved >= 0) pcl_group::post(st, pcl_group::CODE_BOUNDS, 110, moved, from);
  }

  // `step` divides `most`: a chunk is then at most `most` rows, and all but the last of a group's chunks cannot hold all its rows.
  // Rows [begin, begin + n) of chunk `c`, in group `e`, the last whose chunks begin at or before `c`
  __device__ __forceinline__ void find(int groups, int c, int step, int& e, int& begin, int& n) const {
    int hi = groups;   // chunks[e] <= c < chunks[hi]
    e = 0;
    while (hi - e > 1) {
      const int mid = (e + hi) >> 1;
      if (chunks[mid] <= c) e = mid;
      else hi = mid;
    }
    const int rows = bounds[e + 1] - bounds[e], parts = chunks[e + 1] - chunks[e];
    const int size = chunk_size(rows, parts, step);
    begin = bounds[e] + (c - chunks[e]) * size;
    n = min(size, bounds[e + 1] - begin);
  }
};

// One lane of a converged warp.  Loads by the copy engine, products and commits take their operands from the warp's uniform
// registers: issued under this condition by a warp that runs its loop as a whole they cost a few instructions, under
// `lane == 0` several times as many.
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// Whether the phase has passed, without waiting.  The answer takes 85 cycles: asked for the next stage while the products of this one are issued, it
// costs nothing where the stage has arrived.
__device__ __forceinline__ bool has_passed(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

// as mbar_wait, for a barrier that the other CTA of a pair arrives on; the limit grows by `more_ns`
__device__ __forceinline__ bool wait_full(uint64_t* bar, uint32_t parity, volatile int* abort_flag, unsigned long long more_ns = 0) {
  const uint32_t addr = smem_u32(bar);
  unsigned long long t0 = 0;
  for (unsigned it = 0;; ++it) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return true;
    if ((it & 31) == 31) {
      if (*abort_flag) return false;
      const unsigned long long now = pcl_globaltimer();
      if (t0 == 0) t0 = now;
      else if (now - t0 > WAIT_NS + more_ns) return false;
    }
  }
}
// What `steps` stages may take beyond the usual limit (a stage takes a fraction of a microsecond; a reduction over 2^31 rows has 2^25)
__device__ __forceinline__ unsigned long long tile_ns(long long steps) { return 2000ull * (unsigned long long)steps; }

// arrive on a barrier given by its cluster address, after this CTA's writes to its shared memory
__device__ __forceinline__ void arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// raise the abort flag, of both CTAs of a pair
template <int CG>
__device__ __forceinline__ void abort_all(volatile int* abort_flag, uint32_t peer) {
  *abort_flag = 1;
  if (CG == 2)
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(map_to_cta(smem_u32((const void*)abort_flag), peer)), "r"(1) : "memory");
}

// box of a three-dimensional map into this CTA's shared memory; the bytes count on `bar` (of the pair's leader for CG 2)
template <int CG>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  if (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// arrive on the barrier at this shared-memory address (in both CTAs of a pair) once every product issued so far by this thread has finished
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if (CG == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3)
                 : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

template <int CG>
__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  if (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
        : "memory");
}

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, int cols) {
  if (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
}

template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t base, int cols) {
  if (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols));
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols));
}

// A CTA's (or cluster's) tiles, first, first + step, ..: tile c * across + m is block m of chunk c.  No division but at the start, and that in 32 bits: one in
// 64 takes longer than a short tile.
struct Counter {
  int c, m, dc, dm, across;
  __device__ Counter(int first, int step, int across_) : across(across_) {
    c = first / across;
    m = first - c * across;
    dc = step / across;
    dm = step - dc * across;
  }
  __device__ __forceinline__ void next() {
    c += dc;
    m += dm;
    if (m >= across) { m -= across; ++c; }
  }
};

// The same tiles in turn, for a whole warp: its lanes look the next 32 up together, since finding one takes 300 to 800 cycles, most of the time that a warp was
// busy with a short tile (four-bit product of 16384 rows of 32 groups, 4096 x 256: 55 us when each was found by itself, 39 so).  ONE: there is one at most.
template <class Walk, bool ONE>
struct Tiles {
  using Tile = decltype(static_cast<const Walk*>(nullptr)->at(static_cast<const Counter*>(nullptr)[0]));
  const Walk& walk;
  Counter own;
  Tile mine;
  uint32_t there;   // lanes that found one
  int k;

  __device__ __forceinline__ Tiles(const Walk& w, int first, int step)
      : walk(w), own(ONE ? first : first + ((int)threadIdx.x & 31) * step, 32 * step, w.mb), mine{} {
    look();
  }
  __device__ __forceinline__ void look() {
    const bool found = walk.has(own);
    if (found) mine = walk.at(own);
    there = ONE ? found : __ballot_sync(0xffffffffu, found);
    k = 0;
  }
  __device__ __forceinline__ bool has() const { return there >> k & 1u; }
  __device__ __forceinline__ Tile tile() const {
    static_assert(sizeof(Tile) % 4 == 0, "whole words");
    if (ONE) return mine;
    int v[sizeof(Tile) / 4];
    memcpy(v, &mine, sizeof(Tile));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Tile) / 4); ++i) v[i] = __shfl_sync(0xffffffffu, v[i], k);
    Tile t;
    memcpy(&t, v, sizeof(Tile));
    return t;
  }
  __device__ __forceinline__ void next() {
    if (++k < 32 || ONE) return;
    own.next();
    look();
  }
};

// The kernels here are launched while the one before them in the stream may still run, so that their blocks find their place and set up barriers and tensor
// memory meanwhile (2 to 3 us of a call that takes 5 to 10); `after_previous` comes before the first access to global memory.  They let the next one
// begin the same way from their own start: it waits for their end.
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <bool CLUSTER>
__device__ __forceinline__ void sync_cluster_or_block() {
  __syncthreads();
  if (CLUSTER) {
    __syncwarp();
    cluster_sync_all();
  }
}

// Operand tile whose rows are contiguous along the reduction: 128-byte rows, eight of them swizzled together, groups of eight 1 KB apart.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t saddr) { return make_desc_sw128(saddr); }

// Operand tile whose rows are contiguous along m (or j): boxes of 64 values x 64 steps of the reduction (8 KB) side by side, groups of eight
// steps 1 KB apart.
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t saddr) {
  const uint32_t lo = ((saddr >> 4) & 0x3FFFu) | (512u << 16);
  const uint32_t hi = 64u | (1u << 14) | (2u << 29);
  return ((uint64_t)hi << 32) | lo;
}

// 16 lanes x 32 columns of tensor memory: register 4 i + q of thread t holds lane t / 4 + 8 (q / 2), column 8 i + 2 (t mod 4) + q mod 2
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// low half: a, high half: b
static __device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
static __device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Where a warp puts 32 columns x 32 lanes of its accumulator for the copy engine: 2 KB, rows of 64 bytes (a column's 32 lanes)
constexpr int PIECE_BYTES = 2048;

// 8 columns of the warp's 32 lanes
static __device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}

// The tensor cores cut off what they add to an accumulator, always towards zero, so that its error grows with the number of additions: a sum of a million terms of one sign
// lost 0.7 % in one accumulator (1.2e-3 where signs differ).  A reduction of more stages than LONG is therefore done in parts of LONG stages, and the
// parts are added up in fp32, rounded, by the warps that store: the error stays that of 8192 terms (9e-6, 3.5e-5 of one sign).  The tensor cores wait meanwhile: 0 to 2.5 % of such a call
// (one group of 65536 rows, 4096 x 4096: 1503 us in one accumulator, 1534 so; with parts of 64 stages, and the next tile behind the sum's store, 1580).
constexpr int LONG = 128;

// 16 columns of the warp's 32 lanes, from and to tensor memory; loaded registers are read behind a wait that names them
static __device__ __forceinline__ void tmem_ld16_issue(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
static __device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// The warp's columns (32 of every 64 from `first` on, up to n) of the accumulator `part` begin those of `sum`, or are added to them.
static __device__ __noinline__ void add_part(uint32_t part, uint32_t sum, int first, int n, bool begin) {
#pragma unroll 1
  for (int c = first; c < n; c += ((c & 31) == 16 ? 48 : 16)) {
    uint32_t v[16];
    tmem_ld16_issue(part + (uint32_t)c, v);
    if (begin) {
      asm volatile("tcgen05.wait::ld.sync.aligned;"
                   : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                     "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                   :
                   : "memory");
      tmem_st16(sum + (uint32_t)c, v);
    } else {
      uint32_t u[16];
      tmem_ld16_issue(sum + (uint32_t)c, u);
      asm volatile("tcgen05.wait::ld.sync.aligned;"
                   : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                     "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]),
                     "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]), "+r"(u[8]), "+r"(u[9]), "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]),
                     "+r"(u[14]), "+r"(u[15])
                   :
                   : "memory");
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(u[j]));
      tmem_st16(sum + (uint32_t)c, v);
    }
  }
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// n columns lane by lane, a row's 32 neighbours at a time: short code, for the few columns of short calls
template <class TO>
__device__ __forceinline__ void store_singly(uint32_t taddr, int n, TO* dst, long long ldo, int lanes) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int c = 0; c < n; c += 8) {
    uint32_t v[8];
    tmem_ld8(taddr + (uint32_t)c, v);
    if (lane < lanes) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < n) dst[(c + j) * ldo + lane] = pcl_group::to_out<TO>(__uint_as_float(v[j]));
    }
    __syncwarp();
  }
}

// 32 rows of `count` 16-bit values out of `piece` (as store_columns leaves them there) to rows that begin at multiples of sizeof(V) bytes, several a store
template <class V, class TO>
__device__ __forceinline__ void store_words(const uint8_t* piece, TO* dst, long long ldo, int count) {
  constexpr int EACH = sizeof(V) / 2, ACROSS = 32 / EACH;
  const int lane = threadIdx.x & 31, e = lane % ACROSS * EACH;
#pragma unroll 4
  for (int j = lane / ACROSS; j < 32; j += 32 / ACROSS) {
    const uint8_t* from = piece + j * 64 + (((e >> 3) ^ ((j >> 1) & 3)) << 4) + (e & 7) * 2;
    TO* to = dst + j * ldo + e;
    if (e + EACH <= count) {
      *reinterpret_cast<V*>(to) = *reinterpret_cast<const V*>(from);
    } else {
#pragma unroll
      for (int q = 0; q < EACH - 1; ++q)
        if (e + q < count) to[q] = reinterpret_cast<const TO*>(from)[q];
    }
  }
}

// Zeros to part `part` of `parts` of n values, by `threads` threads: 16 bytes a store, but for the ends (by rows of 64 bytes, dW of 8 rows of 64 groups,
// 2048 x 1024, took 60 instead of 46 us)
template <class TO>
__device__ __forceinline__ void zero_part(TO* dst, long long n, int part, int parts, int thread, int threads) {
  TO *from = dst + n * part / parts, *end = dst + n * (part + 1) / parts;
  constexpr int EACH = 16 / sizeof(TO);
  const long long count = end - from;
  const long long head = min(count, (long long)((16 - ((uintptr_t)from & 15)) & 15) / (long long)sizeof(TO)), words = (count - head) / EACH;
  const long long tail = head + words * EACH;
  if (thread < head) from[thread] = pcl_group::to_out<TO>(0.f);
  if (tail + thread < count) from[tail + thread] = pcl_group::to_out<TO>(0.f);
  for (long long q = thread; q < words; q += threads) reinterpret_cast<uint4*>(from + head)[q] = make_uint4(0, 0, 0, 0);
}

// A warp's part of an accumulator goes to out: column j of [0, n) and the warp's 32 lanes to dst[j * ldo + lane], lanes < `lanes` only.  Columns 32 at a time,
// first + 0, 64, 128 ..  16-bit results turn around in shared memory (stmatrix) and leave as boxes of 32 rows
// x 64 bytes, where `boxed` says that the map can take them, or by words of eight or four bytes (the last lanes of rows whose length is no multiple of 16 bytes always); what is left of a chunk, and rows that begin anywhere, are stored lane by lane, a row's 32
// neighbours at a time (stored so throughout, nt of 16 groups of 1024 rows, 2048 x 1024 took 81 instead of 68 us: a store of one row takes an SM 11 cycles, of
// 64 bytes or of 128).
template <class TO>
__device__ __forceinline__ void store_columns(uint32_t taddr, int first, int n, TO* dst, long long ldo, int lanes, bool boxed, uint8_t* piece,
                                              const CUtensorMap* map, int x, int y, int z) {
  const int lane = threadIdx.x & 31;
  const uint32_t bits = (uint32_t)(uintptr_t)dst | (uint32_t)ldo * 2u;
  const int word = (bits & 7) == 0 ? 8 : (bits & 3) == 0 ? 4 : 2;   // bytes
  // The copy engine writes 16 bytes whole, those behind a map's last column among them, which in a strided result are someone else's
  boxed = boxed && (lanes >= 32 || (lanes & 7) == 0);
  for (int c = first; c < n; c += 64) {
    if (sizeof(TO) == 2 && (boxed || word > 2) && c + 32 <= n) {
      uint32_t lo[16], hi[16];
      tmem_ld_16x32(taddr + (uint32_t)c, lo);
      tmem_ld_16x32(taddr + (16u << 16) + (uint32_t)c, hi);
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // the last box has been read
      __syncwarp();
      asm volatile("tcgen05.wait::ld.sync.aligned;"
                   : "+r"(lo[0]), "+r"(lo[1]), "+r"(lo[2]), "+r"(lo[3]), "+r"(lo[4]), "+r"(lo[5]), "+r"(lo[6]), "+r"(lo[7]),
                     "+r"(lo[8]), "+r"(lo[9]), "+r"(lo[10]), "+r"(lo[11]), "+r"(lo[12]), "+r"(lo[13]), "+r"(lo[14]), "+r"(lo[15]),
                     "+r"(hi[0]), "+r"(hi[1]), "+r"(hi[2]), "+r"(hi[3]), "+r"(hi[4]), "+r"(hi[5]), "+r"(hi[6]), "+r"(hi[7]),
                     "+r"(hi[8]), "+r"(hi[9]), "+r"(hi[10]), "+r"(hi[11]), "+r"(hi[12]), "+r"(hi[13]), "+r"(hi[14]), "+r"(hi[15])
                   :
                   : "memory");
      auto two = [&](const uint32_t* r) { return pack2(__uint_as_float(r[0]), __uint_as_float(r[1]), TO()); };
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 8 * i + (lane & 7);
        const uint32_t at = smem_u32(piece) + j * 64 + (((lane >> 3) ^ ((j >> 1) & 3)) << 4);
        asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(two(lo + 4 * i)),
                     "r"(two(lo + 4 * i + 2)), "r"(two(hi + 4 * i)), "r"(two(hi + 4 * i + 2))
                     : "memory");
      }
      if (!boxed) {
        __syncwarp();
        if (word == 8) store_words<uint2>(piece, dst + (long long)c * ldo, ldo, lanes);
        else store_words<uint32_t>(piece, dst + (long long)c * ldo, ldo, lanes);
        __syncwarp();
        continue;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0 && lanes > 0) {
        asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(smem_u32(piece)),
                     "r"(x), "r"(y + c), "r"(z)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    } else {
      store_singly(taddr + (uint32_t)c, min(32, n - c), dst + (long long)c * ldo, ldo, lanes);
    }
    __syncwarp();
  }
}
// 32 bits a value: sixteen columns at a time go through shared memory, and leave as four rows a store where these begin at multiples of 16 bytes (four-bit product
// of 16384 rows of 32 groups, 4096 x 256: 101 us by single rows, 59 so; tn of 1537 rows of 11 groups, 1001 x 776: 26 and 18)
template <>
__device__ __forceinline__ void store_columns<float>(uint32_t taddr, int first, int n, float* dst, long long ldo, int lanes, bool, uint8_t* piece,
                                                     const CUtensorMap*, int, int, int) {
  const int lane = threadIdx.x & 31;
  const bool quads = lanes >= 32 && (((uintptr_t)dst | (uintptr_t)ldo * 4) & 15) == 0;
  for (int c0 = first; c0 < n; c0 += 64) {
#pragma unroll 1
    for (int c = c0; c < min(c0 + 32, n); c += 16) {
      float* to = dst + (long long)c * ldo;
      if (quads && c + 16 <= n) {
        uint32_t v[16];
        tmem_ld8(taddr + (uint32_t)c, v);
        tmem_ld8(taddr + (uint32_t)c + 8, v + 8);
#pragma unroll
        for (int j = 0; j < 16; ++j) *reinterpret_cast<uint32_t*>(piece + j * 128 + lane * 4) = v[j];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = 4 * i + (lane >> 3);
          *reinterpret_cast<uint4*>(to + j * ldo + (lane & 7) * 4) = *reinterpret_cast<const uint4*>(piece + j * 128 + (lane & 7) * 16);
        }
        __syncwarp();
      } else {
        store_singly(taddr + (uint32_t)c, min(16, n - c), to, ldo, lanes);
      }
    }
  }
}

// ---- one tile by a cluster: every CTA has a part of the reduction, and adds up the parts of some of the columns

static __device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}

constexpr int inbox_bytes(int cols) { return (cols + 4 * 8) * 128 * 4; }   // up to `cols` columns, four to each of 8 parts more
__device__ __forceinline__ int columns_of_part(int n, int parts) { return ((n + parts - 1) / parts + 3) & ~3; }

// This warp's quarter of the accumulator (zeros for `none`) to the CTAs that add it up: columns [o * each, (o + 1) * each) go to CTA o, there into
// inbox[rank][column / 4][lane][column mod 4]
static __device__ __forceinline__ void send_columns(uint32_t taddr, int sub, int first, int n, const float* inbox, uint32_t rank, int each,
                                                    bool none = false) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int c = first; c < n; c += ((c & 31) == 24 ? 40 : 8)) {   // 32 columns of every 64, eight at a time
    uint32_t v[8] = {};
    if (!none) tmem_ld8(taddr + (uint32_t)c, v);
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      if (c + j < n) {
        const int owner = (c + j) / each, col = c + j - owner * each;
        const uint32_t at = map_to_cta(smem_u32(inbox + ((int)rank * each + col) * 128 + (sub * 32 + lane) * 4), (uint32_t)owner);
        asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[j]), "r"(v[j + 1]), "r"(v[j + 2]), "r"(v[j + 3]) : "memory");
      }
    }
    __syncwarp();
  }
}

// Behind the cluster's barrier: this CTA's columns, added up in the order of the parts, to dst[column * ldo + lane]; by `threads` threads from `first` on
template <class TO>
__device__ __forceinline__ void add_up(const float* inbox, int n, int each, uint32_t rank, int parts, int first, int threads, TO* dst, long long ldo, int lanes) {
  const int mine = min(each, n - (int)rank * each);
  for (int i = (int)threadIdx.x - first; i < (mine + 3) / 4 * 128; i += threads) {
    const int col = i >> 7 << 2, l = i & 127;
    float v[4] = {};
    for (int p = 0; p < parts; ++p) {
      const float4 u = *reinterpret_cast<const float4*>(inbox + (p * each + col) * 128 + l * 4);
      v[0] += u.x;
      v[1] += u.y;
      v[2] += u.z;
      v[3] += u.w;
    }
    if (l < lanes) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < mine) dst[((long long)rank * each + col + j) * ldo + l] = pcl_group::to_out<TO>(v[j]);
    }
  }
}

// the most chunks of at most `cols` rows that `rows` rows of `groups` groups can make
static inline long long most_chunks(long long rows, int groups, int cols) {
  const long long taken = rows < groups ? rows : groups;   // groups with a row
  return (rows - taken) / cols + taken;
}

// How long a call of single CTAs takes with `chunks` chunks of at most `cols` rows of Q, in units of about 2.5 cycles.  A CTA takes in 52 bytes a cycle
// whatever it computes, so a stage costs its 128 + cols lines of 128 bytes; storing a tile takes 21 cycles a column, beside the
// next tile's stages.
static inline long long tiles_cost(long long chunks, int cols, int mdim, int steps) {
  const long long tiles = chunks * ((mdim + 127) / 128), store = 9ll * cols, main = (long long)steps * (128 + cols);
  return (tiles + SMS - 1) / SMS * (main > store ? main : store) + store;
}

// Chunks that `rows` rows of `groups` groups may be expected to make: half a chunk more for each group, one at least
static inline long long likely_chunks(long long rows, int groups, int cols) {
  const long long taken = rows < groups ? rows : groups, all = (rows + cols - 1) / cols;
  return taken <= 1 ? all : (taken > all + taken / 2 ? taken : all + taken / 2);
}

// Clusters of 1 to 8 CTAs that run at the same time, one CTA to an SM, as the runtime counts them: they do not straddle the processor's parts of some 16 SMs,
// and one more runs alone behind the others (one row times 2048 x 2048: 11.8 us by 16 clusters of 8, 7.2 by 16 of 6).
constexpr int CLUSTERS[] = {0, 148, 74, 45, 33, 26, 22, 15, 15};

// Parts that a tile's reduction of `steps` stages is cut into: as many as `tiles` clusters that run at the same time can have, at most
// eight (the largest portable cluster), and two stages at least for each.  1: not cut.
static inline int parts_of(long long tiles, int steps) {
  int parts = steps < 8 ? 1 : steps < 16 ? steps / 2 : 8;
  while (parts > 1 && tiles > CLUSTERS[parts]) --parts;
  return parts;
}

// A launch in clusters of `cluster` CTAs, behind the previous kernel of the stream as `let_next_begin` says
struct Launch {
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};

  Launch(unsigned grid, int threads, size_t smem, int cluster, cudaStream_t stream) {
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    if (cluster > 1) {
      attr[1].id = cudaLaunchAttributeClusterDimension;
      attr[1].val.clusterDim.x = (unsigned)cluster;
      attr[1].val.clusterDim.y = 1;
      attr[1].val.clusterDim.z = 1;
      cfg.numAttrs = 2;
    }
  }
};

// map of `depth` matrices [rows x inner]; strides in bytes; box: box_in values x box_rows rows x box_mats matrices.  `inner` and box_in count elements of `type`.
static inline int make_map_3d(CUtensorMap* map, CUtensorMapDataType type, const void* ptr, long long inner, long long rows, long long depth,
                              long long row_bytes, long long mat_bytes, int box_in, int box_rows,
                              CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B, int box_mats = 1) {
  encode_fn_t enc = get_encode2();
  if (enc == nullptr) return (int)cudaErrorNotSupported;
  cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)depth};
  cuuint64_t strides[2] = {(cuuint64_t)row_bytes, (cuuint64_t)mat_bytes};
  cuuint32_t box[3] = {(cuuint32_t)box_in, (cuuint32_t)box_rows, (cuuint32_t)box_mats};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(map, type, 3, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

// The map that store_columns writes through, of `depth` results [rows x inner] of 16 bits; false where its rows do not start at multiples of 16
// bytes (or the map cannot be made): then `map` becomes a copy of `other`, and is not used.
static inline bool make_out_map(CUtensorMap* map, const CUtensorMap& other, int out_type, const void* out, long long inner, long long rows, long long depth,
                                long long ldo, long long ld_mat) {
  *map = other;
  if (out_type == pcl_group::TYPE_F32 || ((uintptr_t)out & 15) || (ldo * 2 & 15) || (ld_mat * 2 & 15)) return false;
  const CUtensorMapDataType t = out_type == pcl_group::TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return make_map_3d(map, t, out, inner, rows, depth, ldo * 2, ld_mat * 2, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B) == 0;
}

}  // namespace pcl_tiles
