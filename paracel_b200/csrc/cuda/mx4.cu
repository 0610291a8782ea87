// Matrices in four bits with a shared scale for every 32 values of a row (OCP microscaling format, elements E2M1, scales
// E8M0): quantisation, its reverse, and the product of two of them, also with one right-hand matrix for each group of rows.
//
// Layout, `rows` x K: data [rows, 16 ceil(K / 32)] bytes, value 2 j of a row in the low half of byte j, 2 j + 1 in the high
// half; scales [ceil(K / 128), rows] words of four codes, byte i of word (b, r) is the code of row r's block 4 b + i.
// A word holds the scales of 128 values, and the words of neighbouring rows are neighbours: a tile of rows finds its
// scales in one piece wherever it begins.  A code c stands for 2^(c - 127), 255 for NaN.
#include "tiles_sm100.cuh"

namespace {

using namespace pcl_group;
using namespace pcl_tiles;

// the file is compiled with subnormals flushed to zero: a plain product would lose blocks whose scale is below 2^-126
__device__ __forceinline__ float mul_keep(float a, float b) {
  float d;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ float scale_value(int code) {   // 2^(code - 127)
  return __uint_as_float(code == 255 ? 0x7fc00000u : code == 0 ? 0x00400000u : (uint32_t)code << 23);
}

// eight values in four bits each, v[0] in the lowest: to nearest, ties to the even code, beyond 6 to 6
__device__ __forceinline__ uint32_t pack8(const float* v) {
  uint32_t d;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(d)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return d;
}

// the values of eight codes, v[0] of the lowest: the conversion to fp16 is exact
__device__ __forceinline__ void unpack8(uint32_t codes, float* v) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(h + i));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

struct QuantArgs {
  const void* x;
  long long ldx;
  uint32_t* data;      // 4 bytes = 8 values
  uint32_t* scales;
  long long rows;
  int K, words;        // words: ceil(K / 128)
  int vec;             // rows of x can be read 16 bytes at a time
  int shift;           // log2 of the words side by side in a CTA
};

// A thread takes eight neighbouring values of a row, four lanes make a block of 32 and sixteen a word of scales, 128 values.  A CTA has 16 ITERS words, of which
// 2^shift lie side by side in a row: 1024 columns of eight rows where rows are that long, and 64 rows of 128 columns.  All loads of a thread come before
// the first use, and the words of neighbouring rows are stored together.  Bound by memory: 32768 x 8192 of bf16 takes 120 us (5.7 TB/s) and of fp32 178 us
// (6.8 TB/s), back to bf16 110 us (6.2 TB/s); 1000000 x 128 of fp32 89 us (6.5 TB/s; 418 where a CTA's rows have 1024 columns whatever the matrix has).  The registers are
// bounded so that six blocks share an SM: with five of them quantisation of bf16 takes 164 us, with seven, whose loads no longer fit, 224.
constexpr int QTHREADS = 256;

template <int ITERS>
struct Units {
  static constexpr int COUNT = 16 * ITERS, LOG = ITERS == 4 ? 6 : 4;
  long long r0;
  int word0, shift;

  __device__ Units(int words, int shift_) : shift(shift_) {
    const int across = (words + (1 << shift) - 1) >> shift;
    word0 = (int)(blockIdx.x % across) << shift;
    r0 = (long long)(blockIdx.x / across) << (LOG - shift);
  }
  // of this thread: its word, the same in every pass, its row in the first, and the rows from one pass to the next
  __device__ int word() const { return word0 + ((threadIdx.x >> 4) & ((1 << shift) - 1)); }
  __device__ long long row() const { return r0 + (threadIdx.x >> (4 + shift)); }
  __device__ int step() const { return 16 >> shift; }
};

// The largest magnitude of eight values, as the bits of an fp32 value: compared by their bits NaN and infinity come out on top.  16-bit values are
// compared in pairs, before they are widened.
template <class T>
__device__ __forceinline__ uint32_t top_bits(const uint4* raw);
template <>
__device__ __forceinline__ uint32_t top_bits<float>(const uint4* raw) {
  constexpr uint32_t M = 0x7fffffffu;
  const uint32_t a = max(max(raw[0].x & M, raw[0].y & M), max(raw[0].z & M, raw[0].w & M));
  const uint32_t b = max(max(raw[1].x & M, raw[1].y & M), max(raw[1].z & M, raw[1].w & M));
  return max(a, b);
}
__device__ __forceinline__ uint32_t top_16(const uint4& r) {
  constexpr uint32_t M = 0x7fff7fffu;
  const uint32_t m = __vmaxu2(__vmaxu2(r.x & M, r.y & M), __vmaxu2(r.z & M, r.w & M));
  return max(m & 0xffffu, m >> 16);
}
template <>
__device__ __forceinline__ uint32_t top_bits<__nv_bfloat16>(const uint4* raw) { return top_16(raw[0]) << 16; }
template <>
__device__ __forceinline__ uint32_t top_bits<__half>(const uint4* raw) {
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)top_16(raw[0]))));
}

// Eight values of a block that starts at a multiple of four lanes, `most` the bits of the largest magnitude of these: their codes, and in `word` the word of scales
// of the sixteen lanes around.  `in`: the row has this block.
__device__ __forceinline__ uint32_t encode8(float (&v)[8], uint32_t most, bool in, int part, uint32_t& word) {
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
  const bool bad = most >= 0x7f800000u;
  // floor(log2(most)) - 2, at least -127 (all that is below 2^-125 takes the smallest scale)
  const int code = bad ? 255 : max((int)(most >> 23) - 2, 0);
  const float inv = __uint_as_float((uint32_t)(254 - min(code, 253)) << 23);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = mul_keep(v[j], inv);   // no matter which in a block that is not a number
  word = in ? (uint32_t)code << (8 * (part >> 2)) : 0u;
  word |= __shfl_xor_sync(0xffffffffu, word, 4);
  word |= __shfl_xor_sync(0xffffffffu, word, 8);
  return pack8(v);
}

// VEC: rows start at multiples of 16 bytes and have a multiple of eight values.  ALONG: a CTA has eight words of a row (shift 3) and a thread goes along one
// row instead of down one column (bf16 32768 x 8192: 120 instead of 134 us).
template <int ITERS, bool VEC, bool ALONG, class T>
__global__ void __launch_bounds__(QTHREADS, !VEC ? 1 : sizeof(T) == 4 ? 4 : 6) quantize_kernel(QuantArgs a) {
  // Behind the wait: the product that follows reads its other operand without one of its own, and that may come from the kernel before this
  after_previous();
  let_next_begin();
  using U = Units<ITERS>;
  __shared__ uint32_t words[U::COUNT];
  const U u(a.words, a.shift);
  const int row_words = (a.K + 31) / 32 * 4;           // 4-byte words of a row of data
  const int part = threadIdx.x & 15, step = ALONG ? 0 : u.step();
  const int c = (ALONG ? u.word0 + (int)(threadIdx.x >> 4 & 1) : u.word()) * 128 + part * 8;
  const long long r = ALONG ? u.r0 + (threadIdx.x >> 5) : u.row();
  const int left = ALONG ? (r < a.rows ? 1 : 0) : (int)min(a.rows - r, (long long)U::COUNT);
  auto valid = [&](int i) { return i * step < left && (ALONG ? c + i * 256 < a.K : !VEC || c < a.K); };
  const T* src = static_cast<const T*>(a.x) + r * a.ldx + c;
  const long long src_step = ALONG ? 256 : (long long)step * a.ldx;
  constexpr int PER = sizeof(T) / 2;                   // 16-byte loads of eight values
  uint4 raw[ITERS][PER];
  if (VEC || (a.vec && c + 8 <= a.K)) {
#pragma unroll
    for (int i = 0; i < ITERS; ++i)
#pragma unroll
      for (int q = 0; q < PER; ++q)
        raw[i][q] = valid(i) ? __ldcs(reinterpret_cast<const uint4*>(src + i * src_step) + q) : make_uint4(0, 0, 0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      T v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = i * step < left && c + j < a.K ? src[i * src_step + j] : to_out<T>(0.f);
      memcpy(raw[i], v, sizeof(v));
    }
  }
  uint32_t* dst = a.data + r * row_words + (c >> 3);
  const long long dst_step = ALONG ? 32 : (long long)step * row_words;
  const int slot = ((c / 128 - u.word0) << (U::LOG - u.shift)) + (int)(r - u.r0), slot_step = ALONG ? 16 : step;
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    T t[8];
    memcpy(t, raw[i], sizeof(t));
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32(t[j]);
    const bool in = c + (ALONG ? i * 256 : 0) < row_words * 8;
    uint32_t w;
    const uint32_t codes = encode8(v, top_bits<T>(raw[i]), in, part, w);
    if (in && i * step < left) dst[i * dst_step] = codes;
    if (part == 0) words[slot + i * slot_step] = w;
  }
  __syncthreads();
  const int rows = U::COUNT >> u.shift, word = u.word0 + (int)threadIdx.x / rows;
  const long long row = u.r0 + (threadIdx.x & (rows - 1));
  if (threadIdx.x < U::COUNT && word < a.words && row < a.rows) a.scales[(long long)word * a.rows + row] = words[threadIdx.x];
}

struct DequantArgs {
  const uint32_t* data;
  const uint32_t* scales;
  void* out;
  long long ldo, rows;
  int K, words, vec, shift;
};

template <int ITERS, class T>
__global__ void __launch_bounds__(QTHREADS) dequantize_kernel(DequantArgs a) {
  const Units<ITERS> u(a.words, a.shift);
  const int row_words = (a.K + 31) / 32 * 4;
  const int part = threadIdx.x & 15, c = u.word() * 128 + part * 8, step = u.step();
  const long long r = u.row();
  if (c >= a.K) return;
  const int left = (int)min(a.rows - r, (long long)(16 * ITERS));
  const uint32_t* src = a.data + r * row_words + (c >> 3);
  const uint32_t* scales = a.scales + (long long)u.word() * a.rows + r;
  uint32_t codes[ITERS], scale[ITERS];
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    codes[i] = i * step < left ? __ldcs(src + (long long)(i * step) * row_words) : 0u;
    scale[i] = i * step < left ? scales[i * step] : 0u;
  }
  T* dst = static_cast<T*>(a.out) + r * a.ldo + c;
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    if (i * step >= left) break;
    const float s = scale_value((scale[i] >> (8 * (part >> 2))) & 255u);
    float f[8];
    unpack8(codes[i], f);
    T v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_out<T>(mul_keep(f[j], s));
    if (sizeof(T) == 2 && a.vec && c + 8 <= a.K) {
      uint4 raw;
      memcpy(&raw, v, 16);
      __stcs(reinterpret_cast<uint4*>(dst), raw);
    } else if (sizeof(T) == 4 && a.vec && (c & ~15) + 16 <= a.K) {
      // two lanes have 64 bytes: they change halves, so that each of their two stores is a whole sector (195 instead of 261 us for 32768 x 8192)
      const bool odd = part & 1;
      uint4 lo, hi, other;
      memcpy(&lo, v, 16);
      memcpy(&hi, reinterpret_cast<const char*>(v) + 16, 16);
      const uint4 give = odd ? lo : hi;
      const unsigned pair = 3u << (threadIdx.x & 30);
      other.x = __shfl_xor_sync(pair, give.x, 1);
      other.y = __shfl_xor_sync(pair, give.y, 1);
      other.z = __shfl_xor_sync(pair, give.z, 1);
      other.w = __shfl_xor_sync(pair, give.w, 1);
      __stcs(reinterpret_cast<uint4*>(dst - (odd ? 4 : 0)), odd ? other : lo);
      __stcs(reinterpret_cast<uint4*>(dst + (odd ? 4 : 8)), odd ? hi : other);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < a.K) dst[j] = v[j];
    }
    dst += (long long)step * a.ldo;
  }
}

// ------------------------------------------------------------------------------------------ products
//
// D[m, j] = sum_r P[m, r] Q[j, r] (tiles_sm100.cuh) with P = the rows of B, Q = those of A, by tcgen05.mma kind::mxf4: 64
// values a step, exact products of the four-bit values, scaled by the two blocks' scales, fp32 sums.
//
// The instruction takes the scales from tensor memory, for 128 rows in 32 lanes x 4 columns (row r in lane r mod 32, column r / 32), a word of four
// codes for 128 values of a row; four copies of it stand in the four quarters of the lanes.  A stage of 256 values has two
// such words of every row.  Three warps fetch them (a word of neighbouring rows is one line), one for P, two for Q, put them
// into shared memory in that order, and tcgen05.cp spreads them, behind the operands' arrival and ahead of the products.
//
// Every stage has 24 columns of tensor memory for its scales, which are free when the stage is; two accumulators of at most 208 columns and
// four stages fill the 512.  (224 columns and scales for two stages: a stage's copy then waits for the products of the stage before the last,
// and 1000 cycles go by per stage, 270 us for 8192^3.)
// Roles in a CTA: warp 0 loads operands, warp 1 issues products, warps 2-9 store, warps 10-12 fetch scales.
//
// Measured, in streams of calls: 8192^3 of packed matrices in 261 to 269 us = 4.1 to 4.2 PFLOP/s (nominal peak 9), 32 groups of together 16384 rows x 4096 x 2048 in 100 to 103 us,
// with A from bf16, its quantisation included, 311 to 328 and 120 to 125; one row from bf16 against 8192 x 4096 8.5 to 8.9 us.  Bound by the tensor pipe: a stage takes 600 cycles of it, 416 for the products of 208 columns and 30 for each of the six
// copies of scales; by the bytes that an SM takes in (45 KB a stage) where a reduction is short; by latency, about 4 us, for the smallest.  Pairs of
// CTAs, which load less, took 283 us: the leader has to be told of the other's scales.
constexpr int LANES = 128;
constexpr int BR = 256;                        // values of a row in a stage: 128 bytes
constexpr int P_BYTES = LANES * 128;
constexpr int SCALE_COLS = 24;
constexpr int TMEM_COLS = 512;
constexpr int MAX_STAGES = 7;
constexpr int EPI_WARPS = 8;
constexpr int SCALE_WARP = 2 + EPI_WARPS;
constexpr int THREADS = 32 * (SCALE_WARP + 3);

// Rows of A that a load brings where a tile has not all that fit: up to three times a quarter of them, in whole groups of eight
constexpr int small_box(int cols) { return (cols / 4 + 7) / 8 * 8; }

// COLS: columns of an accumulator, the most rows of A in a tile.  64 of them leave room for seven stages of 27 KB, 128 for five of 35, 208 for four of 45.
// SPLIT: a cluster shares a tile's reduction (COLS 64 only)
// FUSED: A comes as bf16, fp16 or fp32, and a CTA quantises the rows of its one tile into shared memory, where they stay; stages hold P alone (COLS 64 only)
template <int COLS, bool SPLIT, bool FUSED>
struct Form {
  static constexpr int STAGE_BYTES = P_BYTES + (FUSED ? 0 : COLS * 128);
  static constexpr int SCALE_BYTES = (FUSED ? 1 : 3) * 1024;   // P, Q rows 0-127, Q rows 128-255: two blocks of 512 bytes each
  static constexpr int SMALL_BOX = small_box(COLS);
  static constexpr int STAGES = FUSED ? 6 : (192 * 1024 - (SPLIT ? inbox_bytes(64) : 0)) / (STAGE_BYTES + SCALE_BYTES);
  static constexpr int SMEM_BYTES = 1024 + STAGES * (STAGE_BYTES + SCALE_BYTES) + EPI_WARPS * PIECE_BYTES + (SPLIT ? inbox_bytes(64) : 0);   // and Shared
  static_assert(STAGES <= MAX_STAGES, "barriers");
  static_assert(2 * COLS + STAGES * SCALE_COLS <= TMEM_COLS, "accumulators and scales share the tensor memory");
  static_assert(COLS % 16 == 0, "a chunk rounded up to the product's columns fits an accumulator, and none is left empty");
};
constexpr int FEW_COLS = 64, SOME_COLS = 128, MANY_COLS = 208;
constexpr int FUSED_MOST = 44 * 1024;          // bytes of a tile's quantised rows that leave room for the rest
// Bytes of `rows` quantised rows over `steps` stages: 128 of values each, and a block of scales for either half
constexpr int fused_bytes(int rows, int steps) { return steps * (rows * 128 + 1024); }

struct Args {
  const uint32_t* sp;   // words of B's scales [words, groups * N]
  const uint32_t* sq;   // of A's [words, rows]
  void* out;
  long long ldo;
  Offsets off;
  int N, steps, words, blocks, fill;
  bool boxed;   // results leave through mapOut
  bool behind;  // the kernel before is the quantisation of A, and wrote nothing else that is read here
  // FUSED
  const void* x;
  long long ldx;
  int x_type, K, room, cap;   // room: bytes of shared memory for `cap` quantised rows
  bool x_vec;                 // rows of x can be read 16 bytes at a time
};

struct Shared {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES], tfull[2], tempty[2], quantized;
  uint32_t tmem;
  int abort_flag;
  Table table;
};


__device__ PclStatus g_status;

__global__ void take_kernel(PclStatus* to) { take(&g_status, to); }

// a block of 32 rows x 16 bytes without swizzle: eight rows are 128 bytes in one piece
__device__ __forceinline__ uint64_t desc_scales(uint32_t saddr) {
  return ((uint64_t)(8u | (1u << 14)) << 32) | ((saddr >> 4) & 0x3FFFu) | (8u << 16);
}

__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ void umma_mxf4(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
      : "memory");
}

struct Tile {
  int e, m0, j0, n, ncol;   // columns: n of them, ncol with those that the product rounds up to
  int k0, k1;               // stages
};

// The tiles of a call, numbered: those that share rows of A are neighbours.
template <bool SPLIT>
struct Walk {
  const Args& a;
  const Table& t;
  int mb, chunks;

  __device__ Walk(const Args& a_, const Table& t_) : a(a_), t(t_) {
    mb = (a.N + LANES - 1) / LANES;
    chunks = t.chunks[a.off.groups];
  }

  __device__ Counter start(int first, int step) const { return Counter(first, step, mb); }
  __device__ bool has(const Counter& i) const { return i.c < chunks; }

  __device__ Tile at(const Counter& i) const {
    Tile w;
    w.m0 = i.m * LANES;
    t.find(a.off.groups, i.c, 16, w.e, w.j0, w.n);
    w.k0 = 0;
    w.k1 = a.steps;
    if (SPLIT) {
      const int rank = (int)cluster_ctarank(), parts = (int)cluster_size();
      w.k0 = rank * a.steps / parts;
      w.k1 = (rank + 1) * a.steps / parts;
    }
    w.ncol = (w.n + 16 - 1) / (16) * (16);
    return w;
  }
};

// Eight values of a row, from column c on, zeros behind column K; and the bits of their largest magnitude
__device__ __forceinline__ void load8(const Args& a, long long r, int c, float (&v)[8]) {
  const int size = a.x_type == TYPE_F32 ? 4 : 2;
  const char* p = static_cast<const char*>(a.x) + (r * a.ldx + c) * size;
  if (a.x_vec && c + 8 <= a.K) {
    uint4 raw[2];
    raw[0] = *reinterpret_cast<const uint4*>(p);
    if (size == 4) {
      raw[1] = *(reinterpret_cast<const uint4*>(p) + 1);
      memcpy(v, raw, 32);
    } else {
      const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (a.x_type == TYPE_BF16) {
          v[2 * i] = __uint_as_float(w[i] << 16);
          v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(w + i));
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        }
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = 0.f;
    if (c + j < a.K) {
      if (size == 4) v[j] = reinterpret_cast<const float*>(p)[j];
      else if (a.x_type == TYPE_BF16) v[j] = to_f32(reinterpret_cast<const __nv_bfloat16*>(p)[j]);
      else v[j] = to_f32(reinterpret_cast<const __half*>(p)[j]);
    }
  }
}

// FUSED: the rows of the tile into `room`, by warp `w` of QUANT_WARPS: for every stage `cap` rows of 128 bytes, swizzled as an operand, behind them for every stage two
// blocks of scales.  Sixteen lanes take a word of scales, 128 values; two words of each lane are on their way together.
constexpr int QUANT_WARPS = EPI_WARPS + 2;
__device__ __forceinline__ void quantize_tile(const Args& a, const Tile& t, uint8_t* room, int w) {
  const int lane = threadIdx.x & 31, part = lane & 15;
  const int across = 2 * (t.k1 - t.k0), units = t.n * across, row_values = a.blocks * 32;
  uint8_t* scales = room + (t.k1 - t.k0) * a.cap * 128;
  constexpr int AHEAD = 2;
  for (int u0 = w * 2 + (lane >> 4); u0 - (lane >> 4) < units; u0 += 2 * QUANT_WARPS * AHEAD) {
    float v[AHEAD][8];
    int row[AHEAD], word[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int u = u0 + i * 2 * QUANT_WARPS;
      row[i] = u / across;
      word[i] = u - row[i] * across;
      if (u < units) {
        load8(a, (long long)t.j0 + row[i], (t.k0 * 2 + word[i]) * 128 + part * 8, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[i][j]) & 0x7fffffffu);
      const bool in = (t.k0 * 2 + word[i]) * 128 + part * 8 < row_values;
      uint32_t scale;
      const uint32_t codes = encode8(v[i], most, in, part, scale);
      if (u0 + i * 2 * QUANT_WARPS < units) {
        const int r = row[i], step = word[i] >> 1, half = word[i] & 1, chunk = half * 4 + (part >> 2);
        *reinterpret_cast<uint32_t*>(room + (step * a.cap + r) * 128 + ((chunk ^ (r & 7)) << 4) + (part & 3) * 4) = in ? codes : 0u;
        if (part == 0) *reinterpret_cast<uint32_t*>(scales + step * 1024 + half * 512 + (r & 31) * 16 + (r >> 5) * 4) = scale;
      }
    }
  }
}

template <int COLS, bool SPLIT, bool FUSED, class TO>
__global__ void __launch_bounds__(THREADS, 1)
product_kernel(const __grid_constant__ CUtensorMap mapP, const __grid_constant__ CUtensorMap mapQ,
               const __grid_constant__ CUtensorMap mapQ_small, const __grid_constant__ CUtensorMap mapOut, Args a) {
  using F = Form<COLS, SPLIT, FUSED>;
  constexpr int STAGES = F::STAGES, STAGE_BYTES = F::STAGE_BYTES, SCALE_BYTES = F::SCALE_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* room = stages + STAGES * STAGE_BYTES;                              // FUSED
  uint8_t* scales = room + (FUSED ? a.room : 0);
  uint8_t* pieces = scales + STAGES * SCALE_BYTES;
  float* inbox = reinterpret_cast<float*>(pieces + EPI_WARPS * PIECE_BYTES);   // SPLIT
  Shared& s = *reinterpret_cast<Shared*>(pieces + EPI_WARPS * PIECE_BYTES + (SPLIT ? inbox_bytes(64) : 0));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &s.abort_flag;

  if (warp == 0) {
    if (lane < STAGES) {
      mbar_init(s.full + lane, 1 + (FUSED ? 1 : 3) * 32);   // the loads, and every lane that copies scales
      mbar_init(s.empty + lane, 1);
    }
    if (lane < 2) { mbar_init(s.tfull + lane, 1); mbar_init(s.tempty + lane, EPI_WARPS); }
    if (lane == 0) { mbar_init(&s.quantized, QUANT_WARPS); s.abort_flag = 0; }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2 && lane == 0) {
    for (const CUtensorMap* m : {&mapP, &mapQ, &mapQ_small, &mapOut}) asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
  }
  let_next_begin();
  if (!a.behind) after_previous();
  load_bounds(a.off, s.table.bounds, &g_status);
  __syncthreads();
  if (warp == 0) s.table.build(a.off.groups, COLS, &g_status);
  if (warp == 1) tmem_alloc<1>(&s.tmem, TMEM_COLS);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  sync_cluster_or_block<SPLIT>();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = s.tmem;
  const int share = SPLIT ? (int)cluster_size() : 1;
  const int group = blockIdx.x / share, groups = gridDim.x / share;
  const Walk<SPLIT> walk(a, s.table);
  using Turn = Tiles<Walk<SPLIT>, SPLIT || FUSED>;
  bool ok = true;
  auto gave_up = [&](int where, int x, int y) {
    if (lane == 0) post(&g_status, CODE_WAIT, where, x, y);
    *abort_flag = 1;
    ok = false;
  };
  if (FUSED && warp >= 2 && warp != SCALE_WARP && walk.has(walk.start(group, groups))) {
    quantize_tile(a, walk.at(walk.start(group, groups)), room, warp < SCALE_WARP ? warp - 2 : warp - 3);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&s.quantized)) : "memory");
  }

  if (warp == 0) {
    after_previous();   // A may still be being quantised
    int stage = 0;
    uint32_t phase = 0;
    for (Turn i(walk, group, groups); i.has() && ok; i.next()) {
      const Tile w = i.tile();
      constexpr int SMALL_BOX = F::SMALL_BOX;
      const bool whole = w.ncol > 3 * SMALL_BOX;
      const int boxes = whole ? 1 : (w.ncol + SMALL_BOX - 1) / SMALL_BOX;
      const uint32_t bytes = P_BYTES + (FUSED ? 0 : whole ? COLS * 128 : boxes * SMALL_BOX * 128);
      for (int kb = w.k0; kb < w.k1; ++kb) {
        if (!mbar_wait(s.empty + stage, phase ^ 1, abort_flag)) { gave_up(41, kb, stage); break; }
        if (elect()) {
          const uint32_t sp = smem_u32(stages + stage * STAGE_BYTES), sq = sp + P_BYTES;
          const uint32_t bar = smem_u32(s.full + stage);
          mbar_expect_tx(s.full + stage, bytes);
          tma_load_3d<1>(sp, &mapP, bar, kb * 128, w.m0, w.e);
          if (FUSED) {
          } else if (whole) {
            tma_load_3d<1>(sq, &mapQ, bar, kb * 128, w.j0, 0);
          } else {
            for (int b = 0; b < boxes; ++b)
              tma_load_3d<1>(sq + b * SMALL_BOX * 128, &mapQ_small, bar, kb * 128, w.j0 + b * SMALL_BOX, 0);
          }
        }
        __syncwarp();
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
    }
    if (!ok)
      for (int i = 0; i < 2048; ++i) __nanosleep(1000);   // copies in flight land before the shared memory goes away
  } else if (warp == 1) {
    // operands E2M1, scales E8M0
    const uint32_t idesc0 = (1u << 7) | (1u << 10) | (1u << 23) | ((uint32_t)(LANES >> 4) << 24);
    const uint64_t dp0 = desc_k_major(smem_u32(stages)), ds0 = desc_scales(smem_u32(scales));
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;   // bit i of acc_phase: accumulator i
    bool ready = false;                  // the next stage has arrived
    for (Turn i(walk, group, groups); i.has() && ok; i.next()) {
      const Tile w = i.tile();
      if (!mbar_wait(s.tempty + acc, (acc_phase >> acc & 1u) ^ 1u, abort_flag)) { gave_up(42, acc, 0); break; }
      acc_phase ^= 1u << acc;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t idesc = idesc0 | ((uint32_t)(w.ncol >> 3) << 17);
      const uint32_t d = tmem + (uint32_t)(acc * COLS);
      const bool wide = w.ncol > 128;
      if (FUSED && !mbar_wait(&s.quantized, 0, abort_flag)) { gave_up(49, 0, 0); break; }   // a CTA has one tile
      for (int kb = w.k0; kb < w.k1; ++kb) {
        if (!ready && !mbar_wait(s.full + stage, phase, abort_flag)) { gave_up(43, kb, stage); break; }
        const int next = stage + 1 == STAGES ? 0 : stage + 1;
        ready = has_passed(s.full + next, phase ^ (uint32_t)(next == 0));
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (elect()) {
          // the scales were copied for other threads, and have arrived
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          const uint32_t sf = tmem + (uint32_t)(2 * COLS + stage * SCALE_COLS);
          const uint64_t ds = ds0 + (uint32_t)(stage * SCALE_BYTES) / 16;
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            copy_scales(sf + v * 4, ds + v * 32);
            copy_scales(sf + 8 + v * 8, FUSED ? desc_scales(smem_u32(room)) + (uint32_t)((w.k1 - w.k0) * a.cap * 128 + (kb - w.k0) * 1024) / 16 + v * 32 : ds + 64 + v * 32);
            if (wide) copy_scales(sf + 12 + v * 8, ds + 128 + v * 32);
          }
          const uint64_t dp = dp0 + (uint32_t)(stage * STAGE_BYTES) / 16;
          const uint64_t dq = FUSED ? desc_k_major(smem_u32(room)) + (uint32_t)((kb - w.k0) * a.cap * 128) / 16 : dp + P_BYTES / 16;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t id = (uint32_t)(k & 1) * 2;   // codes 0, 1 or 2, 3 of a word
            umma_mxf4(d, dp + 2 * k, dq + 2 * k, idesc | (id << 4) | (id << 29), sf + (k >> 1) * 4, sf + 8 + (k >> 1) * 8,
                          (kb > w.k0 || k > 0) ? 1u : 0u);
          }
          commit<1>(smem_u32(s.empty + stage));
          if (kb + 1 == w.k1) commit<1>(smem_u32(s.tfull + acc));
        }
        __syncwarp();
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
      acc ^= 1;
    }
  } else if (warp >= SCALE_WARP && (!FUSED || warp == SCALE_WARP)) {
    const int part = warp - SCALE_WARP;      // 0: P, 1 and 2: Q
    if (part > 0) after_previous();
    const long long rows = part == 0 ? (long long)a.off.groups * a.N : a.off.rows;
    const uint8_t* src = reinterpret_cast<const uint8_t*>(part == 0 ? a.sp : a.sq);
    // Of 128 rows a lane copies 8 q + lane mod 8 + 32 (lane / 8), q = 0 .. 3: together the lanes read whole sectors and write
    // different banks.  (Words that went through registers took 73 of 311 thousand cycles of 4096 x 8192^2, more the further ahead they were
    // read: the copies are neither waited for nor unrolled.)
    const int row = (lane & 7) + 32 * (lane >> 3);
    const uint32_t dst0 = smem_u32(scales) + part * 1024 + (lane & 7) * 16 + (lane >> 3) * 4;
    const int last_bytes = 4 - (a.words * 4 - a.blocks);   // codes of the last word; those that no block has become zero
    int stage = 0;
    uint32_t phase = 0;
    for (Turn i(walk, group, groups); i.has() && ok; i.next()) {
      const Tile w = i.tile();
      const bool used = part < 2 || w.ncol > 128;
      const long long r0 = part == 0 ? (long long)w.e * a.N + w.m0 : (long long)w.j0 + (part - 1) * 128;
      const uint8_t* at[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) at[q] = src + 4 * min(r0 + row + 8 * q, rows - 1);   // rows of no tile: any scales do
      for (int kb = w.k0; kb < w.k1; ++kb) {
        if (!mbar_wait(s.empty + stage, phase ^ 1, abort_flag)) { gave_up(48, kb, stage); break; }
        if (used) {
          const uint32_t dst = dst0 + stage * SCALE_BYTES;
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const int word = kb * 2 + v;
            const int bytes = word + 1 < a.words ? 4 : word + 1 == a.words ? last_bytes : 0;
            const long long off = word < a.words ? word * rows * 4 : 0;
#pragma unroll
            for (int q = 0; q < 4; ++q)
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + v * 512 + q * 128), "l"(at[q] + off), "r"(bytes) : "memory");
          }
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(s.full + stage)) : "memory");
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp < SCALE_WARP) {
    const int sub = warp & 3;                 // the quarter of the tensor memory's lanes that this warp can read
    const int half = (warp - 2) >> 2;         // two warps share a quarter: 32 columns in turn
    TO* out = static_cast<TO*>(a.out);
    int acc = 0;
    uint32_t acc_phase = 0;                   // bit i: accumulator i
    for (Turn i(walk, group, groups); i.has() && ok; i.next()) {
      const Tile w = i.tile();
      if (!wait_full(s.tfull + acc, acc_phase >> acc & 1u, abort_flag, tile_ns(w.k1 - w.k0))) { gave_up(44, acc, 0); break; }
      acc_phase ^= 1u << acc;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int m = w.m0 + sub * 32;
      TO* dst = out + (long long)w.j0 * a.ldo + m;
      const uint32_t t0 = tmem + ((uint32_t)(sub * 32) << 16) + (uint32_t)(acc * COLS);
      if (SPLIT) {   // the cluster has this one tile
        send_columns(t0, sub, half * 32, w.n, inbox, cluster_ctarank(), columns_of_part(w.n, share));
        continue;
      }
      store_columns<TO>(t0, half * 32, w.n, dst, a.ldo, a.N - m, a.boxed, pieces + (warp - 2) * PIECE_BYTES, &mapOut, m, w.j0, 0);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(smem_u32(s.tempty + acc));
      acc ^= 1;
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // the copy engine has read and written all boxes
    if (a.fill) {
      const int first = s.table.bounds[0], last = s.table.bounds[a.off.groups];
      const int rows = first + (a.off.rows - last);
      for (long long q = (long long)blockIdx.x * EPI_WARPS + warp - 2; q < rows; q += (long long)gridDim.x * EPI_WARPS) {
        TO* row = out + (q < first ? q : q - first + last) * a.ldo;
        for (int c = lane; c < a.N; c += 32) row[c] = to_out<TO>(0.f);
      }
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncwarp();
  sync_cluster_or_block<SPLIT>();   // the parts of a split tile are in their inboxes
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem_free<1>(tmem, TMEM_COLS);
  }
  if (SPLIT && warp >= 2 && warp < SCALE_WARP && walk.has(walk.start(group, groups))) {
    const Tile w = walk.at(walk.start(group, groups));
    add_up<TO>(inbox, w.n, columns_of_part(w.n, share), cluster_ctarank(), share, 64, 32 * EPI_WARPS, static_cast<TO*>(a.out) + (long long)w.j0 * a.ldo + w.m0,
               a.ldo, a.N - w.m0);
  }
}

template <int COLS, bool SPLIT, bool FUSED, class TO>
int launch(const CUtensorMap& p, const CUtensorMap& q, const CUtensorMap& qs, const CUtensorMap& o, const Args& a, int parts, cudaStream_t stream) {
  auto kernel = product_kernel<COLS, SPLIT, FUSED, TO>;
  constexpr int fixed = Form<COLS, SPLIT, FUSED>::SMEM_BYTES + (int)sizeof(Shared);
  // The limit belongs to the function, not to the launch: it is the same in every call, since another thread's call may come between the two
  constexpr int limit = fixed + (FUSED ? FUSED_MOST : 0);
  static_assert(limit <= 227 * 1024, "shared memory of an SM");
  const int smem = fixed + (FUSED ? a.room : 0);
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, limit);
  if (e != cudaSuccess) return (int)e;
  const long long mb = (a.N + LANES - 1) / LANES;
  const long long chunks = most_chunks(a.off.rows, a.off.groups, COLS);
  // a cluster that shares a tile has no other, nor has a CTA that quantises its rows
  const unsigned grid = SPLIT ? (unsigned)(chunks * mb) * parts : FUSED ? (unsigned)(chunks * mb) : (unsigned)min((long long)sms, chunks * mb);
  const Launch l(grid, THREADS, smem, parts, stream);
  e = cudaLaunchKernelEx(&l.cfg, kernel, p, q, qs, o, a);
  return e != cudaSuccess ? (int)e : pcl_last_error();
}

template <int COLS, bool SPLIT, bool FUSED>
int launch_as(int out_type, const CUtensorMap& p, const CUtensorMap& q, const CUtensorMap& qs, const CUtensorMap& o, const Args& a, int parts,
              cudaStream_t stream) {
  if (out_type == TYPE_F32) return launch<COLS, SPLIT, FUSED, float>(p, q, qs, o, a, parts, stream);
  if (out_type == TYPE_BF16) return launch<COLS, SPLIT, FUSED, __nv_bfloat16>(p, q, qs, o, a, parts, stream);
  return launch<COLS, SPLIT, FUSED, __half>(p, q, qs, o, a, parts, stream);
}

// CTAs of the grid, how long their rows are, and whether they go over four words a thread: where that leaves every SM four of them
bool blocks_of(long long rows, int words, long long* n, int* shift, bool* four) {
  for (const int iters : {4, 1}) {
    *shift = 0;
    while ((1 << *shift) < words && *shift < (iters == 4 ? 3 : 1)) ++*shift;
    const int down = 16 * iters >> *shift;
    *n = (rows + down - 1) / down * ((words + (1 << *shift) - 1) >> *shift);
    *four = iters == 4;
    if (*n >= 4 * SMS) break;
  }
  return *n < (1ll << 31);
}

template <class T>
int launch_quantize(unsigned n, bool four, const QuantArgs& a, cudaStream_t stream) {
  const Launch l(n, QTHREADS, 0, 1, stream);
  const bool vec = a.vec && a.K % 8 == 0;
  auto kernel = vec ? (four ? (a.shift == 3 ? quantize_kernel<4, true, true, T> : quantize_kernel<4, true, false, T>) : quantize_kernel<1, true, false, T>)
                    : (four ? quantize_kernel<4, false, false, T> : quantize_kernel<1, false, false, T>);
  return (int)cudaLaunchKernelEx(&l.cfg, kernel, a);
}

template <class T>
void launch_dequantize(unsigned n, bool four, const DequantArgs& a, cudaStream_t stream) {
  if (four) dequantize_kernel<4, T><<<n, QTHREADS, 0, stream>>>(a);
  else dequantize_kernel<1, T><<<n, QTHREADS, 0, stream>>>(a);
}

}  // namespace

static int quantize(const void* x, long long ldx, int in_type, void* data, void* scales, long long rows, int K, cudaStream_t stream) {
  QuantArgs a{x, ldx, static_cast<uint32_t*>(data), static_cast<uint32_t*>(scales), rows, K, (K + 127) / 128, 0, 0};
  const int size = in_type == TYPE_F32 ? 4 : 2;
  a.vec = ((uintptr_t)x & 15) == 0 && (ldx * size & 15) == 0;
  long long n;
  bool four;
  if (rows < 0 || K < 1 || in_type < 0 || in_type > 2 || !blocks_of(rows, a.words, &n, &a.shift, &four)) return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  const int rc = in_type == TYPE_F32    ? launch_quantize<float>((unsigned)n, four, a, stream)
                 : in_type == TYPE_BF16 ? launch_quantize<__nv_bfloat16>((unsigned)n, four, a, stream)
                                        : launch_quantize<__half>((unsigned)n, four, a, stream);
  return rc ? rc : pcl_last_error();
}

// x [rows, K] of in_type (0 fp32, 1 bf16, 2 fp16), rows ldx values apart
PCL_API int pcl_mx4_quantize(const void* x, long long ldx, int in_type, void* data, void* scales, long long rows, int K,
                             cudaStream_t stream) {
  return quantize(x, ldx, in_type, data, scales, rows, K, stream);
}

PCL_API int pcl_mx4_dequantize(const void* data, const void* scales, void* out, long long ldo, int out_type, long long rows,
                               int K, cudaStream_t stream) {
  DequantArgs a{static_cast<const uint32_t*>(data), static_cast<const uint32_t*>(scales), out, ldo, rows, K, (K + 127) / 128, 0, 0};
  const int size = out_type == TYPE_F32 ? 4 : 2;
  a.vec = ((uintptr_t)out & 15) == 0 && (ldo * size & 15) == 0;
  long long n;
  bool four;
  if (rows < 0 || K < 1 || out_type < 0 || out_type > 2 || !blocks_of(rows, a.words, &n, &a.shift, &four)) return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  if (out_type == TYPE_F32) launch_dequantize<float>((unsigned)n, four, a, stream);
  else if (out_type == TYPE_BF16) launch_dequantize<__nv_bfloat16>((unsigned)n, four, a, stream);
  else launch_dequantize<__half>((unsigned)n, four, a, stream);
  return pcl_last_error();
}

struct Plan {
  int cols, parts, cap, room;
  bool fused;
};

// Tiles of the number of rows that takes the shortest time; and whether A, of x_type, is quantised by the product's own CTAs: where each has one tile at most, and the words
// of its rows go through its warps in one pass (QUANT_WARPS * 4 of them).  One row against 8192 x 4096 takes 8.5 us so, 9.6 with a kernel for the quantisation,
// most of it the second launch; 64 rows of 8 words a CTA 20 us, and 8.
static Plan plan_of(int x_type, long long rows, int groups, int N, int K) {
  Plan plan{0, 1, 0, 0, false};
  const int steps = (K + 255) / 256;
  long long least = 0;
  for (const int c : {FEW_COLS, SOME_COLS, MANY_COLS}) {
    const long long t = tiles_cost(likely_chunks(rows, groups, c), c, N, steps);
    if (plan.cols == 0 || t < least) { plan.cols = c; least = t; }
  }
  if (plan.cols != FEW_COLS) return plan;
  const long long tiles = most_chunks(rows, groups, FEW_COLS) * ((N + LANES - 1) / LANES);
  plan.parts = parts_of(tiles, steps);
  const int own = (steps + plan.parts - 1) / plan.parts;
  plan.cap = (int)(rows < FEW_COLS ? (rows + 15) / 16 * 16 : FEW_COLS);
  plan.fused = x_type >= 0 && tiles * plan.parts <= SMS && 2 * own * min(rows, (long long)FEW_COLS) <= 4 * QUANT_WARPS && fused_bytes(plan.cap, own) <= FUSED_MOST;
  plan.room = plan.fused ? fused_bytes(plan.cap, own) : 0;
  return plan;
}

// Bytes that A and its scales have to have room for in a call with an x of x_type
PCL_API long long pcl_mx4_room(int x_type, long long rows, int groups, int N, int K) {
  if (rows < 1 || groups < 1 || N < 1 || K < 1 || plan_of(x_type, rows, groups, N, K).fused) return 0;
  return rows * ((K + 31) / 32 * 16ll + (K + 127) / 128 * 4ll);
}

// A [rows, K], B [groups * N, K], both in four bits -> out [rows, N] of out_type; offsets null: one group of all rows.  x_type 0, 1, 2: A and
// sa are room for x [rows, K] (fp32, bf16, fp16, rows ldx values apart), which is quantised into them first; -1: they are the operand.
PCL_API int pcl_mx4_rows(const void* x, long long ldx, int x_type, void* A, void* sa, const void* B, const void* sb, const void* offsets,
                         int off64, void* out, long long ldo, int out_type, long long rows, int groups, int N, int K, int fill,
                         cudaStream_t stream) {
  if (rows < 0 || rows >= (1ll << 31) - 512 || groups < 1 || groups > MAX_GROUPS || N < 1 || K < 1 ||
      (long long)groups * N >= (1ll << 31) - 512)
    return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  if (out_type < 0 || out_type > 2) return (int)cudaErrorInvalidValue;
  const long long row_bytes = (K + 31) / 32 * 16;
  const Plan plan = plan_of(x_type, rows, groups, N, K);
  const int cols = plan.cols;
  if (x_type >= 0 && !plan.fused) {
    const int rc = quantize(x, ldx, x_type, A, sa, rows, K, stream);
    if (rc) return rc;
  }
  CUtensorMap p, q, qs, o;
  const CUtensorMapDataType t = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  int rc = make_map_3d(&p, t, B, row_bytes, N, groups, row_bytes, row_bytes * N, 128, LANES);
  if (plan.fused) q = qs = p;   // not used
  else if (rc == 0) rc = make_map_3d(&q, t, A, row_bytes, rows, 1, row_bytes, row_bytes, 128, cols);
  if (rc == 0 && !plan.fused) rc = make_map_3d(&qs, t, A, row_bytes, rows, 1, row_bytes, row_bytes, 128, small_box(cols));
  if (rc) return rc;
  Args a{static_cast<const uint32_t*>(sb), static_cast<const uint32_t*>(sa), out, ldo, Offsets{offsets, off64, groups, (int)rows},
         N, (int)((row_bytes + 127) / 128), (K + 127) / 128, (K + 31) / 32, fill, false, x_type >= 0 && !plan.fused,
         x, ldx, x_type, K, plan.room, plan.cap, ((uintptr_t)x & 15) == 0 && (ldx * (x_type == TYPE_F32 ? 4 : 2) & 15) == 0};
  a.boxed = make_out_map(&o, p, out_type, out, N, rows, 1, ldo, ldo);
  if (cols == SOME_COLS) return launch_as<SOME_COLS, false, false>(out_type, p, q, qs, o, a, 1, stream);
  if (cols == MANY_COLS) return launch_as<MANY_COLS, false, false>(out_type, p, q, qs, o, a, 1, stream);
  if (plan.fused)
    return plan.parts > 1 ? launch_as<FEW_COLS, true, true>(out_type, p, q, qs, o, a, plan.parts, stream) : launch_as<FEW_COLS, false, true>(out_type, p, q, qs, o, a, 1, stream);
  return plan.parts > 1 ? launch_as<FEW_COLS, true, false>(out_type, p, q, qs, o, a, plan.parts, stream) : launch_as<FEW_COLS, false, false>(out_type, p, q, qs, o, a, 1, stream);
}

// Moves the report that the status block of these products holds, if any, to `to` in the device's memory, behind what the stream has so far.
PCL_API int pcl_mx4_status(PclStatus* to, cudaStream_t stream) {
  take_kernel<<<1, 1, 0, stream>>>(to);
  return pcl_last_error();
}
