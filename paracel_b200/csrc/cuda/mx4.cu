// Matrices in four bits with a shared scale for every 32 values of a row (OCP microscaling format, elements E2M1, scales
// E8M0): quantisation, its reverse, and the product of two of them, also with one right-hand matrix for each group of rows.
//
// Layout, `rows` x K: data [rows, 16 ceil(K / 32)] bytes, value 2 j of a row in the low half of byte j, 2 j + 1 in the high
// half; scales [ceil(K / 128), rows] words of four codes, byte i of word (b, r) is the code of row r's block 4 b + i.
// A word holds the scales of 128 values, and the words of neighbouring rows are neighbours: a tile of rows finds its
// scales in one piece wherever it begins.  A code c stands for 2^(c - 127), 255 for NaN.
#include "grouped.cuh"

namespace {

using namespace pcl_group;

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

// value of a four-bit code: codes 0 and 1 are 0 and 1/2, above them (2 + mantissa) / 2 * 2^(exponent - 1)
__device__ __forceinline__ float code_value(uint32_t c) {
  const uint32_t m = c & 7u;
  const float v = m < 2u ? 0.5f * (float)m : __uint_as_float((m << 22) + (126u << 23));
  return (c & 8u) ? -v : v;
}

struct QuantArgs {
  const void* x;
  long long ldx;
  uint32_t* data;      // 4 bytes = 8 values
  uint32_t* scales;
  long long rows;
  int K, words;        // words: ceil(K / 128)
  int vec;             // rows of x can be read 16 bytes at a time
};

// A thread takes eight neighbouring values of a row; four lanes make a block of 32, sixteen a word of scales.  A block of
// the grid takes 128 columns of QROWS rows and stores its words of scales side by side.
constexpr int QROWS = 32, QTHREADS = 256;

template <class T>
__global__ void __launch_bounds__(QTHREADS) quantize_kernel(QuantArgs a) {
  __shared__ uint32_t words[QROWS];
  const int word = blockIdx.x % a.words;
  const long long r0 = (long long)(blockIdx.x / a.words) * QROWS;
  const int lane = threadIdx.x & 31, part = threadIdx.x & 15;
  const int c0 = word * 128 + part * 8;
  const int row_bytes4 = (a.K + 31) / 32 * 4;          // 4-byte words of a row of data
#pragma unroll
  for (int i = 0; i < QROWS * 16 / QTHREADS; ++i) {
    const int lr = i * (QTHREADS / 16) + (threadIdx.x >> 4);
    const long long r = r0 + lr;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (r < a.rows && c0 < a.K) {
      const T* src = static_cast<const T*>(a.x) + r * a.ldx + c0;
      if (a.vec && c0 + 8 <= a.K) {
        uint4 raw[sizeof(T) / 2];
#pragma unroll
        for (int q = 0; q < (int)(sizeof(T) / 2); ++q) raw[q] = reinterpret_cast<const uint4*>(src)[q];
        const T* p = reinterpret_cast<const T*>(raw);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_f32(p[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c0 + j < a.K) v[j] = to_f32(src[j]);
      }
    }
    // the largest magnitude of the block, by its bits: NaN and infinity come out on top
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const bool bad = most >= 0x7f800000u;
    // floor(log2(most)) - 2, at least -127 (all that is below 2^-125 takes the smallest scale)
    const int code = bad ? 255 : max((int)(most >> 23) - 2, 0);
    const float inv = __uint_as_float((uint32_t)(254 - min(code, 253)) << 23);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = bad ? 0.f : mul_keep(v[j], inv);
    if (r < a.rows && c0 < row_bytes4 * 8) a.data[r * row_bytes4 + (c0 >> 3)] = pack8(v);
    uint32_t w = (c0 < row_bytes4 * 8) ? (uint32_t)code << (8 * (part >> 2)) : 0u;
    w |= __shfl_xor_sync(0xffffffffu, w, 4);
    w |= __shfl_xor_sync(0xffffffffu, w, 8);
    if (part == 0) words[lr] = w;
  }
  __syncthreads();
  (void)lane;
  if (threadIdx.x < QROWS && r0 + threadIdx.x < a.rows)
    a.scales[(long long)word * a.rows + r0 + threadIdx.x] = words[threadIdx.x];
}

struct DequantArgs {
  const uint32_t* data;
  const uint32_t* scales;
  void* out;
  long long ldo, rows;
  int K, words, vec;
};

template <class T>
__global__ void __launch_bounds__(QTHREADS) dequantize_kernel(DequantArgs a) {
  const int word = blockIdx.x % a.words;
  const long long r0 = (long long)(blockIdx.x / a.words) * QROWS;
  const int part = threadIdx.x & 15;
  const int c0 = word * 128 + part * 8;
  const int row_bytes4 = (a.K + 31) / 32 * 4;
#pragma unroll
  for (int i = 0; i < QROWS * 16 / QTHREADS; ++i) {
    const long long r = r0 + i * (QTHREADS / 16) + (threadIdx.x >> 4);
    if (r >= a.rows || c0 >= a.K) continue;
    const uint32_t codes = a.data[r * row_bytes4 + (c0 >> 3)];
    const float s = scale_value((a.scales[(long long)word * a.rows + r] >> (8 * (part >> 2))) & 255u);
    T* dst = static_cast<T*>(a.out) + r * a.ldo + c0;
    __align__(16) T v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_out<T>(mul_keep(code_value((codes >> (4 * j)) & 15u), s));
    if (a.vec && c0 + 8 <= a.K) {
#pragma unroll
      for (int q = 0; q < (int)(sizeof(T) / 2); ++q) reinterpret_cast<uint4*>(dst)[q] = reinterpret_cast<uint4*>(v)[q];
    } else {
      for (int j = 0; j < 8; ++j)
        if (c0 + j < a.K) dst[j] = v[j];
    }
  }
}

struct RowsArgs {
  const uint8_t* A;
  const uint32_t* sa;
  const uint8_t* B;
  const uint32_t* sb;
  void* out;
  long long ldo;
  Offsets off;
  int N, K, fill;
};

__device__ PclStatus g_status;

constexpr int T = 64, KB = 32, THREADS = 256;

__device__ __forceinline__ float value_at(const uint8_t* data, const uint32_t* scales, long long rows, int row_bytes, long long r, int k) {
  const uint32_t c = data[r * row_bytes + (k >> 1)] >> (4 * (k & 1));
  return mul_keep(code_value(c & 15u), scale_value((scales[(long long)(k >> 7) * rows + r] >> (8 * ((k >> 5) & 3))) & 255u));
}

template <class TO>
__global__ void __launch_bounds__(THREADS) rows_kernel(RowsArgs a) {
  __shared__ int bounds[MAX_GROUPS + 1];
  __shared__ float ps[KB][T], qs[KB][T];
  load_bounds(a.off, bounds, &g_status);
  __syncthreads();
  TO* out = static_cast<TO*>(a.out);
  const int across = (a.N + T - 1) / T;
  int tile = blockIdx.x / across, e = 0;
  for (; e < a.off.groups; ++e) {
    const int n = (bounds[e + 1] - bounds[e] + T - 1) / T;
    if (tile < n) break;
    tile -= n;
  }
  const int c0 = blockIdx.x % across * T;
  if (e == a.off.groups) {   // rows of no group
    if (!a.fill || tile != 0) return;
    for (long long r = threadIdx.x; r < a.off.rows; r += THREADS)
      if (r < bounds[0] || r >= bounds[a.off.groups])
        for (int c = c0; c < min(c0 + T, a.N); ++c) out[r * a.ldo + c] = to_out<TO>(0.f);
    return;
  }
  const int t0 = bounds[e] + tile * T, t1 = bounds[e + 1];
  const int row_bytes = (a.K + 31) / 32 * 16;
  const long long b_rows = (long long)a.off.groups * a.N;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < a.K; k0 += KB) {
    for (int i = threadIdx.x; i < KB * T; i += THREADS) {
      const int k = k0 + i % KB, m = i / KB;
      qs[i % KB][m] = (k < a.K && t0 + m < t1) ? value_at(a.A, a.sa, a.off.rows, row_bytes, t0 + m, k) : 0.f;
      ps[i % KB][m] = (k < a.K && c0 + m < a.N) ? value_at(a.B, a.sb, b_rows, row_bytes, (long long)e * a.N + c0 + m, k) : 0.f;
    }
    __syncthreads();
    const int tm = (threadIdx.x & 15) * 4, tj = (threadIdx.x >> 4) * 4;
#pragma unroll
    for (int r = 0; r < KB; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(ps[r][tm + i], qs[r][tj + j], acc[i][j]);
    __syncthreads();
  }
  const int tm = (threadIdx.x & 15) * 4, tj = (threadIdx.x >> 4) * 4;
  for (int j = 0; j < 4; ++j)
    for (int i = 0; i < 4; ++i)
      if (t0 + tj + j < t1 && c0 + tm + i < a.N) out[(long long)(t0 + tj + j) * a.ldo + c0 + tm + i] = to_out<TO>(acc[i][j]);
}

template <class TO>
int launch_rows(const RowsArgs& a, cudaStream_t stream) {
  const long long grid = ((a.off.rows + T - 1ll) / T + a.off.groups + 1) * ((a.N + T - 1ll) / T);
  if (grid >= (1ll << 31)) return (int)cudaErrorInvalidValue;
  rows_kernel<TO><<<(unsigned)grid, THREADS, 0, stream>>>(a);
  return pcl_last_error();
}

bool blocks_of(long long rows, int words, long long* n) {
  *n = (rows + QROWS - 1) / QROWS * words;
  return *n < (1ll << 31);
}

}  // namespace

// x [rows, K] of in_type (0 fp32, 1 bf16, 2 fp16), rows ldx values apart
PCL_API int pcl_mx4_quantize(const void* x, long long ldx, int in_type, void* data, void* scales, long long rows, int K,
                             cudaStream_t stream) {
  QuantArgs a{x, ldx, static_cast<uint32_t*>(data), static_cast<uint32_t*>(scales), rows, K, (K + 127) / 128, 0};
  const int size = in_type == TYPE_F32 ? 4 : 2;
  a.vec = ((uintptr_t)x & 15) == 0 && (ldx * size & 15) == 0;
  long long n;
  if (rows < 0 || K < 1 || in_type < 0 || in_type > 2 || !blocks_of(rows, a.words, &n)) return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  if (in_type == TYPE_F32) quantize_kernel<float><<<(unsigned)n, QTHREADS, 0, stream>>>(a);
  else if (in_type == TYPE_BF16) quantize_kernel<__nv_bfloat16><<<(unsigned)n, QTHREADS, 0, stream>>>(a);
  else quantize_kernel<__half><<<(unsigned)n, QTHREADS, 0, stream>>>(a);
  return pcl_last_error();
}

PCL_API int pcl_mx4_dequantize(const void* data, const void* scales, void* out, long long ldo, int out_type, long long rows,
                               int K, cudaStream_t stream) {
  DequantArgs a{static_cast<const uint32_t*>(data), static_cast<const uint32_t*>(scales), out, ldo, rows, K, (K + 127) / 128, 0};
  const int size = out_type == TYPE_F32 ? 4 : 2;
  a.vec = ((uintptr_t)out & 15) == 0 && (ldo * size & 15) == 0;
  long long n;
  if (rows < 0 || K < 1 || out_type < 0 || out_type > 2 || !blocks_of(rows, a.words, &n)) return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  if (out_type == TYPE_F32) dequantize_kernel<float><<<(unsigned)n, QTHREADS, 0, stream>>>(a);
  else if (out_type == TYPE_BF16) dequantize_kernel<__nv_bfloat16><<<(unsigned)n, QTHREADS, 0, stream>>>(a);
  else dequantize_kernel<__half><<<(unsigned)n, QTHREADS, 0, stream>>>(a);
  return pcl_last_error();
}

// A [rows, K], B [groups * N, K], both in four bits -> out [rows, N] of out_type; offsets null: one group of all rows
PCL_API int pcl_mx4_rows(const void* A, const void* sa, const void* B, const void* sb, const void* offsets, int off64, void* out,
                         long long ldo, int out_type, long long rows, int groups, int N, int K, int fill,
                         cudaStream_t stream) {
  if (rows < 0 || rows >= (1ll << 31) - 512 || groups < 1 || groups > MAX_GROUPS || N < 1 || K < 1 ||
      (long long)groups * N >= (1ll << 31) - 512)
    return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  RowsArgs a{static_cast<const uint8_t*>(A), static_cast<const uint32_t*>(sa), static_cast<const uint8_t*>(B),
             static_cast<const uint32_t*>(sb), out, ldo, Offsets{offsets, off64, groups, (int)rows}, N, K, fill};
  if (out_type == TYPE_F32) return launch_rows<float>(a, stream);
  if (out_type == TYPE_BF16) return launch_rows<__nv_bfloat16>(a, stream);
  if (out_type == TYPE_F16) return launch_rows<__half>(a, stream);
  return (int)cudaErrorInvalidValue;
}

// Copies the status block of these products to `host` and clears it (waits for the stream).
PCL_API int pcl_mx4_status(PclStatus* host, cudaStream_t stream) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(host, g_status, sizeof(PclStatus), 0, cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess || host->code == 0) return (int)e;
  const PclStatus none{};
  e = cudaMemcpyToSymbolAsync(g_status, &none, sizeof(none), 0, cudaMemcpyHostToDevice, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  return (int)e;
}
