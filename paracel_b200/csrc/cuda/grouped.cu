// Products with one matrix for each group of rows (16-bit storage, fp32 sums).
//
//   rows, nt   Y[t, n] = sum_k X[t, k] W[e, n, k]        t in group e
//   rows, nn   Z[t, k] = sum_n Y[t, n] W[e, n, k]
//   tn         D[e, n, k] = sum_{t in group e} Y[t, n] X[t, k]
//
// One 64 x 64 tile of the output per CTA, 4 x 4 of it per thread, the reduction 16 at a time through shared memory.
#include "grouped.cuh"

namespace {

using namespace pcl_group;

__device__ PclStatus g_status;

struct RowsArgs {
  const void* X;
  const void* W;
  void* out;
  long long ldx, ws_e, ws_n, ldo;
  Offsets off;
  int N, K, fill;
};

constexpr int T = 64, KB = 16, THREADS = 256;

// acc += P Q^T over one step: ps[r][m], qs[r][j]
__device__ __forceinline__ void step(const float (*ps)[T], const float (*qs)[T], float (&acc)[4][4]) {
  const int tm = (threadIdx.x & 15) * 4, tj = (threadIdx.x >> 4) * 4;
#pragma unroll
  for (int r = 0; r < KB; ++r) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(ps[r][tm + i], qs[r][tj + j], acc[i][j]);
  }
}

template <bool NN, class TI, class TO>
__global__ void __launch_bounds__(THREADS) rows_kernel(RowsArgs a) {
  __shared__ int bounds[MAX_GROUPS + 1];
  __shared__ float ps[KB][T], qs[KB][T];
  load_bounds(a.off, bounds, &g_status);
  __syncthreads();
  const int cols = NN ? a.K : a.N, red = NN ? a.N : a.K;
  TO* out = static_cast<TO*>(a.out);
  const int across = (cols + T - 1) / T;
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
        for (int c = c0; c < min(c0 + T, cols); ++c) out[r * a.ldo + c] = to_out<TO>(0.f);
    return;
  }
  const int t0 = bounds[e] + tile * T, t1 = bounds[e + 1];
  const TI* X = static_cast<const TI*>(a.X);
  const TI* W = static_cast<const TI*>(a.W) + (long long)e * a.ws_e;
  float acc[4][4] = {};
  for (int r0 = 0; r0 < red; r0 += KB) {
    for (int i = threadIdx.x; i < KB * T; i += THREADS) {
      const int r = r0 + i % KB, t = t0 + i / KB;
      qs[i % KB][i / KB] = (r < red && t < t1) ? to_f32(X[(long long)t * a.ldx + r]) : 0.f;
      const int wr = NN ? r0 + i / T : r, wc = NN ? c0 + i % T : c0 + i / KB;
      const float w = (wr < red && wc < cols) ? to_f32(NN ? W[(long long)wr * a.ws_n + wc] : W[(long long)wc * a.ws_n + wr]) : 0.f;
      if (NN) ps[i / T][i % T] = w;
      else ps[i % KB][i / KB] = w;
    }
    __syncthreads();
    step(ps, qs, acc);
    __syncthreads();
  }
  const int tm = (threadIdx.x & 15) * 4, tj = (threadIdx.x >> 4) * 4;
  for (int j = 0; j < 4; ++j)
    for (int i = 0; i < 4; ++i)
      if (t0 + tj + j < t1 && c0 + tm + i < cols) out[(long long)(t0 + tj + j) * a.ldo + c0 + tm + i] = to_out<TO>(acc[i][j]);
}

struct TnArgs {
  const void* Y;
  const void* X;
  void* out;
  long long ldy, ldx;
  Offsets off;
  int N, K;
};

template <class TI, class TO>
__global__ void __launch_bounds__(THREADS) tn_kernel(TnArgs a) {
  __shared__ int bounds[MAX_GROUPS + 1];
  __shared__ float ps[KB][T], qs[KB][T];
  load_bounds(a.off, bounds, &g_status);
  __syncthreads();
  const int e = blockIdx.z, k0 = blockIdx.x * T, n0 = blockIdx.y * T;
  const TI* X = static_cast<const TI*>(a.X);
  const TI* Y = static_cast<const TI*>(a.Y);
  float acc[4][4] = {};
  for (int t0 = bounds[e]; t0 < bounds[e + 1]; t0 += KB) {
    for (int i = threadIdx.x; i < KB * T; i += THREADS) {
      const int t = t0 + i / T, c = i % T;
      const bool in = t < bounds[e + 1];
      ps[i / T][c] = (in && k0 + c < a.K) ? to_f32(X[(long long)t * a.ldx + k0 + c]) : 0.f;
      qs[i / T][c] = (in && n0 + c < a.N) ? to_f32(Y[(long long)t * a.ldy + n0 + c]) : 0.f;
    }
    __syncthreads();
    step(ps, qs, acc);
    __syncthreads();
  }
  const int tm = (threadIdx.x & 15) * 4, tj = (threadIdx.x >> 4) * 4;
  TO* out = static_cast<TO*>(a.out) + (long long)e * a.N * a.K;
  for (int j = 0; j < 4; ++j)
    for (int i = 0; i < 4; ++i)
      if (n0 + tj + j < a.N && k0 + tm + i < a.K) out[(long long)(n0 + tj + j) * a.K + k0 + tm + i] = to_out<TO>(acc[i][j]);
}

template <class TI, class TO>
int launch_rows(bool nn, const RowsArgs& a, cudaStream_t stream) {
  const int cols = nn ? a.K : a.N;
  const long long grid = ((a.off.rows + T - 1ll) / T + a.off.groups + 1) * ((cols + T - 1ll) / T);
  if (grid >= (1ll << 31)) return (int)cudaErrorInvalidValue;
  if (nn) rows_kernel<true, TI, TO><<<(unsigned)grid, THREADS, 0, stream>>>(a);
  else rows_kernel<false, TI, TO><<<(unsigned)grid, THREADS, 0, stream>>>(a);
  return pcl_last_error();
}

template <class TI, class TO>
int launch_tn(const TnArgs& a, cudaStream_t stream) {
  const dim3 grid((a.K + T - 1) / T, (a.N + T - 1) / T, a.off.groups);
  tn_kernel<TI, TO><<<grid, THREADS, 0, stream>>>(a);
  return pcl_last_error();
}

bool sizes_ok(long long rows, int groups, int N, int K) {
  return rows >= 0 && rows < (1ll << 31) - 512 && groups >= 1 && groups <= MAX_GROUPS && N >= 1 && K >= 1;
}

}  // namespace

// mode 0: X [rows, K] -> out [rows, N]; mode 1: X [rows, N] -> out [rows, K].  W [groups, N, K] with strides (ws_e, ws_n, 1).
// in_type 1 / 2 (bf16 / fp16), out_type the same or 0 (fp32).  fill: rows of no group become zero, else they are left.
PCL_API int pcl_grouped_rows(int mode, int in_type, int out_type, const void* X, long long ldx, const void* W,
                             long long ws_e, long long ws_n, const void* offsets, int off64, void* out,
                             long long ldo, long long rows, int groups, int N, int K, int fill,
                             cudaStream_t stream) {
  if (!sizes_ok(rows, groups, N, K) || (mode != 0 && mode != 1)) return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  RowsArgs a{X, W, out, ldx, ws_e, ws_n, ldo, Offsets{offsets, off64, groups, (int)rows}, N, K, fill};
  const bool nn = mode == 1;
  if (in_type == TYPE_BF16 && out_type == TYPE_BF16) return launch_rows<__nv_bfloat16, __nv_bfloat16>(nn, a, stream);
  if (in_type == TYPE_BF16 && out_type == TYPE_F32) return launch_rows<__nv_bfloat16, float>(nn, a, stream);
  if (in_type == TYPE_F16 && out_type == TYPE_F16) return launch_rows<__half, __half>(nn, a, stream);
  if (in_type == TYPE_F16 && out_type == TYPE_F32) return launch_rows<__half, float>(nn, a, stream);
  return (int)cudaErrorInvalidValue;
}

// out [groups, N, K] (contiguous): every matrix is written, zeros where a group has no row
PCL_API int pcl_grouped_tn(int in_type, int out_type, const void* Y, long long ldy, const void* X, long long ldx,
                           const void* offsets, int off64, void* out, long long rows, int groups, int N, int K,
                           cudaStream_t stream) {
  if (!sizes_ok(rows, groups, N, K)) return (int)cudaErrorInvalidValue;
  TnArgs a{Y, X, out, ldy, ldx, Offsets{offsets, off64, groups, (int)rows}, N, K};
  if (in_type == TYPE_BF16 && out_type == TYPE_BF16) return launch_tn<__nv_bfloat16, __nv_bfloat16>(a, stream);
  if (in_type == TYPE_BF16 && out_type == TYPE_F32) return launch_tn<__nv_bfloat16, float>(a, stream);
  if (in_type == TYPE_F16 && out_type == TYPE_F16) return launch_tn<__half, __half>(a, stream);
  if (in_type == TYPE_F16 && out_type == TYPE_F32) return launch_tn<__half, float>(a, stream);
  return (int)cudaErrorInvalidValue;
}

// Copies the status block of the grouped products to `host` and clears it (waits for the stream).
PCL_API int pcl_grouped_status(PclStatus* host, cudaStream_t stream) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(host, g_status, sizeof(PclStatus), 0, cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess || host->code == 0) return (int)e;
  const PclStatus none{};
  e = cudaMemcpyToSymbolAsync(g_status, &none, sizeof(none), 0, cudaMemcpyHostToDevice, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  return (int)e;
}
