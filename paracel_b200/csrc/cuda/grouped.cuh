// What the grouped products share: the groups' bounds as the kernels take them, and the conversions of
// what they store.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace pcl_group {

constexpr int MAX_GROUPS = 1024;

// element types of the C entries
constexpr int TYPE_F32 = 0, TYPE_BF16 = 1, TYPE_F16 = 2;

struct Offsets {
  const void* p;   // groups + 1 numbers, null: one group of all rows
  int is64;
  int groups;
  int rows;        // rows of the tensor that they cut up

  __device__ __forceinline__ long long raw(int i) const {
    if (p == nullptr) return i == 0 ? 0 : rows;
    return is64 ? static_cast<const long long*>(p)[i] : static_cast<const int*>(p)[i];
  }
};

// bounds[0..groups] in shared memory as they come, inside the tensor; every thread of the block calls this, and synchronises behind it
static __device__ __forceinline__ void load_bounds(const Offsets& o, int* bounds, PclStatus* st) {
  for (int i = threadIdx.x; i <= o.groups; i += blockDim.x) {
    const long long raw = o.raw(i);
    const int v = (int)min(max(raw, 0ll), (long long)o.rows);
    bounds[i] = v;
    if (v != raw) pcl_report_bad_id(st, 0, 110, i, raw);
  }
}

template <class T> static __device__ __forceinline__ T to_out(float v);
template <> __device__ __forceinline__ float to_out<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 to_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half to_out<__half>(float v) { return __float2half_rn(v); }

static __device__ __forceinline__ float to_f32(float v) { return v; }
static __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
static __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

}  // namespace pcl_group
