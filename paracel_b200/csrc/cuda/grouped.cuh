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

// The products' status block belongs to the device: kernels of all streams report into it, and all threads ask for it.  It keeps its first report until
// that is taken.  Who writes or takes one holds the block (code BUSY) until the fields are complete, so that a report is read whole, and by one caller.
constexpr int CODE_WAIT = 1, CODE_BOUNDS = 2, CODE_BUSY = -1;

// (a function of its own: in line at every wait it made one row x 8192 x 4096 in four bits 8.9 instead of 8.7 us)
static __device__ __noinline__ void post(PclStatus* st, int code, int where, long long expected, long long seen) {
  if (atomicCAS(&st->code, 0, CODE_BUSY) != 0) return;
  st->rank = 0;
  st->wait_id = where;
  st->expected = expected;
  st->seen = seen;
  __threadfence();
  atomicExch(&st->code, code);
}

// by one thread: the report into `to` (code 0: there is none, or not yet), and out of the block
static __device__ __forceinline__ void take(PclStatus* st, PclStatus* to) {
  PclStatus got{};
  const int code = atomicAdd(&st->code, 0);
  if (code > 0 && atomicCAS(&st->code, code, CODE_BUSY) == code) {
    __threadfence();
    const volatile PclStatus* held = st;
    got.code = code;
    got.rank = held->rank;
    got.wait_id = held->wait_id;
    got.expected = held->expected;
    got.seen = held->seen;
    __threadfence();
    atomicExch(&st->code, 0);
  }
  *to = got;
}

// bounds[0..groups] in shared memory as they come, inside the tensor; every thread of the block calls this, and synchronises behind it
static __device__ __forceinline__ void load_bounds(const Offsets& o, int* bounds, PclStatus* st) {
  int moved = -1;
  long long from = 0;
  for (int i = threadIdx.x; i <= o.groups; i += blockDim.x) {
    const long long raw = o.raw(i);
    const int v = (int)min(max(raw, 0ll), (long long)o.rows);
    bounds[i] = v;
    if (v != raw && moved < 0) {
      moved = i;
      from = raw;
    }
  }
  if (moved >= 0) post(st, CODE_BOUNDS, 110, moved, from);
}

template <class T> static __device__ __forceinline__ T to_out(float v);
template <> __device__ __forceinline__ float to_out<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 to_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half to_out<__half>(float v) { return __float2half_rn(v); }

static __device__ __forceinline__ float to_f32(float v) { return v; }
static __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
static __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

}  // namespace pcl_group
