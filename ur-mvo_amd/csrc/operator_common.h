// operator_common.h -- what the operators on caller-owned device tensors share (attention, log probabilities, distillation):
// element types, the device guard of a call, the workgroup barrier.
#pragma once
#include "../../include/urf.h"
#include "urf_common.h"

namespace urf {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

inline int dtype_bytes(int dtype) { return dtype == URF_F32 ? 4 : dtype == URF_F16 || dtype == URF_BF16 ? 2 : 0; }

// The operators leave the calling thread's current device as they found it: their callers own the tensors and have a current
// device of their own (the handles' entry points bind theirs).
struct OnDevice {
  int before = -1;
  hipError_t rc;
  explicit OnDevice(int device) {
    rc = hipGetDevice(&before);
    if (rc == hipSuccess && before == device) before = -1;
    else if (rc == hipSuccess) rc = hipSetDevice(device);
  }
  ~OnDevice() { if (before >= 0) (void)hipSetDevice(before); }
};

// Workgroup barrier with the wait for the wave's own LDS operations written out: hipcc drops that wait at a barrier that heads
// a loop when the pending write sits on the back edge.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

}  // namespace urf
