// Running sums over the lanes of a wave by DPP moves: a dozen instructions, where moves through LDS wait for each step.
#pragma once

#include <hip/hip_runtime.h>

#include "common.h"

AKLR_SCALAR_FP32_BEGIN

namespace aklr {

// What the lane that CTRL names holds, in the rows of 16 lanes of MASK; 0 from no lane.
template <int CTRL, int MASK>
__device__ __forceinline__ int from_lane(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, MASK, 0xF, true);
}
template <int CTRL, int MASK>
__device__ __forceinline__ double from_lane(double x) {
  return __hiloint2double(from_lane<CTRL, MASK>(__double2hiint(x)), from_lane<CTRL, MASK>(__double2loint(x)));
}

// The sum of the lanes up to this one: of its half of the wave, or of the whole.
template <bool WHOLE, typename T>
__device__ __forceinline__ T sum_upto(T x) {
  x += from_lane<0x111, 0xF>(x);  // row_shr:1
  x += from_lane<0x112, 0xF>(x);
  x += from_lane<0x114, 0xF>(x);
  x += from_lane<0x118, 0xF>(x);
  x += from_lane<0x142, 0xA>(x);             // row_bcast:15 into rows 1 and 3
  if (WHOLE) x += from_lane<0x143, 0xC>(x);  // row_bcast:31 into rows 2 and 3
  return x;
}

// The sum of the lanes of a workgroup of THREADS before this one, and of all in `total`. `sums`: THREADS / 64 words of LDS.
template <int THREADS>
__device__ __forceinline__ int block_before(int x, int* sums, int& total) {
  const int s = sum_upto<true>(x), wave = threadIdx.x >> 6;
  __syncthreads();  // the last call's reads are done
  if ((threadIdx.x & 63) == 63) sums[wave] = s;
  __syncthreads();
  int off = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w == wave) off = total;
    total += sums[w];
  }
  return off + s - x;
}

}  // namespace aklr

AKLR_SCALAR_FP32_END
