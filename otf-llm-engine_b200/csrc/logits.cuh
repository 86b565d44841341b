// What the kernels that read rows of logits share.
#pragma once

#include "otf_common.cuh"

namespace otf {

// 0, or from 1e-20 on (log2(e) / T stays finite; its product with a difference of logits need not).  In 64 bits: a number
// that fp32 would hold as 0 is none of them.
__host__ __device__ __forceinline__ bool temperature_ok(double T) { return T == 0.0 || (T >= 1e-20f && T <= 1e20f); }

// Four consecutive values of a row, `pad` behind its end.  Rows that are not 16-byte aligned are read
// value by value by the same threads, so that a row's sums do not depend on where it lies.
__device__ __forceinline__ float4 logits4(const float* x, int i, int end, bool aligned, float pad = -INFINITY) {
  if (aligned && i + 4 <= end) return __ldcs(reinterpret_cast<const float4*>(x + i));
  float4 v;
  v.x = i < end ? __ldcs(x + i) : pad;
  v.y = i + 1 < end ? __ldcs(x + i + 1) : pad;
  v.z = i + 2 < end ? __ldcs(x + i + 2) : pad;
  v.w = i + 3 < end ? __ldcs(x + i + 3) : pad;
  return v;
}

}  // namespace otf
