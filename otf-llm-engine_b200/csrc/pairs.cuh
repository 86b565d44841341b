// Two fp32 operations in one instruction, and a maximum of three.
#pragma once

#include "otf_common.cuh"

namespace otf {

// x = x m + z, y = y m + z.
__device__ __forceinline__ void fma_two(float& x, float& y, float m, float z) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tmov.b64 c, {%3, %3};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}" : "+f"(x), "+f"(y) : "f"(m), "f"(z));
}
__device__ __forceinline__ void add_two(float& x, float& y, float u, float v) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "add.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "+f"(x), "+f"(y) : "f"(u), "f"(v));
}
// sx += x p, sy += y q.
__device__ __forceinline__ void fma_pair(float& sx, float& sy, float x, float y, float p, float q) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%0, %1};\n\t"
      "fma.rn.f32x2 c, a, b, c;\n\tmov.b64 {%0, %1}, c;\n\t}" : "+f"(sx), "+f"(sy) : "f"(x), "f"(y), "f"(p), "f"(q));
}
__device__ __forceinline__ float max_three(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

}  // namespace otf
