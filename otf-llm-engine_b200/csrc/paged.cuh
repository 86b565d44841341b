// What the paged cache's kernels share: the cache as they take it, and its checks on the host.
#pragma once

#include <cuda_bf16.h>

#include <atomic>

#include "otf_common.cuh"

namespace otf {

constexpr int kPagedMaxBatch = 4096;
constexpr int kPagedMaxTokens = 16;  // new tokens of a sequence in one attention call

// otf_paged_cache as the kernels take it.
struct PagedView {
  uint16_t* k;
  uint16_t* v;
  int64_t page_stride, token_stride, head_stride;
  const int* table;
  int64_t ld_table;
  const int* lengths;
  int n_pages, page_size, capacity, kv_heads, batch;
};

template <bool BF>
__device__ __forceinline__ float to_f(uint16_t v) {
  return BF ? __bfloat162float(__ushort_as_bfloat16(v)) : h2f(v);
}
template <bool BF>
__device__ __forceinline__ uint16_t from_f(float v) {
  return BF ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : f2h(v);
}

// Two values as they lie next to one another in memory.
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (BF) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool BF>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  return BF ? make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u))
            : __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// Division of numbers below 2^31 by a fixed one.
struct FastDiv {
  uint32_t mul, shift, d;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  return FastDiv{(uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1), l, d};
}
__device__ __forceinline__ uint32_t operator/(uint32_t n, const FastDiv& f) {
  return (__umulhi(f.mul, n) + n) >> f.shift;
}

// Whether a kernel's attributes still have to be set on the current device (done: per kernel, per device;
// setting them twice does no harm).
inline cudaError_t needs_opt_in(std::atomic<bool> (&done)[64], int& dev, bool& needs) {
  const cudaError_t e = cudaGetDevice(&dev);
  needs = e == cudaSuccess && (dev < 0 || dev >= 64 || !done[dev].load(std::memory_order_acquire));
  return e;
}
inline void opted_in(std::atomic<bool> (&done)[64], int dev) {
  if (dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_release);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The view of a cache, or why there is none.
inline int view_of(const otf_paged_cache* c, PagedView& v) {
  if (!c || !c->k_pages || !c->v_pages || !c->page_table || !c->lengths) return OTF_ERR_INVALID;
  if (c->dtype != OTF_DTYPE_F16 && c->dtype != OTF_DTYPE_BF16) return OTF_ERR_UNSUPPORTED;
  if (c->head_dim != 64 && c->head_dim != 128) return OTF_ERR_UNSUPPORTED;
  if (c->batch <= 0 || c->kv_heads <= 0 || c->page_size <= 0 || c->max_pages <= 0 || c->n_pages <= 0)
    return OTF_ERR_INVALID;
  if (c->batch > kPagedMaxBatch || c->kv_heads > 1024 || c->n_pages > INT32_MAX || c->page_size > INT32_MAX ||
      c->max_pages > INT32_MAX || c->max_pages * c->page_size > (1ll << 30))
    return OTF_ERR_UNSUPPORTED;
  if (c->ld_table < c->max_pages) return OTF_ERR_INVALID;
  if (!aligned16(c->k_pages) || !aligned16(c->v_pages) || c->page_stride % 8 || c->token_stride % 8 ||
      c->head_stride % 8 || c->page_stride < 0 || c->token_stride < c->head_dim || c->head_stride < c->head_dim)
    return OTF_ERR_INVALID;
  v = PagedView{static_cast<uint16_t*>(c->k_pages), static_cast<uint16_t*>(c->v_pages), c->page_stride,
                c->token_stride, c->head_stride, c->page_table, c->ld_table, c->lengths, (int)c->n_pages,
                (int)c->page_size, (int)(c->max_pages * c->page_size), (int)c->kv_heads, (int)c->batch};
  return OTF_OK;
}

// Whether `rows` rows of 16-bit values share memory with as many others (strides and columns of each).
// Views of one buffer whose columns lie beside one another share none.
inline bool rows_overlap(const void* x, int64_t ldx, int64_t colx, const void* y, int64_t ldy, int64_t coly, int64_t rows) {
  const int64_t at = (int64_t)(reinterpret_cast<intptr_t>(y) - reinterpret_cast<intptr_t>(x)) / 2;  // of y, from x on
  if (at >= (rows - 1) * ldx + colx || -at >= (rows - 1) * ldy + coly) return false;
  if (ldx == ldy) {
    const int64_t col = (at % ldx + ldx) % ldx;
    return col < colx || col + coly > ldx;
  }
  for (int64_t i = 0; i < rows; ++i) {  // the first of y's rows that ends behind the start of x's row i
    const int64_t ahead = i * ldx - at - coly, j = ahead < 0 ? 0 : ahead / ldy + 1;
    if (j < rows && at + j * ldy < i * ldx + colx) return true;
  }
  return false;
}
// The same of bytes that lie together.
inline bool bytes_overlap(const void* x, int64_t nx, const void* y, int64_t ny) {
  const intptr_t a = reinterpret_cast<intptr_t>(x), b = reinterpret_cast<intptr_t>(y);
  return a < b + ny && b < a + nx;
}

inline bool rows16(const void* p, int64_t ld, int64_t cols) { return p && aligned16(p) && ld % 8 == 0 && ld >= cols; }

}  // namespace otf
