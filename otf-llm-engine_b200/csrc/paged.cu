// A key/value cache in pages: rotary positions and the write of new tokens (otf_paged_append) and
// the cut of long sequences to a budget (otf_paged_evict); the attention that reads it is in
// paged_attn.cu.  Layout and rules: include/otf_b200.h.
#include <algorithm>

#include "paged.cuh"

namespace otf {

int set_cuda_error(cudaError_t e);  // capi.cu
int check_device();                 // capi.cu
int paged_device_error(int clear);  // read (and optionally clear) the flag below

// Set when a sequence does not fit its pages or names a page outside the pool.
__device__ int g_paged_device_error;
__device__ __forceinline__ void report_bad_page() { atomicExch(&g_paged_device_error, 1); }

// The sequence of row `row` under the row ranges starts[0..batch], found by a warp: as many
// sequences end at or before it.  batch when the row lies behind the last sequence.
__device__ __forceinline__ int sequence_of(const int* starts, int batch, int row) {
  const int lane = threadIdx.x & 31;
  int b = 0;
  for (int i = 0; i < batch; i += 32) {
    const bool ended = i + lane < batch && starts[i + lane + 1] <= row;
    b += __popc(__ballot_sync(0xffffffffu, ended));
  }
  return b;
}

// Rotary positions and the cache write, one CTA per row.
template <bool BF>
__global__ void __launch_bounds__(256) k_paged_append(PagedView c, const double* turns, int rot, float factor,
                                                      int interleaved, const uint16_t* q, int64_t ldq, uint16_t* qo,
                                                      int64_t ldqo, int heads, const uint16_t* k, int64_t ldk,
                                                      const uint16_t* v, int64_t ldv, const int* starts,
                                                      const int* positions, int per, int D) {
  __shared__ float s_c[64], s_s[64];
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.x, tid = threadIdx.x;
  const int b = starts ? sequence_of(starts, c.batch, row) : row / per;
  if (b >= c.batch) return;  // behind the last sequence
  const int t = row - (starts ? starts[b] : b * per);
  const int len = c.lengths[b];
  if (len < 0) return;  // no sequence in this place
  const int64_t slot = (int64_t)len + t;
  if (t < 0 || slot >= c.capacity) {
    if (tid == 0) report_bad_page();
    return;
  }
  const int page = c.table[b * c.ld_table + slot / c.page_size];
  if (page < 0 || page >= c.n_pages) {
    if (tid == 0) report_bad_page();
    return;
  }
  const int half = rot / 2;
  if (tid < half) {
    double turn = (double)(positions ? positions[row] : (int)slot) * turns[tid];
    turn -= rint(turn);
    float sn, cs;
    sincospif(2.0f * (float)turn, &sn, &cs);
    s_c[tid] = cs * factor;
    s_s[tid] = sn * factor;
  }
  __syncthreads();
  const int64_t at = page * c.page_stride + (slot % c.page_size) * c.token_stride;
  const int pairs = D / 2;
  const int turning = (q ? heads : 0) + c.kv_heads;
  for (int e = tid; e < turning * pairs; e += blockDim.x) {
    int h = e / pairs;
    const int i = e - h * pairs;
    const uint16_t* x;
    uint16_t* y;
    if (q && h < heads) {
      x = q + row * ldq + (int64_t)h * D;
      y = qo + row * ldqo + (int64_t)h * D;
    } else {
      if (q) h -= heads;
      x = k + row * ldk + (int64_t)h * D;
      y = c.k + at + h * c.head_stride;
    }
    int i0, i1;
    if (i < half) {
      i0 = interleaved ? 2 * i : i;
      i1 = interleaved ? 2 * i + 1 : i + half;
    } else {
      i0 = 2 * i;
      i1 = 2 * i + 1;
    }
    const uint16_t xa = x[i0], xb = x[i1];
    if (i < half) {
      const float fa = to_f<BF>(xa), fb = to_f<BF>(xb);
      y[i0] = from_f<BF>(fa * s_c[i] - fb * s_s[i]);
      y[i1] = from_f<BF>(fb * s_c[i] + fa * s_s[i]);
    } else {
      y[i0] = xa;
      y[i1] = xb;
    }
  }
  for (int e = tid; e < c.kv_heads * D; e += blockDim.x) {
    const int h = e / D, i = e - h * D;
    c.v[at + h * c.head_stride + i] = v[row * ldv + (int64_t)h * D + i];
  }
}

// ---- eviction -------------------------------------------------------------------------------

// A weight's rank as an unsigned number: larger weights larger, -0 as 0, a NaN the largest.
__device__ __forceinline__ uint32_t weight_key(float w) {
  uint32_t u = __float_as_uint(w);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kEvictThreads = 1024;

// One CTA per (sequence, KV head): the k-th largest key by four rounds of 8 bits, then the kept
// places in order.  Weights move downwards only, tile by tile, so they may be cut in place.
__global__ void __launch_bounds__(kEvictThreads) k_evict_select(const int* lengths, int kv_heads, int capacity,
                                                                const float* weights, int64_t ldw, float* wout,
                                                                int64_t ldwo, int budget, int recent, int* kept) {
  __shared__ int s_hist[256];
  __shared__ int s_need;
  __shared__ uint32_t s_prefix;
  __shared__ int s_g[32], s_e[32];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / kv_heads;
  const float* w = weights + (int64_t)blockIdx.x * ldw;
  float* wo = wout + (int64_t)blockIdx.x * ldwo;
  int* keep = kept + (int64_t)blockIdx.x * budget;
  int len = lengths[b];
  if (len > capacity || len > ldw) {
    if (tid == 0) report_bad_page();
    len = -1;
  }
  if (len < 0) {
    for (int i = tid; i < budget; i += kEvictThreads) keep[i] = -1;
    return;
  }
  const bool in_place = wout == weights;
  if (len <= budget) {
    for (int i = tid; i < budget; i += kEvictThreads) keep[i] = i < len ? i : -1;
    if (!in_place)
      for (int64_t i = tid; i < ldwo; i += kEvictThreads) wo[i] = i < len ? w[i] : 0.0f;
    return;
  }
  const int n = len - recent, k = budget - recent;
  if (tid == 0) {
    s_prefix = 0u;
    s_need = k;
  }
  uint32_t mask = 0u;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) s_hist[tid] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix;
    for (int i = tid; i < n; i += kEvictThreads) {
      const uint32_t u = weight_key(w[i]);
      if ((u & mask) == prefix) atomicAdd(&s_hist[(u >> shift) & 255u], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int need = s_need, bin = 255;
      while (bin > 0 && s_hist[bin] < need) need -= s_hist[bin--];
      s_need = need;
      s_prefix = prefix | ((uint32_t)bin << shift);
    }
    mask |= 255u << shift;
    __syncthreads();
  }
  const uint32_t limit = s_prefix;
  const int need = s_need;  // of the keys equal to the limit, the first ones
  int g0 = 0, e0 = 0;
  for (int base = 0; base < n; base += kEvictThreads) {
    const int i = base + tid;
    const float x = i < n ? w[i] : 0.0f;
    const uint32_t u = weight_key(x);
    const bool gt = k > 0 && i < n && u > limit, eq = k > 0 && i < n && u == limit;
    const unsigned bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) {
      s_g[warp] = __popc(bg);
      s_e[warp] = __popc(be);
    }
    __syncthreads();  // the tile's weights are read, its counts there
    int g = g0, e = e0;
    for (int i2 = 0; i2 < 32; ++i2) {
      if (i2 < warp) {
        g += s_g[i2];
        e += s_e[i2];
      }
      g0 += s_g[i2];
      e0 += s_e[i2];
    }
    const unsigned below = (1u << lane) - 1u;
    g += __popc(bg & below);
    e += __popc(be & below);
    if (gt || (eq && e < need)) {
      const int at = g + min(e, need);
      keep[at] = i;
      wo[at] = x;
    }
    __syncthreads();
  }
  for (int base = 0; base < recent; base += kEvictThreads) {
    const int i = base + tid;
    const float x = i < recent ? w[n + i] : 0.0f;
    __syncthreads();
    if (i < recent) {
      keep[k + i] = n + i;
      wo[k + i] = x;
    }
    __syncthreads();
  }
  const int64_t end = in_place ? len : ldwo;
  for (int64_t i = budget + tid; i < end; i += kEvictThreads) wo[i] = 0.0f;
}

// One CTA per (sequence, KV head, keys or values): the kept rows move to the front, 16 at a
// time in order.  A row's place never rises, so a step's rows are read before any row of the
// step or of a later one is overwritten, and the pages may be the same.
__global__ void __launch_bounds__(256) k_evict_move(PagedView from, PagedView to, const int* kept, int budget, int D,
                                                    int* lengths_out) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x / from.kv_heads, g = blockIdx.x - b * from.kv_heads;
  const uint16_t* src = blockIdx.y ? from.v : from.k;
  uint16_t* dst = blockIdx.y ? to.v : to.k;
  const int* keep = kept + (int64_t)blockIdx.x * budget;
  const int pieces = D / 8, rows = 256 / pieces;
  const int r = threadIdx.x / pieces, piece = threadIdx.x - r * pieces;
  for (int base = 0; base < budget; base += rows) {
    const int j = base + r;
    const int s = j < budget ? keep[j] : -1;
    uint4 x = make_uint4(0, 0, 0, 0);
    bool ok = s >= 0;
    if (ok) {
      const int p = from.table[b * from.ld_table + s / from.page_size];
      ok = p >= 0 && p < from.n_pages;
      if (ok)
        x = *reinterpret_cast<const uint4*>(src + p * from.page_stride + (s % from.page_size) * from.token_stride +
                                            g * from.head_stride + piece * 8);
    }
    __syncthreads();
    if (s >= 0) {
      const int p = to.table[b * to.ld_table + j / to.page_size];
      if (p < 0 || p >= to.n_pages) ok = false;
      if (ok)
        *reinterpret_cast<uint4*>(dst + p * to.page_stride + (j % to.page_size) * to.token_stride +
                                  g * to.head_stride + piece * 8) = x;
      else
        report_bad_page();
    }
    __syncthreads();
  }
  if (g == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
    const int len = from.lengths[b];
    lengths_out[b] = len > from.capacity ? len : min(len, budget);
  }
}

}  // namespace otf

using otf::check_device;
using otf::set_cuda_error;

int otf::paged_device_error(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, otf::g_paged_device_error, sizeof(int)) != cudaSuccess) {
    set_cuda_error(cudaGetLastError());
    return -1;
  }
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(otf::g_paged_device_error, &z, sizeof(int));
  }
  return v;
}

extern "C" OTF_API int otf_paged_append(const otf_paged_cache* cache, const otf_rotary* rotary, const void* q,
                                        int64_t ldq, void* q_out, int64_t ldqo, int64_t heads, const void* k,
                                        int64_t ldk, const void* v, int64_t ldv, const int32_t* starts,
                                        const int32_t* positions, int64_t n, void* stream) {
  otf::PagedView c;
  int st = otf::view_of(cache, c);
  if (st != OTF_OK) return st;
  const int64_t D = cache->head_dim;
  if (n < 0 || n > INT32_MAX || (!starts && n % c.batch)) return OTF_ERR_INVALID;
  if (n == 0) return OTF_OK;
  if (!otf::rows16(k, ldk, c.kv_heads * D) || !otf::rows16(v, ldv, c.kv_heads * D)) return OTF_ERR_INVALID;
  if (q && (heads <= 0 || heads > 65535 || !otf::rows16(q, ldq, heads * D) || !otf::rows16(q_out, ldqo, heads * D)))
    return OTF_ERR_INVALID;
  int rot = 0;
  if (rotary) {
    if (rotary->rot_dim < 0 || rotary->rot_dim > D || rotary->rot_dim % 2 || (rotary->rot_dim && !rotary->turns))
      return OTF_ERR_INVALID;
    rot = (int)rotary->rot_dim;
  }
  st = check_device();
  if (st != OTF_OK) return st;
  auto* kern = cache->dtype == OTF_DTYPE_BF16 ? otf::k_paged_append<true> : otf::k_paged_append<false>;
  return set_cuda_error(otf::launch_pdl(
      kern, dim3((unsigned)n), dim3(256), 0, static_cast<cudaStream_t>(stream), 1u, c, rot ? rotary->turns : nullptr,
      rot, rot ? rotary->factor : 1.0f, rot ? (int)rotary->interleaved : 0, static_cast<const uint16_t*>(q), ldq,
      static_cast<uint16_t*>(q_out), ldqo, (int)heads, static_cast<const uint16_t*>(k), ldk,
      static_cast<const uint16_t*>(v), ldv, starts, positions, (int)(n / c.batch), (int)D));
}

extern "C" OTF_API int otf_paged_evict(const otf_paged_cache* from, const otf_paged_cache* to, const float* weights,
                                       int64_t ldw, float* weights_out, int64_t ldw_out, int64_t budget,
                                       int64_t recent, int32_t* kept, int32_t* lengths_out, void* stream) {
  otf::PagedView f, t;
  int st = otf::view_of(from, f);
  if (st == OTF_OK) st = otf::view_of(to, t);
  if (st != OTF_OK) return st;
  if (!weights || !weights_out || !kept || !lengths_out) return OTF_ERR_INVALID;
  if (from->head_dim != to->head_dim || from->dtype != to->dtype || f.kv_heads != t.kv_heads || f.batch != t.batch ||
      f.page_size != t.page_size)
    return OTF_ERR_INVALID;
  if (budget <= 0 || recent < 0 || recent > budget || budget > t.capacity) return OTF_ERR_INVALID;
  if (ldw < f.capacity || ldw_out < budget || (weights == weights_out && ldw != ldw_out)) return OTF_ERR_INVALID;
  st = check_device();
  if (st != OTF_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned pairs = (unsigned)(f.batch * f.kv_heads);
  cudaError_t e = otf::launch_pdl(otf::k_evict_select, dim3(pairs), dim3(otf::kEvictThreads), 0, s, 1u, f.lengths,
                                  f.kv_heads, f.capacity, weights, ldw, weights_out, ldw_out, (int)budget, (int)recent,
                                  kept);
  if (e != cudaSuccess) return set_cuda_error(e);
  return set_cuda_error(otf::launch_pdl(otf::k_evict_move, dim3(pairs, 2), dim3(256), 0, s, 1u, f, t,
                                        (const int*)kept, (int)budget, (int)from->head_dim, lengths_out));
}
