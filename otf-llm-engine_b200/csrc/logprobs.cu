// Log probabilities of given tokens, with rank, entropy and the likeliest tokens (otf_token_logprobs).
//
// Mathematics.  With m the row's largest logit and d_i = x_i - m, one pass keeps, under a running m,
// l = sum e^d_i over all entries but one of value m, and t = sum e^d_i d_i.  Then log sum e^x_i =
// m + log1p(l), a token's log probability is d - log1p(l), and the entropy log1p(l) - t / (1 + l), two terms
// that are not negative: both keep their relative precision where one token has nearly all of the weight.
// Parts join as l = l_a + (1 + l_b) f, t = t_a + f (t_b + (1 + l_b) (m_b - m_a)) with f = e^(m_b - m_a), m_b <= m_a.
// The likeliest tokens are kept as a sorted list of 32 in a warp's lanes, value before index.  What may belong to
// them gathers in a buffer of 32 that is sorted into the list when it is full; a bar that the warps share (each one's
// last listed value, and at first the top-th largest of its lanes' first maxima) keeps all but a few hundred
// entries of a row out.
//
// Bound: the logits are read once.  A row is cut among the warps of a cluster of CTAs (one CTA where there
// are enough rows), 512 logits at a time, 16 in each lane; their parts meet in the cluster's first CTA.
#include <algorithm>
#include <cfloat>

#include "paged.cuh"
#include "pairs.cuh"

namespace otf {

int set_cuda_error(cudaError_t e);     // capi.cu
int check_device();                    // capi.cu
int logprobs_device_error(int clear);  // read (and optionally clear) the flag below

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpGroup = 512;           // logits that a warp holds at once, 16 a lane
constexpr int kLpCluster = 16;
constexpr int kLpResident = 148 * 4;    // CTAs that run at once
constexpr int kLpMaxTop = 32;

// Set when a token lies outside the vocabulary.
__device__ int g_logprobs_device_error;

struct LogprobArgs {
  const void* x;
  int64_t ld;
  const int64_t* tokens;
  float* logprobs;
  float* entropy;
  int* ranks;
  int64_t* top_tokens;   // [n][top]
  float* top_logprobs;   // [n][top]
  int n, vocab, top;
};

// What is known of a part of a row.
struct __align__(16) LpPart {
  float m, l, t;
  int before;  // entries that come before the token
};
__device__ __forceinline__ LpPart lp_join(const LpPart& p, const LpPart& q) {
  const LpPart& a = p.m >= q.m ? p : q;
  const LpPart& b = p.m >= q.m ? q : p;
  LpPart r = a;
  if (b.m > -INFINITY) {
    const float d = b.m - a.m, f = __expf(d);
    r.l = fmaf(1.0f + b.l, f, a.l);
    r.t = fmaf(f, fmaf(1.0f + b.l, fmaxf(d, -200.0f), b.t), a.t);
  }
  r.before = p.before + q.before;
  return r;
}

// A value and its index as one number, the larger the better: by value, then by the lower index.  0: none.
__device__ __forceinline__ unsigned long long lp_key(float x, int i) {
  const uint32_t u = __float_as_uint(x + 0.0f), v = u & 0x80000000u ? ~u : u | 0x80000000u;  // -0 as 0
  return (unsigned long long)v << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float lp_value(unsigned long long k) {
  const uint32_t v = (uint32_t)(k >> 32);
  return __uint_as_float(v & 0x80000000u ? v & 0x7fffffffu : ~v);
}
// A lane's exchange in a sorting network: the larger of its own and the partner's key, or the smaller.
__device__ __forceinline__ unsigned long long lp_exchange(unsigned long long k, int o, bool larger) {
  const unsigned long long p = __shfl_xor_sync(0xffffffffu, k, o);
  return (p > k) == larger ? p : k;
}
// Keys that rise and then fall (or the reverse) over the lanes, sorted: the largest first.
__device__ __forceinline__ unsigned long long lp_merge(unsigned long long k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = lp_exchange(k, o, !(lane & o));
  return k;
}
__device__ __forceinline__ unsigned long long lp_sort(unsigned long long k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int n = 2; n <= 16; n <<= 1)
#pragma unroll
    for (int o = n / 2; o > 0; o >>= 1) k = lp_exchange(k, o, !(lane & o) == !(lane & n));
  return lp_merge(k);
}
// The 32 largest of two sorted lists, sorted.
__device__ __forceinline__ unsigned long long lp_both(unsigned long long a, unsigned long long b) {
  const unsigned long long r = __shfl_xor_sync(0xffffffffu, b, 31);
  return lp_merge(a > r ? a : r);
}

// 16 logits of each lane from entry i0 of a row on, -inf behind its end.  T: 0 fp32, 1 fp16, 2 bf16.
// Entry j of a lane is i0 + lp_index(j).
template <int T>
__device__ __forceinline__ int lp_index(int j) {
  const int lane = threadIdx.x & 31;
  return T == 0 ? (j >> 2) * 128 + lane * 4 + (j & 3) : (j >> 3) * 256 + lane * 8 + (j & 7);
}
template <int T>
__device__ __forceinline__ void lp_load(const void* row, int i0, int vocab, bool aligned, float (&v)[16]) {
  if (aligned && i0 + kLpGroup <= vocab) {
    if (T == 0) {
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const float4 y = __ldcs(reinterpret_cast<const float4*>(static_cast<const float*>(row) + i0 + lp_index<T>(4 * z)));
        v[4 * z] = y.x;
        v[4 * z + 1] = y.y;
        v[4 * z + 2] = y.z;
        v[4 * z + 3] = y.w;
      }
    } else {
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const uint4 y = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + i0 + lp_index<T>(8 * z)));
        const uint32_t u[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float2 f = unpack2<T == 2>(u[w]);
          v[8 * z + 2 * w] = f.x;
          v[8 * z + 2 * w + 1] = f.y;
        }
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int i = i0 + lp_index<T>(j);
      v[j] = -INFINITY;
      if (i < vocab)
        v[j] = T == 0 ? static_cast<const float*>(row)[i] : to_f<T == 2>(static_cast<const uint16_t*>(row)[i]);
    }
  }
}
// The largest float below x, the smallest above it (x itself for infinities and NaN).
__device__ __forceinline__ float lp_below(float x) { return x > -INFINITY ? nextafterf(x, -INFINITY) : x; }
__device__ __forceinline__ float lp_above(float x) { return x < INFINITY ? nextafterf(x, INFINITY) : x; }
// 1 where x > y, else 0.
__device__ __forceinline__ float lp_greater(float x, float y) {
  float r;
  asm("set.gt.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 32 values over the lanes, the largest first.
__device__ __forceinline__ float lp_sort_values(float x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
    for (int o = n / 2; o > 0; o >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, x, o);
      x = (!(lane & o) == !(lane & n)) ? fmaxf(x, y) : fminf(x, y);
    }
  return x;
}

// A warp's list of the likeliest, and what may belong to it.
struct LpList {
  unsigned long long best;     // the lane's entry of the sorted list
  unsigned long long* buffer;  // [32]
  uint32_t* bar;               // the row's, as the upper half of a key: an entry below it is not among the likeliest
  int held, top;
  float least;                 // entries below it need not be looked at

  // The buffer into the list.
  __device__ __forceinline__ void sort_in() {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    best = lp_both(best, lp_sort(lane < held ? buffer[lane] : 0ull));
    held = 0;
    raise();
    __syncwarp();
  }
  // Later entries of the warp have higher indexes: those as large as the list's last one come behind it.
  __device__ __forceinline__ void raise() {
    const unsigned long long last = __shfl_sync(0xffffffffu, best, top - 1);
    if (last) {
      least = fmaxf(least, lp_above(lp_value(last)));
      if ((threadIdx.x & 31) == 0) atomicMax(bar, (uint32_t)(last >> 32));
    }
  }
};

template <int T, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 4) k_token_logprobs(LogprobArgs a, int ctas) {
  __shared__ LpPart s_part[kLpWarps], s_cta[kLpCluster];
  __shared__ unsigned long long s_list[TOP ? kLpWarps : 1][32], s_cta_list[TOP ? kLpCluster : 1][32];
  __shared__ uint32_t s_bar;
  pdl_trigger();
  if (TOP) {
    if (threadIdx.x == 0) s_bar = 0;
    __syncthreads();
  }
  pdl_wait();
  if (ctas > 1) cluster_arrive_relaxed();
  const int row = blockIdx.x / ctas, rank = blockIdx.x - row * ctas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const char* x = static_cast<const char*>(a.x) + (int64_t)row * a.ld * (T == 0 ? 4 : 2);
  const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const int64_t asked = a.tokens[row];
  const int token = asked >= 0 && asked < a.vocab ? (int)asked : -1;
  float mine = -INFINITY;  // the token's logit; a NaN as -inf, an infinity as the largest number
  if (token >= 0) {
    mine = T == 0 ? reinterpret_cast<const float*>(x)[token] : to_f<T == 2>(reinterpret_cast<const uint16_t*>(x)[token]);
    mine = mine == mine ? fminf(mine, FLT_MAX) : -INFINITY;
  }
  const float mine_below = lp_below(mine);
  float m = -INFINITY, l = 0.0f, t = 0.0f;  // m of the warp, l and t of the lane
  float ahead[2] = {0.0f, 0.0f};  // entries before the token, whole numbers below 2^24 in a lane
  LpList list = {0ull, s_list[TOP ? warp : 0], &s_bar, 0, a.top, -FLT_MAX};  // an entry of -inf is none
  for (int64_t g = (int64_t)(rank * kLpWarps + warp) * kLpGroup; g < a.vocab; g += (int64_t)ctas * kLpWarps * kLpGroup) {
    const int i0 = (int)g;
    float v[16];
    lp_load<T>(x, i0, a.vocab, aligned, v);
    float top = v[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) top = fmaxf(top, v[j]);
    if (__any_sync(0xffffffffu, top == INFINITY)) {
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = v[j] == INFINITY ? FLT_MAX : v[j];
      top = fminf(top, FLT_MAX);
    }
    // the token's rank: entries before it count where they are equal, too
    if (token >= i0 + kLpGroup || token < i0) {
      const float than = token >= i0 ? mine_below : mine;
#pragma unroll
      for (int j = 0; j < 16; j += 2) add_two(ahead[0], ahead[1], lp_greater(v[j], than), lp_greater(v[j + 1], than));
      if (token >= i0 && mine == -INFINITY)  // all of them, NaN too
#pragma unroll
        for (int j = 0; j < 16; ++j) ahead[0] += !(v[j] > -INFINITY);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int i = i0 + lp_index<T>(j);
        ahead[0] += v[j] > mine || (i < token && !(v[j] < mine) && (v[j] == mine || mine == -INFINITY));
      }
    }
    if (TOP) {
      const uint32_t bar = *(volatile uint32_t*)&s_bar;
      if (bar) list.least = fmaxf(list.least, lp_value((unsigned long long)bar << 32));
      if (__any_sync(0xffffffffu, top >= list.least)) {
        if (list.least == -FLT_MAX) {
          // nothing known yet: a.top lanes have an entry that is their a.top-th largest maximum at least
          const float first = __shfl_sync(0xffffffffu, lp_sort_values(top == top ? top : -INFINITY), a.top - 1);
          if (first > -INFINITY) {
            list.least = first;
            if (lane == 0) atomicMax(&s_bar, (uint32_t)(lp_key(first, 0) >> 32));
          }
        }
        const float limit = list.least;  // sorting in may raise it before the entries counted here are taken
        int n = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) n += v[j] >= limit;
        int at = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, at, o);
          if (lane >= o) at += y;
        }
        const int all = __shfl_sync(0xffffffffu, at, 31);
        if (all <= 32) {
          if (list.held + all > 32) list.sort_in();
          at += list.held - n;
          if (n)
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (v[j] >= limit) list.buffer[at++] = lp_key(v[j], i0 + lp_index<T>(j));
          list.held += all;
        } else {
          if (list.held) list.sort_in();
#pragma unroll 1
          for (int j = 0; j < 16; ++j) {
            float x = v[0];
#pragma unroll
            for (int k = 1; k < 16; ++k) x = j == k ? v[k] : x;
            if (__any_sync(0xffffffffu, x >= list.least))
              list.best = lp_both(list.best, lp_sort(x >= list.least ? lp_key(x, i0 + lp_index<T>(j)) : 0ull));
          }
          list.raise();
        }
      }
    }
    // the warp's maximum, and the entry that l leaves out
    if (__any_sync(0xffffffffu, top > m)) {
      float mx = top;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float d = m - mx;
      if (m > -INFINITY) {
        const float f = __expf(d);
        t = f * fmaf(l, fmaxf(d, -200.0f), t);
        l *= f;
        if (lane == 0) {  // the entry left out so far
          l += f;
          t = fmaf(f, fmaxf(d, -200.0f), t);
        }
      }
      m = mx;
      const uint32_t has = __ballot_sync(0xffffffffu, top == mx);
      if (lane == __ffs((int)has) - 1) {
        bool out = false;
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (!out && v[j] == mx) {
            out = true;
            v[j] = -INFINITY;
          }
      }
    }
    // e^-200 is 0 in fp32; so -inf and NaN weigh nothing
    float sl[2] = {0.0f, 0.0f}, st[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      float d = v[j], e = v[j + 1];
      add_two(d, e, -m, -m);
      d = fmaxf(d, -200.0f);
      e = fmaxf(e, -200.0f);
      float p = d, q = e;
      fma_two(p, q, 1.4426950408889634f, 0.0f);
      p = lp_ex2(p);
      q = lp_ex2(q);
      add_two(sl[0], sl[1], p, q);
      fma_pair(st[0], st[1], p, q, d, e);
    }
    l += sl[0] + sl[1];
    t += st[0] + st[1];
  }
  int before = (int)ahead[0] + (int)ahead[1];
  if (TOP && list.held) list.sort_in();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    l += __shfl_xor_sync(0xffffffffu, l, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if (lane == 0) s_part[warp] = LpPart{m, l, t, before};
  if (TOP) s_list[warp][lane] = list.best;
  __syncthreads();
  if (ctas > 1) cluster_wait();  // all CTAs of the cluster run
  LpPart p = s_part[0];
  if (warp == 0) {
    for (int w = 1; w < kLpWarps; ++w) {
      p = lp_join(p, s_part[w]);
      if (TOP) list.best = lp_both(list.best, s_list[w][lane]);
    }
    if (ctas > 1) {
      if (lane == 0) {
        const uint32_t to = mapa_shared(smem_u32(&s_cta[rank]), 0);
        st_cluster_v2(to, __float_as_uint(p.m), __float_as_uint(p.l));
        st_cluster_v2(to + 8, __float_as_uint(p.t), (uint32_t)p.before);
      }
      if (TOP) st_cluster_v2(mapa_shared(smem_u32(&s_cta_list[rank][lane]), 0), (uint32_t)list.best, (uint32_t)(list.best >> 32));
    }
  }
  if (ctas > 1) {
    __syncwarp();
    cluster_sync_all();
    if (rank) return;
    if (warp == 0) {
      p = s_cta[0];
      for (int r = 1; r < ctas; ++r) {
        p = lp_join(p, s_cta[r]);
        if (TOP) list.best = lp_both(list.best, s_cta_list[r][lane]);
      }
    }
  }
  if (warp) return;
  const double lse = log1p((double)p.l);
  auto logprob = [&](float v) { return v > -INFINITY ? (float)(((double)v - (double)p.m) - lse) : -INFINITY; };
  if (lane == 0) {
    if (asked >= a.vocab) atomicExch(&g_logprobs_device_error, 1);
    a.logprobs[row] = token >= 0 ? logprob(mine) : asked < 0 ? 0.0f : __uint_as_float(0x7fc00000u);
    a.ranks[row] = token >= 0 ? p.before : -1;
    a.entropy[row] = (float)(lse - (double)p.t / (1.0 + (double)p.l));
  }
  if (TOP && lane < a.top) {
    a.top_tokens[(int64_t)row * a.top + lane] = list.best ? (int64_t)(int)~(uint32_t)list.best : -1;
    a.top_logprobs[(int64_t)row * a.top + lane] = list.best ? logprob(lp_value(list.best)) : -INFINITY;
  }
}

}  // namespace otf

using otf::check_device;
using otf::set_cuda_error;

int otf::logprobs_device_error(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, otf::g_logprobs_device_error, sizeof(int)) != cudaSuccess) {
    set_cuda_error(cudaGetLastError());
    return -1;
  }
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(otf::g_logprobs_device_error, &z, sizeof(int));
  }
  return v;
}

extern "C" OTF_API int otf_token_logprobs(const void* logits, int64_t ld, int32_t dtype, const int64_t* tokens,
                                          int64_t n, int64_t vocab, int64_t top, float* logprobs, float* entropy,
                                          int32_t* ranks, int64_t* top_tokens, float* top_logprobs, void* stream) {
  if (!logits || !tokens || !logprobs || !entropy || !ranks || n <= 0 || vocab <= 0 || ld < vocab || top < 0 ||
      (top && (!top_tokens || !top_logprobs)))
    return OTF_ERR_INVALID;
  if (dtype != OTF_DTYPE_F16 && dtype != OTF_DTYPE_BF16 && dtype != OTF_DTYPE_F32) return OTF_ERR_UNSUPPORTED;
  const int64_t size = dtype == OTF_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size) return OTF_ERR_INVALID;
  if (top > otf::kLpMaxTop || vocab > (1ll << 30) || n > (1ll << 26)) return OTF_ERR_UNSUPPORTED;
  const int st = check_device();
  if (st != OTF_OK) return st;
  const otf::LogprobArgs a = {logits, ld, tokens, logprobs, entropy, ranks, top_tokens, top_logprobs, (int)n, (int)vocab, (int)top};
  auto* k = dtype == OTF_DTYPE_F32   ? (top ? otf::k_token_logprobs<0, true> : otf::k_token_logprobs<0, false>)
            : dtype == OTF_DTYPE_F16 ? (top ? otf::k_token_logprobs<1, true> : otf::k_token_logprobs<1, false>)
                                     : (top ? otf::k_token_logprobs<2, true> : otf::k_token_logprobs<2, false>);
  int ctas = otf::kLpCluster;
  while (ctas > 1 && (n * ctas > otf::kLpResident || (int64_t)(ctas / 2) * otf::kLpWarps * otf::kLpGroup >= vocab)) ctas /= 2;
  if (ctas > 8) {
    static std::atomic<bool> done[6][64];
    int dev;
    bool needs;
    const int which = dtype == OTF_DTYPE_F32 ? 0 : dtype == OTF_DTYPE_F16 ? 1 : 2;
    cudaError_t e = otf::needs_opt_in(done[2 * which + (top > 0)], dev, needs);
    if (e == cudaSuccess && needs) {
      e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e == cudaSuccess) otf::opted_in(done[2 * which + (top > 0)], dev);
    }
    if (e != cudaSuccess) return set_cuda_error(e);
  }
  return set_cuda_error(otf::launch_pdl(k, dim3((unsigned)(n * ctas)), dim3(otf::kLpThreads), 0,
                                        static_cast<cudaStream_t>(stream), (unsigned)ctas, a, ctas));
}
