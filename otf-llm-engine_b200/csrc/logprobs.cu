// Log probabilities of given tokens, with rank, entropy and the likeliest tokens (otf_token_logprobs).
//
// Mathematics.  With m the row's largest logit and d_i = x_i - m, one pass keeps, under a running m,
// l = sum e^d_i over all entries but one of value m, and t = sum e^d_i d_i.  (A warp's m may be an entry of another
// warp; it then leaves out none.)  Then log sum e^x_i =
// m + log1p(l), a token's log probability is d - log1p(l), and the entropy log1p(l) - t / (1 + l), two terms
// that are not negative: both keep their relative precision where one token has nearly all of the weight.
// Parts join as l = l_a + (h + l_b) f, t = t_a + f (t_b + (h + l_b) (m_b - m_a)) with f = e^(m_b - m_a), m_b <= m_a,
// and h what b left out, 1 or 0.
// For the likeliest tokens the pass leaves the maximum of every 16 logits of a lane (more in long rows) in shared
// memory.  The top-th largest of the lanes' maxima over all is a bar that as many entries reach, and few others: the
// sixteens that reach it, about one for each token wanted, are read again and sorted, value before index.
//
// Bound: the logits are read once.  A row is cut among the warps of a cluster of CTAs (one CTA where there
// are enough rows), 512 logits at a time, 16 in each lane; their parts meet in the cluster's first CTA.
//
// Measured: 2047 rows of 128256 fp32, 1.05 GB, 164 to 183 us = 5.7 to 6.4 TB/s; 1024 rows of 128256 bf16, 0.26 GB, 78 us
// without a list and 98 to 111 with twenty alternatives: instructions bound it, some 13 a logit, and twice the logits come
// with every byte; 4 rows of 32000 with five alternatives 9.5 us.
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
constexpr int kLpPerSm = 4;             // CTAs of an SM (twenty of 1024 x 128256 bf16: 132 us with 3 of 80 registers, 99 with 4 of 64)
constexpr int kLpResident = 148 * kLpPerSm;
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
  int per;  // groups of a slot
};

// What is known of a part of a row.
struct __align__(16) LpPart {
  float m, l, t;
  int before;  // twice the entries that come before the token, and 1 if an entry of value m is left out of l
};
__device__ __forceinline__ LpPart lp_join(const LpPart& p, const LpPart& q) {
  const LpPart& a = p.m >= q.m ? p : q;
  const LpPart& b = p.m >= q.m ? q : p;
  LpPart r = a;
  r.before = (p.before & ~1) + (q.before & ~1) + (a.before & 1);
  const float out = (float)(b.before & 1), l = b.l + out;
  if (b.m == a.m) {
    r.l += b.l + out * (float)(a.before & 1);  // one is left out of both together
    r.t += b.t;
    r.before |= b.before & 1;
  } else if (b.m > -INFINITY) {
    const float d = fmaxf(b.m - a.m, -200.0f), f = __expf(d);
    r.l = fmaf(l, f, a.l);
    r.t = fmaf(f, fmaf(l, d, b.t), a.t);
  }
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
struct LpRaw {
  uint4 x[T == 0 ? 4 : 2];
};
// Two 16-bit logits of a lane's 16, z of 8.
template <int T>
__device__ __forceinline__ uint32_t lp_word(const LpRaw<T>& raw, int z) {
  const uint4& x = raw.x[z >> 2];
  return (z & 3) == 0 ? x.x : (z & 3) == 1 ? x.y : (z & 3) == 2 ? x.z : x.w;
}
template <int T>
__device__ __forceinline__ void lp_load(const void* row, int64_t i0, int vocab, bool aligned, LpRaw<T>& raw) {
  constexpr int N = T == 0 ? 4 : 2, E = 16 / N;
  if (i0 >= vocab) return;
  if (aligned && i0 + kLpGroup <= vocab) {
#pragma unroll
    for (int z = 0; z < N; ++z)
      raw.x[z] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const char*>(row) + (i0 + lp_index<T>(E * z)) * (T == 0 ? 4 : 2)));
  } else {
#pragma unroll
    for (int z = 0; z < N; ++z) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = (int)i0 + lp_index<T>(E * z + (T == 0 ? k : 2 * k));
        if (T == 0) {
          w[k] = i < vocab ? static_cast<const uint32_t*>(row)[i] : 0xFF800000u;
        } else {
          constexpr uint32_t none = T == 1 ? 0xFC00u : 0xFF80u;
          const uint16_t* x = static_cast<const uint16_t*>(row) + i;
          w[k] = (i < vocab ? x[0] : none) | (i + 1 < vocab ? x[1] : none) << 16;
        }
      }
      raw.x[z] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}
template <int T>
__device__ __forceinline__ void lp_values(const LpRaw<T>& raw, float (&v)[16]) {
  constexpr int N = T == 0 ? 4 : 2, E = 16 / N;
#pragma unroll
  for (int z = 0; z < N; ++z) {
    const uint32_t w[4] = {raw.x[z].x, raw.x[z].y, raw.x[z].z, raw.x[z].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (T == 0) {
        v[E * z + k] = __uint_as_float(w[k]);
      } else {
        const float2 f = unpack2<T == 2>(w[k]);
        v[E * z + 2 * k] = f.x;
        v[E * z + 2 * k + 1] = f.y;
      }
    }
  }
}
// The smallest float above x (x itself for an infinity or NaN).
__device__ __forceinline__ float lp_above(float x) { return x < INFINITY ? nextafterf(x, INFINITY) : x; }
// 1 where x > y, or (EQUAL) x >= y, else 0.
template <bool EQUAL>
__device__ __forceinline__ float lp_greater(float x, float y) {
  float r;
  if (EQUAL) asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  else asm("set.gt.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
// How many of a lane's 16 logits are larger than `than`, or (EQUAL) as large: in two halves.
template <int T, bool EQUAL>
__device__ __forceinline__ float2 lp_ahead(const LpRaw<T>& raw, const float (&v)[16], float than) {
  float2 n = make_float2(0.0f, 0.0f);
  if constexpr (T == 0) {
#pragma unroll
    for (int j = 0; j < 16; j += 2) add_two(n.x, n.y, lp_greater<EQUAL>(v[j], than), lp_greater<EQUAL>(v[j + 1], than));
  } else if constexpr (T == 1) {
    const __half2 y = __float2half2_rn(than);  // exact: it is one of the row's
    __half2 sum = __float2half2_rn(0.0f);
#pragma unroll
    for (int z = 0; z < 8; ++z) {
      const uint32_t w = lp_word<T>(raw, z);
      const __half2 x = *reinterpret_cast<const __half2*>(&w);
      sum = __hadd2(sum, EQUAL ? __hge2(x, y) : __hgt2(x, y));
    }
    n = __half22float2(sum);
  } else {
    const __nv_bfloat162 y = __float2bfloat162_rn(than);
    __nv_bfloat162 sum = __float2bfloat162_rn(0.0f);
#pragma unroll
    for (int z = 0; z < 8; ++z) {
      const uint32_t w = lp_word<T>(raw, z);
      const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&w);
      sum = __hadd2(sum, EQUAL ? __hge2(x, y) : __hgt2(x, y));
    }
    n = __bfloat1622float2(sum);
  }
  return n;
}
// The largest of a lane's 16 logits (NaN aside).
template <int T>
__device__ __forceinline__ float lp_top(const LpRaw<T>& raw, const float (&v)[16]) {
  if constexpr (T == 0) {
    float top = v[0];
#pragma unroll
    for (int j = 1; j < 15; j += 2) top = max_three(top, v[j], v[j + 1]);
    return fmaxf(top, v[15]);
  } else {
    uint32_t w[8];
#pragma unroll
    for (int z = 0; z < 8; ++z) w[z] = lp_word<T>(raw, z);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1)
#pragma unroll
      for (int z = 0; z < o; ++z) {
        if (T == 1) {
          const __half2 y = __hmax2(*reinterpret_cast<const __half2*>(&w[z]), *reinterpret_cast<const __half2*>(&w[z + o]));
          w[z] = *reinterpret_cast<const uint32_t*>(&y);
        } else {
          const __nv_bfloat162 y = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&w[z]), *reinterpret_cast<const __nv_bfloat162*>(&w[z + o]));
          w[z] = *reinterpret_cast<const uint32_t*>(&y);
        }
      }
    const float2 y = unpack2<T == 2>(w[0]);
    return fmaxf(y.x, y.y);
  }
}
__device__ __forceinline__ float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 32 values over the lanes, the largest first; and of two such lists the 32 largest.
__device__ __forceinline__ float lp_step(float x, int o, bool larger) {
  const float y = __shfl_xor_sync(0xffffffffu, x, o);
  return larger ? fmaxf(x, y) : fminf(x, y);
}
__device__ __forceinline__ float lp_sort_values(float x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
    for (int o = n / 2; o > 0; o >>= 1) x = lp_step(x, o, !(lane & o) == !(lane & n));
  return x;
}
__device__ __forceinline__ float lp_both_values(float x, float y) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, y, 31));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = lp_step(x, o, !(threadIdx.x & o));
  return x;
}

// Slots of a lane's maxima.  A slot has `per` groups of 16.
constexpr int kLpSlots = 32;

// One logit; a NaN as -inf, an infinity as the largest number.
template <int T>
__device__ __forceinline__ float lp_one(const void* row, int i) {
  const float x = T == 0 ? static_cast<const float*>(row)[i] : to_f<T == 2>(static_cast<const uint16_t*>(row)[i]);
  return x == x ? fminf(x, FLT_MAX) : -INFINITY;
}

// The 32 largest entries of a warp's groups, sorted: those of the slots that reach `bar` are looked at.
template <int T>
__device__ unsigned long long lp_likeliest(const void* row, const float (&slots)[kLpSlots][kLpThreads], int64_t first, int64_t step,
                                           int per, int vocab, float bar, int top) {
  const int lane = threadIdx.x & 31;
  unsigned long long best = 0;
  float least = bar;  // entries below it need not be looked at
  for (int k = 0; k < kLpSlots && first + (int64_t)k * per * step < vocab; ++k) {
    uint32_t in = __ballot_sync(0xffffffffu, slots[k][threadIdx.x] >= least);
    while (in) {
      // two lanes' sixteens at a time, of each group of the slot
      const int one = __ffs((int)in) - 1;
      in &= in - 1;
      const int two = in ? __ffs((int)in) - 1 : -1;
      in &= in - 1;
      const int of = lane < 16 ? one : two, j = lane & 15;
      for (int z = 0; z < per; ++z) {
        const int64_t i0 = first + ((int64_t)k * per + z) * step;
        const int64_t i = i0 + (T == 0 ? (j >> 2) * 128 + of * 4 + (j & 3) : (j >> 3) * 256 + of * 8 + (j & 7));
        const float x = of >= 0 && i < vocab ? lp_one<T>(row, (int)i) : -INFINITY;
        if (__any_sync(0xffffffffu, x >= least)) {
          best = lp_both(best, lp_sort(x >= least ? lp_key(x, (int)i) : 0ull));
          // later slots have higher indexes, but another lane of this one's need not
          const unsigned long long last = __shfl_sync(0xffffffffu, best, top - 1);
          if (last) least = fmaxf(least, lp_value(last));
        }
      }
    }
    const unsigned long long last = __shfl_sync(0xffffffffu, best, top - 1);
    if (last) least = fmaxf(least, lp_above(lp_value(last)));
  }
  return best;
}

template <int T, bool TOP>
__global__ void __launch_bounds__(kLpThreads, kLpPerSm) k_token_logprobs(LogprobArgs a, int ctas) {
  __shared__ LpPart s_part[kLpWarps], s_cta[kLpCluster];
  __shared__ unsigned long long s_list[TOP ? kLpWarps : 1][32], s_cta_list[TOP ? kLpCluster : 1][32];
  __shared__ float s_slots[TOP ? kLpSlots : 1][TOP ? kLpThreads : 1];
  __shared__ float s_first[TOP ? kLpWarps : 1][32], s_max[kLpWarps];
  pdl_trigger();
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
  float m = -INFINITY, l = 0.0f, t = 0.0f;  // m of the warp, l and t of the lane
  float ahead[2] = {0.0f, 0.0f};  // entries before the token, whole numbers below 2^24 in a lane
  float high = -INFINITY, highest = -INFINITY;  // of the lane's slot at hand, of all of them
  int slot = 0, in_slot = 0;
  const int64_t step = (int64_t)ctas * kLpWarps * kLpGroup;
  LpRaw<T> next;  // the group after the one at hand is on its way
  lp_load<T>(x, (int64_t)(rank * kLpWarps + warp) * kLpGroup, a.vocab, aligned, next);
  int out = 0;  // whether an entry of value m is left out of the warp's l
  {
    // m to begin with: the largest of the warps' first groups, so that few warps ever meet a larger one
    float top = -INFINITY;
    if ((int64_t)(rank * kLpWarps + warp) * kLpGroup < a.vocab) {
      float v[16];
      lp_values<T>(next, v);
      top = lp_top<T>(next, v);
      if (top == INFINITY) top = FLT_MAX;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) s_max[warp] = fmaxf(top, -INFINITY);  // a NaN as -inf
    __syncthreads();
    int owner = 0;
#pragma unroll
    for (int w = 0; w < kLpWarps; ++w) {
      if (s_max[w] > m) {
        m = s_max[w];
        owner = w;
      }
    }
    if (owner == warp) m = -INFINITY;  // it meets the entry in its first group
  }
  for (int64_t g = (int64_t)(rank * kLpWarps + warp) * kLpGroup; g < a.vocab; g += step) {
    const int i0 = (int)g;
    const LpRaw<T> raw = next;
    float v[16];
    lp_values<T>(raw, v);
    lp_load<T>(x, g + step, a.vocab, aligned, next);
    float top = lp_top<T>(raw, v);
    if (__any_sync(0xffffffffu, top == INFINITY)) {
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = v[j] == INFINITY ? FLT_MAX : v[j];
      top = fminf(top, FLT_MAX);
    }
    // the token's rank: entries before it count where they are equal, too
    if (token >= i0 + kLpGroup || token < i0) {
      const float2 n = token >= i0 ? lp_ahead<T, true>(raw, v, mine) : lp_ahead<T, false>(raw, v, mine);
      add_two(ahead[0], ahead[1], n.x, n.y);
      if (token >= i0 && mine == -INFINITY)  // a NaN counts as one of -inf
#pragma unroll
        for (int j = 0; j < 16; ++j) ahead[0] += v[j] != v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int i = i0 + lp_index<T>(j);
        ahead[0] += v[j] > mine || (i < token && !(v[j] < mine) && (v[j] == mine || mine == -INFINITY));
      }
    }
    if (TOP) {
      high = fmaxf(high, top);
      if (++in_slot == a.per) {
        s_slots[TOP ? slot : 0][TOP ? tid : 0] = high;
        highest = fmaxf(highest, high);
        high = -INFINITY;
        in_slot = 0;
        ++slot;
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
        if (lane == 0 && out) {  // the entry left out so far
          l += f;
          t = fmaf(f, fmaxf(d, -200.0f), t);
        }
      }
      m = mx;
      out = 1;
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
  unsigned long long list = 0;
  if (TOP) {
    if (in_slot) {
      s_slots[TOP ? slot : 0][TOP ? tid : 0] = high;
      highest = fmaxf(highest, high);
    }
    // entries of -inf are none
    float first = lp_sort_values(fmaxf(highest, -INFINITY));
    s_first[TOP ? warp : 0][lane] = first;
    __syncthreads();
    for (int w = 0; w < kLpWarps; ++w)
      if (w != warp) first = lp_both_values(first, s_first[TOP ? w : 0][lane]);
    const float bar = fmaxf(__shfl_sync(0xffffffffu, first, a.top - 1), -FLT_MAX);
    list = lp_likeliest<T>(x, reinterpret_cast<const float (&)[kLpSlots][kLpThreads]>(s_slots),
                           (int64_t)(rank * kLpWarps + warp) * kLpGroup, step, a.per, a.vocab, bar, a.top);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    l += __shfl_xor_sync(0xffffffffu, l, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if (lane == 0) s_part[warp] = LpPart{m, l, t, 2 * before + out};
  if (TOP) s_list[warp][lane] = list;
  __syncthreads();
  if (TOP)
#pragma unroll
    for (int o = kLpWarps / 2; o > 1; o >>= 1) {
      if (warp < o) s_list[warp][lane] = lp_both(s_list[warp][lane], s_list[warp + o][lane]);
      __syncthreads();
    }
  if (ctas > 1) cluster_wait();  // all CTAs of the cluster run
  LpPart p = s_part[0];
  if (warp == 0) {
    for (int w = 1; w < kLpWarps; ++w) p = lp_join(p, s_part[w]);
    if (TOP) list = lp_both(s_list[0][lane], s_list[TOP ? 1 : 0][lane]);
    if (ctas > 1) {
      if (lane == 0) {
        const uint32_t to = mapa_shared(smem_u32(&s_cta[rank]), 0);
        st_cluster_v2(to, __float_as_uint(p.m), __float_as_uint(p.l));
        st_cluster_v2(to + 8, __float_as_uint(p.t), (uint32_t)p.before);
      }
      if (TOP) st_cluster_v2(mapa_shared(smem_u32(&s_cta_list[rank][lane]), 0), (uint32_t)list, (uint32_t)(list >> 32));
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
        if (TOP) list = lp_both(list, s_cta_list[r][lane]);
      }
    }
  }
  if (warp) return;
  const double lse = log1p((double)p.l);
  auto logprob = [&](float v) { return v > -INFINITY ? (float)(((double)v - (double)p.m) - lse) : -INFINITY; };
  if (lane == 0) {
    if (asked >= a.vocab) atomicExch(&g_logprobs_device_error, 1);
    a.logprobs[row] = token >= 0 ? logprob(mine) : asked < 0 ? 0.0f : __uint_as_float(0x7fc00000u);
    a.ranks[row] = token >= 0 ? p.before >> 1 : -1;
    a.entropy[row] = (float)(lse - (double)p.t / (1.0 + (double)p.l));
  }
  if (TOP && lane < a.top) {
    a.top_tokens[(int64_t)row * a.top + lane] = list ? (int64_t)(int)~(uint32_t)list : -1;
    a.top_logprobs[(int64_t)row * a.top + lane] = list ? logprob(lp_value(list)) : -INFINITY;
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
  otf::LogprobArgs a = {logits, ld, tokens, logprobs, entropy, ranks, top_tokens, top_logprobs, (int)n, (int)vocab, (int)top, 1};
  auto* k = dtype == OTF_DTYPE_F32   ? (top ? otf::k_token_logprobs<0, true> : otf::k_token_logprobs<0, false>)
            : dtype == OTF_DTYPE_F16 ? (top ? otf::k_token_logprobs<1, true> : otf::k_token_logprobs<1, false>)
                                     : (top ? otf::k_token_logprobs<2, true> : otf::k_token_logprobs<2, false>);
  // As many CTAs a row as waste least of the last wave; each costs a start and a meeting, as much as
  // 5000 logits, and with a list of the likeliest three times that.
  int ctas = 1;
  double best = 1e30;
  for (int c = 1; c <= otf::kLpCluster; c *= 2) {
    if (c > 1 && (int64_t)(c / 2) * otf::kLpWarps * otf::kLpGroup >= vocab) break;
    const double waves = (double)((n * c + otf::kLpResident - 1) / otf::kLpResident);
    const double cost = waves * ((double)vocab / c + (top ? 15000.0 : 5000.0));
    if (cost < best) {
      best = cost;
      ctas = c;
    }
  }
  const int64_t groups = (vocab + (int64_t)ctas * otf::kLpWarps * otf::kLpGroup - 1) / ((int64_t)ctas * otf::kLpWarps * otf::kLpGroup);
  a.per = (int)((groups + otf::kLpSlots - 1) / otf::kLpSlots);
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
