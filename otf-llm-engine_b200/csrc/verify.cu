// Verification of drafted tokens against the target model's distribution (otf_verify_drafts).
//
// With p = softmax(target / T) and q = softmax(draft / T), token d_j is taken while
// u_j q(d_j) < p(d_j); the first one refused is replaced by a draw from max(p - q, 0), which
// makes every produced token one of the target's distribution; behind K taken ones a draw from p
// follows.  A draw is argmax_i w_i / e_i with e_i ~ Exp(1) given: the index of the smallest of
// independent exponential times of rates w_i, which is distributed as w.  Unlike a search in
// cumulated weights it has no border between neighbours on which a rounding decides.
#include <algorithm>

#include "otf_common.cuh"

namespace otf {

int set_cuda_error(cudaError_t e);   // capi.cu
int check_device();                  // capi.cu
int verify_device_error(int clear);  // read (and optionally clear) the flag below

constexpr int kVerifyMaxDrafts = 32;
constexpr int kVerifySeg = 8192;     // logits of a row that one CTA reads
constexpr int kVerifyThreads = 256;

// Set when a sequence has no token to draw, or an argument on the device is out of range.
__device__ int g_verify_device_error;

// What one CTA found in its part of a row: the largest logit, its first index, and the sum of
// exp((x - max) / T).
struct __align__(16) RowPart {
  float max, sum;
  int at, pad;
};

// exp(d / T) for d <= 0, with c = log2(e) / T in two floats: the exponent is split into its
// nearest whole number and a rest that keeps the product's low bits, so that the relative error
// stays near 2^-22 for small results too (d c alone, rounded, is off by d c 2^-24).
__device__ __forceinline__ float exp_scaled(float d, float c_hi, float c_lo) {
  const float n = fmaxf(rintf(d * c_hi), -160.0f);
  const float r = fmaf(d, c_lo, fmaf(d, c_hi, -n));
  return d > -INFINITY ? ldexpf(exp2f(r), (int)n) : 0.0f;  // 0 for a NaN too
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 0, or from 1e-20 on (log2(e) / T and its product with a difference of logits stay finite).
__host__ __device__ __forceinline__ bool temperature_ok(float T) { return T == 0.0f || (T >= 1e-20f && T <= 1e20f); }

__device__ __forceinline__ float temperature_of(const float* temperatures, float temperature, int b) {
  return temperatures ? temperatures[b] : temperature;
}

// Four consecutive logits of a row, -inf behind its end.  Rows that are not 16-byte aligned are read
// value by value by the same threads, so that a row's sums do not depend on where it lies.
__device__ __forceinline__ float4 logits4(const float* x, int i, int end, bool aligned) {
  if (aligned && i + 4 <= end) return __ldcs(reinterpret_cast<const float4*>(x + i));
  float4 v;
  v.x = i < end ? __ldcs(x + i) : -INFINITY;
  v.y = i + 1 < end ? __ldcs(x + i + 1) : -INFINITY;
  v.z = i + 2 < end ? __ldcs(x + i + 2) : -INFINITY;
  v.w = i + 3 < end ? __ldcs(x + i + 3) : -INFINITY;
  return v;
}

// One pass over the logits: grid (segments, rows), the rows being the batch x (drafts + 1) of the
// target, then the draft's.  A thread holds its 32 values in registers: their maximum, then the
// sum of exponentials under it, joined over the CTA.  Memory-bound, 5 instructions per logit.
__global__ void __launch_bounds__(kVerifyThreads) k_verify_rows(const float* target, int64_t tseq, int64_t ldt,
                                                                const float* draft, int64_t dseq, int64_t ldd,
                                                                const float* temperatures, float temperature,
                                                                const int* counts, int batch, int drafts, int vocab,
                                                                RowPart* parts) {
  constexpr int N = kVerifySeg / (4 * kVerifyThreads), W = kVerifyThreads / 32;
  __shared__ float s_m[W], s_s[W];
  __shared__ int s_i[W];
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.y, trows = batch * (drafts + 1);
  const bool of_target = row < trows;
  const int per = of_target ? drafts + 1 : drafts;
  const int r = of_target ? row : row - trows;
  const int b = r / per, j = r - b * per;
  const float T = temperature_of(temperatures, temperature, b);
  const int count = counts ? counts[b] : drafts;
  if (of_target ? j > count : (j >= count || T == 0.0f)) return;  // a row that nothing asks for
  const float* x = of_target ? target + b * tseq + j * ldt : draft + b * dseq + j * ldd;
  const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const int i0 = blockIdx.x * kVerifySeg + 4 * threadIdx.x;
  float4 v[N];
#pragma unroll
  for (int z = 0; z < N; ++z) v[z] = logits4(x, i0 + z * 4 * kVerifyThreads, vocab, aligned);
  float m = -INFINITY;  // a NaN is never the largest
#pragma unroll
  for (int z = 0; z < N; ++z) m = fmaxf(m, fmaxf(fmaxf(v[z].x, v[z].y), fmaxf(v[z].z, v[z].w)));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float s = 0.0f;
  int at = INT_MAX;
  if (T == 0.0f) {
#pragma unroll
    for (int z = N - 1; z >= 0; --z) {
      const float e[4] = {v[z].x, v[z].y, v[z].z, v[z].w};
#pragma unroll
      for (int w = 3; w >= 0; --w) {
        const int i = i0 + z * 4 * kVerifyThreads + w;
        if (e[w] == m && i < vocab) at = i;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
      const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
      if (m2 > m || (m2 == m && a2 < at)) {
        m = m2;
        at = a2;
      }
    }
    if (lane == 0) {
      s_m[warp] = m;
      s_i[warp] = at;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < W; ++w)
        if (s_m[w] > m || (s_m[w] == m && s_i[w] < at)) {
          m = s_m[w];
          at = s_i[w];
        }
      parts[(int64_t)row * gridDim.x + blockIdx.x] = RowPart{m, 0.0f, at, 0};
    }
    return;
  }
  const float c_hi = (float)(1.4426950408889634 / (double)T);
  const float c_lo = (float)(1.4426950408889634 / (double)T - (double)c_hi);
  auto term = [&](float x, float max) {  // 0 for -inf and NaN (the maximum drops a NaN)
    const float d = x - max;
    return ex2(fmaxf(fmaf(d, c_hi, d * c_lo), -200.0f));
  };
  const float mt = m == -INFINITY ? 0.0f : m;  // nothing but -inf: the sum is 0
#pragma unroll
  for (int z = 0; z < N; ++z)
    if (i0 + z * 4 * kVerifyThreads < vocab)
      s += (term(v[z].x, mt) + term(v[z].y, mt)) + (term(v[z].z, mt) + term(v[z].w, mt));
  auto join = [&](float m2, float s2) {
    const float M = fmaxf(m, m2);
    if (M != -INFINITY) s = s * term(m, M) + s2 * term(m2, M);  // else both are 0
    m = M;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    join(m2, s2);
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_s[warp] = s;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < W; ++w) join(s_m[w], s_s[w]);
    parts[(int64_t)row * gridDim.x + blockIdx.x] = RowPart{m, s, INT_MAX, 0};
  }
}

// A race's leader: the largest w / e and its index, of what the draft leaves of p and of p itself.
struct Leader {
  float best[2];
  int at[2];
  __device__ __forceinline__ void take(int z, float score, int i) {
    if (score > best[z] || (score == best[z] && i < at[z])) {
      best[z] = score;
      at[z] = i;
    }
  }
};

// A cluster of kPickCluster CTAs per sequence.  Every CTA joins the rows' parts and follows the
// drafted tokens (a few hundred numbers); the race over the vocabulary is cut among them, and
// their leaders meet in rank 0 through distributed shared memory.
constexpr int kPickCluster = 8;
constexpr int kPickThreads = 512;

__global__ void __launch_bounds__(kPickThreads) k_verify_pick(const float* target, int64_t tseq, int64_t ldt,
                                                              const float* draft, int64_t dseq, int64_t ldd,
                                                              const int64_t* tokens, int64_t ldtok, const float* uniforms,
                                                              int64_t ldu, const float* noise, int64_t ldn,
                                                              const float* temperatures, float temperature, const int* counts,
                                                              int64_t* out, int* accepted, int batch, int drafts, int vocab,
                                                              const RowPart* parts, int segs) {
  constexpr int W = kPickThreads / 32;
  __shared__ double s_sum[2 * kVerifyMaxDrafts + 1];
  __shared__ float s_max[2 * kVerifyMaxDrafts + 1];
  __shared__ int s_at[kVerifyMaxDrafts + 1];
  __shared__ int s_taken;
  __shared__ __align__(16) Leader s_lead[W];
  __shared__ __align__(16) Leader s_all[kPickCluster];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x / kPickCluster, rank = (int)cluster_ctarank(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float T = temperature_of(temperatures, temperature, b);
  const int count = counts ? counts[b] : drafts;
  if (count < 0 || count > drafts || !temperature_ok(T) || (T > 0.0f && (!noise || (count && !uniforms)))) {
    if (rank) return;  // as all the others do
    for (int j = tid; j <= drafts; j += kPickThreads) out[(int64_t)b * (drafts + 1) + j] = -1;
    if (tid == 0) {
      accepted[b] = 0;
      atomicExch(&g_verify_device_error, 1);
    }
    return;
  }
  if (T == 0.0f && rank) return;  // no race
  const bool drafted = draft != nullptr && T > 0.0f;
  for (int r = warp; r < count + 1 + (drafted ? count : 0); r += W) {
    const int64_t row = r <= count ? (int64_t)b * (drafts + 1) + r
                                   : (int64_t)batch * (drafts + 1) + (int64_t)b * drafts + (r - count - 1);
    const RowPart* p = parts + row * segs;
    float m = -INFINITY;
    int at = INT_MAX;
    for (int i = lane; i < segs; i += 32) {
      const RowPart q = p[i];
      if (q.max > m || (q.max == m && q.at < at)) {
        m = q.max;
        at = q.at;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
      const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
      if (m2 > m || (m2 == m && a2 < at)) {
        m = m2;
        at = a2;
      }
    }
    double s = 0.0;
    if (T > 0.0f)
      for (int i = lane; i < segs; i += 32) {
        const RowPart q = p[i];
        if (q.sum != 0.0f) s += (double)q.sum * exp(((double)q.max - (double)m) / (double)T);
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) {
      const int to = r <= count ? r : drafts + 1 + (r - count - 1);
      s_max[to] = m;
      s_sum[to] = s;
      if (r <= count) s_at[r] = at;
    }
  }
  __syncthreads();
  if (warp == 0) {
    bool take = false;
    if (lane < count) {
      const int64_t d = tokens[b * ldtok + lane];
      if (d < 0 || d >= vocab) {
        if (rank == 0) atomicExch(&g_verify_device_error, 1);
      } else if (T == 0.0f) {
        take = d == s_at[lane];
      } else {
        const double p = exp(((double)target[b * tseq + lane * ldt + d] - (double)s_max[lane]) / (double)T) / s_sum[lane];
        double q = 1.0;
        if (drafted)
          q = exp(((double)draft[b * dseq + lane * ldd + d] - (double)s_max[drafts + 1 + lane]) / (double)T) /
              s_sum[drafts + 1 + lane];
        if (!(q >= 0.0)) q = 0.0;  // a NaN
        take = (double)uniforms[b * ldu + lane] * q < p;
      }
    }
    const unsigned no = ~__ballot_sync(0xffffffffu, take);
    if (lane == 0) s_taken = no ? __ffs((int)no) - 1 : 32;
  }
  __syncthreads();
  const int taken = min(s_taken, count);
  int64_t last = -1;
  if (T == 0.0f) {
    last = s_at[taken] == INT_MAX ? -1 : s_at[taken];
  } else {
    const bool refused = taken < count;
    const float* x = target + b * tseq + taken * ldt;
    const float* y = drafted && refused ? draft + b * dseq + taken * ldd : nullptr;
    const float* e = noise + b * ldn;
    const bool ax = (reinterpret_cast<uintptr_t>(x) & 15) == 0, ay = (reinterpret_cast<uintptr_t>(y) & 15) == 0,
               ae = (reinterpret_cast<uintptr_t>(e) & 15) == 0;
    const float xm = s_max[taken], xi = (float)(1.0 / s_sum[taken]);
    const float ym = y ? s_max[drafts + 1 + taken] : 0.0f, yi = y ? (float)(1.0 / s_sum[drafts + 1 + taken]) : 0.0f;
    const int64_t out_of = refused && !drafted ? tokens[b * ldtok + taken] : -1;
    const float c_hi = (float)(1.4426950408889634 / (double)T);
    const float c_lo = (float)(1.4426950408889634 / (double)T - (double)c_hi);
    Leader lead = {{0.0f, 0.0f}, {INT_MAX, INT_MAX}};
    for (int i = 4 * (rank * kPickThreads + tid); i < vocab; i += 4 * kPickThreads * kPickCluster) {
      const float4 vx = logits4(x, i, vocab, ax), ve = logits4(e, i, vocab, ae);
      float4 vy = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (y) vy = logits4(y, i, vocab, ay);
      const float fx[4] = {vx.x, vx.y, vx.z, vx.w}, fy[4] = {vy.x, vy.y, vy.z, vy.w}, fe[4] = {ve.x, ve.y, ve.z, ve.w};
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        // products that round by themselves: equal rows leave exactly nothing
        const float p = __fmul_rn(exp_scaled(fx[z] - xm, c_hi, c_lo), xi);
        float left = p;
        if (y) left = __fsub_rn(p, __fmul_rn(exp_scaled(fy[z] - ym, c_hi, c_lo), yi));
        if (i + z == out_of) left = 0.0f;
        if (i + z < vocab && p > 0.0f) {
          lead.take(1, p / fe[z], i + z);
          if (left > 0.0f) lead.take(0, left / fe[z], i + z);
        }
      }
    }
#pragma unroll
    for (int z = 0; z < 2; ++z) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float s2 = __shfl_xor_sync(0xffffffffu, lead.best[z], o);
        const int i2 = __shfl_xor_sync(0xffffffffu, lead.at[z], o);
        lead.take(z, s2, i2);
      }
    }
    if (lane == 0) s_lead[warp] = lead;
    __syncthreads();
    cluster_sync_all();  // rank 0 runs
    if (tid == 0) {
      for (int w = 1; w < W; ++w)
        for (int z = 0; z < 2; ++z) lead.take(z, s_lead[w].best[z], s_lead[w].at[z]);
      const uint32_t to = mapa_shared(smem_u32(&s_all[rank]), 0);
      st_cluster_v2(to, __float_as_uint(lead.best[0]), __float_as_uint(lead.best[1]));
      st_cluster_v2(to + 8, (uint32_t)lead.at[0], (uint32_t)lead.at[1]);
    }
    cluster_sync_all();
    if (rank) return;
    for (int z = 0; z < 2 && last < 0; ++z) {
      Leader w = s_all[0];
      for (int k = 1; k < kPickCluster; ++k) w.take(z, s_all[k].best[z], s_all[k].at[z]);
      if (w.at[z] != INT_MAX) last = w.at[z];
    }
  }
  for (int j = tid; j <= drafts; j += kPickThreads)
    out[(int64_t)b * (drafts + 1) + j] = last < 0 || j > taken ? -1 : j < taken ? tokens[b * ldtok + j] : last;
  if (tid == 0) {
    accepted[b] = last < 0 ? 0 : taken;
    if (last < 0) atomicExch(&g_verify_device_error, 1);
  }
}

}  // namespace otf

using otf::check_device;
using otf::set_cuda_error;

int otf::verify_device_error(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, otf::g_verify_device_error, sizeof(int)) != cudaSuccess) {
    set_cuda_error(cudaGetLastError());
    return -1;
  }
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(otf::g_verify_device_error, &z, sizeof(int));
  }
  return v;
}

extern "C" OTF_API int64_t otf_verify_workspace_bytes(int64_t batch, int64_t drafts, int64_t vocab) {
  if (batch <= 0 || drafts < 0 || drafts > otf::kVerifyMaxDrafts || vocab <= 0 || vocab > INT32_MAX / 2) return -1;
  const int64_t segs = (vocab + otf::kVerifySeg - 1) / otf::kVerifySeg;
  return otf::align_up(batch * (2 * drafts + 1) * segs * (int64_t)sizeof(otf::RowPart), 256);
}

extern "C" OTF_API int otf_verify_drafts(const float* target, int64_t target_seq, int64_t ld_target,
                                         const float* draft, int64_t draft_seq, int64_t ld_draft,
                                         const int64_t* tokens, int64_t ld_tokens, const float* uniforms,
                                         int64_t ld_uniforms, const float* noise, int64_t ld_noise,
                                         const float* temperatures, float temperature, const int32_t* counts,
                                         int64_t* out_tokens, int32_t* accepted, int64_t batch, int64_t drafts,
                                         int64_t vocab, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!target || !out_tokens || !accepted || !workspace || batch <= 0 || drafts < 0 || vocab <= 0)
    return OTF_ERR_INVALID;
  if (drafts > otf::kVerifyMaxDrafts || vocab > INT32_MAX / 2 || batch > 65535 / (2 * drafts + 1))
    return OTF_ERR_UNSUPPORTED;
  if (drafts > 0 && (!tokens || ld_tokens < drafts || (uniforms && ld_uniforms < drafts))) return OTF_ERR_INVALID;
  if (ld_target < vocab || target_seq < 0 || (noise && ld_noise < vocab)) return OTF_ERR_INVALID;
  if (draft && drafts > 0 && (ld_draft < vocab || draft_seq < 0)) return OTF_ERR_INVALID;
  if (!temperatures) {
    if (!otf::temperature_ok(temperature)) return OTF_ERR_INVALID;
    if (temperature > 0.0f && (!noise || (drafts > 0 && !uniforms))) return OTF_ERR_INVALID;
  }
  if ((reinterpret_cast<uintptr_t>(workspace) & 255) ||
      workspace_bytes < otf_verify_workspace_bytes(batch, drafts, vocab))
    return OTF_ERR_INVALID;
  int st = check_device();
  if (st != OTF_OK) return st;
  if (drafts == 0) draft = nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int segs = (int)((vocab + otf::kVerifySeg - 1) / otf::kVerifySeg);
  auto* parts = static_cast<otf::RowPart*>(workspace);
  const int64_t rows = batch * (drafts + 1) + (draft ? batch * drafts : 0);
  cudaError_t e = otf::launch_pdl(otf::k_verify_rows, dim3((unsigned)segs, (unsigned)rows), dim3(otf::kVerifyThreads),
                                  0, s, 1u, target, target_seq, ld_target, draft, draft_seq, ld_draft, temperatures,
                                  temperature, counts, (int)batch, (int)drafts, (int)vocab, parts);
  if (e != cudaSuccess) return set_cuda_error(e);
  return set_cuda_error(otf::launch_pdl(otf::k_verify_pick, dim3((unsigned)batch * otf::kPickCluster),
                                        dim3(otf::kPickThreads), 0, s, (unsigned)otf::kPickCluster, target,
                                        target_seq, ld_target, draft, draft_seq, ld_draft, tokens, ld_tokens, uniforms,
                                        ld_uniforms, noise, ld_noise, temperatures, temperature, counts, out_tokens,
                                        accepted, (int)batch, (int)drafts, (int)vocab, (const otf::RowPart*)parts,
                                        segs));
}
