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
  return d == -INFINITY ? 0.0f : ldexpf(exp2f(r), (int)n);
}

// 0, or from 1e-20 on (log2(e) / T and its product with a difference of logits stay finite).
__host__ __device__ __forceinline__ bool temperature_ok(float T) { return T == 0.0f || (T >= 1e-20f && T <= 1e20f); }

__device__ __forceinline__ float temperature_of(const float* temperatures, float temperature, int b) {
  return temperatures ? temperatures[b] : temperature;
}

// Grid (segments, rows): rows are the batch x (drafts + 1) of the target, then the draft's.
__global__ void __launch_bounds__(kVerifyThreads) k_verify_rows(const float* target, int64_t tseq, int64_t ldt,
                                                                const float* draft, int64_t dseq, int64_t ldd,
                                                                const float* temperatures, float temperature,
                                                                const int* counts, int batch, int drafts, int vocab,
                                                                RowPart* parts) {
  __shared__ float s_m[8], s_s[8];
  __shared__ int s_i[8];
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
  const int i0 = blockIdx.x * kVerifySeg, i1 = min(vocab, i0 + kVerifySeg);
  const float c_hi = (float)(1.4426950408889634 / (double)T);
  const float c_lo = (float)(1.4426950408889634 / (double)T - (double)c_hi);
  float m = -INFINITY, s = 0.0f;
  int at = INT_MAX;
  for (int i = i0 + threadIdx.x; i < i1; i += kVerifyThreads)
    if (x[i] > m || (at == INT_MAX && x[i] == x[i])) {  // a NaN is never the largest
      m = x[i];
      at = i;
    }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto better = [](float m1, int i1_, float m2, int i2_) { return m1 > m2 || (m1 == m2 && i1_ < i2_); };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
    const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
    if (better(m2, a2, m, at)) {
      m = m2;
      at = a2;
    }
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_i[warp] = at;
  }
  __syncthreads();
  for (int w = 0; w < 8; ++w)
    if (better(s_m[w], s_i[w], m, at)) {
      m = s_m[w];
      at = s_i[w];
    }
  if (T != 0.0f && m != -INFINITY)
    for (int i = i0 + threadIdx.x; i < i1; i += kVerifyThreads) s += exp_scaled(x[i] - m, c_hi, c_lo);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) s_s[warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0f;
    for (int w = 0; w < 8; ++w) s += s_s[w];
    parts[(int64_t)row * gridDim.x + blockIdx.x] = RowPart{m, s, at, 0};
  }
}

// One CTA per sequence: the rows' parts joined, the drafted tokens taken or refused, the draw.
__global__ void __launch_bounds__(1024) k_verify_pick(const float* target, int64_t tseq, int64_t ldt,
                                                      const float* draft, int64_t dseq, int64_t ldd,
                                                      const int64_t* tokens, int64_t ldtok, const float* uniforms,
                                                      int64_t ldu, const float* noise, int64_t ldn,
                                                      const float* temperatures, float temperature, const int* counts,
                                                      int64_t* out, int* accepted, int batch, int drafts, int vocab,
                                                      const RowPart* parts, int segs) {
  __shared__ double s_max[2 * kVerifyMaxDrafts + 1], s_sum[2 * kVerifyMaxDrafts + 1];
  __shared__ int s_at[kVerifyMaxDrafts + 1];
  __shared__ int s_taken;
  __shared__ float s_best[2][32];
  __shared__ int s_idx[2][32];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float T = temperature_of(temperatures, temperature, b);
  const int count = counts ? counts[b] : drafts;
  if (count < 0 || count > drafts || !temperature_ok(T) || (T > 0.0f && (!noise || (count && !uniforms)))) {
    for (int j = tid; j <= drafts; j += blockDim.x) out[(int64_t)b * (drafts + 1) + j] = -1;
    if (tid == 0) {
      accepted[b] = 0;
      atomicExch(&g_verify_device_error, 1);
    }
    return;
  }
  const bool drafted = draft != nullptr && T > 0.0f;
  for (int r = warp; r < count + 1 + (drafted ? count : 0); r += 32) {
    const int64_t row = r <= count ? (int64_t)b * (drafts + 1) + r
                                   : (int64_t)batch * (drafts + 1) + (int64_t)b * drafts + (r - count - 1);
    const RowPart* p = parts + row * segs;
    float m = -INFINITY;
    int at = INT_MAX;
    for (int i = lane; i < segs; i += 32)
      if (p[i].max > m || (p[i].max == m && p[i].at < at)) {
        m = p[i].max;
        at = p[i].at;
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
      for (int i = lane; i < segs; i += 32)
        if (p[i].max != -INFINITY) s += (double)p[i].sum * exp(((double)p[i].max - (double)m) / (double)T);
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
        atomicExch(&g_verify_device_error, 1);
      } else if (T == 0.0f) {
        take = d == s_at[lane];
      } else {
        const double p = exp(((double)target[b * tseq + lane * ldt + d] - s_max[lane]) / (double)T) / s_sum[lane];
        double q = 1.0;
        if (drafted)
          q = exp(((double)draft[b * dseq + lane * ldd + d] - s_max[drafts + 1 + lane]) / (double)T) /
              s_sum[drafts + 1 + lane];
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
    const float xm = (float)s_max[taken], xi = (float)(1.0 / s_sum[taken]);
    const float ym = y ? (float)s_max[drafts + 1 + taken] : 0.0f, yi = y ? (float)(1.0 / s_sum[drafts + 1 + taken]) : 0.0f;
    const int64_t out_of = refused && !drafted ? tokens[b * ldtok + taken] : -1;
    const float c_hi = (float)(1.4426950408889634 / (double)T);
    const float c_lo = (float)(1.4426950408889634 / (double)T - (double)c_hi);
    // the race of what is left of p, and of p itself for where nothing is left
    float best[2] = {0.0f, 0.0f};
    int idx[2] = {INT_MAX, INT_MAX};
    for (int i = tid; i < vocab; i += blockDim.x) {
      const float e = noise[b * ldn + i];
      // products that round by themselves: equal rows leave exactly nothing
      const float p = __fmul_rn(exp_scaled(x[i] - xm, c_hi, c_lo), xi);
      float left = p;
      if (y) left = __fsub_rn(p, __fmul_rn(exp_scaled(y[i] - ym, c_hi, c_lo), yi));
      if (i == out_of) left = 0.0f;
      const float w[2] = {left, p};
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const float sc = w[z] > 0.0f ? w[z] / e : 0.0f;
        if (sc > best[z]) {
          best[z] = sc;
          idx[z] = i;
        }
      }
    }
#pragma unroll
    for (int z = 0; z < 2; ++z) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float s2 = __shfl_xor_sync(0xffffffffu, best[z], o);
        const int i2 = __shfl_xor_sync(0xffffffffu, idx[z], o);
        if (s2 > best[z] || (s2 == best[z] && i2 < idx[z])) {
          best[z] = s2;
          idx[z] = i2;
        }
      }
      if (lane == 0) {
        s_best[z][warp] = best[z];
        s_idx[z][warp] = idx[z];
      }
    }
    __syncthreads();
    for (int z = 0; z < 2 && last < 0; ++z) {
      float bs = 0.0f;
      int bi = INT_MAX;
      for (int w = 0; w < 32; ++w)
        if (s_best[z][w] > bs || (s_best[z][w] == bs && s_idx[z][w] < bi)) {
          bs = s_best[z][w];
          bi = s_idx[z][w];
        }
      if (bi != INT_MAX) last = bi;
    }
  }
  for (int j = tid; j <= drafts; j += blockDim.x)
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
  return set_cuda_error(otf::launch_pdl(otf::k_verify_pick, dim3((unsigned)batch), dim3(1024), 0, s, 1u, target,
                                        target_seq, ld_target, draft, draft_seq, ld_draft, tokens, ld_tokens, uniforms,
                                        ld_uniforms, noise, ld_noise, temperatures, temperature, counts, out_tokens,
                                        accepted, (int)batch, (int)drafts, (int)vocab, (const otf::RowPart*)parts,
                                        segs));
}
