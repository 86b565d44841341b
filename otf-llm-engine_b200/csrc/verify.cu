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
constexpr int kVerifySeg = 1024;     // logits of a row that one warp reads
constexpr int kVerifyThreads = 256;

// Set when a sequence has no token to draw, or an argument on the device is out of range.
__device__ int g_verify_device_error;

// What one warp found in its part of a row: the largest logit, its first index, and the sum of
// exp((x - max) / T).
struct __align__(16) RowPart {
  float max, sum;
  int at, pad;
};

// What the draw of a sequence needs: the row it is of, the rows' maxima and 1 / sums, log2(e) / T.
struct __align__(16) Pick {
  int taken, refused, drafted, out_of;  // taken -1: nothing to draw
  float xm, xi, ym, yi, c_hi, c_lo, pad[2];
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

// The logits' place, and what every kernel asks about a sequence.
struct VerifyArgs {
  const float* target;
  const float* draft;  // or null
  int64_t tseq, ldt, dseq, ldd;
  const int64_t* tokens;
  int64_t ldtok;
  const float* uniforms;
  int64_t ldu;
  const float* noise;
  int64_t ldn;
  const float* temperatures;
  float temperature;
  const int* counts;
  int64_t* out;
  int* accepted;
  int drafts, vocab, segs;
  RowPart* parts;  // [batch][2 drafts + 1: the target's rows, then the draft's][segs]
  Pick* picks;     // [batch]

  __device__ __forceinline__ float temp(int b) const { return temperatures ? temperatures[b] : temperature; }
  __device__ __forceinline__ int count(int b) const { return counts ? counts[b] : drafts; }
  // row r of the count + 1 target rows and then count draft rows that sequence b needs
  __device__ __forceinline__ int rows(int b, int n, float T) const {
    return n < 0 || n > drafts ? 0 : n + 1 + (draft && T > 0.0f ? n : 0);
  }
  __device__ __forceinline__ const float* row(int b, int n, int r) const {
    return r <= n ? target + b * tseq + r * ldt : draft + b * dseq + (r - n - 1) * ldd;
  }
  __device__ __forceinline__ int64_t part(int b, int n, int r) const {
    return ((int64_t)b * (2 * drafts + 1) + (r <= n ? r : drafts + r - n)) * segs;
  }
};

// One pass over the logits: grid (blocks of 8 segments, row groups, batch), a warp per segment.  A lane
// holds its 32 values of a row's segment in registers: the warp's maximum, then the sum of
// exponentials under it.  Memory-bound, 7 instructions per logit; the warps of a CTA never meet.  A
// CTA goes through its group's rows, so that rows that a sequence with fewer drafted tokens does
// not have cost nothing.
__global__ void __launch_bounds__(kVerifyThreads) k_verify_rows(VerifyArgs a) {
  constexpr int N = kVerifySeg / 128;
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.z, lane = threadIdx.x & 31, seg = blockIdx.x * (kVerifyThreads / 32) + (threadIdx.x >> 5);
  if (seg >= a.segs) return;
  const float T = a.temp(b);
  const int n = a.count(b), rows = a.rows(b, n, T);
  const int i0 = seg * kVerifySeg + 4 * lane;
  const float c_hi = (float)(1.4426950408889634 / (double)T);
  const float c_lo = (float)(1.4426950408889634 / (double)T - (double)c_hi);
  for (int r = blockIdx.y; r < rows; r += gridDim.y) {
    const float* x = a.row(b, n, r);
    const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    float4 v[N];
#pragma unroll
    for (int z = 0; z < N; ++z) v[z] = logits4(x, i0 + z * 128, a.vocab, aligned);
    float m = -INFINITY;  // a NaN is never the largest
#pragma unroll
    for (int z = 0; z < N; ++z) m = fmaxf(m, fmaxf(fmaxf(v[z].x, v[z].y), fmaxf(v[z].z, v[z].w)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float s = 0.0f;
    int at = INT_MAX;
    if (T == 0.0f) {  // the first of the largest
#pragma unroll
      for (int z = N - 1; z >= 0; --z) {
        const float e[4] = {v[z].x, v[z].y, v[z].z, v[z].w};
#pragma unroll
        for (int w = 3; w >= 0; --w)
          if (e[w] == m && i0 + z * 128 + w < a.vocab) at = i0 + z * 128 + w;
      }
      at = __reduce_min_sync(0xffffffffu, at);
    } else {
      const float mt = m == -INFINITY ? 0.0f : m;  // nothing but -inf: the sum is 0
      auto term = [&](float x) {  // 0 for -inf and NaN (the maximum drops a NaN)
        const float d = x - mt;
        return ex2(fmaxf(fmaf(d, c_hi, d * c_lo), -200.0f));
      };
#pragma unroll
      for (int z = 0; z < N; ++z) s += (term(v[z].x) + term(v[z].y)) + (term(v[z].z) + term(v[z].w));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    if (lane == 0) a.parts[a.part(b, n, r) + seg] = RowPart{m, s, at, 0};
  }
}

__device__ __forceinline__ void write_tokens(const VerifyArgs& a, int b, int taken, int64_t last, int tid, int threads) {
  for (int j = tid; j <= a.drafts; j += threads)
    a.out[(int64_t)b * (a.drafts + 1) + j] = last < 0 || j > taken ? -1 : j < taken ? a.tokens[b * a.ldtok + j] : last;
  if (tid == 0) {
    a.accepted[b] = last < 0 ? 0 : taken;
    if (last < 0) atomicExch(&g_verify_device_error, 1);
  }
}

// A CTA per sequence: the rows' parts joined (a warp per row), the drafted tokens followed, and what
// the draw needs left in picks[b]; with temperature 0 that is all.  Latency-bound: the tokens and
// their logits are requested before the parts are joined.
constexpr int kPickThreads = 512;

__global__ void __launch_bounds__(kPickThreads) k_verify_pick(VerifyArgs a) {
  __shared__ double s_sum[2 * kVerifyMaxDrafts + 1];
  __shared__ float s_max[2 * kVerifyMaxDrafts + 1];
  __shared__ int s_at[kVerifyMaxDrafts + 1];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float T = a.temp(b);
  const int n = a.count(b), rows = a.rows(b, n, T);
  if (rows == 0 || !temperature_ok(T) || (T > 0.0f && (!a.noise || (n && !a.uniforms)))) {
    if (tid == 0) a.picks[b].taken = -1;
    write_tokens(a, b, 0, -1, tid, kPickThreads);
    return;
  }
  const bool drafted = rows > n + 1;
  float xd = 0.0f, yd = 0.0f, u = 0.0f;
  int64_t d = -1;
  if (warp == 0 && lane < n) {
    d = a.tokens[b * a.ldtok + lane];
    if (d >= 0 && d < a.vocab && T > 0.0f) {
      xd = a.target[b * a.tseq + lane * a.ldt + d];
      if (drafted) yd = a.draft[b * a.dseq + lane * a.ldd + d];
      u = a.uniforms[b * a.ldu + lane];
    }
  }
  const double c = T > 0.0f ? 1.4426950408889634 / (double)T : 0.0;
  const float c_hi = (float)c, c_lo = (float)(c - (double)c_hi);
  for (int r = warp; r < rows; r += kPickThreads / 32) {
    const RowPart* p = a.parts + a.part(b, n, r);
    constexpr int U = 4;  // a lane's parts of 128 segments, requested together
    float m = -INFINITY;
    int at = INT_MAX;
    RowPart q[U];
#pragma unroll
    for (int k = 0; k < U; ++k) q[k] = lane + 32 * k < a.segs ? p[lane + 32 * k] : RowPart{-INFINITY, 0.0f, INT_MAX, 0};
    auto top = [&](const RowPart& x) {
      if (x.max > m || (x.max == m && x.at < at)) {
        m = x.max;
        at = x.at;
      }
    };
#pragma unroll
    for (int k = 0; k < U; ++k) top(q[k]);
    for (int i = lane + 32 * U; i < a.segs; i += 32) top(p[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
      const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
      top(RowPart{m2, 0.0f, a2, 0});
    }
    double s = 0.0;
    if (T > 0.0f) {
      auto add = [&](const RowPart& x) {
        if (x.sum != 0.0f) s += (double)(x.sum * exp_scaled(x.max - m, c_hi, c_lo));
      };
#pragma unroll
      for (int k = 0; k < U; ++k) add(q[k]);
      for (int i = lane + 32 * U; i < a.segs; i += 32) add(p[i]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    if (lane == 0) {
      const int to = r <= n ? r : a.drafts + r - n;
      s_max[to] = m;
      s_sum[to] = s;
      if (r <= n) s_at[r] = at;
    }
  }
  __syncthreads();
  if (warp) return;
  bool take = false;
  if (lane < n) {
    if (d < 0 || d >= a.vocab) {
      atomicExch(&g_verify_device_error, 1);
    } else if (T == 0.0f) {
      take = d == s_at[lane];
    } else {
      const double p = exp(((double)xd - (double)s_max[lane]) / (double)T) / s_sum[lane];
      double q = 1.0;
      if (drafted) {
        q = exp(((double)yd - (double)s_max[a.drafts + 1 + lane]) / (double)T) / s_sum[a.drafts + 1 + lane];
        if (!(q >= 0.0)) q = 0.0;  // a NaN
      }
      take = (double)u * q < p;
    }
  }
  const unsigned no = ~__ballot_sync(0xffffffffu, take);
  const int taken = no ? min(__ffs((int)no) - 1, n) : n;
  if (T == 0.0f) {
    write_tokens(a, b, taken, s_at[taken] == INT_MAX ? -1 : s_at[taken], lane, 32);
    if (lane == 0) a.picks[b].taken = -1;
    return;
  }
  const bool refused = taken < n;
  const int64_t out_of = __shfl_sync(0xffffffffu, d, min(taken, 31));
  if (lane == 0) {
    Pick k;
    k.taken = taken;
    k.refused = refused;
    k.drafted = drafted && refused;
    k.out_of = refused && !drafted && out_of >= 0 && out_of < a.vocab ? (int)out_of : -1;
    k.xm = s_max[taken];
    k.xi = (float)(1.0 / s_sum[taken]);
    k.ym = k.drafted ? s_max[a.drafts + 1 + taken] : 0.0f;
    k.yi = k.drafted ? (float)(1.0 / s_sum[a.drafts + 1 + taken]) : 0.0f;
    k.c_hi = c_hi;
    k.c_lo = c_lo;
    a.picks[b] = k;
  }
}

// The leader of the race: the largest w / e, and its index.
struct __align__(8) Leader {
  float best;
  int at;
  __device__ __forceinline__ void take(float score, int i) {
    if (score > best || (score == best && i < at)) {
      best = score;
      at = i;
    }
  }
};

// The draw: a cluster of `ctas` CTAs per sequence, the vocabulary cut among them, their leaders
// exchanged through distributed shared memory.  An entry is weighed with the hardware's exponential
// first, whose error is far below the margin 2^-16; only what may beat its warp's leader by then is
// computed with care (some 10 entries of a warp), so the loop stays near 25 instructions per entry.
// A thread requests kRaceBatch pieces of each row before it uses them.
constexpr int kRaceCluster = 8;
constexpr int kRaceThreads = 256;
constexpr int kRaceBatch = 4;

__global__ void __launch_bounds__(kRaceThreads, 2) k_verify_race(VerifyArgs a, int ctas) {
  constexpr int W = kRaceThreads / 32, U = kRaceBatch;
  __shared__ Leader s_lead[W];
  __shared__ Leader s_all[2][kRaceCluster];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x / ctas, rank = blockIdx.x - b * ctas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Pick k = a.picks[b];
  if (k.taken < 0) return;  // done already; the whole cluster returns
  cluster_arrive_relaxed();
  const float* x = a.target + b * a.tseq + k.taken * a.ldt;
  const float* e = a.noise + b * a.ldn;
  const bool ax = (reinterpret_cast<uintptr_t>(x) & 15) == 0, ae = (reinterpret_cast<uintptr_t>(e) & 15) == 0;
  const float* y = k.drafted ? a.draft + b * a.dseq + k.taken * a.ldd : nullptr;
  int out_of = k.out_of;
  int64_t last = -1;
  const int step = 4 * kRaceThreads * ctas;
  for (int pass = 0;; ++pass) {  // a second one where nothing of p - q is left: p itself
    const bool ay = (reinterpret_cast<uintptr_t>(y) & 15) == 0;
    Leader lead = {0.0f, INT_MAX};
    float bar = 0.0f;  // the warp's leader
    for (int i0 = 4 * (rank * kRaceThreads + warp * 32); i0 < a.vocab; i0 += U * step) {
      float4 vx[U], ve[U], vy[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int i = min(i0 + j * step, a.vocab) + 4 * lane;  // behind the end: -inf without a read
        vx[j] = logits4(x, i, a.vocab, ax);
        ve[j] = logits4(e, i, a.vocab, ae);
        vy[j] = y ? logits4(y, i, a.vocab, ay) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int i = min(i0 + j * step, a.vocab) + 4 * lane;
        const float fx[4] = {vx[j].x, vx[j].y, vx[j].z, vx[j].w}, fy[4] = {vy[j].x, vy[j].y, vy[j].z, vy[j].w},
                    fe[4] = {ve[j].x, ve[j].y, ve[j].z, ve[j].w};
        bool may[4], any = false;
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const float dx = fx[z] - k.xm, dy = fy[z] - k.ym;
          const float p = ex2(fmaxf(fmaf(dx, k.c_hi, dx * k.c_lo), -200.0f)) * k.xi;
          float q = 0.0f;
          if (y) q = ex2(fmaxf(fmaf(dy, k.c_hi, dy * k.c_lo), -200.0f)) * k.yi;
          may[z] = fmaf(p + q, 0x1p-16f, p - q) > bar * fe[z] && i + z != out_of && i + z < a.vocab;
          any |= may[z];
        }
        if (__any_sync(0xffffffffu, any)) {
#pragma unroll
          for (int z = 0; z < 4; ++z)
            if (may[z]) {
              // products that round by themselves: equal rows leave exactly nothing
              float w = __fmul_rn(exp_scaled(fx[z] - k.xm, k.c_hi, k.c_lo), k.xi);
              if (y) w = __fsub_rn(w, __fmul_rn(exp_scaled(fy[z] - k.ym, k.c_hi, k.c_lo), k.yi));
              if (w > 0.0f) lead.take(w / fe[z], i + z);
            }
          bar = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(lead.best)));
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float s2 = __shfl_xor_sync(0xffffffffu, lead.best, o);
      const int i2 = __shfl_xor_sync(0xffffffffu, lead.at, o);
      lead.take(s2, i2);
    }
    if (lane == 0) s_lead[warp] = lead;
    __syncthreads();
    if (pass == 0) cluster_wait();  // all CTAs of the cluster run
    if (tid < ctas) {
      for (int w = 0; w < W; ++w) lead.take(s_lead[w].best, s_lead[w].at);
      st_cluster_v2(mapa_shared(smem_u32(&s_all[pass][rank]), tid), __float_as_uint(lead.best), (uint32_t)lead.at);
    }
    __syncwarp();
    cluster_sync_all();
    Leader all = s_all[pass][0];
    for (int r = 1; r < ctas; ++r) all.take(s_all[pass][r].best, s_all[pass][r].at);
    if (all.at != INT_MAX) last = all.at;
    if (last >= 0 || pass == 1 || !k.refused) break;
    y = nullptr;
    out_of = -1;
  }
  if (rank == 0) write_tokens(a, b, k.taken, last, tid, kRaceThreads);
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
  return otf::align_up(batch * (int64_t)sizeof(otf::Pick), 256) +
         otf::align_up(batch * (2 * drafts + 1) * segs * (int64_t)sizeof(otf::RowPart), 256);
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
  if (drafts > otf::kVerifyMaxDrafts || vocab > INT32_MAX / 2 || batch > 65535)
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int segs = (int)((vocab + otf::kVerifySeg - 1) / otf::kVerifySeg);
  char* w = static_cast<char*>(workspace);
  const otf::VerifyArgs a = {target,
                             drafts ? draft : nullptr,
                             target_seq,
                             ld_target,
                             draft_seq,
                             ld_draft,
                             tokens,
                             ld_tokens,
                             uniforms,
                             ld_uniforms,
                             noise,
                             ld_noise,
                             temperatures,
                             temperature,
                             counts,
                             out_tokens,
                             accepted,
                             (int)drafts,
                             (int)vocab,
                             segs,
                             reinterpret_cast<otf::RowPart*>(w + otf::align_up(batch * (int64_t)sizeof(otf::Pick), 256)),
                             reinterpret_cast<otf::Pick*>(w)};
  // row groups: one per row while all of their CTAs fit the GPU at once, else 4
  const int64_t rows = drafts + 1 + (a.draft ? drafts : 0);
  const int64_t blocks = (segs + 7) / 8;
  const int64_t groups = std::min<int64_t>(rows, batch * blocks * rows <= 4 * 148 ? rows : 4);
  cudaError_t e = otf::launch_pdl(otf::k_verify_rows, dim3((unsigned)blocks, (unsigned)groups, (unsigned)batch),
                                  dim3(otf::kVerifyThreads), 0, s, 1u, a);
  if (e != cudaSuccess) return set_cuda_error(e);
  e = otf::launch_pdl(otf::k_verify_pick, dim3((unsigned)batch), dim3(otf::kPickThreads), 0, s, 1u, a);
  if (e != cudaSuccess || (!temperatures && temperature == 0.0f)) return set_cuda_error(e);
  // CTAs per sequence: as many as all run at once, two on an SM
  int ctas = otf::kRaceCluster;
  while (ctas > 1 && batch * ctas > 2 * 148) ctas /= 2;
  return set_cuda_error(otf::launch_pdl(otf::k_verify_race, dim3((unsigned)(batch * ctas)), dim3(otf::kRaceThreads), 0, s,
                                        (unsigned)ctas, a, ctas));
}
