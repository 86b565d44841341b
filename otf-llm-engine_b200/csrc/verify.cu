// Verification of drafted tokens against the target model's distribution (otf_verify_drafts).
//
// With p = softmax(target / T) and q = softmax(draft / T), token d_j is taken while
// u_j q(d_j) < p(d_j); the first one refused is replaced by a draw from max(p - q, 0), which
// makes every produced token one of the target's distribution; behind K taken ones a draw from p
// follows.  A draw is argmax_i w_i / e_i with e_i ~ Exp(1) given: the index of the smallest of
// independent exponential times of rates w_i, which is distributed as w.  Unlike a search in
// cumulated weights it has no border between neighbours on which a rounding decides.
//
// Three steps: (1) every row's maximum, its first index and the sum of exponentials under it, in one
// pass over the logits (K + 1 rows of the target's, K of the draft's); (2) the drafted tokens, a few
// hundred numbers per sequence; (3) the race over the one or two rows that it needs.  Memory-bound:
// the rows are read once, the drawn ones a second time, from L2 where they still are.
//
// Few logits take one launch, k_verify: a cluster of CTAs per sequence, the vocabulary cut among them,
// the steps' results exchanged through distributed shared memory.  Many take three, whose grids
// fill the GPU in every step whatever the sequences' drafts are: k_verify_rows, k_verify_pick,
// k_verify_race.  What a step computes is shared.
#include <cfloat>

#include <algorithm>

#include "logits.cuh"
#include "paged.cuh"

namespace otf {

int set_cuda_error(cudaError_t e);   // capi.cu
int check_device();                  // capi.cu
int verify_device_error(int clear);  // read (and optionally clear) the flag below

constexpr int kVerifyMaxDrafts = 32;
constexpr int kVerifyMaxRows = 2 * kVerifyMaxDrafts + 1;
constexpr int kVerifySeg = 1024;     // logits that a warp holds at once, 32 a lane
constexpr int kVerifyThreads = 256;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyCluster = 16;   // CTAs of a sequence at most (k_verify)
constexpr int kPickThreads = 1024;   // of k_verify_pick at most
constexpr int kRaceResident = 148 * 4;  // CTAs of k_verify_race that run at once
constexpr int kRaceLeast = 1024;     // entries of a CTA at least (k_verify_race)
// One launch is taken up to 6M logits in all rows and 512K of a sequence (1.5M of at most kVerifyFew
// sequences); its CTAs then have 32 warps where a CTA's slice of the rows is large (kVerifyLarge
// logits), else 8.  Measured, eager calls one after another, one launch against three: 16 sequences x 5
// rows of 32000 (2.4M) 13.8 us against 20.4, x 9 rows (4.4M) 18.8 against 21.0, 32 x 9 (8.8M) 22.5 against
// 22.0; 8 x 5 rows of 128256 (641K each) 22.5 against 21.2; 4 x 11 (1.4M each) 18.8 against 21.2, 4 x 17
// (2.2M) 23.7 against 21.2, one of 33 (4.2M) 31.9 against 21.3.  32 warps against 8: one sequence, 9 rows of
// 128256, 17.4 us against 22.5; 8 x 5 rows of 32000 19.0 against 14.1.
constexpr int kVerifyFew = 4;
constexpr int64_t kVerifyLarge = 1 << 14;

// Set when a sequence has no token to draw, or an argument on the device is out of range.
__device__ int g_verify_device_error;

// What is known of a row, or of a part of it: the largest logit, its first index, and the sum of
// exp((x - max) / T).
struct __align__(16) RowPart {
  float max, sum;
  int at, pad;
};

// What the draw of a sequence needs: the row it is of, the rows' maxima and 1 / sums.
struct __align__(16) Pick {
  int taken, refused, drafted, out_of;  // taken -1: nothing to draw
  float xm, xi, ym, yi;
  unsigned long long lead;  // k_verify_race: the leader so far (see packed), 0 at first
  int done, pad;            // and its CTAs that are done
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
  int drafts, vocab;
  int slice;       // k_verify: a CTA's part of the vocabulary, a multiple of 4
  int segs;        // k_verify_rows: segments of a row
  RowPart* parts;  // [batch][2 drafts + 1: the target's rows, then the draft's][segs]
  Pick* picks;     // [batch]
};

// A sequence as the kernels see it.
struct Sequence {
  const VerifyArgs& a;
  int b, n;        // n: its drafted tokens
  float T, c_hi, c_lo;  // temperature, log2(e) / T in two floats
  bool ok, drafted;     // drafted: the draft's logits count

  __device__ __forceinline__ Sequence(const VerifyArgs& args, int seq) : a(args), b(seq) {
    T = a.temperatures ? a.temperatures[b] : a.temperature;
    n = a.counts ? a.counts[b] : a.drafts;
    ok = n >= 0 && n <= a.drafts && temperature_ok(T) && (T == 0.0f || (a.noise && (n == 0 || a.uniforms)));
    drafted = ok && a.draft && T > 0.0f && n > 0;
    const double c = T > 0.0f ? 1.4426950408889634 / (double)T : 0.0;
    c_hi = (float)c;
    c_lo = (float)(c - (double)c_hi);
  }
  // rows: the target's 0 .. n, then the draft's
  __device__ __forceinline__ int rows() const { return !ok ? 0 : n + 1 + (drafted ? n : 0); }
  __device__ __forceinline__ const float* row(int r) const {
    return r <= n ? a.target + b * a.tseq + r * a.ldt : a.draft + b * a.dseq + (r - n - 1) * a.ldd;
  }
  __device__ __forceinline__ RowPart* part(int r) const {
    return a.parts + ((int64_t)b * (2 * a.drafts + 1) + (r <= n ? r : a.drafts + r - n)) * a.segs;
  }
};

__device__ __forceinline__ void write_tokens(const Sequence& q, int taken, int64_t last, int tid, int threads) {
  const VerifyArgs& a = q.a;
  for (int j = tid; j <= a.drafts; j += threads)
    a.out[(int64_t)q.b * (a.drafts + 1) + j] =
        last < 0 || j > taken ? -1 : j < taken ? a.tokens[q.b * a.ldtok + j] : last;
  if (tid == 0) {
    a.accepted[q.b] = last < 0 ? 0 : taken;
    if (last < 0) atomicExch(&g_verify_device_error, 1);
  }
}

// Step 1 for a warp: the 1024 logits of a row from i0 on (none behind `end`), 32 in each lane: their
// maximum, then the sum of exponentials under it, 7 instructions per logit.  A NaN counts as -inf.
__device__ __forceinline__ RowPart read_segment(const Sequence& q, const float* x, int i0, int end) {
  constexpr int N = kVerifySeg / 128;
  const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  i0 += 4 * (threadIdx.x & 31);
  float4 v[N];
#pragma unroll
  for (int z = 0; z < N; ++z) v[z] = logits4(x, i0 + z * 128, end, aligned);
  float m = -INFINITY;
#pragma unroll
  for (int z = 0; z < N; ++z) m = fmaxf(m, fmaxf(fmaxf(v[z].x, v[z].y), fmaxf(v[z].z, v[z].w)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float s = 0.0f;
  int at = INT_MAX;
  if (q.T == 0.0f) {  // the first of the largest, none among -inf alone
#pragma unroll
    for (int z = N - 1; z >= 0; --z) {
      const float e[4] = {v[z].x, v[z].y, v[z].z, v[z].w};
#pragma unroll
      for (int w = 3; w >= 0; --w)
        if (e[w] == m && m > -INFINITY) at = i0 + z * 128 + w;
    }
    at = __reduce_min_sync(0xffffffffu, at);
  } else {
    const float mt = m == -INFINITY ? 0.0f : m;  // nothing but -inf: the sum is 0
    // 0 for -inf and NaN.  Bounded before the products: the lowest finite logit times a negative c_lo
    // of a small T is +inf.
    const float low = -138.629436f * q.T;  // its exponential is 2^-200, 0 in fp32
    auto term = [&](float x) {
      const float d = fmaxf(x - mt, low);
      return ex2(fmaf(d, q.c_hi, d * q.c_lo));
    };
#pragma unroll
    for (int z = 0; z < N; ++z) s += (term(v[z].x) + term(v[z].y)) + (term(v[z].z) + term(v[z].w));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  }
  return RowPart{m, s, at, 0};
}

__device__ __forceinline__ RowPart no_part() { return RowPart{-INFINITY, 0.0f, INT_MAX, 0}; }

// Two parts of a row as one.
__device__ __forceinline__ RowPart join(const Sequence& q, const RowPart& x, const RowPart& y) {
  RowPart z = x.max > y.max || (x.max == y.max && x.at < y.at) ? x : y;
  z.sum = (x.sum != 0.0f ? x.sum * exp_scaled(x.max - z.max, q.c_hi, q.c_lo) : 0.0f) +
          (y.sum != 0.0f ? y.sum * exp_scaled(y.max - z.max, q.c_hi, q.c_lo) : 0.0f);
  return z;
}
// The parts that `width` neighbouring lanes (a power of two) hold, joined for all of them.
__device__ __forceinline__ RowPart join_lanes(const Sequence& q, const RowPart& p, int width) {
  float m = p.max;
  int at = p.at;
  for (int o = 1; o < width; o <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
    const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
    if (m2 > m || (m2 == m && a2 < at)) {
      m = m2;
      at = a2;
    }
  }
  float s = p.sum != 0.0f ? p.sum * exp_scaled(p.max - m, q.c_hi, q.c_lo) : 0.0f;
  for (int o = 1; o < width; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return RowPart{m, s, at, 0};
}

// Step 2.  A warp's lane j asks for drafted token j and its logits...
struct Drafted {
  int64_t token;
  float x, y, u;
};
__device__ __forceinline__ Drafted ask_drafted(const Sequence& q, int j) {
  const VerifyArgs& a = q.a;
  Drafted d = {-1, 0.0f, 0.0f, 0.0f};
  if (j < q.n) {
    d.token = a.tokens[q.b * a.ldtok + j];
    if (d.token >= 0 && d.token < a.vocab && q.T > 0.0f) {
      d.x = a.target[q.b * a.tseq + j * a.ldt + d.token];
      if (q.drafted) d.y = a.draft[q.b * a.dseq + j * a.ldd + d.token];
      d.u = a.uniforms[q.b * a.ldu + j];
    }
  }
  return d;
}
// ... and follows them, once `row` holds all rows: how many are taken, and what the draw needs.
__device__ __forceinline__ Pick follow(const Sequence& q, const Drafted& d, const RowPart* row, bool report) {
  const int j = threadIdx.x & 31, n = q.n;
  bool take = false;
  if (j < n) {
    if (d.token < 0 || d.token >= q.a.vocab) {
      if (report) atomicExch(&g_verify_device_error, 1);
    } else if (q.T == 0.0f) {
      take = d.token == row[j].at;
    } else {
      const double p = exp(((double)d.x - (double)row[j].max) / (double)q.T) / (double)row[j].sum;
      double r = 1.0;
      if (q.drafted) {
        r = exp(((double)d.y - (double)row[n + 1 + j].max) / (double)q.T) / (double)row[n + 1 + j].sum;
        if (!(r >= 0.0)) r = 0.0;  // a NaN
      }
      take = (double)d.u * r < p;
    }
  }
  const unsigned no = ~__ballot_sync(0xffffffffu, take);
  Pick k;
  k.taken = no ? min(__ffs((int)no) - 1, n) : n;
  k.refused = k.taken < n;
  k.drafted = q.drafted && k.refused;
  const int64_t token = __shfl_sync(0xffffffffu, d.token, min(k.taken, 31));
  k.out_of = k.refused && !q.drafted && token >= 0 && token < q.a.vocab ? (int)token : -1;
  k.xm = row[k.taken].max;
  k.xi = 1.0f / row[k.taken].sum;
  k.ym = k.drafted ? row[n + 1 + k.taken].max : 0.0f;
  k.yi = k.drafted ? 1.0f / row[n + 1 + k.taken].sum : 0.0f;
  return k;
}
// With temperature 0 the token that follows, or -1.
__device__ __forceinline__ int64_t greedy(const RowPart& p) { return p.at == INT_MAX ? -1 : p.at; }

// Step 3.  The leader of the race: the largest w / e, and its index.
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

// A warp's part of the race over entries [i0, end) in pieces of 128, `step` apart, U of them
// requested at a time.  An entry is weighed with the hardware's exponential first, whose error is
// below the margin 2^-15 (2^-23 of the exponent, which is 127 at most); only what may beat the
// bar, a score that some entry of the CTA's has at least (shared_bar, 0 at first), is computed with care, so
// the loop takes 14 instructions per entry.  Behind the end the noise is infinite.  y null: p alone.
template <int U>
__device__ __forceinline__ Leader race(const Sequence& q, const Pick& k, const float* y, int out_of, int i0, int end, int step,
                                       uint32_t* shared_bar) {
  const int lane = threadIdx.x & 31;
  const float* x = q.row(k.taken);
  const float* e = q.a.noise + q.b * q.a.ldn;
  const bool ax = (reinterpret_cast<uintptr_t>(x) & 15) == 0, ay = (reinterpret_cast<uintptr_t>(y) & 15) == 0,
             ae = (reinterpret_cast<uintptr_t>(e) & 15) == 0;
  Leader lead = {0.0f, INT_MAX};
  float bar = 0.0f;
  for (; i0 < end; i0 += U * step) {
    float4 vx[U], ve[U], vy[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = min(i0 + j * step, end) + 4 * lane;  // behind the end: -inf without a read
      vx[j] = logits4(x, i, end, ax);
      ve[j] = logits4(e, i, end, ae, INFINITY);
      vy[j] = y ? logits4(y, i, end, ay) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    bar = fmaxf(bar, __uint_as_float(*(volatile uint32_t*)shared_bar));
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = min(i0 + j * step, end) + 4 * lane;
      const float fx[4] = {vx[j].x, vx[j].y, vx[j].z, vx[j].w}, fy[4] = {vy[j].x, vy[j].y, vy[j].z, vy[j].w},
                  fe[4] = {ve[j].x, ve[j].y, ve[j].z, ve[j].w};
      float high[4], width[4];
      bool any = false;
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const float dx = fx[z] - k.xm, dy = fy[z] - k.ym;
        const float p = ex2(dx * q.c_hi) * k.xi;                 // a NaN is never taken
        const float r = y ? fmaxf(ex2(dy * q.c_hi), 0.0f) * k.yi : 0.0f;  // and counts as 0 here
        width[z] = p + r;
        high[z] = fmaf(width[z], 0x1p-15f, p - r);
        any |= high[z] > bar * fe[z];
      }
      if (__any_sync(0xffffffffu, any)) {
        // what these entries score at least raises the bar, which few of them pass then
        float least = 0.0f;
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const float low = fmaf(width[z], -0x1p-14f, high[z]);
          if (low > 0.0f && i + z != out_of) least = fmaxf(least, low / fe[z]);
        }
        least = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fminf(least, FLT_MAX))));
        if (least > bar) {
          bar = least;
          if (lane == 0) atomicMax(shared_bar, __float_as_uint(bar));
        }
#pragma unroll
        for (int z = 0; z < 4; ++z)
          if (high[z] > bar * fe[z] && i + z != out_of) {
            // products that round by themselves: equal rows leave exactly nothing
            float w = __fmul_rn(exp_scaled(fx[z] - k.xm, q.c_hi, q.c_lo), k.xi);
            if (y) w = __fsub_rn(w, __fmul_rn(exp_scaled(fy[z] - k.ym, q.c_hi, q.c_lo), k.yi));
            if (w > 0.0f) lead.take(w / fe[z], i + z);
          }
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float s2 = __shfl_xor_sync(0xffffffffu, lead.best, o);
    const int i2 = __shfl_xor_sync(0xffffffffu, lead.at, o);
    lead.take(s2, i2);
  }
  return lead;
}

// The race over a cluster: CTA `rank` of `ctas` runs over entries [i0 of its warps, end), the leaders
// meet in every CTA.  Returns the winner, or -1.  The caller's cluster runs by now.
template <int U, int W>
__device__ __forceinline__ int64_t race_cluster(const Sequence& q, const Pick& k, int i0, int end, int step, int rank, int ctas) {
  __shared__ Leader s_lead[W];
  __shared__ Leader s_all[2][kVerifyCluster];
  __shared__ uint32_t s_bar;
  const int tid = threadIdx.x;
  const float* y = k.drafted ? q.row(q.n + 1 + k.taken) : nullptr;
  int out_of = k.out_of;
  if (tid == 0) s_bar = 0u;  // and so it is in a second pass: nothing scored in the first
  __syncthreads();
  for (int pass = 0;; ++pass) {  // a second one where nothing of p - q is left: p itself
    Leader lead = race<U>(q, k, y, out_of, i0, end, step, &s_bar);
    if ((tid & 31) == 0) s_lead[tid >> 5] = lead;
    __syncthreads();
    if (tid < ctas) {
      for (int w = 0; w < W; ++w) lead.take(s_lead[w].best, s_lead[w].at);
      st_cluster_v2(mapa_shared(smem_u32(&s_all[pass][rank]), tid), __float_as_uint(lead.best), (uint32_t)lead.at);
    }
    __syncwarp();
    cluster_sync_all();
    Leader all = s_all[pass][0];
    for (int r = 1; r < ctas; ++r) all.take(s_all[pass][r].best, s_all[pass][r].at);
    if (all.at != INT_MAX) return all.at;
    if (pass == 1 || !k.refused) return -1;
    y = nullptr;
    out_of = -1;
  }
}

// All in one launch: a cluster of `ctas` CTAs per sequence.
template <int W>
__global__ void __launch_bounds__(32 * W, 1024 / (32 * W) < 3 ? 1024 / (32 * W) : 3) k_verify(VerifyArgs a, int ctas) {
  constexpr int kSlots = 8;
  __shared__ RowPart s_part[kVerifyMaxRows][kSlots];         // this slice's rows, by slot
  __shared__ RowPart s_cta[kVerifyMaxRows][kVerifyCluster];  // the rows, by CTA
  __shared__ RowPart s_row[kVerifyMaxRows];
  __shared__ Pick s_pick;
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x / ctas, rank = blockIdx.x - b * ctas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Sequence q(a, b);
  const int rows = q.rows();
  if (rows == 0) {
    if (rank == 0) write_tokens(q, 0, -1, tid, 32 * W);
    return;  // as the whole cluster does
  }
  cluster_arrive_relaxed();
  Drafted d = {-1, 0.0f, 0.0f, 0.0f};
  if (warp == 0) d = ask_drafted(q, lane);
  const int s0 = min(a.vocab, rank * a.slice), s1 = min(a.vocab, s0 + a.slice);
  // The slice's segments go round `slots` warps, the same ones in every row; several rows at once
  // where the slice has few segments.
  const int segs = (a.slice + kVerifySeg - 1) / kVerifySeg;
  const int slots = segs >= kSlots ? kSlots : segs >= 4 ? 4 : segs >= 2 ? 2 : 1;
  for (int r = warp / slots; r < rows; r += W / slots) {
    const float* x = q.row(r);
    RowPart p = no_part();
    for (int seg = warp % slots; seg < segs; seg += slots) p = join(q, p, read_segment(q, x, s0 + seg * kVerifySeg, s1));
    if (lane == 0) s_part[r][warp % slots] = p;
  }
  __syncthreads();
  cluster_wait();  // all CTAs of the cluster run
  for (int r = warp; r < rows; r += W) {
    const RowPart p = join_lanes(q, s_part[r][lane % slots], slots);
    if (lane < ctas) st_cluster_v4(mapa_shared(smem_u32(&s_cta[r][rank]), lane), p.max, p.sum, p.at);
  }
  __syncwarp();
  cluster_sync_all();
  for (int r = warp; r < rows; r += W) {
    const RowPart p = join_lanes(q, s_cta[r][lane % ctas], ctas);
    if (lane == 0) s_row[r] = p;
  }
  __syncthreads();
  if (warp == 0) {
    const Pick k = follow(q, d, s_row, rank == 0);
    if (lane == 0) s_pick = k;
  }
  __syncthreads();
  const Pick k = s_pick;
  const int64_t last = q.T == 0.0f ? greedy(s_row[k.taken])
                                   : race_cluster<2, W>(q, k, s0 + 128 * warp, s1, 128 * W, rank, ctas);
  if (rank == 0) write_tokens(q, k.taken, last, tid, 32 * W);
}

// Step 1 alone: grid (blocks of 8 segments, row groups, batch), a warp per segment; the warps of a CTA
// never meet.  64 sequences of 1 to 11 rows of 128256 and their draft's, 229 MB: 38.5 us by itself, 6.0 TB/s (41.6
// after a flush of the caches).  A CTA goes through its group's rows, so that rows that a sequence with
// fewer drafted tokens does not have cost nothing.
__global__ void __launch_bounds__(kVerifyThreads, 4) k_verify_rows(VerifyArgs a) {
  pdl_trigger();
  pdl_wait();
  const int seg = blockIdx.x * kVerifyWarps + (threadIdx.x >> 5);
  if (seg >= a.segs) return;
  const Sequence q(a, blockIdx.z);
  const int rows = q.rows();
  for (int r = blockIdx.y; r < rows; r += gridDim.y) {
    const RowPart p = read_segment(q, q.row(r), seg * kVerifySeg, a.vocab);
    if ((threadIdx.x & 31) == 0) q.part(r)[seg] = p;
  }
}

// Step 2 alone: a CTA per sequence, a warp per row.  Latency-bound, 6.6 us for those 64 sequences (8.8 after a
// flush of the caches): 32 warps where there are more than 16 rows (4 sequences x 17 rows of 128256 21.0 us
// a call with 16, 19.5 with 32), but not for more sequences than SMs (250 x 3 rows of 10000 23.1 and 26.5).
__global__ void __launch_bounds__(kPickThreads, 1) k_verify_pick(VerifyArgs a) {
  __shared__ RowPart s_row[kVerifyMaxRows];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Sequence q(a, blockIdx.x);
  const int rows = q.rows();
  if (rows == 0) {
    if (tid == 0) a.picks[q.b].taken = -1;
    write_tokens(q, 0, -1, tid, blockDim.x);
    return;
  }
  Drafted d = {-1, 0.0f, 0.0f, 0.0f};
  if (warp == 0) d = ask_drafted(q, lane);
  for (int r = warp; r < rows; r += blockDim.x / 32) {
    constexpr int U = 4;  // a lane's parts of 128 segments, requested together
    const RowPart* p = q.part(r);
    RowPart x[U];
#pragma unroll
    for (int k = 0; k < U; ++k) x[k] = lane + 32 * k < a.segs ? p[lane + 32 * k] : no_part();
    RowPart z = x[0];
#pragma unroll
    for (int k = 1; k < U; ++k) z = join(q, z, x[k]);
    for (int i = lane + 32 * U; i < a.segs; i += 32) z = join(q, z, p[i]);
    z = join_lanes(q, z, 32);
    if (lane == 0) s_row[r] = z;
  }
  __syncthreads();
  if (warp) return;
  Pick k = follow(q, d, s_row, true);
  if (q.T == 0.0f) {
    write_tokens(q, k.taken, greedy(s_row[k.taken]), lane, 32);
    k.taken = -1;
  }
  k.lead = 0ull;
  k.done = 0;
  if (lane == 0) a.picks[q.b] = k;
}

// A leader as one number, the larger the better: its score, then the lower index; 0 for none.
__device__ __forceinline__ unsigned long long packed(const Leader& l) {
  return l.at == INT_MAX ? 0ull : (unsigned long long)__float_as_uint(l.best) << 32 | (uint32_t)~l.at;
}

// Step 3 alone: grid (CTAs of a sequence, batch), a CTA `per` entries.  The leaders meet in the
// sequence's Pick by a maximum, which no order of the CTAs changes; the last CTA writes.  All CTAs run
// at once, four on an SM: a second wave pays the start again (some 4 us: 64 sequences of 128256 entries 61 us
// a call with 592 CTAs, 65 with 1184; 65 with two on an SM that request four pieces at a time; 64.7 with a
// cluster of 4 per sequence, which left SMs with one CTA beside SMs with two).  By itself 20 us, 23 after a
// flush of the caches, 85 MB.
__global__ void __launch_bounds__(kVerifyThreads, 4) k_verify_race(VerifyArgs a, int per) {
  constexpr int U = 2, W = kVerifyWarps;
  __shared__ unsigned long long s_lead[W], s_best;
  __shared__ int s_last;
  __shared__ uint32_t s_bar;
  pdl_trigger();
  if (threadIdx.x == 0) s_bar = 0u;
  __syncthreads();
  pdl_wait();
  const Sequence q(a, blockIdx.y);
  Pick* pick = a.picks + blockIdx.y;
  const Pick k = *pick;
  if (k.taken < 0) return;  // done already
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float* y = k.drafted ? q.row(q.n + 1 + k.taken) : nullptr;
  auto best = [&](const Leader& lead) {  // of the CTA, in thread 0
    if (lane == 0) s_lead[warp] = packed(lead);
    __syncthreads();
    unsigned long long x = s_lead[0];
#pragma unroll
    for (int w = 1; w < W; ++w) x = max(x, s_lead[w]);
    return x;
  };
  const int i0 = blockIdx.x * per, end = min(a.vocab, i0 + per);
  unsigned long long all = best(race<U>(q, k, y, k.out_of, i0 + 128 * warp, end, 128 * W, &s_bar));
  if (tid == 0) {
    if (all) atomicMax(&pick->lead, all);
    __threadfence();
    s_last = atomicAdd(&pick->done, 1) == (int)gridDim.x - 1;
    if (s_last) {
      __threadfence();
      s_best = atomicMax(&pick->lead, 0ull);
    }
  }
  __syncthreads();
  if (!s_last) return;
  all = s_best;
  if (!all && k.refused) all = best(race<U>(q, k, nullptr, -1, 128 * warp, a.vocab, 128 * W, &s_bar));  // nothing of p - q: p itself
  write_tokens(q, k.taken, all ? (int64_t)(uint32_t)~(uint32_t)all : -1, tid, kVerifyThreads);
}

template <int W>
static cudaError_t launch_verify(const VerifyArgs& a, int batch, int ctas, cudaStream_t s) {
  static std::atomic<bool> done[64];  // clusters of 16 are beyond the portable size
  int dev;
  bool needs;
  cudaError_t e = needs_opt_in(done, dev, needs);
  if (e != cudaSuccess) return e;
  if (needs) {
    e = cudaFuncSetAttribute(k_verify<W>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    opted_in(done, dev);
  }
  return launch_pdl(k_verify<W>, dim3((unsigned)(batch * ctas)), dim3(32 * W), 0, s, (unsigned)ctas, a, ctas);
}

// One launch, or the workspace of three.
static bool one_launch(int64_t batch, int64_t rows, int64_t vocab) {
  return batch * rows * vocab <= 6ll << 20 && rows * vocab <= (batch <= kVerifyFew ? 3ll << 19 : 1ll << 19);
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

extern "C" OTF_API int64_t otf_verify_workspace_bytes(int64_t batch, int64_t drafts, int64_t vocab, int with_draft) {
  if (batch <= 0 || batch > 65535 || drafts < 0 || drafts > otf::kVerifyMaxDrafts || vocab <= 0 || vocab > (1 << 30))
    return -1;
  if (otf::one_launch(batch, drafts + 1 + (with_draft ? drafts : 0), vocab)) return 0;
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
  if (!target || !out_tokens || !accepted || batch <= 0 || drafts < 0 || vocab <= 0) return OTF_ERR_INVALID;
  if (drafts > otf::kVerifyMaxDrafts || vocab > (1 << 30) || batch > 65535) return OTF_ERR_UNSUPPORTED;
  if (drafts > 0 && (!tokens || ld_tokens < drafts || (uniforms && ld_uniforms < drafts))) return OTF_ERR_INVALID;
  if (ld_target < vocab || target_seq < 0 || (noise && ld_noise < vocab)) return OTF_ERR_INVALID;
  if (drafts == 0) draft = nullptr;
  if (draft && (ld_draft < vocab || draft_seq < 0)) return OTF_ERR_INVALID;
  if (!temperatures) {
    if (!otf::temperature_ok(temperature)) return OTF_ERR_INVALID;
    if (temperature > 0.0f && (!noise || (drafts > 0 && !uniforms))) return OTF_ERR_INVALID;
  }
  const int64_t bytes = otf_verify_workspace_bytes(batch, drafts, vocab, draft != nullptr);
  if (bytes > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < bytes))
    return OTF_ERR_INVALID;
  int st = check_device();
  if (st != OTF_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  otf::VerifyArgs a = {};
  a.target = target;
  a.tseq = target_seq;
  a.ldt = ld_target;
  a.draft = draft;
  a.dseq = draft_seq;
  a.ldd = ld_draft;
  a.tokens = tokens;
  a.ldtok = ld_tokens;
  a.uniforms = uniforms;
  a.ldu = ld_uniforms;
  a.noise = noise;
  a.ldn = ld_noise;
  a.temperatures = temperatures;
  a.temperature = temperature;
  a.counts = counts;
  a.out = out_tokens;
  a.accepted = accepted;
  a.drafts = (int)drafts;
  a.vocab = (int)vocab;
  const int64_t rows = drafts + 1 + (draft ? drafts : 0);
  if (bytes == 0) {
    // CTAs per sequence: 16 (of such clusters 14 run at once), 8, or as many as all run at once, three
    // on an SM; no more than the vocabulary has segments
    int ctas = batch <= 8 ? 16 : 8;
    while (ctas > 1 && (batch * ctas > 3 * 148 || (int64_t)(ctas - 1) * otf::kVerifySeg >= vocab)) ctas /= 2;
    a.slice = (int)(((vocab + ctas - 1) / ctas + 3) & ~3ll);
    const bool large = batch <= otf::kVerifyFew && rows * a.slice >= otf::kVerifyLarge;
    return set_cuda_error(large ? otf::launch_verify<32>(a, (int)batch, ctas, s) : otf::launch_verify<8>(a, (int)batch, ctas, s));
  }
  a.segs = (int)((vocab + otf::kVerifySeg - 1) / otf::kVerifySeg);
  a.picks = static_cast<otf::Pick*>(workspace);
  a.parts = reinterpret_cast<otf::RowPart*>(static_cast<char*>(workspace) +
                                            otf::align_up(batch * (int64_t)sizeof(otf::Pick), 256));
  // row groups: as many as all of their CTAs run at once, at least 4 (one sequence x 65 rows of 128256
  // 42.5 us a call with 4, 24.6 with 37)
  const int64_t blocks = (a.segs + otf::kVerifyWarps - 1) / otf::kVerifyWarps;
  const int64_t groups = std::min(rows, std::max<int64_t>(4, 4 * 148 / (batch * blocks)));
  cudaError_t e = otf::launch_pdl(otf::k_verify_rows, dim3((unsigned)blocks, (unsigned)groups, (unsigned)batch),
                                  dim3(otf::kVerifyThreads), 0, s, 1u, a);
  if (e != cudaSuccess) return set_cuda_error(e);
  e = otf::launch_pdl(otf::k_verify_pick, dim3((unsigned)batch),
                      dim3(rows > 16 && batch <= 148 ? otf::kPickThreads : otf::kPickThreads / 2), 0, s, 1u, a);
  if (e != cudaSuccess || (!temperatures && temperature == 0.0f)) return set_cuda_error(e);
  // CTAs per sequence: as many as all run at once
  const int64_t ctas = std::max<int64_t>(1, std::min(otf::kRaceResident / batch, vocab / otf::kRaceLeast));
  const int per = (int)(((vocab + ctas - 1) / ctas + 127) & ~127ll);
  return set_cuda_error(otf::launch_pdl(otf::k_verify_race, dim3((unsigned)((vocab + per - 1) / per), (unsigned)batch),
                                        dim3(otf::kVerifyThreads), 0, s, 1u, a, per));
}
