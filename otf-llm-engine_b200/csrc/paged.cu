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

// What k_paged_append gets beside the cache.
struct AppendArgs {
  PagedView c;
  const double* turns;
  int rot, interleaved;
  float factor;
  const uint16_t* q;
  uint16_t* qo;
  const uint16_t* k;
  const uint16_t* v;
  int64_t ldq, ldqo, ldk, ldv;
  int heads;  // 0: keys and values alone
  const int* starts;
  const int* positions;
  int per;    // rows of a sequence, without starts
  float* weights;  // or null: their entries of the new tokens are cleared
  int64_t ldw;
};

// Where a row goes: the offset of its token's page row, or -1 (all its threads agree; `t` of `threads`).
// The rotary position's sines and cosines go to s_c and s_s.
__device__ __forceinline__ int64_t append_place(const AppendArgs& a, int row, int t, int threads, float* s_c, float* s_s) {
  const PagedView& c = a.c;
  const int b = a.starts ? sequence_of(a.starts, c.batch, row) : row / a.per;
  if (b >= c.batch) return -1;  // behind the last sequence
  const int i = row - (a.starts ? a.starts[b] : b * a.per);
  const int len = c.lengths[b];
  if (len < 0) return -1;  // no sequence in this place
  const int64_t slot = (int64_t)len + i;
  if (i < 0 || slot >= c.capacity) {
    if (t == 0) report_bad_page();
    return -1;
  }
  const int in = (int)slot / c.page_size;
  const int page = c.table[b * c.ld_table + in];
  if (page < 0 || page >= c.n_pages) {
    if (t == 0) report_bad_page();
    return -1;
  }
  if (a.weights)
    for (int g = t; g < c.kv_heads; g += threads) a.weights[((int64_t)b * c.kv_heads + g) * a.ldw + slot] = 0.0f;
  const int position = a.positions ? a.positions[row] : (int)slot;
  for (int p = t; p < a.rot / 2; p += threads) {
    // the angle in turns, 64 bits until the whole turns are gone: what is left keeps 2^-25 of a turn
    double turn = (double)position * a.turns[p];
    turn -= rint(turn);
    float sn, cs;
    sincospif(2.0f * (float)turn, &sn, &cs);
    s_c[p] = cs * a.factor;
    s_s[p] = sn * a.factor;
  }
  return page * c.page_stride + (int64_t)((int)slot - in * c.page_size) * c.token_stride;
}

// Where head h of a row is read from and goes to: queries, keys, values in this order.
template <int D>
__device__ __forceinline__ const uint16_t* append_source(const AppendArgs& a, int64_t row, int h) {
  const int k = h - a.heads, v = k - a.c.kv_heads;
  return k < 0 ? a.q + row * a.ldq + (int64_t)h * D : v < 0 ? a.k + row * a.ldk + (int64_t)k * D : a.v + row * a.ldv + (int64_t)v * D;
}
template <int D>
__device__ __forceinline__ uint16_t* append_target(const AppendArgs& a, int64_t row, int64_t at, int h) {
  const int k = h - a.heads, v = k - a.c.kv_heads;
  return k < 0   ? a.qo + row * a.ldqo + (int64_t)h * D
         : v < 0 ? a.c.k + at + (int64_t)k * a.c.head_stride
                 : a.c.v + at + (int64_t)v * a.c.head_stride;
}

// Rotary positions and the cache write in units of two 16-byte pieces whose values turn together:
// pieces i and i + rot / 16 of a head (half layout), or 2i and 2i + 1.  Memory-bound: a row is read
// and written once (15125 rows of 80 heads of 128, 620 MB: 94.8 us, 6.5 TB/s).  The values are requested before the row's place in the cache and its angles are
// known, kAppendBatch units at a time; a thread has the same i in every head, whose 8 sines and
// cosines it keeps in registers.  WR warps a row: 4, or 1 for rows that a warp holds at once (27500 rows
// of 18 heads of 64: 62.5 us with 4, 37.6 with 1; of 80 heads of 128: 168.6 with 4, 171.8 with 1; 256
// of them 5.1 and 8.3).
constexpr int kAppendThreads = 128;
constexpr int kAppendBatch = 5;

template <bool BF, int D, int WR>
__global__ void __launch_bounds__(kAppendThreads) k_paged_append(AppendArgs a, int n) {
  constexpr int UH = D / 16, T = 32 * WR, R = kAppendThreads / T;  // units of a head, threads of a row, rows of the CTA
  __shared__ __align__(16) float s_c[R][64], s_s[R][64];
  pdl_trigger();
  pdl_wait();
  const int mine = threadIdx.x / T, t = threadIdx.x % T, row = blockIdx.x * R + mine;
  if (row >= n) return;  // a whole warp's, and with more warps a row there is one row
  const int turning = a.heads + a.c.kv_heads, heads = turning + a.c.kv_heads, i = t % UH;
  const bool turns = i < a.rot / 16, halves = turns && !a.interleaved;
  const int p0 = halves ? i * 8 : i * 16, p1 = halves ? i * 8 + a.rot / 2 : i * 16 + 8;
  float cs[8], sn[8];
  int64_t at = 0;
  constexpr int HC = T / UH;  // heads that the row's threads cover at once
  for (int h0 = 0; h0 < heads; h0 += kAppendBatch * HC) {
    uint4 x[kAppendBatch][2];
#pragma unroll
    for (int j = 0; j < kAppendBatch; ++j) {
      const int h = h0 + j * HC + t / UH;
      if (h < heads) {
        const uint16_t* src = append_source<D>(a, row, h);
        x[j][0] = *reinterpret_cast<const uint4*>(src + (h < turning ? p0 : i * 16));  // values never turn
        x[j][1] = *reinterpret_cast<const uint4*>(src + (h < turning ? p1 : i * 16 + 8));
      }
    }
    if (h0 == 0) {
      at = append_place(a, row, t, T, s_c[mine], s_s[mine]);
      if (at < 0) return;
      if (WR > 1) __syncthreads(); else __syncwarp();
      if (turns)
#pragma unroll
        for (int z = 0; z < 8; ++z) {
          cs[z] = s_c[mine][8 * i + z];
          sn[z] = s_s[mine][8 * i + z];
        }
    }
#pragma unroll
    for (int j = 0; j < kAppendBatch; ++j) {
      const int h = h0 + j * HC + t / UH;
      if (h >= heads) break;
      uint16_t* dst = append_target<D>(a, row, at, h);
      if (turns && h < turning) {
        uint32_t* w0 = reinterpret_cast<uint32_t*>(&x[j][0]);
        uint32_t* w1 = reinterpret_cast<uint32_t*>(&x[j][1]);
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          if (halves) {  // pairs (w0, w1) place by place
            const float2 u = unpack2<BF>(w0[z]), v = unpack2<BF>(w1[z]);
            w0[z] = pack2<BF>(u.x * cs[2 * z] - v.x * sn[2 * z], u.y * cs[2 * z + 1] - v.y * sn[2 * z + 1]);
            w1[z] = pack2<BF>(v.x * cs[2 * z] + u.x * sn[2 * z], v.y * cs[2 * z + 1] + u.y * sn[2 * z + 1]);
          } else {       // pairs within a word, four in each piece
            const float2 u = unpack2<BF>(w0[z]), v = unpack2<BF>(w1[z]);
            w0[z] = pack2<BF>(u.x * cs[z] - u.y * sn[z], u.y * cs[z] + u.x * sn[z]);
            w1[z] = pack2<BF>(v.x * cs[z + 4] - v.y * sn[z + 4], v.y * cs[z + 4] + v.x * sn[z + 4]);
          }
        }
      }
      *reinterpret_cast<uint4*>(dst + (h < turning ? p0 : i * 16)) = x[j][0];
      *reinterpret_cast<uint4*>(dst + (h < turning ? p1 : i * 16 + 8)) = x[j][1];
    }
  }
}

// The same for a rot that is no multiple of 16, where the partners of a 16-byte piece lie across two
// others: the heads go through shared memory, kAppendHeads at a time, whose threads share out the pairs.
constexpr int kAppendHeads = 32;

template <bool BF, int D>
__global__ void __launch_bounds__(kAppendThreads) k_paged_append_any(AppendArgs a) {
  constexpr int P = D / 8, N = kAppendHeads * P / kAppendThreads;  // pieces of a head, of a thread
  __shared__ float s_c[64], s_s[64];
  __shared__ __align__(16) uint16_t s_x[kAppendHeads][D];
  pdl_trigger();
  pdl_wait();
  const int64_t row = blockIdx.x;
  const int half = a.rot / 2, turning = a.heads + a.c.kv_heads, heads = turning + a.c.kv_heads;
  int64_t at = 0;
  for (int h0 = 0; h0 < heads; h0 += kAppendHeads) {
    uint4 x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = j * kAppendThreads + threadIdx.x, h = h0 + e / P;
      if (h < heads) x[j] = *reinterpret_cast<const uint4*>(append_source<D>(a, row, h) + e % P * 8);
    }
    if (h0 == 0) {
      at = append_place(a, (int)row, threadIdx.x, kAppendThreads, s_c, s_s);
      if (at < 0) return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = j * kAppendThreads + threadIdx.x;
      if (h0 + e / P < turning) *reinterpret_cast<uint4*>(&s_x[e / P][e % P * 8]) = x[j];
    }
    __syncthreads();
    const int pairs = min(kAppendHeads, turning - h0) * half;
    for (int e = threadIdx.x; e < pairs; e += kAppendThreads) {
      const int h = e / half, p = e - h * half;
      uint16_t& u = s_x[h][a.interleaved ? 2 * p : p];
      uint16_t& v = s_x[h][a.interleaved ? 2 * p + 1 : p + half];
      const float fu = to_f<BF>(u), fv = to_f<BF>(v);
      u = from_f<BF>(fu * s_c[p] - fv * s_s[p]);
      v = from_f<BF>(fv * s_c[p] + fu * s_s[p]);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = j * kAppendThreads + threadIdx.x, h = h0 + e / P;
      if (h >= heads) break;
      if (h < turning && e % P * 8 < a.rot) x[j] = *reinterpret_cast<const uint4*>(&s_x[e / P][e % P * 8]);
      *reinterpret_cast<uint4*>(append_target<D>(a, row, at, h) + e % P * 8) = x[j];
    }
    __syncthreads();  // before the next heads
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

constexpr int kEvictThreads = 512;
constexpr int kEvictKeys = 16;       // weights of a thread
constexpr int kEvictStrip = kEvictThreads * kEvictKeys;
constexpr int kEvictCluster = 8;     // CTAs that may share one (sequence, KV head)

// Which places stay: a cluster per (sequence, KV head), each CTA a contiguous slice of the n
// weights that are not among the recent ones, a thread 16 neighbours.  Rounds of BITS bits find the
// k-th largest key (each round: counts of the slice's keys in shared memory, summed over the cluster
// through distributed shared memory), and what the CTAs before this one count above the limit and at
// it is where its own places begin.  Of the keys equal to the k-th largest the first ones stay.
// Bound by the rounds' latencies, not by bytes: ONE holds the keys of a slice of up to kEvictStrip
// in registers through all rounds, longer ones are read again (from L2).  16 x 8 heads of 8191 weights
// take 11.3 us (12.9 after a flush of the caches).  BITS 11 (three rounds) for a CTA by itself, 8 (four) in
// a cluster, whose CTAs read one another's counts: 65536 weights of 8 heads, with the copy, 26.1 us with
// 11, 21.6 us with 8.
template <bool ONE, int BITS>
__global__ void __launch_bounds__(kEvictThreads) k_evict_select(const int* lengths, int kv_heads, int capacity,
                                                                const float* weights, int64_t ldw, int budget,
                                                                int recent, int* kept, int ctas) {
  constexpr int W = kEvictThreads / 32, V = kEvictKeys, BINS = 1 << BITS, ROUNDS = (31 + BITS) / BITS;
  constexpr int ND = BINS > kEvictThreads ? BINS / kEvictThreads : 1;  // digits of a thread, of the first BINS / ND
  __shared__ __align__(16) int s_hist[ROUNDS][BINS];
  __shared__ int s_cut[2];    // this round's digit, and how many keys of it are needed
  __shared__ int s_count[2];  // kept keys above the limit, and keys at it, in the slices before
  __shared__ int s_warp[W];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = ctas > 1 ? (int)cluster_ctarank() : 0;
  const int pair = blockIdx.x / ctas, b = pair / kv_heads;
  const float* w = weights + (int64_t)pair * ldw;
  int* keep = kept + (int64_t)pair * budget;
  int len = lengths[b];
  if (len > capacity) {
    if (tid == 0) report_bad_page();
    len = -1;
  }
  if (len <= budget) {  // the whole cluster returns
    for (int i = rank * kEvictThreads + tid; i < budget; i += ctas * kEvictThreads) keep[i] = i < len ? i : -1;
    return;
  }
  const int n = len - recent, k = budget - recent;
  for (int i = rank * kEvictThreads + tid; i < recent; i += ctas * kEvictThreads) keep[k + i] = n + i;
  if (k == 0) return;
  const int per = ((n + ctas - 1) / ctas + 3) & ~3, i0 = min(n, rank * per), i1 = min(n, i0 + per);
  const bool aligned = (reinterpret_cast<uintptr_t>(w) & 15) == 0;
  // this thread's keys of the strip from `base` on: u[0 .. there)
  uint32_t u[V];
  auto load = [&](int base) -> int {
    const int i = base + tid * V, there = max(0, min(V, i1 - i));
#pragma unroll
    for (int z = 0; z < V; z += 4) {
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (aligned && z + 4 <= there) {
        x = *reinterpret_cast<const float4*>(w + i + z);
      } else {
        if (z < there) x.x = w[i + z];
        if (z + 1 < there) x.y = w[i + z + 1];
        if (z + 2 < there) x.z = w[i + z + 2];
        if (z + 3 < there) x.w = w[i + z + 3];
      }
      u[z] = weight_key(x.x);
      u[z + 1] = weight_key(x.y);
      u[z + 2] = weight_key(x.z);
      u[z + 3] = weight_key(x.w);
    }
    return there;
  };
  int there = ONE ? load(i0) : 0;
  for (int i = tid; i < ROUNDS * BINS / 4; i += kEvictThreads)
    reinterpret_cast<int4*>(&s_hist[0][0])[i] = make_int4(0, 0, 0, 0);
  if (tid < 2) s_count[tid] = 0;
  __syncthreads();
  uint32_t limit = 0u, mask = 0u;
  int need = k;
  int g0 = 0, e0 = 0;  // this thread's digits' share of the keys above the limit, and at it, in the slices before
#pragma unroll 1
  for (int round = 0; round < ROUNDS; ++round) {
    const int shift = max(0, 32 - BITS * (round + 1));
    const uint32_t bits = round == ROUNDS - 1 ? (1u << (32 - BITS * (ROUNDS - 1))) - 1u : BINS - 1u;
    for (int base = i0; base < i1; base += kEvictStrip) {
      if (!ONE) there = load(base);
#pragma unroll
      for (int z = 0; z < V; ++z)
        if (z < there && (u[z] & mask) == limit) atomicAdd(&s_hist[round][(u[z] >> shift) & bits], 1);
    }
    if (ctas > 1) cluster_sync_all(); else __syncthreads();
    // thread t: the ND digits from high - ND + 1 to high, of the cluster and of the CTAs before this one
    const int high = BINS - 1 - ND * tid;
    int c[ND], lower[ND], all = 0;
#pragma unroll
    for (int i = 0; i < ND; ++i) c[i] = lower[i] = 0;
    if (high >= 0) {
      const int* mine = &s_hist[round][high - ND + 1];
      if (ctas > 1) {
#pragma unroll
        for (int r = 0; r < kEvictCluster; ++r)
          if (r < ctas)
#pragma unroll
            for (int i = 0; i < ND; ++i) {
              const int x = ld_cluster_s32(mapa_shared(smem_u32(mine + i), r));
              c[i] += x;
              if (r < rank) lower[i] += x;
            }
      } else {
#pragma unroll
        for (int i = 0; i < ND; ++i) c[i] = mine[i];
      }
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) all += c[i];
    int before = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += x;
    }
    if (lane == 31) s_warp[warp] = before;
    __syncthreads();
    before -= all;
#pragma unroll
    for (int x = 0; x < W; ++x)
      if (x < warp) before += s_warp[x];
    if (before < need && before + all >= need) {  // one thread's
      bool found = false;
#pragma unroll
      for (int i = ND - 1; i >= 0; --i) {
        if (!found && before + c[i] >= need) {
          found = true;
          s_cut[0] = high - ND + 1 + i;
          s_cut[1] = need - before;
        }
        before += c[i];
      }
    }
    __syncthreads();
    // every thread has used what it read: after the last round the others may leave (waited for at the end)
    if (ctas > 1 && round == ROUNDS - 1) cluster_arrive_relaxed();
    const int cut = s_cut[0];
    limit |= (uint32_t)cut << shift;
    need = s_cut[1];
    mask |= bits << shift;
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const int digit = high - ND + 1 + i;
      if (digit > cut) g0 += lower[i];
      if (round == ROUNDS - 1 && digit == cut) e0 += lower[i];
    }
  }
  if (ctas > 1) {  // the threads' shares as one sum
    g0 = __reduce_add_sync(0xffffffffu, g0);
    e0 = __reduce_add_sync(0xffffffffu, e0);
    if (lane == 0) {
      atomicAdd(&s_count[0], g0);
      atomicAdd(&s_count[1], e0);
    }
    __syncthreads();
    g0 = s_count[0];
    e0 = s_count[1];
  }
  // keys above the limit in the low, at it in the high half
  auto count = [&] {
    uint32_t c = 0;
#pragma unroll
    for (int z = 0; z < V; ++z)
      if (z < there) c += u[z] > limit ? 1u : u[z] == limit ? 0x10000u : 0u;
    return c;
  };
  for (int base = i0; base < i1; base += kEvictStrip) {
    if (!ONE) there = load(base);
    const uint32_t mine = count();
    uint32_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (lane == 31) s_warp[warp] = (int)inc;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int x = 0; x < W; ++x) {
      if (x == warp) before = all;
      all += (uint32_t)s_warp[x];
    }
    before += inc - mine;
    int g = g0 + (int)(before & 0xffffu), e = e0 + (int)(before >> 16);
#pragma unroll
    for (int z = 0; z < V; ++z)
      if (z < there) {
        const bool eq = u[z] == limit;
        if (u[z] > limit || (eq && e < need)) keep[g + min(e, need)] = base + tid * V + z;
        g += u[z] > limit;
        e += eq;
      }
    g0 += (int)(all & 0xffffu);
    e0 += (int)(all >> 16);
    __syncthreads();
  }
  __syncwarp();
  if (ctas > 1) cluster_wait();  // no CTA leaves while another reads its counts
}

// The kept rows' keys, values and weights, where source and target are apart: grid (pairs, tiles
// of kMoveRows kept places).  One pass, memory-bound: 16 x 8 heads, 2048 rows kept, 233 MB in 39 us after
// a flush of the caches, 6.0 TB/s, 42 us behind other calls, whose writes are still to leave L2.
constexpr int kMoveRows = 64;

struct MoveArgs {
  PagedView from, to;
  const int* kept;
  const float* weights;
  float* wout;
  int64_t ldw, ldwo;
  int budget;
  int* lengths_out;
};

// Offset of a sequence's token in a pool, -1 (and the flag) when its page is not in it.
__device__ __forceinline__ int64_t token_offset(const PagedView& c, int b, int s) {
  const int at = s / c.page_size;
  const int page = c.table[b * c.ld_table + at];
  if (page < 0 || page >= c.n_pages) {
    report_bad_page();
    return -1;
  }
  return page * c.page_stride + (int64_t)(s - at * c.page_size) * c.token_stride;
}

__device__ __forceinline__ void set_length(const MoveArgs& a, int b) {
  const int len = a.from.lengths[b];
  a.lengths_out[b] = len > a.from.capacity ? len : min(len, a.budget);
}

template <int D>
__global__ void __launch_bounds__(256) k_evict_copy(MoveArgs a) {
  constexpr int P = D / 8, R = 256 / P, N = kMoveRows / R;
  __shared__ int64_t s_from[kMoveRows], s_to[kMoveRows];
  pdl_trigger();
  pdl_wait();
  const int pair = blockIdx.x, b = pair / a.from.kv_heads, g = pair - b * a.from.kv_heads, tid = threadIdx.x;
  const int base = blockIdx.y * kMoveRows;
  const int* keep = a.kept + (int64_t)pair * a.budget;
  if (a.from.lengths[b] < 0 || a.from.lengths[b] > a.from.capacity) {
    if (g == 0 && blockIdx.y == 0 && tid == 0) set_length(a, b);
    return;
  }
  if (tid < kMoveRows) {
    const int j = base + tid, s = j < a.budget ? keep[j] : -1;
    int64_t x = -1, y = -1;
    if (s >= 0) {
      a.wout[pair * a.ldwo + j] = a.weights[pair * a.ldw + s];
      x = token_offset(a.from, b, s);
      y = token_offset(a.to, b, j);
    } else if (j < a.budget) {
      a.wout[pair * a.ldwo + j] = 0.0f;
    }
    s_from[tid] = y < 0 ? -1 : x;
    s_to[tid] = y;
  }
  if (blockIdx.y == 0)
    for (int64_t i = a.budget + tid; i < a.ldwo; i += 256) a.wout[pair * a.ldwo + i] = 0.0f;
  __syncthreads();
  const int r = tid / P, piece = tid - r * P;
  uint4 x[N][2];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t at = s_from[i * R + r];
    if (at >= 0) {
      const int64_t o = at + g * a.from.head_stride + piece * 8;
      x[i][0] = ld_stream16(a.from.k + o);
      x[i][1] = ld_stream16(a.from.v + o);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (s_from[i * R + r] >= 0) {
      const int64_t o = s_to[i * R + r] + g * a.to.head_stride + piece * 8;
      *reinterpret_cast<uint4*>(a.to.k + o) = x[i][0];
      *reinterpret_cast<uint4*>(a.to.v + o) = x[i][1];
    }
  if (g == 0 && blockIdx.y == 0 && tid == 0) set_length(a, b);
}

// The same in place: a CTA per (pair, keys / values, 64-byte column of the rows), or for a pair's
// weights, goes through the kept places in order, a tile of 256 at a time.  A row never moves to
// a higher place, so what a tile overwrites lies before all rows that later tiles read, and
// the next tile's rows can be requested before this one's are written; only within a tile must
// every row be read (the barrier) before one is written.  Rows that stay where they are are skipped.
__global__ void __launch_bounds__(128) k_evict_shift(MoveArgs a, int columns) {
  constexpr int N = 8, R = 32, T = N * R;  // rows of a thread, of the CTA at once, of a tile
  pdl_trigger();
  pdl_wait();
  const int pair = blockIdx.x, b = pair / a.from.kv_heads, g = pair - b * a.from.kv_heads, tid = threadIdx.x;
  const int len = a.from.lengths[b];
  if (len <= a.budget || len > a.from.capacity) return;  // nothing moves
  const int* keep = a.kept + (int64_t)pair * a.budget;
  if ((int)blockIdx.y == 2 * columns) {
    float* w = a.wout + pair * a.ldwo;
    for (int base = 0; base < a.budget; base += N * 128) {
      float x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = base + i * 128 + tid;
        x[i] = j < a.budget ? w[keep[j]] : 0.0f;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = base + i * 128 + tid;
        if (j < a.budget) w[j] = x[i];
      }
    }
    __syncthreads();
    for (int i = a.budget + tid; i < len; i += 128) w[i] = 0.0f;
    return;
  }
  uint16_t* pool = ((int)blockIdx.y < columns ? a.from.k : a.from.v) + g * a.from.head_stride +
                   ((int)blockIdx.y % columns) * 32 + (tid & 3) * 8;
  const int r = tid >> 2;
  struct Rows {
    uint4 x[N];
    int64_t to[N];
  };
  auto load = [&](int base, Rows& v) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = base + i * R + r;
      const int s = j < a.budget ? keep[j] : j;
      v.to[i] = -1;
      if (s != j) {
        const int64_t at = token_offset(a.from, b, s);
        if (at >= 0) {
          v.to[i] = token_offset(a.from, b, j);
          v.x[i] = *reinterpret_cast<const uint4*>(pool + at);
        }
      }
    }
  };
  auto store = [&](const Rows& v) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (v.to[i] >= 0) *reinterpret_cast<uint4*>(pool + v.to[i]) = v.x[i];
  };
  Rows even, odd;
  load(0, even);
  for (int base = 0; base < a.budget; base += 2 * T) {
    load(base + T, odd);
    __syncthreads();
    store(even);
    if (base + T >= a.budget) break;
    load(base + 2 * T, even);
    __syncthreads();
    store(odd);
  }
}

// In place the lengths change when nobody reads them any more.
__global__ void k_evict_lengths(MoveArgs a) {
  pdl_trigger();
  pdl_wait();
  for (int b = blockIdx.x * blockDim.x + threadIdx.x; b < a.from.batch; b += gridDim.x * blockDim.x) set_length(a, b);
}

// The taken nodes of a tree (otf_paged_keep): keys and values of the places lengths + path[j] move to
// lengths + 1 + j.  A CTA per sequence and KV head fetches all of them before it writes the first, so that
// the ways may cross; latency-bound: a chain of the path, the table, the rows.  Measured: 64 sequences, 32 KV heads of
// 128, up to 8 nodes each (9.4 MB) 4.0 us; one sequence, 8 KV heads, 5 nodes 2.5 us.
constexpr int kKeepThreads = 128;
constexpr int kKeepMost = 63;

template <int D>
__global__ void __launch_bounds__(kKeepThreads) k_paged_keep(PagedView c, const int* path, int64_t ldp, const int* accepted, int depth) {
  constexpr int P = D / 8;  // 16-byte pieces of a row
  __shared__ int64_t s_from[kKeepMost], s_to[kKeepMost];
  extern __shared__ uint4 s_rows[];  // [2 n P]
  pdl_trigger();
  pdl_wait();
  const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int len = c.lengths[b], n = accepted[b];
  if (len < 0 || n == 0) return;
  if (n < 0 || n > depth) {
    if (tid == 0 && g == 0) report_bad_page();
    return;
  }
  auto place = [&](int64_t s) -> int64_t {
    if (s >= c.capacity) return -1;
    const int page = c.table[b * c.ld_table + s / c.page_size];
    return page < 0 || page >= c.n_pages ? -1 : page * c.page_stride + s % c.page_size * c.token_stride;
  };
  if (tid < n) {
    const int from = path[b * ldp + tid];
    int64_t x = -1, y = -1;
    if (from >= 0) {
      x = place((int64_t)len + from);
      y = place((int64_t)len + 1 + tid);
    }
    if (x < 0 || y < 0) {
      report_bad_page();
      x = -1;
    } else if (x == y) {
      x = -1;  // there already
    }
    s_from[tid] = x;
    s_to[tid] = y;
  }
  __syncthreads();
  const int64_t head = g * c.head_stride;
#pragma unroll 4
  for (int i = tid; i < 2 * n * P; i += kKeepThreads) {
    const int j = i / (2 * P), piece = i % P;
    const int64_t x = s_from[j];
    if (x >= 0) s_rows[i] = *reinterpret_cast<const uint4*>((i / P & 1 ? c.v : c.k) + x + head + piece * 8);
  }
  __syncthreads();
#pragma unroll 4
  for (int i = tid; i < 2 * n * P; i += kKeepThreads) {
    const int j = i / (2 * P), piece = i % P;
    if (s_from[j] >= 0) *reinterpret_cast<uint4*>((i / P & 1 ? c.v : c.k) + s_to[j] + head + piece * 8) = s_rows[i];
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
  return otf_paged_append_weights(cache, rotary, q, ldq, q_out, ldqo, heads, k, ldk, v, ldv, starts, positions, n,
                                  nullptr, 0, stream);
}

extern "C" OTF_API int otf_paged_append_weights(const otf_paged_cache* cache, const otf_rotary* rotary, const void* q,
                                                int64_t ldq, void* q_out, int64_t ldqo, int64_t heads, const void* k,
                                                int64_t ldk, const void* v, int64_t ldv, const int32_t* starts,
                                                const int32_t* positions, int64_t n, float* weights, int64_t ldw,
                                                void* stream) {
  otf::PagedView c;
  int st = otf::view_of(cache, c);
  if (st != OTF_OK) return st;
  const int64_t D = cache->head_dim;
  if (n < 0 || n > INT32_MAX || (!starts && n % c.batch)) return OTF_ERR_INVALID;
  if (n == 0) return OTF_OK;
  if (!otf::rows16(k, ldk, c.kv_heads * D) || !otf::rows16(v, ldv, c.kv_heads * D)) return OTF_ERR_INVALID;
  if (q && (heads <= 0 || heads > 65535 || !otf::rows16(q, ldq, heads * D) || !otf::rows16(q_out, ldqo, heads * D)))
    return OTF_ERR_INVALID;
  if (weights && ldw < c.capacity) return OTF_ERR_INVALID;
  if (q && (((q_out != q || ldqo != ldq) && otf::rows_overlap(q, ldq, heads * D, q_out, ldqo, heads * D, n)) ||
            otf::rows_overlap(k, ldk, c.kv_heads * D, q_out, ldqo, heads * D, n) ||
            otf::rows_overlap(v, ldv, c.kv_heads * D, q_out, ldqo, heads * D, n)))
    return OTF_ERR_INVALID;
  int rot = 0;
  if (rotary) {
    if (rotary->rot_dim < 0 || rotary->rot_dim > D || rotary->rot_dim % 2 || (rotary->rot_dim && !rotary->turns))
      return OTF_ERR_INVALID;
    rot = (int)rotary->rot_dim;
  }
  st = check_device();
  if (st != OTF_OK) return st;
  otf::AppendArgs a = {c,
                       rot ? rotary->turns : nullptr,
                       rot,
                       rot ? (int)(rotary->interleaved != 0) : 0,
                       rot ? rotary->factor : 1.0f,
                       static_cast<const uint16_t*>(q),
                       static_cast<uint16_t*>(q_out),
                       static_cast<const uint16_t*>(k),
                       static_cast<const uint16_t*>(v),
                       ldq,
                       ldqo,
                       ldk,
                       ldv,
                       q ? (int)heads : 0,
                       starts,
                       positions,
                       (int)(n / c.batch),
                       weights,
                       ldw};
  const bool bf = cache->dtype == OTF_DTYPE_BF16;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)n);
  if (rot % 16)
    return set_cuda_error(otf::launch_pdl(D == 128 ? (bf ? otf::k_paged_append_any<true, 128> : otf::k_paged_append_any<false, 128>)
                                                   : (bf ? otf::k_paged_append_any<true, 64> : otf::k_paged_append_any<false, 64>),
                                          grid, dim3(otf::kAppendThreads), 0, s, 1u, a));
  // a warp per row where its threads hold the whole row at once
  const bool short_rows = ((q ? heads : 0) + 2 * c.kv_heads) * (D / 16) <= 32 * otf::kAppendBatch;
  auto* kern = D == 128 ? (short_rows ? (bf ? otf::k_paged_append<true, 128, 1> : otf::k_paged_append<false, 128, 1>)
                                : (bf ? otf::k_paged_append<true, 128, 4> : otf::k_paged_append<false, 128, 4>))
                        : (short_rows ? (bf ? otf::k_paged_append<true, 64, 1> : otf::k_paged_append<false, 64, 1>)
                                : (bf ? otf::k_paged_append<true, 64, 4> : otf::k_paged_append<false, 64, 4>));
  return set_cuda_error(otf::launch_pdl(kern, dim3((unsigned)(short_rows ? (n + 3) / 4 : n)), dim3(otf::kAppendThreads), 0, s, 1u,
                                        a, (int)n));
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
  if (budget > 65535ll * otf::kMoveRows) return OTF_ERR_UNSUPPORTED;
  // cut in place: the same pools under the same table, and the weights with them
  const bool in_place = to->page_table == from->page_table && to->k_pages == from->k_pages && to->v_pages == from->v_pages;
  if (in_place != (weights == weights_out) || (!in_place && lengths_out == from->lengths)) return OTF_ERR_INVALID;
  const int64_t pairs = f.batch * (int64_t)f.kv_heads;
  if (!in_place && otf::bytes_overlap(weights, pairs * ldw * 4, weights_out, pairs * ldw_out * 4)) return OTF_ERR_INVALID;
  if (lengths_out != from->lengths && otf::bytes_overlap(lengths_out, f.batch * 4, from->lengths, f.batch * 4))
    return OTF_ERR_INVALID;
  st = check_device();
  if (st != OTF_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // CTAs per (sequence, KV head): as many as hold the weights that there can be in registers, while
  // that leaves less than two CTAs per SM
  int ctas = 1;
  while (ctas < otf::kEvictCluster && (int64_t)ctas * otf::kEvictStrip < f.capacity && pairs * ctas <= 148) ctas *= 2;
  const bool one = (((f.capacity + ctas - 1) / ctas + 3) & ~3) <= otf::kEvictStrip;
  auto* select = ctas > 1 ? (one ? otf::k_evict_select<true, 8> : otf::k_evict_select<false, 8>)
                          : (one ? otf::k_evict_select<true, 11> : otf::k_evict_select<false, 11>);
  cudaError_t e = otf::launch_pdl(select, dim3((unsigned)(pairs * ctas)), dim3(otf::kEvictThreads), 0, s,
                                  (unsigned)ctas, f.lengths, f.kv_heads, f.capacity, weights, ldw, (int)budget,
                                  (int)recent, kept, ctas);
  if (e != cudaSuccess) return set_cuda_error(e);
  const otf::MoveArgs a = {f, t, kept, weights, weights_out, ldw, ldw_out, (int)budget, lengths_out};
  if (in_place) {
    const int columns = (int)(from->head_dim / 32);
    e = otf::launch_pdl(otf::k_evict_shift, dim3((unsigned)pairs, 2 * columns + 1), dim3(128), 0, s, 1u, a, columns);
    if (e != cudaSuccess) return set_cuda_error(e);
    return set_cuda_error(otf::launch_pdl(otf::k_evict_lengths, dim3((unsigned)((f.batch + 255) / 256)), dim3(256), 0, s, 1u, a));
  }
  const int64_t tiles = (budget + otf::kMoveRows - 1) / otf::kMoveRows;
  return set_cuda_error(otf::launch_pdl(from->head_dim == 128 ? otf::k_evict_copy<128> : otf::k_evict_copy<64>,
                                        dim3((unsigned)pairs, (unsigned)tiles), dim3(256), 0, s, 1u, a));
}

extern "C" OTF_API int otf_paged_keep(const otf_paged_cache* cache, const int32_t* path, int64_t ld_path,
                                      const int32_t* accepted, int64_t depth, void* stream) {
  otf::PagedView c;
  int st = otf::view_of(cache, c);
  if (st != OTF_OK) return st;
  if (!accepted || depth < 0 || (depth && (!path || ld_path < depth))) return OTF_ERR_INVALID;
  if (depth > otf::kKeepMost) return OTF_ERR_UNSUPPORTED;
  st = check_device();
  if (st != OTF_OK || depth == 0) return st;
  const int64_t bytes = 2 * depth * cache->head_dim * 2;
  return set_cuda_error(otf::launch_pdl(cache->head_dim == 128 ? otf::k_paged_keep<128> : otf::k_paged_keep<64>,
                                        dim3((unsigned)c.kv_heads, (unsigned)c.batch), dim3(otf::kKeepThreads), (size_t)bytes,
                                        static_cast<cudaStream_t>(stream), 1u, c, path, ld_path, accepted, (int)depth));
}
