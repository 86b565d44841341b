// Attention of rows of any number per sequence over a key/value cache in pages (otf_paged_attn_rows):
// prompts and decoded tokens, through a sliding window with some first tokens that stay visible, and
// trees of drafted tokens.
//
// Mathematics.  A row sees the keys of a set that a few numbers describe: the first `sinks` ones and
// those from `lo` to `hi`, or (trees) to the last cached one and the nodes of a 64-bit mask.  With
// s_j = scale log2(e) q k_j one pass over the keys keeps a reference m near the running maximum,
// l = sum_j 2^(s_j - m) and o = sum_j 2^(s_j - m) v_j; out = o / l.  Parts (m, l, o) of disjoint key
// ranges join as M = max m, L = sum l 2^(m - M), O = sum o 2^(m - M).
//
// Split.  An item is a (sequence, block of rows, KV head), the rows being (token, query head of the KV
// head) in that order; its keys are cut into chunks of 128, of which those that no row sees are left
// out.  All items' chunks, in order, are dealt out evenly to one CTA per SM in contiguous runs: a run
// may cross items, and an item may be shared by several CTAs, which then leave parts that a second
// kernel joins in order.  Lengths and row ranges are read on the device, so that a step can be captured.
//
// A CTA has two groups of four warps that turn scores into probabilities, a thread per row; a warp that
// issues the matrix products (tcgen05, 128 rows x 128 keys and 128 rows x head_dim, scores, probabilities
// and outputs in tensor memory); a warp that fetches queries, and four that fetch keys and values through
// a ring of shared-memory slots by 16-byte asynchronous copies, page by page, whatever the page size is.
// TILES 2, for many rows: the groups have 128 rows each and share every chunk.  TILES 1, for few rows:
// the groups have the same rows and every other chunk each, and join at the item's end.
#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace otf {

int set_cuda_error(cudaError_t e);       // capi.cu
int check_device();                      // capi.cu
int paged_rows_device_error(int clear);  // read (and optionally clear) the flag below

constexpr int kPrKeys = 128;      // keys of a chunk
constexpr int kPrGrid = 148;      // a CTA on each SM
constexpr int kPrMma = 8, kPrQuery = 9, kPrScan = 10, kPrLoad = 12;  // that issue products, fetch queries, look values through (2), fetch keys (4)
constexpr int kPrThreads = 512;
// Registers: 128 a thread at launch, of which half of the threads give 32 to the others, which hold rows.
constexpr int kPrRowRegs = 160, kPrOtherRegs = 96;
constexpr int kPrMaxNodes = 64;
constexpr int kPrItemUnits = 2;   // what an item's start and end cost, in chunks
constexpr float kPrLog2e = 1.4426950408889634f;

// Set when a sequence does not fit its pages, names a page outside the pool, or has rows or parents out of range.
__device__ int g_paged_rows_device_error;
__device__ __forceinline__ void report_bad_rows() { atomicExch(&g_paged_rows_device_error, 1); }

// The item that several CTAs share and that begins in a CTA's run.
struct __align__(16) SharedItem {
  int there, b, rb, g;
  int first_part, last_cta, pad[2];
};

struct RowsArgs {
  PagedView c;
  FastDiv page, rep_div;
  const uint16_t* q;
  int64_t ldq;
  uint16_t* out;
  int64_t ldo;
  const int* starts;   // or null: `per` rows each
  const int* parents;  // or null: rows in a line
  int per, n, rep;
  int window, sinks;   // window 0: none
  float scale;         // |scale| log2(e)
  uint32_t sign;       // of the scale, on two 16-bit queries
  float* part;         // [2 x grid][rows of a block][head_dim]: o of a part
  float2* part_ml;     // [2 x grid][rows of a block]: its m and l
  SharedItem* shared;  // [grid]
};

__device__ __forceinline__ float pr_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The reference m of a row follows its maximum only when a score rises 2^7 above it: probabilities reach
// 2^(shift + 7), 2^15 in fp16, and what lies 2^-32 below the reference still counts there.
constexpr float kPrHeadroom = 7.0f;
template <bool BF>
constexpr float kPrShift = BF ? 0.0f : 8.0f;

// ---- what a row sees --------------------------------------------------------------------------

// A sequence's rows: `tokens` of them from row `r0` on, behind `len` cached tokens.  tokens 0: nothing to do.
struct RowRange {
  int tokens, len, r0;
};
template <bool TREE>
__device__ __forceinline__ RowRange range_of(const RowsArgs& a, int b, bool report) {
  RowRange s;
  s.len = a.c.lengths[b];
  s.r0 = a.starts ? a.starts[b] : b * a.per;
  const int end = a.starts ? a.starts[b + 1] : s.r0 + a.per;
  s.tokens = end - s.r0;
  if (s.len < 0) s.tokens = 0;
  if (s.len >= 0 && (s.r0 < 0 || end < s.r0 || end > a.n || (int64_t)s.len + s.tokens > a.c.capacity ||
                     (TREE && s.tokens > kPrMaxNodes))) {
    if (report) report_bad_rows();
    s.tokens = 0;
  }
  return s;
}

// The keys of a block of rows: those in [0, sinks) and [low, end), in chunks: `sink_chunks` from the first
// key on, then those from chunk `low_chunk` on.  From key `full` on a row may not see a key that another does,
// and so below key `low_full`, from the sinks on.
struct Keys {
  int t0, t1;  // its first and last token
  int low, low_full, full, end, sink_chunks, low_chunk, chunks;
};
template <bool TREE, int ROWS>
__device__ __forceinline__ Keys keys_of(const RowsArgs& a, const RowRange& s, int rb) {
  Keys k;
  const int row0 = rb * ROWS, row1 = min(s.tokens * a.rep, row0 + ROWS);
  k.t0 = (uint32_t)row0 / a.rep_div;
  k.t1 = (uint32_t)(row1 - 1) / a.rep_div;
  k.low = k.low_full = k.sink_chunks = k.low_chunk = 0;
  if (a.window) {
    k.low = max(0, s.len + (TREE ? 0 : k.t0) - a.window + 1);
    k.low_full = max(0, s.len + (TREE ? s.tokens - 1 : k.t1) - a.window + 1);
    k.low_chunk = k.low / kPrKeys;
    k.sink_chunks = min((a.sinks + kPrKeys - 1) / kPrKeys, k.low_chunk);
  }
  k.full = TREE ? s.len : s.len + k.t0 + 1;
  k.end = TREE ? s.len + s.tokens : s.len + k.t1 + 1;
  k.chunks = k.sink_chunks + (k.end + kPrKeys - 1) / kPrKeys - k.low_chunk;
  return k;
}
// The first key of chunk v.
__device__ __forceinline__ int first_key(const Keys& k, int v) {
  return (v < k.sink_chunks ? v : k.low_chunk + v - k.sink_chunks) * kPrKeys;
}

// Whether a chunk has keys that some of the block's rows see and others do not, beyond a single token's.
__device__ __forceinline__ bool some_do_not_see(const Keys& k, int v, int sinks) {
  const int k0 = first_key(k, v);
  return k.t1 > k.t0 && (k0 + kPrKeys > k.full || (k0 < k.low_full && k0 + kPrKeys > sinks));
}

// What one row sees.
struct RowView {
  int lo, hi;  // keys lo .. hi; trees: lo .. hi and the nodes of `nodes` behind them
  uint64_t nodes;
};
__device__ __forceinline__ uint32_t ones(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
// Which of the 32 keys from k0 on.
template <bool TREE>
__device__ __forceinline__ uint32_t seen32(const RowsArgs& a, const RowView& v, int k0) {
  uint32_t x = ones(v.hi + 1 - k0) & (~ones(v.lo - k0) | ones(a.sinks - k0));
  if (TREE) {
    const int at = k0 - v.hi - 1;  // of the first key among the nodes
    if (at > -32 && at < kPrMaxNodes) x |= (uint32_t)(at >= 0 ? v.nodes >> at : v.nodes << -at);
  }
  return x;
}

// ---- a CTA's run ------------------------------------------------------------------------------

struct RunStart {
  int64_t u0, u1, total, ctas, at;  // its units; where its first item begins
  int b, rb, g, pad;
};

// An item of a run, with the chunks [c0, c1) that the run has of it.
template <bool TREE, int ROWS>
struct Item {
  const RowsArgs& a;
  const int64_t u0, u1;
  int64_t at;
  int b, rb, g, c0, c1;
  RowRange s;
  Keys k;
  bool first = true;  // of the run

  __device__ __forceinline__ Item(const RowsArgs& args, const RunStart& r)
      : a(args), u0(r.u0), u1(r.u1), at(r.at), b(r.b), rb(r.rb), g(r.g) {}
  __device__ __forceinline__ bool clip() {
    c0 = (int)max((int64_t)0, u0 - at - kPrItemUnits);
    c1 = (int)min((int64_t)k.chunks, u1 - at - kPrItemUnits);
    return c1 > c0;
  }
  __device__ __forceinline__ bool begin() {
    if (u0 >= u1) return false;
    s = range_of<TREE>(a, b, false);
    k = keys_of<TREE, ROWS>(a, s, rb);
    return clip() || next_with_chunks();
  }
  __device__ __forceinline__ bool next() {
    first = false;
    return next_with_chunks();
  }
  __device__ __forceinline__ bool next_with_chunks() {
    do {
      at += k.chunks + kPrItemUnits;
      if (at + kPrItemUnits >= u1) return false;
      if (++g == a.c.kv_heads) {
        g = 0;
        if ((int64_t)(++rb) * ROWS >= (int64_t)s.tokens * a.rep) {
          rb = 0;
          do {
            if (++b >= a.c.batch) return false;
            s = range_of<TREE>(a, b, false);
          } while (s.tokens == 0);
        }
        k = keys_of<TREE, ROWS>(a, s, rb);
      }
    } while (!clip());
    return true;
  }
  __device__ __forceinline__ bool whole() const { return c0 == 0 && c1 == k.chunks; }
};

template <int D, int TILES>
struct RowsShape {
  static constexpr int rows = 128 * TILES;
  static constexpr int tile = 128 * D * 2;               // bytes of 128 queries, keys or values
  static constexpr int slots = D == 128 ? 5 : 10;        // of the ring
  static constexpr int meet = TILES == 1 ? 128 * 64 * 4 : 0;  // where the groups' outputs meet, 64 columns at a time
  static constexpr int ring = TILES * tile + meet;
  static constexpr int small = ring + slots * tile;      // barriers and the like
  static constexpr int bytes = 1024 + small + 2048;
};

// The small part of the shared memory, behind the ring.
struct RowsSmall {
  uint64_t kv_full[10], kv_empty[10], v_landed[10];
  uint64_t q_full[2], q_empty[2], s_full[2], p_full[2], o_done[2];
  RunStart run;
  int64_t sums[16];
  float2 ml[128];
  uint32_t tmem;
  int gave_up;   // a wait ran out: no more waiting
  int odd;       // an infinity or NaN was taken out of some values
};
static_assert(sizeof(RowsSmall) <= 2048, "");

// A bounded wait: after a second the CTA gives up, raises the flag and runs to its end without waiting.
__device__ __forceinline__ void rows_wait(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
  const uint32_t at = smem_u32(bar);
  if (mbar_try_wait(at, parity)) return;
  const uint64_t t0 = global_ns();
  while (!*gave_up) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (mbar_try_wait(at, parity)) return;
    if (global_ns() - t0 > 1000000000ull) {
      *gave_up = 1;
      report_bad_rows();
    }
  }
}

__device__ __forceinline__ void mbar_arrive_n(uint32_t addr, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(addr), "r"(n) : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 lanes x 32 consecutive 32-bit columns of tensor memory, complete on return, and back.
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
// The descriptor of 16-bit values stored [key][64 dims] in 128-byte swizzled rows, eight keys in 1024
// bytes, the next 64 dims 128 keys on, as the operand whose contraction runs over the keys.
__device__ __forceinline__ uint64_t values_desc(uint32_t at) {
  return (uint64_t)((at >> 4) & 0x3FFFu) | ((uint64_t)(128 * 128 >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) |
         ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}

// Whether one of two 16-bit values is an infinity or NaN.
template <bool BF>
__device__ __forceinline__ bool odd2(uint32_t x) {
  constexpr uint32_t e = BF ? 0x7F80u : 0x7C00u;
  return (x & e) == e || (x & (e << 16)) == e << 16;
}
template <bool BF>
__device__ __forceinline__ uint32_t without_odd2(uint32_t x) {
  constexpr uint32_t e = BF ? 0x7F80u : 0x7C00u;
  if ((x & e) == e) x &= 0xffff0000u;
  if ((x & (e << 16)) == e << 16) x &= 0xffffu;
  return x;
}

// Offset of key s of sequence b in the pools, -1 where its page lies outside.
__device__ __forceinline__ int64_t key_place(const RowsArgs& a, int b, int s) {
  const uint32_t in = (uint32_t)s / a.page;
  const int page = a.c.table[b * a.c.ld_table + in];
  if (page < 0 || page >= a.c.n_pages) {
    report_bad_rows();
    return -1;
  }
  return page * a.c.page_stride + (int64_t)(s - (int)(in * a.page.d)) * a.c.token_stride;
}

// The infinities and NaN that were taken out of a block's values, given back to the rows that see them:
// columns [col, col + 32) of the outputs o that a warp's lanes hold a row of each.
template <bool BF, int D, bool TREE, int ROWS>
__device__ __noinline__ void add_odd(const Item<TREE, ROWS>& it, const RowView& view, float* o, int col) {
  const RowsArgs& a = it.a;
  for (int v = it.c0; v < it.c1; ++v) {
    if (!some_do_not_see(it.k, v, a.sinks)) continue;
    const int k0 = first_key(it.k, v);
    for (int s = k0; s < min(k0 + kPrKeys, it.k.end); ++s) {
      if (s < it.k.low && s >= a.sinks) continue;
      const int64_t at = key_place(a, it.b, s);
      if (at < 0) continue;
      const uint16_t* x = a.c.v + at + it.g * a.c.head_stride + col;
      const float mine = to_f<BF>(x[threadIdx.x & 31]);
      if (!__any_sync(0xffffffffu, !isfinite(mine))) continue;
      const bool sees = (seen32<TREE>(a, view, s & ~31) >> (s & 31)) & 1u;
      for (int i = 0; i < 32; ++i) {
        const float y = __shfl_sync(0xffffffffu, mine, i);
        if (sees && !isfinite(y)) o[i] += y;
      }
    }
  }
}

// ---- the kernel -------------------------------------------------------------------------------

template <bool BF, int D, int TILES, bool TREE>
__global__ void __launch_bounds__(kPrThreads, 1) k_paged_rows(const __grid_constant__ RowsArgs a) {
  using S = RowsShape<D, TILES>;
  using It = Item<TREE, S::rows>;
  constexpr int NS = S::slots;
  constexpr uint32_t kFormat = (1u << 4) | (BF ? 1u << 7 | 1u << 10 : 0u) | ((uint32_t)(128 >> 4) << 24);
  constexpr uint32_t kScores = kFormat | ((uint32_t)(kPrKeys >> 3) << 17);
  constexpr uint32_t kOutputs = kFormat | ((uint32_t)(D >> 3) << 17) | (1u << 16);  // values: keys across
  constexpr uint32_t kOut = 256;  // tensor memory: 128 columns of scores for each group, then its outputs
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  RowsSmall& sm = *reinterpret_cast<RowsSmall*>(smem + S::small);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_trigger();
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(smem_u32(&sm.kv_full[i]), 128);
      mbar_init(smem_u32(&sm.v_landed[i]), 128);
      mbar_init(smem_u32(&sm.kv_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sm.q_full[i]), 1);
      mbar_init(smem_u32(&sm.q_empty[i]), 1);
      mbar_init(smem_u32(&sm.s_full[i]), 1);
      mbar_init(smem_u32(&sm.p_full[i]), 4);
      mbar_init(smem_u32(&sm.o_done[i]), 1);
    }
    mbar_fence_init();
    sm.gave_up = sm.odd = 0;
  }
  if (warp == kPrMma) {
    tmem_alloc(smem_u32(&sm.tmem), 512);
    tmem_relinquish();
  }
  pdl_wait();

  // every sequence's units, then this CTA's run
  {
    int64_t* units = reinterpret_cast<int64_t*>(smem + S::ring);
    int64_t sum = 0;
    for (int b = warp; b < a.c.batch; b += kPrThreads / 32) {
      const RowRange s = range_of<TREE>(a, b, blockIdx.x == 0 && lane == 0);
      int64_t x = 0;
      for (int rb = lane; (int64_t)rb * S::rows < (int64_t)s.tokens * a.rep; rb += 32)
        x += keys_of<TREE, S::rows>(a, s, rb).chunks + kPrItemUnits;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      x *= a.c.kv_heads;
      if (lane == 0) units[b] = x;
      sum += x;
    }
    if (lane == 0) sm.sums[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      int64_t total = lane < kPrThreads / 32 ? sm.sums[lane] : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      RunStart r = {};
      r.total = total;
      r.ctas = max((int64_t)1, min((int64_t)kPrGrid, total / (kPrItemUnits + 1)));
      r.u0 = blockIdx.x < r.ctas ? blockIdx.x * total / r.ctas : total;
      r.u1 = blockIdx.x < r.ctas ? (blockIdx.x + 1) * total / r.ctas : total;
      if (lane == 0) sm.run = r;
      __syncwarp();
      int64_t base = 0;
      int found = -1;
      for (int b0 = 0; b0 < a.c.batch && r.u0 < r.u1; b0 += 32) {
        const int64_t mine = b0 + lane < a.c.batch ? units[b0 + lane] : 0;
        int64_t inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += x;
        }
        const uint32_t in = __ballot_sync(0xffffffffu, r.u0 >= base + inc - mine && r.u0 < base + inc);
        if (in) {
          found = b0 + __ffs((int)in) - 1;
          base += __shfl_sync(0xffffffffu, inc - mine, __ffs((int)in) - 1);
          break;
        }
        base += __shfl_sync(0xffffffffu, inc, 31);
      }
      if (found >= 0) {
        const RowRange s = range_of<TREE>(a, found, false);
        for (int r0 = 0;; r0 += 32) {
          const int per = (int64_t)(r0 + lane) * S::rows < (int64_t)s.tokens * a.rep
                              ? keys_of<TREE, S::rows>(a, s, r0 + lane).chunks + kPrItemUnits : 0;
          const int64_t mine = (int64_t)per * a.c.kv_heads;
          int64_t inc = mine;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += x;
          }
          if (mine && r.u0 >= base + inc - mine && r.u0 < base + inc) {
            const int64_t off = r.u0 - (base + inc - mine);
            sm.run.b = found;
            sm.run.rb = r0 + lane;
            sm.run.g = (int)(off / per);
            sm.run.at = base + inc - mine + off / per * per;
          }
          base += __shfl_sync(0xffffffffu, inc, 31);
          if (base > r.u0 || __all_sync(0xffffffffu, mine == 0)) break;
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&sm.tmem);
  const RunStart run = sm.run;
  It it(a, run);
  volatile int* gave_up = &sm.gave_up;

  if (warp >= 8)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPrOtherRegs));
  else
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPrRowRegs));

  if (warp >= kPrLoad) {
    // Keys and values: chunk after chunk a slot of keys, then one of values, 32 rows a warp.
    constexpr int P = D / 8, R = 32 / P;  // 16-byte pieces of a row, rows of a copy instruction
    const int w = warp - kPrLoad, piece = lane % P, sub = lane / P;
    const uint32_t ring = smem_u32(smem + S::ring);
    const uint32_t to = (uint32_t)((piece >> 3) * 128 * 128 + (32 * w + sub) * 128);
    uint32_t fill = 0;
    auto places = [&](int v) -> int64_t {
      const int s = first_key(it.k, v) + 32 * w + lane;
      return s < it.k.end && (s >= it.k.low || s < a.sinks) ? key_place(a, it.b, s) : -1;
    };
    auto put = [&](const uint16_t* base, int64_t place, uint64_t* full) {
      const uint32_t slot = fill % NS;
      if (fill >= NS) rows_wait(&sm.kv_empty[slot], (fill / NS - 1) & 1u, gave_up);
      const uint32_t dst = ring + slot * S::tile + to;
#pragma unroll
      for (int i = 0; i < 32 / R; ++i) {
        const int64_t at = __shfl_sync(0xffffffffu, place, sub + i * R);
        cp_async16(dst + i * R * 128 + (((piece & 7) ^ ((sub + i * R) & 7)) << 4), base + (at >= 0 ? at : 0), at >= 0 ? 16u : 0u);
      }
      cp_async_mbar_arrive(smem_u32(full + slot));  // when they have landed
      ++fill;
    };
    if (it.begin()) {
      int64_t place = places(it.c0);
      int v = it.c0;
      for (;;) {
        const bool odd = some_do_not_see(it.k, v, a.sinks);
        const int64_t head = it.g * a.c.head_stride + piece * 8, now = place;
        bool more = true;
        if (++v == it.c1) {
          more = it.next();
          v = it.c0;
        }
        if (more) place = places(v);
        put(a.c.k + head, now, sm.kv_full);
        put(a.c.v + head, now, odd ? sm.v_landed : sm.kv_full);
        if (!more) break;
      }
    }
    cp_async_wait<0>();
  } else if (warp >= kPrScan) {
    // Values that not every row of the block sees: a weight of 0 does not keep an infinity or NaN from a row, so
    // they are taken out before the products (and given back at the item's end).  A warp has half of a slot.
    const int h = warp - kPrScan;
    uint32_t fill = 0;
    uint32_t turns = 0;  // how often each slot's landing came around, a bit per slot
    for (bool more = it.begin(); more; more = it.next())
      for (int v = it.c0; v < it.c1; ++v, fill += 2) {
        if (!some_do_not_see(it.k, v, a.sinks)) continue;
        const uint32_t slot = (fill + 1) % NS;
        rows_wait(&sm.v_landed[slot], turns >> slot & 1u, gave_up);
        turns ^= 1u << slot;
        uint4* x = reinterpret_cast<uint4*>(smem + S::ring + slot * S::tile + h * (S::tile / 2));
        bool odd = false;
#pragma unroll 4
        for (int i = lane; i < S::tile / 32; i += 32) {
          const uint4 y = x[i];
          if (odd2<BF>(y.x) || odd2<BF>(y.y) || odd2<BF>(y.z) || odd2<BF>(y.w)) {
            x[i] = make_uint4(without_odd2<BF>(y.x), without_odd2<BF>(y.y), without_odd2<BF>(y.z), without_odd2<BF>(y.w));
            odd = true;
          }
        }
        if (odd) *(volatile int*)&sm.odd = 1;
        __syncwarp();
        if (lane == 0) mbar_arrive_n(smem_u32(&sm.kv_full[slot]), 64);
      }
  } else if (warp == kPrQuery) {
    // Queries: rows that there are, 128 of a tile; the others' scores are never looked at.
    constexpr int P = D / 8, R = 32 / P;
    const int piece = lane % P, sub = lane / P;
    uint32_t n = 0;
    for (bool more = it.begin(); more; more = it.next(), ++n)
      for (int w = 0; w < TILES; ++w) {
        if (n > 0) rows_wait(&sm.q_empty[w], (n - 1) & 1u, gave_up);
        const int row0 = it.rb * S::rows + w * 128, rows = min(128, it.s.tokens * a.rep - row0);
        unsigned char* tile = smem + w * S::tile + (piece >> 3) * 128 * 128;
        for (int r = sub; r < rows; r += R) {
          const uint32_t row = row0 + r, t = row / a.rep_div;
          const uint16_t* x = a.q + (it.s.r0 + (int64_t)t) * a.ldq + (int64_t)(it.g * a.rep + row - t * a.rep) * D + piece * 8;
          cp_async16(smem_u32(tile + r * 128 + (((piece & 7) ^ (r & 7)) << 4)), x, 16u);
        }
        cp_async_commit();
        cp_async_wait<0>();
        if (a.sign)  // a negative scale's, so that a larger product weighs more
          for (int r = sub; r < rows; r += R) {
            uint4* x = reinterpret_cast<uint4*>(tile + r * 128 + (((piece & 7) ^ (r & 7)) << 4));
            const uint4 y = *x;
            *x = make_uint4(y.x ^ a.sign, y.y ^ a.sign, y.z ^ a.sign, y.w ^ a.sign);
          }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.q_full[w]));
      }
  } else if (warp == kPrMma) {
    if (lane == 0) {
      uint32_t items = 0, fill = 0, probs[2] = {0, 0};
      const uint32_t q0 = smem_u32(smem), ring = smem_u32(smem + S::ring);
      auto scores = [&](int w, uint32_t f) {  // of group w, from the keys of fill f
        const uint32_t q = q0 + (TILES == 2 ? w : 0) * S::tile, k = ring + f % NS * S::tile;
#pragma unroll
        for (int x = 0; x < D / 16; ++x)
          tc_mma_f16(tmem + w * 128, tc_desc_sw128(q + (x >> 2) * 128 * 128 + (x & 3) * 32),
                     tc_desc_sw128(k + (x >> 2) * 128 * 128 + (x & 3) * 32), kScores, x > 0);
        tc_commit(smem_u32(&sm.s_full[w]));
      };
      auto outputs = [&](int w, uint32_t f, bool add) {  // of group w, from the values of fill f
        const uint32_t v = ring + f % NS * S::tile, p = tmem + w * 128;
#pragma unroll
        for (int x = 0; x < kPrKeys / 16; ++x) {
          if (TILES == 2) {
            tc_mma_f16_ta(tmem + kOut + w * 128, p + 8 * x, values_desc(v + x * 2048), kOutputs, add || x > 0);
          } else {
            tc_mma_f16_ta(tmem + kOut + w * 128, p + 32 * (x >> 1) + 8 * (x & 1), values_desc(v + x * 2048), kOutputs, add || x > 0);
            tc_mma_f16_ta(tmem + kOut + w * 128, p + 32 * (x >> 1) + 8 * (x & 1) + 16, values_desc(v + x * 2048), kOutputs, 1u);
          }
        }
      };
      auto filled = [&](uint32_t f) {
        rows_wait(&sm.kv_full[f % NS], f / NS & 1u, gave_up);
        fence_async_shared();  // the copies are of the generic proxy, the products of the other
      };
      auto release = [&](uint32_t f) { tc_commit(smem_u32(&sm.kv_empty[f % NS])); };
      auto ready = [&](int w) {
        rows_wait(&sm.p_full[w], probs[w] & 1u, gave_up);
        ++probs[w];
        tc_fence_after_sync();
      };
      for (bool more = it.begin(); more; more = it.next(), ++items) {
        const int m = it.c1 - it.c0;
        for (int w = 0; w < TILES; ++w) rows_wait(&sm.q_full[w], items & 1u, gave_up);
        tc_fence_after_sync();
        if (TILES == 2) {
          filled(fill);
          scores(0, fill);
          scores(1, fill);
          release(fill);
          for (int j = 0; j < m; ++j, fill += 2) {
            filled(fill + 1);
            ready(0);
            outputs(0, fill + 1, j > 0);
            if (j + 1 < m) {
              filled(fill + 2);
              scores(0, fill + 2);
            } else {
              tc_commit(smem_u32(&sm.q_empty[0]));
              tc_commit(smem_u32(&sm.o_done[0]));
            }
            ready(1);
            outputs(1, fill + 1, j > 0);
            release(fill + 1);
            if (j + 1 < m) {
              scores(1, fill + 2);
              release(fill + 2);
            } else {
              tc_commit(smem_u32(&sm.q_empty[1]));
              tc_commit(smem_u32(&sm.o_done[1]));
            }
          }
        } else {
          for (int j = 0; j < min(m, 2); ++j) {
            filled(fill + 2 * j);
            scores(j, fill + 2 * j);
            release(fill + 2 * j);
          }
          if (m <= 2) tc_commit(smem_u32(&sm.q_empty[0]));
          for (int j = 0; j < m; ++j, fill += 2) {
            const int w = j & 1;
            filled(fill + 1);
            ready(w);
            outputs(w, fill + 1, j > 1);
            release(fill + 1);
            if (j + 2 < m) {
              filled(fill + 4);
              scores(w, fill + 4);
              release(fill + 4);
              if (j + 3 == m) tc_commit(smem_u32(&sm.q_empty[0]));
            } else {
              tc_commit(smem_u32(&sm.o_done[w]));
            }
          }
        }
      }
    }
    __syncwarp();
  } else if (warp < 8) {
    // The rows: thread r of group w has row r of its tile, which is lane r of tensor memory.
    const int w = warp >> 2, r = tid & 127, quarter = warp & 3;
    const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
    const uint32_t s_at = tmem + lanes + w * 128, o_at = tmem + lanes + kOut + w * 128;
    uint32_t chunk_count = 0, item_count = 0;
    for (bool more = it.begin(); more; more = it.next()) {
      const int row = it.rb * S::rows + (TILES == 2 ? w * 128 : 0) + r, rows = it.s.tokens * a.rep;
      const bool there = row < rows, warp_there = row - lane < rows;
      const int t = there ? (int)((uint32_t)row / a.rep_div) : it.k.t1;
      RowView view;
      if (TREE) {
        // the way up, through the nodes' parents in the lanes
        int up[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = lane + 32 * h;
          up[h] = i < it.s.tokens ? a.parents[it.s.r0 + i] : -1;
          if (up[h] >= i || up[h] < -1) {
            report_bad_rows();
            up[h] = -1;
          }
        }
        view.nodes = 0;
        for (int at = t; __any_sync(0xffffffffu, at >= 0);) {
          const int x = __shfl_sync(0xffffffffu, up[0], at & 31), y = __shfl_sync(0xffffffffu, up[1], at & 31);
          if (at >= 0) {
            view.nodes |= 1ull << at;
            at = at < 32 ? x : y;
          }
        }
        view.hi = it.s.len - 1;
        view.lo = a.window ? it.s.len + __popcll(view.nodes) - a.window : 0;
      } else {
        view.hi = it.s.len + t;
        view.lo = a.window ? view.hi - a.window + 1 : 0;
        view.nodes = 0;
      }
      float m = -INFINITY, l = 0.0f;
      bool any = false;  // a chunk of this group came before
      for (int v = it.c0 + (TILES == 1 ? w : 0); v < it.c1; v += TILES == 1 ? 2 : 1) {
        rows_wait(&sm.s_full[w], chunk_count & 1u, gave_up);
        ++chunk_count;
        tc_fence_after_sync();
        if (warp_there) {
          const int k0 = first_key(it.k, v);
          const bool edge = k0 + kPrKeys > it.k.full || (k0 < it.k.low_full && k0 + kPrKeys > a.sinks);
          uint32_t see[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) see[c] = edge ? seen32<TREE>(a, view, k0 + 32 * c) : 0xffffffffu;
          auto load = [&](int c, float (&s)[32]) {
            uint32_t x[32];
            tmem_ld32(s_at + 32 * c, x);
#pragma unroll
            for (int i = 0; i < 32; ++i) s[i] = __uint_as_float(x[i]);
            if (edge)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(see[c] >> i & 1u)) s[i] = -INFINITY;
          };
          float top = -INFINITY;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float s[32];
            load(c, s);
#pragma unroll
            for (int i = 0; i < 32; ++i) top = fmaxf(top, s[i]);
          }
          top *= a.scale;
          // lanes without a row hold what happens to lie there
          if (__any_sync(0xffffffffu, there && top > (m == -INFINITY ? -INFINITY : m + kPrHeadroom))) {
            const float mx = fmaxf(m, top), f = m == -INFINITY ? 0.0f : pr_ex2(m - mx);
            m = mx;
            l *= f;
            // the scores of a chunk are complete after the outputs of the one before it
            if (any)
#pragma unroll 1
              for (int c = 0; c < D; c += 32) {
                uint32_t x[32];
                tmem_ld32(o_at + c, x);
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * f);
                tmem_st32(o_at + c, x);
              }
          }
          const float z = kPrShift<BF> - (m == -INFINITY ? 0.0f : m);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float s[32];
            load(c, s);
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              s[i] = pr_ex2(fmaf(s[i], a.scale, z));
              sum[i & 3] += s[i];
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if (TILES == 2) {
              uint32_t p[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) p[i] = pack2<BF>(s[2 * i], s[2 * i + 1]);
              tmem_st16(s_at + 16 * c, p);
            } else {
              uint32_t p[32];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                p[i] = pack2<BF>(s[2 * i], s[2 * i + 1]);
                const float2 y = unpack2<BF>(p[i]);
                p[16 + i] = pack2<BF>(s[2 * i] - y.x, s[2 * i + 1] - y.y);
              }
              tmem_st32(s_at + 32 * c, p);
            }
          }
          tmem_wait_st();
        }
        any = true;
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.p_full[w]));
      }

      // The item's end in this run.
      if (any) {
        rows_wait(&sm.o_done[w], item_count & 1u, gave_up);
        ++item_count;
        tc_fence_after_sync();
      }
      const bool two = TILES == 1 && it.c1 - it.c0 > 1;  // the groups meet
      float f0 = 1.0f, f1 = 0.0f;
      const bool whole = it.whole();
      const int64_t part = (int64_t)(2 * blockIdx.x + (it.first ? 0 : 1)) * S::rows + (TILES == 2 ? w * 128 : 0) + r;
      const bool odd = *(volatile int*)&sm.odd;
#pragma unroll 1
      for (int half = 0; half < (TILES == 1 ? D / 64 : 1); ++half) {
        float* meet = reinterpret_cast<float*>(smem + TILES * S::tile) + r * 64;
        if (two) {
          if (w == 1 && warp_there) {
#pragma unroll 1
            for (int c = 0; c < 64; c += 32) {
              uint32_t x[32];
              tmem_ld32(o_at + half * 64 + c, x);
              if (there)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  *reinterpret_cast<uint4*>(meet + ((((c >> 2) + i) ^ (r & 15)) << 2)) =
                      make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
            }
            if (half == 0) sm.ml[r] = make_float2(m, l);
          }
          named_barrier_sync(1, 256);
          if (w == 0 && half == 0) {
            const float2 ml = sm.ml[r];
            const float mx = fmaxf(m, ml.x);
            f0 = m == -INFINITY ? 0.0f : pr_ex2(m - mx);
            f1 = ml.x == -INFINITY ? 0.0f : pr_ex2(ml.x - mx);
            m = mx;
            l = l * f0 + ml.y * f1;
          }
        }
        if ((TILES == 2 || w == 0) && warp_there) {
          const float inv = whole ? 1.0f / l : 1.0f;
          const int head = it.g * a.rep + row - t * a.rep;
#pragma unroll 1
          for (int c = TILES == 1 ? half * 64 : 0; c < (TILES == 1 ? half * 64 + 64 : D); c += 32) {
            uint32_t x[32];
            float o[32];
            tmem_ld32(o_at + c, x);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(x[i]);
            if (two && there) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 y = *reinterpret_cast<const float4*>(meet + (((((c & 63) >> 2) + i) ^ (r & 15)) << 2));
                o[4 * i] = fmaf(o[4 * i], f0, y.x * f1);
                o[4 * i + 1] = fmaf(o[4 * i + 1], f0, y.y * f1);
                o[4 * i + 2] = fmaf(o[4 * i + 2], f0, y.z * f1);
                o[4 * i + 3] = fmaf(o[4 * i + 3], f0, y.w * f1);
              }
            }
            if (odd) {
              const It here = it;  // copies: what lies in memory for the call
              const RowView mine = view;
              float y[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) y[i] = o[i];
              add_odd<BF, D>(here, mine, y, c);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = y[i];
            }
            if (there) {
              if (whole) {
                uint4* to = reinterpret_cast<uint4*>(a.out + (it.s.r0 + (int64_t)t) * a.ldo + (int64_t)head * D + c);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  to[i] = make_uint4(pack2<BF>(o[8 * i] * inv, o[8 * i + 1] * inv), pack2<BF>(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                     pack2<BF>(o[8 * i + 4] * inv, o[8 * i + 5] * inv), pack2<BF>(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
              } else {
                float4* to = reinterpret_cast<float4*>(a.part + part * D + c);
#pragma unroll
                for (int i = 0; i < 8; ++i) to[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
              }
            }
          }
          if (!whole && there && half == 0) a.part_ml[part] = make_float2(m, l);
        }
        if (two) named_barrier_sync(1, 256);  // before the columns are written again
      }
    }
  }

  // what the joining kernel needs of this run: the item that begins in it and goes on behind it
  if (tid == 0) {
    SharedItem x = {};
    It last(a, run);
    for (bool more = last.begin(); more; more = last.next())
      if (last.c0 == 0 && last.c1 < last.k.chunks) {
        const int64_t end = last.at + kPrItemUnits + last.k.chunks - 1;  // the unit of its last chunk
        x = SharedItem{1, last.b, last.rb, last.g, 2 * (int)blockIdx.x + (last.first ? 0 : 1),
                       (int)(((end + 1) * run.ctas - 1) / run.total), {0, 0}};
      }
    a.shared[blockIdx.x] = x;
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == kPrMma) tmem_dealloc(tmem, 512);
}

// The parts of an item that several CTAs shared, joined in the keys' order: grid (CTAs, rows / 8), a warp
// per row.
template <bool BF, int D, int TILES, bool TREE>
__global__ void __launch_bounds__(256) k_paged_rows_join(const __grid_constant__ RowsArgs a) {
  constexpr int ROWS = 128 * TILES, PL = D / 32;
  pdl_trigger();
  pdl_wait();
  const SharedItem x = a.shared[blockIdx.x];
  if (!x.there) return;
  const RowRange s = range_of<TREE>(a, x.b, false);
  const int lane = threadIdx.x & 31, r = blockIdx.y * 8 + (threadIdx.x >> 5), row = x.rb * ROWS + r;
  if (row >= s.tokens * a.rep) return;
  const int n = x.last_cta - (int)blockIdx.x + 1;
  auto part = [&](int i) { return (int64_t)(i == 0 ? x.first_part : 2 * ((int)blockIdx.x + i)) * ROWS + r; };
  float M = -INFINITY, L = 0.0f, acc[PL] = {};
  for (int i = lane; i < n; i += 32) M = fmaxf(M, a.part_ml[part(i)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float2 ml = a.part_ml[part(i)];
    const float f = ml.x == -INFINITY ? 0.0f : pr_ex2(ml.x - M);
    const float* y = a.part + part(i) * D + lane * PL;
    L = fmaf(ml.y, f, L);
    if (ml.x != -INFINITY)
#pragma unroll
      for (int j = 0; j < PL; ++j) acc[j] = fmaf(y[j], f, acc[j]);
  }
  const int t = (uint32_t)row / a.rep_div, head = x.g * a.rep + row - t * a.rep;
  uint32_t* to = reinterpret_cast<uint32_t*>(a.out + (s.r0 + (int64_t)t) * a.ldo + (int64_t)head * D + lane * PL);
#pragma unroll
  for (int j = 0; j < PL / 2; ++j) to[j] = pack2<BF>(acc[2 * j] / L, acc[2 * j + 1] / L);
}

// Blocks of 256 rows where sequences have more than 128 rows of a KV head on average.
static int rows_tiles(int64_t n, int64_t rep, int64_t batch) { return n * rep > 128 * batch ? 2 : 1; }

struct RowsSpace {
  int64_t part, part_ml, shared;
  int64_t bytes() const { return part + part_ml + shared; }
};
static RowsSpace rows_space(int64_t n, int64_t heads, int64_t kv_heads, int64_t D, int64_t batch) {
  const int64_t rows = 128 * rows_tiles(n, heads / kv_heads, batch);
  return RowsSpace{2 * kPrGrid * rows * D * 4, 2 * kPrGrid * rows * 8, align_up(kPrGrid * (int64_t)sizeof(SharedItem), 256)};
}
static bool rows_limits(int64_t batch, int64_t n, int64_t heads, int64_t kv_heads, int64_t D) {
  return batch <= kPagedMaxBatch && heads <= 65535 && kv_heads <= 1024 && (D == 64 || D == 128) && n <= INT32_MAX &&
         n * (heads / kv_heads) <= INT32_MAX;
}

template <bool BF, int D, int TILES, bool TREE>
static cudaError_t launch_rows(const RowsArgs& a, cudaStream_t s) {
  auto* k = k_paged_rows<BF, D, TILES, TREE>;
  constexpr int bytes = RowsShape<D, TILES>::bytes;
  static std::atomic<bool> done[64];
  int dev;
  bool needs;
  cudaError_t e = needs_opt_in(done, dev, needs);
  if (e != cudaSuccess) return e;
  if (needs) {
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    opted_in(done, dev);
  }
  e = launch_pdl(k, dim3(kPrGrid), dim3(kPrThreads), bytes, s, 1u, a);
  if (e != cudaSuccess) return e;
  return launch_pdl(k_paged_rows_join<BF, D, TILES, TREE>, dim3(kPrGrid, 16 * TILES), dim3(256), 0, s, 1u, a);
}
template <bool BF, int D>
static cudaError_t launch_rows_of(const RowsArgs& a, int tiles, cudaStream_t s) {
  if (a.parents) return tiles == 2 ? launch_rows<BF, D, 2, true>(a, s) : launch_rows<BF, D, 1, true>(a, s);
  return tiles == 2 ? launch_rows<BF, D, 2, false>(a, s) : launch_rows<BF, D, 1, false>(a, s);
}

}  // namespace otf

using otf::check_device;
using otf::set_cuda_error;

int otf::paged_rows_device_error(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, otf::g_paged_rows_device_error, sizeof(int)) != cudaSuccess) {
    set_cuda_error(cudaGetLastError());
    return -1;
  }
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(otf::g_paged_rows_device_error, &z, sizeof(int));
  }
  return v;
}

extern "C" OTF_API int64_t otf_paged_attn_rows_workspace_bytes(int64_t batch, int64_t n, int64_t heads, int64_t kv_heads,
                                                               int64_t head_dim) {
  if (batch <= 0 || n <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads ||
      !otf::rows_limits(batch, n, heads, kv_heads, head_dim))
    return -1;
  return otf::rows_space(n, heads, kv_heads, head_dim, batch).bytes();
}

extern "C" OTF_API int otf_paged_attn_rows(const otf_paged_cache* cache, const void* q, int64_t ldq, int64_t heads,
                                           const int32_t* starts, int64_t n, const int32_t* parents, int64_t window,
                                           int64_t sinks, float scale, void* out, int64_t ldo, void* workspace,
                                           int64_t workspace_bytes, void* stream) {
  otf::RowsArgs a = {};
  int st = otf::view_of(cache, a.c);
  if (st != OTF_OK) return st;
  const int64_t D = cache->head_dim;
  if (heads <= 0 || heads % a.c.kv_heads || n <= 0 || (!starts && n % a.c.batch) || !std::isfinite(scale * otf::kPrLog2e) ||
      window < 0 || sinks < 0 || (sinks && !window) || (parents && window && window < otf::kPrMaxNodes))
    return OTF_ERR_INVALID;
  if (!otf::rows_limits(a.c.batch, n, heads, a.c.kv_heads, D) || (parents && !starts && n / a.c.batch > otf::kPrMaxNodes))
    return OTF_ERR_UNSUPPORTED;
  if (!otf::rows16(q, ldq, heads * D) || !otf::rows16(out, ldo, heads * D)) return OTF_ERR_INVALID;
  if (otf::rows_overlap(q, ldq, heads * D, out, ldo, heads * D, n)) return OTF_ERR_INVALID;
  const otf::RowsSpace space = otf::rows_space(n, heads, a.c.kv_heads, D, a.c.batch);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < space.bytes())
    return OTF_ERR_INVALID;
  st = check_device();
  if (st != OTF_OK) return st;
  a.rep = (int)(heads / a.c.kv_heads);
  a.page = otf::fast_div((uint32_t)a.c.page_size);
  a.rep_div = otf::fast_div((uint32_t)a.rep);
  a.q = static_cast<const uint16_t*>(q);
  a.ldq = ldq;
  a.out = static_cast<uint16_t*>(out);
  a.ldo = ldo;
  a.starts = starts;
  a.parents = parents;
  a.per = starts ? 0 : (int)(n / a.c.batch);
  a.n = (int)n;
  // a window as long as any cache hides nothing
  a.window = window > (1ll << 30) ? 0 : (int)window;
  a.sinks = a.window ? (int)std::min<int64_t>(sinks, 1ll << 30) : 0;
  // a masked -inf stays one under a scale of 0, and no finite score counts under 2^-149
  a.scale = fmaxf(fabsf(scale * otf::kPrLog2e), 0x1p-149f);
  a.sign = scale < 0.0f ? 0x80008000u : 0u;
  char* w = static_cast<char*>(workspace);
  a.part = reinterpret_cast<float*>(w);
  a.part_ml = reinterpret_cast<float2*>(w + space.part);
  a.shared = reinterpret_cast<otf::SharedItem*>(w + space.part + space.part_ml);
  const int tiles = otf::rows_tiles(n, a.rep, a.c.batch);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = cache->dtype == OTF_DTYPE_BF16;
  return set_cuda_error(D == 128 ? (bf ? otf::launch_rows_of<true, 128>(a, tiles, s) : otf::launch_rows_of<false, 128>(a, tiles, s))
                                 : (bf ? otf::launch_rows_of<true, 64>(a, tiles, s) : otf::launch_rows_of<false, 64>(a, tiles, s)));
}
