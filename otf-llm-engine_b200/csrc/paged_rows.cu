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
// A CTA has two groups of four warps that turn scores into probabilities, a thread per row; a warp that issues the matrix
// products (tcgen05, 128 rows x 128 keys and 128 rows x head_dim, scores, probabilities and outputs in tensor memory); a warp
// that fetches queries and looks values through; and two that fetch keys and values through a ring of shared-memory slots:
// by tensor copies, a page at a time, where all of a chunk's keys are there, else by 16-byte copies.  Blocks of more than 128
// rows: the groups have 128 rows each and share every chunk.  Blocks of fewer: the groups have the same rows and every other
// chunk each, and join at the item's end; and where there are 64 rows or fewer they lie there two or four times, each copy
// with its own keys of a chunk (its other probabilities are 0), so that all warps have work.
//
// Bound.  Many rows: 4 head_dim flops a row and key on the matrix pipe and one exponential, of which an SM makes 16 a cycle:
// a chunk's 256 x 128 scores take it as long as their products, 2048 cycles, and the two overlap in part.  Few rows: keys and
// values are read once, 4 head_dim bytes a token and KV head.  Measured (head_dim 128, 64 heads over 8): 16,382 prompt rows
// through a window of 4096, 2.20 TFLOP, 2.3 to 2.5 ms = 880 to 950 TFLOP/s at the power limit; a token of each of 64 sequences
// through such a window, 0.90 GB, 166 to 208 us = 4.3 to 5.4 TB/s; trees of 8 to 64 nodes of 32 sequences on up to 8190
// tokens, 0.2 TFLOP and 0.6 GB, 245 to 287 us; one token through a window of 1024 (32 heads) 13.5 us.
//
// Probabilities go into the products as 16-bit numbers, as tcgen05 takes them beside 16-bit values.  Blocks of 128 rows or fewer
// have room on the matrix pipe for two, the rounding and the rest, and outputs off by little but their own rounding.  Blocks of
// more take one: with two the prompts above take 3.03 in place of 2.45 ms and the trees 324 in place of 269 us, and their
// root mean square error falls from 2.7e-4 (fp16) and 2.2e-3 (bf16) of the outputs to 2.0e-4 and 1.7e-3, that of the
// outputs' rounding alone.  Sums are of the probabilities before either.
//
// The products of one thread run in the order of their issue: scores that overwrite a chunk's probabilities wait for its
// outputs, and a chunk's scores are complete after the outputs of the chunk before (nothing else guards either).
// Halves of a chunk whose scores are there ahead of time (64 keys a product) were slower: 2.76 against 2.44 ms on the prompts.
#include <cuda.h>

#include <algorithm>
#include <cmath>
#include <numeric>

#include "paged.cuh"
#include "pairs.cuh"

namespace otf {

int set_cuda_error(cudaError_t e);       // capi.cu
int check_device();                      // capi.cu
int paged_rows_device_error(int clear);  // read (and optionally clear) the flag below
bool encode_tiled_4d_swizzled(void* map, const void* base, const uint64_t* dims, const uint64_t* strides, const uint32_t* box);  // capi.cu

constexpr int kPrKeys = 128;      // keys of a chunk
constexpr int kPrRows = 256;      // rows of a block
constexpr int kPrGrid = 148;      // a CTA on each SM
constexpr int kPrMma = 8, kPrQuery = 9, kPrLoad = 10;  // warps that issue products, fetch queries, and two that fetch keys and values
constexpr int kPrThreads = 384;
constexpr int kPrMaxNodes = 64;
// What an item's start and end cost, in chunks.  With 2, 3 and 4 on one GPU: a batch's step (as above) 194, 188 and 185 us,
// trees 266, 265 and 268, prompts 2.50, 2.51 and 2.52 ms (between GPUs they differ by more).
constexpr int kPrItemUnits = 3;
constexpr float kPrLog2e = 1.4426950408889634f;

// Set when a sequence does not fit its pages, names a page outside the pool, or has rows or parents out of range.
__device__ int g_paged_rows_device_error;
__device__ __forceinline__ void report_bad_rows() { atomicExch(&g_paged_rows_device_error, 1); }

// The item that several CTAs share and that begins in a CTA's run.
struct __align__(16) SharedItem {
  int there, g, row0, rows;  // row0: of the sequence's; rows of the block
  int first_part, last_cta, r0, pad;
};

struct RowsArgs {
  // Boxes of 64 dims of `box` tokens of a page, as the ring holds them, and of `rest` tokens for what is left of it.
  CUtensorMap kmap, vmap, kmap_rest, vmap_rest;
  CUtensorMap qmap;        // boxes of 64 dims of 32 rows: a KV head's query heads of some tokens
  int box, rest, q_box;    // box, q_box: 0 for no tensor copies
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
  int part_rows;       // rows of a block that there can be
  float* part;         // [2 x grid][part_rows][head_dim]: o of a part
  float2* part_ml;     // [2 x grid][part_rows]: its m and l
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
  int t0, t1;  // the first and last token whose keys and rows it has
  int low, low_full, full, end, sink_chunks, low_chunk, chunks;
};
template <bool TREE>
__device__ __forceinline__ Keys keys_of(const RowsArgs& a, const RowRange& s, int rb) {
  Keys k;
  const int row0 = rb * kPrRows, row1 = min(s.tokens * a.rep, row0 + kPrRows);
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
  if (TREE) {  // all nodes' keys are there for every block
    k.t0 = 0;
    k.t1 = s.tokens - 1;
  }
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

// What a run has of an item: the chunks [c0, c1).  Without any it is the run's end.
struct __align__(16) Portion {
  int b, rb, g, rows;  // rows of the block
  int c0, c1, first;   // first: of the run
  RowRange s;
  Keys k;
  int pad;
  __device__ __forceinline__ bool whole() const { return c0 == 0 && c1 == k.chunks; }
  // The ring's order, that of the products: of m chunks the j-th one's keys and values are these fills.  With groups that
  // share chunks K0 V0 K1 V1 ..., with groups that take turns K0 K1 V0 K2 V1 ...: what is fetched later is held shorter.
  __device__ __forceinline__ uint32_t key_fill(int j) const { return rows > 128 || j == 0 ? 2 * j : 2 * j - 1; }
  __device__ __forceinline__ uint32_t value_fill(int j) const {
    return rows > 128 || j + 1 == c1 - c0 ? 2 * j + 1 : 2 * j + 2;
  }
  // Copies of the rows: 1 << fold.
  __device__ __forceinline__ int fold() const { return rows <= 32 ? 2 : rows <= 64 ? 1 : 0; }
};
static_assert(sizeof(Portion) == 80, "");

// The portions of a run, one after another.
template <bool TREE>
struct Walk {
  const RowsArgs& a;
  const int64_t u0, u1;
  int64_t at;  // the item's first unit
  Portion p;

  __device__ __forceinline__ Walk(const RowsArgs& args, const RunStart& r) : a(args), u0(r.u0), u1(r.u1), at(r.at) {
    p.b = r.b;
    p.rb = r.rb;
    p.g = r.g;
    p.first = 1;
  }
  __device__ __forceinline__ void block() {
    p.k = keys_of<TREE>(a, p.s, p.rb);
    p.rows = min(kPrRows, p.s.tokens * a.rep - p.rb * kPrRows);
  }
  __device__ __forceinline__ bool clip() {
    p.c0 = (int)max((int64_t)0, u0 - at - kPrItemUnits);
    p.c1 = (int)min((int64_t)p.k.chunks, u1 - at - kPrItemUnits);
    return p.c1 > p.c0;
  }
  __device__ __forceinline__ bool begin() {
    if (u0 >= u1) return false;
    p.s = range_of<TREE>(a, p.b, false);
    block();
    return clip() || find();
  }
  __device__ __forceinline__ bool next() {
    p.first = 0;
    return find();
  }
  __device__ __forceinline__ bool find() {
    do {
      at += p.k.chunks + kPrItemUnits;
      if (at + kPrItemUnits >= u1) return false;
      if (++p.g == a.c.kv_heads) {
        p.g = 0;
        if ((int64_t)(++p.rb) * kPrRows >= (int64_t)p.s.tokens * a.rep) {
          p.rb = 0;
          do {
            if (++p.b >= a.c.batch) return false;
            p.s = range_of<TREE>(a, p.b, false);
          } while (p.s.tokens == 0);
        }
        block();
      }
    } while (!clip());
    return true;
  }
};

constexpr int kPrSmall = 3 * 1024;

template <int D>
struct RowsShape {
  static constexpr int tile = 128 * D * 2;               // bytes of 128 queries, keys or values
  static constexpr int slots = D == 128 ? 5 : 10;        // of the ring
  static constexpr int ring = D == 128 ? 2 * tile : tile + 128 * 64 * 4;  // behind two tiles of queries, or one and `meet`
  static constexpr int small = ring + slots * tile;      // barriers and the like
  static constexpr int bytes = small + kPrSmall;  // the runtime's own kilobyte lies before a 1024-byte border
};
// Behind the first tile of queries, where there is no second one: 64 columns of the outputs of 128 rows, where
// the groups and copies meet.

// The small part of the shared memory, behind the ring.
struct RowsSmall {
  uint64_t kv_full[10], kv_empty[10], v_landed[10];
  uint64_t q_full[2], q_empty[2], s_full[2], p_half[2], p_full[2], o_done[2];
  uint64_t item_full[4], item_empty[4], meet_free[2], both;
  Portion items[4];  // the run's next ones, from the warp that fetches keys to all others
  RunStart run;
  int64_t sums[16];
  float2 ml[256];
  uint32_t tmem;
  int gave_up;   // a wait ran out: no more waiting
  // Slot n & 7 holds n where an infinity or NaN was taken out of values of the run's n-th portion.  Any warp is at most four
  // portions ahead of another (`items`), so that no slot is written for a later portion while an earlier one's is read.
  uint32_t odd[8];
};
static_assert(sizeof(RowsSmall) <= kPrSmall, "");

// A bounded wait: after a second the CTA gives up, raises the flag and runs to its end without waiting.  The warp that
// fetches queries waits for whole items, of up to millions of chunks: a minute.  For a whole warp, whose lanes go on together:
// what follows are instructions of all of them.
constexpr uint64_t kPrWait = 1000000000ull, kPrLongWait = 60 * kPrWait;
__device__ __forceinline__ void rows_wait(uint64_t* bar, uint32_t parity, volatile int* gave_up, uint64_t most = kPrWait) {
  const uint32_t at = smem_u32(bar);
  bool there = mbar_try_wait(at, parity);
  if (!there) {
    const uint64_t t0 = global_ns();
    while (!there && !*gave_up) {
#pragma unroll 1
      for (int i = 0; i < 32 && !there; ++i) there = mbar_try_wait(at, parity);
      if (!there && global_ns() - t0 > most) {
        *gave_up = 1;
        report_bad_rows();
      }
    }
  }
  __syncwarp();
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* tmap, int x, int y, int z, int u, uint32_t mbar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(u), "r"(mbar) : "memory");
}
// True in one lane of a warp that runs together.
__device__ __forceinline__ bool one_lane() {
  uint32_t x;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(x));
  return x != 0;
}
// A warp's view of the run's portions.
struct Feed {
  RowsSmall& sm;
  volatile int* gave_up;
  uint32_t n = 0;
  __device__ __forceinline__ Feed(RowsSmall& small) : sm(small), gave_up(&small.gave_up) {}
  __device__ __forceinline__ bool next(Portion& p, uint64_t most = kPrWait) {
    const uint32_t slot = n & 3;
    rows_wait(&sm.item_full[slot], n >> 2 & 1u, gave_up, most);
    p = sm.items[slot];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&sm.item_empty[slot]));
    ++n;
    // one answer for the warp: where a lane has given up, the lanes may hold different portions
    return !__any_sync(0xffffffffu, *gave_up) && p.c1 > p.c0;
  }
};

__device__ __forceinline__ void mbar_arrive_n(uint32_t addr, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(addr), "r"(n) : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 lanes x 32 or 16 consecutive 32-bit columns of tensor memory, complete on return, and back.
__device__ __forceinline__ void tmem_ld32(uint32_t at, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%1"
      "7,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%1"
      "7,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
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

// Two 16-bit values, an infinity or NaN as 0.
template <bool BF>
__device__ __forceinline__ uint32_t without_odd2(uint32_t x) {
  constexpr uint32_t e = BF ? 0x7F80u : 0x7C00u;
  if ((x & e) == e) x &= 0xffff0000u;
  if ((x & (e << 16)) == e << 16) x &= 0xffffu;
  return x;
}

// The page of a key, as the table names it (0 where there is no key), and the key's offset in the pools under it: -1
// where the page lies outside.
struct KeyPlace {
  int page, rest;
  bool there;
};
__device__ __forceinline__ KeyPlace ask_key(const RowsArgs& a, int b, int s, bool there) {
  const uint32_t in = (uint32_t)s / a.page;
  return KeyPlace{there ? a.c.table[b * a.c.ld_table + in] : 0, s - (int)(in * a.page.d), there};
}
__device__ __forceinline__ int64_t offset_of(const RowsArgs& a, const KeyPlace& k) {
  if (!k.there) return -1;
  if (k.page < 0 || k.page >= a.c.n_pages) {
    report_bad_rows();
    return -1;
  }
  return k.page * a.c.page_stride + (int64_t)k.rest * a.c.token_stride;
}

// The infinities and NaN that were taken out of a block's values, given back to the rows that see them:
// columns [col, col + N) of the outputs o that a warp's lanes hold a row of each (the same columns).
template <bool BF, int D, bool TREE, int N>
__device__ __noinline__ void add_odd(const RowsArgs& a, const Portion& it, const RowView& view, float* o, int col) {
  for (int v = it.c0; v < it.c1; ++v) {
    if (!some_do_not_see(it.k, v, a.sinks)) continue;
    const int k0 = first_key(it.k, v);
    for (int s = k0; s < min(k0 + kPrKeys, it.k.end); ++s) {
      if (s < it.k.low && s >= a.sinks) continue;
      const int64_t at = offset_of(a, ask_key(a, it.b, s, true));
      if (at < 0) continue;
      const float mine = to_f<BF>(a.c.v[at + it.g * a.c.head_stride + col + (threadIdx.x & (N - 1))]);
      if (!__any_sync(0xffffffffu, !isfinite(mine))) continue;
      const bool sees = (seen32<TREE>(a, view, s & ~31) >> (s & 31)) & 1u;
      for (int i = 0; i < N; ++i) {
        const float y = __shfl_sync(0xffffffffu, mine, i);
        if (sees && !isfinite(y)) o[i] += y;
      }
    }
  }
}
// (The call keeps some 240 to 430 bytes a thread in local memory; blocks without odd values never make it.)
template <bool BF, int D, bool TREE, int N>
__device__ __forceinline__ void give_back(const RowsArgs& a, const Portion& it, const RowView& view, float (&o)[N], int col) {
  const Portion here = it;  // copies: what lies in memory for the call
  const RowView mine = view;
  float y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = o[i];
  add_odd<BF, D, TREE, N>(a, here, mine, y, col);
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = y[i];
}

// ---- scores to probabilities ------------------------------------------------------------------

// 4 x 4 16-byte pieces across four lanes: lane q's piece i becomes lane i's piece q.
__device__ __forceinline__ void turn_pieces(uint32_t (&x)[4][4]) {
#pragma unroll
  for (int step = 1; step <= 2; step <<= 1) {
    const bool upper = threadIdx.x & step;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!(i & step))
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? x[i][k] : x[i + step][k], step);
          if (upper) x[i][k] = got;
          else x[i + step][k] = got;
        }
  }
}

// A row's state.
struct RowState {
  float m, l;
  bool any;  // a chunk came before
};

// The scores of the keys' groups of 32, c0 .. c1 - 1 of a chunk's four, become probabilities: one 16-bit number each,
// 16 columns a group, or (TWO) the rounding and the rest, 16 columns of each in the place of 32 scores.  Loops over
// the groups, the scores fetched twice: with all 128 in registers the code was four times as long and its fetching
// took more time than the second look (prompts of 64 heads, some 16400 rows, 2.94 ms against 2.69).
template <bool BF, int D, bool TWO, bool TREE, bool EDGE>
__device__ __forceinline__ void turn_chunk(const RowsArgs& a, uint32_t s_at, uint32_t o_at, int c0, int c1, const RowView& view, int k0,
                                     bool there, RowState& r, uint64_t* half_bar) {
  const float scale = a.scale;
  auto fetch = [&](int c, float (&s)[32]) {
    tmem_ld32(s_at + 32 * c, s);
    if (EDGE) {
      const uint32_t see = seen32<TREE>(a, view, k0 + 32 * c);
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (!(see >> i & 1u)) s[i] = -INFINITY;
    }
  };
  float tops[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
  for (int c = c0; c < c1; ++c) {
    float s[32];
    fetch(c, s);
#pragma unroll
    for (int i = 0; i < 32; i += 2) tops[(i >> 1) & 1] = max_three(tops[(i >> 1) & 1], s[i], s[i + 1]);
  }
  const float top = fmaxf(tops[0], tops[1]) * scale;
  // lanes without a row hold what happens to lie there
  if (__any_sync(0xffffffffu, there && top > (r.m == -INFINITY ? -INFINITY : r.m + kPrHeadroom))) {
    const float mx = fmaxf(r.m, top), f = r.m == -INFINITY ? 0.0f : pr_ex2(r.m - mx);
    r.m = mx;
    r.l *= f;
    if (r.any)  // the outputs of the chunk before are complete, as this one's scores are
#pragma unroll 1
      for (int c = 0; c < D; c += 16) {
        uint32_t x[16];
        tmem_ld16(o_at + c, x);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * f);
        tmem_st16(o_at + c, x);
      }
  }
  const float z = kPrShift<BF> - (r.m == -INFINITY ? 0.0f : r.m);
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
  for (int c = c0; c < c1; ++c) {
    float s[32];
    fetch(c, s);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      fma_two(s[i], s[i + 1], scale, z);
      s[i] = pr_ex2(s[i]);
      s[i + 1] = pr_ex2(s[i + 1]);
      add_two(sum[i & 2], sum[(i & 2) + 1], s[i], s[i + 1]);
    }
    if (TWO) {
      uint32_t p[32];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = pack2<BF>(s[2 * i], s[2 * i + 1]);
        const float2 y = unpack2<BF>(p[i]);
        p[16 + i] = pack2<BF>(s[2 * i] - y.x, s[2 * i + 1] - y.y);
      }
      tmem_st32(s_at + 32 * c, p);
    } else {
      uint32_t p[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = pack2<BF>(s[2 * i], s[2 * i + 1]);
      tmem_st16(s_at + 16 * c, p);
    }
    if (c == 1 && c1 - c0 == 4) {  // the products with the first half of the keys' values may begin
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(half_bar));
    }
  }
  if (TWO && c1 - c0 < 4) {  // a copy's other keys
    const uint32_t none[32] = {};
#pragma unroll 1
    for (int c = 0; c < 4; ++c)
      if (c < c0 || c >= c1) tmem_st32(s_at + 32 * c, none);
  }
  r.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

template <bool BF, int D, bool TWO, bool TREE>
__device__ __forceinline__ void turn(const RowsArgs& a, uint32_t s_at, uint32_t o_at, int c0, int c1, bool edge, const RowView& view, int k0,
                                     bool there, RowState& r, uint64_t* half_bar) {
  if (edge)
    turn_chunk<BF, D, TWO, TREE, true>(a, s_at, o_at, c0, c1, view, k0, there, r, half_bar);
  else
    turn_chunk<BF, D, TWO, TREE, false>(a, s_at, o_at, c0, c1, view, k0, there, r, half_bar);
}

// ---- the kernel -------------------------------------------------------------------------------

template <bool BF, int D, bool TREE>
__global__ void __launch_bounds__(kPrThreads, 1) k_paged_rows(const __grid_constant__ RowsArgs a) {
  using S = RowsShape<D>;
  constexpr int NS = S::slots;
  constexpr uint32_t kFormat = (1u << 4) | (BF ? 1u << 7 | 1u << 10 : 0u) | ((uint32_t)(128 >> 4) << 24);
  constexpr uint32_t kScores = kFormat | ((uint32_t)(kPrKeys >> 3) << 17);
  constexpr uint32_t kOutputs = kFormat | ((uint32_t)(D >> 3) << 17) | (1u << 16);  // values: keys across
  constexpr uint32_t kOut = 256;  // tensor memory: 128 columns of scores for each group, then its outputs
  extern __shared__ __align__(1024) unsigned char smem[];
  RowsSmall& sm = *reinterpret_cast<RowsSmall*>(smem + S::small);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_trigger();
  if (smem_u32(smem) & 1023u) {  // the swizzles count on it
    pdl_wait();
    if (tid == 0) {
      report_bad_rows();
      a.shared[blockIdx.x] = SharedItem{};
    }
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(smem_u32(&sm.kv_full[i]), 64);
      mbar_init(smem_u32(&sm.v_landed[i]), 64);
      mbar_init(smem_u32(&sm.kv_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sm.q_full[i]), 1);
      mbar_init(smem_u32(&sm.q_empty[i]), 1);
      mbar_init(smem_u32(&sm.s_full[i]), 1);
      mbar_init(smem_u32(&sm.p_half[i]), 4);
      mbar_init(smem_u32(&sm.p_full[i]), 4);
      mbar_init(smem_u32(&sm.o_done[i]), 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&sm.meet_free[i]), 8);
    mbar_init(smem_u32(&sm.both), 8);
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(&sm.item_full[i]), 1);
      mbar_init(smem_u32(&sm.item_empty[i]), kPrThreads / 32 - 1);
    }
    mbar_fence_init();
    sm.gave_up = 0;
    for (int i = 0; i < 8; ++i) sm.odd[i] = 0;
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
      for (int rb = lane; (int64_t)rb * kPrRows < (int64_t)s.tokens * a.rep; rb += 32)
        x += keys_of<TREE>(a, s, rb).chunks + kPrItemUnits;
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
      r.ctas = max((int64_t)1, min((int64_t)kPrGrid, total));
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
          const int per = (int64_t)(r0 + lane) * kPrRows < (int64_t)s.tokens * a.rep
                              ? keys_of<TREE>(a, s, r0 + lane).chunks + kPrItemUnits : 0;
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
  fence_async_shared();  // the units lie where tensor copies go
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&sm.tmem);
  const RunStart run = sm.run;
  volatile int* gave_up = &sm.gave_up;
  Feed feed(sm);
  Portion it;

  if (warp >= kPrLoad) {
    // Keys and values: chunk after chunk a slot of keys, then one of values, 64 rows a warp.
    constexpr int P = D / 8, R = 32 / P;  // 16-byte pieces of a row, rows of a copy instruction
    const int w = warp - kPrLoad, piece = lane % P, sub = lane / P;
    const uint32_t ring = smem_u32(smem + S::ring);
    const uint32_t to = (uint32_t)((piece >> 3) * 128 * 128 + (64 * w + sub) * 128);
    uint32_t fill = 0;
    // What a chunk's copies need to know, asked for a chunk ahead: of two of the warp's keys, 32 apart, or where all
    // keys are there and tensor copies are open, of the first key in a lane's page (one page a lane).
    struct Asked {
      KeyPlace key[2];
      bool boxes;
    };
    auto ask = [&](int v) {
      const int k0 = first_key(it.k, v);
      Asked x;
      x.boxes = a.box && k0 + kPrKeys <= it.k.end && (k0 >= it.k.low || k0 + kPrKeys <= a.sinks);
      if (x.boxes) {
        const int64_t first = ((int64_t)((uint32_t)k0 / a.page) + lane) * a.page.d;
        const bool there = first < k0 + kPrKeys;
        x.key[0] = ask_key(a, it.b, there ? max(k0, (int)first) : 0, there);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int s = k0 + 64 * w + 32 * h + lane;
          x.key[h] = ask_key(a, it.b, s, s < it.k.end && (s >= it.k.low || s < a.sinks));
        }
      }
      return x;
    };
    auto empty = [&](uint32_t f) {
      if (f >= NS) rows_wait(&sm.kv_empty[f % NS], (f / NS - 1) & 1u, gave_up);
    };
    // The first of the two warps finds the run's portions for all.
    Walk<TREE> walk(a, run);
    SharedItem over = {};
    uint32_t found = 0;
    auto next_portion = [&](bool begin) -> bool {
      if (w) return feed.next(it);
      const bool more = (begin ? walk.begin() : walk.next()) && !__any_sync(0xffffffffu, *gave_up);
      if (!more) walk.p.c0 = walk.p.c1 = 0;
      it = walk.p;
      if (it.c0 == 0 && it.c1 > 0 && it.c1 < it.k.chunks) {
        // begins in this run and goes on behind it: what the joining kernel needs to know
        const int64_t end = walk.at + kPrItemUnits + it.k.chunks - 1;  // the unit of its last chunk
        over = SharedItem{1, it.g, it.rb * kPrRows, it.rows, 2 * (int)blockIdx.x + (it.first ? 0 : 1),
                          (int)(((end + 1) * run.ctas - 1) / run.total), it.s.r0, 0};
      }
      const uint32_t slot = found & 3;
      if (found >= 4) rows_wait(&sm.item_empty[slot], ((found >> 2) - 1) & 1u, gave_up);
      __syncwarp();
      if (lane == 0) {
        sm.items[slot] = it;
        mbar_arrive(smem_u32(&sm.item_full[slot]));
      }
      ++found;
      return more;
    };
    if (next_portion(true)) {
      const int64_t v_from_k = a.c.v - a.c.k;
      Asked next = ask(it.c0);
      for (int v = it.c0;;) {
        const bool odd = some_do_not_see(it.k, v, a.sinks);
        const int g = it.g;
        const Asked x = next;
        const uint32_t kf = fill + it.key_fill(v - it.c0), vf = fill + it.value_fill(v - it.c0);
        bool more = true;
        if (++v == it.c1) {
          fill += 2 * (it.c1 - it.c0);
          more = next_portion(false);
          v = it.c0;
        }
        if (more) next = ask(v);
        const uint32_t ks = kf % NS, vs = vf % NS;
        if (x.boxes) {
          // the first warp the keys, the second one the values
          const uint32_t slot = w ? vs : ks, bar = smem_u32(w && odd ? &sm.v_landed[slot] : &sm.kv_full[slot]);
          empty(w ? vf : kf);
          __syncwarp();
          if (lane == 0) {
            mbar_arrive_expect_tx(bar, S::tile);
            mbar_arrive_n(bar, 63);
          }
          __syncwarp();
          const int first = __shfl_sync(0xffffffffu, x.key[0].rest, 0);
          if (x.key[0].there) {
            int page = x.key[0].page, from = x.key[0].rest;
            if (page < 0 || page >= a.c.n_pages) {
              report_bad_rows();
              page = a.c.n_pages;  // reads as zeros
            }
            // the first lane's page may have begun before the chunk, the last one's may go on behind it
            const int d = (int)a.page.d;
            int row = lane ? lane * d - first : 0;
            const int end = min(kPrKeys, (lane + 1) * d - first);
            uint32_t dst = ring + slot * S::tile + row * 128;
            while (row < end) {
              const bool big = end - row >= a.box;
              const CUtensorMap* map = w ? (big ? &a.vmap : &a.vmap_rest) : (big ? &a.kmap : &a.kmap_rest);
#pragma unroll
              for (int h = 0; h < D / 64; ++h) tma_load_4d(dst + h * (128 * 128), map, h * 64, g, from, page, bar);
              const int n = big ? a.box : a.rest;
              row += n;
              from += n;
              dst += n * 128;
            }
          }
        } else {
          empty(kf);
          empty(vf);
          const uint16_t* const base = a.c.k + g * a.c.head_stride + piece * 8;
          const uint32_t dst = ring + ks * S::tile + to, across = (vs - ks) * S::tile;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int64_t mine = offset_of(a, x.key[h]);
#pragma unroll 4
            for (int i = 0; i < 32 / R; ++i) {
              const int64_t at = __shfl_sync(0xffffffffu, mine, sub + i * R);
              const uint16_t* y = base + (at >= 0 ? at : 0);  // an address, not read where there is no key
              const uint32_t to_key = dst + (32 * h + i * R) * 128 + (((piece & 7) ^ ((sub + i * R) & 7)) << 4), bytes = at >= 0 ? 16u : 0u;
              cp_async16(to_key, y, bytes);
              cp_async16(to_key + across, y + v_from_k, bytes);
            }
          }
          cp_async_mbar_arrive(smem_u32(&sm.kv_full[ks]));  // when they have landed
          cp_async_mbar_arrive(smem_u32(odd ? &sm.v_landed[vs] : &sm.kv_full[vs]));
        }
        if (!more) break;
      }
    }
    if (w == 0 && lane == 0) a.shared[blockIdx.x] = over;
    cp_async_wait<0>();
  } else if (warp == kPrQuery) {
    // Queries: rows that there are, 128 of a tile; the others' scores are never looked at.  Then, once they have
    // landed, the item's values that not every row of the block sees: a weight of 0 does not keep an infinity or NaN
    // from a row, so they are taken out before the products (and given back at the item's end).
    constexpr int P = D / 8, R = 32 / P;
    const int piece = lane % P, sub = lane / P;
    uint32_t n[2] = {0, 0}, fill = 0;
    uint32_t turns = 0;  // how often each slot's landing came around, a bit per slot
    uint32_t meets = 0;
    bool met = false;    // the portion before uses `meet`
    while (feed.next(it, kPrLongWait)) {
      const int all = it.rows, fold = it.fold();
      for (int w = 0; w < 2; ++w) {
        if (w == 1) {
          // The second tile lies where the groups of the portion before may still be meeting.  Two barriers in turn:
          // with one the portion at hand, whose first tile is there, might be through before this warp has looked.
          if (met) {
            rows_wait(&sm.meet_free[meets & 1], meets >> 1 & 1u, gave_up, kPrLongWait);
            ++meets;
          }
          met = all <= 128;
          if (met) break;
        }
        if (n[w] > 0) rows_wait(&sm.q_empty[w], (n[w] - 1) & 1u, gave_up, kPrLongWait);
        ++n[w];
        const int row0 = it.rb * kPrRows + w * 128, rows = min(128, all - w * 128);
        unsigned char* tile = smem + w * S::tile + (piece >> 3) * 128 * 128;
        auto at = [&](int r) { return reinterpret_cast<uint4*>(tile + r * 128 + (((piece & 7) ^ (r & 7)) << 4)); };
        if (a.q_box) {
          constexpr int H = D / 64;
          const int from = lane / H & ((4 >> fold) - 1);  // a lane's box, which lies there 1 << fold times
          const bool mine = lane < 4 * H && from * 32 < rows;
          const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, mine)), bar = smem_u32(&sm.q_full[w]);
          if (lane == 0) mbar_arrive_expect_tx(bar, boxes * 32 * 128);
          __syncwarp();
          if (mine)
            tma_load_4d(smem_u32(smem + w * S::tile) + lane % H * (128 * 128) + lane / H * (32 * 128), &a.qmap, lane % H * 64,
                        it.g * a.rep, it.s.r0 + (int)((uint32_t)row0 / a.rep_div) + from * a.q_box, 0, bar);
          continue;
        }
        for (int r = sub; r < rows; r += R) {
          const uint32_t row = row0 + r, t = row / a.rep_div;
          const uint16_t* x = a.q + (it.s.r0 + (int64_t)t) * a.ldq + (int64_t)(it.g * a.rep + row - t * a.rep) * D + piece * 8;
          for (int c = 0; c < 128; c += 128 >> fold) cp_async16(smem_u32(at(c + r)), x, 16u);
        }
        cp_async_commit();
        cp_async_wait<0>();
        if (a.sign)  // a negative scale's, so that a larger product weighs more
          for (int r = sub; r < rows; r += R)
            for (int c = 0; c < 128; c += 128 >> fold) {
              const uint4 y = *at(c + r);
              *at(c + r) = make_uint4(y.x ^ a.sign, y.y ^ a.sign, y.z ^ a.sign, y.w ^ a.sign);
            }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.q_full[w]));
      }
      for (int v = it.c0; v < it.c1; ++v) {
        if (!some_do_not_see(it.k, v, a.sinks)) continue;
        const uint32_t slot = (fill + it.value_fill(v - it.c0)) % NS;
        rows_wait(&sm.v_landed[slot], turns >> slot & 1u, gave_up, kPrLongWait);
        turns ^= 1u << slot;
        uint4* x = reinterpret_cast<uint4*>(smem + S::ring + slot * S::tile);
        uint32_t high = 0;  // an exponent of ones plus one carries into the sign's place
#pragma unroll 16
        for (int i = lane; i < S::tile / 16; i += 32) {
          constexpr uint32_t e = BF ? 0x7F807F80u : 0x7C007C00u, one = BF ? 0x00800080u : 0x04000400u;
          const uint4 y = x[i];
          high |= ((y.x & e) + one) | ((y.y & e) + one) | ((y.z & e) + one) | ((y.w & e) + one);
        }
        if (high & 0x80008000u) {
          for (int i = lane; i < S::tile / 16; i += 32) {
            const uint4 y = x[i];
            x[i] = make_uint4(without_odd2<BF>(y.x), without_odd2<BF>(y.y), without_odd2<BF>(y.z), without_odd2<BF>(y.w));
          }
          *(volatile uint32_t*)&sm.odd[feed.n & 7] = feed.n;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_n(smem_u32(&sm.kv_full[slot]), 64);
      }
      fill += 2 * (it.c1 - it.c0);
    }
  } else if (warp == kPrMma) {
    // The whole warp keeps count, one lane issues: descriptors then are a warp's, not a lane's.
    uint32_t fill = 0, probs[2] = {0, 0}, items[2] = {0, 0};
    const uint32_t q0 = smem_u32(smem), ring = smem_u32(smem + S::ring);
    auto scores = [&](int w, uint32_t q, uint32_t f) {  // of group w, from the keys of fill f
      const uint64_t qd = tc_desc_sw128(q), kd = tc_desc_sw128(ring + f % NS * S::tile);
      if (one_lane()) {
#pragma unroll
        for (int x = 0; x < D / 16; ++x)
          tc_mma_f16(tmem + w * 128, qd + (x >> 2) * (128 * 128 / 16) + (x & 3) * 2, kd + (x >> 2) * (128 * 128 / 16) + (x & 3) * 2,
                     kScores, x > 0);
        tc_commit(smem_u32(&sm.s_full[w]));
      }
    };
    // Outputs of group w from the values of fill f, the keys of the chunk's first or second half.
    auto outputs = [&](int w, uint32_t f, int half, uint32_t add) {
      const uint64_t vd = values_desc(ring + f % NS * S::tile) + half * (64 * 128 / 16);
      const uint32_t p = tmem + w * 128 + 32 * half, o = tmem + kOut + w * 128;
      if (one_lane())
#pragma unroll
        for (int x = 0; x < 4; ++x) tc_mma_f16_ta(o, p + 8 * x, vd + x * (2048 / 16), kOutputs, x > 0 ? 1u : add);
    };
    auto outputs_two = [&](int w, uint32_t f, int half, uint32_t add) {  // the same from probabilities of two numbers
      const uint64_t vd = values_desc(ring + f % NS * S::tile) + half * (64 * 128 / 16);
      const uint32_t p = tmem + w * 128 + 64 * half, o = tmem + kOut + w * 128;
      if (one_lane())
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          tc_mma_f16_ta(o, p + 32 * (x >> 1) + 8 * (x & 1), vd + x * (2048 / 16), kOutputs, x > 0 ? 1u : add);
          tc_mma_f16_ta(o, p + 32 * (x >> 1) + 8 * (x & 1) + 16, vd + x * (2048 / 16), kOutputs, 1u);
        }
    };
    auto commit = [&](uint64_t* bar) {
      if (one_lane()) tc_commit(smem_u32(bar));
    };
    auto filled = [&](uint32_t f) {
      rows_wait(&sm.kv_full[f % NS], f / NS & 1u, gave_up);
      fence_async_shared();  // the copies are of the generic proxy, the products of the other
      __syncwarp();
    };
    auto release = [&](uint32_t f) { commit(&sm.kv_empty[f % NS]); };
    auto ready = [&](int w, int half) {
      rows_wait(half ? &sm.p_full[w] : &sm.p_half[w], probs[w] & 1u, gave_up);
      probs[w] += half;
      tc_fence_after_sync();
      __syncwarp();
    };
    while (feed.next(it)) {
      const int m = it.c1 - it.c0;
      const bool pair = it.rows > 128;
      for (int w = 0; w < (pair ? 2 : 1); ++w) rows_wait(&sm.q_full[w], items[w]++ & 1u, gave_up);
      tc_fence_after_sync();
      __syncwarp();
      if (pair) {
        filled(fill);
        scores(0, q0, fill);
        scores(1, q0 + S::tile, fill);
        release(fill);
#pragma unroll 1
        for (int j = 0; j < m; ++j, fill += 2) {
          filled(fill + 1);
          if (j + 1 < m) filled(fill + 2);
          ready(0, 0);
          outputs(0, fill + 1, 0, j > 0);
          ready(0, 1);
          outputs(0, fill + 1, 1, 1u);
          if (j + 1 < m) {
            scores(0, q0, fill + 2);
          } else {
            commit(&sm.q_empty[0]);
            commit(&sm.o_done[0]);
          }
          ready(1, 0);
          outputs(1, fill + 1, 0, j > 0);
          ready(1, 1);
          outputs(1, fill + 1, 1, 1u);
          release(fill + 1);
          if (j + 1 < m) {
            scores(1, q0 + S::tile, fill + 2);
            release(fill + 2);
          } else {
            commit(&sm.q_empty[1]);
            commit(&sm.o_done[1]);
          }
        }
      } else {
        auto next_scores = [&](int j) {
          const uint32_t f = fill + it.key_fill(j);
          filled(f);
          scores(j & 1, q0, f);
          release(f);
        };
        next_scores(0);
        if (m > 1) next_scores(1);
        if (m <= 2) commit(&sm.q_empty[0]);
#pragma unroll 1
        for (int j = 0; j < m; ++j) {
          const int w = j & 1;
          const uint32_t f = fill + it.value_fill(j);
          filled(f);
          ready(w, 0);
          outputs_two(w, f, 0, j > 1);
          ready(w, 1);
          outputs_two(w, f, 1, 1u);
          release(f);
          if (j + 2 < m) {
            next_scores(j + 2);
            if (j + 3 == m) commit(&sm.q_empty[0]);
          } else {
            commit(&sm.o_done[w]);
          }
        }
        fill += 2 * m;
      }
    }
    __syncwarp();
  } else if (warp < 8) {
    // The rows: thread r of group w has row r of its tile, which is lane r of tensor memory.
    const int w = warp >> 2, r = tid & 127, quarter = warp & 3;
    const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
    const uint32_t s_at = tmem + lanes + w * 128, o_at = tmem + lanes + kOut + w * 128;
    uint32_t chunk_count = 0, item_count = 0, meets = 0, boths = 0;
    // The groups' eight warps meet (a wait that ends, as all others).
    auto both = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sm.both));
      rows_wait(&sm.both, boths++ & 1u, gave_up);
      __syncwarp();
    };
    while (feed.next(it)) {
      const bool pair = it.rows > 128;
      const int fold = it.fold(), size = 128 >> fold, copy = r >> (7 - fold);
      const int row = it.rb * kPrRows + (pair ? w * 128 : 0) + (r & (size - 1)), rows = it.s.tokens * a.rep;
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
      RowState state = {-INFINITY, 0.0f, false};
#pragma unroll 1
      for (int v = it.c0 + (pair ? 0 : w); v < it.c1; v += pair ? 1 : 2) {
        rows_wait(&sm.s_full[w], chunk_count & 1u, gave_up);
        ++chunk_count;
        tc_fence_after_sync();
        if (warp_there) {
          const int k0 = first_key(it.k, v);
          const bool edge = k0 + kPrKeys > it.k.full || (k0 < it.k.low_full && k0 + kPrKeys > a.sinks);
          if (pair)
            turn<BF, D, false, TREE>(a, s_at, o_at, 0, 4, edge, view, k0, there, state, &sm.p_half[w]);
          else
            turn<BF, D, true, TREE>(a, s_at, o_at, copy * (4 >> fold), (copy + 1) * (4 >> fold), edge, view, k0, there, state, &sm.p_half[w]);
          tmem_wait_st();
        }
        state.any = true;
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (fold || !warp_there) mbar_arrive(smem_u32(&sm.p_half[w]));
          mbar_arrive(smem_u32(&sm.p_full[w]));
        }
      }

      // The item's end in this run.
      if (state.any) {
        rows_wait(&sm.o_done[w], item_count & 1u, gave_up);
        ++item_count;
        tc_fence_after_sync();
      }
      if (!pair && it.c1 - it.c0 > 1) both();  // the other group's values have been looked through, too
      auto any_odd = [&] { return *(volatile uint32_t*)&sm.odd[feed.n & 7] == feed.n; };
      const bool whole = it.whole(), odd = __any_sync(0xffffffffu, any_odd());  // the warp goes one way: what it gives back takes all lanes
      const int64_t part = (int64_t)(2 * blockIdx.x + (it.first ? 0 : 1)) * a.part_rows + (row - it.rb * kPrRows);
      uint16_t* const to = a.out + (it.s.r0 + (int64_t)t) * a.ldo + (int64_t)(it.g * a.rep + row - t * a.rep) * D;
      // Columns [c, c + 32) of the warp's rows.  Four lanes turn their rows' 16-byte pieces, so that they write 64 bytes of
      // one row together.
      auto store = [&](float (&o)[32], int c, float l) {
        if (odd) give_back<BF, D, TREE, 32>(a, it, view, o, c);
        if (whole) {
          const float inv = 1.0f / l;
          uint32_t x[4][4];
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i >> 2][i & 3] = pack2<BF>(o[2 * i] * inv, o[2 * i + 1] * inv);
          turn_pieces(x);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int from = (lane & 28) + i;
            uint16_t* y = reinterpret_cast<uint16_t*>(__shfl_sync(0xffffffffu, (unsigned long long)to, from)) + c + (lane & 3) * 8;
            if (row - lane + from < rows) *reinterpret_cast<uint4*>(y) = make_uint4(x[i][0], x[i][1], x[i][2], x[i][3]);
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t x[4][4];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i >> 2][i & 3] = __float_as_uint(o[16 * h + i]);
            turn_pieces(x);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int from = (lane & 28) + i;
              if (row - lane + from < rows)
                *reinterpret_cast<uint4*>(a.part + (part - lane + from) * D + c + 16 * h + (lane & 3) * 4) =
                    make_uint4(x[i][0], x[i][1], x[i][2], x[i][3]);
            }
          }
        }
      };
      if (pair) {
        if (warp_there) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t x[32];
            float o[32];
            tmem_ld32(o_at + c, x);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(x[i]);
            store(o, c, state.l);
          }
          if (!whole && there) a.part_ml[part] = make_float2(state.m, state.l);
        }
      } else {
        const bool two = it.c1 - it.c0 > 1;  // both groups have chunks
        float* const meet = reinterpret_cast<float*>(smem + S::tile);
        if (fold) {
          // The groups' and copies' parts of each row: as many columns at a time as `meet` has room for, then all
          // threads add up four columns of a row at a time.
          const int rows_here = it.rows, parts = (two ? 2 : 1) << fold, mine = (w << fold) + copy;
          const int wide = rows_here <= 8 ? 7 : rows_here <= 16 ? 6 : 5, cols = min(D, 1 << wide);  // 8 parts x rows x cols <= 8192
          const int lr = r & (size - 1);
          if (state.any && there) sm.ml[(mine * size + lr) & 255] = make_float2(state.m, state.l);
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += cols) {
            if (state.any && warp_there)
#pragma unroll 1
              for (int c = 0; c < cols; c += 32) {
                uint32_t x[32];
                float o[32];
                tmem_ld32(o_at + c0 + c, x);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(x[i]);
                if (odd && mine == 0) give_back<BF, D, TREE, 32>(a, it, view, o, c0 + c);
                if (there)
#pragma unroll
                  for (int i = 0; i < 32; i += 4)  // turned by the row against bank conflicts
                    *reinterpret_cast<float4*>(meet + (mine * rows_here + lr) * cols + ((c + i) ^ ((lr & 7) << 2))) =
                        make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
              }
            both();
            const bool given = any_odd();  // a group without chunks only now knows
#pragma unroll 1
            for (int e = tid * 4; e < rows_here * cols; e += 256 * 4) {
              const int rr = e / cols, c = e - rr * cols;
              float mx = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
              for (int k = 0; k < parts; ++k) mx = fmaxf(mx, sm.ml[k * size + rr].x);
#pragma unroll 4
              for (int k = 0; k < parts; ++k) {
                const float2 ml = sm.ml[k * size + rr];
                // A part without a key that the row sees holds nothing, whatever its outputs are, but for what the first one
                // was given back; one whose keys are all NaN has no maximum either, and its sum says so.
                if (ml.x != -INFINITY || ml.y != 0.0f || (given && k == 0)) {
                  const float f = ml.x == -INFINITY ? 0.0f : pr_ex2(ml.x - mx);
                  const float4 y = *reinterpret_cast<const float4*>(meet + (k * rows_here + rr) * cols + (c ^ ((rr & 7) << 2)));
                  l = fmaf(ml.y, f, l);
                  o[0] = fmaf(y.x, f, o[0]);
                  o[1] = fmaf(y.y, f, o[1]);
                  o[2] = fmaf(y.z, f, o[2]);
                  o[3] = fmaf(y.w, f, o[3]);
                }
              }
              if (whole) {
                const int rt = (uint32_t)(it.rb * kPrRows + rr) / a.rep_div, head = it.g * a.rep + it.rb * kPrRows + rr - rt * a.rep;
                const float inv = 1.0f / l;
                *reinterpret_cast<uint2*>(a.out + (it.s.r0 + (int64_t)rt) * a.ldo + (int64_t)head * D + c0 + c) =
                    make_uint2(pack2<BF>(o[0] * inv, o[1] * inv), pack2<BF>(o[2] * inv, o[3] * inv));
              } else {
                const int64_t at = (int64_t)(2 * blockIdx.x + (it.first ? 0 : 1)) * a.part_rows + rr;
                *reinterpret_cast<float4*>(a.part + at * D + c0 + c) = make_float4(o[0], o[1], o[2], o[3]);
                if (c0 + c == 0) a.part_ml[at] = make_float2(mx, l);
              }
            }
            both();  // before the columns are written again
          }
        } else if (w == 0 || two) {
          auto place = [&](int row, int c) {  // of four columns, turned by the row against bank conflicts
            return reinterpret_cast<float4*>(meet + row * 64 + (((c >> 2) ^ (row & 15)) << 2));
          };
          float f0 = 1.0f, f1 = 0.0f;
#pragma unroll 1
          for (int half = 0; half < D; half += 64) {
            if (w == 1) {
              if (warp_there)
#pragma unroll 1
                for (int c = 0; c < 64; c += 32) {
                  uint32_t x[32];
                  tmem_ld32(o_at + half + c, x);
                  if (there)
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                      *place(r, c + i) = make_float4(__uint_as_float(x[i]), __uint_as_float(x[i + 1]),
                                                     __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
                }
              if (half == 0) sm.ml[r] = make_float2(state.m, state.l);
            }
            if (two) both();
            if (w == 0) {
              if (half == 0 && two) {
                const float2 ml = sm.ml[r];
                const float mx = fmaxf(state.m, ml.x);
                f0 = state.m == -INFINITY ? 0.0f : pr_ex2(state.m - mx);
                f1 = ml.x == -INFINITY ? 0.0f : pr_ex2(ml.x - mx);
                state.m = mx;
                state.l = state.l * f0 + ml.y * f1;
              }
              if (warp_there)
#pragma unroll 1
                for (int c = 0; c < 64; c += 32) {
                  uint32_t x[32];
                  float o[32];
                  tmem_ld32(o_at + half + c, x);
#pragma unroll
                  for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(x[i]);
                  if (two && there)
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                      const float4 y = *place(r, c + i);
                      o[i] = fmaf(o[i], f0, y.x * f1);
                      o[i + 1] = fmaf(o[i + 1], f0, y.y * f1);
                      o[i + 2] = fmaf(o[i + 2], f0, y.z * f1);
                      o[i + 3] = fmaf(o[i + 3], f0, y.w * f1);
                    }
                  store(o, half + c, state.l);
                }
              if (!whole && there && half == 0) a.part_ml[part] = make_float2(state.m, state.l);
            }
            if (two) both();  // before the columns are written again
          }
        }
        fence_async_shared();  // before the tensor copies that may follow there
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.meet_free[meets & 1]));
        ++meets;
      }
    }
  }

  if (*gave_up) {  // what is still on its way ends within microseconds
    const uint64_t t0 = global_ns();
    while (global_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == kPrMma) tmem_dealloc(tmem, 512);
}

// The parts of an item that several CTAs shared, joined in the keys' order: grid (CTAs, rows / 8), a warp
// per row.  Latency-bound: what the item is, then all parts' m and l and, eight at a time, their o.
template <bool BF, int D>
__global__ void __launch_bounds__(256) k_paged_rows_join(const __grid_constant__ RowsArgs a) {
  constexpr int PL = D / 32, U = 8;
  pdl_trigger();
  pdl_wait();
  const SharedItem x = a.shared[blockIdx.x];
  const int lane = threadIdx.x & 31, r = blockIdx.y * 8 + (threadIdx.x >> 5);
  if (!x.there || r >= x.rows) return;
  const int n = x.last_cta - (int)blockIdx.x + 1;
  auto part = [&](int i) { return (int64_t)(i == 0 ? x.first_part : 2 * ((int)blockIdx.x + i)) * a.part_rows + r; };
  float y[U][PL];
  auto fetch = [&](int base) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (base + k >= n) break;
      const float* z = a.part + part(base + k) * D + lane * PL;
      if (D == 128) {
        const float4 v = *reinterpret_cast<const float4*>(z);
        y[k][0] = v.x;
        y[k][1] = v.y;
        y[k][PL - 2] = v.z;
        y[k][PL - 1] = v.w;
      } else {
        const float2 v = *reinterpret_cast<const float2*>(z);
        y[k][0] = v.x;
        y[k][1] = v.y;
      }
    }
  };
  fetch(0);  // on their way while the maxima are found
  float2 ml = lane < n ? a.part_ml[part(lane)] : make_float2(-INFINITY, 0.0f);  // of the lane's part among 32
  float M = ml.x, L = 0.0f, acc[PL] = {};
  for (int i = lane + 32; i < n; i += 32) M = fmaxf(M, a.part_ml[part(i)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  for (int base = 0; base < n; base += U) {
    if (base) fetch(base);
    if (base && (base & 31) == 0) ml = base + lane < n ? a.part_ml[part(base + lane)] : make_float2(-INFINITY, 0.0f);
    const float mine = ml.x == -INFINITY ? 0.0f : pr_ex2(ml.x - M);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (base + k >= n) break;
      const float f = __shfl_sync(0xffffffffu, mine, (base + k) & 31), l = __shfl_sync(0xffffffffu, ml.y, (base + k) & 31);
      const float m = __shfl_sync(0xffffffffu, ml.x, (base + k) & 31);
      if (m != -INFINITY || l != 0.0f) {  // else nothing that the row sees, or nothing at all, lies there (l of NaN keys alone is one)
        L = fmaf(l, f, L);
#pragma unroll
        for (int j = 0; j < PL; ++j) acc[j] = fmaf(y[k][j], f, acc[j]);
      }
    }
  }
  const int row = x.row0 + r, t = (uint32_t)row / a.rep_div, head = x.g * a.rep + row - t * a.rep;
  uint32_t* to = reinterpret_cast<uint32_t*>(a.out + (x.r0 + (int64_t)t) * a.ldo + (int64_t)head * D + lane * PL);
#pragma unroll
  for (int j = 0; j < PL / 2; ++j) to[j] = pack2<BF>(acc[2 * j] / L, acc[2 * j + 1] / L);
}

struct RowsSpace {
  int64_t rows, part, part_ml, shared;
  int64_t bytes() const { return part + part_ml + shared; }
};
static RowsSpace rows_space(int64_t n, int64_t rep, int64_t D) {
  RowsSpace s;
  s.rows = std::min<int64_t>(kPrRows, align_up(n * rep, 8));
  s.part = align_up(2 * kPrGrid * s.rows * D * 4, 256);
  s.part_ml = align_up(2 * kPrGrid * s.rows * 8, 256);
  s.shared = align_up(kPrGrid * (int64_t)sizeof(SharedItem), 256);
  return s;
}
static bool rows_limits(int64_t batch, int64_t n, int64_t heads, int64_t kv_heads, int64_t D) {
  return batch <= kPagedMaxBatch && heads <= 65535 && kv_heads <= 1024 && (D == 64 || D == 128) && n <= INT32_MAX &&
         n * (heads / kv_heads) <= INT32_MAX - kPrRows;
}

template <bool BF, int D, bool TREE>
static cudaError_t launch_rows(const RowsArgs& a, cudaStream_t s) {
  auto* k = k_paged_rows<BF, D, TREE>;
  static std::atomic<bool> done[64];
  int dev;
  bool needs;
  cudaError_t e = needs_opt_in(done, dev, needs);
  if (e != cudaSuccess) return e;
  if (needs) {
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, RowsShape<D>::bytes);
    if (e != cudaSuccess) return e;
    opted_in(done, dev);
  }
  e = launch_pdl(k, dim3(kPrGrid), dim3(kPrThreads), RowsShape<D>::bytes, s, 1u, a);
  if (e != cudaSuccess) return e;
  return launch_pdl(k_paged_rows_join<BF, D>, dim3(kPrGrid, (unsigned)(a.part_rows / 8)), dim3(256), 0, s, 1u, a);
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
  return otf::rows_space(n, heads / kv_heads, head_dim).bytes();
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
  const otf::RowsSpace space = otf::rows_space(n, heads / a.c.kv_heads, D);
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
  // Tensor copies where chunks cut pages into groups of 4 tokens or more (`rest`), in larger boxes as far as they go:
  // a box costs the copy unit some 40 cycles whatever is in it (pages of 20, trees of 32 sequences: boxes of 4 alone
  // 321 us, with boxes of 16 277).  Else, and for the chunks that are not all there, 16-byte copies.
  const int rest = std::gcd((int)a.c.page_size, otf::kPrKeys);
  if (rest >= 4) {
    int box = rest;
    while (rest < 16 && box * 2 <= std::min(16, a.c.page_size)) box *= 2;
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)a.c.kv_heads, (uint64_t)a.c.page_size, (uint64_t)a.c.n_pages};
    const uint64_t strides[3] = {(uint64_t)a.c.head_stride * 2, (uint64_t)a.c.token_stride * 2, (uint64_t)a.c.page_stride * 2};
    const uint32_t boxes[4] = {64, 1, (uint32_t)box, 1}, rests[4] = {64, 1, (uint32_t)rest, 1};
    if (otf::encode_tiled_4d_swizzled(&a.kmap, a.c.k, dims, strides, boxes) &&
        otf::encode_tiled_4d_swizzled(&a.vmap, a.c.v, dims, strides, boxes) &&
        (rest == box || (otf::encode_tiled_4d_swizzled(&a.kmap_rest, a.c.k, dims, strides, rests) &&
                         otf::encode_tiled_4d_swizzled(&a.vmap_rest, a.c.v, dims, strides, rests)))) {
      a.box = box;
      a.rest = rest;
    }
  }
  if (a.rep <= 32 && 32 % a.rep == 0 && !a.sign) {
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)heads, (uint64_t)n, 1};
    const uint64_t strides[3] = {(uint64_t)D * 2, (uint64_t)ldq * 2, (uint64_t)ldq * 2};
    const uint32_t boxes[4] = {64, (uint32_t)a.rep, (uint32_t)(32 / a.rep), 1};
    if (otf::encode_tiled_4d_swizzled(&a.qmap, a.q, dims, strides, boxes)) a.q_box = 32 / a.rep;
  }
  char* w = static_cast<char*>(workspace);
  a.part = reinterpret_cast<float*>(w);
  a.part_ml = reinterpret_cast<float2*>(w + space.part);
  a.shared = reinterpret_cast<otf::SharedItem*>(w + space.part + space.part_ml);
  a.part_rows = (int)space.rows;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = cache->dtype == OTF_DTYPE_BF16;
  auto* launch = parents ? (D == 128 ? (bf ? otf::launch_rows<true, 128, true> : otf::launch_rows<false, 128, true>)
                                     : (bf ? otf::launch_rows<true, 64, true> : otf::launch_rows<false, 64, true>))
                         : (D == 128 ? (bf ? otf::launch_rows<true, 128, false> : otf::launch_rows<false, 128, false>)
                                     : (bf ? otf::launch_rows<true, 64, false> : otf::launch_rows<false, 64, false>));
  return set_cuda_error(launch(a, s));
}
