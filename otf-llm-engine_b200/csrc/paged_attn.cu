// Attention of a few new tokens per sequence over a key/value cache in pages (otf_paged_attn).
//
// Mathematics.  For a query row r of a KV head, with s_j = scale log2(e) q_r k_j, one pass over the
// cached tokens keeps the running maximum m, l = sum_j 2^(s_j - m) and o = sum_j 2^(s_j - m) v_j,
// rescaled when m grows; out = o / l.  Parts (m, l, o) of disjoint token ranges join as
// M = max m, L = sum l 2^(m - M), O = sum o 2^(m - M).
//
// Bound: the keys and values are read once, 2 x head_dim x 2 bytes per token and KV head; the
// products are 4 x head_dim x rows flops on them, below the matrix pipe's rate up to some tens
// of rows.  So the aim is to keep enough loads in flight on every SM.
//
// Split.  An item is a (sequence, KV head, block of up to 32 query rows); its tokens are cut into
// chunks, and all items' chunks, in order, are dealt out evenly to a fixed grid in contiguous runs,
// whatever the lengths are: a run may cross items, and an item may be shared by several CTAs, which
// then leave parts that a second kernel joins in order.  Neither launch depends on lengths (they are
// read on the device), so a step can be captured.
//
// Inside a CTA each warp is on its own: it takes 16 (head_dim 64: 32) tokens of every chunk through its
// own ring of shared-memory stages, filled by 16-byte asynchronous copies some chunks ahead and
// across items, and runs q k and p v on m16n8k16 matrix instructions.  The warps meet only at an
// item's end.  Up to 8 rows the loads decide (94 to 97% of the measured copy rate), and other products
// would change nothing; at 20 rows memory is at 48%, held back by starts, item ends and 255 registers a
// thread.  The asynchronous 5th-generation products would fit that side (keys, then dims, as their 128
// rows, the query rows as the narrow side, outputs in tensor memory); they are not tried here.
//
// Measured (16-bit, head_dim 128, 8 KV heads; the whole call in a graph, calls on different inputs one
// after another, caches as they leave them): one sequence of 131071
// tokens, 64 heads, 537 MB, 87.8 us = 6.1 TB/s (k_paged_attn by itself 83 us, 6.4 TB/s); 64 sequences
// of 127 to 8190 tokens, 1.09 GB, 181.7 us = 6.0 TB/s; one of 700 tokens 8.3 us, of which the joining
// launch, 4.1 by itself, is 3; 16 of 62 to 4001 tokens, 20 rows an item, 39 us without and 56.3 us with weights.
//
// The newest keys, which not every row sees, are masked in the steps that hold them; what they hold
// cannot reach the other rows (see the loop).
#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace otf {

int set_cuda_error(cudaError_t e);       // capi.cu
int check_device();                      // capi.cu
int paged_attn_device_error(int clear);  // read (and optionally clear) the flag below

constexpr int kPaWarps = 4;
constexpr int kPaThreads = kPaWarps * 32;
constexpr int kPaStages = 3;
constexpr int kPaStage = 8192;  // bytes of a warp's stage: its tokens' keys, then values
constexpr int kPaGrid = 296;    // two CTAs on each of 148 SMs
constexpr float kLog2e = 1.4426950408889634f;

// Set when a sequence does not fit its pages or names a page outside the pool.
__device__ int g_paged_attn_device_error;
__device__ __forceinline__ void report_bad_attn_page() { atomicExch(&g_paged_attn_device_error, 1); }

// Division of numbers below 2^31 by a fixed one.
struct FastDiv {
  uint32_t mul, shift, d;
};
static FastDiv fast_div(uint32_t d) {
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  return FastDiv{(uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1), l, d};
}
__device__ __forceinline__ uint32_t operator/(uint32_t n, const FastDiv& f) {
  return (__umulhi(f.mul, n) + n) >> f.shift;
}

struct AttnArgs {
  PagedView c;
  FastDiv page;
  const uint16_t* q;
  int64_t ldq;
  uint16_t* out;
  int64_t ldo;
  float scale;         // with log2(e)
  int rep, tokens;     // query heads per KV head, new tokens per sequence
  int rows, blocks;    // rep x tokens rows in so many row blocks
  int chunk_units, item_units;
  int64_t* prefix;     // [batch + 1] units before each sequence
  float* part;         // [2 x grid][rows of a block][head_dim]: o of a part
  float4* part_ml;     // [2 x grid][rows of a block]: its m, l and unrounded l
  float* lse;          // [batch, kv_heads, ld_scores] log2 of the sum, when weights are wanted
  float* scores;       // [batch, kv_heads, max_keys, ld_scores] likewise, a row's score in each column
  int64_t max_keys;
  int ld_scores;       // rows, rounded up to 4
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool BF>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}
__device__ __forceinline__ void lds128(uint32_t addr, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint16_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts128_zero(uint32_t addr) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(addr), "r"(0) : "memory");
}
// The transposed 8 x 8 matrix of 16-bit values, a row in the lanes 4 i .. 4 i + 3.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// PL consecutive values of a row to fp32, and back.
template <bool BF, int PL>
__device__ __forceinline__ void load_row(const uint16_t* x, float (&v)[PL]) {
#pragma unroll
  for (int i = 0; i < PL / 2; ++i) {
    const float2 w = unpack2<BF>(reinterpret_cast<const uint32_t*>(x)[i]);
    v[2 * i] = w.x;
    v[2 * i + 1] = w.y;
  }
}
template <bool BF, int PL>
__device__ __forceinline__ void store_row(uint16_t* y, const float (&v)[PL], float f) {
#pragma unroll
  for (int i = 0; i < PL / 2; ++i) reinterpret_cast<uint32_t*>(y)[i] = pack2<BF>(v[2 * i] * f, v[2 * i + 1] * f);
}

// The running reference m of a row follows its maximum only when a score rises 2^7 above it, which
// saves the reductions and rescalings of most steps: probabilities reach 2^(shift + 7), 2^15 in
// fp16, and what lies 2^-32 below the reference still counts there.
constexpr float kHeadroom = 7.0f;
template <bool BF>
constexpr float kProbShift = BF ? 0.0f : 8.0f;

// Work is dealt out in units: a chunk is one, and an item's start and end cost about as much as
// kPaItemUnits more (queries fetched, warps joined), which short items would otherwise pile up in one CTA.
constexpr int kPaItemUnits = 2;
// Where no sequence can have more tokens than this, an item is one unit, no CTA shares one, and the
// joining launch falls away.  Measured, eager calls of one sequence, 8 KV heads: 256 tokens 10.3 us
// whole against 12.5 split, 512 tokens 12.9 against 12.4, 1024 tokens 21.7 against 12.6.
constexpr int kPaWholeTokens = 256;

// Where a walk over a CTA's run stands: sequence, item (KV head and row block), chunk, and the
// units left (a chunk is there while they are positive).  A chunk takes a.chunk_units of them, an
// item's start a.item_units: 1 and kPaItemUnits, or 0 and 1 where items stay whole.
struct Walk {
  int b, item, chunk, chunks;
  int64_t left;
};

template <int D>
struct Tile {
  static constexpr int keys = D == 128 ? 16 : 32;   // of a warp's stage
  static constexpr int groups = keys / 16;
  static constexpr int chunk = keys * kPaWarps;
  static constexpr int pieces = D / 8;              // 16-byte pieces of a row
  static constexpr int rows = 32 / pieces;          // rows that a warp's copy instruction covers
};

// `end`: a sequence's tokens, the new ones among them; 0 for a place without one.
template <int D>
__device__ __forceinline__ int chunks_of(int end) {
  return (end + Tile<D>::chunk - 1) / Tile<D>::chunk;
}
template <int D>
__device__ __forceinline__ int64_t units_of(const AttnArgs& a, int end, int items) {
  return end == 0 ? 0 : (int64_t)(chunks_of<D>(end) * a.chunk_units + a.item_units) * items;
}

// ALIGNED: a page holds a multiple of 16 tokens, so that 16 neighbours from a multiple of 16 on lie
// in one page and one look-up serves them; otherwise every lane looks up its own token.
// NT: the block's rows in eights.
template <bool BF, int D, int NT, bool ALIGNED>
__global__ void __launch_bounds__(kPaThreads, 2) k_paged_attn(AttnArgs a) {
  constexpr int KT = Tile<D>::keys, CH = Tile<D>::chunk, NS = kPaStages, RB = 8 * NT, G = Tile<D>::groups;
  constexpr bool QS = NT > 3;  // queries in shared memory: the outputs take the registers
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* s_q = smem + kPaWarps * NS * kPaStage;  // [RB][D] when it does not fit the registers
  float* s_m = reinterpret_cast<float*>(s_q + (QS ? RB * D * 2 : 0));
  float* s_l = s_m + kPaWarps * 16;
  float* s_exact = s_l + kPaWarps * 16;
  int* s_end = reinterpret_cast<int*>(s_exact + kPaWarps * 16);
  __shared__ int64_t s_sum[kPaWarps];
  __shared__ Walk s_walk;
  pdl_trigger();
  pdl_wait();
  const PagedView& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int items = c.kv_heads * a.blocks;

  // the lengths, and this CTA's run of units [u0, u1)
  int64_t sum = 0;
  for (int b = tid; b < c.batch; b += kPaThreads) {
    const int len = c.lengths[b];
    int end = 0;
    if (len >= 0) {
      if ((int64_t)len + a.tokens <= c.capacity) end = len + a.tokens;
      else if (blockIdx.x == 0) report_bad_attn_page();
    }
    s_end[b] = end;
    sum += units_of<D>(a, end, items);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kPaWarps; ++w) total += s_sum[w];
  const int64_t ctas = min((int64_t)kPaGrid, total);
  const int64_t u0 = blockIdx.x < ctas ? blockIdx.x * total / ctas : total;
  const int64_t u1 = blockIdx.x < ctas ? (blockIdx.x + 1) * total / ctas : total;
  if (warp == 0 && (u0 < u1 || blockIdx.x == 0)) {
    int64_t base = 0;
    for (int b0 = 0; b0 < c.batch; b0 += 32) {
      const int b = b0 + lane;
      const int n = b < c.batch ? chunks_of<D>(s_end[b]) : 0;
      const int64_t mine = b < c.batch ? units_of<D>(a, s_end[b], items) : 0;
      int64_t inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
      }
      const int64_t first = base + inc - mine;
      if (u0 >= first && u0 < first + mine) {
        const int per = n * a.chunk_units + a.item_units, item = (int)((u0 - first) / per);
        const int x = (int)(u0 - first - (int64_t)item * per);
        s_walk = a.chunk_units ? Walk{b, item, max(0, x - kPaItemUnits), n, u1 - u0 - max(0, kPaItemUnits - x)}
                               : Walk{b, item, 0, n, u1 - u0};
      }
      if (blockIdx.x == 0 && b < c.batch) {
        a.prefix[b] = first;
        if (b == c.batch - 1) a.prefix[c.batch] = total;
      }
      base += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  __syncthreads();
  if (u0 >= u1 || s_walk.left <= 0) return;

  auto advance = [&](Walk& w) {
    w.left -= a.chunk_units;
    if (++w.chunk < w.chunks) return;
    w.left -= a.item_units;
    w.chunk = 0;
    if (++w.item < items || w.left <= 0) return;
    w.item = 0;
    do ++w.b;
    while (w.b < c.batch && s_end[w.b] == 0);
    if (w.b < c.batch) w.chunks = chunks_of<D>(s_end[w.b]);
  };

  // Offsets in the pools of the walk's chunk for this warp: of each group of 16 tokens (ALIGNED), or
  // of the lane's token; -1 where there is none.
  struct Places {
    int64_t at[ALIGNED ? G : 1];
  };
  auto places = [&](const Walk& w) {
    Places p;
#pragma unroll
    for (int g = 0; g < (ALIGNED ? G : 1); ++g) {
      const int key = w.chunk * CH + warp * KT + (ALIGNED ? g * 16 : lane);
      p.at[g] = -1;
      if (w.left > 0 && (ALIGNED || lane < KT) && key < s_end[w.b]) {
        const uint32_t in = (uint32_t)key / a.page;
        const int page = c.table[w.b * c.ld_table + in];
        if (page >= 0 && page < c.n_pages)
          p.at[g] = page * c.page_stride + (int64_t)(key - (int)(in * a.page.d)) * c.token_stride;
        else
          report_bad_attn_page();
      }
    }
    return p;
  };
  const uint32_t ring = smem_u32(smem) + warp * NS * kPaStage;
  const int my_row = lane / Tile<D>::pieces, my_piece = lane % Tile<D>::pieces;
  const int64_t v_from_k = c.v - c.k, my_off = my_row * c.token_stride + my_piece * 8;
  auto fetch = [&](const Walk& w, const Places& p, int slot) {
    const int64_t head = (int64_t)(w.item / a.blocks) * c.head_stride;
    const uint32_t dst = ring + slot * kPaStage;
    const int there = s_end[w.b] - (w.chunk * CH + warp * KT);  // tokens of the tile that there are
#pragma unroll
    for (int i = 0; i < KT / Tile<D>::rows; ++i) {
      const int r = i * Tile<D>::rows + my_row;
      const uint16_t* x;
      bool ok;
      if (ALIGNED) {
        constexpr int per = 16 / Tile<D>::rows;  // instructions of a group
        ok = r < there && p.at[i / per] >= 0;
        x = c.k + p.at[i / per] + head + my_off + (int64_t)((i % per) * Tile<D>::rows) * c.token_stride;
      } else {
        const int64_t off = __shfl_sync(0xffffffffu, p.at[0], r);
        ok = off >= 0;
        x = c.k + off + head + my_piece * 8;
      }
      if (!ok) x = c.k;  // an address, not read
      const uint32_t to = dst + r * (D * 2) + ((my_piece ^ (r & 7)) << 4);
      cp_async16(to, x, ok ? 16u : 0u);
      cp_async16(to + KT * D * 2, ok ? x + v_from_k : x, ok ? 16u : 0u);
    }
  };

  Walk get = s_walk, load = s_walk;
  Places next = places(load);
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    if (load.left > 0) {
      fetch(load, next, i);
      advance(load);
      next = places(load);
    }
    cp_async_commit();
  }

  // Everything is transposed, so that the few rows are the narrow side of the matrix instruction: the
  // products are keys x rows (16 x 8), the outputs dims x rows, both m16n8k16; the probabilities
  // change sides by an 8 x 8 transposition.  Lane l holds rows 2 (l % 4) and the next of each eight.
  uint32_t qf[QS ? 1 : D / 16][NT][2];
  float o[D / 16][NT][4], m[NT][2], l[NT][4], exact[NT][2];
  // A probability goes into the products as two 16-bit numbers, its rounding and the rest: rounded once
  // its error would equal that of the output's own rounding (1.4 times the error in all); the second
  // product costs nothing while the loads decide (up to 16 rows; 5% at 24, 14% at 32).  A row of ones
  // beside the values sums them into l as the products see them, so that what is left of the rounding
  // cancels; `exact` sums them in fp32, for the weights.
  const uint32_t one2 = BF ? 0x3F803F80u : 0x3C003C00u;
  const uint32_t ones[4] = {one2, one2, one2, one2};
  const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;  // on q, so that a larger product weighs more
  // a masked -inf stays one under a scale of 0, and no finite score counts under 2^-149
  const float scale = fmaxf(fabsf(a.scale), 0x1p-149f);
  const int lrow = lane & 7, lmat = lane >> 3;
  // a 16 x 16 tile's four 8 x 8 matrices, rows first and columns first
  const uint32_t rows_first = ((lmat & 1) * 8 + lrow) * (D * 2) + (((lmat >> 1) ^ lrow) << 4);
  const uint32_t cols_first = ((lmat >> 1) * 8 + lrow) * (D * 2) + (((lmat & 1) ^ lrow) << 4);
  const uint32_t q_lane = smem_u32(s_q) + cols_first;
  int parts = 0, began = get.chunk, slot = 0;
  bool fresh = true;
  while (get.left > 0) {
    const int g = get.item / a.blocks, rb = get.item - g * a.blocks;
    const int end = s_end[get.b], len = end - a.tokens;  // row t sees the keys 0 .. len + t
    if (fresh) {
      fresh = false;
      // the row block's queries: matrix fragments in registers, or rows in shared memory for ldmatrix
      if (!QS) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int r = rb * RB + n * 8 + (lane >> 2), tok = r / a.rep;
          const uint32_t* x = reinterpret_cast<const uint32_t*>(a.q + ((int64_t)get.b * a.tokens + tok) * a.ldq +
                                                                (int64_t)(g * a.rep + r - tok * a.rep) * D) + (lane & 3);
#pragma unroll
          for (int k = 0; k < (QS ? 1 : D / 16); ++k) {
            qf[k][n][0] = r < a.rows ? x[k * 8] ^ sign : 0u;
            qf[k][n][1] = r < a.rows ? x[k * 8 + 4] ^ sign : 0u;
          }
        }
      } else {
#pragma unroll
        for (int e = tid; e < RB * D / 8; e += kPaThreads) {
          const int w = e / (D / 8), piece = e % (D / 8), r = rb * RB + w, tok = r / a.rep;
          uint4 x = make_uint4(0, 0, 0, 0);
          if (r < a.rows)
            x = *reinterpret_cast<const uint4*>(a.q + ((int64_t)get.b * a.tokens + tok) * a.ldq +
                                                (int64_t)(g * a.rep + r - tok * a.rep) * D + piece * 8);
          *reinterpret_cast<uint4*>(s_q + w * D * 2 + ((piece ^ (w & 7)) << 4)) =
              make_uint4(x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign);
        }
        __syncthreads();
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = l[n][2] = l[n][3] = exact[n][0] = exact[n][1] = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[j][n][i] = 0.0f;
      }
    }
    cp_async_wait<NS - 2>();
    __syncwarp();
    // the stage read one round ago takes the chunk NS - 1 ahead
    if (load.left > 0) {
      fetch(load, next, slot == 0 ? NS - 1 : slot - 1);
      advance(load);
      next = places(load);
    }
    cp_async_commit();
    const int key0 = get.chunk * CH + warp * KT;
    if (key0 < end) {
      const uint32_t kb = ring + slot * kPaStage + rows_first, vb = ring + slot * kPaStage + KT * D * 2 + cols_first;
      float s[KT / 16][NT][4];  // 16 keys x 8 rows: keys lane / 4 and 8 on, two rows each
#pragma unroll
      for (int h = 0; h < KT / 16; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[h][n][i] = 0.0f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t qk[NT][2];
        if (QS) {
#pragma unroll
          for (int n = 0; n + 1 < NT; n += 2)
            ldmatrix_x4((q_lane ^ (k << 5)) + n * 8 * D * 2, qk[n][0], qk[n][1], qk[n + 1][0], qk[n + 1][1]);
        } else {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            qk[n][0] = qf[QS ? 0 : k][n][0];
            qk[n][1] = qf[QS ? 0 : k][n][1];
          }
        }
#pragma unroll
        for (int h = 0; h < KT / 16; ++h) {
          uint32_t ka[4];
          ldmatrix_x4((kb ^ (k << 5)) + h * 16 * D * 2, ka[0], ka[1], ka[2], ka[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<BF>(s[h][n], ka, qk[n][0], qk[n][1]);
        }
      }
      const bool edge = key0 + KT > len + 1;  // not every row sees every key
      if (edge) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int seen = len + (rb * RB + n * 8 + (lane & 3) * 2 + i) / a.rep;
#pragma unroll
            for (int h = 0; h < KT / 16; ++h) {
              if (key0 + h * 16 + (lane >> 2) > seen) s[h][n][i] = -INFINITY;
              if (key0 + h * 16 + (lane >> 2) + 8 > seen) s[h][n][i + 2] = -INFINITY;
            }
          }
      }
      if (a.scores) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int r = rb * RB + n * 8 + (lane & 3) * 2;
          float* to = a.scores + (((int64_t)get.b * c.kv_heads + g) * a.max_keys + key0 + (lane >> 2)) * a.ld_scores + r;
          if (r < a.ld_scores)  // an odd row's neighbour is padding
#pragma unroll
            for (int h = 0; h < KT / 16; ++h)
#pragma unroll
              for (int z = 0; z < 2; ++z)
                if (key0 + h * 16 + z * 8 + (lane >> 2) < end)
                  *reinterpret_cast<float2*>(to + (int64_t)(h * 16 + z * 8) * a.ld_scores) =
                      make_float2(s[h][n][2 * z] * scale, s[h][n][2 * z + 1] * scale);
        }
      }
      uint32_t p[KT / 16][NT][2], rest[KT / 16][NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        // the exponents scale s - m + shift against the reference m; where one of them leaves the
        // headroom (or a row has no reference yet) m becomes the true maximum so far
        float e[KT / 16][4];
        auto exponents = [&] {
          const float z[2] = {kProbShift<BF> - (m[n][0] == -INFINITY ? 0.0f : m[n][0]),
                              kProbShift<BF> - (m[n][1] == -INFINITY ? 0.0f : m[n][1])};
#pragma unroll
          for (int h = 0; h < KT / 16; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) e[h][i] = fmaf(s[h][n][i], scale, z[i & 1]);
        };
        exponents();
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int h = 0; h < KT / 16; ++h) {
          top[0] = fmaxf(top[0], fmaxf(e[h][0], e[h][2]));
          top[1] = fmaxf(top[1], fmaxf(e[h][1], e[h][3]));
        }
        const bool grow = top[0] > (m[n][0] == -INFINITY ? -INFINITY : kProbShift<BF> + kHeadroom) ||
                          top[1] > (m[n][1] == -INFINITY ? -INFINITY : kProbShift<BF> + kHeadroom);
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float mx = -INFINITY;
#pragma unroll
            for (int h = 0; h < KT / 16; ++h) mx = fmaxf(mx, fmaxf(s[h][n][i], s[h][n][i + 2]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mx = fmaxf(mx * scale, m[n][i]);
            const float f = m[n][i] == -INFINITY ? 0.0f : ex2(m[n][i] - mx);
            l[n][i] *= f;
            l[n][i + 2] *= f;
            exact[n][i] *= f;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
              o[j][n][i] *= f;
              o[j][n][i + 2] *= f;
            }
            m[n][i] = mx;
          }
          exponents();
        }
#pragma unroll
        for (int h = 0; h < KT / 16; ++h) {
#pragma unroll
          for (int i = 0; i < 4; ++i) e[h][i] = ex2(e[h][i]);
          if (a.scores) {
            exact[n][0] += e[h][0] + e[h][2];
            exact[n][1] += e[h][1] + e[h][3];
          }
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint32_t high = pack2<BF>(e[h][2 * z], e[h][2 * z + 1]);
            const float2 rounded = unpack2<BF>(high);
            p[h][n][z] = transpose8x8(high);
            rest[h][n][z] = transpose8x8(pack2<BF>(e[h][2 * z] - rounded.x, e[h][2 * z + 1] - rounded.y));
          }
          mma16816<BF>(l[n], ones, p[h][n][0], p[h][n][1]);
          mma16816<BF>(l[n], ones, rest[h][n][0], rest[h][n][1]);
        }
      }
      if (edge && a.tokens > 1) {
        // A weight of 0 does not keep an infinity or NaN among the newest values from the rows that do
        // not see them: where there is one, its key's values are added row by row on plain arithmetic
        // and taken out of the stage.
        uint32_t bad = 0;
        const uint32_t v0 = ring + slot * kPaStage + KT * D * 2;
        const int first = max(0, len + 1 - key0), behind = min(KT, end - key0);
        for (int r = first; r < behind; ++r) {
          bool odd = false;
          if (lane < D / 8) {
            uint32_t x[4];
            lds128(v0 + r * (D * 2) + (lane << 4), x);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              constexpr uint32_t e = BF ? 0x7F80u : 0x7C00u;
              odd |= (x[i] & e) == e || (x[i] & (e << 16)) == e << 16;
            }
          }
          if (__any_sync(0xffffffffu, odd)) bad |= 1u << r;
        }
        for (; bad; bad &= bad - 1) {
          const int r = __ffs((int)bad) - 1;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int w = (lane & 3) * 2 + i;  // its probability lies transposed, in lane 4 w + key / 2
              uint32_t x = 0, x2 = 0;
#pragma unroll
              for (int h = 0; h < KT / 16; ++h)
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                  const uint32_t y = __shfl_sync(0xffffffffu, p[h][n][z], w * 4 + ((r & 7) >> 1));
                  const uint32_t y2 = __shfl_sync(0xffffffffu, rest[h][n][z], w * 4 + ((r & 7) >> 1));
                  if (r >> 3 == 2 * h + z) {
                    x = y;
                    x2 = y2;
                  }
                }
              const float2 two = unpack2<BF>(x), two2 = unpack2<BF>(x2);
              const float pr = r & 1 ? two.y + two2.y : two.x + two2.x;
              if (key0 + r <= len + (rb * RB + n * 8 + w) / a.rep)
#pragma unroll
                for (int j = 0; j < D / 16; ++j)
#pragma unroll
                  for (int z = 0; z < 2; ++z) {
                    const int d = j * 16 + z * 8 + (lane >> 2);
                    const uint16_t v = lds16(v0 + r * (D * 2) + (((d >> 3) ^ (r & 7)) << 4) + (d & 7) * 2);
                    o[j][n][i + 2 * z] = fmaf(pr, to_f<BF>(v), o[j][n][i + 2 * z]);
                  }
            }
          __syncwarp();
          if (lane < D / 8) sts128_zero(v0 + r * (D * 2) + (lane << 4));
          __syncwarp();
        }
      }
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int h = 0; h < KT / 16; ++h) {
          uint32_t va[4];
          ldmatrix_x4_trans((vb ^ (j << 5)) + h * 16 * D * 2, va[0], va[1], va[2], va[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<BF>(o[j][n], va, p[h][n][0], p[h][n][1]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<BF>(o[j][n], va, rest[h][n][0], rest[h][n][1]);
        }
    }
    const Walk now = get;
    const bool last = now.chunk + 1 == now.chunks;
    advance(get);
    if (last || get.left <= 0) {
      // The item's end in this run: the warps' parts join, through the stage just read, all 16 rows
      // of a block at once: 8 threads per row, each the 4 values from j * 32 + 4 * part on.
      const bool whole = last && began == 0;
      float* mine = reinterpret_cast<float*>(smem + warp * NS * kPaStage + slot * kPaStage);
      const int r = tid >> 3, part = tid & 7;
      auto turn = [](int row) { return ((row >> 1) & 3) << 3; };
#pragma unroll
      for (int t = 0; t < (NT + 1) / 2; ++t) {
        const int rr = rb * RB + t * 16 + r;
        const bool there = t * 16 + r < RB && rr < a.rows;
        const int tok = rr / a.rep, head = g * a.rep + rr - tok * a.rep;
        const int64_t row = (int64_t)now.b * a.tokens + tok;
        __syncwarp();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n = 2 * t + h;
          if (n < NT)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int w = h * 8 + (lane & 3) * 2 + i;
              float x = exact[n < NT ? n : 0][i];
              x += __shfl_xor_sync(0xffffffffu, x, 4);
              x += __shfl_xor_sync(0xffffffffu, x, 8);
              x += __shfl_xor_sync(0xffffffffu, x, 16);
              if (lane < 4) {
                s_exact[warp * 16 + w] = x;
                s_m[warp * 16 + w] = m[n < NT ? n : 0][i];
                s_l[warp * 16 + w] = l[n < NT ? n : 0][i];
              }
#pragma unroll
              for (int j = 0; j < D / 16; ++j) {  // columns turned by the row, against bank conflicts
                mine[w * D + ((j * 16 + (lane >> 2)) ^ turn(w))] = o[j][n < NT ? n : 0][i];
                mine[w * D + ((j * 16 + 8 + (lane >> 2)) ^ turn(w))] = o[j][n < NT ? n : 0][i + 2];
              }
            }
        }
        __syncthreads();
        float M = -INFINITY, L = 0.0f, E = 0.0f, acc[D / 32][4];
#pragma unroll
        for (int w = 0; w < kPaWarps; ++w) M = fmaxf(M, s_m[w * 16 + r]);
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
#pragma unroll
        for (int w = 0; w < kPaWarps; ++w) {
          const float lw = s_l[w * 16 + r];
          const float f = lw == 0.0f ? 0.0f : ex2(s_m[w * 16 + r] - M);
          const float* x = reinterpret_cast<const float*>(smem + w * NS * kPaStage + slot * kPaStage) + r * D;
          if (lw != 0.0f) {
            L = fmaf(lw, f, L);
            E = fmaf(s_exact[w * 16 + r], f, E);
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
              const float4 y = *reinterpret_cast<const float4*>(x + ((j * 32 + part * 4) ^ turn(r)));
              acc[j][0] = fmaf(y.x, f, acc[j][0]);
              acc[j][1] = fmaf(y.y, f, acc[j][1]);
              acc[j][2] = fmaf(y.z, f, acc[j][2]);
              acc[j][3] = fmaf(y.w, f, acc[j][3]);
            }
          }
        }
        if (there) {
          if (whole) {
#pragma unroll
            for (int j = 0; j < D / 32; ++j)
              store_row<BF, 4>(a.out + row * a.ldo + (int64_t)head * D + j * 32 + part * 4, acc[j], 1.0f / L);
            if (a.lse && part == 0)
              a.lse[((int64_t)now.b * c.kv_heads + g) * a.ld_scores + rr] = M + log2f(E) - kProbShift<BF>;
          } else {
            const int64_t at = (int64_t)(2 * blockIdx.x + (parts > 0 ? 1 : 0)) * RB + t * 16 + r;
#pragma unroll
            for (int j = 0; j < D / 32; ++j)
              *reinterpret_cast<float4*>(a.part + at * D + j * 32 + part * 4) =
                  make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
            if (part == 0) a.part_ml[at] = make_float4(M, L, E, 0.0f);
          }
        }
        __syncthreads();  // before the stages are filled again, or the next 16 rows come
      }
      ++parts;
      began = 0;
      fresh = true;
    }
    slot = slot + 1 == NS ? 0 : slot + 1;
  }
  cp_async_wait<0>();
}

// The parts of an item that several CTAs shared, joined in the cache's order: grid (items, rows / rows
// of a CTA), WR of the CTA's four warps on a row, each adding up every WR-th part.  Latency-bound:
// after the parts' m and l come their o, eight in flight per warp.
constexpr int kJoinWarps = 4;

template <bool BF, int D, int WR>
__global__ void __launch_bounds__(kJoinWarps * 32) k_paged_attn_join(AttnArgs a, int RB) {
  constexpr int PL = D / 32, W = kJoinWarps;
  __shared__ float s_l[W], s_e[W];
  __shared__ __align__(16) float s_o[WR > 1 ? W : 1][D];
  pdl_trigger();
  const PagedView& c = a.c;
  const int items = c.kv_heads * a.blocks;
  const int b = blockIdx.x / items, item = blockIdx.x - b * items, g = item / a.blocks, rb = item - g * a.blocks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WR;
  const int r = blockIdx.y * (W / WR) + warp / WR, rr = rb * RB + r;
  pdl_wait();
  const int64_t p0 = a.prefix[b], p1 = a.prefix[b + 1], total = a.prefix[c.batch];
  if (p0 == p1 || rr >= a.rows) return;  // with WR > 1 the whole CTA
  // the CTAs whose runs meet the item's chunks, units [c0, c1) behind its kPaItemUnits: 32-bit
  // divisions where they do; and whether the item is not the first of CTA i0's run
  const int64_t ctas = min((int64_t)kPaGrid, total);
  int i0, i1;
  bool second;
  if (total < (1 << 23)) {
    const uint32_t n = (uint32_t)(p1 - p0) / items, at = (uint32_t)p0 + item * n, t = (uint32_t)total, u = (uint32_t)ctas;
    i0 = (int)(((at + kPaItemUnits + 1) * u - 1) / t);
    i1 = (int)(((at + n) * u - 1) / t);
    second = i0 * t / u < at;
  } else {
    const int64_t n = (p1 - p0) / items, at = p0 + item * n;
    i0 = (int)(((at + kPaItemUnits + 1) * ctas - 1) / total);
    i1 = (int)(((at + n) * ctas - 1) / total);
    second = i0 * total / ctas < at;
  }
  if (i0 == i1) return;  // one CTA had it whole
  const int n = i1 + 1 - i0;
  auto part = [&](int i) { return (2 * (i0 + i) + (i == 0 && second ? 1 : 0)) * RB + r; };
  float M = -INFINITY, L = 0.0f, E = 0.0f, acc[PL];
#pragma unroll
  for (int j = 0; j < PL; ++j) acc[j] = 0.0f;
#pragma unroll 4
  for (int i = lane; i < n; i += 32) M = fmaxf(M, a.part_ml[part(i)].x);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
  for (int base = sub; base < n; base += 8 * WR) {
    float x[8][PL], f = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = base + k * WR;
      const float* y = a.part + (int64_t)part(min(i, n - 1)) * D + lane * PL;
      if (D == 128) {
        const float4 z = *reinterpret_cast<const float4*>(y);
        x[k][0] = z.x;
        x[k][1] = z.y;
        x[k][PL - 2] = z.z;
        x[k][PL - 1] = z.w;
      } else {
        const float2 z = *reinterpret_cast<const float2*>(y);
        x[k][0] = z.x;
        x[k][1] = z.y;
      }
    }
    if (lane < 8 && base + lane * WR < n) {  // lane k holds the factor of the k-th of them
      const float4 ml = a.part_ml[part(base + lane * WR)];
      f = ml.y == 0.0f ? 0.0f : ex2(ml.x - M);
      L = fmaf(ml.y, f, L);
      E = fmaf(ml.z, f, E);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float w = __shfl_sync(0xffffffffu, f, k);
      if (base + k * WR < n)
#pragma unroll
        for (int j = 0; j < PL; ++j) acc[j] = fmaf(x[k][j], w, acc[j]);
    }
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {
    L += __shfl_xor_sync(0xffffffffu, L, x);
    E += __shfl_xor_sync(0xffffffffu, E, x);
  }
  if (WR > 1) {
    if (lane == 0) {
      s_l[warp] = L;
      s_e[warp] = E;
    }
#pragma unroll
    for (int j = 0; j < PL; ++j) s_o[warp % (WR > 1 ? W : 1)][lane * PL + j] = acc[j];
    __syncthreads();
    if (sub) return;
    L = E = 0.0f;
#pragma unroll
    for (int j = 0; j < PL; ++j) acc[j] = 0.0f;
#pragma unroll
    for (int w = 0; w < WR; ++w) {
      L += s_l[warp + w];
      E += s_e[warp + w];
#pragma unroll
      for (int j = 0; j < PL; ++j) acc[j] += s_o[(warp + w) % (WR > 1 ? W : 1)][lane * PL + j];
    }
  }
  const int tok = rr / a.rep, head = g * a.rep + rr - tok * a.rep;
  store_row<BF, PL>(a.out + ((int64_t)b * a.tokens + tok) * a.ldo + (int64_t)head * D + lane * PL, acc, 1.0f / L);
  if (a.lse && lane == 0) a.lse[((int64_t)b * c.kv_heads + g) * a.ld_scores + rr] = M + log2f(E) - kProbShift<BF>;
}

// weights[b, g, s] += sum over the item's rows of 2^(score - lse): a thread per token, rows in order.
// Memory-bound: the scores are read once, mostly from L2.  The grid covers all tokens that the table has room
// for only up to kWeightCtas CTAs, which then go on to further tokens, so that room for long sequences costs
// short ones little: whole calls, 64 sequences of 100 tokens, 8 KV heads, room for 8192 tokens, 22.8 us with
// 8192 CTAs, 31 with 16384, 48 with all 32768 (for 131072 tokens the same, and 554 with all); 64 of 4000
// tokens, 32 rows, room for 4096, 435 us with 8192, 428 with 16384, 426 with all.
constexpr int kWeightThreads = 128;
constexpr int64_t kWeightCtas = 16384;

__global__ void __launch_bounds__(kWeightThreads, 16) k_paged_attn_weights(AttnArgs a, float* weights, int64_t ldw) {
  pdl_trigger();
  pdl_wait();
  const PagedView& c = a.c;
  const int g = blockIdx.y, b = blockIdx.z, len = c.lengths[b];
  if (len < 0 || (int64_t)len + a.tokens > c.capacity) return;
  const int64_t item = (int64_t)b * c.kv_heads + g;
  const float* lse = a.lse + item * a.ld_scores;
  auto term = [](float v, float l) { return v == -INFINITY ? 0.0f : ex2(v - l); };
#pragma unroll 1
  for (int s = blockIdx.x * kWeightThreads + threadIdx.x; s < len + a.tokens; s += gridDim.x * kWeightThreads) {
    const float* x = a.scores + (item * a.max_keys + s) * a.ld_scores;
    float sum = 0.0f;
#pragma unroll 4
    for (int r = 0; r < a.rows; r += 4) {
      const float4 v = *reinterpret_cast<const float4*>(x + r), l = *reinterpret_cast<const float4*>(lse + r);
      sum += term(v.x, l.x);
      if (r + 1 < a.rows) sum += term(v.y, l.y);
      if (r + 2 < a.rows) sum += term(v.z, l.z);
      if (r + 3 < a.rows) sum += term(v.w, l.w);
    }
    weights[item * ldw + s] += sum;
  }
}

// The sizes that there are limits for.  Within them a head's scores take 2^52 bytes at most.
static bool attn_limits(int64_t batch, int64_t heads, int64_t kv_heads, int64_t D, int64_t tokens, int64_t max_tokens) {
  return batch <= kPagedMaxBatch && heads <= 65535 && kv_heads <= 1024 && (D == 64 || D == 128) &&
         tokens <= kPagedMaxTokens && max_tokens <= 1ll << 30;
}

// With weights, the scores that one pass may keep: rows x capacity x 4 bytes of a KV head, whatever the
// lengths are.  Calls with more of them go through several passes, one after another, of as many sequences
// as fit, or of as many KV heads of one sequence (one at least).
constexpr int64_t kPaScoreBytes = 2ll << 30;

// Bytes of the workspace's parts, in order, and the sequences and KV heads of a pass.
struct AttnSpace {
  int64_t prefix, part, part_ml, lse, scores, ld_scores;
  int64_t batch, kv_heads;
  int64_t bytes() const { return prefix + part + part_ml + lse + scores; }
};
// Rows of a block: eights, 32 at most.
static int block_rows(int64_t rows) { return rows >= 32 ? 32 : (int)((rows + 7) / 8 * 8); }
static AttnSpace attn_space(int64_t batch, int64_t heads, int64_t kv_heads, int64_t D, int64_t tokens, int64_t max_tokens,
                            bool weights) {
  AttnSpace s;
  const int64_t rows = heads / kv_heads * tokens, RB = block_rows(rows);
  s.prefix = align_up((batch + 1) * 8, 256);
  s.part = align_up(2 * kPaGrid * RB * D * 4, 256);
  s.part_ml = align_up(2 * kPaGrid * RB * 16, 256);
  s.ld_scores = align_up(rows, 4);
  s.batch = batch;
  s.kv_heads = kv_heads;
  s.lse = s.scores = 0;
  if (weights) {
    const int64_t each = s.ld_scores * max_tokens * 4, fit = std::max<int64_t>(1, kPaScoreBytes / each);
    s.kv_heads = std::min(kv_heads, fit);
    s.batch = std::min(batch, std::max<int64_t>(1, fit / kv_heads));
    s.lse = align_up(s.batch * s.kv_heads * s.ld_scores * 4, 256);
    s.scores = align_up(s.batch * s.kv_heads * each, 256);
  }
  return s;
}

template <bool BF, int D>
static cudaError_t launch_join(const AttnArgs& a, int RB, cudaStream_t s) {
  // Few rows are shared by many CTAs each: a join CTA per row, its four warps on a quarter of the parts
  // each; many rows by few: a warp per row.
  const int64_t items = (int64_t)a.c.batch * a.c.kv_heads * a.blocks;
  const int rows = std::min(a.rows, RB);
  if (items * rows <= kPaGrid * 4)
    return launch_pdl(k_paged_attn_join<BF, D, 4>, dim3((unsigned)items, (unsigned)rows), dim3(kJoinWarps * 32), 0, s, 1u, a, RB);
  return launch_pdl(k_paged_attn_join<BF, D, 1>, dim3((unsigned)items, (unsigned)(rows + 3) / 4), dim3(kJoinWarps * 32), 0,
                    s, 1u, a, RB);
}

template <bool BF, int D, int NT, bool ALIGNED>
static cudaError_t launch_attn_kernel(const AttnArgs& a, size_t dyn, cudaStream_t s) {
  auto* k = k_paged_attn<BF, D, NT, ALIGNED>;
  static std::atomic<bool> done[64];  // the shared-memory opt-in, for the largest batch
  int dev;
  bool needs;
  cudaError_t e = needs_opt_in(done, dev, needs);
  if (e != cudaSuccess) return e;
  if (needs) {
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kPaWarps * kPaStages * kPaStage + kPaWarps * 16 * 12 + 32 * D * 2 +
                                 kPagedMaxBatch * 4);
    if (e != cudaSuccess) return e;
    opted_in(done, dev);
  }
  return launch_pdl(k, dim3(kPaGrid), dim3(kPaThreads), dyn, s, 1u, a);
}

template <bool BF, int D>
static cudaError_t launch_attn(const AttnArgs& a, float* weights, int64_t ldw, cudaStream_t s) {
  const int RB = block_rows(a.rows);
  const size_t dyn = (size_t)kPaWarps * kPaStages * kPaStage + (size_t)kPaWarps * 16 * 12 + (RB > 24 ? RB * D * 2 : 0) +
                     (size_t)a.c.batch * 4;
  const bool aligned = a.c.page_size % 16 == 0;
  cudaError_t e = RB == 8    ? (aligned ? launch_attn_kernel<BF, D, 1, true>(a, dyn, s) : launch_attn_kernel<BF, D, 1, false>(a, dyn, s))
                  : RB == 16 ? (aligned ? launch_attn_kernel<BF, D, 2, true>(a, dyn, s) : launch_attn_kernel<BF, D, 2, false>(a, dyn, s))
                  : RB == 24 ? (aligned ? launch_attn_kernel<BF, D, 3, true>(a, dyn, s) : launch_attn_kernel<BF, D, 3, false>(a, dyn, s))
                             : (aligned ? launch_attn_kernel<BF, D, 4, true>(a, dyn, s) : launch_attn_kernel<BF, D, 4, false>(a, dyn, s));
  if (e != cudaSuccess) return e;
  if (a.chunk_units) e = launch_join<BF, D>(a, RB, s);
  if (e != cudaSuccess || !weights) return e;
  const int64_t blocks = (a.c.capacity + kWeightThreads - 1) / kWeightThreads;
  const int64_t most = std::max<int64_t>(1, kWeightCtas / ((int64_t)a.c.kv_heads * a.c.batch));
  return launch_pdl(k_paged_attn_weights,
                    dim3((unsigned)std::min(blocks, most), (unsigned)a.c.kv_heads, (unsigned)a.c.batch),
                    dim3(kWeightThreads), 0, s, 1u, a, weights, ldw);
}

}  // namespace otf

using otf::check_device;
using otf::set_cuda_error;

int otf::paged_attn_device_error(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, otf::g_paged_attn_device_error, sizeof(int)) != cudaSuccess) {
    set_cuda_error(cudaGetLastError());
    return -1;
  }
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(otf::g_paged_attn_device_error, &z, sizeof(int));
  }
  return v;
}

extern "C" OTF_API int64_t otf_paged_attn_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads,
                                                          int64_t head_dim, int64_t tokens, int64_t max_tokens,
                                                          int with_weights) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || tokens <= 0 || max_tokens <= 0 ||
      !otf::attn_limits(batch, heads, kv_heads, head_dim, tokens, max_tokens))
    return -1;
  return otf::attn_space(batch, heads, kv_heads, head_dim, tokens, max_tokens, with_weights != 0).bytes();
}

extern "C" OTF_API int otf_paged_attn(const otf_paged_cache* cache, const void* q, int64_t ldq, int64_t heads,
                                      int64_t tokens, float scale, void* out, int64_t ldo, float* weights,
                                      int64_t ldw, void* workspace, int64_t workspace_bytes, void* stream) {
  otf::AttnArgs a = {};
  int st = otf::view_of(cache, a.c);
  if (st != OTF_OK) return st;
  const int64_t D = cache->head_dim;
  if (heads <= 0 || heads % a.c.kv_heads || tokens <= 0 || !std::isfinite(scale * otf::kLog2e)) return OTF_ERR_INVALID;
  if (!otf::attn_limits(a.c.batch, heads, a.c.kv_heads, D, tokens, a.c.capacity)) return OTF_ERR_UNSUPPORTED;
  if (!otf::rows16(q, ldq, heads * D) || !otf::rows16(out, ldo, heads * D)) return OTF_ERR_INVALID;
  if (otf::rows_overlap(q, ldq, heads * D, out, ldo, heads * D, a.c.batch * tokens)) return OTF_ERR_INVALID;
  if (weights && ldw < a.c.capacity) return OTF_ERR_INVALID;
  const otf::AttnSpace space = otf::attn_space(a.c.batch, heads, a.c.kv_heads, D, tokens, a.c.capacity, weights != nullptr);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < space.bytes())
    return OTF_ERR_INVALID;
  st = check_device();
  if (st != OTF_OK) return st;
  a.page = otf::fast_div((uint32_t)a.c.page_size);
  a.q = static_cast<const uint16_t*>(q);
  a.ldq = ldq;
  a.out = static_cast<uint16_t*>(out);
  a.ldo = ldo;
  a.scale = scale * otf::kLog2e;
  a.rep = (int)(heads / a.c.kv_heads);
  a.tokens = (int)tokens;
  a.rows = (int)(a.rep * tokens);
  const bool whole = a.c.capacity <= otf::kPaWholeTokens;
  a.chunk_units = whole ? 0 : 1;
  a.item_units = whole ? 1 : otf::kPaItemUnits;
  a.blocks = (a.rows + 31) / 32;
  char* w = static_cast<char*>(workspace);
  a.prefix = reinterpret_cast<int64_t*>(w);
  a.part = reinterpret_cast<float*>(w += space.prefix);
  a.part_ml = reinterpret_cast<float4*>(w += space.part);
  w += space.part_ml;
  if (weights) {
    a.lse = reinterpret_cast<float*>(w);
    a.scores = reinterpret_cast<float*>(w + space.lse);
    a.ld_scores = (int)space.ld_scores;
    a.max_keys = a.c.capacity;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = cache->dtype == OTF_DTYPE_BF16;
  auto* launch = D == 128 ? (bf ? otf::launch_attn<true, 128> : otf::launch_attn<false, 128>)
                          : (bf ? otf::launch_attn<true, 64> : otf::launch_attn<false, 64>);
  for (int64_t b = 0; b < a.c.batch; b += space.batch)
    for (int64_t g = 0; g < a.c.kv_heads; g += space.kv_heads) {  // more than one only with one sequence a pass
      otf::AttnArgs p = a;
      p.c.batch = (int)std::min(space.batch, a.c.batch - b);
      p.c.kv_heads = (int)std::min(space.kv_heads, a.c.kv_heads - g);
      p.c.table += b * a.c.ld_table;
      p.c.lengths += b;
      p.c.k += g * a.c.head_stride;
      p.c.v += g * a.c.head_stride;
      p.q += b * tokens * ldq + g * a.rep * D;
      p.out += b * tokens * ldo + g * a.rep * D;
      const cudaError_t e = launch(p, weights ? weights + (b * a.c.kv_heads + g) * ldw : nullptr, ldw, s);
      if (e != cudaSuccess) return set_cuda_error(e);
    }
  return OTF_OK;
}
