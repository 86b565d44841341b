// A way through a tree of drafted tokens (otf_verify_tree).
//
// At each node, from the root on, the token that follows is drawn from the target's own distribution behind
// that node, p = softmax(target / T), as argmax_i p_i / e_i with e_i ~ Exp(1) given; a child that holds it is
// taken and the walk goes on there, else it ends.  Whatever the tree holds, every token is one of the
// target's distribution.  In logarithms the leader is the largest x_i / T - log e_i, which needs no sum:
// a step is one pass over one row of logits and one of noise, and only the rows on the way are read.
//
// An entry is weighed in fp32, 5 instructions, with a bound on the error; only those that may lead are computed in 64 bits.
//
// Many logits: a sequence is walked by a cluster of CTAs that cut the vocabulary among them (k_verify_tree); a step's
// leaders meet in distributed shared memory.  A step's rows are 8 bytes per entry, but a step cannot start before the
// one before it has ended: some 4 us.  Few logits: every node's leader is found at once by the whole GPU, with the
// noise of the node's depth, and the way is then followed in a second launch (k_tree_leaders, k_tree_walk).
//
// Measured: 64 sequences of 5 to 40 nodes over 128256 at temperature 0.8, ways of 2 rows on average and of 6 or 7 the longest,
// 0.13 to 0.14 GB, 54 to 67 us: 2 to 2.6 TB/s, bound by the longest ways' steps, one after another, while the CTAs of ways
// that have ended idle; one of 26 nodes over 32000, greedy, 7.5 to 7.9 us.
#include <algorithm>

#include "logits.cuh"
#include "paged.cuh"

namespace otf {

int set_cuda_error(cudaError_t e);        // capi.cu
int check_device();                       // capi.cu
int verify_tree_device_error(int clear);  // read (and optionally clear) the flag below

constexpr int kTreeMaxNodes = 64;
constexpr int kTreeThreads = 256;
constexpr int kTreeWarps = kTreeThreads / 32;
constexpr int kTreeCluster = 16;
constexpr int kTreeResident = 148 * 4;  // CTAs that run at once
constexpr int kTreeSlice = 8192;        // entries of a CTA of k_tree_leaders
// Logits of all nodes up to which they are looked at at once.  At once takes as long whatever the way is, clusters some 4 us a
// step and so less for short ways.  The host does not know how long a way is; the border lies where long ways no longer gain,
// and below it short ones lose.  Measured, one way each, clusters against at once, greedy (long ways) and at temperature 0.8
// (shorter ones): one sequence of 26 nodes over 32000 23.5 against 7.6 us and 9.1 against 7.9, of 64
// over 128256 (8.2M) 27 against 19 and 6.5 against 22, 16 of 26 over 32000 (13.3M) 29 against 16 and 30 against 21, 4 of
// 40 over 128256 (20.5M) 30 against 29 and 22 against 37, 16 of 26 over 128256 (53M) 38 against 63 and 35 against 76.
constexpr int64_t kTreeAtOnce = 13ll << 20;

// Set when a sequence has no token to draw, or an argument on the device is out of range.
__device__ int g_verify_tree_device_error;

struct TreeArgs {
  const float* target;
  int64_t ldt;
  const int64_t* tokens;
  const int* parents;
  const int* starts;  // or null: `per` nodes each
  const float* noise;
  int64_t nseq, ldn;
  const float* temperatures;
  double temperature;
  int64_t* out;       // [batch][depth + 1]
  int* path;          // [batch][depth]
  int* accepted;
  int per, n, depth, vocab;
  int batch, slices;
  struct TreeLeader* leaders;  // [n][slices], k_tree_leaders alone
};

struct TreeLeader {
  double score;
  int at;
  int seq;  // in the leaders of k_tree_leaders: whose temperature and noise it was found with, -1: nobody's
};
__device__ __forceinline__ bool leads(double s, int i, const TreeLeader& l) { return s > l.score || (s == l.score && i < l.at); }

// x / T - log e in 64 bits, or x at temperature 0.
__device__ __forceinline__ double tree_score(float x, float e, double T) {
  return T == 0.0 ? (double)x : (double)x / T - log((double)e);
}

// The leader of two lanes' at every lane.
__device__ __forceinline__ TreeLeader tree_leader_of_warp(TreeLeader l) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double s = __shfl_xor_sync(0xffffffffu, l.score, o);
    const int i = __shfl_xor_sync(0xffffffffu, l.at, o);
    if (i != INT_MAX && leads(s, i, l)) l = {s, i, 0};
  }
  return l;
}

// The leader among entries first .. first + 3 and so on, `stride` apart, below `end`, of a row of logits x and of noise e
// (null at temperature 0) that the CTA's threads cut among them: of the warp, at every lane.  s_top: [kTreeWarps].
// In fp32 a score d = x c - log2 e is off by 2^-20 (|x c| + |log2 e| + 1) at most (two roundings, the logarithm's error), and
// |log2 e| <= 150 where d is finite, so what lies 2^-19 (|d| + 304) below the largest d cannot lead.  The entries of a
// thread that has one above are looked at again, by its warp, in 64 bits.
__device__ __forceinline__ TreeLeader tree_leader(const float* x, const float* e, double T, float c, int first, int stride, int end,
                                                  float* s_top) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool ax = (reinterpret_cast<uintptr_t>(x) & 15) == 0, ae = (reinterpret_cast<uintptr_t>(e) & 15) == 0;
  auto weigh = [&](float fx, float fe) { return e ? fmaf(fx, c, -__log2f(fe)) : fx; };
  constexpr int U = 4;
  float top = -INFINITY;  // of the thread; a NaN is none
  for (int i0 = first; i0 < end; i0 += U * stride) {
    float4 vx[U], ve[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (int)min((int64_t)i0 + (int64_t)u * stride, (int64_t)end);  // behind the end: -inf without a read
      vx[u] = logits4(x, i, end, ax);
      if (e) ve[u] = logits4(e, i, end, ae, INFINITY);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      top = fmaxf(top, fmaxf(fmaxf(weigh(vx[u].x, ve[u].x), weigh(vx[u].y, ve[u].y)), fmaxf(weigh(vx[u].z, ve[u].z), weigh(vx[u].w, ve[u].w))));
  }
  float most = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if (lane == 0) s_top[warp] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kTreeWarps; ++w) most = fmaxf(most, s_top[w]);
  // an infinity (a logit's, a noise of 0, or a product's) and -inf alone (small temperatures) are weighed in 64 bits as they are
  const float bar = !e || fabsf(most) == INFINITY ? most : most - 0x1p-19f * (fabsf(most) + 304.0f);
  TreeLeader mine = {-INFINITY, INT_MAX, 0};
  for (uint32_t in = __ballot_sync(0xffffffffu, top >= bar); in; in &= in - 1) {
    const int64_t from = __shfl_sync(0xffffffffu, first, __ffs((int)in) - 1);
    for (int k = lane;; k += 32) {
      const int64_t i = from + (int64_t)(k >> 2) * stride + (k & 3);
      if (i >= end) {
        if ((k & 3) == 0 || from + (int64_t)(k >> 2) * stride >= end) break;
        continue;
      }
      const float fx = x[i], fe = e ? e[i] : 1.0f;
      if (weigh(fx, fe) >= bar) {
        const double s = tree_score(fx, fe, T);
        if (s > -INFINITY && leads(s, (int)i, mine)) mine = {s, (int)i, 0};
      }
    }
    __syncwarp();
  }
  return tree_leader_of_warp(mine);
}

__global__ void __launch_bounds__(kTreeThreads, 4) k_verify_tree(TreeArgs a, int ctas) {
  __shared__ TreeLeader s_warp[kTreeWarps], s_all[2][kTreeCluster];
  __shared__ float s_bar[kTreeWarps];
  __shared__ int64_t s_tokens[kTreeMaxNodes + 1];
  __shared__ int s_path[kTreeMaxNodes], s_at;
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x / ctas, rank = blockIdx.x - b * ctas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r0 = a.starts ? a.starts[b] : b * a.per, r1 = a.starts ? a.starts[b + 1] : r0 + a.per, nodes = r1 - r0;
  const double T = a.temperatures ? (double)a.temperatures[b] : a.temperature;
  const bool ok = r0 >= 0 && r1 <= a.n && nodes > 0 && nodes <= kTreeMaxNodes && temperature_ok(T) && (T == 0.0 || a.noise);
  cluster_arrive_relaxed();
  // the nodes, two in each lane of the first warp
  int64_t token[2] = {-1, -1};
  int parent[2] = {-1, -1};
  if (ok && warp == 0)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (lane + 32 * h < nodes) {
        token[h] = a.tokens[r0 + lane + 32 * h];
        parent[h] = a.parents[r0 + lane + 32 * h];
        // not a node before it: it hangs nowhere
        if (parent[h] >= lane + 32 * h || parent[h] < -1) {
          if (rank == 0) atomicExch(&g_verify_tree_device_error, 1);
          parent[h] = -1;
        }
      }
  int at = 0, taken = 0;
  bool failed = !ok;
  const float c = T > 0.0 ? (float)(1.4426950408889634 / T) : 0.0f;
  cluster_wait();  // all CTAs of the cluster run
  for (int step = 0; !failed; ++step) {
    const float* x = a.target + (int64_t)(r0 + at) * a.ldt;
    const float* e = T > 0.0 ? a.noise + b * a.nseq + step * a.ldn : nullptr;
    TreeLeader mine = tree_leader(x, e, T, c, 4 * (rank * kTreeThreads + tid), 4 * kTreeThreads * ctas, a.vocab, s_bar);
    if (lane == 0) s_warp[warp] = mine;
    __syncthreads();
    if (warp == 0) {
      mine = tree_leader_of_warp(lane < kTreeWarps ? s_warp[lane] : TreeLeader{-INFINITY, INT_MAX, 0});
      if (lane < ctas) {
        const long long bits = __double_as_longlong(mine.score);
        st_cluster_v4(mapa_shared(smem_u32(&s_all[step & 1][rank]), lane), __uint_as_float((uint32_t)bits),
                      __uint_as_float((uint32_t)(bits >> 32)), mine.at);
      }
    }
    __syncwarp();
    cluster_sync_all();
    if (warp == 0) {
      const TreeLeader all = tree_leader_of_warp(lane < ctas ? s_all[step & 1][lane] : TreeLeader{-INFINITY, INT_MAX, 0});
      int child = -1;  // goes on there; -1: ends, -2: nothing to draw
      if (all.at == INT_MAX) {
        child = -2;
      } else {
        if (step < a.depth) {
          const uint32_t h0 = __ballot_sync(0xffffffffu, lane > 0 && parent[0] == at && token[0] == all.at);
          const uint32_t h1 = __ballot_sync(0xffffffffu, parent[1] == at && token[1] == all.at);
          child = h0 ? __ffs((int)h0) - 1 : h1 ? 31 + __ffs((int)h1) : -1;
        }
        if (lane == 0) {
          s_tokens[step] = all.at;
          if (child >= 0) s_path[step] = child;
        }
      }
      if (lane == 0) s_at = child;
    }
    __syncthreads();
    at = s_at;
    if (at == -2) failed = true;
    if (at < 0) break;
    ++taken;
  }
  if (rank) return;
  __syncthreads();
  for (int j = tid; j <= a.depth; j += kTreeThreads) {
    a.out[(int64_t)b * (a.depth + 1) + j] = !failed && j <= taken ? s_tokens[j] : -1;
    if (j < a.depth) a.path[(int64_t)b * a.depth + j] = !failed && j < taken ? s_path[j] : -1;
  }
  if (tid == 0) {
    a.accepted[b] = failed ? 0 : taken;
    if (failed && nodes != 0) atomicExch(&g_verify_tree_device_error, 1);
  }
}

// The leaders of all nodes' rows, grid (slices, n).
__global__ void __launch_bounds__(kTreeThreads, 4) k_tree_leaders(TreeArgs a) {
  __shared__ float s_bar[kTreeWarps];
  __shared__ TreeLeader s_warp[kTreeWarps];
  __shared__ int s_seq, s_level;
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 0) {
    // the first sequence that has the row, and the node's depth, up through its parents in the lanes
    int b = -1, level = 0, r0 = 0, r1 = 0;
    if (a.starts) {
      for (int i = 0; i < a.batch && b < 0; i += 32) {
        const int x = i + lane < a.batch ? a.starts[i + lane] : 0, y = i + lane < a.batch ? a.starts[i + lane + 1] : 0;
        const uint32_t in = __ballot_sync(0xffffffffu, x >= 0 && x <= row && row < y && y <= a.n && y - x <= kTreeMaxNodes);
        if (in) {
          const int from = __ffs((int)in) - 1;
          b = i + from;
          r0 = __shfl_sync(0xffffffffu, x, from);
          r1 = __shfl_sync(0xffffffffu, y, from);
        }
      }
    } else {
      b = row / a.per;
      r0 = b * a.per;
      r1 = r0 + a.per;
    }
    if (b >= 0) {
      int up[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = lane + 32 * h;
        up[h] = r0 + i < r1 ? a.parents[r0 + i] : -1;
        if (up[h] >= i || up[h] < -1) up[h] = -1;
      }
      for (int at = row - r0;;) {
        const int p = at < 32 ? __shfl_sync(0xffffffffu, up[0], at) : __shfl_sync(0xffffffffu, up[1], at - 32);
        if (p < 0) {
          if (at) b = -1;  // does not hang on the root: never reached
          break;
        }
        at = p;
        ++level;
      }
      if (level > a.depth) b = -1;
    }
    if (lane == 0) {
      s_seq = b;
      s_level = level;
    }
  }
  __syncthreads();
  const int b = s_seq;
  TreeLeader* const to = a.leaders + (int64_t)row * a.slices + blockIdx.x;
  const double T = b < 0 ? -1.0 : a.temperatures ? (double)a.temperatures[b] : a.temperature;
  if (!temperature_ok(T) || (T > 0.0 && !a.noise)) {  // k_tree_walk reports a sequence's
    if (tid == 0) *to = {-INFINITY, INT_MAX, -1};
    return;
  }
  const float c = T > 0.0 ? (float)(1.4426950408889634 / T) : 0.0f;
  const float* x = a.target + (int64_t)row * a.ldt;
  const float* e = T > 0.0 ? a.noise + b * a.nseq + s_level * a.ldn : nullptr;
  const int i0 = blockIdx.x * kTreeSlice, end = min(a.vocab, i0 + kTreeSlice);
  const TreeLeader mine = tree_leader(x, e, T, c, i0 + 4 * tid, 4 * kTreeThreads, end, s_bar);
  if (lane == 0) s_warp[warp] = mine;
  __syncthreads();
  if (warp == 0) {
    const TreeLeader all = tree_leader_of_warp(lane < kTreeWarps ? s_warp[lane] : TreeLeader{-INFINITY, INT_MAX, 0});
    if (lane == 0) *to = {all.score, all.at, b};
  }
}

// And the ways through them: a warp per sequence.  Rows that another sequence has too (starts that fall) were looked at
// for the first of them; the others look for themselves.
__global__ void __launch_bounds__(32) k_tree_walk(TreeArgs a) {
  __shared__ int64_t s_tokens[kTreeMaxNodes];
  __shared__ int s_path[kTreeMaxNodes];
  __shared__ int s_drawn[kTreeMaxNodes];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x, lane = threadIdx.x;
  const int r0 = a.starts ? a.starts[b] : b * a.per, r1 = a.starts ? a.starts[b + 1] : r0 + a.per, nodes = r1 - r0;
  const double T = a.temperatures ? (double)a.temperatures[b] : a.temperature;
  bool failed = !(r0 >= 0 && r1 <= a.n && nodes > 0 && nodes <= kTreeMaxNodes && temperature_ok(T) && (T == 0.0 || a.noise));
  int64_t token[2] = {-1, -1};
  int parent[2] = {-1, -1};
  if (!failed) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (lane + 32 * h < nodes) {
        token[h] = a.tokens[r0 + lane + 32 * h];
        parent[h] = a.parents[r0 + lane + 32 * h];
        if (parent[h] >= lane + 32 * h || parent[h] < -1) {
          atomicExch(&g_verify_tree_device_error, 1);
          parent[h] = -1;
        }
      }
    // a lane's nodes' leaders
#pragma unroll 1
    for (int i = lane; i < nodes; i += 32) {
      const TreeLeader* l = a.leaders + (int64_t)(r0 + i) * a.slices;
      TreeLeader all = {-INFINITY, INT_MAX, 0};
#pragma unroll 4
      for (int k = 0; k < a.slices; ++k) {
        const TreeLeader y = l[k];
        if (y.at != INT_MAX && leads(y.score, y.at, all)) all = y;
      }
      s_drawn[i] = l[0].seq == b ? all.at : -1;
    }
  }
  __syncwarp();
  int at = 0, taken = 0;
  while (!failed) {
    int drawn = s_drawn[at];
    if (drawn < 0) {
      const float* x = a.target + (int64_t)(r0 + at) * a.ldt;
      const float* e = T > 0.0 ? a.noise + b * a.nseq + taken * a.ldn : nullptr;
      TreeLeader mine = {-INFINITY, INT_MAX, 0};
      for (int i = lane; i < a.vocab; i += 32) {
        const double s = tree_score(x[i], e ? e[i] : 1.0f, T);
        if (s > -INFINITY && leads(s, i, mine)) mine = {s, i, 0};
      }
      drawn = tree_leader_of_warp(mine).at;
    }
    if (drawn == INT_MAX) {
      failed = true;
      break;
    }
    if (lane == 0) s_tokens[taken] = drawn;
    if (taken == a.depth) break;
    const uint32_t h0 = __ballot_sync(0xffffffffu, lane > 0 && parent[0] == at && token[0] == drawn);
    const uint32_t h1 = __ballot_sync(0xffffffffu, parent[1] == at && token[1] == drawn);
    if (!(h0 | h1)) break;
    at = h0 ? __ffs((int)h0) - 1 : 31 + __ffs((int)h1);
    if (lane == 0) s_path[taken] = at;
    ++taken;
  }
  __syncwarp();
  for (int j = lane; j <= a.depth; j += 32) {
    a.out[(int64_t)b * (a.depth + 1) + j] = !failed && j <= taken ? s_tokens[j] : -1;
    if (j < a.depth) a.path[(int64_t)b * a.depth + j] = !failed && j < taken ? s_path[j] : -1;
  }
  if (lane == 0) {
    a.accepted[b] = failed ? 0 : taken;
    if (failed && nodes != 0) atomicExch(&g_verify_tree_device_error, 1);
  }
}

}  // namespace otf

using otf::check_device;
using otf::set_cuda_error;

int otf::verify_tree_device_error(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, otf::g_verify_tree_device_error, sizeof(int)) != cudaSuccess) {
    set_cuda_error(cudaGetLastError());
    return -1;
  }
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(otf::g_verify_tree_device_error, &z, sizeof(int));
  }
  return v;
}

extern "C" OTF_API int64_t otf_verify_tree_workspace_bytes(int64_t n, int64_t vocab) {
  if (n <= 0 || vocab <= 0 || n > INT32_MAX || vocab > (1ll << 30)) return -1;
  if (n > 65535 || n * vocab > otf::kTreeAtOnce) return 0;
  return n * ((vocab + otf::kTreeSlice - 1) / otf::kTreeSlice) * (int64_t)sizeof(otf::TreeLeader);
}

extern "C" OTF_API int otf_verify_tree(const float* target, int64_t ld_target, const int64_t* tokens,
                                       const int32_t* parents, const int32_t* starts, int64_t n, const float* noise,
                                       int64_t noise_seq, int64_t ld_noise, const float* temperatures,
                                       double temperature, int64_t* out_tokens, int32_t* path, int32_t* accepted,
                                       int64_t batch, int64_t depth, int64_t vocab, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  if (!target || !tokens || !parents || !out_tokens || (!path && depth) || !accepted) return OTF_ERR_INVALID;
  if (batch <= 0 || depth < 0 || vocab <= 0 || n <= 0 || (!starts && n % batch) || ld_target < vocab) return OTF_ERR_INVALID;
  if (!temperatures && !otf::temperature_ok(temperature)) return OTF_ERR_INVALID;
  if (!noise && (temperatures || temperature > 0.0)) return OTF_ERR_INVALID;
  if (noise && (ld_noise < vocab || noise_seq < 0)) return OTF_ERR_INVALID;
  if (batch > 65535 || depth >= otf::kTreeMaxNodes || vocab > (1ll << 30) || n > INT32_MAX ||
      (!starts && n / batch > otf::kTreeMaxNodes))
    return OTF_ERR_UNSUPPORTED;
  const int64_t bytes = otf_verify_tree_workspace_bytes(n, vocab);
  if (bytes && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < bytes)) return OTF_ERR_INVALID;
  const int st = check_device();
  if (st != OTF_OK) return st;
  otf::TreeArgs a = {target, ld_target, tokens, parents, starts, noise, noise_seq, ld_noise, temperatures, temperature,
                     out_tokens, path, accepted, starts ? 0 : (int)(n / batch), (int)n, (int)depth, (int)vocab,
                     (int)batch, (int)((vocab + otf::kTreeSlice - 1) / otf::kTreeSlice), static_cast<otf::TreeLeader*>(workspace)};
  if (bytes) {
    const cudaError_t e = otf::launch_pdl(otf::k_tree_leaders, dim3((unsigned)a.slices, (unsigned)n), dim3(otf::kTreeThreads), 0,
                                          static_cast<cudaStream_t>(stream), 1u, a);
    if (e != cudaSuccess) return set_cuda_error(e);
    return set_cuda_error(otf::launch_pdl(otf::k_tree_walk, dim3((unsigned)batch), dim3(32), 0, static_cast<cudaStream_t>(stream), 1u, a));
  }
  static std::atomic<bool> done[64];
  int dev;
  bool needs;
  cudaError_t e = otf::needs_opt_in(done, dev, needs);
  if (e != cudaSuccess) return set_cuda_error(e);
  if (needs) {
    e = cudaFuncSetAttribute(otf::k_verify_tree, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return set_cuda_error(e);
    otf::opted_in(done, dev);
  }
  int ctas = otf::kTreeCluster;
  while (ctas > 1 && (batch * ctas > otf::kTreeResident || (int64_t)(ctas / 2) * otf::kTreeThreads * 4 >= vocab)) ctas /= 2;
  return set_cuda_error(otf::launch_pdl(otf::k_verify_tree, dim3((unsigned)(batch * ctas)), dim3(otf::kTreeThreads), 0,
                                        static_cast<cudaStream_t>(stream), (unsigned)ctas, a, ctas));
}
