// Verification of a tree of drafted tokens against the target's logits, and the tree's plan, on sm_100a.
//
// The walk starts at the root (node 0). At a node with logits z the target's distribution is
// p = softmax(cap(z) / temperature), cap(z) = softcap tanh(z / softcap) (the framework's LM head, reference
// utils/model.py:206-208; 0: none), and its children in their order, drawn from the draft's distribution q at that node,
// are judged with r = p, S = 1 at first: child c with token x and random number u_c is accepted if
// u_c S q(x) < r(x); else r = max(r / S - q, 0), S = sum r, and the next child's turn. The walk goes on from an
// accepted child. Where none is, the next token is drawn from r by the race of given exponential numbers E:
// argmax r_v / E_v, the lowest of equals. Accepted and drawn tokens together are distributed as the target's.
// Without q the drafts were picked, not drawn: q is 1 at the child's token. At temperature 0 a child is accepted if
// its token is the largest logit's, and that is the next token (the lowest of equals).
//
// Only the rows that the walk visits are read, once each. A cluster of CTAs takes one sequence, each CTA a slice of the
// vocabulary in shared memory; a node is one pass with a running maximum and sum, a rejection one more over the slice.
// What the children's tests need of their own tokens is read by one warp beside the row, so a test costs no pass. All
// CTAs of a cluster combine the same parts in the same order, so they take the same turns. Sums are in fp32.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "noise_b200.h"

namespace cg = cooperative_groups;

namespace noise {
namespace verify {

constexpr int NT = 1024, WARPS = NT / 32, MAX_NODES = 64, MAX_CTAS = 8, MAX_SLICE = 49152;

struct Params {
  const void* logits;
  int64_t seq_stride, node_stride;
  const float* probs;  // [seqs, nodes, vocab] or NULL
  int64_t probs_seq, probs_node;
  const int64_t* tokens;
  const int* parents;
  const float* u;
  const float* race;  // [seqs, vocab]
  int seqs, nodes, vocab, slice;
  float temperature, softcap;
  int* count;
  int* path;
  int64_t* token;
};

struct Pair {
  float a, b;
};

// (maximum, sum of exp(x - maximum)) of two parts.
__device__ __forceinline__ Pair soft_join(Pair x, Pair y) {
  const float m = fmaxf(x.a, y.a);
  if (m == -INFINITY) return {m, x.b + y.b};  // (NaN sums stay)
  return {m, x.b * expf(x.a - m) + y.b * expf(y.a - m)};
}

// The larger value, the lower index of equals. a: value, b: index as an int's bits.
__device__ __forceinline__ Pair best_join(Pair x, Pair y) {
  const bool other = y.a > x.a || (y.a == x.a && __float_as_int(y.b) < __float_as_int(x.b));
  return other ? y : x;
}

__device__ __forceinline__ Pair sum_join(Pair x, Pair y) { return {x.a + y.a, 0.f}; }

// One value from all threads of the cluster; the parts of the warps and of the CTAs are combined in their order.
template <typename F>
__device__ __forceinline__ Pair reduce(Pair v, F join, Pair* warps, Pair (*ctas)[MAX_CTAS], int& turn) {
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, size = cluster.num_blocks();
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)  // butterfly: lower lanes first, alike in every lane
  {
    const Pair w = {__shfl_xor_sync(0xffffffffu, v.a, o), __shfl_xor_sync(0xffffffffu, v.b, o)};
    v = lane & o ? join(w, v) : join(v, w);
  }
  __syncthreads();  // the last turn's parts were read
  if (lane == 0) warps[warp] = v;
  __syncthreads();
  v = warps[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Pair w = {__shfl_xor_sync(0xffffffffu, v.a, o), __shfl_xor_sync(0xffffffffu, v.b, o)};
    v = lane & o ? join(w, v) : join(v, w);
  }
  if (size == 1) return v;
  if (static_cast<int>(threadIdx.x) < size) cluster.map_shared_rank(&ctas[turn][0], threadIdx.x)[cluster.block_rank()] = v;
  cluster.sync();
  v = ctas[turn][0];
  for (int i = 1; i < size; ++i) v = join(v, ctas[turn][i]);
  turn ^= 1;
  return v;
}

template <typename T>
__device__ __forceinline__ float logit(const Params& p, const T* row, int64_t v, bool greedy) {
  float z = static_cast<float>(row[v]);
  if (p.softcap > 0.f) z = p.softcap * tanhf(z / p.softcap);
  return greedy ? z : z / p.temperature;
}

template <typename T>
__global__ void __launch_bounds__(NT) verify_kernel(const Params p) {
  extern __shared__ float left[];  // the slice of r: exp(z - top) before the first rejection
  __shared__ Pair warps[WARPS];
  __shared__ Pair ctas[2][MAX_CTAS];
  __shared__ int parents[MAX_NODES];
  __shared__ int kids[MAX_NODES];
  __shared__ float kid_logit[MAX_NODES], kid_u[MAX_NODES], kid_q[MAX_NODES];
  __shared__ int64_t kid_token[MAX_NODES];
  __shared__ int kid_count;
  cg::cluster_group cluster = cg::this_cluster();
  const auto everyone = [&] {  // all threads of the cluster
    if (cluster.num_blocks() > 1) cluster.sync();
    else __syncthreads();
  };
  const int rank = cluster.block_rank(), seq = blockIdx.x / cluster.num_blocks(), tid = threadIdx.x;
  const int v0 = rank * p.slice, n = min(p.slice, p.vocab - v0);  // n < 1: an empty slice
  const bool greedy = p.temperature == 0.f;
  const int64_t* tokens = p.tokens + static_cast<int64_t>(seq) * p.nodes;
  if (tid < p.nodes) parents[tid] = p.parents[seq * p.nodes + tid];
  everyone();  // the cluster's other CTAs have started too
  int at = 0, count = 0, turn = 0;
  Pair best = {-INFINITY, 0.f};
  int* path = p.path + seq * p.nodes;
  if (rank == 0 && tid < p.nodes) path[tid] = tid == 0 ? 0 : -1;
  while (true) {
    const T* row = static_cast<const T*>(p.logits) + seq * p.seq_stride + at * p.node_stride;
    const float* probs = p.probs ? p.probs + seq * p.probs_seq + at * p.probs_node : nullptr;
    // the children, in their order, and what their tests read
    if (tid < 32) {
      int found = 0;
#pragma unroll
      for (int i = 0; i < MAX_NODES; i += 32) {
        const int c = i + tid;
        const bool is = c < p.nodes && c > at && parents[c] == at;
        const unsigned all = __ballot_sync(0xffffffffu, is);
        if (is) {
          const int k = found + __popc(all & ((1u << tid) - 1));
          const int64_t x = tokens[c];
          const bool real = x >= 0 && x < p.vocab;  // a token that is none is never accepted
          kids[k] = c;
          kid_token[k] = real ? x : -1;
          kid_u[k] = p.u ? p.u[seq * p.nodes + c] : 0.f;
          kid_q[k] = real && probs ? probs[x] : 1.f;
          kid_logit[k] = real ? logit(p, row, x, greedy) : -INFINITY;
        }
        found += __popc(all);
      }
      if (tid == 0) kid_count = found;
    }
    int next = -1;
    if (greedy) {
      Pair b = {-INFINITY, __int_as_float(p.vocab)};
      for (int i = tid; i < n; i += NT) {
        const Pair x = {logit(p, row, v0 + i, true), __int_as_float(v0 + i)};
        b = best_join(b, x);
      }
      best = reduce(b, best_join, warps, ctas, turn);
      for (int k = 0; k < kid_count && next < 0; ++k)
        if (kid_token[k] == __float_as_int(best.b)) next = kids[k];
    } else {
      Pair mine = {-INFINITY, 0.f};
      for (int i = tid; i < n; i += NT) {
        const float z = logit(p, row, v0 + i, false);
        left[i] = z;
        mine.a = fmaxf(mine.a, z);
      }
      if (mine.a != -INFINITY)
        for (int i = tid; i < n; i += NT) mine.b += expf(left[i] - mine.a);
      const Pair all = reduce(mine, soft_join, warps, ctas, turn);
      const float top = all.a, total = all.b;
      for (int i = tid; i < n; i += NT) left[i] = expf(left[i] - top) / total;
      float mass = 1.f;
      bool first = true;
      for (int k = 0; k < kid_count; ++k) {
        const int64_t x = kid_token[k];
        // r(x): p(x), less q(x) once for each sibling before
        float value = expf(kid_logit[k] - top) / total;
        if (!first) {  // the owner's slice has it
          value = 0.f;
          const int owner = x >= 0 ? static_cast<int>(x / p.slice) : 0;
          if (x >= 0) value = cluster.map_shared_rank(left, owner)[x - static_cast<int64_t>(owner) * p.slice];
        }
        if (x >= 0 && kid_u[k] * mass * kid_q[k] < value) {
          next = kids[k];
          break;
        }
        if (!first) everyone();  // everyone has read the value
        const float div = mass > 0.f ? mass : 1.f;
        Pair s = {0.f, 0.f};
        for (int i = tid; i < n; i += NT) {
          const float q = probs ? probs[v0 + i] : v0 + i == x ? 1.f : 0.f;
          const float r = fmaxf(left[i] / div - q, 0.f);
          left[i] = r;
          s.a += r;
        }
        mass = reduce(s, sum_join, warps, ctas, turn).a;
        first = false;
      }
      if (next < 0) {
        const float* race = p.race + static_cast<int64_t>(seq) * p.vocab;
        Pair b = {-INFINITY, __int_as_float(p.vocab)};
        for (int i = tid; i < n; i += NT) {
          // nothing left of r (the drafts' own distribution): p
          const float r = mass > 0.f ? left[i] : expf(logit(p, row, v0 + i, false) - top) / total;
          const Pair x = {r / race[v0 + i], __int_as_float(v0 + i)};
          b = best_join(b, x);
        }
        best = reduce(b, best_join, warps, ctas, turn);
      }
    }
    everyone();  // the children's list and the slices were read
    if (next < 0) break;
    at = next;
    ++count;
    if (rank == 0 && tid == 0) path[count] = at;
  }
  if (rank == 0 && tid == 0) {
    p.count[seq] = count;
    const int v = __float_as_int(best.b);
    p.token[seq] = v < p.vocab ? v : -1;  // (no logit above -inf)
  }
}

// mask: a node's ancestors and itself; depth: its distance from the root. A parent that is not -1 or an earlier node that is
// itself part of the tree makes a node padding: mask 0, depth -1. One warp a sequence.
__global__ void __launch_bounds__(128) plan_kernel(const int* parents, int seqs, int nodes, int64_t* mask, int* depth) {
  __shared__ int up[4][MAX_NODES];
  __shared__ unsigned long long seen[4][MAX_NODES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, seq = blockIdx.x * 4 + warp;
  if (seq >= seqs) return;
  for (int i = lane; i < nodes; i += 32) {
    const int x = parents[static_cast<int64_t>(seq) * nodes + i];
    up[warp][i] = x >= -1 && x < i ? x : -2;
    seen[warp][i] = 1ull << i;
  }
  __syncwarp();
  for (int step = 1; step < MAX_NODES; step <<= 1) {  // pointer doubling: 2^k ancestors after k steps
    int to[2];
    unsigned long long m[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = lane + 32 * j;
      if (i >= nodes) continue;
      const int x = up[warp][i];
      m[j] = seen[warp][i] | (x >= 0 ? seen[warp][x] : 0ull);
      to[j] = x >= 0 ? up[warp][x] : x;
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = lane + 32 * j;
      if (i >= nodes) continue;
      seen[warp][i] = m[j];
      up[warp][i] = to[j];
    }
    __syncwarp();
  }
  for (int i = lane; i < nodes; i += 32) {
    const bool real = up[warp][i] == -1;
    const unsigned long long m = seen[warp][i];
    mask[static_cast<int64_t>(seq) * nodes + i] = real ? static_cast<int64_t>(m) : 0;
    depth[static_cast<int64_t>(seq) * nodes + i] = real ? __popcll(m) - 1 : -1;
  }
}

template <typename T>
int run(const Params& p, int ctas, cudaStream_t s) {
  const auto kernel = verify_kernel<T>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SLICE * 4) != cudaSuccess)
    return NOISE_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.seqs * ctas);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = p.temperature == 0.f ? 0 : p.slice * 4;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? NOISE_OK : NOISE_ERR_CUDA;
}

}  // namespace verify
}  // namespace noise

extern "C" {

int noise_tree_plan(const int* parents, int seqs, int nodes, int64_t* mask, int* depth, void* stream) {
  if (seqs < 0 || nodes < 1 || nodes > noise::verify::MAX_NODES) return NOISE_ERR_SHAPE;
  if (seqs == 0) return NOISE_OK;
  if (!parents || !mask || !depth) return NOISE_ERR_ARGUMENT;
  noise::verify::plan_kernel<<<(seqs + 3) / 4, 128, 0, static_cast<cudaStream_t>(stream)>>>(parents, seqs, nodes, mask,
                                                                                            depth);
  return cudaGetLastError() == cudaSuccess ? NOISE_OK : NOISE_ERR_CUDA;
}

int noise_verify_tree(const void* logits, int logits_dtype, int64_t seq_stride, int64_t node_stride,
                      const int64_t* tokens, const int* parents, const float* u, const float* race,
                      const float* probs, int64_t probs_seq_stride, int64_t probs_node_stride, int seqs, int nodes,
                      int vocab, float temperature, float softcap, int* count, int* path, int64_t* token,
                      void* stream) {
  using namespace noise::verify;
  if (logits_dtype != NOISE_DTYPE_F32 && logits_dtype != NOISE_DTYPE_BF16) return NOISE_ERR_ARGUMENT;
  if (seqs < 0 || seqs > (1 << 24) || nodes < 1 || nodes > MAX_NODES || vocab < 1 || vocab > MAX_CTAS * MAX_SLICE)
    return NOISE_ERR_SHAPE;
  if (!(temperature >= 0.f) || !(temperature < INFINITY) || !(softcap >= 0.f) || !(softcap < INFINITY))
    return NOISE_ERR_ARGUMENT;
  if (seqs == 0) return NOISE_OK;
  if (!logits || !tokens || !parents || !count || !path || !token || (temperature > 0.f && (!u || !race)))
    return NOISE_ERR_ARGUMENT;
  // a cluster of the fewest CTAs with at most 8 values a thread, 8 CTAs at most
  int ctas = 1;
  while (ctas < MAX_CTAS && (vocab + ctas - 1) / ctas > 8 * NT) ctas *= 2;
  Params p = {logits, seq_stride, node_stride, probs, probs_seq_stride, probs_node_stride, tokens, parents, u, race,
              seqs, nodes, vocab, (vocab + ctas - 1) / ctas, temperature, softcap, count, path, token};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return logits_dtype == NOISE_DTYPE_F32 ? run<float>(p, ctas, s) : run<__nv_bfloat16>(p, ctas, s);
}

}  // extern "C"
