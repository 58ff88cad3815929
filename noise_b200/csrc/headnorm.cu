// Per-head RMS norm of queries and keys with the position rotation in the same pass, and its gradient, on sm_100a
// (reference utils/model.py:46-47 norm, :55-58 apply_rotary_emb, :93-94 their use, as an operator of its own).
//
// A row x of D values (one token's head) has r = rsqrt(mean x^2 + eps), xh = r x, a = w xh (w: the learned weight of the
// D dimensions, shared by the heads; none: 1), and with the cos c and sin s of the token's position over the halves
// y1 = a1 c + a2 s, y2 = a2 c - a1 s. The rotation keeps a row's norm, so without w this is norm(rope(x)) too.
// Backward: g = the rotation back of dy, h = w g, dx = r (h - xh mean(h xh)), dw = sum over rows of g xh.
//
// Both directions read and write each value once and do some ten operations on it: memory-bound. A lane holds the
// same VEC places of both halves, so the rotation needs no exchange and the row's sum is a few shuffles; a warp takes
// one token's heads, so cos and sin are read once for all of them. Sums are held in 32 bits.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "noise_b200.h"

namespace noise {
namespace headnorm {

constexpr int WARPS = 8;

struct Rows {  // [tokens, heads, D], the last dimension contiguous
  const void* x;
  const void* dy;
  int64_t token, head, dy_token, dy_head;
  int heads;
  const void* weight;
  void* out;  // contiguous
};

struct Args {
  Rows q, k;
  const void* cos;
  const void* sin;
  int table_rows;
  const int* positions;
  int tokens, dim;
  float eps;
  int q_chunks, k_chunks;  // warps' shares of a token's heads
  int q_blocks;            // blocks of the gradient that take queries
  float* partial;          // [blocks, D] weight gradients
};

template <int N, typename T>
__device__ __forceinline__ void load(const T* p, float (&v)[N]) {
  constexpr int BYTES = N * sizeof(T);
  if constexpr (BYTES % 4 == 0) {
    uint32_t w[BYTES / 4];
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(w)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else if constexpr (BYTES == 8) {
      *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<float>(p[i]);
  }
}

template <int N, typename T>
__device__ __forceinline__ void store(T* p, const float (&v)[N]) {
  if constexpr (sizeof(T) == 4 && N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
      reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else if constexpr (sizeof(T) == 2 && N == 8) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = static_cast<T>(v[i]);
  }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// T: the rows' type; TT: the tables'; a row is LPR lanes with VEC values of each half ITER times. U rows a lane are
// loaded before the first is used.
template <typename T, typename TT, int VEC, int LPR, int ITER, int U>
__global__ void __launch_bounds__(32 * WARPS) forward_kernel(const Args a) {
  const int lane = threadIdx.x & 31, sub = lane % LPR, grp = lane / LPR;
  const int half = a.dim / 2, chunks = a.q_chunks + a.k_chunks;
  const int64_t item = blockIdx.x * static_cast<int64_t>(WARPS) + (threadIdx.x >> 5);
  const int token = static_cast<int>(item / chunks);
  if (token >= a.tokens) return;
  const int chunk = static_cast<int>(item - static_cast<int64_t>(token) * chunks);
  const bool is_k = chunk >= a.q_chunks;
  const Rows& r = is_k ? a.k : a.q;
  const int h0 = (is_k ? chunk - a.q_chunks : chunk) * (32 / LPR) * U + grp;
  const T* src = static_cast<const T*>(r.x) + token * r.token;
  float x[U][ITER][2][VEC];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u * (32 / LPR);
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int i = (it * LPR + sub) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[u][it][0][e] = x[u][it][1][e] = 0.f;
      if (h < r.heads && i < half) {
        load<VEC>(src + h * r.head + i, x[u][it][0]);
        load<VEC>(src + h * r.head + half + i, x[u][it][1]);
      }
    }
  }
  const int pos = a.positions[token];
  const bool known = pos >= 0 && pos < a.table_rows;  // a position without a table row gives NaN
  float c[ITER][VEC], s[ITER][VEC];
#pragma unroll
  for (int it = 0; it < ITER; ++it) {
    const int i = (it * LPR + sub) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) c[it][e] = s[it][e] = __int_as_float(0x7fc00000);
    if (known && i < half) {
      load<VEC>(static_cast<const TT*>(a.cos) + static_cast<int64_t>(pos) * half + i, c[it]);
      load<VEC>(static_cast<const TT*>(a.sin) + static_cast<int64_t>(pos) * half + i, s[it]);
    }
  }
  float w[ITER][2][VEC];
#pragma unroll
  for (int it = 0; it < ITER; ++it) {
    const int i = (it * LPR + sub) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) w[it][0][e] = w[it][1][e] = 1.f;
    if (r.weight && i < half) {
      load<VEC>(static_cast<const T*>(r.weight) + i, w[it][0]);
      load<VEC>(static_cast<const T*>(r.weight) + half + i, w[it][1]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float sq = 0.f;
#pragma unroll
    for (int it = 0; it < ITER; ++it)
#pragma unroll
      for (int e = 0; e < VEC; ++e) sq += x[u][it][0][e] * x[u][it][0][e] + x[u][it][1][e] * x[u][it][1][e];
    const float rr = rsqrtf(row_sum<LPR>(sq) / a.dim + a.eps);
    const int h = h0 + u * (32 / LPR);
    if (h >= r.heads) continue;
    T* dst = static_cast<T*>(r.out) + (static_cast<int64_t>(token) * r.heads + h) * a.dim;
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int i = (it * LPR + sub) * VEC;
      float y1[VEC], y2[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float a1 = x[u][it][0][e] * rr * w[it][0][e], a2 = x[u][it][1][e] * rr * w[it][1][e];
        y1[e] = a1 * c[it][e] + a2 * s[it][e];
        y2[e] = a2 * c[it][e] - a1 * s[it][e];
      }
      if (i < half) {
        store<VEC>(dst + i, y1);
        store<VEC>(dst + half + i, y2);
      }
    }
  }
}

// Blocks [0, q_blocks) take the queries, the others the keys, so a lane sums one weight's gradient over all its rows;
// a block's sums go to partial[block] (no atomics: the order is the same from call to call).
template <typename T, typename TT, int VEC, int LPR, int ITER>
__global__ void __launch_bounds__(32 * WARPS) backward_kernel(const Args a) {
  __shared__ float sums[WARPS][2 * LPR * VEC * ITER];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LPR, grp = lane / LPR;
  const int half = a.dim / 2;
  const bool is_k = blockIdx.x >= a.q_blocks;
  const Rows& r = is_k ? a.k : a.q;
  const int chunks = is_k ? a.k_chunks : a.q_chunks;
  const int block = is_k ? blockIdx.x - a.q_blocks : blockIdx.x;
  const int blocks = is_k ? gridDim.x - a.q_blocks : a.q_blocks;
  float w[ITER][2][VEC], dw[ITER][2][VEC];
#pragma unroll
  for (int it = 0; it < ITER; ++it) {
    const int i = (it * LPR + sub) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[it][0][e] = w[it][1][e] = 1.f;
      dw[it][0][e] = dw[it][1][e] = 0.f;
    }
    if (r.weight && i < half) {
      load<VEC>(static_cast<const T*>(r.weight) + i, w[it][0]);
      load<VEC>(static_cast<const T*>(r.weight) + half + i, w[it][1]);
    }
  }
  const int64_t items = static_cast<int64_t>(a.tokens) * chunks;
  for (int64_t item = block * static_cast<int64_t>(WARPS) + warp; item < items;
       item += static_cast<int64_t>(blocks) * WARPS) {
    const int token = static_cast<int>(item / chunks);
    const int h = static_cast<int>(item - static_cast<int64_t>(token) * chunks) * (32 / LPR) + grp;
    const bool here = h < r.heads;
    const T* src = static_cast<const T*>(r.x) + token * r.token + h * r.head;
    const T* dsrc = static_cast<const T*>(r.dy) + token * r.dy_token + h * r.dy_head;
    float x[ITER][2][VEC], g[ITER][2][VEC], c[ITER][VEC], s[ITER][VEC];
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int i = (it * LPR + sub) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[it][0][e] = x[it][1][e] = g[it][0][e] = g[it][1][e] = 0.f;
      if (here && i < half) {
        load<VEC>(src + i, x[it][0]);
        load<VEC>(src + half + i, x[it][1]);
        load<VEC>(dsrc + i, g[it][0]);
        load<VEC>(dsrc + half + i, g[it][1]);
      }
    }
    const int pos = a.positions[token];
    const bool known = pos >= 0 && pos < a.table_rows;
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int i = (it * LPR + sub) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) c[it][e] = s[it][e] = i < half ? __int_as_float(0x7fc00000) : 0.f;
      if (known && i < half) {
        load<VEC>(static_cast<const TT*>(a.cos) + static_cast<int64_t>(pos) * half + i, c[it]);
        load<VEC>(static_cast<const TT*>(a.sin) + static_cast<int64_t>(pos) * half + i, s[it]);
      }
    }
    float sq = 0.f, dot = 0.f;  // dot: sum h x
#pragma unroll
    for (int it = 0; it < ITER; ++it)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d1 = g[it][0][e], d2 = g[it][1][e];
        g[it][0][e] = d1 * c[it][e] - d2 * s[it][e];
        g[it][1][e] = d1 * s[it][e] + d2 * c[it][e];
        sq += x[it][0][e] * x[it][0][e] + x[it][1][e] * x[it][1][e];
        dot += g[it][0][e] * w[it][0][e] * x[it][0][e] + g[it][1][e] * w[it][1][e] * x[it][1][e];
      }
    const float rr = rsqrtf(row_sum<LPR>(sq) / a.dim + a.eps);
    const float m = row_sum<LPR>(dot) * rr / a.dim;  // mean(h xh)
    T* dst = static_cast<T*>(r.out) + (static_cast<int64_t>(token) * r.heads + h) * a.dim;
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int i = (it * LPR + sub) * VEC;
      float o[2][VEC];
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float xh = x[it][p][e] * rr;
          o[p][e] = rr * (g[it][p][e] * w[it][p][e] - xh * m);
          if (here) dw[it][p][e] += g[it][p][e] * xh;
        }
      if (here && i < half) {
        store<VEC>(dst + i, o[0]);
        store<VEC>(dst + half + i, o[1]);
      }
    }
  }
  if (!a.partial) return;
#pragma unroll
  for (int it = 0; it < ITER; ++it)
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float v = dw[it][p][e];
#pragma unroll
        for (int o = 16; o >= LPR; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        const int i = (it * LPR + sub) * VEC + e;
        if (grp == 0 && i < half) sums[warp][p * half + i] = v;
      }
  __syncthreads();
  for (int i = threadIdx.x; i < a.dim; i += 32 * WARPS) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) v += sums[k][i];
    a.partial[static_cast<int64_t>(blockIdx.x) * a.dim + i] = v;
  }
}

// dw[i] = sum over blocks of partial[block][i]: 32 columns a block, 32 rows at a time. blockIdx.y: queries, keys.
__global__ void __launch_bounds__(1024) weight_kernel(const float* partial, int q_blocks, int blocks, int dim,
                                                      float* q_out, float* k_out) {
  __shared__ float sums[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), row = threadIdx.x >> 5;
  const int first = blockIdx.y ? q_blocks : 0, last = blockIdx.y ? blocks : q_blocks;
  float* out = blockIdx.y ? k_out : q_out;
  cudaGridDependencySynchronize();
  if (!out) return;
  float v = 0.f;
  if (col < dim)
    for (int b = first + row; b < last; b += 32) v += partial[static_cast<int64_t>(b) * dim + col];
  sums[row][threadIdx.x & 31] = v;
  __syncthreads();
  if (row == 0 && col < dim) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += sums[k][threadIdx.x];
    out[col] = t;
  }
}

constexpr int GRAD_BLOCKS = 148 * 3;  // three blocks of 8 warps fit an SM: one wave

inline int lanes_of(int half, int vec) {
  int l = 1;
  while (l * vec < half) l *= 2;
  return l;
}

template <typename T, typename TT, int VEC, int LPR, int ITER>
cudaError_t run(Args a, bool backward, float* q_dw, float* k_dw, cudaStream_t s) {
  constexpr int U = ITER > 1 || LPR == 32 ? 1 : 2;
  if (!backward) {
    constexpr int HEADS = 32 / LPR * U;
    a.q_chunks = (a.q.heads + HEADS - 1) / HEADS;
    a.k_chunks = (a.k.heads + HEADS - 1) / HEADS;
    const int64_t items = static_cast<int64_t>(a.tokens) * (a.q_chunks + a.k_chunks);
    forward_kernel<T, TT, VEC, LPR, ITER, U>
        <<<static_cast<unsigned>((items + WARPS - 1) / WARPS), 32 * WARPS, 0, s>>>(a);
    return cudaGetLastError();
  }
  constexpr int HEADS = 32 / LPR;
  a.q_chunks = (a.q.heads + HEADS - 1) / HEADS;
  a.k_chunks = (a.k.heads + HEADS - 1) / HEADS;
  const int64_t q_need = (static_cast<int64_t>(a.tokens) * a.q_chunks + WARPS - 1) / WARPS;
  const int64_t k_need = (static_cast<int64_t>(a.tokens) * a.k_chunks + WARPS - 1) / WARPS;
  int64_t q_most = static_cast<int64_t>(GRAD_BLOCKS) * a.q_chunks / (a.q_chunks + a.k_chunks);
  if (q_most < 1) q_most = 1;
  const int64_t k_most = GRAD_BLOCKS - q_most > 1 ? GRAD_BLOCKS - q_most : 1;
  a.q_blocks = static_cast<int>(q_need < q_most ? q_need : q_most);
  const int blocks = a.q_blocks + static_cast<int>(k_need < k_most ? k_need : k_most);
  if (!q_dw && !k_dw) a.partial = nullptr;
  backward_kernel<T, TT, VEC, LPR, ITER><<<blocks, 32 * WARPS, 0, s>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !a.partial) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((a.dim + 31) / 32, 2);
  cfg.blockDim = dim3(1024);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, weight_kernel, static_cast<const float*>(a.partial), a.q_blocks, blocks, a.dim,
                            q_dw, k_dw);
}

template <typename T, typename TT>
cudaError_t by_lanes(const Args& a, bool wide, bool backward, float* q_dw, float* k_dw, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  if (!wide) return run<T, TT, 1, 32, 4>(a, backward, q_dw, k_dw, s);  // any address: one value at a time
  switch (lanes_of(a.dim / 2, VEC)) {
    case 1: return run<T, TT, VEC, 1, 1>(a, backward, q_dw, k_dw, s);
    case 2: return run<T, TT, VEC, 2, 1>(a, backward, q_dw, k_dw, s);
    case 4: return run<T, TT, VEC, 4, 1>(a, backward, q_dw, k_dw, s);
    case 8: return run<T, TT, VEC, 8, 1>(a, backward, q_dw, k_dw, s);
    case 16: return run<T, TT, VEC, 16, 1>(a, backward, q_dw, k_dw, s);
    default: return run<T, TT, VEC, 32, 1>(a, backward, q_dw, k_dw, s);
  }
}

template <typename T>
bool wide_rows(const Rows& r, int dim) {
  const auto ok = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const int64_t v = 16 / sizeof(T);
  return ok(r.x) && ok(r.dy) && ok(r.weight) && ok(r.out) && r.token % v == 0 && r.head % v == 0 &&
         r.dy_token % v == 0 && r.dy_head % v == 0 && (dim / 2) % v == 0;
}

int launch(const noise_heads_t* q, const noise_heads_t* k, const noise_heads_t* dq, const noise_heads_t* dk,
           const void* cos, const void* sin, int table_dtype, int table_rows, const int* positions, int tokens, int dim,
           int dtype, const void* q_weight, const void* k_weight, float eps, void* q_out, void* k_out, float* q_dw,
           float* k_dw, float* partial, bool backward, void* stream) {
  if (!q || !k || (backward && (!dq || !dk))) return NOISE_ERR_ARGUMENT;
  if ((dtype != NOISE_DTYPE_F32 && dtype != NOISE_DTYPE_BF16) ||
      (table_dtype != NOISE_DTYPE_F32 && table_dtype != NOISE_DTYPE_BF16))
    return NOISE_ERR_ARGUMENT;
  if (tokens < 0 || dim < 2 || dim > 256 || dim % 2 || table_rows < 1 || q->heads < 1 || k->heads < 1 ||
      q->heads > 4096 || k->heads > 4096)
    return NOISE_ERR_SHAPE;
  if (!(eps >= 0.f)) return NOISE_ERR_ARGUMENT;
  if (tokens == 0) return NOISE_OK;
  if (!q->data || !k->data || !cos || !sin || !positions || !q_out || !k_out) return NOISE_ERR_ARGUMENT;
  if (backward && (!dq->data || !dk->data || dq->heads != q->heads || dk->heads != k->heads))
    return NOISE_ERR_ARGUMENT;
  Args a = {};
  a.q = {q->data, backward ? dq->data : nullptr, q->token_stride, q->head_stride, backward ? dq->token_stride : 0,
         backward ? dq->head_stride : 0, q->heads, q_weight, q_out};
  a.k = {k->data, backward ? dk->data : nullptr, k->token_stride, k->head_stride, backward ? dk->token_stride : 0,
         backward ? dk->head_stride : 0, k->heads, k_weight, k_out};
  a.cos = cos;
  a.sin = sin;
  a.table_rows = table_rows;
  a.positions = positions;
  a.tokens = tokens;
  a.dim = dim;
  a.eps = eps;
  a.partial = partial;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool tables = reinterpret_cast<uintptr_t>(cos) % 16 == 0 && reinterpret_cast<uintptr_t>(sin) % 16 == 0;
  cudaError_t e;
  if (dtype == NOISE_DTYPE_F32) {
    const bool wide = tables && wide_rows<float>(a.q, dim) && wide_rows<float>(a.k, dim);
    e = table_dtype == NOISE_DTYPE_F32 ? by_lanes<float, float>(a, wide, backward, q_dw, k_dw, s)
                                       : by_lanes<float, __nv_bfloat16>(a, wide, backward, q_dw, k_dw, s);
  } else {
    const bool wide = tables && wide_rows<__nv_bfloat16>(a.q, dim) && wide_rows<__nv_bfloat16>(a.k, dim);
    e = table_dtype == NOISE_DTYPE_F32 ? by_lanes<__nv_bfloat16, float>(a, wide, backward, q_dw, k_dw, s)
                                       : by_lanes<__nv_bfloat16, __nv_bfloat16>(a, wide, backward, q_dw, k_dw, s);
  }
  return e == cudaSuccess ? NOISE_OK : NOISE_ERR_CUDA;
}

}  // namespace headnorm
}  // namespace noise

extern "C" {

int noise_head_norm_rope(const noise_heads_t* q, const noise_heads_t* k, const void* cos, const void* sin,
                         int table_dtype, int table_rows, const int* positions, int tokens, int dim, int dtype,
                         const void* q_weight, const void* k_weight, float eps, void* q_out, void* k_out,
                         void* stream) {
  return noise::headnorm::launch(q, k, nullptr, nullptr, cos, sin, table_dtype, table_rows, positions, tokens, dim,
                                 dtype, q_weight, k_weight, eps, q_out, k_out, nullptr, nullptr, nullptr, false,
                                 stream);
}

size_t noise_head_norm_rope_backward_workspace_bytes(int dim) {
  return dim < 2 || dim > 256 ? 0 : static_cast<size_t>(noise::headnorm::GRAD_BLOCKS) * dim * sizeof(float);
}

int noise_head_norm_rope_backward(const noise_heads_t* dq, const noise_heads_t* dk, const noise_heads_t* q,
                                  const noise_heads_t* k, const void* cos, const void* sin, int table_dtype,
                                  int table_rows, const int* positions, int tokens, int dim, int dtype,
                                  const void* q_weight, const void* k_weight, float eps, void* dq_in, void* dk_in,
                                  float* dq_weight, float* dk_weight, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if ((dq_weight || dk_weight) &&
      (!workspace || workspace_bytes < noise_head_norm_rope_backward_workspace_bytes(dim)))
    return NOISE_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return NOISE_ERR_ALIGN;
  if (tokens == 0) {  // no rows: zero weight gradients
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    for (float* w : {dq_weight, dk_weight})
      if (w && dim > 0 && dim <= 256 && cudaMemsetAsync(w, 0, dim * sizeof(float), s) != cudaSuccess)
        return NOISE_ERR_CUDA;
  }
  return noise::headnorm::launch(q, k, dq, dk, cos, sin, table_dtype, table_rows, positions, tokens, dim, dtype,
                                 q_weight, k_weight, eps, dq_in, dk_in, dq_weight, dk_weight,
                                 static_cast<float*>(workspace), true, stream);
}

}  // extern "C"
