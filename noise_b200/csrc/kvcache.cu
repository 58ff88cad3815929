// Writing tokens' keys and values into the paged cache, quantised on the way, and reading them back, on sm_100a.
//
// Token i of a call goes to position pos[i] of sequence seq[i]: page table[seq, pos / page_size], slot
// pos % page_size. Quantising a row x of D values: 2^e the least power of two with max|x| <= 2^e * 448 (e4m3) or 127
// (int8), code = round(x / 2^e), ties to even. Each value is read once, its code written once: memory-bound. A lane
// takes 8 values, the row's maximum is a few shuffles; a group of lanes does K and V of its (token, head), both loaded
// before either is used.
#include <cuda_runtime.h>

#include "kv.cuh"
#include "ptx.cuh"

namespace noise {
namespace kv {

constexpr int NT = 256;

struct Io {
  noise_kv_cache_t c;
  const void* k;  // write: the rows; read: unused
  const void* v;
  int64_t k_layer, k_token, k_head, v_layer, v_token, v_head;
  void* k_out;  // read: [layers, tokens, heads, D]
  void* v_out;
  int layer0, layers, tokens, source_rows;
  const int* seq;
  const int* pos;
  const int* rows;
  const int* table;
  int seqs, width, page_shift;
};

// The page and slot of token i: 0 found, 1 to be skipped (a negative sequence, position or row), 2 out of range.
__device__ __forceinline__ int place(const Io& a, int i, int& row, int64_t& page, int& slot) {
  row = a.rows ? a.rows[i] : i;
  const int s = a.seq[i], p = a.pos[i];
  if (s < 0 || p < 0 || row < 0) return 1;
  const int at = p >> a.page_shift;
  slot = p & (a.c.page_size - 1);
  if (s >= a.seqs || at >= a.width || row >= a.source_rows) return 2;
  page = a.table[static_cast<int64_t>(s) * a.width + at];
  return page >= 0 && page < a.c.pages ? 0 : 2;
}

template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (!WIDE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(p[i]);
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The codes of the 8 values and the row's scale byte; LPR lanes hold the row.
template <int KIND, int LPR>
__device__ __forceinline__ uint32_t quantise(const float (&x)[8], uint32_t (&code)[2]) {
  uint32_t top = 0;  // of the bits of |x|: orders NaN above infinity above the finite
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (top >= 0x7f800000u) {
    code[0] = code[1] = 0;
    return 255;
  }
  const uint32_t b = scale_byte<KIND>(top);
  const float m = power(254 - static_cast<int>(b));
  code[0] = encode4<KIND>(x[0] * m, x[1] * m, x[2] * m, x[3] * m);
  code[1] = encode4<KIND>(x[4] * m, x[5] * m, x[6] * m, x[7] * m);
  return b;
}

template <typename T, int KIND, int LPR, bool WIDE>
__global__ void __launch_bounds__(NT) write_kernel(const Io a) {
  const int sub = threadIdx.x % LPR, d = sub * 8;
  const int64_t group = blockIdx.x * static_cast<int64_t>(NT / LPR) + threadIdx.x / LPR;
  const int token = static_cast<int>(group / a.c.heads);
  const int h = static_cast<int>(group - static_cast<int64_t>(token) * a.c.heads);
  const int layer = blockIdx.y;
  int row = 0, slot = 0, found = 1;
  int64_t page = 0;
  if (token < a.tokens) found = place(a, token, row, page, slot);
  if (found == 2 && sub == 0) record_error(a.c.status, NOISE_DEV_BAD_INDEX);
  const bool active = found == 0 && d < a.c.dim;
  float k[8], v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) k[i] = v[i] = 0.f;
  if (active) {
    load8<T, WIDE>(static_cast<const T*>(a.k) + layer * a.k_layer + row * a.k_token + h * a.k_head + d, k);
    load8<T, WIDE>(static_cast<const T*>(a.v) + layer * a.v_layer + row * a.v_token + h * a.v_head + d, v);
  }
  const int64_t cell = ((static_cast<int64_t>(a.layer0 + layer) * a.c.pages + page) * a.c.heads + h) * a.c.page_size;
  const int64_t k_at = (cell + slot) * a.c.dim + d;
  const int64_t v_at = ((cell >> 2) + (slot >> 2)) * a.c.dim * 4 + d * 4 + (slot & 3);
  if constexpr (KIND == NOISE_KV_BF16) {
    if (!active) return;
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.c.k) + k_at) =
        make_uint4(pack2(k[0], k[1]), pack2(k[2], k[3]), pack2(k[4], k[5]), pack2(k[6], k[7]));
    __nv_bfloat16* to = static_cast<__nv_bfloat16*>(a.c.v) + v_at;
#pragma unroll
    for (int i = 0; i < 8; ++i) to[4 * i] = __float2bfloat16_rn(v[i]);
  } else {
    uint32_t kc[2], vc[2];
    const uint32_t kb = quantise<KIND, LPR>(k, kc), vb = quantise<KIND, LPR>(v, vc);
    if (!active) return;
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.c.k) + k_at) = make_uint2(kc[0], kc[1]);
    uint8_t* to = static_cast<uint8_t*>(a.c.v) + v_at;
#pragma unroll
    for (int i = 0; i < 8; ++i) to[4 * i] = static_cast<uint8_t>(vc[i >> 2] >> (8 * (i & 3)));
    if (sub == 0) {
      a.c.k_scale[cell + slot] = static_cast<uint8_t>(kb);
      a.c.v_scale[cell + slot] = static_cast<uint8_t>(vb);
    }
  }
}

template <int KIND>
__device__ __forceinline__ void scaled8(uint32_t lo, uint32_t hi, uint32_t b, float (&x)[8]) {
  uint32_t h[4];
  decode4<KIND>(lo, h[0], h[1]);
  decode4<KIND>(hi, h[2], h[3]);
  const float m = b == 255 ? __int_as_float(0x7fc00000) : b ? power(b) : 5.877471754111438e-39f;  // 2^-127
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    x[2 * i] = f.x * m;
    x[2 * i + 1] = f.y * m;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]),
                                              pack2(x[6], x[7]));
  }
}

template <typename T, int KIND, int LPR>
__global__ void __launch_bounds__(NT) read_kernel(const Io a) {
  const int sub = threadIdx.x % LPR, d = sub * 8;
  const int64_t group = blockIdx.x * static_cast<int64_t>(NT / LPR) + threadIdx.x / LPR;
  const int token = static_cast<int>(group / a.c.heads);
  if (token >= a.tokens || d >= a.c.dim) return;
  const int h = static_cast<int>(group - static_cast<int64_t>(token) * a.c.heads);
  const int layer = blockIdx.y;
  int row, slot = 0;
  int64_t page = 0;
  const int found = place(a, token, row, page, slot);
  if (found == 2 && sub == 0) record_error(a.c.status, NOISE_DEV_BAD_INDEX);
  float k[8], v[8];
  if (found == 0) {
    const int64_t cell =
        ((static_cast<int64_t>(a.layer0 + layer) * a.c.pages + page) * a.c.heads + h) * a.c.page_size;
    const int64_t k_at = (cell + slot) * a.c.dim + d;
    const int64_t v_at = ((cell >> 2) + (slot >> 2)) * a.c.dim * 4 + d * 4 + (slot & 3);
    if constexpr (KIND == NOISE_KV_BF16) {
      load8<__nv_bfloat16, true>(static_cast<const __nv_bfloat16*>(a.c.k) + k_at, k);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __bfloat162float(static_cast<const __nv_bfloat16*>(a.c.v)[v_at + 4 * i]);
    } else {
      const uint2 kc = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.c.k) + k_at);
      uint32_t vc[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        vc[i >> 2] |= static_cast<uint32_t>(static_cast<const uint8_t*>(a.c.v)[v_at + 4 * i]) << (8 * (i & 3));
      scaled8<KIND>(kc.x, kc.y, a.c.k_scale[cell + slot], k);
      scaled8<KIND>(vc[0], vc[1], a.c.v_scale[cell + slot], v);
    }
  } else {  // skipped: zeros; out of range: NaN
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = v[i] = found == 1 ? 0.f : __int_as_float(0x7fc00000);
  }
  const int64_t to = ((static_cast<int64_t>(layer) * a.tokens + token) * a.c.heads + h) * a.c.dim + d;
  store8(static_cast<T*>(a.k_out) + to, k);
  store8(static_cast<T*>(a.v_out) + to, v);
}

template <typename T, int KIND, int LPR>
cudaError_t run(const Io& a, bool write, bool wide, cudaStream_t s) {
  const int64_t groups = static_cast<int64_t>(a.tokens) * a.c.heads;
  const dim3 grid(static_cast<unsigned>((groups + NT / LPR - 1) / (NT / LPR)), a.layers);
  if (!write)
    read_kernel<T, KIND, LPR><<<grid, NT, 0, s>>>(a);
  else if (wide)
    write_kernel<T, KIND, LPR, true><<<grid, NT, 0, s>>>(a);
  else
    write_kernel<T, KIND, LPR, false><<<grid, NT, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T, int KIND>
cudaError_t by_lanes(const Io& a, bool write, bool wide, cudaStream_t s) {
  if (a.c.dim <= 16) return run<T, KIND, 2>(a, write, wide, s);
  if (a.c.dim <= 32) return run<T, KIND, 4>(a, write, wide, s);
  if (a.c.dim <= 64) return run<T, KIND, 8>(a, write, wide, s);
  if (a.c.dim <= 128) return run<T, KIND, 16>(a, write, wide, s);
  return run<T, KIND, 32>(a, write, wide, s);
}

template <typename T>
cudaError_t by_kind(const Io& a, bool write, bool wide, cudaStream_t s) {
  if (a.c.kind == NOISE_KV_E4M3) return by_lanes<T, NOISE_KV_E4M3>(a, write, wide, s);
  if (a.c.kind == NOISE_KV_INT8) return by_lanes<T, NOISE_KV_INT8>(a, write, wide, s);
  return by_lanes<T, NOISE_KV_BF16>(a, write, wide, s);
}

int check_cache(const noise_kv_cache_t* c) {
  if (!c || !c->k || !c->v || !c->status) return NOISE_ERR_ARGUMENT;
  if (c->kind != NOISE_KV_BF16 && c->kind != NOISE_KV_E4M3 && c->kind != NOISE_KV_INT8) return NOISE_ERR_ARGUMENT;
  if (c->kind != NOISE_KV_BF16 && (!c->k_scale || !c->v_scale)) return NOISE_ERR_ARGUMENT;
  if (c->layers < 1 || c->pages < 1 || c->heads < 1 || c->heads > 4096 || c->dim < 16 || c->dim > 256 ||
      c->dim % 16 || c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)))
    return NOISE_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(c->k) % 16 || reinterpret_cast<uintptr_t>(c->v) % 16 ||
      reinterpret_cast<uintptr_t>(c->k_scale) % 16 || reinterpret_cast<uintptr_t>(c->v_scale) % 16)
    return NOISE_ERR_ALIGN;
  return NOISE_OK;
}

int launch(Io& a, int dtype, bool write, void* stream) {
  if (dtype != NOISE_DTYPE_F32 && dtype != NOISE_DTYPE_BF16) return NOISE_ERR_ARGUMENT;
  if (a.tokens < 0 || a.seqs < 0 || a.width < 0 || a.source_rows < 0 || a.layers < 1 || a.layers > 65535 ||
      a.layer0 < 0 || a.layer0 > a.c.layers - a.layers)
    return NOISE_ERR_SHAPE;
  if (static_cast<int64_t>(a.tokens) * a.c.heads > (static_cast<int64_t>(1) << 33)) return NOISE_ERR_SHAPE;
  if (a.tokens == 0) return NOISE_OK;
  if (!a.seq || !a.pos || (a.seqs > 0 && a.width > 0 && !a.table)) return NOISE_ERR_ARGUMENT;
  a.page_shift = __builtin_ctz(static_cast<unsigned>(a.c.page_size));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int v = dtype == NOISE_DTYPE_F32 ? 4 : 8;
  bool wide = reinterpret_cast<uintptr_t>(a.k) % 16 == 0 && reinterpret_cast<uintptr_t>(a.v) % 16 == 0;
  for (int64_t stride : {a.k_layer, a.k_token, a.k_head, a.v_layer, a.v_token, a.v_head})
    wide = wide && stride % v == 0;
  const cudaError_t e = dtype == NOISE_DTYPE_F32 ? by_kind<float>(a, write, wide, s)
                                                 : by_kind<__nv_bfloat16>(a, write, wide, s);
  return e == cudaSuccess ? NOISE_OK : NOISE_ERR_CUDA;
}

}  // namespace kv
}  // namespace noise

extern "C" {

int noise_kv_write(const noise_kv_cache_t* cache, int layer, int layers, const void* k, int64_t k_layer_stride,
                   int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_layer_stride,
                   int64_t v_token_stride, int64_t v_head_stride, int source_rows, int dtype, int tokens,
                   const int* seq, const int* pos, const int* rows, const int* table, int seqs, int width,
                   void* stream) {
  if (const int e = noise::kv::check_cache(cache)) return e;
  if (tokens > 0 && source_rows > 0 && (!k || !v)) return NOISE_ERR_ARGUMENT;
  noise::kv::Io a = {};
  a.c = *cache;
  a.k = k;
  a.v = v;
  a.k_layer = k_layer_stride, a.k_token = k_token_stride, a.k_head = k_head_stride;
  a.v_layer = v_layer_stride, a.v_token = v_token_stride, a.v_head = v_head_stride;
  a.layer0 = layer, a.layers = layers, a.tokens = tokens, a.source_rows = source_rows;
  a.seq = seq, a.pos = pos, a.rows = rows, a.table = table, a.seqs = seqs, a.width = width;
  return noise::kv::launch(a, dtype, true, stream);
}

int noise_kv_read(const noise_kv_cache_t* cache, int layer, int layers, void* k, void* v, int dtype, int tokens,
                  const int* seq, const int* pos, const int* table, int seqs, int width, void* stream) {
  if (const int e = noise::kv::check_cache(cache)) return e;
  if (tokens > 0 && (!k || !v)) return NOISE_ERR_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16) return NOISE_ERR_ALIGN;
  noise::kv::Io a = {};
  a.c = *cache;
  a.k_out = k;
  a.v_out = v;
  a.layer0 = layer, a.layers = layers, a.tokens = tokens, a.source_rows = tokens;
  a.seq = seq, a.pos = pos, a.table = table, a.seqs = seqs, a.width = width;
  return noise::kv::launch(a, dtype, false, stream);
}

}  // extern "C"
