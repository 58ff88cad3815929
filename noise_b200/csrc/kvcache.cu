// Writing tokens' keys and values into the paged cache, quantised on the way, and reading them back, on sm_100a.
//
// Entry i of a call goes to position pos[i] of sequence seq[i]: page table[seq, pos / page_size], slot
// pos % page_size. Quantising a row x of D values: 2^e the least power of two with max|x| <= 2^e * 448 (e4m3) or 127
// (int8), code = round(x / 2^e), ties to even. Each value is read once, its code written once: memory-bound. A lane
// takes 8 values of a row, the row's maximum is a few shuffles.
//
// V keeps four neighbouring positions side by side, so a lane takes four entries at once: where they are the four of
// one quad its codes are 32 (bf16: 64) bytes in a row, else single codes. Group i of lanes takes the quad that entry 4 i
// is in, as far as its neighbours in the call are its neighbours in the sequence, and of entries 4 i .. 4 i + 3 those that
// are in no group's quad; so a run of positions that begins anywhere is written by whole quads, and any order is right.
// Measured: 32,768 tokens of 8 int8 heads of 128 written and read back: 90 us, 4.5 TB/s; the write's instructions (some 8
// a value: the maximum, the rounding, V's transposition) keep the issue slots 68% busy and DRAM 44%.
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

struct Place {
  int64_t cell;  // of the page's head: slot 0 of [layers, pages, heads, page_size]
  int row, slot;
  bool real;
};

template <typename T, bool WIDE>
struct Row8 {  // 8 values as they lie in memory
  uint32_t w[sizeof(T) * 2];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + i);
        w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(p[i]);
    } else {
      const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = q[2 * i] | static_cast<uint32_t>(q[2 * i + 1]) << 16;
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) * 2; ++i) w[i] = 0;
  }
  __device__ __forceinline__ uint32_t top() const {  // the largest of the bits of |x|, or some NaN's
    if constexpr (sizeof(T) == 4) {
      uint32_t t = w[0] & 0x7fffffffu;
#pragma unroll
      for (int i = 1; i < 8; ++i) t = max(t, w[i] & 0x7fffffffu);
      return t;
    } else {
      const auto two = [&](int i) { return __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])); };
      const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(two(0), two(1)), __hmax2_nan(two(2), two(3)));
      const uint32_t t = *reinterpret_cast<const uint32_t*>(&m);
      return max(t << 16, t & 0xffff0000u);
    }
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
  }
};

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Rows transposed: out[d] = byte d of each of the four rows, for the four d of a word.
__device__ __forceinline__ void bytes4x4(const uint32_t (&r)[4], uint32_t (&out)[4]) {
  const uint32_t a = __byte_perm(r[0], r[1], 0x5140), b = __byte_perm(r[2], r[3], 0x5140);
  const uint32_t c = __byte_perm(r[0], r[1], 0x7362), d = __byte_perm(r[2], r[3], 0x7362);
  out[0] = __byte_perm(a, b, 0x5410);
  out[1] = __byte_perm(a, b, 0x7632);
  out[2] = __byte_perm(c, d, 0x5410);
  out[3] = __byte_perm(c, d, 0x7632);
}

// The codes of the 8 values (bf16: the values) and the row's scale byte; LPR lanes hold the row.
template <int KIND, int LPR, typename R>
__device__ __forceinline__ uint32_t quantise(const R& x, uint32_t (&code)[KIND == NOISE_KV_BF16 ? 4 : 2]) {
  if constexpr (KIND == NOISE_KV_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) code[i] = pack2(x[2 * i], x[2 * i + 1]);
    return 0;
  } else {
    uint32_t top = x.top();  // the bits of the largest |x|: orders NaN above infinity above the finite
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
}

template <int KIND>
__device__ __forceinline__ void scaled8(const uint32_t (&code)[KIND == NOISE_KV_BF16 ? 4 : 2], uint32_t b,
                                        float (&x)[8]) {
  if constexpr (KIND == NOISE_KV_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(code[i] << 16);
      x[2 * i + 1] = __uint_as_float(code[i] & 0xffff0000u);
    }
  } else {
    uint32_t h[4];
    decode4<KIND>(code[0], h[0], h[1]);
    decode4<KIND>(code[1], h[2], h[3]);
    const float m = b == 255 ? __int_as_float(0x7fc00000) : b ? power(b) : 5.877471754111438e-39f;  // 2^-127
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
      x[2 * i] = f.x * m;
      x[2 * i + 1] = f.y * m;
    }
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

// The entries that group i of lanes takes: the quad of entry 4 i, then strays; at most 4 + 3.
struct Group {
  int first;       // entry of the quad's first position (may be before 4 i, or before the call's first)
  unsigned quad;   // bit e: entry first + e is there, and at the quad's position e
  unsigned stray;  // bit e: entry 4 i + e is in no group's quad

  __device__ __forceinline__ Group() : first(0), quad(0), stray(0) {}
  __device__ __forceinline__ Group(const Io& a, int i) {
    const int at = 4 * i;
    // sequence and position of entries at - 3 .. at + 7, as far as the call goes
    const auto in = [&](int e) { return e >= 0 && e < a.tokens; };
    const int s0 = __ldg(a.seq + at), p0 = __ldg(a.pos + at), phase = p0 & 3;
    const bool more = in(at + 4);
    const int s1 = more ? __ldg(a.seq + at + 4) : -1, p1 = more ? __ldg(a.pos + at + 4) : 0;
    first = at - phase;
    quad = stray = 0;
#pragma unroll
    for (int d = -3; d < 4; ++d) {
      const int e = at + d;
      if (!in(e)) continue;
      const int s = __ldg(a.seq + e), p = __ldg(a.pos + e);
      const int k = d + phase;
      if (s0 >= 0 && p0 >= 0 && k >= 0 && k < 4 && s == s0 && p - p0 == d) {
        quad |= 1u << k;
      } else if (d > 0) {  // in the quad of entry at + 4?
        const int k1 = d - 4 + (p1 & 3);
        if (!(more && s1 >= 0 && p1 >= 0 && k1 >= 0 && s == s1 && p - p1 == d - 4)) stray |= 1u << d;
      } else if (d == 0) {
        stray |= 1u;  // entry 4 i itself is to be skipped
      }
    }
  }
};

// Slot 0's cell of the page that holds position p of sequence s, or -1.
__device__ __forceinline__ int64_t cell_of(const Io& a, int s, int p, int h, int layer) {
  const int at = p >> a.page_shift;
  if (s >= a.seqs || at >= a.width) return -1;
  const int page = __ldg(a.table + static_cast<int64_t>(s) * a.width + at);
  if (page < 0 || page >= a.c.pages) return -1;
  return ((static_cast<int64_t>(a.layer0 + layer) * a.c.pages + page) * a.c.heads + h) << a.page_shift;
}

// Where entry e goes: real, or to be skipped; report: say so if it is out of range.
__device__ __forceinline__ Place place(const Io& a, int e, int h, int layer, bool report) {
  Place to = {0, a.rows ? __ldg(a.rows + e) : e, 0, false};
  const int s = __ldg(a.seq + e), p = __ldg(a.pos + e);
  if (s < 0 || p < 0 || to.row < 0) return to;
  to.slot = p & (a.c.page_size - 1);
  to.cell = to.row < a.source_rows ? cell_of(a, s, p, h, layer) : -1;
  to.real = to.cell >= 0;
  if (!to.real && report) record_error(a.c.status, NOISE_DEV_BAD_INDEX);
  return to;
}

// blockIdx.x: groups of PER entries, blockIdx.y: heads, blockIdx.z: layers. PER 4: quads and strays as above; PER 1: an
// entry a group, for calls so small that they last as long as one group does.
template <typename T, int KIND, int LPR, bool WIDE, int PER>
__global__ void __launch_bounds__(NT) write_kernel(const Io a) {
  constexpr bool BF = KIND == NOISE_KV_BF16;
  constexpr int CW = BF ? 4 : 2;  // words of 8 codes
  const int sub = threadIdx.x % LPR, d = sub * 8, h = blockIdx.y, layer = blockIdx.z;
  const int i = blockIdx.x * (NT / LPR) + threadIdx.x / LPR;
  const bool here = PER * i < a.tokens, mine = d < a.c.dim;
  const T* ks = static_cast<const T*>(a.k) + layer * a.k_layer + h * a.k_head + d;
  const T* vs = static_cast<const T*>(a.v) + layer * a.v_layer + h * a.v_head + d;
  Group g;
  if constexpr (PER == 4) {
    if (here) g = Group(a, i);
  } else {
    g.stray = here ? 1u : 0u;
  }
  // the rows of all entries are loaded before the first is used
  const auto put = [&](const Place (&to)[PER], bool quad) {
    Row8<T, WIDE> k[PER], v[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      k[e].zero();
      v[e].zero();
      if (to[e].real && mine) {
        k[e].load(ks + to[e].row * a.k_token);
        v[e].load(vs + to[e].row * a.v_token);
      }
    }
    uint32_t code[PER][CW], kb = 0, vb = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      kb |= quantise<KIND, LPR>(k[e], code[e]) << (8 * e);
      if (to[e].real && mine) {
        const int64_t at = (to[e].cell + to[e].slot) * a.c.dim + d;
        if constexpr (BF)
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.c.k) + at) =
              make_uint4(code[e][0], code[e][1], code[e][2], code[e][3]);
        else
          *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.c.k) + at) = make_uint2(code[e][0], code[e][1]);
      }
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) vb |= quantise<KIND, LPR>(v[e], code[e]) << (8 * e);
    if (!mine) return;
    if constexpr (PER == 4) {
      if (quad) {  // to[0].slot is a multiple of 4
        const int64_t cell = to[0].cell + to[0].slot;
        if constexpr (BF) {
          uint4* out = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.c.v) + cell * a.c.dim + d * 4);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            out[j] = make_uint4(
                __byte_perm(code[0][j], code[1][j], 0x5410), __byte_perm(code[2][j], code[3][j], 0x5410),
                __byte_perm(code[0][j], code[1][j], 0x7632), __byte_perm(code[2][j], code[3][j], 0x7632));
        } else {
          uint4* out = reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.c.v) + cell * a.c.dim + d * 4);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t r[4] = {code[0][j], code[1][j], code[2][j], code[3][j]};
            uint32_t t[4];
            bytes4x4(r, t);
            out[j] = make_uint4(t[0], t[1], t[2], t[3]);
          }
          if (sub == 0) {
            *reinterpret_cast<uint32_t*>(a.c.k_scale + cell) = kb;
            *reinterpret_cast<uint32_t*>(a.c.v_scale + cell) = vb;
          }
        }
        return;
      }
    }
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (to[e].real) {
        const int64_t at = ((to[e].cell >> 2) + (to[e].slot >> 2)) * a.c.dim * 4 + d * 4 + (to[e].slot & 3);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (BF)
            static_cast<unsigned short*>(a.c.v)[at + 4 * j] =
                static_cast<unsigned short>(code[e][j >> 1] >> (16 * (j & 1)));
          else
            static_cast<uint8_t*>(a.c.v)[at + 4 * j] = static_cast<uint8_t>(code[e][j >> 2] >> (8 * (j & 3)));
        }
        if (!BF && sub == 0) {
          a.c.k_scale[to[e].cell + to[e].slot] = static_cast<uint8_t>(kb >> (8 * e));
          a.c.v_scale[to[e].cell + to[e].slot] = static_cast<uint8_t>(vb >> (8 * e));
        }
      }
  };
  Place to[PER];
  if constexpr (PER == 4) {
    const int p0 = here ? __ldg(a.pos + 4 * i) : 0;  // one page holds the quad
    const int64_t cell = g.quad ? cell_of(a, __ldg(a.seq + 4 * i), p0, h, layer) : -1;
    unsigned real = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = g.quad >> e & 1;
      const int row = !in ? -1 : a.rows ? __ldg(a.rows + g.first + e) : g.first + e;
      to[e] = {cell, row, (p0 & (a.c.page_size - 4)) + e, row >= 0 && row < a.source_rows && cell >= 0};
      if (row >= 0 && !to[e].real && sub == 0) record_error(a.c.status, NOISE_DEV_BAD_INDEX);
      if (to[e].real) real |= 1u << e;
    }
    put(to, real == 15u);
    if (!__any_sync(0xffffffffu, g.stray != 0)) return;
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    to[e] = {0, 0, 0, false};
    if (g.stray >> e & 1) to[e] = place(a, PER * i + e, h, layer, sub == 0);
  }
  put(to, false);
}

template <typename T, int KIND, int LPR, int PER>
__global__ void __launch_bounds__(NT) read_kernel(const Io a) {
  constexpr bool BF = KIND == NOISE_KV_BF16;
  constexpr int CW = BF ? 4 : 2;
  const int sub = threadIdx.x % LPR, d = sub * 8, h = blockIdx.y, layer = blockIdx.z;
  const int i = blockIdx.x * (NT / LPR) + threadIdx.x / LPR;
  if (PER * i >= a.tokens || d >= a.c.dim) return;
  Group g;
  if constexpr (PER == 4) g = Group(a, i);
  else g.stray = 1u;
  T* const ko = static_cast<T*>(a.k_out) + (static_cast<int64_t>(layer) * a.tokens * a.c.heads + h) * a.c.dim + d;
  T* const vo = static_cast<T*>(a.v_out) + (static_cast<int64_t>(layer) * a.tokens * a.c.heads + h) * a.c.dim + d;
  const int64_t token = static_cast<int64_t>(a.c.heads) * a.c.dim;
  const auto load_k = [&](const Place& at, uint32_t (&c)[CW]) {
    if constexpr (BF) {
      const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.c.k) +
                                                      (at.cell + at.slot) * a.c.dim + d);
      c[0] = u.x, c[1] = u.y, c[2] = u.z, c[3] = u.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.c.k) + (at.cell + at.slot) * a.c.dim + d);
      c[0] = u.x, c[1] = u.y;
    }
  };
  const auto put = [&](T* to, int e, const uint32_t (&c)[CW], uint32_t b) {
    float x[8];
    scaled8<KIND>(c, b, x);
    store8(to + e * token, x);
  };
  const auto fill = [&](int e, float f) {  // skipped: zeros; out of range: NaN
    const float x[8] = {f, f, f, f, f, f, f, f};
    store8(ko + e * token, x);
    store8(vo + e * token, x);
  };
  const auto bad = [&](int e) { return a.seq[e] < 0 || a.pos[e] < 0 ? 0.f : __int_as_float(0x7fc00000); };
  if (PER == 4 && g.quad) {  // the whole quad's codes, of which the entries that are there are put out
    Place at = {0, 0, 0, false};
#pragma unroll
    for (int e = 3; e >= 0; --e)
      if (g.quad >> e & 1) at = place(a, g.first + e, h, layer, sub == 0);
    if (at.real) {
      const int64_t cell = at.cell + (at.slot & ~3);
      uint32_t kc[4][CW], vc[4][CW], kb = 0, vb = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) load_k({at.cell, 0, (at.slot & ~3) + e, true}, kc[e]);
      if constexpr (BF) {
        const uint4* in = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.c.v) + cell * a.c.dim + d * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 u = in[j];
          vc[0][j] = __byte_perm(u.x, u.z, 0x5410), vc[1][j] = __byte_perm(u.x, u.z, 0x7632);
          vc[2][j] = __byte_perm(u.y, u.w, 0x5410), vc[3][j] = __byte_perm(u.y, u.w, 0x7632);
        }
      } else {
        const uint4* in = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.c.v) + cell * a.c.dim + d * 4);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint4 u = in[j];
          const uint32_t r[4] = {u.x, u.y, u.z, u.w};
          uint32_t t[4];
          bytes4x4(r, t);
#pragma unroll
          for (int e = 0; e < 4; ++e) vc[e][j] = t[e];
        }
        kb = *reinterpret_cast<const uint32_t*>(a.c.k_scale + cell);
        vb = *reinterpret_cast<const uint32_t*>(a.c.v_scale + cell);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (g.quad >> e & 1) {
          put(ko, g.first + e, kc[e], kb >> (8 * e) & 0xffu);
          put(vo, g.first + e, vc[e], vb >> (8 * e) & 0xffu);
        }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (g.quad >> e & 1) fill(g.first + e, bad(g.first + e));
    }
  }
  if (!g.stray) return;
  Place at[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    at[e] = {0, 0, 0, false};
    if (g.stray >> e & 1) at[e] = place(a, PER * i + e, h, layer, sub == 0);
  }
  uint32_t kc[PER][CW], vc[PER][CW], kb[PER], vb[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    if (!at[e].real) continue;
    load_k(at[e], kc[e]);
    const int64_t from = ((at[e].cell >> 2) + (at[e].slot >> 2)) * a.c.dim * 4 + d * 4 + (at[e].slot & 3);
#pragma unroll
    for (int j = 0; j < CW; ++j) vc[e][j] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (BF)
        vc[e][j >> 1] |= static_cast<uint32_t>(static_cast<const unsigned short*>(a.c.v)[from + 4 * j]) << (16 * (j & 1));
      else
        vc[e][j >> 2] |= static_cast<uint32_t>(static_cast<const uint8_t*>(a.c.v)[from + 4 * j]) << (8 * (j & 3));
    }
    kb[e] = BF ? 0u : a.c.k_scale[at[e].cell + at[e].slot];
    vb[e] = BF ? 0u : a.c.v_scale[at[e].cell + at[e].slot];
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    if (!(g.stray >> e & 1)) continue;
    if (at[e].real) {
      put(ko, PER * i + e, kc[e], kb[e]);
      put(vo, PER * i + e, vc[e], vb[e]);
    } else {
      fill(PER * i + e, bad(PER * i + e));
    }
  }
}

template <typename T, int KIND, int LPR, int PER>
cudaError_t run(const Io& a, bool write, bool wide, cudaStream_t s) {
  const int groups = a.tokens / PER + (a.tokens % PER != 0);
  const dim3 grid((groups + NT / LPR - 1) / (NT / LPR), a.c.heads, a.layers);
  if (!write)
    read_kernel<T, KIND, LPR, PER><<<grid, NT, 0, s>>>(a);
  else if (wide)
    write_kernel<T, KIND, LPR, true, PER><<<grid, NT, 0, s>>>(a);
  else
    write_kernel<T, KIND, LPR, false, PER><<<grid, NT, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T, int KIND, int LPR>
cudaError_t by_size(const Io& a, bool write, bool wide, cudaStream_t s) {
  // an entry a group where all entries fit the SMs' threads at once. Written and read, 8 int8 heads of 64, an entry a group
  // and four: 5 and 12 us for 8 tokens, 12.3 and 15.4 for 4,736, 55 and 52 for 32,768 (of 128: 149 and 91)
  return static_cast<int64_t>(a.tokens) * a.c.heads * a.layers * LPR <= 148 * 2048
             ? run<T, KIND, LPR, 1>(a, write, wide, s)
             : run<T, KIND, LPR, 4>(a, write, wide, s);
}

template <typename T, int KIND>
cudaError_t by_lanes(const Io& a, bool write, bool wide, cudaStream_t s) {
  if (a.c.dim <= 16) return by_size<T, KIND, 2>(a, write, wide, s);
  if (a.c.dim <= 32) return by_size<T, KIND, 4>(a, write, wide, s);
  if (a.c.dim <= 64) return by_size<T, KIND, 8>(a, write, wide, s);
  if (a.c.dim <= 128) return by_size<T, KIND, 16>(a, write, wide, s);
  return by_size<T, KIND, 32>(a, write, wide, s);
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
  if (a.tokens < 0 || a.tokens > (1 << 30) || a.seqs < 0 || a.width < 0 || a.source_rows < 0 || a.layers < 1 ||
      a.layers > 65535 || a.layer0 < 0 || a.layer0 > a.c.layers - a.layers)
    return NOISE_ERR_SHAPE;
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
