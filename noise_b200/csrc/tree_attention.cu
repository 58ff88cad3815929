// Attention of a tree of drafted tokens over the paged cache, on sm_100a; one node a sequence is a decoding step, a
// chain a chunk of a prompt (the block's attention, reference utils/model.py:17-31, for the tokens that come next).
//
// Sequence b has len cached tokens and N nodes; node n stands at position len + depth[n] and sees the cached tokens
// that its window reaches and the nodes in its mask: o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q k_j - m). The rows
// of all query heads that share a key head form one tile (row r: node r / group, head r % group), so K and V are read
// once for them. A depth below 0 marks a node that is padding: its row is zero.
//
// A cached key costs D codes of K and of V and 4 D operations a row: with up to some 64 rows of 8-bit codes the
// kernel is bound by the cache's bytes. So it is built to stream them:
//  - Each warp walks the keys 16 at a time and keeps a running maximum, sum and output (32 bits) for its rows. A lane
//    copies its own fragments (cp.async, 16 bytes each, a ring of STAGES steps) and reads back only what it copied
//    itself: no barrier, and the loads of the next steps stay in flight while a step computes.
//  - The order of a contraction's index is free, so it is chosen for the loads: for S = Q K^T a lane takes 16
//    consecutive bytes of a key's row, for P V four neighbouring keys of one dimension, which lie in one word of V's
//    layout; codes become fp16 in registers.
//  - The keys of all sequences, heads and row tiles form one line of units of 64 keys, cut into equal spans, one a
//    CTA, whatever the lengths are. Parts of an item are joined by a second kernel.
// Roundings: Q to fp16 under a power of two per row (an element loses bits only below 2^-14 of the row's largest),
// P 2^(scale of V) to fp16 relative to the largest scale seen; for a bf16 cache and for the nodes' own bf16 keys, P
// to bf16, the type of V. All sums are in fp32.
#include <cuda_runtime.h>

#include <cmath>

#include "kv.cuh"
#include "ptx.cuh"
#include "warp_mma.cuh"

namespace noise {
namespace tree {

constexpr int KW = 4;            // warps that share a row tile's keys: a unit is 16 keys of each
constexpr int UNIT = 16 * KW;
constexpr int MAX_SEQS = 4096;
constexpr int VREF = 127 - 20;   // the output's first unit is 2^-20: V rows with less than that as a scale lose bits
constexpr float NEG = -INFINITY;

struct Params {
  noise_kv_cache_t c;
  int64_t layer_cell;  // layer * pages
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  int64_t q_seq, q_node, q_head, k_seq, k_node, k_head, v_seq, v_node, v_head;
  const int* table;
  const int* lengths;
  const uint64_t* mask;
  const int* depth;
  __nv_bfloat16* out;
  float* partial;  // [2 * grid][RT][D] then m, l [2 * grid][RT]
  int seqs, nodes, group, heads, width, window, page_shift, tiles, grid;
  float scale_log2;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {
  const int n = real ? 16 : 0;  // else zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool real) {
  const int n = real ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float low_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// ---- the line of units ------------------------------------------------------------------------------------------

__device__ __forceinline__ int length_of(const Params& p, int b) {
  const int len = p.lengths[b];
  const int64_t room = static_cast<int64_t>(p.width) << p.page_shift;
  return len < 0 ? 0 : len > room ? static_cast<int>(room) : len;
}

// First unit of 64 keys that some node's window reaches (the least depth of a real node is 0).
__device__ __forceinline__ int first_unit(const Params& p, int len) {
  return p.window < 0 || p.window >= len ? 0 : (len - p.window) / UNIT;
}

// Units of one item of sequence b: one for its nodes, then its cached keys'.
__device__ __forceinline__ int units_of(const Params& p, int b) {
  const int len = length_of(p, b);
  return 1 + (len + UNIT - 1) / UNIT - first_unit(p, len);
}

// before[b] = units of one item of each sequence before b; every thread of the block calls it.
__device__ __forceinline__ void line_of(const Params& p, int* before) {
  for (int b = threadIdx.x; b < p.seqs; b += blockDim.x) before[b + 1] = units_of(p, b);
  __syncthreads();
  if (threadIdx.x < 32) {
    int carry = 0;
    for (int b0 = 0; b0 < p.seqs; b0 += 32) {
      const int b = b0 + threadIdx.x;
      int x = b < p.seqs ? before[b + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (static_cast<int>(threadIdx.x) >= o) x += y;
      }
      if (b < p.seqs) before[b + 1] = carry + x;
      carry += __shfl_sync(0xffffffffu, x, 31);
    }
    if (threadIdx.x == 0) before[0] = 0;
  }
  __syncthreads();
}

struct Spans {  // CTA i takes units [cut(i), cut(i + 1))
  int64_t total;
  int ctas;
  __device__ __forceinline__ Spans(const Params& p, const int* before) {
    total = static_cast<int64_t>(before[p.seqs]) * p.heads * p.tiles;
    const int64_t most = total / 2;  // at least two units each: a shorter span is all overhead
    ctas = most < 1 ? 1 : most < p.grid ? static_cast<int>(most) : p.grid;
  }
  __device__ __forceinline__ int64_t cut(int i) const { return total * i / ctas; }
  __device__ __forceinline__ int owner(int64_t u) const {  // the CTA whose span holds unit u
    int i = static_cast<int>(u * ctas / total);
    while (cut(i) > u) --i;
    while (cut(i + 1) <= u) ++i;
    return i;
  }
};

// ---- one item's part --------------------------------------------------------------------------------------------

template <int KIND, int D, int MT, int RW>
struct Shape {
  static constexpr bool BF = KIND == NOISE_KV_BF16;
  static constexpr int KS = D / 16;                  // steps of Q K^T
  static constexpr int NB = D / 8;                   // columns of 8 of the output
  static constexpr int NL = BF ? D / 16 : D / 32;    // 16-byte loads a lane of K, and of V
  static constexpr int NT = 32 * KW * RW;
  static constexpr int RT = 16 * MT * RW;
  static constexpr int STEP = 2 * NL * 512 + (BF ? 0 : 256);  // bytes of a warp's 16 keys
  static constexpr int STAGES = STEP <= 2500 ? 4 : 3;
  static constexpr bool QREG = MT * KS <= 8;         // Q's fragments in registers, else in shared memory
  static constexpr int RING = STAGES * STEP;
  static constexpr int JOIN = 32 * (4 * MT * NB + 4 * MT) * 4;  // a warp's output, maxima and sums
  static constexpr int QBYTES = QREG ? 0 : RW * MT * KS * 512;
  static constexpr int WORK = KW * RW * RING > 2 * RW * JOIN ? KW * RW * RING : 2 * RW * JOIN;
  static constexpr int SMEM = WORK + QBYTES;
  // the dimension that word (ks) of lane t starts at in Q K^T: 16 consecutive bytes of a key's row a lane
  __device__ static __forceinline__ int dim_of(int ks, int t) {
    return BF ? (ks >> 1) * 32 + t * 8 + (ks & 1) * 4 : (ks >> 2) * 64 + t * 16 + (ks & 3) * 4;
  }
};

template <int KIND, int D, int MT, int RW>
struct Part {
  using S = Shape<KIND, D, MT, RW>;
  float acc[MT][S::NB][4];
  float m[MT][2], l[MT][2], rf[MT][2];  // maxima of the scores before the row's factor rf
  int lo[MT][2];                        // the first cached position in the row's window
  int vref;                             // acc holds the output in units of 2^(vref - 127) (8-bit kinds)

  // Scores s (masked: -inf) to probabilities, the running maximum and sum and the output's rescaling.
  __device__ __forceinline__ void soften(float (&s)[MT][2][4], int new_ref) {
    bool up = new_ref != vref;
    float top[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x = fmaxf(fmaxf(s[mt][0][2 * h], s[mt][0][2 * h + 1]), fmaxf(s[mt][1][2 * h], s[mt][1][2 * h + 1]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        top[mt][h] = fmaxf(m[mt][h], x);
        up |= top[mt][h] > m[mt][h];
      }
    if (__any_sync(0xffffffffu, up)) {
      const float unit = ex2(static_cast<float>(vref - new_ref));
      vref = new_ref;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float f = top[mt][h] > m[mt][h] ? ex2((m[mt][h] - top[mt][h]) * rf[mt][h]) : 1.f;
          m[mt][h] = top[mt][h];
          l[mt][h] *= f;
          const float g = f * unit;
#pragma unroll
          for (int nb = 0; nb < S::NB; ++nb) {
            acc[mt][nb][2 * h] *= g;
            acc[mt][nb][2 * h + 1] *= g;
          }
        }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float off = m[mt][h] == NEG ? 0.f : -m[mt][h] * rf[mt][h];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = s[mt][j][2 * h + e];
            x = ex2(fmaf(x, rf[mt][h], off));
            l[mt][h] += x;
          }
      }
  }
};

// P's fragment of a 16 x 16 tile: columns 2t, 2t + 1 of both blocks of 8 are the lane's four keys 4t .. 4t + 3.
template <bool BF>
__device__ __forceinline__ void p_fragment(const float (&s)[2][4], const float (&f)[4], uint32_t (&a)[4]) {
  if constexpr (BF) {
    a[0] = pack_bf16(s[0][0] * f[0], s[0][1] * f[1]);
    a[1] = pack_bf16(s[0][2] * f[0], s[0][3] * f[1]);
    a[2] = pack_bf16(s[1][0] * f[2], s[1][1] * f[3]);
    a[3] = pack_bf16(s[1][2] * f[2], s[1][3] * f[3]);
  } else {
    a[0] = pack_f16(s[0][0] * f[0], s[0][1] * f[1]);
    a[1] = pack_f16(s[0][2] * f[0], s[0][3] * f[1]);
    a[2] = pack_f16(s[1][0] * f[2], s[1][1] * f[3]);
    a[3] = pack_f16(s[1][2] * f[2], s[1][3] * f[3]);
  }
}

// P V of bf16 values where a probability may be 0 because the key is masked: such a key's infinities and NaN must
// not count, a visible key's must. Values that are not finite are left out of the product and put in by hand: vis has
// 1 for the keys that the row sees, and the products of vis with marks of +inf and of -inf (NaN: both) say what to add.
template <int MT, int NB>
__device__ __forceinline__ void pv_special(float (&acc)[MT][NB][4], int nb, const uint32_t (&a)[MT][4],
                                           const uint32_t (&vis)[MT][4], uint32_t b0, uint32_t b1) {
  const auto special = [](uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; };
  if (!__any_sync(0xffffffffu, special(b0) || special(b1))) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) mma_bf16(acc[mt][nb], a[mt][0], a[mt][1], a[mt][2], a[mt][3], b0, b1);
    return;
  }
  uint32_t b[2] = {b0, b1}, plus[2] = {0, 0}, minus[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int sh = 0; sh < 32; sh += 16) {
      const uint32_t x = b[i] >> sh & 0xffffu;
      if ((x & 0x7f80u) != 0x7f80u) continue;
      const bool nan = (x & 0x7fu) != 0;
      if (nan || !(x & 0x8000u)) plus[i] |= 0x3f80u << sh;
      if (nan || (x & 0x8000u)) minus[i] |= 0x3f80u << sh;
      b[i] &= ~(0xffffu << sh);
    }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    mma_bf16(acc[mt][nb], a[mt][0], a[mt][1], a[mt][2], a[mt][3], b[0], b[1]);
    float up[4] = {0.f, 0.f, 0.f, 0.f}, down[4] = {0.f, 0.f, 0.f, 0.f};
    mma_bf16(up, vis[mt][0], vis[mt][1], vis[mt][2], vis[mt][3], plus[0], plus[1]);
    mma_bf16(down, vis[mt][0], vis[mt][1], vis[mt][2], vis[mt][3], minus[0], minus[1]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (up[e] > 0.f) acc[mt][nb][e] += INFINITY;
      if (down[e] > 0.f) acc[mt][nb][e] -= INFINITY;
    }
  }
}

template <int MT>
__device__ __forceinline__ void visible(const float (&s)[MT][2][4], uint32_t (&vis)[MT][4]) {  // scores, before soften
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = i >> 1, h = i & 1;
      vis[mt][i] = (s[mt][j][2 * h] != NEG ? 0x3f80u : 0u) | (s[mt][j][2 * h + 1] != NEG ? 0x3f800000u : 0u);
    }
}

template <int KIND, int D, int MT, int RW>
__global__ void __launch_bounds__(Shape<KIND, D, MT, RW>::NT)
    attend_kernel(const Params p) {
  using S = Shape<KIND, D, MT, RW>;
  constexpr bool BF = S::BF;
  constexpr int NL = S::NL, KS = S::KS, NB = S::NB;
  extern __shared__ __align__(16) uint8_t smem[];
  uint4* const qs = reinterpret_cast<uint4*>(smem + S::WORK);
  int* const before = reinterpret_cast<int*>(smem + S::SMEM);
  cudaTriggerProgrammaticLaunchCompletion();
  line_of(p, before);
  const Spans spans(p, before);
  if (static_cast<int>(blockIdx.x) >= spans.ctas) return;
  const int64_t first = spans.cut(blockIdx.x), last = spans.cut(blockIdx.x + 1);
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int warp = threadIdx.x >> 5, kw = warp % KW, rw = warp / KW;
  const int rows = p.nodes * p.group, hr = p.heads * p.tiles;
  uint8_t* const ring = smem + warp * S::RING;
  const uint32_t ring_at = smem_u32(ring) + lane * 16;
  int b;
  {
    int low = 0, high = p.seqs - 1;  // the last sequence that begins at or before the span
    while (low < high) {
      const int mid = (low + high + 1) >> 1;
      if (static_cast<int64_t>(before[mid]) * hr <= first) low = mid;
      else high = mid - 1;
    }
    b = low;
  }
  for (int64_t at = first; at < last;) {
    const int64_t base = static_cast<int64_t>(before[b]) * hr;
    const int per = before[b + 1] - before[b];
    const int item = static_cast<int>((at - base) / per);
    const int u0 = static_cast<int>(at - base - static_cast<int64_t>(item) * per);
    const int u1 = last - at < per - u0 ? u0 + static_cast<int>(last - at) : per;
    const int h = item / p.tiles, tile = item - h * p.tiles;
    const int row0 = tile * S::RT + rw * 16 * MT;
    const int len = length_of(p, b);
    const int unit0 = first_unit(p, len) - 1;  // unit u holds the keys from (unit0 + u) * 64 on

    // ---- the cached keys' first copies: issued before Q is read
    const int* table = p.table + static_cast<int64_t>(b) * p.width;
    const int cshift = p.page_shift - 4;
    int chunk = (unit0 + (u0 > 1 ? u0 : 1)) * KW + kw;  // of 16 keys
    const int chunk_end = min((unit0 + u1) * KW, (len + 15) >> 4);
    int ahead = chunk, page0 = -64, pages = 0;
    bool lost = false;
    const auto fetch = [&](int stage) {
      if (ahead < chunk_end) {
        const int pi = ahead >> cshift;
        if (pi >= page0 + 32) {  // the next 32 entries of the table, one a lane
          page0 = pi;
          pages = page0 + lane < p.width ? table[page0 + lane] : 0;
        }
        int page = __shfl_sync(0xffffffffu, pages, pi - page0);
        if (page < 0 || page >= p.c.pages) {
          lost = true;
          page = 0;
        }
        const int64_t cell =
            (((p.layer_cell + page) * p.heads + h) << p.page_shift) + ((ahead & ((1 << cshift) - 1)) << 4);
        const uint32_t to = ring_at + stage * S::STEP;
        const uint8_t* k = static_cast<const uint8_t*>(p.c.k) + cell * D * (BF ? 2 : 1);
        const uint8_t* v = static_cast<const uint8_t*>(p.c.v) + cell * D * (BF ? 2 : 1);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int key = 4 * (g >> 1) + (g & 1) + 2 * j;
#pragma unroll
          for (int c = 0; c < NL / 2; ++c)
            copy16(to + (j * (NL / 2) + c) * 512, k + key * D * (BF ? 2 : 1) + c * 64 + t * 16, true);
        }
#pragma unroll
        for (int c = 0; c < NL; ++c)
          copy16(to + (NL + c) * 512, v + (t * D + c * (BF ? 16 : 32)) * (BF ? 8 : 4) + g * 16, true);
        if constexpr (!BF) {
          const uint32_t s4 = smem_u32(ring) + stage * S::STEP + 2 * NL * 512 + lane * 4;
          copy4(s4, p.c.k_scale + cell + 4 * t, true);
          copy4(s4 + 128, p.c.v_scale + cell + 4 * t, true);
        }
      }
      cp_async_commit();
      ahead += KW;
    };
    for (int i = 0; i < S::STAGES - 1; ++i) fetch(i);

    // ---- Q's fragments
    Part<KIND, D, MT, RW> part;
    uint32_t qr[S::QREG ? MT : 1][S::QREG ? KS : 1][4];
    const __nv_bfloat16* qb = p.q + b * p.q_seq;
    const auto q_row = [&](int mt, int hh, bool& real) {
      const int r = row0 + mt * 16 + hh * 8 + g;
      real = r < rows;
      const int node = real ? r / p.group : 0;
      return qb + node * p.q_node + (h * p.group + (real ? r - node * p.group : 0)) * p.q_head;
    };
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      uint32_t frag[KS][4];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        bool real;
        const __nv_bfloat16* q = q_row(mt, hh, real);
        uint2 x[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          x[ks] = real ? *reinterpret_cast<const uint2*>(q + S::dim_of(ks, t)) : make_uint2(0, 0);
        part.rf[mt][hh] = p.scale_log2;
        if constexpr (!BF) {  // fp16 under a power of two: the row's largest is brought to [1, 2)
          uint32_t top = 0;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            top = max(top, max(x[ks].x & 0x7fffu, x[ks].x >> 16 & 0x7fffu));
            top = max(top, max(x[ks].y & 0x7fffu, x[ks].y >> 16 & 0x7fffu));
          }
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          int e = static_cast<int>(top >> 7);
          e = e == 255 || e < 1 ? 127 : e < 67 ? 67 : e > 253 ? 253 : e;  // (not finite or zero: as it is)
          const float f = kv::power(254 - e);
          part.rf[mt][hh] *= kv::power(e);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            frag[ks][hh] = pack_f16(low_f(x[ks].x) * f, high_f(x[ks].x) * f);
            frag[ks][2 + hh] = pack_f16(low_f(x[ks].y) * f, high_f(x[ks].y) * f);
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            frag[ks][hh] = x[ks].x;
            frag[ks][2 + hh] = x[ks].y;
          }
        }
        const int r = row0 + mt * 16 + hh * 8 + g;
        const int node = r < rows ? r / p.group : 0;
        part.lo[mt][hh] = p.window < 0 ? 0 : len + p.depth[b * p.nodes + node] - p.window;
        part.m[mt][hh] = NEG;
        part.l[mt][hh] = 0.f;
      }
      if constexpr (S::QREG) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int i = 0; i < 4; ++i) qr[mt][ks][i] = frag[ks][i];
      } else if (kw == 0) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          qs[((rw * MT + mt) * KS + ks) * 32 + lane] = make_uint4(frag[ks][0], frag[ks][1], frag[ks][2], frag[ks][3]);
      }
    }
    if constexpr (!S::QREG) __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 4; ++e) part.acc[mt][nb][e] = 0.f;
    part.vref = BF ? 127 : VREF;

    // ---- the tree's own keys: 16 nodes a warp, unquantised, in bf16
    if (u0 == 0 && kw * 16 < p.nodes) {
      float s[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mt][j][e] = 0.f;
      const __nv_bfloat16* kb = p.k + b * p.k_seq + h * p.k_head;
      const __nv_bfloat16* vb = p.v + b * p.v_seq + h * p.v_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint2 kk[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int node = kw * 16 + 4 * (g >> 1) + (g & 1) + 2 * j;
          kk[j] = node < p.nodes ? *reinterpret_cast<const uint2*>(kb + node * p.k_node + S::dim_of(ks, t))
                                 : make_uint2(0, 0);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t a[4];
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            bool real;
            const __nv_bfloat16* q = q_row(mt, hh, real);
            const uint2 x = real ? *reinterpret_cast<const uint2*>(q + S::dim_of(ks, t)) : make_uint2(0, 0);
            a[hh] = x.x;
            a[2 + hh] = x.y;
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) mma_bf16(s[mt][j], a[0], a[1], a[2], a[3], kk[j].x, kk[j].y);
        }
      }
      int dk[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int node = kw * 16 + 4 * t + i;
        dk[i] = node < p.nodes ? p.depth[b * p.nodes + node] : 0;
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int r = row0 + mt * 16 + hh * 8 + g;
          const int node = r < rows ? r / p.group : 0;
          const uint64_t mask = r < rows ? p.mask[b * p.nodes + node] : 0;
          const float f = p.scale_log2 / part.rf[mt][hh];  // scores in the units of the cached keys' (a power of two)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = kw * 16 + 4 * t + i;
            // lo - len = depth - window
            const bool see = key < p.nodes && (mask >> key & 1) && (p.window < 0 || dk[i] >= part.lo[mt][hh] - len);
            float& x = s[mt][i >> 1][2 * hh + (i & 1)];
            x = see ? x * f : NEG;
          }
        }
      uint32_t vis[MT][4], a[MT][4];
      visible<MT>(s, vis);
      part.soften(s, part.vref);
      constexpr float UNITS = BF ? 1.f : 1048576.f;  // 1 in units of 2^(VREF - 127)
      const float one[4] = {UNITS, UNITS, UNITS, UNITS};
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) p_fragment<true>(s[mt], one, a[mt]);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int d = BF ? (nb >> 1) * 16 + 2 * g + (nb & 1) : (nb >> 2) * 32 + 4 * g + (nb & 3);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int node = kw * 16 + 4 * t + i;
          w[i] = node < p.nodes ? __ldg(reinterpret_cast<const unsigned short*>(vb + node * p.v_node + d)) : 0u;
        }
        pv_special<MT, NB>(part.acc, nb, a, vis, w[0] | w[1] << 16, w[2] | w[3] << 16);
      }
    }

    // ---- the cached keys
    int stage = 0;
    for (; chunk < chunk_end; chunk += KW) {
      cp_async_wait<S::STAGES - 2>();
      fetch(stage == 0 ? S::STAGES - 1 : stage - 1);  // the step read last is free
      const uint8_t* step = ring + stage * S::STEP;
      const uint4* own = reinterpret_cast<const uint4*>(step) + lane;
      float s[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mt][j][e] = 0.f;
#pragma unroll
      for (int c = 0; c < NL / 2; ++c) {
        constexpr int PER = BF ? 2 : 4;  // steps in 16 bytes
        uint32_t w[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint4 u = own[(j * (NL / 2) + c) * 32];
          w[j][0] = u.x, w[j][1] = u.y, w[j][2] = u.z, w[j][3] = u.w;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int ks = c * PER + i;
          uint32_t kk[2][2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if constexpr (BF) {
              kk[j][0] = w[j][2 * i], kk[j][1] = w[j][2 * i + 1];
            } else {
              kv::decode4<KIND>(w[j][i], kk[j][0], kk[j][1]);
            }
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint32_t a[4];
            if constexpr (S::QREG) {
#pragma unroll
              for (int e = 0; e < 4; ++e) a[e] = qr[mt][ks][e];
            } else {
              const uint4 u = qs[((rw * MT + mt) * KS + ks) * 32 + lane];
              a[0] = u.x, a[1] = u.y, a[2] = u.z, a[3] = u.w;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if constexpr (BF) mma_bf16(s[mt][j], a[0], a[1], a[2], a[3], kk[j][0], kk[j][1]);
              else mma_f16(s[mt][j], a, kk[j][0], kk[j][1]);
            }
          }
        }
      }
      const int key0 = chunk << 4;
      // some key is past the end, or before the window of the deepest node there could be
      const bool edge = key0 + 16 > len || (p.window >= 0 && key0 < len + p.nodes - p.window);
      uint32_t vb4 = 0;
      bool nan_v = false;
      if constexpr (!BF) {
        const uint32_t kb4 = reinterpret_cast<const uint32_t*>(step + 2 * NL * 512)[lane];
        vb4 = reinterpret_cast<const uint32_t*>(step + 2 * NL * 512)[32 + lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t kbyte = kb4 >> (8 * i) & 0xffu;
          const float f = kbyte == 255 ? __int_as_float(0x7fc00000) : kv::power(kbyte);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            s[mt][i >> 1][i & 1] *= f;
            s[mt][i >> 1][2 + (i & 1)] *= f;
          }
        }
      }
      uint32_t keep = 0xffffffffu;  // a byte for each of the lane's four keys that exist
      if (edge) {
        const int k0 = key0 + 4 * t, left = len - k0;
        keep = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : 0xffffffffu >> (32 - 8 * left);
        vb4 &= keep;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (i >= left || k0 + i < part.lo[mt][hh]) s[mt][i >> 1][2 * hh + (i & 1)] = NEG;
      }
      float f[4] = {1.f, 1.f, 1.f, 1.f};
      int ref = part.vref;
      if constexpr (!BF) {
        uint32_t top = __vmaxu4(vb4, vb4 >> 16);
        top = max(top & 0xffu, top >> 8 & 0xffu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (top == 255) {  // a row of V that reads as NaN: such keys are taken out here, and put into the sum below
          nan_v = true;
          top = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x = vb4 >> (8 * i) & 0xffu;
            top = max(top, x == 255 ? 0u : x);
          }
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        }
        ref = max(ref, static_cast<int>(top));
      }
      uint32_t vis[BF ? MT : 1][4];
      if constexpr (BF) {
        if (edge) visible<MT>(s, vis);
      }
      if (nan_v) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((vb4 >> (8 * i) & 0xffu) == 255) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int hh = 0; hh < 2; ++hh)
                if (s[mt][i >> 1][2 * hh + (i & 1)] != NEG) part.l[mt][hh] = __int_as_float(0x7fc00000);
          }
      }
      part.soften(s, ref);
      if constexpr (!BF) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int x = static_cast<int>(vb4 >> (8 * i) & 0xffu), e = x - ref + 127;
          f[i] = x == 255 || e <= 0 ? 0.f : kv::power(e);
        }
      }
      uint32_t a[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) p_fragment<BF>(s[mt], f, a[mt]);
#pragma unroll
      for (int c = 0; c < NL; ++c) {
        const uint4 u = own[(NL + c) * 32];
        uint32_t w[4] = {u.x, u.y, u.z, u.w};
        if constexpr (BF) {
          if (edge) {
            const uint32_t lo = __byte_perm(keep, 0, 0x1100), hi = __byte_perm(keep, 0, 0x3322);
            w[0] &= lo, w[1] &= hi, w[2] &= lo, w[3] &= hi;
#pragma unroll
            for (int i = 0; i < 2; ++i)
              pv_special<MT, NB>(part.acc, c * 2 + i, a, vis, w[2 * i], w[2 * i + 1]);
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
                mma_bf16(part.acc[mt][c * 2 + i], a[mt][0], a[mt][1], a[mt][2], a[mt][3], w[2 * i], w[2 * i + 1]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t b0, b1;
            kv::decode4<KIND>(w[i] & keep, b0, b1);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) mma_f16(part.acc[mt][c * 4 + i], a[mt], b0, b1);
          }
        }
      }
      stage = stage + 1 == S::STAGES ? 0 : stage + 1;
    }
    cp_async_wait<0>();
    if (lost) {
      record_error(p.c.status, NOISE_DEV_BAD_INDEX);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) part.l[mt][0] = part.l[mt][1] = __int_as_float(0x7fc00000);
    }

    // ---- the warps' parts joined: those of the upper half handed to the lower, then 1 to 0
    if constexpr (!BF) {
      const float unit = ex2(static_cast<float>(part.vref - 127));
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) part.acc[mt][nb][e] *= unit;
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float x = part.l[mt][hh];
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        part.l[mt][hh] = x + __shfl_xor_sync(0xffffffffu, x, 2);
      }
#pragma unroll
    for (int from = KW / 2; from >= 1; from >>= 1) {
      __syncthreads();  // everyone is done with the ring, or with the last round's hand-over
      float4* slab = reinterpret_cast<float4*>(smem + (rw * 2 + kw % from) * S::JOIN) + lane;
      if (kw >= from && kw < 2 * from) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            slab[(mt * NB + nb) * 32] =
                make_float4(part.acc[mt][nb][0], part.acc[mt][nb][1], part.acc[mt][nb][2], part.acc[mt][nb][3]);
          slab[(MT * NB + mt) * 32] = make_float4(part.m[mt][0], part.m[mt][1], part.l[mt][0], part.l[mt][1]);
        }
      }
      __syncthreads();
      if (kw < from) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const float4 o = slab[(MT * NB + mt) * 32];
          const float om[2] = {o.x, o.y}, ol[2] = {o.z, o.w};
          float mine[2], theirs[2];
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const float top = fmaxf(part.m[mt][hh], om[hh]);
            mine[hh] = part.m[mt][hh] == NEG ? 0.f : ex2((part.m[mt][hh] - top) * part.rf[mt][hh]);
            theirs[hh] = om[hh] == NEG ? 0.f : ex2((om[hh] - top) * part.rf[mt][hh]);
            // a row that saw no key may still hold the NaN of a lost page
            part.l[mt][hh] = (part.m[mt][hh] == NEG ? part.l[mt][hh] : part.l[mt][hh] * mine[hh]) +
                             (om[hh] == NEG ? ol[hh] : ol[hh] * theirs[hh]);
            part.m[mt][hh] = top;
          }
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const float4 x = slab[(mt * NB + nb) * 32];
            part.acc[mt][nb][0] = part.acc[mt][nb][0] * mine[0] + x.x * theirs[0];
            part.acc[mt][nb][1] = part.acc[mt][nb][1] * mine[0] + x.y * theirs[0];
            part.acc[mt][nb][2] = part.acc[mt][nb][2] * mine[1] + x.z * theirs[1];
            part.acc[mt][nb][3] = part.acc[mt][nb][3] * mine[1] + x.w * theirs[1];
          }
        }
      }
    }
    if (kw == 0) {
      const bool whole = u0 == 0 && u1 == per;
      const int slot = 2 * blockIdx.x + (at == first ? 0 : 1);
      float* po = p.partial + static_cast<int64_t>(slot) * S::RT * D;
      float* pm = p.partial + static_cast<int64_t>(2 * p.grid) * S::RT * D + static_cast<int64_t>(slot) * 2 * S::RT;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int in = rw * 16 * MT + mt * 16 + hh * 8 + g, r = tile * S::RT + in;
          if (r >= rows) continue;
          const int node = r / p.group;
          const bool pad = p.depth[b * p.nodes + node] < 0;
          const float l = part.l[mt][hh];
          const float f = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
          __nv_bfloat16* out =
              p.out + ((static_cast<int64_t>(b) * p.nodes + node) * p.heads * p.group + h * p.group + r - node * p.group) * D;
          if (!whole && t == 0) {
            pm[in] = part.m[mt][hh] * part.rf[mt][hh];
            pm[S::RT + in] = l;
          }
          constexpr int RUN = BF ? 2 : 4;  // the lane's consecutive dimensions: 2 RUN
#pragma unroll
          for (int c = 0; c < NB / RUN; ++c) {
            float x[2 * RUN];
#pragma unroll
            for (int i = 0; i < RUN; ++i) {
              x[i] = pad ? 0.f : part.acc[mt][c * RUN + i][2 * hh] * f;
              x[RUN + i] = pad ? 0.f : part.acc[mt][c * RUN + i][2 * hh + 1] * f;
            }
            const int d = c * 8 * RUN + t * 2 * RUN;
            if (whole) {
              if constexpr (BF)
                *reinterpret_cast<uint2*>(out + d) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
              else
                *reinterpret_cast<uint4*>(out + d) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]),
                                                                pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
            } else {
#pragma unroll
              for (int i = 0; i < 2 * RUN; i += 4)
                *reinterpret_cast<float4*>(po + in * D + d + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
            }
          }
        }
    }
    at += u1 - u0;
    if (u1 == per && item == hr - 1) ++b;
    __syncthreads();  // the hand-over's memory is the next item's ring
  }
}

// Joins the parts of one item (a block each): o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i, in the parts' order.
__global__ void __launch_bounds__(256) join_kernel(const Params p, int rt, int dim) {
  extern __shared__ int before[];
  line_of(p, before);
  const Spans spans(p, before);
  const int hr = p.heads * p.tiles;
  const int b = blockIdx.x / hr, item = blockIdx.x - b * hr;
  const int per = before[b + 1] - before[b];
  const int64_t u = static_cast<int64_t>(before[b]) * hr + static_cast<int64_t>(item) * per;
  const int c0 = spans.owner(u), c1 = spans.owner(u + per - 1);
  cudaGridDependencySynchronize();
  if (c0 == c1) return;  // it was written whole
  const int slot0 = 2 * c0 + (spans.cut(c0) == u ? 0 : 1);
  const int h = item / p.tiles, tile = item - h * p.tiles, rows = p.nodes * p.group;
  const float* sums = p.partial + static_cast<int64_t>(2 * p.grid) * rt * dim;
  const int quads = dim / 4;
  for (int i = threadIdx.x; i < rt * quads; i += blockDim.x) {
    const int in = i / quads, d = (i - in * quads) * 4, r = tile * rt + in;
    if (r >= rows) return;
    const int node = r / p.group;
    float top = NEG;
    for (int c = c0; c <= c1; ++c)
      top = fmaxf(top, sums[static_cast<int64_t>(c == c0 ? slot0 : 2 * c) * 2 * rt + in]);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = c0; c <= c1; ++c) {
      const int64_t slot = c == c0 ? slot0 : 2 * c;
      const float m = sums[slot * 2 * rt + in], sl = sums[slot * 2 * rt + rt + in];
      const float4 x = *reinterpret_cast<const float4*>(p.partial + (slot * rt + in) * dim + d);
      const float f = m == NEG ? 0.f : ex2(m - top);
      l += m == NEG ? sl : sl * f;
      o.x += x.x * f, o.y += x.y * f, o.z += x.z * f, o.w += x.w * f;
    }
    const bool none = l == 0.f || p.depth[b * p.nodes + node] < 0;
    const float f = none ? 0.f : 1.f / l;
    __nv_bfloat16* out =
        p.out + ((static_cast<int64_t>(b) * p.nodes + node) * p.heads * p.group + h * p.group + r - node * p.group) * dim;
    *reinterpret_cast<uint2*>(out + d) = none ? make_uint2(0, 0)
                                              : make_uint2(pack_bf16(o.x * f, o.y * f), pack_bf16(o.z * f, o.w * f));
  }
}

// ---- host -------------------------------------------------------------------------------------------------------

constexpr int MAX_GRID = 148 * 8;

// The row tile and grid of a call: 16 rows a tile where they hold all, else 32, else 64.
inline int tile_rows(int rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

inline int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return n;
}

template <int KIND, int D, int MT, int RW>
int run(Params& p, size_t workspace_bytes, cudaStream_t s) {
  using S = Shape<KIND, D, MT, RW>;
  const auto kernel = attend_kernel<KIND, D, MT, RW>;
  const int smem = S::SMEM + (p.seqs + 1) * 4;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM + (MAX_SEQS + 1) * 4) !=
      cudaSuccess)
    return NOISE_ERR_CUDA;
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, S::NT, smem) != cudaSuccess || per_sm < 1)
    return NOISE_ERR_CUDA;
  const int sms = sm_count();
  if (sms < 1) return NOISE_ERR_CUDA;
  p.grid = sms * per_sm;
  if (p.grid > MAX_GRID) p.grid = MAX_GRID;
  const int64_t room = static_cast<int64_t>(p.width) << p.page_shift;
  const int64_t units = static_cast<int64_t>(p.seqs) * p.heads * p.tiles * (1 + (room + UNIT - 1) / UNIT);
  if (units / 2 < p.grid) p.grid = units < 4 ? 1 : static_cast<int>(units / 2);
  if (static_cast<size_t>(2) * p.grid * S::RT * (D + 2) * sizeof(float) > workspace_bytes) return NOISE_ERR_WORKSPACE;
  kernel<<<p.grid, S::NT, smem, s>>>(p);
  if (cudaGetLastError() != cudaSuccess) return NOISE_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.seqs * p.heads * p.tiles);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = (p.seqs + 1) * 4;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join_kernel, static_cast<const Params>(p), static_cast<int>(S::RT), D) == cudaSuccess
             ? NOISE_OK
             : NOISE_ERR_CUDA;
}

template <int KIND, int D>
int by_rows(Params& p, size_t bytes, cudaStream_t s) {
  const int rows = p.nodes * p.group;
  if (rows <= 16) return run<KIND, D, 1, 1>(p, bytes, s);
  if (rows <= 32) return run<KIND, D, 2, 1>(p, bytes, s);
  return run<KIND, D, 2, 2>(p, bytes, s);
}

template <int KIND>
int by_dim(Params& p, size_t bytes, cudaStream_t s) {
  return p.c.dim == 64 ? by_rows<KIND, 64>(p, bytes, s) : by_rows<KIND, 128>(p, bytes, s);
}

}  // namespace tree
}  // namespace noise

extern "C" {

size_t noise_tree_attention_workspace_bytes(int seqs, int nodes, int q_heads, int heads, int dim) {
  if (seqs < 1 || nodes < 1 || heads < 1 || q_heads < heads || q_heads % heads || (dim != 64 && dim != 128)) return 0;
  return static_cast<size_t>(2) * noise::tree::MAX_GRID * noise::tree::tile_rows(nodes * (q_heads / heads)) *
         (dim + 2) * sizeof(float);
}

int noise_tree_attention(const noise_kv_cache_t* cache, int layer, const void* q, int64_t q_seq_stride,
                         int64_t q_node_stride, int64_t q_head_stride, int q_heads, const void* k,
                         int64_t k_seq_stride, int64_t k_node_stride, int64_t k_head_stride, const void* v,
                         int64_t v_seq_stride, int64_t v_node_stride, int64_t v_head_stride, int seqs, int nodes,
                         const int* table, int width, const int* lengths, const int64_t* mask, const int* depth,
                         int window, float scale, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace noise::tree;
  if (!cache || !cache->k || !cache->v || !cache->status) return NOISE_ERR_ARGUMENT;
  if (cache->kind != NOISE_KV_BF16 && cache->kind != NOISE_KV_E4M3 && cache->kind != NOISE_KV_INT8)
    return NOISE_ERR_ARGUMENT;
  if (cache->kind != NOISE_KV_BF16 && (!cache->k_scale || !cache->v_scale)) return NOISE_ERR_ARGUMENT;
  if (cache->layers < 1 || cache->pages < 1 || cache->heads < 1 || cache->heads > 4096 ||
      (cache->dim != 64 && cache->dim != 128) || cache->page_size < 16 || cache->page_size > 4096 ||
      (cache->page_size & (cache->page_size - 1)))
    return NOISE_ERR_SHAPE;
  if (layer < 0 || layer >= cache->layers || seqs < 0 || seqs > MAX_SEQS || nodes < 1 || nodes > 64 || width < 0 ||
      q_heads < cache->heads || q_heads % cache->heads || q_heads / cache->heads > 64 ||
      static_cast<int64_t>(width) * cache->page_size > (1 << 30) ||
      seqs * (static_cast<int64_t>(width) * cache->page_size / UNIT + 2) > 0x7fffffff)
    return NOISE_ERR_SHAPE;
  if (!(scale >= 1e-18f) || !(scale <= 1e18f)) return NOISE_ERR_ARGUMENT;
  if (seqs == 0) return NOISE_OK;
  if (!q || !k || !v || !lengths || !mask || !depth || !out || (width > 0 && !table)) return NOISE_ERR_ARGUMENT;
  for (const void* p : {static_cast<const void*>(cache->k), static_cast<const void*>(cache->v),
                        static_cast<const void*>(cache->k_scale), static_cast<const void*>(cache->v_scale), q, k,
                        static_cast<const void*>(out), static_cast<const void*>(workspace)})
    if (reinterpret_cast<uintptr_t>(p) % 16) return NOISE_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(k) % 8 || reinterpret_cast<uintptr_t>(v) % 2) return NOISE_ERR_ALIGN;
  for (int64_t stride : {q_seq_stride, q_node_stride, q_head_stride, k_seq_stride, k_node_stride, k_head_stride})
    if (stride % 4) return NOISE_ERR_ALIGN;
  const int group = q_heads / cache->heads, tile = tile_rows(nodes * group);
  const int tiles = (nodes * group + tile - 1) / tile;
  if (static_cast<int64_t>(seqs) * cache->heads * tiles > 0x7fffffff) return NOISE_ERR_SHAPE;
  if (!workspace) return NOISE_ERR_WORKSPACE;
  Params p = {};
  p.c = *cache;
  p.layer_cell = static_cast<int64_t>(layer) * cache->pages;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.q_seq = q_seq_stride, p.q_node = q_node_stride, p.q_head = q_head_stride;
  p.k_seq = k_seq_stride, p.k_node = k_node_stride, p.k_head = k_head_stride;
  p.v_seq = v_seq_stride, p.v_node = v_node_stride, p.v_head = v_head_stride;
  p.table = table, p.lengths = lengths, p.mask = reinterpret_cast<const uint64_t*>(mask), p.depth = depth;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.partial = static_cast<float*>(workspace);
  p.seqs = seqs, p.nodes = nodes, p.group = group, p.heads = cache->heads, p.width = width, p.window = window;
  p.page_shift = __builtin_ctz(static_cast<unsigned>(cache->page_size));
  p.tiles = tiles;
  p.scale_log2 = scale * 1.4426950408889634f;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cache->kind == NOISE_KV_E4M3) return by_dim<NOISE_KV_E4M3>(p, workspace_bytes, s);
  if (cache->kind == NOISE_KV_INT8) return by_dim<NOISE_KV_INT8>(p, workspace_bytes, s);
  return by_dim<NOISE_KV_BF16>(p, workspace_bytes, s);
}

}  // extern "C"
