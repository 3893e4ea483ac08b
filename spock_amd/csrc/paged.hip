// paged.hip -- a serving step over a paged key/value cache: rotary positions
// with several axes and the store into the pages (spk_mrope_append), and the
// attention of each sequence's new tokens over its pages
// (spk_paged_attention).
#include <algorithm>
#include <cmath>

#include "capi_common.hpp"
#include "numerics.hpp"
#include "paged.hpp"

namespace {

using spk_paged::Cache;
using spk_paged::Seq;

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

// The two 16-bit types: conversions (round to nearest even) and products.
template <bool BF>
struct Half;
template <>
struct Half<false> {
  // Weights are stored as 2^7 of themselves: with the running maximum at most
  // 8 binades behind they stay below 2^15, and a weight keeps all its bits
  // down to 2^-21 of the row's largest instead of 2^-14.
  static constexpr float kShift = 7.0f;
  static __device__ __forceinline__ float2_t unpack(uint32_t u) {
    half2_t h = __builtin_bit_cast(half2_t, u);
    return float2_t{(float)h.x, (float)h.y};
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, half2_t{(_Float16)a, (_Float16)b});
  }
  static __device__ __forceinline__ uint16_t one(float a) { return __builtin_bit_cast(uint16_t, (_Float16)a); }
  static __device__ __forceinline__ float widen(uint16_t u) { return (float)__builtin_bit_cast(_Float16, u); }
  // an infinity or NaN among the two
  static __device__ __forceinline__ bool odd(uint32_t u) {
    return (u & 0x7c00u) == 0x7c00u || (u & 0x7c000000u) == 0x7c000000u;
  }
  // the two with such values as zeros
  static __device__ __forceinline__ uint32_t finite(uint32_t u) {
    return ((u & 0x7c00u) == 0x7c00u ? 0u : u & 0xffffu) | ((u & 0x7c000000u) == 0x7c000000u ? 0u : u & 0xffff0000u);
  }
  static __device__ __forceinline__ floatx4 mfma16(uint4 a, uint4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0,
                                                  0, 0);
  }
  static __device__ __forceinline__ floatx16 mfma32(uint4 a, uint4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0,
                                                  0, 0);
  }
};
template <>
struct Half<true> {
  static constexpr float kShift = 0.0f;  // the exponent range is fp32's
  static __device__ __forceinline__ float2_t unpack(uint32_t u) {
    return float2_t{__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)};
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, bf2_t{(__bf16)a, (__bf16)b});
  }
  static __device__ __forceinline__ uint16_t one(float a) { return __builtin_bit_cast(uint16_t, (__bf16)a); }
  static __device__ __forceinline__ float widen(uint16_t u) { return __uint_as_float((uint32_t)u << 16); }
  static __device__ __forceinline__ bool odd(uint32_t u) {
    return (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u;
  }
  static __device__ __forceinline__ uint32_t finite(uint32_t u) {
    return ((u & 0x7f80u) == 0x7f80u ? 0u : u & 0xffffu) | ((u & 0x7f800000u) == 0x7f800000u ? 0u : u & 0xffff0000u);
  }
  static __device__ __forceinline__ floatx4 mfma16(uint4 a, uint4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8_t, a), __builtin_bit_cast(bf8_t, b), c, 0, 0,
                                                   0);
  }
  static __device__ __forceinline__ floatx16 mfma32(uint4 a, uint4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8_t, a), __builtin_bit_cast(bf8_t, b), c, 0, 0,
                                                   0);
  }
};

// ---------------------------------------------------------------------------
// Rotary positions and the store into the pages.
// ---------------------------------------------------------------------------

struct Mrope {
  Cache c;
  const uint16_t *q, *k, *v, *qw, *kw;
  uint16_t *qo, *kc, *vc;
  int64_t qt, qh, kt, kh, vt, vh, ot, oh;
  const int32_t* positions;
  int64_t pos_stride;
  const float* rope;
  int32_t rope_rows, rot, heads, kv_heads;
  float eps;
  uint8_t axis[128];
};

// One wave per token.  D / 16 lanes hold a head, 16 elements each: chunks of 8
// that rotate together (HALVES: chunk j and j + rot/16; ADJACENT: the pairs
// lie inside a chunk), so the angles of a lane are the same for every head of
// the token and are read once.
template <int D, bool BF, bool ADJ>
__global__ __launch_bounds__(256) void mrope_append_kernel(Mrope a) {
  constexpr int L = D / 16, RG = 64 / L;  // lanes of a head, heads at a time
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.c.total_tokens) return;
  const int s = spk_paged::seq_of_token(a.c.cu, a.c.num_seqs, t, lane);
  if (s >= a.c.num_seqs) return;
  const Seq sq = spk_paged::seq_at(a.c, s);
  if (t < sq.first || t >= sq.first + sq.n) return;
  const int pos = sq.ctx - sq.n + (t - sq.first);
  const int64_t slot = pos < 0 ? -1 : spk_paged::offset_of(a.c, s, pos);

  // chunks of this lane, and its 8 pairs' angles
  const int j = lane % L, rg = lane / L;
  const int turning = a.rot / 16;  // lanes that rotate
  const bool turns = j < turning;
  const int c0 = ADJ ? 2 * j : turns ? j : 2 * j;
  const int c1 = ADJ ? 2 * j + 1 : turns ? j + turning : 2 * j + 1;
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.0f;
    sn[e] = 0.0f;
    if (turns) {
      const int pair = 8 * j + e;
      int row = a.positions[a.axis[pair] * a.pos_stride + t];
      row = min(max(row, 0), a.rope_rows - 1);
      const float2 v = *reinterpret_cast<const float2*>(a.rope + (int64_t)row * a.rot + 2 * pair);
      cs[e] = v.x;
      sn[e] = v.y;
    }
  }

  const int rows = a.heads + 2 * a.kv_heads;
  for (int r = rg; r < rows; r += RG) {
    const bool isq = r < a.heads, isv = r >= a.heads + a.kv_heads;
    const int h = isq ? r : isv ? r - a.heads - a.kv_heads : r - a.heads;
    const uint16_t* src = isq ? a.q + t * a.qt + h * a.qh : isv ? a.v + t * a.vt + h * a.vh : a.k + t * a.kt + h * a.kh;
    uint16_t* dst = isq ? a.qo + t * a.ot + h * a.oh : (isv ? a.vc : a.kc) + slot + h * a.c.head_stride;
    const uint16_t* w = isq ? a.qw : isv ? nullptr : a.kw;
    uint4 u0 = *reinterpret_cast<const uint4*>(src + 8 * c0);
    uint4 u1 = *reinterpret_cast<const uint4*>(src + 8 * c1);
    if (!isv) {
      float x[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2_t lo = Half<BF>::unpack((&u0.x)[i]), hi = Half<BF>::unpack((&u1.x)[i]);
        x[2 * i] = lo.x;
        x[2 * i + 1] = lo.y;
        x[8 + 2 * i] = hi.x;
        x[8 + 2 * i + 1] = hi.y;
      }
      if (w) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
#pragma unroll
        for (int m = L / 2; m; m >>= 1) ss += __shfl_xor(ss, m);
        const float inv = spk::rsqrt_det(ss / (float)D + a.eps);
        const uint4 w0 = *reinterpret_cast<const uint4*>(w + 8 * c0), w1 = *reinterpret_cast<const uint4*>(w + 8 * c1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2_t lo = Half<BF>::unpack((&w0.x)[i]), hi = Half<BF>::unpack((&w1.x)[i]);
          x[2 * i] *= inv * (1.0f + lo.x);
          x[2 * i + 1] *= inv * (1.0f + lo.y);
          x[8 + 2 * i] *= inv * (1.0f + hi.x);
          x[8 + 2 * i + 1] *= inv * (1.0f + hi.y);
        }
      }
      if (turns) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i1 = ADJ ? 2 * e : e, i2 = ADJ ? 2 * e + 1 : 8 + e;
          const float x1 = x[i1], x2 = x[i2];
          x[i1] = __builtin_fmaf(x1, cs[e], -(x2 * sn[e]));
          x[i2] = __builtin_fmaf(x2, cs[e], x1 * sn[e]);
        }
      }
      if (w || turns) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          (&u0.x)[i] = Half<BF>::pack(x[2 * i], x[2 * i + 1]);
          (&u1.x)[i] = Half<BF>::pack(x[8 + 2 * i], x[8 + 2 * i + 1]);
        }
      }
    }
    if (isq || slot >= 0) {
      *reinterpret_cast<uint4*>(dst + 8 * c0) = u0;
      *reinterpret_cast<uint4*>(dst + 8 * c1) = u1;
    }
  }
}

// ---------------------------------------------------------------------------
// Attention over the pages.
// ---------------------------------------------------------------------------

struct Attn {
  Cache c;
  const uint16_t *q, *k, *v, *gate;
  uint16_t* out;
  float* lse;
  float* part;  // [splits][total_tokens * heads][D + 2] where splits > 1
  int64_t qt, qh, gt, gh, ot, oh;
  int32_t heads, kv_heads, group, window, one_tile;
  // key ranges of a tile and the least keys of one: [0] sequences of few rows, [1] of many
  int32_t splits[2], chunk[2], tile_rows[2];
  int32_t many;      // a sequence has many rows from this on
  float scale_log2;  // scale * log2(e)
};

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kBehind = 8.0f;  // binades that the running maximum may lag

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Keys in one range of a tile that sees [lo, hi): the plan's, or more where
// the lengths pass the host's bound.
__device__ __forceinline__ int range_keys(const Attn& a, int kind, int lo, int hi) {
  const int span = max(hi - (lo & ~31), 0), splits = a.splits[kind];
  return max(a.chunk[kind], (int)((((int64_t)span + splits - 1) / splits + 127) & ~127));
}

// Tile `at` of the row tiles of the sequences of few (kind 0) or many (1) rows
// (n * group rows of a sequence, `rows` to a tile, sequences in order): its
// sequence and its index there.  false past the last.
__device__ __forceinline__ bool find_tile(const Attn& a, int kind, int rows, int at, int lane, int* seq, int* tile) {
  for (int s0 = 0; s0 < a.c.num_seqs; s0 += 64) {
    int mine = 0;
    if (s0 + lane < a.c.num_seqs) {
      const int n = spk_paged::make_seq(a.c, a.c.cu[s0 + lane], a.c.cu[s0 + lane + 1], 0).n * a.group;
      if ((n >= a.many) == (kind == 1)) mine = (n + rows - 1) / rows;
    }
    int sum = mine;  // inclusive scan
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    const int total = __shfl(sum, 63);
    if (at < total) {
      const int l = __popcll(__ballot(sum <= at));
      *seq = s0 + l;
      *tile = at - (__shfl(sum, l) - __shfl(mine, l));
      return true;
    }
    at -= total;
  }
  return false;
}

// out (gated, rounded) of 4-aligned elements d .. d + N of a row.
template <bool BF, int N>
__device__ __forceinline__ void store_out(const Attn& a, int token, int head, int d, const float (&o)[N]) {
  float x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = o[i];
  if (a.gate) {
    const uint16_t* g = a.gate + token * a.gt + head * a.gh + d;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2_t v = Half<BF>::unpack(*reinterpret_cast<const uint32_t*>(g + i));
      x[i] = x[i] / (1.0f + exp2_fast(v.x * -1.44269504f));
      x[i + 1] = x[i + 1] / (1.0f + exp2_fast(v.y * -1.44269504f));
    }
  }
  uint16_t* out = a.out + token * a.ot + head * a.oh + d;
#pragma unroll
  for (int i = 0; i < N; i += 4)
    *reinterpret_cast<uint2*>(out + i) =
        make_uint2(Half<BF>::pack(x[i], x[i + 1]), Half<BF>::pack(x[i + 2], x[i + 3]));
}

// Few rows per sequence and KV head.  A workgroup takes 16 * MT of the
// n * group rows and a range of the keys; each of its 4 waves takes every
// fourth step of 32 keys by itself, straight from memory into registers (the
// rows share each K and V element, nothing is staged), and the waves' softmax
// states are joined in LDS at the end.
//
// Scores are formed transposed, S^T = K Q^T (16x16x32), so that a lane holds
// 8 keys' scores of one row: the running maximum and sum need no exchange
// while the maximum lags by less than 8 binades, and the 8 weights are
// directly the B operand of O^T += V^T P^T.  The order of the 32 keys in that
// product is free: lane group g supplies keys 4g..4g+3 and 16+4g..+3, which are the
// ones its scores are.  V's A operand (8 keys of one dimension) is made from
// 16-byte row pieces by pairing halfwords of two keys.
template <int D, int MT, bool BF>
__global__ __launch_bounds__(256) void paged_rows_kernel(Attn a) {
  using H = Half<BF>;
  constexpr int DC = D / 32;             // contraction steps of the scores
  constexpr int EV = D >= 128 ? 8 : 4;   // elements of V in one load
  constexpr int NH = D / (16 * EV);      // loads that cover a row
  constexpr int LD = D + 4;              // padded rows of the joint
  __shared__ __align__(16) float joint[4][16][LD];
  __shared__ float stat[4][16][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ln = lane & 15, g = lane >> 4;
  const int split = blockIdx.x, kvh = blockIdx.y;
  int seq = blockIdx.z, tile = 0;
  if (!a.one_tile && !find_tile(a, 0, 16 * MT, blockIdx.z, lane, &seq, &tile)) return;
  const Seq sq = spk_paged::seq_at(a.c, seq);
  const int rows = sq.n * a.group;
  const int r0 = tile * 16 * MT;
  if (r0 >= rows) return;
  // keys that any row of the tile sees, and those that all see
  int lo, hi, lo_all, hi_all;
  spk_paged::visible(sq, r0 / a.group, a.window, &lo, &hi_all);
  spk_paged::visible(sq, (min(r0 + 16 * MT, rows) - 1) / a.group, a.window, &lo_all, &hi);
  const int keys = range_keys(a, 0, lo, hi);
  const int begin = (int)min((int64_t)(lo & ~31) + (int64_t)split * keys, (int64_t)hi);
  const int end = begin + min(keys, hi - begin);
  if (begin >= end && a.splits[0] > 1) return;

  // this lane's row of each 16-row tile
  uint4 q[MT][DC];
  int row_lo[MT], row_hi[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = min(r0 + 16 * mt + ln, rows - 1);
    const int i = r / a.group;
    spk_paged::visible(sq, i, a.window, &row_lo[mt], &row_hi[mt]);
    const uint16_t* src = a.q + (sq.first + i) * a.qt + (kvh * a.group + r - i * a.group) * a.qh;
#pragma unroll
    for (int c = 0; c < DC; ++c) q[mt][c] = *reinterpret_cast<const uint4*>(src + 32 * c + 8 * g);
  }
  float m[MT], base[MT], l[MT];
  floatx4 acc[MT][NH][EV];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt] = -INFINITY;
    base[mt] = 0.0f;
    l[mt] = 0.0f;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int e = 0; e < EV; ++e) acc[mt][h][e] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const int32_t* table = a.c.table + (int64_t)seq * a.c.table_stride;
  const uint16_t* kbase = a.k + kvh * a.c.head_stride;
  const uint16_t* vbase = a.v + kvh * a.c.head_stride;

  for (int k0 = begin + 32 * wave; k0 < end; k0 += 128) {
    // lane l looks up key k0 + l % 32; keys outside the range or without a
    // page read the pool's first row and are masked
    const int key = k0 + (lane & 31);
    int64_t off = -1;
    if (key >= lo && key < end) off = spk_paged::offset_in(a.c, table[spk_paged::divide(a.c.div, (uint32_t)key)], key);
    const uint32_t valid = (uint32_t)__ballot(off >= 0);
    if (off < 0) off = 0;
    const bool full = valid == 0xffffffffu && k0 >= lo_all && k0 + 32 <= hi_all;
    uint4 v[8][NH];
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      const int64_t at = __shfl(off, 16 * (kk >> 2) + 4 * g + (kk & 3));
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const uint16_t* p = vbase + at + 16 * EV * h + EV * ln;
        if constexpr (EV == 8) {
          v[kk][h] = *reinterpret_cast<const uint4*>(p);
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(p);
          v[kk][h] = make_uint4(w.x, w.y, 0, 0);
        }
      }
    }
    floatx4 s[MT][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint16_t* p = kbase + __shfl(off, 16 * t + ln) + 8 * g;
      uint4 kf[DC];
#pragma unroll
      for (int c = 0; c < DC; ++c) kf[c] = *reinterpret_cast<const uint4*>(p + 32 * c);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        s[mt][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < DC; ++c) s[mt][t] = H::mfma16(kf[c], q[mt][c], s[mt][t]);
      }
    }
    uint32_t odd_keys = 0;
    if (!full) {
      // a value that is not finite must not meet the zero weight of a row that
      // does not see it: rows of V without a key become zero, and keys whose
      // values hold an infinity or NaN are taken out and added row by row
      uint32_t mine = 0;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const bool has = (valid >> (16 * (kk >> 2) + 4 * g + (kk & 3))) & 1u;
        bool odd = false;
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          if (!has) v[kk][h] = make_uint4(0, 0, 0, 0);
          odd = odd || H::odd(v[kk][h].x) || H::odd(v[kk][h].y) || H::odd(v[kk][h].z) || H::odd(v[kk][h].w);
        }
        const unsigned long long b = __ballot(odd);
#pragma unroll
        for (int gg = 0; gg < 4; ++gg)
          if ((b >> (16 * gg)) & 0xffffull) odd_keys |= 1u << (16 * (kk >> 2) + 4 * gg + (kk & 3));
        mine |= (odd_keys >> (16 * (kk >> 2) + 4 * g + (kk & 3)) & 1u) << kk;
      }
      if (odd_keys) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
#pragma unroll
          for (int h = 0; h < NH; ++h)
            if (mine >> kk & 1u) v[kk][h] = make_uint4(0, 0, 0, 0);
      }
    }
    uint4 p[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = s[mt][i >> 2][i & 3];
        if (!full) {
          const int kl = 16 * (i >> 2) + 4 * g + (i & 3);
          const bool see = (valid >> kl & 1u) && k0 + kl >= row_lo[mt] && k0 + kl < row_hi[mt];
          x[i] = see ? x[i] : -INFINITY;
        }
      }
      float top = x[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
      top *= a.scale_log2;
      if (__any(top > m[mt] + kBehind)) {
        top = fmaxf(top, spk::lane_xor16(top));
        top = fmaxf(top, spk::lane_xor32(top));
        const float now = fmaxf(m[mt], top);
        const float nb = now == -INFINITY ? 0.0f : now;
        const float f = m[mt] == -INFINITY ? 0.0f : exp2_fast(m[mt] - nb);
        m[mt] = now;
        base[mt] = nb;
        l[mt] = l[mt] * f;
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int e = 0; e < EV; ++e) acc[mt][h][e] *= f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = exp2_fast(__builtin_fmaf(x[i], a.scale_log2, H::kShift - base[mt]));
        l[mt] += x[i];
      }
      p[mt] = make_uint4(H::pack(x[0], x[1]), H::pack(x[2], x[3]), H::pack(x[4], x[5]), H::pack(x[6], x[7]));
    }
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        // element e of the 8 keys' pieces
        uint4 f;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          (&f.x)[w] = __builtin_amdgcn_perm((&v[2 * w + 1][h].x)[e >> 1], (&v[2 * w][h].x)[e >> 1],
                                            e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[mt][h][e] = H::mfma16(f, p[mt], acc[mt][h][e]);
      }
    while (odd_keys) {
      const int kl = __ffs(odd_keys) - 1;
      odd_keys &= odd_keys - 1;
      const uint16_t* vr = vbase + __shfl(off, kl);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t pair = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          if (w == 2 * (kl >> 4) + ((kl & 3) >> 1)) pair = (&p[mt].x)[w];
        pair = __shfl((int)pair, ln + 16 * ((kl >> 2) & 3));
        const float weight = H::widen((uint16_t)(kl & 1 ? pair >> 16 : pair));
        if (k0 + kl >= row_lo[mt] && k0 + kl < row_hi[mt]) {
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int e = 0; e < EV; ++e)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                acc[mt][h][e][i] += weight * H::widen(vr[16 * EV * h + EV * (4 * g + i) + e]);
        }
      }
    }
  }

  // join the waves, one 16-row tile at a time
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    l[mt] += spk::lane_xor16(l[mt]);
    l[mt] += spk::lane_xor32(l[mt]);
    if (mt) __syncthreads();
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < EV; e += 4)
          *reinterpret_cast<float4*>(&joint[wave][ln][16 * EV * h + EV * (4 * g + i) + e]) =
              make_float4(acc[mt][h][e][i], acc[mt][h][e + 1][i], acc[mt][h][e + 2][i], acc[mt][h][e + 3][i]);
    if (g == 0) {
      stat[wave][ln][0] = m[mt];
      stat[wave][ln][1] = l[mt];
    }
    __syncthreads();
    const int row = threadIdx.x >> 4, r = r0 + 16 * mt + row;
    if (r < rows) {
      float top = -INFINITY, sum = 0.0f, f[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[w][row][0]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        f[w] = top == -INFINITY ? 1.0f : exp2_fast(stat[w][row][0] - top);
        sum += f[w] * stat[w][row][1];
      }
      const int i = r / a.group, token = sq.first + i, head = kvh * a.group + r - i * a.group;
      const int64_t at = (int64_t)token * a.heads + head;
      float* part = a.part + (at + (int64_t)split * a.c.total_tokens * a.heads) * (D + 2);
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const int d = 64 * c + 4 * (threadIdx.x & 15);
        float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(&joint[w][row][d]);
          o[0] += f[w] * x.x;
          o[1] += f[w] * x.y;
          o[2] += f[w] * x.z;
          o[3] += f[w] * x.w;
        }
        if (a.splits[0] == 1) {
#pragma unroll
          for (int n = 0; n < 4; ++n) o[n] *= inv;
          store_out<BF, 4>(a, token, head, d, o);
        } else {
          *reinterpret_cast<float2*>(part + 2 + d) = make_float2(o[0], o[1]);
          *reinterpret_cast<float2*>(part + 4 + d) = make_float2(o[2], o[3]);
        }
      }
      if ((threadIdx.x & 15) == 0) {
        if (a.splits[0] > 1) {
          part[0] = top;
          part[1] = sum;
        } else if (a.lse) {
          a.lse[at] = sum == 0.0f ? -INFINITY : (top - H::kShift + __builtin_amdgcn_logf(sum)) * kLn2;
        }
      }
    }
  }
}

// Many rows per sequence and KV head: a workgroup of 8 waves takes 256 of the
// n * group rows, 32 to a wave, and walks the keys in tiles of KT that all
// waves share in LDS, the next tile loading while this one is used.
//
// Scores are again S^T = K Q^T (32x32x16): a lane holds 16 keys' scores of one
// row, and its weights are the B operand of O^T += V^T P^T as they are (lane
// half h supplies keys 4h..4h+3 and 8+4h..+3 of each 16).  Both A operands are
// one 16-byte LDS read of a lane.  K rows lie as in memory, their 16-byte
// pieces exchanged by the row number so that 16 rows' pieces are in different
// banks.  V is turned on the way in: a thread takes 8 keys' pieces of 4
// dimensions and writes 4 dimensions' pieces of 8 keys, in fragment order; the
// dimension of row m of output tile 4 u + e is 4 (m + 32 u) + e, which makes
// these writes (and a lane's output) contiguous.
template <int D, bool BF>
__global__ __launch_bounds__(512, 2) void paged_tiles_kernel(Attn a) {
  using H = Half<BF>;
  constexpr int KT = D == 256 ? 64 : 128;  // keys of a tile
  constexpr int KS = D / 16;               // contraction steps of the scores
  constexpr int QR = D == 256 ? 14 : KS;   // of the queries' pieces in registers, the rest in LDS
  constexpr int DT = D / 32;               // output tiles
  constexpr int CH = D / 8;                // 16-byte pieces of a row
  constexpr int RPW = 64 / CH;             // rows of K in one wave-wide load
  constexpr int KL = KT / 8 / RPW;         // such loads of a wave per tile
  constexpr int RS = 32 / RPW;             // distance of its rows: load x of 32 keys holds rows x, x + RS, ...
  constexpr int LG = D / 4;                // lanes that cover a row of V (8 bytes each)
  constexpr int GW = 64 / LG;              // groups of 8 keys of a wave
  constexpr int VW = KT / 8 / GW;          // waves that load V
  constexpr int U = KT / 64;               // lookups of a lane per tile
  // two tiles, as separate arrays: a load into one is then known not to touch the other
  __shared__ __align__(16) uint4 k0s[KT * CH / 64 * 65], k1s[KT * CH / 64 * 65], v0s[KT * CH], v1s[KT * CH];
  __shared__ __align__(16) uint4 qs[KS > QR ? (KS - QR) * 512 : 1];
  __shared__ uint32_t odd_of[3][KT / 32];  // keys of a tile with values that are not finite (tile number % 3)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 31, h = lane >> 5;
  const int kvh = blockIdx.y, split = blockIdx.x;
  int seq, tile;
  if (!find_tile(a, 1, 256, blockIdx.z, lane, &seq, &tile)) return;
  seq = __builtin_amdgcn_readfirstlane(seq);
  tile = __builtin_amdgcn_readfirstlane(tile);
  const Seq sq = spk_paged::seq_at(a.c, seq);
  const int rows = sq.n * a.group;
  const int r0 = tile * 256, r1 = min(r0 + 256, rows);
  int lo, hi, lo_all, hi_all;
  spk_paged::visible(sq, r0 / a.group, a.window, &lo, &hi_all);
  spk_paged::visible(sq, (r1 - 1) / a.group, a.window, &lo_all, &hi);
  const int keys = range_keys(a, 1, lo, hi);
  const int begin = (int)min((int64_t)(lo & ~31) + (int64_t)split * keys, (int64_t)hi);
  const int end = begin + min(keys, hi - begin);
  if (begin >= end && a.splits[1] > 1) return;

  const int r = min(r0 + 32 * wave + ln, rows - 1);
  const int ri = r / a.group, head = kvh * a.group + r - ri * a.group, token = sq.first + ri;
  int row_lo, row_hi, wave_lo, wave_hi, wave_lo_all, wave_hi_all;
  spk_paged::visible(sq, ri, a.window, &row_lo, &row_hi);
  spk_paged::visible(sq, min(r0 + 32 * wave, rows - 1) / a.group, a.window, &wave_lo, &wave_hi_all);
  spk_paged::visible(sq, min(r0 + 32 * wave + 31, rows - 1) / a.group, a.window, &wave_lo_all, &wave_hi);
  uint4 q[QR];
  {
    const uint16_t* src = a.q + token * a.qt + head * a.qh + 8 * h;
#pragma unroll
    for (int c = 0; c < QR; ++c) q[c] = *reinterpret_cast<const uint4*>(src + 16 * c);
#pragma unroll
    for (int c = QR; c < KS; ++c) qs[(c - QR) * 512 + tid] = *reinterpret_cast<const uint4*>(src + 16 * c);
  }
  floatx16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
  float m = -INFINITY, base = 0.0f, l = 0.0f;
  const int32_t* table = a.c.table + (int64_t)seq * a.c.table_stride;
  const uint16_t* kbase = a.k + kvh * a.c.head_stride;
  const uint16_t* vbase = a.v + kvh * a.c.head_stride;

  // key k0 + 64 u + lane of the tile that is loaded next
  int64_t off[U];
  unsigned long long valid[U];
  auto look_up = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = k0 + 64 * u + lane;
      off[u] = -1;
      if (key >= lo && key < end) off[u] = spk_paged::offset_in(a.c, table[spk_paged::divide(a.c.div, (uint32_t)key)], key);
      valid[u] = __ballot(off[u] >= 0);
      if (off[u] < 0) off[u] = 0;
    }
  };
  auto offset = [&](int kl) -> int64_t {  // of key kl of the tile, from its lane
    int64_t o = off[0];
    if constexpr (U == 2) o = kl & 64 ? off[1] : off[0];
    return __shfl(o, kl & 63);
  };
  auto scalar_offset = [&](int kl) -> int64_t {  // the same for a key that the whole wave asks for
    return (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)off[0], kl) |
           (int64_t)__builtin_amdgcn_readlane((int)(off[0] >> 32), kl) << 32;
  };
  uint2 vr[8];
  const int vg = GW == 1 ? wave : wave * GW + lane / LG, dc = lane % LG;  // V: group of 8 keys, piece of 4 dimensions
  auto load_k = [&](uint4* ks) {
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int x = wave * KL + i;
      const int row = x % RS + 32 * (x / RS);
      int64_t at;
      if constexpr (RPW == 2)
        at = h ? scalar_offset(row + RS) : scalar_offset(row);
      else
        at = offset(row + RS * (lane / CH));
      const uint16_t* src = kbase + at + 8 * (lane % CH);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                       (__attribute__((address_space(3))) void*)&ks[x * 65], 16, 0, 0);
    }
  };
  const int kread = (ln % RS) * 65 + (ln / RS) * CH + h;  // of this lane's row and half in the 32 keys' loads
  auto v_key = [&](int kk) { return 16 * (vg >> 1) + 8 * (kk >> 2) + 4 * (vg & 1) + (kk & 3); };
  auto load_v = [&]() {
    if (VW == 8 || wave < VW) {
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        int64_t at;
        if constexpr (GW == 1)
          at = scalar_offset(v_key(kk));
        else
          at = offset(v_key(kk));
        vr[kk] = *reinterpret_cast<const uint2*>(vbase + at + 4 * dc);
      }
    }
  };
  // Some row of the workgroup does not see the whole tile at k0.  Then a value
  // that is not finite must not meet the zero weight of a row that does not
  // see it: such elements are stored as zeros, and added row by row.
  auto partial = [&](int k0) {
    bool all = k0 >= lo_all && k0 + KT <= min(hi_all, end);
#pragma unroll
    for (int u = 0; u < U; ++u) all = all && valid[u] == ~0ull;
    return !all;
  };
  auto store_v = [&](uint4* vs, int k0, int third) {
    if (VW < 8 && wave >= VW) return;
    if (partial(k0)) {
      uint32_t odd = 0;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const int kl = v_key(kk);
        const bool has = (U == 2 && (kl & 64) ? valid[U - 1] : valid[0]) >> (kl & 63) & 1ull;
        if (!has) vr[kk] = make_uint2(0, 0);
        if (H::odd(vr[kk].x) || H::odd(vr[kk].y)) odd |= 1u << kk;
        vr[kk] = make_uint2(H::finite(vr[kk].x), H::finite(vr[kk].y));
      }
      while (odd) {
        const int kl = v_key(__ffs(odd) - 1);
        odd &= odd - 1;
        atomicOr(&odd_of[third][kl >> 5], 1u << (kl & 31));
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint4 f;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        (&f.x)[w] = __builtin_amdgcn_perm((&vr[2 * w + 1].x)[e >> 1], (&vr[2 * w].x)[e >> 1],
                                          e & 1 ? 0x07060302u : 0x05040100u);
      const int t = D >= 128 ? e + 4 * (dc / 32) : e >> 1, row = D >= 128 ? dc % 32 : dc + 16 * (e & 1);
      vs[((vg >> 1) * DT + t) * 64 + row + 32 * (vg & 1)] = f;
    }
  };
  auto dim_of = [&](int t, int row) { return D >= 128 ? 4 * (row + 32 * (t >> 2)) + (t & 3) : 4 * (row & 15) + 2 * t + (row >> 4); };

  if (tid < 3 * (KT / 32)) odd_of[tid / (KT / 32)][tid % (KT / 32)] = 0;
  int third = 0;
  unsigned long long now[U];
  bool part = true;
  auto step = [&](int k0, uint4* ks, uint4* vs, uint4* ks_next, uint4* vs_next) __attribute__((always_inline)) {
    const bool more = k0 + KT < end;
    const int after = third == 2 ? 0 : third + 1;
    part = partial(k0);
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = valid[u];
    if (tid < KT / 32) odd_of[after == 2 ? 0 : after + 1][tid] = 0;  // the tile before this one's
    if (more) {
      look_up(k0 + KT);
      load_k(ks_next);
    }
#pragma unroll 1
    for (int j = 0; j < KT / 32; ++j) {
      const int kj = k0 + 32 * j;
      if (j == KT / 32 - 1 && more) load_v();
      if (kj >= min(wave_hi, end) || kj + 32 <= wave_lo) continue;
      const uint32_t has = (uint32_t)((U == 2 && j > 1 ? now[U - 1] : now[0]) >> (32 * (j & 1)));
      const bool full = has == 0xffffffffu && kj >= wave_lo_all && kj + 32 <= wave_hi_all;
      floatx16 s;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
      for (int c = 0; c < KS; ++c) s = H::mfma32(ks[j * RS * 65 + kread + 2 * c], c < QR ? q[c] : qs[(c - QR) * 512 + tid], s);
      if (!full) {
        // bit n: this row sees key n of the 32; shifted so that a lane's keys are at constant places
        const int first = min(max(row_lo - kj, 0), 31), last = min(max(row_hi - kj, 0), 32);
        uint32_t see = row_lo - kj > 31 || last == 0 ? 0u : has & (0xffffffffu << first) & (0xffffffffu >> (32 - last));
        see >>= 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = see >> (8 * (i >> 2) + (i & 3)) & 1u ? s[i] : -INFINITY;
      }
      float top = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
      top *= a.scale_log2;
      if (__any(top > m + kBehind)) {
        top = fmaxf(top, spk::lane_xor32(top));
        const float next = fmaxf(m, top);
        const float nb = next == -INFINITY ? 0.0f : next;
        const float f = m == -INFINITY ? 0.0f : exp2_fast(m - nb);
        m = next;
        base = nb;
        l *= f;
#pragma unroll
        for (int t = 0; t < DT; ++t) acc[t] *= f;
      }
      uint4 p[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = exp2_fast(__builtin_fmaf(s[i], a.scale_log2, H::kShift - base));
        l += s[i];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        p[i] = make_uint4(H::pack(s[8 * i], s[8 * i + 1]), H::pack(s[8 * i + 2], s[8 * i + 3]),
                          H::pack(s[8 * i + 4], s[8 * i + 5]), H::pack(s[8 * i + 6], s[8 * i + 7]));
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < DT; ++t) acc[t] = H::mfma32(vs[((2 * j + i) * DT + t) * 64 + lane], p[i], acc[t]);
      if (part) {
        uint32_t odd = __builtin_amdgcn_readfirstlane(odd_of[third][j]);
        while (odd) {
          const int kl = __ffs(odd) - 1;
          odd &= odd - 1;
          const uint16_t* row = vbase + spk_paged::offset_of(a.c, seq, kj + kl);
          const uint4 quad = kl & 16 ? p[1] : p[0];
          uint32_t pair = kl & 8 ? (kl & 2 ? quad.w : quad.z) : (kl & 2 ? quad.y : quad.x);
          pair = __shfl((int)pair, ln + 32 * ((kl >> 2) & 1));
          const float weight = H::widen((uint16_t)(kl & 1 ? pair >> 16 : pair));
          if (kj + kl >= row_lo && kj + kl < row_hi) {
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const uint16_t x = row[dim_of(t, 8 * (i >> 2) + 4 * h + (i & 3))];
                if (H::odd(x)) acc[t][i] += weight * H::widen(x);
                __builtin_amdgcn_sched_barrier(0);  // one at a time: this path takes no registers from the others
              }
          }
        }
      }
    }
    if (more) {
      store_v(vs_next, k0 + KT, after);
    }
    third = after;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the keys' loads into LDS
    __syncthreads();
  };
  if (begin < end) {
    look_up(begin);
    load_k(k0s);
    load_v();
    __syncthreads();
    store_v(v0s, begin, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int k0 = begin; k0 < end; k0 += 2 * KT) {
      step(k0, k0s, v0s, k1s, v1s);
      if (k0 + KT >= end) break;
      step(k0 + KT, k1s, v1s, k0s, v0s);
    }
  }

  l += spk::lane_xor32(l);
  if (r0 + 32 * wave + ln >= rows) return;
  const int64_t at = (int64_t)token * a.heads + head;
  if (a.splits[1] > 1) {
    float* part = a.part + (at + (int64_t)split * a.c.total_tokens * a.heads) * (D + 2);
    if (h == 0) {
      part[0] = m;
      part[1] = l;
    }
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) part[2 + dim_of(t, 8 * (i >> 2) + 4 * h + (i & 3))] = acc[t][i];
    return;
  }
  if (a.lse && h == 0) a.lse[at] = l == 0.0f ? -INFINITY : (m - H::kShift + __builtin_amdgcn_logf(l)) * kLn2;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if constexpr (D >= 128) {
#pragma unroll
    for (int u = 0; u < DT / 4; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float o[4] = {acc[4 * u][i] * inv, acc[4 * u + 1][i] * inv, acc[4 * u + 2][i] * inv, acc[4 * u + 3][i] * inv};
        store_out<BF, 4>(a, token, head, dim_of(4 * u, 8 * (i >> 2) + 4 * h + (i & 3)), o);
      }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // rows m and m + 16 hold dimensions 4 (m % 16) + 2 t + 0 and 1
      const float o[4] = {acc[0][i] * inv, acc[0][i + 8] * inv, acc[1][i] * inv, acc[1][i + 8] * inv};
      store_out<BF, 4>(a, token, head, dim_of(0, 8 * (i >> 2) + 4 * h + (i & 3)), o);
    }
  }
}

// Joins the key ranges of a row: one wave per (token, head).
template <int D, bool BF>
__global__ __launch_bounds__(256) void paged_join_kernel(Attn a) {
  constexpr int N = D / 64 >= 2 ? D / 64 : 1;
  const int lane = threadIdx.x & 63;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int token = (int)(at / a.heads), head = (int)(at - (int64_t)token * a.heads);
  if (token >= a.c.total_tokens) return;
  const int s = spk_paged::seq_of_token(a.c.cu, a.c.num_seqs, token, lane);
  if (s >= a.c.num_seqs) return;
  const Seq sq = spk_paged::seq_at(a.c, s);
  if (token < sq.first || token >= sq.first + sq.n) return;
  // the ranges that the row's tile had
  const int rows = sq.n * a.group, r = (token - sq.first) * a.group + head % a.group;
  const int kind = rows >= a.many, tile_rows = a.tile_rows[kind];
  if (a.splits[kind] == 1) return;
  const int r0 = r / tile_rows * tile_rows;
  int lo, hi, x;
  spk_paged::visible(sq, r0 / a.group, a.window, &lo, &x);
  spk_paged::visible(sq, (min(r0 + tile_rows, rows) - 1) / a.group, a.window, &x, &hi);
  const int span = hi - (lo & ~31);
  const int keys = range_keys(a, kind, lo, hi);
  const int n = span <= 0 ? 0 : (int)(((int64_t)span + keys - 1) / keys);
  const int64_t step = (int64_t)a.c.total_tokens * a.heads * (D + 2);
  const float* part = a.part + at * (D + 2);
  float top = -INFINITY, sum = 0.0f, o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.0f;
  for (int j = 0; j < n; ++j) top = fmaxf(top, part[j * step]);
  for (int j = 0; j < n; ++j) {
    const float f = top == -INFINITY ? 1.0f : exp2_fast(part[j * step] - top);
    sum += f * part[j * step + 1];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] += f * part[j * step + 2 + N * lane + i];
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  uint16_t* out = a.out + token * a.ot + head * a.oh + N * lane;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float y = o[i] * inv;
    if (a.gate) {
      const float v = Half<BF>::widen(a.gate[token * a.gt + head * a.gh + N * lane + i]);
      y = y / (1.0f + exp2_fast(v * -1.44269504f));
    }
    out[i] = Half<BF>::one(y);
  }
  if (lane == 0 && a.lse)
    a.lse[at] = sum == 0.0f ? -INFINITY : (top - Half<BF>::kShift + __builtin_amdgcn_logf(sum)) * kLn2;
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

bool strides_ok(int64_t token, int64_t head) {
  return token >= 0 && head >= 0 && token % 8 == 0 && head % 8 == 0;
}

// Checks the cache and fills the kernels' view of it.
int check_cache(const SpkPagedCache& p, const char* who, Cache* c) {
  if (p.dtype != SPK_F16 && p.dtype != SPK_BF16)
    return spk::fail(SPK_ERR_ARG, "%s: dtype %d (SPK_F16 or SPK_BF16)", who, p.dtype);
  if (p.head_dim != 64 && p.head_dim != 128 && p.head_dim != 256)
    return spk::fail(SPK_ERR_SHAPE, "%s: head_dim %d (64, 128 or 256)", who, p.head_dim);
  if (p.num_kv_heads <= 0 || p.page_size <= 0 || p.num_pages <= 0 || p.max_pages <= 0 || p.num_seqs < 0 ||
      p.total_tokens < 0)
    return spk::fail(SPK_ERR_SHAPE, "%s: kv_heads %d page_size %d num_pages %d max_pages %d num_seqs %d total_tokens %d",
                     who, p.num_kv_heads, p.page_size, p.num_pages, p.max_pages, p.num_seqs, p.total_tokens);
  if ((int64_t)p.max_pages * p.page_size > INT32_MAX - 64)
    return spk::fail(SPK_ERR_SHAPE, "%s: max_pages %d of %d tokens pass 2^31 positions", who, p.max_pages, p.page_size);
  if (p.num_seqs && p.total_tokens) {
    if (!p.k_cache || !p.v_cache || !p.block_table || !p.cu_seqlens || !p.context_lens)
      return spk::fail(SPK_ERR_NULL, "%s: k_cache, v_cache, block_table, cu_seqlens or context_lens is NULL", who);
    if (!spk::aligned(p.k_cache, 16) || !spk::aligned(p.v_cache, 16) || !strides_ok(p.token_stride, p.head_stride) ||
        p.page_stride < 0 || p.page_stride % 8)
      return spk::fail(SPK_ERR_ALIGN, "%s: the cache and its strides (page %lld token %lld head %lld) must be 16-byte aligned",
                       who, (long long)p.page_stride, (long long)p.token_stride, (long long)p.head_stride);
    if (p.table_stride < p.max_pages && p.num_seqs > 1)
      return spk::fail(SPK_ERR_SHAPE, "%s: table_stride %lld < max_pages %d", who, (long long)p.table_stride, p.max_pages);
  }
  c->table = p.block_table;
  c->cu = p.cu_seqlens;
  c->ctx = p.context_lens;
  c->table_stride = p.table_stride;
  c->page_stride = p.page_stride;
  c->token_stride = p.token_stride;
  c->head_stride = p.head_stride;
  c->num_seqs = p.num_seqs;
  c->total_tokens = p.total_tokens;
  c->page_size = p.page_size;
  c->num_pages = p.num_pages;
  c->max_pages = p.max_pages;
  c->div = spk_paged::page_div((uint32_t)p.page_size);
  return SPK_OK;
}

// How a call's rows and keys are dealt to the two kernels.
struct Plan {
  int mt, one_tile, many;
  int tiles[2], splits[2], chunk[2], tile_rows[2];
};

Plan plan_of(const SpkPagedAttnArgs& p) {
  const SpkPagedCache& c = p.cache;
  const int group = p.num_q_heads / c.num_kv_heads;
  const int64_t tokens = std::min(p.max_query_len, c.total_tokens);
  const int64_t longest = tokens * group, all = (int64_t)c.total_tokens * group;
  Plan r;
  r.many = 65;
  const bool any_many = longest >= r.many;
  const int64_t few = std::min<int64_t>(longest, r.many - 1);
  r.mt = few <= 16 ? 1 : 2;
  r.tile_rows[0] = 16 * r.mt;
  r.tile_rows[1] = 256;
  r.one_tile = !any_many && few <= r.tile_rows[0];
  // sequences of few rows: all of them, unless the longest takes every row
  r.tiles[0] = r.one_tile ? c.num_seqs
               : any_many && c.num_seqs == 1
                   ? 0
                   : (int)std::min<int64_t>(all / r.tile_rows[0] + c.num_seqs, INT32_MAX);
  r.tiles[1] = any_many ? (int)std::min<int64_t>(all / 256 + std::min<int64_t>(c.num_seqs, all / r.many), INT32_MAX) : 0;
  int64_t span = std::min<int64_t>(p.max_context_len, (int64_t)c.max_pages * c.page_size);
  if (p.window > 0) span = std::min<int64_t>(span, (int64_t)p.window + tokens + 31);
  for (int kind = 0; kind < 2; ++kind) {
    const int64_t groups = (int64_t)r.tiles[kind] * c.num_kv_heads;
    const int64_t want = std::max<int64_t>(1, (kind ? 256 : 1024) / std::max<int64_t>(groups, 1));
    const int64_t least = kind ? 4 : 1;  // steps of 128 keys
    const int64_t steps = std::max<int64_t>(1, (span + 127) / 128);
    const int64_t per = std::max(least, (steps + want - 1) / want);
    r.chunk[kind] = (int)(128 * per);
    r.splits[kind] = r.tiles[kind] ? (int)((steps + per - 1) / per) : 1;
  }
  return r;
}

int check_attn(const SpkPagedAttnArgs* p, Cache* c) {
  if (!p) return spk::fail(SPK_ERR_NULL, "spk_paged_attention: NULL args");
  if (const int rc = check_cache(p->cache, "spk_paged_attention", c)) return rc;
  if (p->num_q_heads <= 0 || p->num_q_heads % p->cache.num_kv_heads)
    return spk::fail(SPK_ERR_SHAPE, "spk_paged_attention: %d query heads over %d KV heads", p->num_q_heads,
                     p->cache.num_kv_heads);
  if (!(p->scale >= 0.0f) || p->scale > 1e30f)
    return spk::fail(SPK_ERR_ARG, "spk_paged_attention: scale %g (positive, or 0 for 1/sqrt(head_dim))", (double)p->scale);
  if (p->max_query_len < 0 || p->max_context_len < 0 || p->window < 0)
    return spk::fail(SPK_ERR_SHAPE, "spk_paged_attention: max_query_len %d max_context_len %d window %d",
                     p->max_query_len, p->max_context_len, p->window);
  if ((int64_t)p->cache.total_tokens * p->num_q_heads > INT32_MAX - 65536)
    return spk::fail(SPK_ERR_SHAPE, "spk_paged_attention: %d tokens of %d heads", p->cache.total_tokens, p->num_q_heads);
  return SPK_OK;
}

size_t workspace_of(const SpkPagedAttnArgs& p) {
  const Plan r = plan_of(p);
  const int splits = std::max(r.splits[0], r.splits[1]);
  if (splits <= 1) return 0;
  return (size_t)splits * p.cache.total_tokens * p.num_q_heads * (p.cache.head_dim + 2) * sizeof(float);
}

template <int D, bool BF>
void launch_attn(const Attn& a, const Plan& r, hipStream_t s) {
  const dim3 grid(r.splits[0], a.kv_heads, r.tiles[0]);
  if (r.tiles[0] && r.mt == 1)
    hipLaunchKernelGGL((paged_rows_kernel<D, 1, BF>), grid, dim3(256), 0, s, a);
  else if (r.tiles[0])
    hipLaunchKernelGGL((paged_rows_kernel<D, 2, BF>), grid, dim3(256), 0, s, a);
  if (r.tiles[1])
    hipLaunchKernelGGL((paged_tiles_kernel<D, BF>), dim3(r.splits[1], a.kv_heads, r.tiles[1]), dim3(512), 0, s, a);
  if (r.splits[0] > 1 || r.splits[1] > 1) {
    const int64_t rows = (int64_t)a.c.total_tokens * a.heads;
    hipLaunchKernelGGL((paged_join_kernel<D, BF>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
  }
}

template <int D, bool BF>
void launch_mrope(const Mrope& a, bool adjacent, hipStream_t s) {
  const dim3 grid((a.c.total_tokens + 3) / 4);
  if (adjacent)
    hipLaunchKernelGGL((mrope_append_kernel<D, BF, true>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((mrope_append_kernel<D, BF, false>), grid, dim3(256), 0, s, a);
}

}  // namespace

extern "C" int spk_mrope_append(const SpkMropeArgs* p, spk_stream_t stream) {
  const char* who = "spk_mrope_append";
  if (!p) return spk::fail(SPK_ERR_NULL, "%s: NULL args", who);
  Mrope a{};
  if (const int rc = check_cache(p->cache, who, &a.c)) return rc;
  const SpkPagedCache& c = p->cache;
  if (p->num_q_heads <= 0) return spk::fail(SPK_ERR_SHAPE, "%s: %d query heads", who, p->num_q_heads);
  if (p->rot_dim <= 0 || p->rot_dim % 16 || p->rot_dim > c.head_dim)
    return spk::fail(SPK_ERR_SHAPE, "%s: rot_dim %d (a multiple of 16 up to head_dim %d)", who, p->rot_dim, c.head_dim);
  if (p->pairing != SPK_ROPE_HALVES && p->pairing != SPK_ROPE_ADJACENT)
    return spk::fail(SPK_ERR_ARG, "%s: pairing %d", who, p->pairing);
  if (p->num_axes < 1 || p->num_axes > 4) return spk::fail(SPK_ERR_SHAPE, "%s: num_axes %d (1 to 4)", who, p->num_axes);
  if (!p->pair_axis) return spk::fail(SPK_ERR_NULL, "%s: pair_axis is NULL", who);
  for (int i = 0; i < p->rot_dim / 2; ++i) {
    if (p->pair_axis[i] >= p->num_axes)
      return spk::fail(SPK_ERR_ARG, "%s: pair_axis[%d] = %d of %d axes", who, i, p->pair_axis[i], p->num_axes);
    a.axis[i] = p->pair_axis[i];
  }
  if (p->rope_rows <= 0) return spk::fail(SPK_ERR_SHAPE, "%s: rope_rows %d", who, p->rope_rows);
  if (c.num_seqs == 0 || c.total_tokens == 0) return SPK_OK;
  if (!p->positions || !p->rope || !p->q || !p->k || !p->v || !p->q_out)
    return spk::fail(SPK_ERR_NULL, "%s: positions, rope, q, k, v or q_out is NULL", who);
  if (p->positions_stride < c.total_tokens && p->num_axes > 1)
    return spk::fail(SPK_ERR_SHAPE, "%s: positions_stride %lld < total_tokens %d", who, (long long)p->positions_stride,
                     c.total_tokens);
  const void* ptrs[] = {p->q, p->k, p->v, p->q_out, p->q_norm_w, p->k_norm_w};
  for (const void* x : ptrs)
    if (!spk::aligned(x, 16)) return spk::fail(SPK_ERR_ALIGN, "%s: q, k, v, q_out and weights must be 16-byte aligned", who);
  if (!spk::aligned(p->rope, 8)) return spk::fail(SPK_ERR_ALIGN, "%s: rope must be 8-byte aligned", who);
  if (!strides_ok(p->q_token_stride, p->q_head_stride) || !strides_ok(p->k_token_stride, p->k_head_stride) ||
      !strides_ok(p->v_token_stride, p->v_head_stride) || !strides_ok(p->out_token_stride, p->out_head_stride))
    return spk::fail(SPK_ERR_ALIGN, "%s: strides of q, k, v and q_out must be multiples of 8 elements", who);
  a.q = static_cast<const uint16_t*>(p->q);
  a.k = static_cast<const uint16_t*>(p->k);
  a.v = static_cast<const uint16_t*>(p->v);
  a.qw = static_cast<const uint16_t*>(p->q_norm_w);
  a.kw = static_cast<const uint16_t*>(p->k_norm_w);
  a.qo = static_cast<uint16_t*>(p->q_out);
  a.kc = static_cast<uint16_t*>(c.k_cache);
  a.vc = static_cast<uint16_t*>(c.v_cache);
  a.qt = p->q_token_stride;
  a.qh = p->q_head_stride;
  a.kt = p->k_token_stride;
  a.kh = p->k_head_stride;
  a.vt = p->v_token_stride;
  a.vh = p->v_head_stride;
  a.ot = p->out_token_stride;
  a.oh = p->out_head_stride;
  a.positions = p->positions;
  a.pos_stride = p->positions_stride;
  a.rope = p->rope;
  a.rope_rows = p->rope_rows;
  a.rot = p->rot_dim;
  a.heads = p->num_q_heads;
  a.kv_heads = c.num_kv_heads;
  a.eps = p->eps > 0.0f ? p->eps : 1e-6f;
  hipStream_t s = spk::to_hip(stream);
  const bool adj = p->pairing == SPK_ROPE_ADJACENT, bf = c.dtype == SPK_BF16;
  if (c.head_dim == 64)
    bf ? launch_mrope<64, true>(a, adj, s) : launch_mrope<64, false>(a, adj, s);
  else if (c.head_dim == 128)
    bf ? launch_mrope<128, true>(a, adj, s) : launch_mrope<128, false>(a, adj, s);
  else
    bf ? launch_mrope<256, true>(a, adj, s) : launch_mrope<256, false>(a, adj, s);
  return spk::check_launch(who);
}

extern "C" size_t spk_paged_attention_workspace_size(const SpkPagedAttnArgs* p) {
  Cache c;
  if (check_attn(p, &c) || p->cache.num_seqs == 0 || p->cache.total_tokens == 0) return 0;
  return workspace_of(*p);
}

extern "C" int spk_paged_attention(const SpkPagedAttnArgs* p, spk_stream_t stream) {
  const char* who = "spk_paged_attention";
  Attn a{};
  if (const int rc = check_attn(p, &a.c)) return rc;
  const SpkPagedCache& c = p->cache;
  if (c.num_seqs == 0 || c.total_tokens == 0) return SPK_OK;
  if (!p->q || !p->out) return spk::fail(SPK_ERR_NULL, "%s: q or out is NULL", who);
  if (!spk::aligned(p->q, 16) || !spk::aligned(p->out, 16) || !spk::aligned(p->gate, 16) ||
      !strides_ok(p->q_token_stride, p->q_head_stride) || !strides_ok(p->out_token_stride, p->out_head_stride) ||
      (p->gate && !strides_ok(p->gate_token_stride, p->gate_head_stride)))
    return spk::fail(SPK_ERR_ALIGN, "%s: q, gate and out and their strides must be 16-byte aligned", who);
  const Plan r = plan_of(*p);
  const size_t need = workspace_of(*p);
  if (need && (!p->workspace || p->workspace_bytes < need || !spk::aligned(p->workspace, 256)))
    return spk::fail(p->workspace ? SPK_ERR_ARG : SPK_ERR_NULL, "%s: workspace of %zu bytes, %zu needed (256-byte aligned)",
                     who, p->workspace ? p->workspace_bytes : (size_t)0, need);
  if (c.num_kv_heads > 65535 || r.tiles[0] > 65535 || r.tiles[1] > 65535)
    return spk::fail(SPK_ERR_SHAPE, "%s: %d KV heads, %d row tiles (65535 at most)", who, c.num_kv_heads,
                     std::max(r.tiles[0], r.tiles[1]));
  a.q = static_cast<const uint16_t*>(p->q);
  a.k = static_cast<const uint16_t*>(c.k_cache);
  a.v = static_cast<const uint16_t*>(c.v_cache);
  a.gate = static_cast<const uint16_t*>(p->gate);
  a.out = static_cast<uint16_t*>(p->out);
  a.lse = p->lse;
  a.part = static_cast<float*>(p->workspace);
  a.qt = p->q_token_stride;
  a.qh = p->q_head_stride;
  a.gt = p->gate_token_stride;
  a.gh = p->gate_head_stride;
  a.ot = p->out_token_stride;
  a.oh = p->out_head_stride;
  a.heads = p->num_q_heads;
  a.kv_heads = c.num_kv_heads;
  a.group = p->num_q_heads / c.num_kv_heads;
  a.window = p->window;
  for (int kind = 0; kind < 2; ++kind) {
    a.splits[kind] = r.splits[kind];
    a.chunk[kind] = r.chunk[kind];
    a.tile_rows[kind] = r.tile_rows[kind];
  }
  a.one_tile = r.one_tile;
  a.many = r.many;
  const float scale = p->scale != 0.0f ? p->scale : 1.0f / std::sqrt((float)c.head_dim);
  a.scale_log2 = scale * 1.44269504088896341f;
  hipStream_t s = spk::to_hip(stream);
  const bool bf = c.dtype == SPK_BF16;
  if (c.head_dim == 64)
    bf ? launch_attn<64, true>(a, r, s) : launch_attn<64, false>(a, r, s);
  else if (c.head_dim == 128)
    bf ? launch_attn<128, true>(a, r, s) : launch_attn<128, false>(a, r, s);
  else
    bf ? launch_attn<256, true>(a, r, s) : launch_attn<256, false>(a, r, s);
  return spk::check_launch(who);
}
