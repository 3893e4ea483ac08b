// paged.hip -- a serving step over a paged key/value cache: rotary positions
// with several axes and the store into the pages (spk_mrope_append), and the
// attention of each sequence's new tokens over its pages
// (spk_paged_attention).
#include <algorithm>
#include <cmath>

#include "capi_common.hpp"
#include "numerics.hpp"
#include "paged.hpp"
#include "paged_deal.hpp"

namespace {

using spk_paged::Cache;
using spk_paged::Plan;
using spk_paged::Seq;
using spk_paged::Share;

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

// Both halfwords less one, no lower than zero.
__device__ __forceinline__ uint32_t step_down(uint32_t u) {
  typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(__builtin_bit_cast(ushort2_t, u), ushort2_t{1, 1}));
}

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
  // Two numbers >= 0, each rounded toward zero and one step further: what is left
  // of a number is then larger than zero wherever the rounded one is, so that
  // both parts of a weight give an infinity its sign.  Rounded to nearest, what is
  // left may be zero or less, and a row that sees an infinity got NaN.
  static __device__ __forceinline__ uint32_t below(float a, float b) {
    return step_down(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b)));
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
  static __device__ __forceinline__ uint32_t below(float a, float b) {
    return step_down(__builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u));
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

// A load of what is read once.
__device__ __forceinline__ uint4 load_once(const uint16_t* p) {
  typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(p)));
}

// One wave per token.  D / 16 lanes hold a head, 16 elements each: chunks of 8
// that rotate together (HALVES: chunk j and j + rot/16; ADJACENT: the pairs
// lie inside a chunk), so the angles of a lane are the same for every head of
// the token and are read once.
//
// What bounds it: memory.  32,768 tokens of 16 + 4 + 4 heads of 128 take 107 us for
// 405 MB read and written, 3.8 TB/s (a plain copy reaches 5.1); a lane's next row
// loaded while it turns one costs registers that other waves' loads need (115
// us).  Rows are read past the caches' replacement: 120 us from call to result for
// 129.  A decode step's is the launch.
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
    uint4 u0 = load_once(src + 8 * c0);
    uint4 u1 = load_once(src + 8 * c1);
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

struct Attn : spk_paged::Deal {
  const uint16_t *q, *k, *v, *gate;
  uint16_t* out;
  float* lse;
  float* shared;  // few rows: [shares][share_rows][D + 2], of the shares that are not alone
  int2* ranges;   // [total_tokens * heads]: where the row's first part lies in `shared` (-1: in `part`) and how many; NULL: no join
  float* part;    // many rows: [splits][total_tokens * heads][D + 2] where splits > 1
  int64_t qt, qh, gt, gh, ot, oh;
  int32_t heads;
  int32_t few;       // the join has [num_seqs][kv_heads][few] rows; 0: [total_tokens][heads]
  float scale_log2;  // scale * log2(e)
};

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kBehind = 8.0f;  // binades that the running maximum may lag

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }


// Sum over the wave, in every lane; and the inclusive running sum.  Lane swaps
// and DPP moves: an LDS permute is ten times as long, and every workgroup
// stands still for these.
__device__ __forceinline__ int wave_sum(int v) {
  v += (int)spk::lane_xor32_u((uint32_t)v);
  v += (int)spk::lane_xor16_u((uint32_t)v);
  v += (int)spk::row_ror_u<8>((uint32_t)v);
  v += (int)spk::row_ror_u<4>((uint32_t)v);
  v += (int)spk::row_ror_u<2>((uint32_t)v);
  v += (int)spk::row_ror_u<1>((uint32_t)v);
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
  v += spk::lane_xor32(v);
  v += spk::lane_xor16(v);
  v += __uint_as_float(spk::row_ror_u<8>(__float_as_uint(v)));
  v += __uint_as_float(spk::row_ror_u<4>(__float_as_uint(v)));
  v += __uint_as_float(spk::row_ror_u<2>(__float_as_uint(v)));
  v += __uint_as_float(spk::row_ror_u<1>(__float_as_uint(v)));
  return v;
}
__device__ __forceinline__ int wave_max(int v) {
  v = max(v, (int)spk::lane_xor32_u((uint32_t)v));
  v = max(v, (int)spk::lane_xor16_u((uint32_t)v));
  v = max(v, (int)spk::row_ror_u<8>((uint32_t)v));
  v = max(v, (int)spk::row_ror_u<4>((uint32_t)v));
  v = max(v, (int)spk::row_ror_u<2>((uint32_t)v));
  return max(v, (int)spk::row_ror_u<1>((uint32_t)v));
}
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // lane 15 of a row to the next row
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // lane 31 to the upper half
  return v;
}

// What the dealing of work does with a wave together (the lengths that it finds
// are the same in all lanes: in scalar registers from there on).
struct Wave {
  static __device__ __forceinline__ int first(int v) { return __builtin_amdgcn_readfirstlane(v); }
  static __device__ __forceinline__ int at(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
  static __device__ __forceinline__ int count(bool b) { return __popcll(__ballot(b)); }
  static __device__ __forceinline__ int sum(int v) { return wave_sum(v); }
  static __device__ __forceinline__ int max(int v) { return wave_max(v); }
  static __device__ __forceinline__ int scan(int v) { return wave_scan(v); }
};

// Tells the join where the parts of row r of a piece or tile lie.
__device__ __forceinline__ void tell(const Attn& a, const Seq& sq, int kvh, int r, int first, int ranges) {
  const int i = r / a.group;
  a.ranges[(int64_t)(sq.first + i) * a.heads + kvh * a.group + r - i * a.group] = make_int2(first, ranges);
}

// Bit n: a row that sees keys [lo, hi) sees key k0 + n, where `has` says that
// the key exists.
__device__ __forceinline__ uint32_t seen(uint32_t has, int k0, int lo, int hi) {
  const int first = lo - k0, last = hi - k0;
  if (first > 31 || last <= 0) return 0;
  return has & (0xffffffffu << max(first, 0)) & (0xffffffffu >> (32 - min(last, 32)));
}

// 16 lanes' 8-byte pieces of 4 rows (4 lanes a row) turned: lane l of the 16
// gets column l's four.
__device__ __forceinline__ uint2 transposed(const uint2* p) {
  typedef short short4_t __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(
      uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)p));
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

// Few rows per sequence and KV head.  A workgroup takes 16 of the
// n * group rows and a range of the keys; each of its 4 waves takes every
// fourth step of 32 keys by itself, straight from memory into registers (the
// rows share each K and V element, nothing is staged), and the waves' softmax
// states are joined in LDS at the end.  The next step's keys are loaded into
// the registers that the scores have used, its values into those that the
// output has: every wave has 16 to 32 KiB in flight all the time.
//
// Scores are formed transposed, S^T = K Q^T (16x16x32), so that a lane holds
// 8 keys' scores of one row: the running maximum and sum need no exchange
// while the maximum lags by less than 8 binades, and the 8 weights are
// directly the B operand of O^T += V^T P^T.  The order of the 32 keys in that
// product is free: lane group g supplies keys 4g..4g+3 and 16+4g..+3, which are the
// ones its scores are.  V's A operand (8 keys of one dimension) is made from
// 16-byte row pieces by pairing halfwords of two keys.  A weight enters as
// two 16-bit parts (value and remainder, `below`: some 20 bits together in fp16,
// 14 in bf16): the kernel waits for memory, and the second product keeps a few
// heavy keys' rounding out of the result.
//
// What bounds it: memory.  64 sequences of 300 to 16000 keys, heads of 256: 1.07 GB
// in 182 us, 5.9 TB/s, where reading alone reaches 7.1; one sequence of 130,001 keys:
// 96 us, 5.5 TB/s.  Values are loaded past the caches' replacement (they are
// read once); the keys, whose rows' other halves come later, are not.
template <int D, bool BF>
__global__ __launch_bounds__(256, 2) void paged_rows_kernel(Attn a) {
  using H = Half<BF>;
  constexpr int DC = D / 32;             // contraction steps of the scores
  constexpr int EV = D >= 128 ? 8 : 4;   // elements of V in one load
  constexpr int NH = D / (16 * EV);      // loads that cover a row
  constexpr int LD = D + 4;              // padded rows of the joint
  constexpr bool QL = D == 256;          // the queries lie in LDS, in fragment order
  __shared__ __align__(16) float joint[4][16][LD];
  __shared__ float stat[4][16][2];
  __shared__ __align__(16) uint4 qs[QL ? DC * 64 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ln = lane & 15, g = lane >> 4;
  Share sh;
  if (!spk_paged::find_share<Wave>(a, blockIdx.x, lane, &sh)) return;
  const int seq = sh.seq, kvh = sh.kvh;
  const Seq sq = spk_paged::seq_at(a.c, seq);
  const int rows = sq.n * a.group;
  const int r0 = sh.tile * 16;
  if (a.ranges && sh.range == 0 && threadIdx.x < 16 && r0 + (int)threadIdx.x < rows)
    tell(a, sq, kvh, r0 + threadIdx.x, sh.first * 16 + threadIdx.x, sh.ranges);
  // keys of the range that any row of the tile sees, and those that all see
  int lo, hi, lo_all, hi_all;
  spk_paged::visible(sq, r0 / a.group, a.window, &lo, &hi_all);
  spk_paged::visible(sq, (min(r0 + 16, rows) - 1) / a.group, a.window, &lo_all, &hi);
  const int begin = (int)min((int64_t)sh.lo + (int64_t)sh.range * sh.keys, (int64_t)hi);
  const int end = begin + min(sh.keys, hi - begin);

  const int32_t* table = a.c.table + (int64_t)seq * a.c.table_stride;
  const uint16_t* kbase = a.k + kvh * a.c.head_stride;
  const uint16_t* vbase = a.v + kvh * a.c.head_stride;
  // lane l asks for key k0 + l % 32; keys outside the range or without a page
  // read the pool's first row and are masked.  A step's page ids are loaded two
  // steps ahead, before the next step's keys, so that no wait for them is a
  // wait for keys or values still on their way.
  auto load_page = [&](int k0) {
    const int key = k0 + (lane & 31);
    return key >= lo && key < end ? table[spk_paged::divide(a.c.div, (uint32_t)key)] : -1;
  };
  int64_t off = 0;
  uint32_t valid = 0;
  auto look_up = [&](int k0, int page) {
    off = spk_paged::offset_in(a.c, page, k0 + (lane & 31));
    valid = (uint32_t)__ballot(off >= 0);
    if (off < 0) off = 0;
  };
  // lane l of a wave as the compiler cannot know it: the lanes asked for below
  // are then formed where they are used, not held in registers throughout
  auto here = [&]() {
    int l = lane;
    asm volatile("" : "+v"(l));
    return l;
  };
  uint4 kf[2][DC], v[8][NH];
  auto load_k = [&]() {
    const int x = here();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint16_t* p = kbase + (__shfl(off, 16 * t + (x & 15)) + 8 * (x >> 4));
#pragma unroll
      for (int c = 0; c < DC; ++c) kf[t][c] = *reinterpret_cast<const uint4*>(p + 32 * c);
    }
  };
  auto load_v = [&]() {
    const int x = here();
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      const uint16_t* p = vbase + (__shfl(off, 16 * (kk >> 2) + 4 * (x >> 4) + (kk & 3)) + EV * (x & 15));
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        if constexpr (EV == 8) {
          v[kk][h] = load_once(p + 16 * EV * h);
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(p + 16 * EV * h);
          v[kk][h] = make_uint4(w.x, w.y, 0, 0);
        }
      }
    }
  };

  int k0 = begin + 32 * wave;
  int page = -1;  // of the step after the one that is loaded
  if (k0 < end) {
    const int first = load_page(k0);
    page = load_page(k0 + 128);
    look_up(k0, first);
    load_k();
    load_v();
  }
  const int r = min(r0 + ln, rows - 1);  // this lane's row
  uint4 q[DC];
  int row_lo, row_hi;
  {
    const int i = r / a.group;
    spk_paged::visible(sq, i, a.window, &row_lo, &row_hi);
    const uint16_t* src = a.q + (sq.first + i) * a.qt + (kvh * a.group + r - i * a.group) * a.qh + 8 * g;
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      if constexpr (!QL)
        q[c] = *reinterpret_cast<const uint4*>(src + 32 * c);
      else if (c % 4 == wave)
        qs[c * 64 + lane] = *reinterpret_cast<const uint4*>(src + 32 * c);
    }
  }
  if constexpr (QL) __syncthreads();
  float m = -INFINITY, base = 0.0f, l = 0.0f;
  floatx4 acc[NH][EV];
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int e = 0; e < EV; ++e) acc[h][e] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  for (; k0 < end; k0 += 128) {
    const bool full = valid == 0xffffffffu && k0 >= lo_all && k0 + 32 <= hi_all;
    const uint32_t has = valid;
    const bool more = k0 + 128 < end;
    floatx4 s0 = floatx4{0.0f, 0.0f, 0.0f, 0.0f}, s1 = s0;
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      const uint4 qf = QL ? qs[c * 64 + lane] : q[c];
      s0 = H::mfma16(kf[0][c], qf, s0);
      s1 = H::mfma16(kf[1][c], qf, s1);
    }
    if (more) {
      look_up(k0 + 128, page);
      page = load_page(k0 + 256);
      load_k();
    }
    float w[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = s0[i];
      w[4 + i] = s1[i];
    }
    if (!full) {
      const uint32_t see = seen(has, k0, row_lo, row_hi) >> (4 * g);  // a lane's keys at constant places
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = see >> (16 * (i >> 2) + (i & 3)) & 1u ? w[i] : -INFINITY;
    }
    float top = w[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, w[i]);
    top *= a.scale_log2;
    if (__any(top > m + kBehind)) {
      top = fmaxf(top, spk::lane_xor16(top));
      top = fmaxf(top, spk::lane_xor32(top));
      const float now = fmaxf(m, top);
      const float nb = now == -INFINITY ? 0.0f : now;
      const float f = m == -INFINITY ? 0.0f : exp2_fast(m - nb);
      m = now;
      base = nb;
      l *= f;
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int e = 0; e < EV; ++e) acc[h][e] *= f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = exp2_fast(__builtin_fmaf(w[i], a.scale_log2, H::kShift - base));
      l += w[i];
    }
    uint4 p0, p1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = H::below(w[2 * i], w[2 * i + 1]);
      const float2_t x = H::unpack(u);
      (&p0.x)[i] = u;
      (&p1.x)[i] = H::pack(w[2 * i] - x.x, w[2 * i + 1] - x.y);
    }
    uint32_t odd_keys = 0;
    if (!full) {
      // a value that is not finite must not meet the zero weight of a row that
      // does not see it: rows of V without a key become zero, and keys whose
      // values hold an infinity or NaN are taken out and added row by row
      uint32_t mine = 0;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const int kl = 16 * (kk >> 2) + 4 * g + (kk & 3);
        bool odd = false;
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          if (!(has >> kl & 1u)) v[kk][h] = make_uint4(0, 0, 0, 0);
          odd = odd || H::odd(v[kk][h].x) || H::odd(v[kk][h].y) || H::odd(v[kk][h].z) || H::odd(v[kk][h].w);
        }
        const unsigned long long b = __ballot(odd);
#pragma unroll
        for (int gg = 0; gg < 4; ++gg)
          if ((b >> (16 * gg)) & 0xffffull) odd_keys |= 1u << (16 * (kk >> 2) + 4 * gg + (kk & 3));
        mine |= (odd_keys >> kl & 1u) << kk;
      }
      if (odd_keys) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
#pragma unroll
          for (int h = 0; h < NH; ++h)
            if (mine >> kk & 1u) v[kk][h] = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        // element e of the 8 keys' pieces
        uint4 f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          (&f.x)[i] = __builtin_amdgcn_perm((&v[2 * i + 1][h].x)[e >> 1], (&v[2 * i][h].x)[e >> 1],
                                            e & 1 ? 0x07060302u : 0x05040100u);
        acc[h][e] = H::mfma16(f, p0, acc[h][e]);
        acc[h][e] = H::mfma16(f, p1, acc[h][e]);
      }
    if (more) load_v();
    while (odd_keys) {
      const int kl = __ffs(odd_keys) - 1;
      odd_keys &= odd_keys - 1;
      const uint16_t* vr = vbase + max(spk_paged::offset_of(a.c, seq, k0 + kl), (int64_t)0);
      float weight = 0.0f;
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const uint4 quad = part ? p1 : p0;
        uint32_t pair = kl & 16 ? (kl & 2 ? quad.w : quad.z) : (kl & 2 ? quad.y : quad.x);
        pair = __shfl((int)pair, ln + 16 * ((kl >> 2) & 3));
        weight += H::widen((uint16_t)(kl & 1 ? pair >> 16 : pair));
      }
      if (k0 + kl >= row_lo && k0 + kl < row_hi) {
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int e = 0; e < EV; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              acc[h][e][i] += weight * H::widen(vr[16 * EV * h + EV * (4 * g + i) + e]);
              __builtin_amdgcn_sched_barrier(0);  // one at a time: this path takes no registers from the others
            }
      }
    }
  }

  // join the waves
  l += spk::lane_xor16(l);
  l += spk::lane_xor32(l);
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < EV; e += 4)
        *reinterpret_cast<float4*>(&joint[wave][ln][16 * EV * h + EV * (4 * g + i) + e]) =
            make_float4(acc[h][e][i], acc[h][e + 1][i], acc[h][e + 2][i], acc[h][e + 3][i]);
  if (g == 0) {
    stat[wave][ln][0] = m;
    stat[wave][ln][1] = l;
  }
  __syncthreads();
  const int row = threadIdx.x >> 4, rj = r0 + row;
  if (rj >= rows) return;
  float top = -INFINITY, sum = 0.0f, f[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[w][row][0]);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = top == -INFINITY ? 1.0f : exp2_fast(stat[w][row][0] - top);
    sum += f[w] * stat[w][row][1];
  }
  const int i = rj / a.group, token = sq.first + i, head = kvh * a.group + rj - i * a.group;
  const int64_t at = (int64_t)token * a.heads + head;
  float* part = a.shared + ((int64_t)blockIdx.x * 16 + row) * (D + 2);
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
    if (sh.ranges == 1) {
#pragma unroll
      for (int n = 0; n < 4; ++n) o[n] *= inv;
      store_out<BF, 4>(a, token, head, d, o);
    } else {
      *reinterpret_cast<float2*>(part + 2 + d) = make_float2(o[0], o[1]);
      *reinterpret_cast<float2*>(part + 4 + d) = make_float2(o[2], o[3]);
    }
  }
  if ((threadIdx.x & 15) == 0) {
    if (sh.ranges > 1) {
      part[0] = top;
      part[1] = sum;
    } else if (a.lse) {
      a.lse[at] = sum == 0.0f ? -INFINITY : (top - H::kShift + __builtin_amdgcn_logf(sum)) * kLn2;
    }
  }
}

// A middle number of rows per sequence and KV head (17 .. 128, in pieces of 64: a
// few drafted tokens): too many for the registers of one wave beside the keys on their
// way, too few to be bound by anything but memory.  A workgroup takes 64 rows,
// 16 to each of its 4 waves, and all waves read every step of 32 keys from
// LDS.  A wave loads its part of a step's keys and values two steps ahead, into
// registers, two steps lie in LDS, and two workgroups share a CU.
// The waves have their own rows, so nothing is joined.
//
// The arithmetic is paged_rows_kernel's.  Rows lie in LDS as in memory, one
// load's 1 KiB (rows x, x + RS, ...) apart by 16 bytes more for the keys, whose
// rows 0..7 are read side by side, and by 32 for the values, which are read
// by the transposing load: 16 lanes take 4 keys' pieces of 16 dimensions and
// get 4 keys of a dimension each.
//
// What bounds it: 16 sequences with 9 tokens of 4 heads (36 rows), heads of 256, take
// 44 us for 168 MB, 3.8 TB/s.  Matrix instructions run 9% of the time and LDS
// reads 14%; some 10 us are the way to the first keys (lengths, shares, page ids),
// the rest is memory.  Heads of 256 fill the registers: 20 bytes of a lane's
// addresses lie in memory, outside the products.
template <int D, bool BF>
__global__ __launch_bounds__(256, 2) void paged_mid_kernel(Attn a) {
  using H = Half<BF>;
  constexpr int DC = D / 32;      // contraction steps of the scores
  constexpr int DT = D / 16;      // output tiles
  constexpr int CH = D / 8;       // 16-byte pieces of a row
  constexpr int RPW = 64 / CH;    // rows of one load
  constexpr int RS = 32 / RPW;    // loads of 32 keys, and the distance of a load's rows
  constexpr int LW = RS / 4;      // loads of a wave
  __shared__ __align__(16) uint4 kss[2][RS * 65], vss[2][RS * 66];
  __shared__ __align__(16) uint32_t there[2][4];  // per step and wave: its rows' keys that exist
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 15, g = lane >> 4;
  Share sh;
  if (!spk_paged::find_share<Wave>(a, blockIdx.x, lane, &sh)) return;
  const int seq = sh.seq, kvh = sh.kvh;
  const Seq sq = spk_paged::seq_at(a.c, seq);
  const int rows = sq.n * a.group;
  const int r0 = sh.tile * 64;
  if (a.ranges && sh.range == 0 && tid < 64 && r0 + tid < rows) tell(a, sq, kvh, r0 + tid, sh.first * 64 + tid, sh.ranges);
  int lo, hi, lo_all, hi_all, x;
  spk_paged::visible(sq, r0 / a.group, a.window, &lo, &x);
  spk_paged::visible(sq, (min(r0 + 64, rows) - 1) / a.group, a.window, &x, &hi);
  const int begin = (int)min((int64_t)sh.lo + (int64_t)sh.range * sh.keys, (int64_t)hi);
  const int end = begin + min(sh.keys, hi - begin);

  // the row of this lane; the keys that all rows of the wave see
  const int r = min(r0 + 16 * wave + ln, rows - 1);
  const int ri = r / a.group, token = sq.first + ri, head = kvh * a.group + r - ri * a.group;
  int row_lo, row_hi;
  spk_paged::visible(sq, ri, a.window, &row_lo, &row_hi);
  spk_paged::visible(sq, min(r0 + 16 * wave, rows - 1) / a.group, a.window, &x, &hi_all);
  spk_paged::visible(sq, min(r0 + 16 * wave + 15, rows - 1) / a.group, a.window, &lo_all, &x);
  const bool idle = r0 + 16 * wave >= rows;
  uint4 q[DC];
  {
    const uint16_t* src = a.q + token * a.qt + head * a.qh + 8 * g;
#pragma unroll
    for (int c = 0; c < DC; ++c) q[c] = *reinterpret_cast<const uint4*>(src + 32 * c);
  }
  const int32_t* table = a.c.table + (int64_t)seq * a.c.table_stride;
  const uint16_t* kbase = a.k + kvh * a.c.head_stride;
  const uint16_t* vbase = a.v + kvh * a.c.head_stride;
  // A wave's part of a step, on its way, and the page ids of the one that
  // takes its place two steps on: vector loads return in order, so an id
  // is asked for before everything that may still be under way when it is used.
  struct Part {
    uint4 k[LW], v[LW];
    int page[LW];
    uint32_t mine;  // its keys that exist
  };
  const int own = wave * LW + RS * (lane / CH);  // this lane's first row of a step
  auto look_up = [&](int k0, Part& p) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LW; ++i)
      p.page[i] = table[spk_paged::divide(a.c.div, (uint32_t)min(max(k0 + own + i, lo), end - 1))];
  };
  auto load = [&](int k0, Part& p) __attribute__((always_inline)) {
    p.mine = 0;
    int64_t at[LW];
#pragma unroll
    for (int i = 0; i < LW; ++i) {
      const int key = k0 + own + i;
      const int64_t o = spk_paged::offset_in(a.c, p.page[i], key);
      const bool there = key >= lo && key < end && o >= 0;
      at[i] = there ? o : 0;  // a key without a place reads the pool's first row and is masked
      const unsigned long long b = __ballot(there);
#pragma unroll
      for (int j = 0; j < RPW; ++j) p.mine |= (uint32_t)(b >> (CH * j) & 1) << (wave * LW + i + RS * j);
    }
    look_up(k0 + 64, p);
#pragma unroll
    for (int i = 0; i < LW; ++i) {
      p.k[i] = load_once(kbase + (at[i] + 8 * (lane % CH)));
      p.v[i] = load_once(vbase + (at[i] + 8 * (lane % CH)));
    }
  };
  floatx4 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, base = 0.0f, l = 0.0f;
  constexpr int K16 = CH * 16 / RS;                       // 16 rows on, in 16-byte pieces
  const int kread = (ln % RS) * 65 + (ln / RS) * CH + g;  // + 4 c
  const int vrow = 4 * g + (ln >> 2);                     // of the transposing load
  const int vread = (vrow % RS) * 132 + (vrow / RS) * 2 * CH + (ln & 3);  // in 8-byte pieces, + 4 t

  auto step = [&](int k0, int buf, Part& p) __attribute__((always_inline)) {
    uint4* ks = kss[buf];
    uint4* vs = vss[buf];
#pragma unroll
    for (int i = 0; i < LW; ++i) {
      ks[(wave * LW + i) * 65 + lane] = p.k[i];
      vs[(wave * LW + i) * 66 + lane] = p.v[i];
    }
    if (lane == 0) there[buf][wave] = p.mine;
    load(k0 + 64, p);
    // every wave's part is there, and every wave has done with the step before
    // the last, whose place this one's took
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (idle || k0 >= end) return;
    const uint4 four = *reinterpret_cast<const uint4*>(&there[buf][0]);
    const uint32_t has = __builtin_amdgcn_readfirstlane(four.x | four.y | four.z | four.w);
    const bool full = has == 0xffffffffu && k0 >= lo_all && k0 + 32 <= min(hi_all, end);
    floatx4 s0 = floatx4{0.0f, 0.0f, 0.0f, 0.0f}, s1 = s0;
    constexpr int KA = DC < 4 ? DC : 4;  // pieces of the keys that are read ahead
    uint4 kf[2][KA];
#pragma unroll
    for (int c = 0; c < KA; ++c) {
      kf[0][c] = ks[kread + 4 * c];
      kf[1][c] = ks[kread + K16 + 4 * c];
    }
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      const uint4 u = kf[0][c % KA], v = kf[1][c % KA];
      if (c + KA < DC) {
        kf[0][c % KA] = ks[kread + 4 * (c + KA)];
        kf[1][c % KA] = ks[kread + K16 + 4 * (c + KA)];
      }
      __builtin_amdgcn_sched_barrier(0);  // the reads go out before the products that wait for earlier ones
      s0 = H::mfma16(u, q[c], s0);
      s1 = H::mfma16(v, q[c], s1);
    }
    float w[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = s0[i];
      w[4 + i] = s1[i];
    }
    if (!full) {
      const uint32_t see = seen(has, k0, row_lo, row_hi) >> (4 * g);  // a lane's keys at constant places
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = see >> (16 * (i >> 2) + (i & 3)) & 1u ? w[i] : -INFINITY;
    }
    float top = w[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, w[i]);
    top *= a.scale_log2;
    if (__any(top > m + kBehind)) {
      top = fmaxf(top, spk::lane_xor16(top));
      top = fmaxf(top, spk::lane_xor32(top));
      const float now = fmaxf(m, top);
      const float nb = now == -INFINITY ? 0.0f : now;
      const float f = m == -INFINITY ? 0.0f : exp2_fast(m - nb);
      m = now;
      base = nb;
      l *= f;
#pragma unroll
      for (int t = 0; t < DT; ++t) acc[t] *= f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = exp2_fast(__builtin_fmaf(w[i], a.scale_log2, H::kShift - base));
      l += w[i];
    }
    uint4 p0, p1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = H::below(w[2 * i], w[2 * i + 1]);
      const float2_t v = H::unpack(u);
      (&p0.x)[i] = u;
      (&p1.x)[i] = H::pack(w[2 * i] - v.x, w[2 * i + 1] - v.y);
    }
    auto values = [&](int t) {  // 8 keys of dimension 16 t + ln
      const auto* at = reinterpret_cast<const uint2*>(vs) + vread + 4 * t;
      const uint2 u = transposed(at), v = transposed(at + 2 * K16);
      return make_uint4(u.x, u.y, v.x, v.y);
    };
    // as in paged_rows_kernel: no value that is not finite meets a zero weight
    const uint32_t exists = has >> (4 * g);
    uint32_t odd = 0;  // bit i: of this lane's keys 2 i and 2 i + 1
    auto clean = [&](uint4& f) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t two = exists >> (16 * (i >> 1) + 2 * (i & 1));
        const uint32_t u = (&f.x)[i] & ((two & 1u ? 0xffffu : 0u) | (two & 2u ? 0xffff0000u : 0u));
        if (H::odd(u)) odd |= 1u << i;
        (&f.x)[i] = H::finite(u);
      }
    };
    constexpr int A = 4;  // tiles whose values are read ahead
    uint4 f[A];
#pragma unroll
    for (int t = 0; t < A; ++t) f[t] = values(t);
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      uint4 u = f[t % A];
      if (t + A < DT) f[t % A] = values(t + A);
      if (!full) clean(u);
      acc[t] = H::mfma16(u, p0, acc[t]);
      acc[t] = H::mfma16(u, p1, acc[t]);
    }
    if (full) return;
    uint32_t odd_keys = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned long long b = __ballot(odd >> i & 1u);
#pragma unroll
      for (int gg = 0; gg < 4; ++gg)
        if ((b >> (16 * gg)) & 0xffffull) odd_keys |= 3u << (16 * (i >> 1) + 4 * gg + 2 * (i & 1));
    }
    while (odd_keys) {
      const int kl = __ffs(odd_keys) - 1;
      odd_keys &= odd_keys - 1;
      if (!(has >> kl & 1u)) continue;
      const uint16_t* row = a.v + kvh * a.c.head_stride + spk_paged::offset_of(a.c, seq, k0 + kl);
      float weight = 0.0f;
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const uint4 quad = part ? p1 : p0;
        uint32_t pair = kl & 16 ? (kl & 2 ? quad.w : quad.z) : (kl & 2 ? quad.y : quad.x);
        pair = __shfl((int)pair, ln + 16 * ((kl >> 2) & 3));
        weight += H::widen((uint16_t)(kl & 1 ? pair >> 16 : pair));
      }
      if (k0 + kl >= row_lo && k0 + kl < row_hi) {
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint16_t u = row[16 * t + 4 * g + i];
            if (H::odd(u)) acc[t][i] += weight * H::widen(u);
            __builtin_amdgcn_sched_barrier(0);  // one at a time: this path takes no registers from the others
          }
      }
    }
  };
  if (begin < end) {
    Part pa, pb;
    look_up(begin, pa);
    look_up(begin + 32, pb);
    load(begin, pa);
    load(begin + 32, pb);
    // the second step may lie past the end and is empty then: with a way out
    // between the two, the wait for the older part would be one for both
    for (int k0 = begin; k0 < end; k0 += 64) {
      step(k0, 0, pa);
      step(k0 + 32, 1, pb);
    }
  }

  l += spk::lane_xor16(l);
  l += spk::lane_xor32(l);
  if (r0 + 16 * wave + ln >= rows) return;
  const int64_t at = (int64_t)token * a.heads + head;
  if (sh.ranges > 1) {
    float* part = a.shared + ((int64_t)blockIdx.x * 64 + 16 * wave + ln) * (D + 2);
    if (g == 0) {
      part[0] = m;
      part[1] = l;
    }
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      *reinterpret_cast<float2*>(part + 2 + 16 * t + 4 * g) = make_float2(acc[t][0], acc[t][1]);
      *reinterpret_cast<float2*>(part + 4 + 16 * t + 4 * g) = make_float2(acc[t][2], acc[t][3]);
    }
    return;
  }
  if (a.lse && g == 0) a.lse[at] = l == 0.0f ? -INFINITY : (m - H::kShift + __builtin_amdgcn_logf(l)) * kLn2;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int t = 0; t < DT; ++t) {
    const float o[4] = {acc[t][0] * inv, acc[t][1] * inv, acc[t][2] * inv, acc[t][3] * inv};
    store_out<BF, 4>(a, token, head, 16 * t + 4 * g, o);
  }
}

// use(c, read(c)) for c below N, with the reads AHEAD of their use, or as the
// compiler has them.
template <int N, int AHEAD, typename Read, typename Use>
__device__ __forceinline__ void in_turn(Read read, Use use) {
  if constexpr (AHEAD == 0) {
#pragma unroll
    for (int c = 0; c < N; ++c) use(c, read(c));
  } else {
    uint4 f[N];
#pragma unroll
    for (int c = 0; c < (AHEAD < N ? AHEAD : N); ++c) f[c] = read(c);
    __builtin_amdgcn_sched_barrier(6);  // only scalar and vector arithmetic may move past it
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if (c + AHEAD < N) f[c + AHEAD] = read(c + AHEAD);
      use(c, f[c]);
      __builtin_amdgcn_sched_barrier(6);
    }
  }
}

// Many rows per sequence and KV head: a workgroup of 8 waves takes 256 of the
// n * group rows, 32 to a wave, and walks the keys in tiles of KT (16 KiB of
// keys) that all waves share in LDS.  Loads go straight into LDS, the keys' two
// tiles ahead and the values' three: a tile takes less time than a load.
//
// Scores are again S^T = K Q^T (32x32x16): a lane holds 16 keys' scores of one
// row, and its weights are the B operand of O^T += V^T P^T as they are (lane
// half h supplies keys 4h..4h+3 and 8+4h..+3 of each 16).  Both A operands are
// one 16-byte LDS read of a lane.  K rows lie as in memory, one load's 1 KiB
// (rows x, x + RS, ...) apart by 16 bytes more, so that rows read side by side
// are in different banks.  V is turned in LDS a tile before it is used: a
// thread reads 2 dimensions of 8 keys and writes 8 keys of each, in fragment
// order; the dimension of row m of output tile 2 u + e is 2 (m + 32 u) + e,
// which makes these writes (and a lane's output) contiguous.
//
// A weight enters the product with V as one 16-bit value, half a step off at
// most; the sum of weights has it unrounded.  In two parts, as the other kernels
// have them, the product is twice as many matrix instructions: 453 us for 337 with
// the first shape below, 249 for 191 with the second, for an error of 2.1e-4 instead
// of 2.8e-4 (fp16, 2-norm against 64 bits) and 1.65e-3 instead of 2.2e-3 (bf16),
// most of which is the result's own rounding.
//
// What bounds it: one workgroup of 8 waves to a CU (a wave's outputs and queries
// fill its registers).  2048 tokens at 16384 keys, heads of 256: 295 to 325 us
// without the join (one chip's clock under load and another's), 790 to 870
// TFLOP/s; matrix instructions run 37% of the time at some 2 GHz, LDS reads 25%,
// waves wait for one or the other in half of theirs, as no registers are left to
// read ahead.  Six ragged prompts, heads of 128: 167 to 180 us, 600 to 650
// TFLOP/s: a step's exponentials take as long as its matrix instructions, and the
// longest tile alone is three quarters of the time.
template <int D, bool BF>
__global__ __launch_bounds__(512, 2) void paged_tiles_kernel(Attn a) {
  using H = Half<BF>;
  constexpr int KT = 8192 / D;             // keys of a tile
  constexpr int KS = D / 16;               // contraction steps of the scores
  constexpr int QR = D == 256 ? 14 : KS;   // of the queries' pieces in registers, the rest in LDS
  constexpr int DT = D / 32;               // output tiles
  constexpr int CH = D / 8;                // 16-byte pieces of a row
  constexpr int RPW = 64 / CH;             // rows of K in one wave-wide load, of which a wave has two
  constexpr int RS = 32 / RPW;             // distance of its rows: load x of 32 keys holds rows x, x + RS, ...
  constexpr int LG = D / 2;                // threads that cover a row of V
  constexpr int U = KT > 64 ? 2 : 1;       // lookups of a lane per tile
  constexpr int NB = D == 256 ? 1 : 2;     // blocks of 32 keys at a time
  // LDS reads ahead of the matrix instruction that uses them.  Heads of 256 have
  // no registers left for it: the kernel keeps 28 bytes of a lane's address
  // arithmetic in memory as it is, outside the products, and 44 with reads 2 ahead,
  // which take 321 us for 317.  With heads of 128, 4 ahead take 181 us for 189.
  constexpr int AHEAD = D == 256 ? 0 : 4;
  // keys, values as they come: three tiles, as separate arrays: a load into one is then known not to touch the others
  __shared__ __align__(16) uint4 ka[16 * 65], kb[16 * 65], kc[16 * 65], ra[1024], rb[1024], rc[1024];
  __shared__ __align__(16) uint4 vss[2 * 1024];  // values turned: two tiles
  __shared__ __align__(16) uint4 qs[KS > QR ? (KS - QR) * 512 : 1];
  __shared__ uint32_t odd_of[3][KT / 32];  // keys of a tile with values that are not finite (tile number % 3)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 31, h = lane >> 5;
  // Workgroups go to the 8 XCDs in turn.  Every 8 tiles another range goes to an
  // XCD, or one has all the short last ranges (2048 tokens at 16384 keys: 335 us ->
  // 316; with another at every tile, which shares fewer keys in an L2, 324).
  const int kvh = blockIdx.y, split = (blockIdx.x + (blockIdx.z >> 3)) % gridDim.x;
  int seq, tile;
  if (!spk_paged::find_tile<Wave>(a, blockIdx.z, gridDim.z - 1, lane, &seq, &tile)) return;
  seq = __builtin_amdgcn_readfirstlane(seq);
  tile = __builtin_amdgcn_readfirstlane(tile);
  const Seq sq = spk_paged::seq_at(a.c, seq);
  const int rows = sq.n * a.group;
  const int r0 = tile * 256, r1 = min(r0 + 256, rows);
  int lo, hi, lo_all, hi_all;
  spk_paged::visible(sq, r0 / a.group, a.window, &lo, &hi_all);
  spk_paged::visible(sq, (r1 - 1) / a.group, a.window, &lo_all, &hi);
  const int keys = spk_paged::range_keys(a, lo, hi);
  const int begin = (int)min((int64_t)(lo & ~31) + (int64_t)split * keys, (int64_t)hi);
  const int end = begin + min(keys, hi - begin);
  if (begin >= end && split > 0) return;
  const bool alone = hi - (lo & ~31) <= keys;  // the tile's one range
  if (a.ranges && split == 0 && tid < r1 - r0)
    tell(a, sq, kvh, r0 + tid, -1, alone ? 1 : (hi - (lo & ~31) + keys - 1) / keys);

  const int r = min(r0 + 32 * wave + ln, rows - 1);
  int row_lo, row_hi, wave_lo, wave_hi, wave_lo_all, wave_hi_all;
  spk_paged::visible(sq, r / a.group, a.window, &row_lo, &row_hi);
  spk_paged::visible(sq, min(r0 + 32 * wave, rows - 1) / a.group, a.window, &wave_lo, &wave_hi_all);
  spk_paged::visible(sq, min(r0 + 32 * wave + 31, rows - 1) / a.group, a.window, &wave_lo_all, &wave_hi);
  wave_hi = min(wave_hi, end);
  uint4 q[QR];
  {
    const int i = r / a.group;
    const uint16_t* src = a.q + (sq.first + i) * a.qt + (kvh * a.group + r - i * a.group) * a.qh + 8 * h;
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
  float m = -INFINITY, shift = H::kShift, l = 0.0f;  // shift: less the maximum that the weights are relative to
  const int32_t* table = a.c.table + (int64_t)seq * a.c.table_stride;
  const uint16_t* vbase = a.v + kvh * a.c.head_stride;

  // Key k0 + 64 u + lane (32 keys: lane % 32) of the tile whose values are loaded
  // next; its page id was asked for a tile earlier.
  const int klane = KT == 32 ? ln : lane;
  int page[U];
  int64_t off[U];
  unsigned long long valid[U];
  auto ask = [&](int k0, int (&page)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      page[u] = table[spk_paged::divide(a.c.div, (uint32_t)min(max(k0 + 64 * u + klane, lo), end - 1))];
  };
  auto look_up = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = k0 + 64 * u + klane;
      off[u] = spk_paged::offset_in(a.c, page[u], key);
      const bool there = key >= lo && key < end && off[u] >= 0;
      valid[u] = __ballot(there);
      off[u] = there ? off[u] : 0;  // a key without a place reads the pool's first row and is masked
    }
  };
  // a wave's two loads of a tile, its rows at `off`, into `to`, loads `apart`;
  // lane l brings piece l % CH ^ other of its row
  auto load = [&](const uint16_t* from, uint4* to, int apart, int other) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int x = wave * 2 + i, row = x % RS + 32 * (x / RS);
      int64_t at;
      if constexpr (RPW == 2) {
        const int64_t first = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)off[0], row) |
                              (int64_t)__builtin_amdgcn_readlane((int)(off[0] >> 32), row) << 32;
        const int64_t second = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)off[0], row + RS) |
                               (int64_t)__builtin_amdgcn_readlane((int)(off[0] >> 32), row + RS) << 32;
        at = h ? second : first;
      } else {
        const int kl = row + RS * (lane / CH);
        int64_t o = off[0];
        if constexpr (U == 2) o = row & 64 ? off[1] : off[0];
        at = __shfl(o, kl & 63);
      }
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + (at + 8 * (lane % CH ^ other))),
                                       (__attribute__((address_space(3))) void*)&to[x * apart], 16, 0, 0);
    }
  };
  // Rows that share a load have their halves exchanged in turn, so that 16 rows
  // read side by side are in different banks: of heads of 128 every other row,
  // of 64 every other two.
  auto swapped = [](int row) { return CH == 16 ? 8 * (row & 1) : CH == 8 ? 4 * (row >> 1 & 1) : 0; };
  const int kload = swapped(lane / CH), kswap = swapped(ln / RS);
  const int kread = (ln % RS) * 65 + (ln / RS) * CH + h;  // of this lane's row and half in the 32 keys' loads
  const int klow = kread + kswap, khigh = kread - kswap;  // its first and its second half's pieces
  // Some row of the workgroup does not see the whole tile at k0.  Then a value
  // that is not finite must not meet the zero weight of a row that does not
  // see it: such elements are turned into zeros, and added row by row.
  auto partial = [&](int k0, const unsigned long long (&exist)[U]) {
    bool all = k0 >= lo_all && k0 + KT <= min(hi_all, end);
#pragma unroll
    for (int u = 0; u < U; ++u) all = all && exist[u] == ~0ull;
    return !all;
  };
  // V: this thread's group of 8 keys, and its piece of 2 dimensions
  const int vg = LG >= 64 ? wave / (LG / 64) : tid / LG, dc = tid % LG;
  auto v_key = [&](int kk) { return 16 * (vg >> 1) + 8 * (kk >> 2) + 4 * (vg & 1) + (kk & 3); };
  auto turn = [&](const uint4* raw, uint4* vs, bool part, const unsigned long long (&exist)[U], uint32_t* odd_keys)
                  __attribute__((always_inline)) {
    uint32_t vr[8];
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      const int kl = v_key(kk), x = kl % RS + RS * (kl / 32);
      vr[kk] = reinterpret_cast<const uint32_t*>(raw)[(x * 64 + (kl % 32) / RS * CH) * 4 + dc];
    }
    if (part) {
      uint32_t odd = 0;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const int kl = v_key(kk);
        const bool has = (U == 2 && (kl & 64) ? exist[U - 1] : exist[0]) >> (kl & 63) & 1ull;
        if (!has) vr[kk] = 0;
        if (H::odd(vr[kk])) odd |= 1u << kk;
        vr[kk] = H::finite(vr[kk]);
      }
      while (odd) {
        const int kl = v_key(__ffs(odd) - 1);
        odd &= odd - 1;
        atomicOr(&odd_keys[kl >> 5], 1u << (kl & 31));
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint4 f;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        (&f.x)[w] = __builtin_amdgcn_perm(vr[2 * w + 1], vr[2 * w], e & 1 ? 0x07060302u : 0x05040100u);
      vs[((vg >> 1) * DT + e + 2 * (dc / 32)) * 64 + dc % 32 + 32 * (vg & 1)] = f;
    }
  };
  auto dim_of = [&](int t, int row) { return 2 * (row + 32 * (t >> 1)) + (t & 1); };

  if (tid < 3 * (KT / 32)) odd_of[tid / (KT / 32)][tid % (KT / 32)] = 0;
  // the keys that exist of this tile and the two after it
  unsigned long long now[U], next[U], second[U];
  auto meet = [&]() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // Tile number n at k0 (n % 3 = third, n % 2 = vs' half): loads the keys of tile
  // n + 2 and the values of tile n + 3, uses tile n, turns the values of n + 1.
  auto step = [&](int k0, int third, int parity, const uint4* ks, uint4* ks_load, const uint4* raw, uint4* raw_load)
                  __attribute__((always_inline)) {
    int asked[U];
    ask(k0 + 4 * KT, asked);
    load(a.k + kvh * a.c.head_stride, ks_load, 65, kload);  // at the offsets that the step before found
    look_up(k0 + 3 * KT);
    load(vbase, raw_load, 64, 0);
    const uint4* vs = &vss[parity * 1024];
    if (tid < KT / 32) odd_of[third == 0 ? 2 : third - 1][tid] = 0;  // the tile before this one's
    const bool part = partial(k0, now);
#pragma unroll 1
    for (int j = 0; j < KT / 32; j += NB) {
      const int kj = k0 + 32 * j;
      if (kj >= wave_hi || kj + 32 * NB <= wave_lo) continue;  // also past the end
      floatx16 s[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
      in_turn<NB * KS, AHEAD>([&](int x) { return ks[(j + x % NB) * RS * 65 + (x / NB < KS / 2 ? klow : khigh) + 2 * (x / NB)]; }, [&](int x, uint4 k) {
        const int c = x / NB;
        s[x % NB] = H::mfma32(k, c < QR ? q[c] : qs[(c - QR) * 512 + tid], s[x % NB]);
      });
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int kb = kj + 32 * b;
        const uint32_t has = (uint32_t)((U == 2 && j > 1 ? now[U - 1] : now[0]) >> (32 * ((j + b) & 1)));
        if (has == 0xffffffffu && kb >= wave_lo_all && kb + 32 <= wave_hi_all) continue;
        const uint32_t see = seen(has, kb, row_lo, row_hi) >> (4 * h);  // a lane's keys at constant places
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][i] = see >> (8 * (i >> 2) + (i & 3)) & 1u ? s[b][i] : -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
      top *= a.scale_log2;
      if (__any(top > m + kBehind)) {
        top = fmaxf(top, spk::lane_xor32(top));
        const float next = fmaxf(m, top);
        const float f = m == -INFINITY ? 0.0f : exp2_fast(m - next);
        m = next;
        shift = H::kShift - (next == -INFINITY ? 0.0f : next);
        l *= f;
#pragma unroll
        for (int t = 0; t < DT; ++t) acc[t] *= f;
      }
      // the weights of 16 keys while the product of the 16 before them runs
      uint4 p[2 * NB];
      auto weigh = [&](int i, int e0, int e1) __attribute__((always_inline)) {
        floatx16& x = s[i >> 1];
#pragma unroll
        for (int e = 8 * (i & 1) + e0; e < 8 * (i & 1) + e1; ++e) {
          x[e] = exp2_fast(__builtin_fmaf(x[e], a.scale_log2, shift));
          l += x[e];
        }
        if (e1 == 8) {
          const int f = 8 * (i & 1);
          p[i] = make_uint4(H::pack(x[f], x[f + 1]), H::pack(x[f + 2], x[f + 3]), H::pack(x[f + 4], x[f + 5]),
                            H::pack(x[f + 6], x[f + 7]));
        }
      };
      weigh(0, 0, 8);
      in_turn<2 * NB * DT, AHEAD>([&](int c) { return vs[(2 * j * DT + c) * 64 + lane]; }, [&](int c, uint4 v) {
        const int i = c / DT, t = c % DT;
        acc[t] = H::mfma32(v, p[i], acc[t]);
        if (i + 1 < 2 * NB) weigh(i + 1, 8 * t / DT, 8 * (t + 1) / DT);
      });
      if (part) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          uint32_t odd = __builtin_amdgcn_readfirstlane(odd_of[third][j + b]);
          while (odd) {
            const int kl = __ffs(odd) - 1, key = kj + 32 * b + kl;
            odd &= odd - 1;
            const uint16_t* row = vbase + max(spk_paged::offset_of(a.c, seq, key), (int64_t)0);
            const uint4 p0 = p[2 * b], p1 = p[2 * b + 1];
            uint32_t pair = kl & 16 ? (kl & 8 ? (kl & 2 ? p1.w : p1.z) : (kl & 2 ? p1.y : p1.x))
                                    : (kl & 8 ? (kl & 2 ? p0.w : p0.z) : (kl & 2 ? p0.y : p0.x));
            pair = __shfl((int)pair, ln + 32 * ((kl >> 2) & 1));
            const float weight = H::widen((uint16_t)(kl & 1 ? pair >> 16 : pair));
            if (key >= row_lo && key < row_hi) {
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
    }
    turn(raw, &vss[(parity ^ 1) * 1024], partial(k0 + KT, next), next, odd_of[third == 2 ? 0 : third + 1]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      now[u] = next[u];
      next[u] = second[u];
      second[u] = valid[u];
    }
    // all but this step's own four loads have arrived
#pragma unroll
    for (int u = 0; u < U; ++u) page[u] = asked[u];
    asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    meet();
  };
  if (begin < end) {
    const uint16_t* kbase = a.k + kvh * a.c.head_stride;
    ask(begin, page);
    look_up(begin);
    ask(begin + KT, page);
    load(kbase, ka, 65, kload);
    load(vbase, ra, 64, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = valid[u];
    look_up(begin + KT);
    ask(begin + 2 * KT, page);
    load(kbase, kb, 65, kload);
    load(vbase, rb, 64, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = valid[u];
    look_up(begin + 2 * KT);
    ask(begin + 3 * KT, page);
    load(vbase, rc, 64, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) second[u] = valid[u];
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    meet();
    turn(ra, vss, partial(begin, now), now, odd_of[0]);
    meet();
    // steps past the end are empty: with a way out between the steps, what is
    // under way would not be known where they meet
    int parity = 0;
    for (int k0 = begin; k0 < end; k0 += 3 * KT, parity ^= 1) {
      step(k0, 0, parity, ka, kc, rb, ra);
      step(k0 + KT, 1, parity ^ 1, kb, ka, rc, rb);
      step(k0 + 2 * KT, 2, parity, kc, kb, ra, rc);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // loads past the end still write LDS
  }

  l += spk::lane_xor32(l);
  if (r0 + 32 * wave + ln >= rows) return;
  const int ri = r / a.group, head = kvh * a.group + r - ri * a.group, token = sq.first + ri;
  const int64_t at = (int64_t)token * a.heads + head;
  float* part = a.part + (at + (int64_t)split * a.c.total_tokens * a.heads) * (D + 2);
  if (h == 0) {
    if (!alone) {
      part[0] = m;
      part[1] = l;
    } else if (a.lse) {
      a.lse[at] = l == 0.0f ? -INFINITY : (m - H::kShift + __builtin_amdgcn_logf(l)) * kLn2;
    }
  }
  const float inv = !alone ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int u = 0; u < DT / 2; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = acc[2 * u + (j & 1)][4 * i + (j >> 1)] * inv;
      const int d = dim_of(2 * u, 8 * i + 4 * h);
      if (!alone) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) *reinterpret_cast<float2*>(part + 2 + d + j) = make_float2(o[j], o[j + 1]);
      } else {
        store_out<BF, 8>(a, token, head, d, o);
      }
    }
}

// Joins the key ranges of a row: a wave to each, as fast as a whole workgroup to
// each where there are few rows of many ranges (32 rows of 64: 106 us with the
// attention either way) and faster where there are many (1024 rows: 24 us, 27).
// The ranges' maxima and sums are read by the lanes side by side; D / 4 lanes
// add a range's output, the other lanes take other ranges, and LDS joins them.
// Where the parts lie the kernels that made them say (`tell`).
template <int D, bool BF>
__global__ __launch_bounds__(256) void paged_join_kernel(Attn a) {
  constexpr int L = D / 4, W = 64 / L;  // lanes of a range, ranges at a time
  __shared__ float weights[4][64];
  __shared__ float4 all[4][W][L];
  const int lane = threadIdx.x & 63, mine = threadIdx.x >> 6;
  float* weight = weights[mine];
  auto together = [&]() {  // of a wave's lanes
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  int64_t at = (int64_t)blockIdx.x * 4 + mine;
  int token, head;
  int2 ranges;
  if (a.few) {
    const int r = (int)(at % a.few), s = (int)(at / a.few / a.kv_heads), kvh = (int)(at / a.few) - s * a.kv_heads;
    if (s >= a.c.num_seqs) return;
    const Seq sq = spk_paged::seq_at(a.c, s);
    if (r >= sq.n * a.group || sq.n * a.group >= a.many) return;
    token = sq.first + r / a.group;
    head = kvh * a.group + r % a.group;
    at = (int64_t)token * a.heads + head;
    ranges = a.ranges[at];
  } else {
    token = (int)(at / a.heads);
    head = (int)(at - (int64_t)token * a.heads);
    if (token >= a.c.total_tokens) return;
    ranges = a.ranges[at];  // asked for before the lengths: of a row of no sequence it is anything
    bool there = false;
    for (int s0 = 0; s0 < a.c.num_seqs && !there; s0 += 64) {
      const int s = min(s0 + lane, a.c.num_seqs - 1);
      there = __any(a.c.cu[s] <= token && token < a.c.cu[s + 1]);
    }
    if (!there) return;
  }
  const bool many = ranges.x < 0;
  // what a row of sequences that overlap left unwritten stays inside the workspace
  const int most = many ? a.splits : (int)(((int64_t)a.shares * a.share_rows - 1 - ranges.x) / a.share_rows) + 1;
  const int n = min(ranges.y, most);
  if (n <= 1) return;
  const int64_t step = many ? (int64_t)a.c.total_tokens * a.heads * (D + 2) : (int64_t)a.share_rows * (D + 2);
  const float* part = many ? a.part + at * (D + 2) : a.shared + (int64_t)ranges.x * (D + 2);

  float2 ml = lane < n ? *reinterpret_cast<const float2*>(part + lane * step) : make_float2(-INFINITY, 0.0f);
  float top = ml.x;
  for (int j = lane + 64; j < n; j += 64) top = fmaxf(top, part[j * step]);
  top = spk::wave_max(top);
  float sum = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int j0 = 0;;) {
    together();
    if (j0 + lane < n) {
      const float f = top == -INFINITY ? 1.0f : exp2_fast(ml.x - top);
      weight[lane] = f;
      sum += f * ml.y;
    }
    together();
    const int m = min(64, n - j0);
    constexpr int B = 8;  // loads under way, without a branch between them
    for (int j = lane / L; j < m; j += B * W) {
      float2 u[B], v[B];
#pragma unroll
      for (int i = 0; i < B; ++i) {
        const float* p = part + (j0 + min(j + i * W, m - 1)) * step + 2 + 4 * (lane % L);
        u[i] = *reinterpret_cast<const float2*>(p);
        v[i] = *reinterpret_cast<const float2*>(p + 2);
      }
#pragma unroll
      for (int i = 0; i < B; ++i) {
        const bool there = j + i * W < m;
        const float f = weight[min(j + i * W, m - 1)];
        o.x += there ? f * u[i].x : 0.0f;
        o.y += there ? f * u[i].y : 0.0f;
        o.z += there ? f * v[i].x : 0.0f;
        o.w += there ? f * v[i].y : 0.0f;
      }
    }
    j0 += 64;
    if (j0 >= n) break;
    ml = *reinterpret_cast<const float2*>(part + min(j0 + lane, n - 1) * step);
  }
  sum = wave_sum(sum);
  if constexpr (W > 1) {
    all[mine][lane / L][lane % L] = o;
    together();
    if (lane < L) {
#pragma unroll
      for (int w = 1; w < W; ++w) {
        const float4 u = all[mine][w][lane];
        o.x += u.x;
        o.y += u.y;
        o.z += u.z;
        o.w += u.w;
      }
    }
  }
  if (lane < L) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    store_out<BF, 4>(a, token, head, 4 * lane, y);
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

// Checks the cache (its sizes alone where there are no buffers yet) and fills the
// kernels' view of it.
int check_cache(const SpkPagedCache& p, const char* who, Cache* c, bool buffers) {
  if (p.dtype != SPK_F16 && p.dtype != SPK_BF16)
    return spk::fail(SPK_ERR_ARG, "%s: dtype %d (SPK_F16 or SPK_BF16)", who, p.dtype);
  if (p.head_dim != 64 && p.head_dim != 128 && p.head_dim != 256)
    return spk::fail(SPK_ERR_SHAPE, "%s: head_dim %d (64, 128 or 256)", who, p.head_dim);
  if (p.num_kv_heads <= 0 || p.page_size <= 0 || p.num_pages <= 0 || p.max_pages <= 0 || p.num_seqs < 0 ||
      p.total_tokens < 0)
    return spk::fail(SPK_ERR_SHAPE, "%s: kv_heads %d page_size %d num_pages %d max_pages %d num_seqs %d total_tokens %d",
                     who, p.num_kv_heads, p.page_size, p.num_pages, p.max_pages, p.num_seqs, p.total_tokens);
  if ((int64_t)p.max_pages * p.page_size > INT32_MAX - 4096)
    return spk::fail(SPK_ERR_SHAPE, "%s: max_pages %d of %d tokens pass 2^31 positions", who, p.max_pages, p.page_size);
  if (buffers && p.num_seqs && p.total_tokens) {
    if (!p.k_cache || !p.v_cache || !p.block_table || !p.cu_seqlens || !p.context_lens)
      return spk::fail(SPK_ERR_NULL, "%s: k_cache, v_cache, block_table, cu_seqlens or context_lens is NULL", who);
    if (!spk::aligned(p.k_cache, 16) || !spk::aligned(p.v_cache, 16) || !strides_ok(p.token_stride, p.head_stride) ||
        p.page_stride < 0 || p.page_stride % 8)
      return spk::fail(SPK_ERR_ALIGN, "%s: the cache and its strides (page %lld token %lld head %lld) must be 16-byte aligned",
                       who, (long long)p.page_stride, (long long)p.token_stride, (long long)p.head_stride);
    if (p.page_stride > UINT32_MAX || p.token_stride > UINT32_MAX)
      return spk::fail(SPK_ERR_SHAPE, "%s: page_stride %lld, token_stride %lld (below 2^32)", who,
                       (long long)p.page_stride, (long long)p.token_stride);
    if (p.table_stride < p.max_pages && p.num_seqs > 1)
      return spk::fail(SPK_ERR_SHAPE, "%s: table_stride %lld < max_pages %d", who, (long long)p.table_stride, p.max_pages);
  }
  c->table = p.block_table;
  c->cu = p.cu_seqlens;
  c->ctx = p.context_lens;
  c->table_stride = p.table_stride;
  c->page_stride = (uint32_t)p.page_stride;
  c->token_stride = (uint32_t)p.token_stride;
  c->head_stride = p.head_stride;
  c->num_seqs = p.num_seqs;
  c->total_tokens = p.total_tokens;
  c->page_size = p.page_size;
  c->num_pages = p.num_pages;
  c->max_pages = p.max_pages;
  c->div = spk_paged::page_div((uint32_t)p.page_size);
  return SPK_OK;
}

int check_attn(const SpkPagedAttnArgs* p, Cache* c, bool buffers) {
  if (!p) return spk::fail(SPK_ERR_NULL, "spk_paged_attention: NULL args");
  if (const int rc = check_cache(p->cache, "spk_paged_attention", c, buffers)) return rc;
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

template <int D, bool BF>
void launch_attn(const Attn& a, const Plan& r, hipStream_t s) {
  if (r.shares && r.share_rows == 16)
    hipLaunchKernelGGL((paged_rows_kernel<D, BF>), dim3(r.shares), dim3(256), 0, s, a);
  else if (r.shares)
    hipLaunchKernelGGL((paged_mid_kernel<D, BF>), dim3(r.shares), dim3(256), 0, s, a);
  if (r.tiles)
    hipLaunchKernelGGL((paged_tiles_kernel<D, BF>), dim3(r.splits, a.kv_heads, r.tiles), dim3(512), 0, s, a);
  if (!r.join) return;
  hipLaunchKernelGGL((paged_join_kernel<D, BF>), dim3((unsigned)((r.join_rows + 3) / 4)), dim3(256), 0, s, a);
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
  if (const int rc = check_cache(p->cache, who, &a.c, true)) return rc;
  const SpkPagedCache& c = p->cache;
  if (p->num_q_heads <= 0 || c.total_tokens > 4 * spk_paged::kMostGroups)
    return spk::fail(SPK_ERR_SHAPE, "%s: %d query heads, %d tokens (%lld at most)", who, p->num_q_heads, c.total_tokens,
                     (long long)(4 * spk_paged::kMostGroups));
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
  if (check_attn(p, &c, false) || p->cache.num_seqs == 0 || p->cache.total_tokens == 0) return 0;
  return spk_paged::workspace_bound(*p);
}

extern "C" size_t spk_paged_attention_workspace_need(const SpkPagedAttnArgs* p) {
  Cache c;
  if (check_attn(p, &c, false) || p->cache.num_seqs == 0 || p->cache.total_tokens == 0) return 0;
  return spk_paged::workspace_of(*p, spk_paged::plan_of(*p));
}

extern "C" int spk_paged_attention(const SpkPagedAttnArgs* p, spk_stream_t stream) {
  const char* who = "spk_paged_attention";
  Attn a{};
  if (const int rc = check_attn(p, &a.c, true)) return rc;
  const SpkPagedCache& c = p->cache;
  if (c.num_seqs == 0 || c.total_tokens == 0) return SPK_OK;
  if (!p->q || !p->out) return spk::fail(SPK_ERR_NULL, "%s: q or out is NULL", who);
  if (!spk::aligned(p->q, 16) || !spk::aligned(p->out, 16) || !spk::aligned(p->gate, 16) ||
      !strides_ok(p->q_token_stride, p->q_head_stride) || !strides_ok(p->out_token_stride, p->out_head_stride) ||
      (p->gate && !strides_ok(p->gate_token_stride, p->gate_head_stride)))
    return spk::fail(SPK_ERR_ALIGN, "%s: q, gate and out and their strides must be 16-byte aligned", who);
  const Plan r = spk_paged::plan_of(*p);
  if (r.shares > spk_paged::kMostGroups || (r.join && (r.join_rows + 3) / 4 > spk_paged::kMostGroups))
    return spk::fail(SPK_ERR_SHAPE, "%s: %d tokens of %d heads, %d sequences are more than one launch holds", who,
                     c.total_tokens, p->num_q_heads, c.num_seqs);
  const size_t need = spk_paged::workspace_of(*p, r);
  if (need && (!p->workspace || p->workspace_bytes < need || !spk::aligned(p->workspace, 256)))
    return spk::fail(p->workspace ? SPK_ERR_ARG : SPK_ERR_NULL, "%s: workspace of %zu bytes, %zu needed (256-byte aligned)",
                     who, p->workspace ? p->workspace_bytes : (size_t)0, need);
  if (c.num_kv_heads > 65535 || r.tiles > 65535)
    return spk::fail(SPK_ERR_SHAPE, "%s: %d KV heads, %d row tiles (65535 at most)", who, c.num_kv_heads, r.tiles);
  a.q = static_cast<const uint16_t*>(p->q);
  a.k = static_cast<const uint16_t*>(c.k_cache);
  a.v = static_cast<const uint16_t*>(c.v_cache);
  a.gate = static_cast<const uint16_t*>(p->gate);
  a.out = static_cast<uint16_t*>(p->out);
  a.lse = p->lse;
  a.shared = static_cast<float*>(p->workspace);
  if (r.join) a.ranges = reinterpret_cast<int2*>(static_cast<char*>(p->workspace) + shared_bytes(*p, r));
  a.part = reinterpret_cast<float*>(static_cast<char*>(p->workspace) + shared_bytes(*p, r) + ranges_bytes(*p, r));
  a.qt = p->q_token_stride;
  a.qh = p->q_head_stride;
  a.gt = p->gate_token_stride;
  a.gh = p->gate_head_stride;
  a.ot = p->out_token_stride;
  a.oh = p->out_head_stride;
  static_cast<spk_paged::Deal&>(a) = spk_paged::deal_of(*p, r, a.c);
  a.heads = p->num_q_heads;
  a.few = r.join_few ? spk_paged::kFew : 0;
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
