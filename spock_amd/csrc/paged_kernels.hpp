// paged_kernels.hpp -- what the kernels over a paged cache share, whatever its
// type: the 16-bit types, the rotation of a row, the softmax helpers, the join of
// key ranges, and the checks of the arguments.  Included by paged.hip and
// paged_mx4.hip.
#pragma once

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

// The 8 pairs' angles that lane j of a head turns by at row t of the step.
__device__ __forceinline__ void angles(const Mrope& a, int t, int j, bool turns, float (&cs)[8], float (&sn)[8]) {
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
}

// A lane's 16 elements of a row, the chunks c0 and c1 of 8: normalised where there is
// a weight, rotated where the lane turns.
template <int D, bool BF, bool ADJ>
__device__ __forceinline__ void turn_row(uint4& u0, uint4& u1, const uint16_t* w, int c0, int c1, bool turns,
                                         const float (&cs)[8], const float (&sn)[8], float eps) {
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
    for (int m = D / 32; m; m >>= 1) ss += __shfl_xor(ss, m);
    const float inv = spk::rsqrt_det(ss / (float)D + eps);
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

// use(c, read(c)) for c below N, with the reads AHEAD of their use, or as the
// compiler has them.
template <int N, int AHEAD, typename T = uint4, typename Read, typename Use>
__device__ __forceinline__ void in_turn(Read read, Use use) {
  if constexpr (AHEAD == 0) {
#pragma unroll
    for (int c = 0; c < N; ++c) use(c, read(c));
  } else {
    T f[N];
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

int check_attn(const SpkPagedAttnArgs* p, const char* who, Cache* c, bool buffers) {
  if (!p) return spk::fail(SPK_ERR_NULL, "%s: NULL args", who);
  if (const int rc = check_cache(p->cache, who, c, buffers)) return rc;
  if (p->num_q_heads <= 0 || p->num_q_heads % p->cache.num_kv_heads)
    return spk::fail(SPK_ERR_SHAPE, "%s: %d query heads over %d KV heads", who, p->num_q_heads,
                     p->cache.num_kv_heads);
  if (!(p->scale >= 0.0f) || p->scale > 1e30f)
    return spk::fail(SPK_ERR_ARG, "%s: scale %g (positive, or 0 for 1/sqrt(head_dim))", who, (double)p->scale);
  if (p->max_query_len < 0 || p->max_context_len < 0 || p->window < 0)
    return spk::fail(SPK_ERR_SHAPE, "%s: max_query_len %d max_context_len %d window %d", who,
                     p->max_query_len, p->max_context_len, p->window);
  if ((int64_t)p->cache.total_tokens * p->num_q_heads > INT32_MAX - 65536)
    return spk::fail(SPK_ERR_SHAPE, "%s: %d tokens of %d heads", who, p->cache.total_tokens, p->num_q_heads);
  return SPK_OK;
}

// Checks the arguments of a rotation and store and fills the kernels' view of them.
// 1: there is nothing to do.
int fill_mrope(const SpkMropeArgs* p, const char* who, Mrope* a) {
  if (!p) return spk::fail(SPK_ERR_NULL, "%s: NULL args", who);
  if (const int rc = check_cache(p->cache, who, &a->c, true)) return rc;
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
    a->axis[i] = p->pair_axis[i];
  }
  if (p->rope_rows <= 0) return spk::fail(SPK_ERR_SHAPE, "%s: rope_rows %d", who, p->rope_rows);
  if (c.num_seqs == 0 || c.total_tokens == 0) return 1;
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
  a->q = static_cast<const uint16_t*>(p->q);
  a->k = static_cast<const uint16_t*>(p->k);
  a->v = static_cast<const uint16_t*>(p->v);
  a->qw = static_cast<const uint16_t*>(p->q_norm_w);
  a->kw = static_cast<const uint16_t*>(p->k_norm_w);
  a->qo = static_cast<uint16_t*>(p->q_out);
  a->kc = static_cast<uint16_t*>(c.k_cache);
  a->vc = static_cast<uint16_t*>(c.v_cache);
  a->qt = p->q_token_stride;
  a->qh = p->q_head_stride;
  a->kt = p->k_token_stride;
  a->kh = p->k_head_stride;
  a->vt = p->v_token_stride;
  a->vh = p->v_head_stride;
  a->ot = p->out_token_stride;
  a->oh = p->out_head_stride;
  a->positions = p->positions;
  a->pos_stride = p->positions_stride;
  a->rope = p->rope;
  a->rope_rows = p->rope_rows;
  a->rot = p->rot_dim;
  a->heads = p->num_q_heads;
  a->kv_heads = c.num_kv_heads;
  a->eps = p->eps > 0.0f ? p->eps : 1e-6f;
  return SPK_OK;
}

// Checks the arguments of an attention, plans it and fills the kernels' view of
// them.  1: there is nothing to do.
int fill_attn(const SpkPagedAttnArgs* p, const char* who, Plan (*plan_of)(const SpkPagedAttnArgs&), Attn* a, Plan* plan) {
  if (const int rc = check_attn(p, who, &a->c, true)) return rc;
  const SpkPagedCache& c = p->cache;
  if (c.num_seqs == 0 || c.total_tokens == 0) return 1;
  if (!p->q || !p->out) return spk::fail(SPK_ERR_NULL, "%s: q or out is NULL", who);
  if (!spk::aligned(p->q, 16) || !spk::aligned(p->out, 16) || !spk::aligned(p->gate, 16) ||
      !strides_ok(p->q_token_stride, p->q_head_stride) || !strides_ok(p->out_token_stride, p->out_head_stride) ||
      (p->gate && !strides_ok(p->gate_token_stride, p->gate_head_stride)))
    return spk::fail(SPK_ERR_ALIGN, "%s: q, gate and out and their strides must be 16-byte aligned", who);
  const Plan r = *plan = plan_of(*p);
  if (r.shares > spk_paged::kMostGroups || (r.join && (r.join_rows + 3) / 4 > spk_paged::kMostGroups))
    return spk::fail(SPK_ERR_SHAPE, "%s: %d tokens of %d heads, %d sequences are more than one launch holds", who,
                     c.total_tokens, p->num_q_heads, c.num_seqs);
  const size_t need = spk_paged::workspace_of(*p, r);
  if (need && (!p->workspace || p->workspace_bytes < need || !spk::aligned(p->workspace, 256)))
    return spk::fail(p->workspace ? SPK_ERR_ARG : SPK_ERR_NULL, "%s: workspace of %zu bytes, %zu needed (256-byte aligned)",
                     who, p->workspace ? p->workspace_bytes : (size_t)0, need);
  if (c.num_kv_heads > 65535 || r.tiles > 65535)
    return spk::fail(SPK_ERR_SHAPE, "%s: %d KV heads, %d row tiles (65535 at most)", who, c.num_kv_heads, r.tiles);
  a->q = static_cast<const uint16_t*>(p->q);
  a->k = static_cast<const uint16_t*>(c.k_cache);
  a->v = static_cast<const uint16_t*>(c.v_cache);
  a->gate = static_cast<const uint16_t*>(p->gate);
  a->out = static_cast<uint16_t*>(p->out);
  a->lse = p->lse;
  a->shared = static_cast<float*>(p->workspace);
  if (r.join) a->ranges = reinterpret_cast<int2*>(static_cast<char*>(p->workspace) + shared_bytes(*p, r));
  a->part = reinterpret_cast<float*>(static_cast<char*>(p->workspace) + shared_bytes(*p, r) + ranges_bytes(*p, r));
  a->qt = p->q_token_stride;
  a->qh = p->q_head_stride;
  a->gt = p->gate_token_stride;
  a->gh = p->gate_head_stride;
  a->ot = p->out_token_stride;
  a->oh = p->out_head_stride;
  static_cast<spk_paged::Deal&>(*a) = spk_paged::deal_of(*p, r, a->c);
  a->heads = p->num_q_heads;
  a->few = r.join_few ? spk_paged::kFew : 0;
  const float scale = p->scale != 0.0f ? p->scale : 1.0f / std::sqrt((float)c.head_dim);
  a->scale_log2 = scale * 1.44269504088896341f;
  return SPK_OK;
}

}  // namespace
