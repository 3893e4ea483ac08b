// paged_mx4.hip -- the serving step over a paged cache of microscaled 4-bit keys
// and values: rotary positions and the store (spk_mrope_append_mx4), and the
// attention of each sequence's new tokens (spk_paged_attention_mx4).
#include "mx4.hpp"
#include "paged_kernels.hpp"

namespace {

// Where the scales lie: strides in bytes, as those of the codes are here.
struct Scales {
  int64_t head_stride;
  uint32_t page_stride, token_stride;
};

// Offsets of a position's codes and scales of KV head 0, or -1: no page.
struct Place {
  int64_t codes, scales;
};

__device__ __forceinline__ Place place_in(const Cache& c, const Scales& s, int32_t page, int32_t pos) {
  if ((uint32_t)page >= (uint32_t)c.num_pages) return {-1, -1};
  const uint32_t at = (uint32_t)pos - spk_paged::divide(c.div, (uint32_t)pos) * (uint32_t)c.page_size;
  return {(int64_t)((uint64_t)(uint32_t)page * c.page_stride + (uint64_t)at * c.token_stride),
          (int64_t)((uint64_t)(uint32_t)page * s.page_stride + (uint64_t)at * s.token_stride)};
}

__device__ __forceinline__ Place place_of(const Cache& c, const Scales& sc, int32_t s, int32_t pos) {
  return place_in(c, sc, c.table[(int64_t)s * c.table_stride + spk_paged::divide(c.div, (uint32_t)pos)], pos);
}

// Above this byte a scale times 6 leaves the 16-bit type.
template <bool BF>
constexpr uint32_t kMost = BF ? 252 : 140;

// A cached block's scale in the 16-bit type: no number where it passes the type.
template <bool BF>
__device__ __forceinline__ float cached_scale(uint32_t byte) {
  return byte > kMost<BF> ? __builtin_inff() : spk_mx4::scale_of(byte);
}

// ---------------------------------------------------------------------------
// Rotary positions and the store into the pages.
// ---------------------------------------------------------------------------

struct MropeMx4 : Mrope {
  uint8_t *kcode, *vcode, *kscale, *vscale;
  Scales sc;
};

// One wave per token, the queries as in spk_mrope_append (the same arithmetic and
// lanes).  A lane holds the two chunks of 8 of a key that rotate together; the
// blocks of 32 are four chunks, whose largest exponents meet in LDS.  The keys'
// norm and rotation are in 64 bits and rounded once, to the code: in 32 a value
// next to a border between two codes, half of its size apart, went by the order
// of the sum of squares.  Values are quantised as they are.
template <int D, bool BF, bool ADJ>
__global__ __launch_bounds__(256) void mrope_append_mx4_kernel(MropeMx4 a) {
  constexpr int L = D / 16, RG = 64 / L;  // lanes of a head, heads at a time
  __shared__ int chunk_top[4][RG][D / 8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = blockIdx.x * 4 + wave;
  if (t >= a.c.total_tokens) return;
  const int s = spk_paged::seq_of_token(a.c.cu, a.c.num_seqs, t, lane);
  if (s >= a.c.num_seqs) return;
  const Seq sq = spk_paged::seq_at(a.c, s);
  if (t < sq.first || t >= sq.first + sq.n) return;
  const int pos = sq.ctx - sq.n + (t - sq.first);
  const Place slot = pos < 0 ? Place{-1, -1} : place_of(a.c, a.sc, s, pos);

  const int j = lane % L, rg = lane / L;
  const int turning = a.rot / 16;  // lanes that rotate
  const bool turns = j < turning;
  const int c0 = ADJ ? 2 * j : turns ? j : 2 * j;
  const int c1 = ADJ ? 2 * j + 1 : turns ? j + turning : 2 * j + 1;
  float cs[8], sn[8];
  angles(a, t, j, turns, cs, sn);

  for (int h = rg; h < a.heads; h += RG) {
    uint4 u0 = load_once(a.q + t * a.qt + h * a.qh + 8 * c0);
    uint4 u1 = load_once(a.q + t * a.qt + h * a.qh + 8 * c1);
    turn_row<D, BF, ADJ>(u0, u1, a.qw, c0, c1, turns, cs, sn, a.eps);
    uint16_t* dst = a.qo + t * a.ot + h * a.oh;
    *reinterpret_cast<uint4*>(dst + 8 * c0) = u0;
    *reinterpret_cast<uint4*>(dst + 8 * c1) = u1;
  }
  if (slot.codes < 0) return;

  // values: 16 elements side by side, two lanes a block
  for (int h = rg; h < a.kv_heads; h += RG) {
    const uint16_t* src = a.v + t * a.vt + h * a.vh + 16 * j;
    const uint4 u0 = load_once(src), u1 = load_once(src + 8);
    uint32_t most = max(spk_mx4::most_of(u0), spk_mx4::most_of(u1));
    most = max(most, spk::lane_xor1_u(most));
    const uint32_t byte = spk_mx4::scale_byte16<BF>(most);
    const float scale = spk_mx4::scale_of(byte);
    uint2 codes = make_uint2(spk_mx4::codes_of<BF>(u0, scale), spk_mx4::codes_of<BF>(u1, scale));
    if (byte == spk_mx4::kNone) codes = make_uint2(0, 0);
    *reinterpret_cast<uint2*>(a.vcode + slot.codes + h * a.c.head_stride + 8 * j) = codes;
    if ((j & 1) == 0) a.vscale[slot.scales + h * a.sc.head_stride + j / 2] = (uint8_t)byte;
  }

  for (int h0 = 0; h0 < a.kv_heads; h0 += RG) {
    const int h = min(h0 + rg, a.kv_heads - 1);  // lanes past the last head do its work again and store nothing
    const uint16_t* src = a.k + t * a.kt + h * a.kh;
    const uint4 u0 = load_once(src + 8 * c0), u1 = load_once(src + 8 * c1);
    double x[16];
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2_t lo = Half<BF>::unpack((&u0.x)[i]), hi = Half<BF>::unpack((&u1.x)[i]);
      x[2 * i] = lo.x;
      x[2 * i + 1] = lo.y;
      x[8 + 2 * i] = hi.x;
      x[8 + 2 * i + 1] = hi.y;
    }
    if (a.kw) {
      double ss = 0.0;
#pragma unroll
      for (int i = 0; i < 16; ++i) ss = __builtin_fma(x[i], x[i], ss);
#pragma unroll
      for (int m = L / 2; m; m >>= 1) ss += __shfl_xor(ss, m);
      const double inv = 1.0 / sqrt(ss / (double)D + (double)a.eps);
      const uint4 w0 = *reinterpret_cast<const uint4*>(a.kw + 8 * c0), w1 = *reinterpret_cast<const uint4*>(a.kw + 8 * c1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2_t lo = Half<BF>::unpack((&w0.x)[i]), hi = Half<BF>::unpack((&w1.x)[i]);
        x[2 * i] *= inv * (1.0 + (double)lo.x);
        x[2 * i + 1] *= inv * (1.0 + (double)lo.y);
        x[8 + 2 * i] *= inv * (1.0 + (double)hi.x);
        x[8 + 2 * i + 1] *= inv * (1.0 + (double)hi.y);
      }
    }
    if (turns) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i1 = ADJ ? 2 * e : e, i2 = ADJ ? 2 * e + 1 : 8 + e;
        const double x1 = x[i1], x2 = x[i2], c = cs[e], n = sn[e];
        x[i1] = __builtin_fma(x1, c, -(x2 * n));
        x[i2] = __builtin_fma(x2, c, x1 * n);
      }
    }
    // exponents of the chunks' largest (2047: an infinity or NaN)
    int top[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
      top[i >> 3] = max(top[i >> 3], (int)(__builtin_bit_cast(uint64_t, x[i]) >> 52 & 0x7ff));
    __builtin_amdgcn_wave_barrier();
    chunk_top[wave][rg][c0] = top[0];
    chunk_top[wave][rg][c1] = top[1];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int c = b ? c1 : c0;
      const int* four = &chunk_top[wave][rg][c & ~3];
      const int e = max(max(four[0], four[1]), max(four[2], four[3])) - 1023 - 2;
      odd = e == 2047 - 1023 - 2;
      const int byte = odd ? (int)spk_mx4::kNone : min(max(e + 127, 0), (int)kMost<BF>);
      // each rounded to the odd one of its two neighbours in 32 bits, so that the
      // rounding to a code is as of the unrounded value
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double v = x[8 * b + i];
        const float f = (float)v;
        const double back = (double)f;
        uint32_t u = __float_as_uint(f);
        if (back != v) u = (u - (fabs(back) > fabs(v) ? 1u : 0u)) | 1u;
        y[i] = __uint_as_float(u);
      }
      uint32_t codes = spk_mx4::codes_of(y, spk_mx4::scale_of((uint32_t)byte));
      if (odd) codes = 0;
      if (h0 + rg < a.kv_heads) {
        *reinterpret_cast<uint32_t*>(a.kcode + slot.codes + h * a.c.head_stride + 4 * c) = codes;
        if ((c & 3) == 0) a.kscale[slot.scales + h * a.sc.head_stride + c / 4] = (uint8_t)byte;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // read before the next heads' are written
    __builtin_amdgcn_wave_barrier();
  }
}

// ---------------------------------------------------------------------------
// Attention over the pages.
// ---------------------------------------------------------------------------

struct AttnMx4 : Attn {
  const uint8_t *kcode, *vcode, *kscale, *vscale;
  Scales sc;
};

// Few rows per sequence and KV head: spk_paged_attention's form for them (16 rows of
// a sequence and a range of its keys to a workgroup, every fourth step of 32 keys
// to a wave, scores transposed, the waves' states joined in LDS), from 4 bits.
//
// A lane of the scores' A operand holds 32 codes of a key that lie side by side,
// one block and one scale (heads of 64: half a block), as 4 contraction steps of
// 8; the queries' dimensions are dealt the same way.  Of the values it holds 8
// dimensions (heads of 64: 4) of its 8 keys.  Codes become 16-bit values with
// their scale in the conversion: exact but for what the type cannot hold.  A weight
// enters the second product rounded to 16 bits: the cache's own rounding is a
// hundred times as much.
template <int D, bool BF>
__global__ __launch_bounds__(256, 2) void mx4_rows_kernel(AttnMx4 a) {
  using H = Half<BF>;
  constexpr int NB = D >= 128 ? D / 128 : 1;  // blocks of a key in a lane
  constexpr int NC = D >= 128 ? 4 : 2;        // contraction steps of one
  constexpr int EV = D >= 128 ? 8 : 4;        // dimensions of a lane's values that lie side by side
  constexpr int NH = D / (16 * EV);           // such pieces
  constexpr int LD = D + 4;                   // padded rows of the joint
  __shared__ __align__(16) float joint[4][16][LD];
  __shared__ float stat[4][16][2];
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
  int lo, hi, lo_all, hi_all;
  spk_paged::visible(sq, r0 / a.group, a.window, &lo, &hi_all);
  spk_paged::visible(sq, (min(r0 + 16, rows) - 1) / a.group, a.window, &lo_all, &hi);
  const int begin = (int)min((int64_t)sh.lo + (int64_t)sh.range * sh.keys, (int64_t)hi);
  const int end = begin + min(sh.keys, hi - begin);

  const int32_t* table = a.c.table + (int64_t)seq * a.c.table_stride;
  const uint8_t* kcode = a.kcode + kvh * a.c.head_stride;
  const uint8_t* vcode = a.vcode + kvh * a.c.head_stride;
  const uint8_t* kscale = a.kscale + kvh * a.sc.head_stride;
  const uint8_t* vscale = a.vscale + kvh * a.sc.head_stride;
  auto load_page = [&](int k0) {
    const int key = k0 + (lane & 31);
    return key >= lo && key < end ? table[spk_paged::divide(a.c.div, (uint32_t)key)] : -1;
  };
  Place off{0, 0};
  uint32_t valid = 0;
  auto look_up = [&](int k0, int page) {
    off = place_in(a.c, a.sc, page, k0 + (lane & 31));
    valid = (uint32_t)__ballot(off.codes >= 0);
    if (off.codes < 0) off = Place{0, 0};
  };
  constexpr int kLaneCodes = D >= 128 ? 16 : 8;  // bytes of a lane's part of a key's block
  uint4 kf[2][NB];
  uint32_t ks[2][NB];
  uint32_t v[8][NH], vs[8][NH];
  auto load_k = [&]() {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* p = kcode + __shfl(off.codes, 16 * t + ln) + kLaneCodes * g;
      const uint8_t* q = kscale + __shfl(off.scales, 16 * t + ln) + (D >= 128 ? g : g / 2);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if constexpr (D >= 128) {
          kf[t][b] = *reinterpret_cast<const uint4*>(p + 64 * b);
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(p);
          kf[t][b] = make_uint4(w.x, w.y, 0, 0);
        }
        ks[t][b] = q[4 * b];
      }
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      const int kl = 16 * (kk >> 2) + 4 * g + (kk & 3);
      const uint8_t* p = vcode + __shfl(off.codes, kl) + EV / 2 * ln;
      const uint8_t* q = vscale + __shfl(off.scales, kl) + EV * ln / 32;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        if constexpr (EV == 8)
          v[kk][h] = *reinterpret_cast<const uint32_t*>(p + 64 * h);
        else
          v[kk][h] = *reinterpret_cast<const uint16_t*>(p);
        vs[kk][h] = q[4 * h];
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
  uint4 q[NB][NC];
  int row_lo, row_hi;
  {
    const int i = r / a.group;
    spk_paged::visible(sq, i, a.window, &row_lo, &row_hi);
    const uint16_t* src = a.q + (sq.first + i) * a.qt + (kvh * a.group + r - i * a.group) * a.qh + 2 * kLaneCodes * g;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int c = 0; c < NC; ++c) q[b][c] = *reinterpret_cast<const uint4*>(src + 128 * b + 8 * c);
  }
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
    floatx4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const float scale = cached_scale<BF>(ks[t][b]);
#pragma unroll
        for (int c = 0; c < NC; ++c) s[t] = H::mfma16(spk_mx4::expand<BF>((&kf[t][b].x)[c], scale), q[b][c], s[t]);
      }
    }
    if (more) {
      look_up(k0 + 128, page);
      page = load_page(k0 + 256);
      load_k();
    }
    float w[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = s[0][i];
      w[4 + i] = s[1][i];
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
    const uint4 p = make_uint4(H::pack(w[0], w[1]), H::pack(w[2], w[3]), H::pack(w[4], w[5]), H::pack(w[6], w[7]));
    uint32_t odd_keys = 0;
    if (!full) {
      // a block without a number must not meet the zero weight of a row that does
      // not see it: it counts as zeros here, and is added row by row
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const int kl = 16 * (kk >> 2) + 4 * g + (kk & 3);
        bool odd = false;
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          const bool none = vs[kk][h] > kMost<BF>;
          odd = odd || (none && (has >> kl & 1u));
          if (none) {
            v[kk][h] = 0;
            vs[kk][h] = 127;
          }
        }
        const unsigned long long b = __ballot(odd);
#pragma unroll
        for (int gg = 0; gg < 4; ++gg)
          if ((b >> (16 * gg)) & 0xffffull) odd_keys |= 1u << (16 * (kk >> 2) + 4 * gg + (kk & 3));
      }
    }
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      uint4 x[8];
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) x[kk] = spk_mx4::expand<BF>(v[kk][h], cached_scale<BF>(vs[kk][h]));
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        uint4 f;  // dimension e of the 8 keys
#pragma unroll
        for (int i = 0; i < 4; ++i)
          (&f.x)[i] = __builtin_amdgcn_perm((&x[2 * i + 1].x)[e >> 1], (&x[2 * i].x)[e >> 1],
                                            e & 1 ? 0x07060302u : 0x05040100u);
        acc[h][e] = H::mfma16(f, p, acc[h][e]);
      }
    }
    if (more) load_v();
    while (odd_keys) {
      const int kl = __ffs(odd_keys) - 1;
      odd_keys &= odd_keys - 1;
      const uint8_t* row = vscale + max(place_of(a.c, a.sc, seq, k0 + kl).scales, (int64_t)0);
      if (k0 + kl >= row_lo && k0 + kl < row_hi) {
#pragma unroll
        for (int h = 0; h < NH; ++h)
          if (row[D >= 128 ? 4 * h + g : g / 2] > kMost<BF>) {
#pragma unroll
            for (int e = 0; e < EV; ++e) acc[h][e] = floatx4{NAN, NAN, NAN, NAN};
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

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

// Checks the scales, and the codes' alignment, which is a row piece's.
int check_scales(const SpkPagedCache& c, const SpkPagedScales* s, const char* who, Scales* out) {
  if (!s) return spk::fail(SPK_ERR_NULL, "%s: scales is NULL", who);
  if (c.page_stride % 16 || c.token_stride % 16 || c.head_stride % 16)
    return spk::fail(SPK_ERR_ALIGN, "%s: the codes' strides (page %lld token %lld head %lld bytes) must be multiples of 16",
                     who, (long long)c.page_stride, (long long)c.token_stride, (long long)c.head_stride);
  if (!s->k_scales || !s->v_scales) return spk::fail(SPK_ERR_NULL, "%s: k_scales or v_scales is NULL", who);
  if (s->page_stride < 0 || s->token_stride < 0 || s->head_stride < 0 || s->page_stride > UINT32_MAX ||
      s->token_stride > UINT32_MAX)
    return spk::fail(SPK_ERR_SHAPE, "%s: the scales' strides (page %lld token %lld head %lld; below 2^32)", who,
                     (long long)s->page_stride, (long long)s->token_stride, (long long)s->head_stride);
  out->page_stride = (uint32_t)s->page_stride;
  out->token_stride = (uint32_t)s->token_stride;
  out->head_stride = s->head_stride;
  return SPK_OK;
}

template <int D, bool BF>
void launch_attn(const AttnMx4& a, const Plan& r, hipStream_t s) {
  hipLaunchKernelGGL((mx4_rows_kernel<D, BF>), dim3(r.shares), dim3(256), 0, s, a);
  if (!r.join) return;
  hipLaunchKernelGGL((paged_join_kernel<D, BF>), dim3((unsigned)((r.join_rows + 3) / 4)), dim3(256), 0, s, a);
}

template <int D, bool BF>
void launch_mrope(const MropeMx4& a, bool adjacent, hipStream_t s) {
  const dim3 grid((a.c.total_tokens + 3) / 4);
  if (adjacent)
    hipLaunchKernelGGL((mrope_append_mx4_kernel<D, BF, true>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((mrope_append_mx4_kernel<D, BF, false>), grid, dim3(256), 0, s, a);
}

}  // namespace

extern "C" int spk_mrope_append_mx4(const SpkMropeArgs* p, const SpkPagedScales* scales, spk_stream_t stream) {
  const char* who = "spk_mrope_append_mx4";
  MropeMx4 a{};
  if (const int rc = fill_mrope(p, who, &a)) return rc < 0 ? rc : SPK_OK;
  const SpkPagedCache& c = p->cache;
  if (const int rc = check_scales(c, scales, who, &a.sc)) return rc;
  a.kcode = static_cast<uint8_t*>(c.k_cache);
  a.vcode = static_cast<uint8_t*>(c.v_cache);
  a.kscale = scales->k_scales;
  a.vscale = scales->v_scales;
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

extern "C" size_t spk_paged_attention_mx4_workspace_size(const SpkPagedAttnArgs* p) {
  Cache c;
  if (check_attn(p, "spk_paged_attention_mx4", &c, false) || p->cache.num_seqs == 0 || p->cache.total_tokens == 0) return 0;
  return spk_paged::workspace_bound(*p);
}

extern "C" size_t spk_paged_attention_mx4_workspace_need(const SpkPagedAttnArgs* p) {
  Cache c;
  if (check_attn(p, "spk_paged_attention_mx4", &c, false) || p->cache.num_seqs == 0 || p->cache.total_tokens == 0) return 0;
  return spk_paged::workspace_of(*p, spk_paged::plan_mx4(*p));
}

extern "C" int spk_paged_attention_mx4(const SpkPagedAttnArgs* p, const SpkPagedScales* scales, spk_stream_t stream) {
  const char* who = "spk_paged_attention_mx4";
  AttnMx4 a{};
  Plan r;
  if (const int rc = fill_attn(p, who, spk_paged::plan_mx4, &a, &r)) return rc < 0 ? rc : SPK_OK;
  const SpkPagedCache& c = p->cache;
  if (const int rc = check_scales(c, scales, who, &a.sc)) return rc;
  a.kcode = static_cast<const uint8_t*>(c.k_cache);
  a.vcode = static_cast<const uint8_t*>(c.v_cache);
  a.kscale = scales->k_scales;
  a.vscale = scales->v_scales;
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
