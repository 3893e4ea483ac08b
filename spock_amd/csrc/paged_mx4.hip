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
//
// Memory bounds it where there are many tokens, the chain of loads (lengths, page, angles)
// where there are few: 32768 tokens of 16 + 4 + 4 heads of 128 in bf16 115 us, 4.0 TB/s (133
// with the 140 registers and three waves to a SIMD that the compiler takes by itself, 151 with each
// head's loads where they are used), 64 tokens 11 us.  (Pairs side by side in fp16 do not fit.)
template <int D, bool BF, bool ADJ>
__global__ __launch_bounds__(256, ADJ && !BF ? 3 : 4) void mrope_append_mx4_kernel(MropeMx4 a) {
  constexpr int L = D / 16, RG = 64 / L;  // lanes of a head, heads at a time
  __shared__ int chunk_top[4][RG][D / 8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = blockIdx.x * 4 + wave;
  if (t >= a.c.total_tokens) return;
  const int j = lane % L, rg = lane / L;
  const int turning = a.rot / 16;  // lanes that rotate
  const bool turns = j < turning;
  const int c0 = ADJ ? 2 * j : turns ? j : 2 * j;
  const int c1 = ADJ ? 2 * j + 1 : turns ? j + turning : 2 * j + 1;
  // the first heads, all asked for at once and before the token's place is known
  struct Row {
    uint4 lo, hi;
  };
  auto row = [&](const uint16_t* x, int64_t xt, int64_t xh, int h, int lo, int hi) __attribute__((always_inline)) {
    const uint16_t* src = x + t * xt + h * xh;
    return Row{load_once(src + 8 * lo), load_once(src + 8 * hi)};
  };
  const int qlast = a.heads - 1, klast = a.kv_heads - 1;
  Row q = row(a.q, a.qt, a.qh, min(rg, qlast), c0, c1);
  Row v = row(a.v, a.vt, a.vh, min(rg, klast), 2 * j, 2 * j + 1);
  Row k = row(a.k, a.kt, a.kh, min(rg, klast), c0, c1);
  const int s = spk_paged::seq_of_token(a.c.cu, a.c.num_seqs, t, lane);
  if (s >= a.c.num_seqs) return;
  const Seq sq = spk_paged::seq_at(a.c, s);
  if (t < sq.first || t >= sq.first + sq.n) return;
  const int pos = sq.ctx - sq.n + (t - sq.first);
  const Place slot = pos < 0 ? Place{-1, -1} : place_of(a.c, a.sc, s, pos);

  float cs[8], sn[8];
  angles(a, t, j, turns, cs, sn);

  for (int h = rg; h < a.heads; h += RG) {
    uint4 u0 = q.lo, u1 = q.hi;
    if (h + RG < a.heads) q = row(a.q, a.qt, a.qh, h + RG, c0, c1);
    turn_row<D, BF, ADJ>(u0, u1, a.qw, c0, c1, turns, cs, sn, a.eps);
    uint16_t* dst = a.qo + t * a.ot + h * a.oh;
    *reinterpret_cast<uint4*>(dst + 8 * c0) = u0;
    *reinterpret_cast<uint4*>(dst + 8 * c1) = u1;
  }
  if (slot.codes < 0) return;

  // values: 16 elements side by side, two lanes a block
  for (int h = rg; h < a.kv_heads; h += RG) {
    const uint4 u0 = v.lo, u1 = v.hi;
    if (h + RG < a.kv_heads) v = row(a.v, a.vt, a.vh, h + RG, 2 * j, 2 * j + 1);
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
    const int h = min(h0 + rg, klast);  // lanes past the last head do its work again and store nothing
    const uint4 u0 = k.lo, u1 = k.hi;
    if (h0 + RG < a.kv_heads) k = row(a.k, a.kt, a.kh, min(h0 + RG + rg, klast), c0, c1);
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

// Two weights as what they are in the 16-bit type and what that leaves of them, both to
// nearest: some 22 bits together in fp16, 16 in bf16.  (A cached value is finite, or its block is
// no number: there is no infinity whose sign the smaller part could turn.)
template <bool BF>
__device__ __forceinline__ void two_parts(float a, float b, uint32_t* most, uint32_t* rest) {
  *most = Half<BF>::pack(a, b);
  const float2_t x = Half<BF>::unpack(*most);
  *rest = Half<BF>::pack(a - x.x, b - x.y);
}

// Few rows per sequence and KV head: spk_paged_attention's form for them (16 rows of
// a sequence and a range of its keys to a workgroup, every fourth step of 32 keys
// to a wave, scores transposed, the waves' states joined in LDS), from 4 bits.
//
// A step's codes, scales and page ids go straight into the wave's own LDS, whole rows to
// neighbouring lanes: read from memory in the operands' order they took four times
// the loads (4 bytes a lane of the values, 1 of the scales), and the pipe of addresses was
// the bound (64 sequences, heads of 128: 174 us, 3.3 TB/s).  At each step a wave asks for
// the step N - 1 further on, whose page ids it asked for N steps ago, and waits for its
// own.  Keys lie in LDS as in memory but for pieces exchanged by the row's number, so that
// 8 rows read side by side are in different banks; key 4 g + j of 16 values lies in row 4 j + g,
// so that what the four lane groups read lies together.
//
// A lane of the scores' A operand holds 32 codes of a key that lie side by side,
// one block and one scale (heads of 64: half a block), as 4 contraction steps of
// 8; the queries' dimensions are dealt the same way.  Of the values it holds D / 16
// dimensions of its 8 keys.  Codes become 16-bit values with their scale in the conversion:
// exact but for what the type cannot hold.  A weight enters the second product
// in two parts (`two_parts`): the products of the second one take 2 us of 39 with drafted
// tokens (16 sequences of 36 rows, heads of 256) and nothing where memory bounds it.
// Memory bounds long contexts (64 sequences, heads of 128: 144 us, 3.9 TB/s with the join's),
// the way to the first keys short ones (1500 keys: 15 us).
// BYTES: the scales' rows are not aligned to 4 bytes (or have 2), and are loaded by the byte.
template <int D, bool BF, bool BYTES>
__global__ __launch_bounds__(256, D == 64 ? 3 : (D == 128 ? 3 : 2) - BYTES) void mx4_rows_kernel(AttnMx4 a) {
  using H = Half<BF>;
  constexpr int NB = D >= 128 ? D / 128 : 1;   // blocks of a key in a lane
  constexpr int NC = D >= 128 ? 4 : 2;         // contraction steps of one
  constexpr int EV = D / 16;                   // dimensions of a lane's values
  constexpr int CP = D / 32;                   // 16-byte pieces of a row of codes, and blocks
  constexpr int RL = 64 / CP;                  // rows of a load
  constexpr int NL = 32 / RL;                  // loads of a step's keys
  constexpr int SB = BYTES ? 1 : 4;            // bytes of a lane's load of scales
  constexpr int NS = CP / SB;                  // such loads, lanes 0..31 of the keys, 32..63 of the values
  constexpr int N = D == 256 ? 2 : 3;          // steps in LDS
  constexpr int P = 2 * NL + NS + 1;           // loads of a step
  constexpr int KW = 32 * CP;                  // 16-byte pieces of a step's keys
  constexpr int SIZE = 2 * KW + NS * 16;       // of a step
  constexpr int JW = 68, JOINT = 4 * 16 * JW / 4;  // padded rows of the joint, and its pieces
  constexpr int FIRST = 4 * SIZE > JOINT ? 4 * SIZE : JOINT;
  // an array to each step: a load into one is then known not to touch the others
  __shared__ __align__(16) uint4 sa[FIRST], sb[4 * SIZE], sc[N == 3 ? 4 * SIZE : 1];
  __shared__ int32_t ia[128], ib[128], ic[N == 3 ? 128 : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
  const uint8_t* scales = lane < 32 ? kscale : vscale;
  // the lower lanes ask for the pages of the keys from k0 on
  auto ask = [&](int k0, int32_t* ids) __attribute__((always_inline)) {
    if (lane < 32)
      spk_mx4::load_lds<4>(table + spk_paged::divide(a.c.div, (uint32_t)min(max(k0 + lane, lo), end - 1)), ids + 32 * wave);
  };
  // what row r of a step's keys and of its values in LDS holds
  const int kfirst = lane / CP, kpiece = lane % CP ^ (CP == 8 ? kfirst & 7 : CP == 4 ? kfirst >> 1 & 3 : 0);
  const int idat = 32 * wave + (lane & 31);
  auto value_key = [](int r) { return (r & ~15) + 4 * (r & 3) + (r >> 2 & 3); };
  // Asks for the codes and scales of the step at k0; the keys of it that exist.
  auto load = [&](int k0, const int32_t* ids, uint4* to) __attribute__((always_inline)) {
    const int key = k0 + (lane & 31);
    Place off = place_in(a.c, a.sc, ids[idat], min(max(key, lo), end - 1));
    const bool there = key >= lo && key < end && off.codes >= 0;
    if (!there) off = Place{0, 0};  // the pool's first row, masked
    uint4* x = to + SIZE * wave;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int64_t k = __shfl(off.codes, RL * i + kfirst), v = __shfl(off.codes, value_key(RL * i + kfirst));
      spk_mx4::load_lds<16>(kcode + k + 16 * kpiece, x + 64 * i);
      spk_mx4::load_lds<16>(vcode + v + 16 * (lane % CP), x + KW + 64 * i);
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) spk_mx4::load_lds<SB>(scales + off.scales + SB * i, x + 2 * KW + 16 * i);
    return (uint32_t)__ballot(there);
  };
  const int r = min(r0 + ln, rows - 1);  // this lane's row
  uint4 q[NB][NC];
  int row_lo, row_hi;
  {
    const int i = r / a.group;
    spk_paged::visible(sq, i, a.window, &row_lo, &row_hi);
    const uint16_t* src = a.q + (sq.first + i) * a.qt + (kvh * a.group + r - i * a.group) * a.qh + (D >= 128 ? 32 : 16) * g;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int c = 0; c < NC; ++c) q[b][c] = *reinterpret_cast<const uint4*>(src + 128 * b + 8 * c);
  }
  float m = -INFINITY, base = 0.0f, l = 0.0f;
  floatx4 acc[EV];
#pragma unroll
  for (int e = 0; e < EV; ++e) acc[e] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  // Where this lane's parts of a step lie, in bytes.  (As one number each: of an address made
  // of many parts the compiler no longer knows the array, and waits for all loads before it reads.)
  const int mine = 16 * SIZE * wave, kflip = CP == 8 ? ln & 7 : ln >> 1 & 3;
  const int kat0 = D >= 128 ? mine + 16 * (ln * CP + (g ^ kflip)) : mine + 32 * ln + 8 * g;
  const int kat1 = mine + 16 * (ln * CP + (4 + g ^ kflip));  // heads of 256: the second block's
  const int vat = mine + 16 * KW + 16 * CP * g + EV / 2 * ln;
  auto scale_at = [&](int b, int key) { return mine + 32 * KW + 4 * (b / SB * 64 + key) + b % SB; };  // values: key + 32
  const int ksat0 = scale_at(D >= 128 ? g : g / 2, ln), ksat1 = scale_at(4 + g, ln), vsat = scale_at(ln * EV / 32, 32 + 4 * g);
  // The step at k0, which lies in `at`; asks for the one N - 1 further, into `to`.
  auto step = [&](int k0, const uint4* at, uint32_t has, int32_t* ids, uint4* to, uint32_t& next) __attribute__((always_inline)) {
    next = load(k0 + 128 * (N - 1), ids, to);
    ask(k0 + 128 * (2 * N - 1), ids);
    spk_mx4::arrived<(N - 1) * P>();
    if (k0 >= end) return;
    const auto* x = reinterpret_cast<const uint8_t*>(at);
    const bool full = has == 0xffffffffu && k0 >= lo_all && k0 + 32 <= hi_all;
    uint32_t ksc[2][NB], vsc[8], most = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int b = 0; b < NB; ++b) ksc[t][b] = x[(b ? ksat1 : ksat0) + 64 * t];
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) vsc[kk] = x[vsat + 64 * (kk >> 2) + 4 * (kk & 3)];
    floatx4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        most = max(most, ksc[t][b]);
        uint4 u;
        if constexpr (D >= 128) {
          u = *reinterpret_cast<const uint4*>(x + (b ? kat1 : kat0) + 256 * CP * t);
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(x + kat0 + 512 * t);
          u = make_uint4(w.x, w.y, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
          s[t] = H::mfma16(spk_mx4::expand<BF>((&u.x)[c], spk_mx4::scale_of(ksc[t][b])), q[b][c], s[t]);
      }
    }
    float w[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = s[0][i];
      w[4 + i] = s[1][i];
    }
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) most = max(most, vsc[kk]);
    const bool odd = __any(most > kMost<BF>);  // some block is no number
    if (odd) {
      // a key that has one is none: its score is no number, where it is seen
      uint32_t none = 0;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        bool bad = false;
#pragma unroll
        for (int b = 0; b < NB; ++b) bad = bad || ksc[t][b] > kMost<BF>;
        const unsigned long long v = __ballot(bad);
        none |= (uint32_t)((v | v >> 16 | v >> 32 | v >> 48) & 0xffff) << (16 * t);
      }
      none >>= 4 * g;
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = none >> (16 * (i >> 2) + (i & 3)) & 1u ? NAN : w[i];
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
      for (int e = 0; e < EV; ++e) acc[e] *= f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = exp2_fast(__builtin_fmaf(w[i], a.scale_log2, H::kShift - base));
      l += w[i];
    }
    uint4 p0, p1;
#pragma unroll
    for (int i = 0; i < 4; ++i) two_parts<BF>(w[2 * i], w[2 * i + 1], &(&p0.x)[i], &(&p1.x)[i]);
    // a block of values that is no number must not meet the zero weight of a row that
    // does not see it: it counts as zeros here, and is added row by row below
    uint32_t odd_keys = 0, zeros = 0;
    if (odd) {
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const bool none = vsc[kk] > kMost<BF>;
        zeros |= (none ? 1u : 0u) << kk;
        const unsigned long long b = __ballot(none && (has >> (16 * (kk >> 2) + 4 * g + (kk & 3)) & 1u));
#pragma unroll
        for (int gg = 0; gg < 4; ++gg)
          if ((b >> (16 * gg)) & 0xffffull) odd_keys |= 1u << (16 * (kk >> 2) + 4 * gg + (kk & 3));
      }
    }
#pragma unroll
    for (int e0 = 0; e0 < EV; e0 += 8) {  // 8 dimensions (heads of 64: 4) at a time
      uint4 v[8];
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const auto* from = x + vat + 16 * CP * (16 * (kk >> 2) + 4 * (kk & 3)) + e0 / 2;
        uint32_t u;
        if constexpr (EV == 4)
          u = *reinterpret_cast<const uint16_t*>(from);
        else
          u = *reinterpret_cast<const uint32_t*>(from);
        v[kk] = spk_mx4::expand<BF>(u, spk_mx4::scale_of(vsc[kk]));
      }
      if (odd) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          if (zeros >> kk & 1u) v[kk] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int e = e0; e < (EV < e0 + 8 ? EV : e0 + 8); ++e) {
        uint4 f;  // dimension e of the 8 keys
#pragma unroll
        for (int i = 0; i < 4; ++i)
          (&f.x)[i] = __builtin_amdgcn_perm((&v[2 * i + 1].x)[(e & 7) >> 1], (&v[2 * i].x)[(e & 7) >> 1],
                                            e & 1 ? 0x07060302u : 0x05040100u);
        acc[e] = H::mfma16(f, p0, acc[e]);
        acc[e] = H::mfma16(f, p1, acc[e]);
      }
    }
    while (odd_keys) {
      const int kl = __ffs(odd_keys) - 1;
      odd_keys &= odd_keys - 1;
      if (k0 + kl >= row_lo && k0 + kl < row_hi) {
#pragma unroll
        for (int i = 0; i < 4; ++i)  // this lane's outputs are dimensions EV (4 g + i) + e
          if (x[scale_at(EV * (4 * g + i) / 32, 32 + kl)] > kMost<BF>) {
#pragma unroll
            for (int e = 0; e < EV; ++e) acc[e][i] = NAN;
          }
      }
    }
  };
  int k0 = begin + 32 * wave;
  if (k0 < end) {
    uint32_t ha, hb, hc = 0;
    // the first N steps' page ids, then the first N - 1 steps and N further page ids in the
    // order in which steps ask for them
    ask(k0, ia);
    ask(k0 + 128, ib);
    if constexpr (N == 3) ask(k0 + 256, ic);
    spk_mx4::arrived<0>();
    if constexpr (N == 3) {
      ha = load(k0, ia, sa);
      ask(k0 + 384, ia);
      hb = load(k0 + 128, ib, sb);
      ask(k0 + 512, ib);
      // step n reads slot n + 2 (mod 3): ids of step 2 are in ic, of 3 in ia, of 4 in ib
      for (; k0 < end; k0 += 384) {
        step(k0, sa, ha, ic, sc, hc);
        step(k0 + 128, sb, hb, ia, sa, ha);
        step(k0 + 256, sc, hc, ib, sb, hb);
      }
    } else {
      ha = load(k0, ia, sa);
      ask(k0 + 256, ia);
      for (; k0 < end; k0 += 256) {
        step(k0, sa, ha, ib, sb, hb);
        step(k0 + 128, sb, hb, ia, sa, ha);
      }
    }
  }
  spk_mx4::arrived<0>();  // loads past the end still write LDS

  // join the waves, 4 dimensions of each 16th of a row at a time
  l += spk::lane_xor16(l);
  l += spk::lane_xor32(l);
  auto stat = reinterpret_cast<float(*)[16][2]>(sb);
  __syncthreads();
  if (g == 0) {
    stat[wave][ln][0] = m;
    stat[wave][ln][1] = l;
  }
  auto joint = reinterpret_cast<float(*)[16][JW]>(sa);
  const int row = threadIdx.x >> 4, part = threadIdx.x & 15, rj = r0 + row;
  const int i = rj / a.group, token = sq.first + i, head = kvh * a.group + rj - i * a.group;
  const int64_t at = (int64_t)token * a.heads + head;
  float* out = a.shared + ((int64_t)blockIdx.x * 16 + row) * (D + 2);
  float top = -INFINITY, sum = 0.0f, f[4];
#pragma unroll
  for (int c = 0; c < EV; c += 4) {
    __syncthreads();
#pragma unroll
    for (int n = 0; n < 4; ++n)
      *reinterpret_cast<float4*>(&joint[wave][ln][4 * (4 * g + n)]) = make_float4(acc[c][n], acc[c + 1][n], acc[c + 2][n], acc[c + 3][n]);
    __syncthreads();
    if (c == 0) {
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[w][row][0]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        f[w] = top == -INFINITY ? 1.0f : exp2_fast(stat[w][row][0] - top);
        sum += f[w] * stat[w][row][1];
      }
    }
    if (rj >= rows) continue;
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(&joint[w][row][4 * part]);
      o[0] += f[w] * x.x;
      o[1] += f[w] * x.y;
      o[2] += f[w] * x.z;
      o[3] += f[w] * x.w;
    }
    const int d = EV * part + c;
    if (sh.ranges == 1) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (int n = 0; n < 4; ++n) o[n] *= inv;
      store_out<BF, 4>(a, token, head, d, o);
    } else {
      *reinterpret_cast<float2*>(out + 2 + d) = make_float2(o[0], o[1]);
      *reinterpret_cast<float2*>(out + 4 + d) = make_float2(o[2], o[3]);
    }
  }
  if (part == 0 && rj < rows) {
    if (sh.ranges > 1) {
      out[0] = top;
      out[1] = sum;
    } else if (a.lse) {
      a.lse[at] = sum == 0.0f ? -INFINITY : (top - H::kShift + __builtin_amdgcn_logf(sum)) * kLn2;
    }
  }
}

// All LDS work of this wave is done, and the workgroup meets.
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0) alone
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Many rows per sequence and KV head: spk_paged_attention's form for them (256 rows to a
// workgroup of 8 waves, 32 to a wave, the keys in tiles of 8192 / D that all waves
// share, scores transposed), from 4 bits.
//
// A thread holds 16 codes of a key and 16 of a value, a half of a block, loaded into
// registers three tiles ahead, and turns them into 16-bit values in LDS one tile before they
// are used: once for 256 rows.  Keys and values lie in LDS alike, rows of pieces of 16
// bytes exchanged by the row's number: 8 keys' pieces side by side (the scores' operand) and 4
// values' halves of 32 dimensions (the transposing load's) lie in 128 bytes of banks without
// sharing any.  That is half of the 64 banks: the other rows that a cycle of 256 bytes
// could read have the same ones.  Counted are 2.5 conflict cycles for each LDS instruction
// (2048 tokens at 16384 keys: 39.9 million in 177 million busy CU cycles), which that arithmetic gives: 4 for a key
// read, 2 for a transposing one, some 8 for a store, none for the queries' pieces.
// The transposing load makes of 4 keys' values the output's operand.
// A weight enters the product with V in two parts here too, for half as many matrix instructions
// more: rounded to one part 2048 tokens at 16384 keys, 8 heads of 256, take 285 us and two
// prompts of heads of 64 91, in two parts 370 and 106.  But the error is then the plain form's (2-norm
// against 64 bits: fp16 2.1e-4, bf16 1.7e-3), where one part has a third more, and the same for all
// numbers of rows.
// The matrix instructions, busy for 53% of the time, and the LDS reads that feed them bound it: those
// 370 us are 700 TFLOP/s of the attention's own operations, 1050 with the second parts.
template <int D, bool BF>
__global__ __launch_bounds__(512, 2) void mx4_tiles_kernel(AttnMx4 a) {
  using H = Half<BF>;
  constexpr int KT = 8192 / D;             // keys of a tile
  constexpr int KS = D / 16;               // contraction steps of the scores
  constexpr int QR = D == 256 ? 8 : KS;   // of the queries' pieces in registers, the rest in LDS
  constexpr int DT = D / 32;               // output tiles
  constexpr int CH = D / 8;                // 16-byte pieces of a row
  constexpr int TK = D / 16;               // threads of a key
  constexpr int WK = 64 / TK;              // keys of a wave's threads
  constexpr int NB = D == 256 ? 1 : 2;     // blocks of 32 keys at a time
  // LDS reads ahead of the product that uses them, and of the queries' 16 pieces those in
  // registers, as the registers allow: 2048 tokens at 16384 keys, heads of 256, take 368 us with
  // (1, 8), 370 with (1, 6) and (2, 6), 385 with (0, 10); (1, 10) would keep 40 bytes of a lane on the
  // private stack.  Heads of 128 (six prompts): 175 us 4 and 6 ahead, 178 2 ahead.
  constexpr int AHEAD = D == 256 ? 1 : 4;
  __shared__ __align__(16) uint4 ks[2][1024], vs[2][1024];
  __shared__ __align__(16) uint4 qs[KS > QR ? (KS - QR) * 512 : 1];
  __shared__ __align__(16) uint32_t there[2][8];  // keys of a tile that exist, by wave of the threads that hold them
  __shared__ uint32_t odd_of[3][KT / 32];  // keys of a tile with blocks that are no numbers (tile number % 3)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 31, h = lane >> 5;
  const int kvh = blockIdx.y, split = (blockIdx.x + (blockIdx.z >> 3)) % gridDim.x;  // another range to an XCD every 8 tiles
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

  // this wave's rows, and the lane's
  const int w0 = r0 + 32 * wave;
  int row_lo, row_hi, wave_lo, wave_hi, wave_lo_all, wave_hi_all;
  spk_paged::visible(sq, min(w0, rows - 1) / a.group, a.window, &wave_lo, &wave_hi_all);
  spk_paged::visible(sq, min(w0 + 31, rows - 1) / a.group, a.window, &wave_lo_all, &wave_hi);
  wave_hi = min(wave_hi, end);
  uint4 q[QR];
  {
    const int r = min(w0 + ln, rows - 1), i = r / a.group;
    spk_paged::visible(sq, i, a.window, &row_lo, &row_hi);
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

  // this thread's key of a tile, and its 16 dimensions
  const int kt = tid / TK, part = tid % TK;
  const uint8_t* kcode = a.kcode + kvh * a.c.head_stride;
  const uint8_t* vcode = a.vcode + kvh * a.c.head_stride;
  const uint8_t* kscale = a.kscale + kvh * a.sc.head_stride;
  const uint8_t* vscale = a.vscale + kvh * a.sc.head_stride;
  struct Part {
    uint2 k, v;
    uint32_t kscale, vscale;
    bool there;
  };
  auto ask = [&](int k0) __attribute__((always_inline)) {
    return table[spk_paged::divide(a.c.div, (uint32_t)min(max(k0 + kt, lo), end - 1))];
  };
  auto load = [&](int k0, int page, Part& p) __attribute__((always_inline)) {
    const int key = k0 + kt;
    const Place o = place_in(a.c, a.sc, page, min(max(key, lo), end - 1));
    p.there = key >= lo && key < end && o.codes >= 0;
    // without a place the pool's first row, masked
    const int64_t code = (p.there ? o.codes : 0) + 8 * part, scale = (p.there ? o.scales : 0) + part / 2;
    p.k = *reinterpret_cast<const uint2*>(kcode + code);
    p.v = *reinterpret_cast<const uint2*>(vcode + code);
    p.kscale = kscale[scale];
    p.vscale = vscale[scale];
  };
  // Both exchanges are one: rows 0..7 have 0, 2, 4, 6, 1, 3, 5, 7.
  auto swapped = [](int row) { return (row & 3) << 1 | (row >> 2 & 1); };
  const int put = kt * CH + (2 * part ^ swapped(kt));  // the first piece's place; the other's is put ^ 1
  // A block of values that is no number must not meet the zero weight of a row that does
  // not see it: where some row of the workgroup does not, it counts as zeros, and is added
  // row by row.
  auto store = [&](int k0, int buf, int third, const Part& p) __attribute__((always_inline)) {
    const float s = cached_scale<BF>(p.kscale);
    const bool none = p.vscale > kMost<BF> && (k0 + kt < lo_all || k0 + kt >= hi_all);
    if (p.there && none) atomicOr(&odd_of[third][kt >> 5], 1u << (kt & 31));
    const bool take = p.there && !none;
    const float t = take ? cached_scale<BF>(p.vscale) : 0.0f;
    ks[buf][put] = spk_mx4::expand<BF>(p.k.x, s);
    ks[buf][put ^ 1] = spk_mx4::expand<BF>(p.k.y, s);
    vs[buf][put] = spk_mx4::expand<BF>(take ? p.v.x : 0, t);
    vs[buf][put ^ 1] = spk_mx4::expand<BF>(take ? p.v.y : 0, t);
    const bool mine = __shfl((int)p.there, lane * TK & 63);
    const uint32_t bits = (uint32_t)__ballot(mine && lane < WK);
    if (lane == 0) there[buf][wave] = bits;
  };
  // piece 2 c + h of a key: 2 c exchanges bits of the place of piece h
  const int kread = ln * CH + (h ^ swapped(ln));
  // the transposing load's row, half of 32 dimensions, and 8-byte piece
  const int vrow = 4 * h + (lane >> 2 & 3), vflip = swapped(vrow), vpiece = 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
  const int vread = 2 * (vrow * CH + (vpiece ^ (vflip & 3))) + (lane & 1);
  if (tid < 3 * (KT / 32)) odd_of[tid / (KT / 32)][tid % (KT / 32)] = 0;

  // Tile number n at k0 (n % 3 = third, n % 2 = buf): the values of n + 1 go to LDS, the
  // codes of n + 3 are loaded, tile n is used.
  int page = 0;  // of tile n + 3
  auto step = [&](int k0, int third, int buf, Part& p) __attribute__((always_inline)) {
    store(k0 + KT, buf ^ 1, third == 2 ? 0 : third + 1, p);
    const int next = ask(k0 + 4 * KT);
    load(k0 + 3 * KT, page, p);
    page = next;
    if (tid < KT / 32) odd_of[third == 0 ? 2 : third - 1][tid] = 0;  // the tile before this one's
    uint32_t has[KT / 32];
#pragma unroll
    for (int j = 0; j < KT / 32; ++j) {
      has[j] = 0;
#pragma unroll
      for (int w = 0; w < 32 / WK; ++w) has[j] |= there[buf][j * (32 / WK) + w] << (w * WK % 32);
    }
    const bool some = k0 < lo_all || k0 + KT > hi_all;  // some row does not see some key
    const uint4* kk = ks[buf];
    const uint2* vv = reinterpret_cast<const uint2*>(vs[buf]);
#pragma unroll
    for (int j = 0; j < KT / 32; j += NB) {
      const int kj = k0 + 32 * j;
      if (kj >= wave_hi || kj + 32 * NB <= wave_lo) continue;  // also past the end
      floatx16 s[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i] = 0.0f;
      in_turn<NB * KS, AHEAD>(
          [&](int x) {
            const int c = x / NB;
            return kk[32 * (j + x % NB) * CH + (c & ~3) * 2 + (kread ^ 2 * (c & 3))];
          },
          [&](int x, uint4 k) {
            const int c = x / NB;
            s[x % NB] = H::mfma32(k, c < QR ? q[c] : qs[(c - QR) * 512 + tid], s[x % NB]);
          });
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int kb = kj + 32 * n;
        const uint32_t exist = __builtin_amdgcn_readfirstlane(has[j + n]);
        if (exist == 0xffffffffu && kb >= wave_lo_all && kb + 32 <= wave_hi_all) continue;
        const uint32_t see = seen(exist, kb, row_lo, row_hi) >> (4 * h);  // a lane's keys at constant places
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i] = see >> (8 * (i >> 2) + (i & 3)) & 1u ? s[n][i] : -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[n][i]);
      top *= a.scale_log2;
      if (__any(top > m + kBehind)) {
        const float next = fmaxf(m, fmaxf(top, spk::lane_xor32(top)));
        const float f = m == -INFINITY ? 0.0f : exp2_fast(m - next);
        m = next;
        shift = H::kShift - (next == -INFINITY ? 0.0f : next);
        l *= f;
#pragma unroll
        for (int t = 0; t < DT; ++t) acc[t] *= f;
      }
      // the weights of 16 keys while the product of the 16 before them runs
      uint4 p0[2 * NB], p1[2 * NB];
      auto weigh = [&](int i, int e0, int e1) __attribute__((always_inline)) {
        floatx16& x = s[i >> 1];
#pragma unroll
        for (int e = 8 * (i & 1) + e0; e < 8 * (i & 1) + e1; ++e) {
          x[e] = exp2_fast(__builtin_fmaf(x[e], a.scale_log2, shift));
          l += x[e];
        }
        if (e1 == 8) {
          const int f = 8 * (i & 1);
#pragma unroll
          for (int n = 0; n < 4; ++n) two_parts<BF>(x[f + 2 * n], x[f + 2 * n + 1], &(&p0[i].x)[n], &(&p1[i].x)[n]);
        }
      };
      weigh(0, 0, 8);
      in_turn<2 * NB * DT, AHEAD>(
          [&](int c) {
            // dimension 32 t + ln of keys 16 i + 4 h .. + 3 and 8 further
            const int i = c / DT, t = c % DT;
            const uint2* at = vv + 2 * (32 * j + 16 * i) * CH + 8 * (t & ~1) + (vread + 8 * ((t & 1) ^ (vflip >> 2)));
            const uint2 u = transposed(at), w = transposed(at + 16 * CH);
            return make_uint4(u.x, u.y, w.x, w.y);
          },
          [&](int c, uint4 v) {
            const int i = c / DT, t = c % DT;
            acc[t] = H::mfma32(v, p0[i], acc[t]);
            acc[t] = H::mfma32(v, p1[i], acc[t]);
            if (i + 1 < 2 * NB) weigh(i + 1, 8 * t / DT, 8 * (t + 1) / DT);
          });
      if (some) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          uint32_t odd = __builtin_amdgcn_readfirstlane(odd_of[third][j + n]);
          while (odd) {
            const int key = kj + 32 * n + __ffs(odd) - 1;
            odd &= odd - 1;
            const uint8_t* row = a.vscale + kvh * a.sc.head_stride + max(place_of(a.c, a.sc, seq, key).scales, (int64_t)0);
            if (key >= row_lo && key < row_hi) {
#pragma unroll
              for (int t = 0; t < DT; ++t)
                if (row[t] > kMost<BF>) {
#pragma unroll
                  for (int i = 0; i < 16; ++i) acc[t][i] = NAN;
                }
            }
          }
        }
      }
    }
    meet();
  };
  if (begin < end) {
    Part pa, pb;
    const int first = ask(begin), second = ask(begin + KT), last = ask(begin + 2 * KT);
    page = ask(begin + 3 * KT);
    load(begin, first, pa);
    load(begin + KT, second, pb);
    __syncthreads();  // odd_of is clear
    store(begin, 0, 0, pa);
    load(begin + 2 * KT, last, pa);
    meet();
    int third = 0;
    for (int k0 = begin; k0 < end; k0 += 2 * KT) {
      step(k0, third, 0, pb);
      third = third == 2 ? 0 : third + 1;
      step(k0 + KT, third, 1, pa);
      third = third == 2 ? 0 : third + 1;
    }
  }

  l += spk::lane_xor32(l);
  const int r = w0 + ln;
  if (r >= rows) return;
  const int ri = r / a.group, head = kvh * a.group + r - ri * a.group, token = sq.first + ri;
  const int64_t at = (int64_t)token * a.heads + head;
  float* out = a.part + (at + (int64_t)split * a.c.total_tokens * a.heads) * (D + 2);
  if (h == 0) {
    if (!alone) {
      out[0] = m;
      out[1] = l;
    } else if (a.lse) {
      a.lse[at] = l == 0.0f ? -INFINITY : (m - H::kShift + __builtin_amdgcn_logf(l)) * kLn2;
    }
  }
  const float inv = !alone ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float o[4] = {acc[t][4 * i] * inv, acc[t][4 * i + 1] * inv, acc[t][4 * i + 2] * inv, acc[t][4 * i + 3] * inv};
      const int d = 32 * t + 8 * i + 4 * h;
      if (!alone) {
        *reinterpret_cast<float2*>(out + 2 + d) = make_float2(o[0], o[1]);
        *reinterpret_cast<float2*>(out + 4 + d) = make_float2(o[2], o[3]);
      } else {
        store_out<BF, 4>(a, token, head, d, o);
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
void launch_attn(const AttnMx4& a, const Plan& r, bool bytes, hipStream_t s) {
  if (r.shares && bytes)
    hipLaunchKernelGGL((mx4_rows_kernel<D, BF, true>), dim3(r.shares), dim3(256), 0, s, a);
  else if (r.shares)
    hipLaunchKernelGGL((mx4_rows_kernel<D, BF, D == 64>), dim3(r.shares), dim3(256), 0, s, a);
  if (r.tiles) hipLaunchKernelGGL((mx4_tiles_kernel<D, BF>), dim3(r.splits, a.kv_heads, r.tiles), dim3(512), 0, s, a);
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
  return spk_paged::workspace_bound_mx4(*p);
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
  // a position's scales are whole dwords
  const bool bytes = (a.sc.page_stride | a.sc.token_stride | a.sc.head_stride) % 4 || !spk::aligned(a.kscale, 4) ||
                     !spk::aligned(a.vscale, 4);
  if (c.head_dim == 64)
    bf ? launch_attn<64, true>(a, r, bytes, s) : launch_attn<64, false>(a, r, bytes, s);
  else if (c.head_dim == 128)
    bf ? launch_attn<128, true>(a, r, bytes, s) : launch_attn<128, false>(a, r, bytes, s);
  else
    bf ? launch_attn<256, true>(a, r, bytes, s) : launch_attn<256, false>(a, r, bytes, s);
  return spk::check_launch(who);
}
