// mx4.hip -- microscaled 4-bit floating point: quantisation and back
// (spk_mx4_quantize, spk_mx4_dequantize) and the products with such weights
// (spk_mx4_matmul).
#include "mx4.hpp"

#include "capi_common.hpp"
#include "numerics.hpp"
#include "paged.hpp"

namespace {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef int intx8 __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------
// Quantisation.
// ---------------------------------------------------------------------------

// Rows cut into groups of 8 values, a group to a thread: four groups are a block,
// and its four lanes find the largest magnitude together.  16 or 32 bytes to a lane in
// and 4 out (or back), all read and written once: memory bounds it (248320 x 1024 in bf16 there and
// back 233 us, 5.5 TB/s, a copy's rate 5.2), few rows the launch (16 x 1024: 4.6 us both, the
// host's calls longer).
struct Rows {
  const void* x;
  void* y;
  uint8_t *codes, *scales;
  int64_t stride, code_stride, scale_stride;  // of x or y in elements
  uint32_t groups, per_row;
  spk_paged::PageDiv div;  // by per_row
};

struct Group {
  int64_t row;
  uint32_t at;  // in the row
};

__device__ __forceinline__ Group group_of(const Rows& a, uint32_t i) {
  const uint32_t row = spk_paged::divide(a.div, i);
  return {(int64_t)row, i - row * a.per_row};
}

template <typename T>
__device__ __forceinline__ T xor_max4(T v) {  // over the four lanes of a block
  v = max(v, (T)spk::lane_xor1_u((uint32_t)v));
  return max(v, (T)spk::lane_xor2_u((uint32_t)v));
}

template <int DT>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(Rows a) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.groups) return;  // whole blocks: groups is a multiple of 4
  const Group g = group_of(a, i);
  uint32_t byte, codes;
  if constexpr (DT == SPK_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.x) + g.row * a.stride + 8 * (int64_t)g.at);
    const float4 u = p[0], v = p[1];
    const float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) most = max(most, __float_as_uint(x[k]) & 0x7fffffffu);
    byte = spk_mx4::scale_byte(xor_max4(most));
    codes = spk_mx4::codes_of(x, spk_mx4::scale_of(byte));
  } else {
    constexpr bool BF = DT == SPK_BF16;
    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + g.row * a.stride + 8 * (int64_t)g.at);
    byte = spk_mx4::scale_byte16<BF>(xor_max4(spk_mx4::most_of(u)));
    codes = spk_mx4::codes_of<BF>(u, spk_mx4::scale_of(byte));
  }
  if (byte == spk_mx4::kNone) codes = 0;
  *reinterpret_cast<uint32_t*>(a.codes + g.row * a.code_stride + 4 * (int64_t)g.at) = codes;
  if ((g.at & 3) == 0) a.scales[g.row * a.scale_stride + g.at / 4] = (uint8_t)byte;
}

template <int DT>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(Rows a) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.groups) return;
  const Group g = group_of(a, i);
  const uint32_t u = *reinterpret_cast<const uint32_t*>(a.codes + g.row * a.code_stride + 4 * (int64_t)g.at);
  const float scale = spk_mx4::scale_of(a.scales[g.row * a.scale_stride + g.at / 4]);
  const int64_t to = g.row * a.stride + 8 * (int64_t)g.at;
  if constexpr (DT == SPK_F32) {
    const auto p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, scale, 0), q = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, scale, 1);
    const auto r = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, scale, 2), s = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, scale, 3);
    float4* y = reinterpret_cast<float4*>(static_cast<float*>(a.y) + to);
    y[0] = make_float4(p[0], p[1], q[0], q[1]);
    y[1] = make_float4(r[0], r[1], s[0], s[1]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.y) + to) = spk_mx4::expand<DT == SPK_BF16>(u, scale);
  }
}

// ---------------------------------------------------------------------------
// Products.
// ---------------------------------------------------------------------------

struct Mm {
  const uint16_t* x;
  const uint8_t *xc, *xs, *wc, *ws;
  const uint16_t* res;
  uint16_t* out;
  int64_t xt, xct, xst, wct, wst, rt, ot;
  int32_t rows, cols, depth;  // of the product: m, n, k
};

__device__ const uint4 kZero[4] = {};  // what lanes past the last value of a row read

template <bool BF>
__device__ __forceinline__ floatx4 mfma16(uint4 a, uint4 b, floatx4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8_t, a), __builtin_bit_cast(bf8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

template <bool BF>
__device__ __forceinline__ floatx16 mfma32(uint4 a, uint4 b, floatx16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8_t, a), __builtin_bit_cast(bf8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

// Four codes' dwords as an operand of the scaled products (of 8, the upper are not read).
__device__ __forceinline__ intx8 four_bits(uint4 u) {
  return intx8{(int)u.x, (int)u.y, (int)u.z, (int)u.w, 0, 0, 0, 0};
}

template <bool BF>
__device__ __forceinline__ float widen(uint16_t u) {
  if constexpr (BF) return __uint_as_float((uint32_t)u << 16);
  return (float)__builtin_bit_cast(_Float16, u);
}
template <bool BF>
__device__ __forceinline__ uint16_t narrow(float f) {
  if constexpr (BF) return __builtin_bit_cast(uint16_t, (__bf16)f);
  return __builtin_bit_cast(uint16_t, (_Float16)f);
}

// Few rows of x, 16 to a workgroup (XR = 4: up to 4): a wave takes 16 NT rows of w and every
// KW-th step of 128 values of their depth, and the KW waves' sums meet in LDS, in their
// order.  A lane of the 16x16 products' A operand holds one block of a row of w, 32 codes
// under one scale, as four contraction steps of 8 (rows in 16 bits) or as they
// are (rows in 4 bits, whose scales the instruction applies).
//
// In that order neighbouring lanes read different rows, and a load takes 64 cycles of the
// address pipe, one for each line that four lanes touch (57 measured, 16 where four lanes
// share a line): one row times 248320 x 1024 took 36 us that way, whatever the tile.  So
// codes, scales and x go straight into the wave's own LDS, row by row, two steps ahead,
// their pieces exchanged so that rows read side by side are in different banks.
// Memory bounds one row times many (1 x 248320 x 1024: 30 us, 4.5 TB/s), the time to the
// first steps and the sums' meeting a small w (17 x 1024 x 3584: 5 us), the conversions and the 16
// rows' own reads of w more rows (64 x 4096 x 14336: 21 us).
// SB: bytes of a load of scales (4: a step's scales of a row are an aligned dword).
template <bool X4, bool BF, int XR, int NT, int KW, int SB>
__global__ __launch_bounds__(KW > 4 ? 64 * KW : 256) void mx4_few_rows_kernel(Mm a) {
  constexpr int W = KW > 4 ? KW : 4, TILES = W / KW;  // waves, and groups of them that share rows of w
  constexpr int XL = X4 ? 1 : XR / 4;                 // loads of x
  constexpr int NS = 4 / SB;
  constexpr int P = NT + XL + NS * (X4 ? 2 : 1);      // loads of a step
  constexpr int SIZE = 64 * (NT + XL) + 16 * NS * (X4 ? 2 : 1);  // 16-byte pieces of a step
  constexpr int SUMS = 16 * (16 * NT + 1) / 4;        // of a wave's sums
  constexpr int FIRST = W * (SIZE > SUMS ? SIZE : SUMS);
  // an array to each step: a load into one is then known not to touch the others
  __shared__ __align__(16) uint4 sa[FIRST], sb[W * SIZE], sc[W * SIZE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 15, g = lane >> 4;
  const int kw = wave % KW;
  const int n0 = (blockIdx.x * TILES + wave / KW) * 16 * NT, m0 = blockIdx.y * 16;
  const int blocks = a.depth / 32, steps = (blocks + 3) / 4;

  const int wpiece = lane % 4 ^ (lane >> 3 & 3);  // of row lane / 4 in its place
  const uint8_t *wp[NT], *wsp, *xp[XL], *xsp = nullptr;
#pragma unroll
  for (int t = 0; t < NT; ++t) wp[t] = a.wc + min(n0 + 16 * t + lane / 4, a.cols - 1) * a.wct + 16 * wpiece;
  wsp = a.ws + min(n0 + lane % (16 * NT), a.cols - 1) * a.wst;
  int xpiece[XL];
  if constexpr (X4) {
    xpiece[0] = wpiece;
    xp[0] = a.xc + min(m0 + lane / 4, a.rows - 1) * a.xct + 16 * wpiece;
    xsp = a.xs + min(m0 + lane % 16, a.rows - 1) * a.xst;
  } else {
#pragma unroll
    for (int i = 0; i < XL; ++i) {
      const int row = 4 * i + lane / 16;
      xpiece[i] = lane % 16 ^ (row & 7);
      xp[i] = reinterpret_cast<const uint8_t*>(a.x + min(m0 + row, a.rows - 1) * a.xt) + 16 * xpiece[i];
    }
  }
  auto load = [&](int st, uint4* to) __attribute__((always_inline)) {
    st = min(st, steps - 1);  // past the end the last one again, which nobody uses
    const uint8_t* zero = reinterpret_cast<const uint8_t*>(kZero);
    uint4* w = to + SIZE * wave;
    uint4 *x = w + 64 * NT, *s = x + 64 * XL;
#pragma unroll
    for (int t = 0; t < NT; ++t)
      spk_mx4::load_lds<16>(SB == 4 || 4 * st + wpiece < blocks ? wp[t] + 64 * (int64_t)st : zero, w + 64 * t);
#pragma unroll
    for (int i = 0; i < XL; ++i)
      spk_mx4::load_lds<16>(SB == 4 || 4 * st + (X4 ? xpiece[i] : xpiece[i] / 4) < blocks ? xp[i] + (X4 ? 64 : 256) * (int64_t)st : zero, x + 64 * i);
#pragma unroll
    for (int b = 0; b < NS; ++b) {
      spk_mx4::load_lds<SB>(SB == 4 || 4 * st + b < blocks ? wsp + 4 * (int64_t)st + b : zero, s + 16 * b);
      if constexpr (X4) spk_mx4::load_lds<SB>(SB == 4 || 4 * st + b < blocks ? xsp + 4 * (int64_t)st + b : zero, s + 16 * (NS + b));
    }
  };
  // Where this lane's operands lie, in bytes.  (As one number each: of an address made of many
  // parts the compiler no longer knows the array, and waits for all loads before it reads.)
  const int mine = 16 * SIZE * wave, wat = mine + 16 * (4 * ln + (g ^ (ln >> 1 & 3)));
  const int xrow = ln & (XR - 1);
  const int xat = mine + 1024 * NT + 16 * (X4 ? 4 * ln + (g ^ (ln >> 1 & 3)) : 16 * xrow + (4 * g ^ (xrow & 7)));
  const int sat = mine + 1024 * (NT + XL) + (SB == 4 ? 4 * ln + g : 256 * g + 4 * ln);
  floatx4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  auto step = [&](int st, const uint4* at, uint4* to) __attribute__((always_inline)) {
    load(st + 2 * KW, to);
    spk_mx4::arrived<2 * P>();
    if (st < steps) {
      const auto* p = reinterpret_cast<const uint8_t*>(at);
      uint4 w[NT], x[4];
      uint32_t s[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        w[t] = *reinterpret_cast<const uint4*>(p + wat + 1024 * t);
        s[t] = p[sat + 64 * t];
      }
      if constexpr (X4) {
        x[0] = *reinterpret_cast<const uint4*>(p + xat);
        const uint32_t xs = p[sat + 256 * NS];
#pragma unroll
        for (int t = 0; t < NT; ++t)
          acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(four_bits(w[t]), four_bits(x[0]), acc[t], 4, 4, 0, (int)s[t], 0,
                                                                    (int)xs);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = *reinterpret_cast<const uint4*>(p + (xat ^ 16 * e));
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int t = 0; t < NT; ++t)
            acc[t] = mfma16<BF>(spk_mx4::expand<BF>((&w[t].x)[e], spk_mx4::scale_of(s[t])), x[e], acc[t]);
      }
    }
  };
  load(kw, sa);
  load(kw + KW, sb);
  for (int st = kw; st < steps; st += 3 * KW) {
    step(st, sa, sc);
    step(st + KW, sb, sa);
    step(st + 2 * KW, sc, sb);
  }
  spk_mx4::arrived<0>();  // loads past the end still write LDS
  __syncthreads();
  auto sums = reinterpret_cast<float(*)[16][16 * NT + 1]>(sa);
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][ln][16 * t + 4 * g + i] = acc[t][i];
  __syncthreads();
  // neighbouring threads have neighbouring columns
  for (int i = threadIdx.x; i < 256 * NT * TILES; i += 64 * W) {
    const int m = i / (16 * NT * TILES), c = i - m * (16 * NT * TILES), n = blockIdx.x * 16 * NT * TILES + c;
    if (m0 + m >= a.rows || n >= a.cols) continue;
    const int first = c / (16 * NT) * KW, at = c % (16 * NT);
    float sum = sums[first][m][at];
#pragma unroll
    for (int w = 1; w < KW; ++w) sum += sums[first + w][m][at];
    if (a.res) sum += widen<BF>(a.res[(m0 + m) * a.rt + n]);
    a.out[(m0 + m) * a.ot + n] = narrow<BF>(sum);
  }
}

// A wave's tiles into out: row m and column n are this lane's first.  vec: out's and
// residual's groups of four values are aligned.
template <bool BF, int TM, int TN>
__device__ __forceinline__ void store_tile(const Mm& a, int vec, int m, int n, const floatx16 (&acc)[TN][TM]) {
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t row = m + 32 * i;
    if (row >= a.rows) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int col = n + 32 * j + 2 * e;
        float y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = acc[j][i][e + k];
        uint16_t* to = a.out + row * a.ot + col;
        const uint16_t* r = a.res + row * a.rt + col;
        if (vec && col + 4 <= a.cols) {
          if (a.res) {
            const ushort4 u = *reinterpret_cast<const ushort4*>(r);
            y[0] += widen<BF>(u.x);
            y[1] += widen<BF>(u.y);
            y[2] += widen<BF>(u.z);
            y[3] += widen<BF>(u.w);
          }
          *reinterpret_cast<ushort4*>(to) = make_ushort4(narrow<BF>(y[0]), narrow<BF>(y[1]), narrow<BF>(y[2]), narrow<BF>(y[3]));
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (col + k >= a.cols) continue;
            if (a.res) y[k] += widen<BF>(r[k]);
            to[k] = narrow<BF>(y[k]);
          }
        }
      }
  }
}

// All loads but the newest N of this wave have arrived, its LDS reads are done, and so are
// those of the workgroup's other waves.
template <int N>
__device__ __forceinline__ void meet_after() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The tile of a workgroup: those of an XCD (its ids are 8 apart) side by side, 8 tiles
// of rows to each tile of columns, so that what they share is in its L2.
__device__ __forceinline__ void tile_at(int id, int tiles_m, int tiles_n, int* tm, int* tn) {
  const int total = tiles_m * tiles_n, q = total / 8, r = total % 8, xcd = id % 8;
  int t = xcd * q + min(xcd, r) + id / 8;
  const int panel = t / (8 * tiles_n), high = min(8, tiles_m - 8 * panel);
  t -= panel * 8 * tiles_n;
  *tn = t / high;
  *tm = 8 * panel + t - *tn * high;
}

// Many rows: a workgroup of WM x WN waves takes a tile of rows of x and rows of w, a wave TM x TN
// tiles of 32 x 32 of it, the depth in stages that go straight into LDS, ahead of
// their use.  The tile is formed transposed (w is the A operand), so that a lane's
// outputs lie side by side in a row of out.  All that is loaded goes to LDS, also
// the scales: a load to registers among the others would make the compiler wait for all.
//
// What is read of a row at a time are whole lines, 128 bytes to 8 lanes: a line of which 64 or
// 32 bytes are taken is fetched again for the rest, and the loads were the bound
// (8192 x 8192 x 8192 in 4 bits with 64 bytes a time: 406 us, without products 397; so
// 344, 3.2 PFLOP/s, products alone 207, and the loads, all of whose lines an XCD's workgroups
// wait for together, still bound it; 2001 x 14336 x 4096 in 16 bits 200 us, 1.2 PFLOP/s).
// Pieces of 16 bytes lie in LDS exchanged within their line by the row's number (p ^ row % 8),
// so that 8 rows read side by side are in different banks.
// What lies past the depth is zero in x and w.
//
// The wave's rows of a matrix: L lanes to a row, which take B bytes each of a line of it.
// (A pointer to each load's rows took 30 registers more than there are.)
template <int B, int L>
struct Lines {
  const uint8_t* at;  // of this lane in the first 64 / L rows
  int64_t stride;     // of 64 / L rows
  int left;           // rows from this lane's on

  __device__ __forceinline__ Lines(const uint8_t* rows, int64_t row_stride, int first, int end, int bytes) {
    const int row = (threadIdx.x & 63) / L;
    at = rows + (first + row) * row_stride + bytes;
    stride = 64 / L * row_stride;
    left = end - first - row;
  }
  // The i-th 64 / L rows, `bytes` further; zeros where `within` is false or there are no more rows.
  __device__ __forceinline__ void load(int i, int64_t bytes, bool within, void* to) const {
    const uint8_t* here = at;
    asm("" : "+v"(here));  // the sum is formed each time, and takes no registers in between
    spk_mx4::load_lds<B>(within && 64 / L * i < left ? here + (i * stride + bytes) : reinterpret_cast<const uint8_t*>(kZero), to);
  }
};

// The scales of a wave's RW rows, a group of stages of 256 values (8 blocks) at a time: 16 bytes
// to each of L lanes of a row (SB = 16), or a byte to a dword where rows of scales are not
// of aligned 16 bytes (SB = 1).  (4 bytes of a row's line at each stage: 40 us of 380.)
template <int SB, int L, int RW>
struct Scales {
  static constexpr int kGroup = SB == 16 ? 2 * L : 1, kLanes = SB == 16 ? L : 8;
  static constexpr int kLoads = RW * kLanes / 64, kWords = SB == 16 ? 4 * L : 8;  // dwords of a row
  Lines<SB, kLanes> lines;

  __device__ __forceinline__ Scales(const uint8_t* rows, int64_t row_stride, int first, int end)
      : lines(rows, row_stride, first, end, SB * ((int)threadIdx.x % kLanes)) {}
  static __device__ __forceinline__ int half(int st) { return st / kGroup & 1; }
  // the group of stage st to the wave's place in its half
  __device__ __forceinline__ void load(int st, int blocks, uint32_t* to) const {
    const int first = st / kGroup * (8 * kGroup);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) lines.load(i, first, first + SB * ((int)threadIdx.x % kLanes) < blocks, to + (SB == 16 ? 256 : 64) * i);
  }
  // blocks 4 n + h and 4 n + 2 + h of row r in bytes 0 and 2 (SB = 16), else block 2 c + h
  static __device__ __forceinline__ uint32_t of(const uint32_t* s, int r, int st, int c, int h) {
    return SB == 16 ? s[kWords * r + 2 * (st % kGroup) + c / 2] >> (8 * h) : s[8 * r + 2 * c + h];
  }
};

// Rows in 16 bits.  64 values of x are a stage, 256 of w one: a lane's 16 bytes are a
// block, whose 4 dwords of codes are 4 products' operands.
template <bool BF, int WM, int WN, int TM, int TN, int SB>
__global__ __launch_bounds__(64 * WM * WN, 2) void mx4_tiles16_kernel(Mm a, int vec) {
  constexpr int NW = WM * WN, BM = 32 * WM * TM, BN = 32 * WN * TN;
  constexpr int PX = BM / (8 * NW), PW = BN / (8 * NW);  // loads of a wave
  static_assert(BM == 32 * NW && BN == 32 * NW, "a wave loads 32 rows of x and of w");
  using S = Scales<SB, 2, 32>;
  // an array to each stage: a load into one is then known not to touch the others
  __shared__ __align__(16) uint4 xa[BM * 8], xb[BM * 8], wa[BN * 8], wb[BN * 8];
  __shared__ __align__(16) uint32_t sc[2 * BN * S::kWords];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 31, h = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;
  int tm, tn;
  tile_at(blockIdx.x, (a.rows + BM - 1) / BM, (a.cols + BN - 1) / BN, &tm, &tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int blocks = a.depth / 32, stages = (blocks + 7) / 8;

  const int piece = lane % 8 ^ lane / 8;
  const Lines<16, 8> xl(reinterpret_cast<const uint8_t*>(a.x), 2 * a.xt, m0 + 32 * wave, a.rows, 16 * piece);
  const Lines<16, 8> wl(a.wc, a.wct, n0 + 32 * wave, a.cols, 16 * piece);
  const S scales(a.ws, a.wst, n0 + 32 * wave, a.cols);
  auto load_x = [&](int st, uint4* x) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PX; ++i) xl.load(i, 128 * (int64_t)st, 2 * st + piece / 4 < blocks, x + 64 * (PX * wave + i));
  };
  auto load_w = [&](int st, int i, uint4* w) __attribute__((always_inline)) {
    wl.load(i, 128 * (int64_t)st, 8 * st + piece < blocks, w + 64 * (PW * wave + i));
  };
  auto load_s = [&](int st) __attribute__((always_inline)) {
    scales.load(st, blocks, sc + (S::half(st) * BN + 32 * wave) * S::kWords);
  };
  floatx16 acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.0f;
  const int xbase = (32 * wm * TM + ln) * 8, nbase = 32 * wn * TN + ln, flip = ln & 7;
  // Quarter q of stage st of w, with the stage of x at `x`; the next ones to xn and wnext.
  auto step = [&](int st, int q, const uint4* x, uint4* xn, const uint4* w, uint4* wnext) __attribute__((always_inline)) {
    uint4 codes[TN], v[2][TM];
    float scale[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const uint32_t* s = sc + S::half(st) * BN * S::kWords;
      scale[j] = spk_mx4::scale_of(S::of(s, nbase + 32 * j, st, q, h) >> (SB == 16 ? 16 * (q & 1) : 0) & 255);
      codes[j] = w[8 * nbase + 256 * j + ((2 * q + h) ^ flip)];
    }
    __builtin_amdgcn_sched_barrier(0);  // the scales, whose halves the compiler does not tell apart, before loads of them
    if (q == 0 && (st + 1) % S::kGroup == 0) load_s(st + 1);
    load_w(st + 1, q, wnext);
    load_x(4 * st + q + 1, xn);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < TM; ++i) v[0][i] = x[xbase + 256 * i + (4 * h ^ flip)];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (c < 3) {
#pragma unroll
        for (int i = 0; i < TM; ++i) v[(c + 1) & 1][i] = x[xbase + 256 * i + ((4 * h + c + 1) ^ flip)];
      }
      uint4 f[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) f[j] = spk_mx4::expand<BF>((&codes[j].x)[c], scale[j]);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[j][i] = mfma32<BF>(f[j], v[c & 1][i], acc[j][i]);
    }
    meet_after<0>();
  };
  auto stage = [&](int st, const uint4* w, uint4* wnext) __attribute__((always_inline)) {
    step(st, 0, xa, xb, w, wnext);
    step(st, 1, xb, xa, w, wnext);
    step(st, 2, xa, xb, w, wnext);
    step(st, 3, xb, xa, w, wnext);
  };
  load_s(0);
#pragma unroll
  for (int c = 0; c < 4; ++c) load_w(0, c, wa);
  load_x(0, xa);
  meet_after<0>();
  int st = 0;
  for (; st + 2 <= stages; st += 2) {
    stage(st, wa, wb);
    stage(st + 1, wb, wa);
  }
  if (st < stages) stage(st, wa, wb);
  store_tile<BF, TM, TN>(a, vec, m0 + 32 * wm * TM + ln, n0 + 32 * wn * TN + 4 * h, acc);
}

// Rows in 4 bits: a stage is 256 values of x and of w and their eight scales, which
// the products apply.
template <bool BF, int WM, int WN, int TM, int TN, int SB>
__global__ __launch_bounds__(64 * WM * WN, 2) void mx4_tiles4_kernel(Mm a, int vec) {
  constexpr int NW = WM * WN, BM = 32 * WM * TM, BN = 32 * WN * TN, R = BM + BN;
  static_assert(BM == 32 * NW && BN == 32 * NW, "a wave loads 64 rows, all of x or all of w");
  using S = Scales<SB, 1, 64>;
  __shared__ __align__(16) uint4 sa[R * 8], sb[R * 8];
  __shared__ __align__(16) uint32_t sc[2 * R * S::kWords], unused[SB == 16 ? 64 * NW : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 31, h = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;
  int tm, tn;
  tile_at(blockIdx.x, (a.rows + BM - 1) / BM, (a.cols + BN - 1) / BN, &tm, &tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int blocks = a.depth / 32, stages = (blocks + 7) / 8;

  // rows of x, then of w
  const int piece = lane % 8 ^ lane / 8;
  const bool x_wave = wave < NW / 2;
  const int row = x_wave ? m0 + 64 * wave : n0 + 64 * wave - BM, end = x_wave ? a.rows : a.cols;
  const Lines<16, 8> lines(x_wave ? a.xc : a.wc, x_wave ? a.xct : a.wct, row, end, 16 * piece);
  const S scales(x_wave ? a.xs : a.ws, x_wave ? a.xst : a.wst, row, end);
  auto load = [&](int st, uint4* to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) lines.load(i, 128 * (int64_t)st, 8 * st + piece < blocks, to + 64 * (8 * wave + i));
  };
  auto load_s = [&](int st) __attribute__((always_inline)) {
    scales.load(st, blocks, sc + (S::half(st) * R + 64 * wave) * S::kWords);
  };
  // A line that comes from memory keeps all of an XCD's workgroups waiting for it that share it:
  // each asks two stages ahead for a part of those it has in common with its neighbours,
  // of which a dword comes that nobody uses (8192 x 8192 x 8192: 361 us without, 344).
  const bool ofx = lane < 32;
  const int arow = ofx ? min(m0 + BM / 4 * (tn % 4) + 8 * wave + lane / 4, a.rows - 1)
                       : min(n0 + BN / 4 * (tm % 4) + 8 * wave + lane / 4 - 8, a.cols - 1);
  const uint8_t* ap = ofx ? a.xc + arow * a.xct : a.wc + arow * a.wct;
  auto ahead = [&](int st) __attribute__((always_inline)) {
    if constexpr (SB == 16)  // with SB = 1 there is no room for it
      spk_mx4::load_lds<4>(8 * (st + 2) < blocks ? ap + 128 * (int64_t)(st + 2) : reinterpret_cast<const uint8_t*>(kZero), unused + 64 * wave);
  };
  floatx16 acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.0f;
  const int mbase = 32 * wm * TM + ln, nbase = BM + 32 * wn * TN + ln, flip = ln & 7;
  auto step = [&](int st, const uint4* x, uint4* to) __attribute__((always_inline)) {
    const uint32_t* s = sc + S::half(st) * R * S::kWords;
    uint32_t xsc[4][TM], wsc[4][TN];
#pragma unroll
    for (int c = 0; c < 4; c += SB == 16 ? 2 : 1) {
#pragma unroll
      for (int i = 0; i < TM; ++i) xsc[c][i] = S::of(s, mbase + 32 * i, st, c, h);
#pragma unroll
      for (int j = 0; j < TN; ++j) wsc[c][j] = S::of(s, nbase + 32 * j, st, c, h);
    }
    __builtin_amdgcn_sched_barrier(0);  // the scales, whose halves the compiler does not tell apart, before loads of them
    if ((st + 1) % S::kGroup == 0) load_s(st + 1);
    uint4 f[2][TN], v[2][TM];
    auto operands = [&](int c) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < TN; ++j) f[c & 1][j] = x[8 * nbase + 256 * j + ((2 * c + h) ^ flip)];
#pragma unroll
      for (int i = 0; i < TM; ++i) v[c & 1][i] = x[8 * mbase + 256 * i + ((2 * c + h) ^ flip)];
    };
    load(st + 1, to);
    __builtin_amdgcn_sched_barrier(0);
    operands(0);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (c < 3) operands(c + 1);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          if (SB == 16 && c % 2)
            acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(four_bits(f[c & 1][j]), four_bits(v[c & 1][i]), acc[j][i], 4, 4,
                                                                        2, (int)wsc[c & 2][j], 2, (int)xsc[c & 2][i]);
          else
            acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(four_bits(f[c & 1][j]), four_bits(v[c & 1][i]), acc[j][i], 4, 4,
                                                                        0, (int)wsc[c][j], 0, (int)xsc[c][i]);
        }
    }
    ahead(st);
    meet_after<SB == 16>();  // all but that
  };
  load_s(0);
  load(0, sa);
  meet_after<0>();
  int st = 0;
  for (; st + 2 <= stages; st += 2) {
    step(st, sa, sb);
    step(st + 1, sb, sa);
  }
  if (st < stages) step(st, sa, sb);
  spk_mx4::arrived<0>();
  store_tile<BF, TM, TN>(a, vec, m0 + 32 * wm * TM + ln, n0 + 32 * wn * TN + 4 * h, acc);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

size_t size_of(int dtype) { return dtype == SPK_F32 ? 4 : 2; }

int check_mx4(const SpkMx4& m, int64_t rows, int32_t cols, const char* who, const char* name) {
  if (!m.codes || !m.scales) return spk::fail(SPK_ERR_NULL, "%s: codes or scales of %s is NULL", who, name);
  if (!spk::aligned(m.codes, 16) || m.code_stride % 16)
    return spk::fail(SPK_ERR_ALIGN, "%s: codes of %s and their stride (%lld bytes) must be 16-byte aligned", who, name,
                     (long long)m.code_stride);
  if (rows > 1 && (m.code_stride < cols / 2 || m.scale_stride < cols / 32))
    return spk::fail(SPK_ERR_SHAPE, "%s: strides of %s (codes %lld, scales %lld) are less than a row of %d values", who,
                     name, (long long)m.code_stride, (long long)m.scale_stride, cols);
  return SPK_OK;
}

// The arguments that quantisation and its inverse share.  1: there is nothing to do.
int fill_rows(const SpkMx4* m, const void* x, int32_t dtype, int64_t stride, int64_t rows, int32_t cols, const char* who,
              Rows* a) {
  if (!m) return spk::fail(SPK_ERR_NULL, "%s: NULL args", who);
  if (dtype != SPK_F32 && dtype != SPK_F16 && dtype != SPK_BF16)
    return spk::fail(SPK_ERR_ARG, "%s: dtype %d (SPK_F32, SPK_F16 or SPK_BF16)", who, dtype);
  if (rows < 0 || cols < 0 || cols % 32)
    return spk::fail(SPK_ERR_SHAPE, "%s: %lld rows of %d values (a multiple of 32)", who, (long long)rows, cols);
  if (rows == 0 || cols == 0) return 1;
  if (rows > INT32_MAX || rows * (cols / 8) > INT32_MAX)
    return spk::fail(SPK_ERR_SHAPE, "%s: %lld rows of %d values (below 2^34 in all)", who, (long long)rows, cols);
  if (!x) return spk::fail(SPK_ERR_NULL, "%s: the rows are NULL", who);
  if (!spk::aligned(x, 16) || stride * (int64_t)size_of(dtype) % 16)
    return spk::fail(SPK_ERR_ALIGN, "%s: the rows and their stride (%lld elements) must be 16-byte aligned", who,
                     (long long)stride);
  if (rows > 1 && stride < cols)
    return spk::fail(SPK_ERR_SHAPE, "%s: stride %lld of rows of %d values", who, (long long)stride, cols);
  if (const int rc = check_mx4(*m, rows, cols, who, "the 4-bit rows")) return rc;
  a->codes = m->codes;
  a->scales = m->scales;
  a->stride = stride;
  a->code_stride = m->code_stride;
  a->scale_stride = m->scale_stride;
  a->groups = (uint32_t)(rows * (cols / 8));
  a->per_row = (uint32_t)cols / 8;
  a->div = spk_paged::page_div(a->per_row);
  return SPK_OK;
}

template <bool X4, bool BF, int WM, int WN, int TM, int TN>
void launch_tiles(const Mm& a, int vec, hipStream_t s) {
  constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN;
  const dim3 grid(((a.rows + BM - 1) / BM) * ((a.cols + BN - 1) / BN)), block(64 * WM * WN);
  const auto whole = [&](const uint8_t* scales, int64_t stride) { return a.depth % 512 == 0 && stride % 16 == 0 && spk::aligned(scales, 16); };
  const bool wide = whole(a.ws, a.wst) && (!X4 || whole(a.xs, a.xst));
  if constexpr (X4) {
    if (wide)
      hipLaunchKernelGGL((mx4_tiles4_kernel<BF, WM, WN, TM, TN, 16>), grid, block, 0, s, a, vec);
    else
      hipLaunchKernelGGL((mx4_tiles4_kernel<BF, WM, WN, TM, TN, 1>), grid, block, 0, s, a, vec);
  } else if (wide) {
    hipLaunchKernelGGL((mx4_tiles16_kernel<BF, WM, WN, TM, TN, 16>), grid, block, 0, s, a, vec);
  } else {
    hipLaunchKernelGGL((mx4_tiles16_kernel<BF, WM, WN, TM, TN, 1>), grid, block, 0, s, a, vec);
  }
}

template <bool X4, bool BF, int XR, int NT, int KW>
void launch_few(const Mm& a, hipStream_t s) {
  constexpr int W = KW > 4 ? KW : 4, N = 16 * NT * W / KW;
  const dim3 grid((a.cols + N - 1) / N, (a.rows + 15) / 16), block(64 * W);
  const bool dwords = a.depth % 128 == 0 && a.wst % 4 == 0 && spk::aligned(a.ws, 4) && (!X4 || (a.xst % 4 == 0 && spk::aligned(a.xs, 4)));
  if (dwords)
    hipLaunchKernelGGL((mx4_few_rows_kernel<X4, BF, XR, NT, KW, 4>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((mx4_few_rows_kernel<X4, BF, XR, NT, KW, 1>), grid, block, 0, s, a);
}

// Tiles of 16 x 16 of the result.
int64_t small_tiles(const Mm& a) { return (int64_t)((a.cols + 15) / 16) * ((a.rows + 15) / 16); }

int64_t big_tiles(const Mm& a) { return (int64_t)((a.cols + 255) / 256) * ((a.rows + 255) / 256); }

// As many columns to a wave as leave some 800 waves, each with a quarter of the depth until
// there are enough without (1 row, us with (4, 1), (4, 4), (2, 4), (1, 4) of NT and KW: 1024 x 3584
// -, 5.7, 4.6, 4.1; 14336 x 4096 -, 8.2, 8.7, 10.9; 32768 x 4096 24.1, 14.6, -, -; 248320 x 1024
// 29.1, 32.4, -, -).
template <bool X4, bool BF, int XR>
void launch_few_rows(const Mm& a, hipStream_t s) {
  const int64_t tiles = small_tiles(a);
  if (tiles >= 8192)
    launch_few<X4, BF, XR, 4, 1>(a, s);
  else if (tiles >= 800)
    launch_few<X4, BF, XR, 4, 4>(a, s);
  else if (tiles >= 400)
    launch_few<X4, BF, XR, 2, 4>(a, s);
  else
    launch_few<X4, BF, XR, 1, 4>(a, s);
}

template <bool X4, bool BF>
void launch_matmul(const Mm& a, hipStream_t s) {
  const int vec = spk::aligned(a.out, 8) && a.ot % 4 == 0 && (!a.res || (spk::aligned(a.res, 8) && a.rt % 4 == 0));
  // Few rows, us with the kernel for them and with tiles of 128 x 128 (which take about the same time
  // until the chip is full): 300 times 4096 x 4096 (4864 small tiles) 33 and 39, 400 (6400) 45 and
  // 40; 64 times 14336 x 4096 (3584) 29 and 39, 100 (6272) 46 and 40.  Rows in 4 bits: 100 times
  // 4096 x 4096 (1792) 12 and 15, 200 (3328) 19 and 16; 64 times 14336 x 4096 23 and 17.
  // Tiles of 256 x 256 pay once most of the chip has one (us with them and with tiles of 128 x 128): 2000
  // times 4096 x 4096 (128 tiles) 91 and 69, 2700 (176) 100 and 100, 3300 (208) 104 and 122; rows in 4
  // bits 42 and 31, 47 and 47, 48 and 54; 2000 times 7168 x 1024 (224) 38 and 40, 22.7 and 23.4.
  if (a.rows <= 16 || small_tiles(a) < (X4 ? 2200 : 5000))
    a.rows <= 4 && !X4 ? launch_few_rows<X4, BF, 4>(a, s) : launch_few_rows<X4, BF, 16>(a, s);
  else if (big_tiles(a) >= 200)
    launch_tiles<X4, BF, 2, 4, 4, 2>(a, vec, s);
  else
    launch_tiles<X4, BF, 2, 2, 2, 2>(a, vec, s);
}

}  // namespace

extern "C" int spk_mx4_quantize(const void* x, int32_t dtype, int64_t x_stride, int64_t rows, int32_t cols,
                                const SpkMx4* out, spk_stream_t stream) {
  const char* who = "spk_mx4_quantize";
  Rows a{};
  if (const int rc = fill_rows(out, x, dtype, x_stride, rows, cols, who, &a)) return rc < 0 ? rc : SPK_OK;
  a.x = x;
  hipStream_t s = spk::to_hip(stream);
  const dim3 grid((a.groups + 255) / 256);
  if (dtype == SPK_F32)
    hipLaunchKernelGGL(mx4_quantize_kernel<SPK_F32>, grid, dim3(256), 0, s, a);
  else if (dtype == SPK_F16)
    hipLaunchKernelGGL(mx4_quantize_kernel<SPK_F16>, grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(mx4_quantize_kernel<SPK_BF16>, grid, dim3(256), 0, s, a);
  return spk::check_launch(who);
}

extern "C" int spk_mx4_dequantize(const SpkMx4* m, int64_t rows, int32_t cols, int32_t dtype, void* y, int64_t y_stride,
                                  spk_stream_t stream) {
  const char* who = "spk_mx4_dequantize";
  Rows a{};
  if (const int rc = fill_rows(m, y, dtype, y_stride, rows, cols, who, &a)) return rc < 0 ? rc : SPK_OK;
  a.y = y;
  hipStream_t s = spk::to_hip(stream);
  const dim3 grid((a.groups + 255) / 256);
  if (dtype == SPK_F32)
    hipLaunchKernelGGL(mx4_dequantize_kernel<SPK_F32>, grid, dim3(256), 0, s, a);
  else if (dtype == SPK_F16)
    hipLaunchKernelGGL(mx4_dequantize_kernel<SPK_F16>, grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(mx4_dequantize_kernel<SPK_BF16>, grid, dim3(256), 0, s, a);
  return spk::check_launch(who);
}

extern "C" int spk_mx4_matmul(const SpkMx4MatmulArgs* p, spk_stream_t stream) {
  const char* who = "spk_mx4_matmul";
  if (!p) return spk::fail(SPK_ERR_NULL, "%s: NULL args", who);
  if (p->dtype != SPK_F16 && p->dtype != SPK_BF16)
    return spk::fail(SPK_ERR_ARG, "%s: dtype %d (SPK_F16 or SPK_BF16)", who, p->dtype);
  if (p->rows < 0 || p->out_dim < 0 || p->in_dim <= 0 || p->in_dim % 32)
    return spk::fail(SPK_ERR_SHAPE, "%s: rows %d out_dim %d in_dim %d (a positive multiple of 32)", who, p->rows, p->out_dim,
                     p->in_dim);
  if (p->rows == 0 || p->out_dim == 0) return SPK_OK;
  if (p->rows > 1 << 30 || p->out_dim > 1 << 30 || (int64_t)((p->rows + 255) / 256) * ((p->out_dim + 255) / 256) >= 1 << 23)
    return spk::fail(SPK_ERR_SHAPE, "%s: rows %d out_dim %d (up to 2^30 each and 2^39 results)", who, p->rows, p->out_dim);
  if (const int rc = check_mx4(p->w, p->out_dim, p->in_dim, who, "w")) return rc;
  if (p->x) {
    if (!spk::aligned(p->x, 16) || p->x_stride % 8)
      return spk::fail(SPK_ERR_ALIGN, "%s: x and its stride (%lld elements) must be 16-byte aligned", who, (long long)p->x_stride);
    if (p->rows > 1 && p->x_stride < p->in_dim)
      return spk::fail(SPK_ERR_SHAPE, "%s: x_stride %lld < in_dim %d", who, (long long)p->x_stride, p->in_dim);
  } else if (const int rc = check_mx4(p->x4, p->rows, p->in_dim, who, "x4")) {
    return rc;
  }
  if (!p->out) return spk::fail(SPK_ERR_NULL, "%s: out is NULL", who);
  if (!spk::aligned(p->out, 2) || !spk::aligned(p->residual, 2))
    return spk::fail(SPK_ERR_ALIGN, "%s: out and residual must be 2-byte aligned", who);
  if (p->rows > 1 && (p->out_stride < p->out_dim || (p->residual && p->residual_stride < p->out_dim)))
    return spk::fail(SPK_ERR_SHAPE, "%s: out_stride %lld, residual_stride %lld < out_dim %d", who, (long long)p->out_stride,
                     (long long)p->residual_stride, p->out_dim);
  if (p->out == p->residual && p->rows > 1 && p->out_stride != p->residual_stride)
    return spk::fail(SPK_ERR_ARG, "%s: out is residual with another stride", who);
  Mm a{};
  a.x = static_cast<const uint16_t*>(p->x);
  a.xc = p->x4.codes;
  a.xs = p->x4.scales;
  a.wc = p->w.codes;
  a.ws = p->w.scales;
  a.res = static_cast<const uint16_t*>(p->residual);
  a.out = static_cast<uint16_t*>(p->out);
  a.xt = p->x_stride;
  a.xct = p->x4.code_stride;
  a.xst = p->x4.scale_stride;
  a.wct = p->w.code_stride;
  a.wst = p->w.scale_stride;
  a.rt = p->residual_stride;
  a.ot = p->out_stride;
  a.rows = p->rows;
  a.cols = p->out_dim;
  a.depth = p->in_dim;
  hipStream_t s = spk::to_hip(stream);
  if (p->dtype == SPK_BF16)
    p->x ? launch_matmul<false, true>(a, s) : launch_matmul<true, true>(a, s);
  else
    p->x ? launch_matmul<false, false>(a, s) : launch_matmul<true, false>(a, s);
  return spk::check_launch(who);
}
