// verify.hip -- verification of drafted tokens against the target's
// distribution (spk_verify_drafts): how many drafts of each sequence are
// accepted, and the token drawn from what the first refused one leaves.
//
// Three steps, each one launch:
//   1. row statistics (logits only): maximum, sum of exponentials and the
//      lowest index of the maximum, of pieces of every row;
//   2. per sequence and piece of the vocabulary: the acceptances in order
//      (every workgroup of a sequence finds the same stop), then the piece's
//      share of the residual max(p - q, 0) of the row that stopped;
//   3. per sequence: the piece in which the running sum passes u * total, and
//      the token in it.
// The outcome hangs on comparisons, so what enters one is fp64 (products u q(d) of
// two values, the exponentials of the drawn row, the running sums) but for what
// normalises a row of logits: that sum is of fp32 exponentials, each off by a few
// units in the last place but none in common (log2(e) / T enters as two floats),
// eight at a time in fp32 and those in fp64 (fp64 exponentials of every row would
// take several times as long as step 2, which has them for two a sequence).
//
// What bounds it (64 sequences, 222 rows and 158 drafts' rows of 248,320 fp16
// logits): step 1 reads 190 MB in 39 us, 4.8 TB/s, with as much time in its
// exponentials (10 vector instructions' time an entry) as in the reads; step 2
// takes 36 us, of which the two fp64 exponentials of an entry need about 20 and
// the way to the row that stopped, a chain of loads, the rest (as a launch of its
// own it gains 2 us there and costs 3 with one sequence); step 3 takes 9 us, a
// chain of loads and meetings of one workgroup.
#include <algorithm>

#include "capi_common.hpp"
#include "numerics.hpp"
#include "paged.hpp"

namespace {

typedef _Float16 half_t;
typedef __bf16 bf_t;

struct Verify {
  const void *target, *draft;
  int64_t target_stride, draft_stride;
  const int32_t *cu, *tokens, *context;
  const float *temperature, *u_accept, *u_sample;
  int32_t *out, *accepted, *context_out;
  float* logprobs;
  struct Stat* stats;   // [2][total_tokens][parts]
  struct Left* left;    // [num_seqs]
  double* mass;         // [num_seqs][pieces][2]: residual, target
  int32_t vocab, num_seqs, total, parts, part_len, pieces;
  int32_t probs;
};

struct Stat {
  float max;
  int32_t arg;  // lowest index of the maximum, -1 where nothing is larger than -inf
  double sum;
};

// What a sequence's draw needs of the row that stopped.
struct Left {
  double p_max, p_sum, q_max, q_sum;
  int32_t row;      // -1: nothing is drawn
  int32_t refused;  // the draft after the row, -1 where there was none
};

constexpr int kMaxParts = 64;   // of a row's statistics: one for each lane

__device__ __forceinline__ bool better(float m, int a, float om, int oa) {
  return om > m || (om == m && (uint32_t)oa < (uint32_t)a);  // -1 is the largest index
}

// log2(e) / T, also as two floats; greedy rows count at T = 1.  Both are larger
// than 0, so that a logit of -inf stays one: T is at most the largest finite
// float, and the second, a denormal from some 7e30 on, at least the smallest of
// them (off by half a step of theirs, 1.7e-7 of log2(e) / T where T is largest).
struct Heat {
  float c, lo;
  double scale;
  bool greedy;
};
__device__ __forceinline__ Heat heat_of(const Verify& a, int s) {
  float t = a.temperature && s < a.num_seqs ? a.temperature[s] : 1.0f;
  Heat h;
  h.greedy = !(t > 0.0f);
  if (h.greedy) t = 1.0f;
  h.scale = 1.4426950408889634 / fmin(fmax((double)t, 1e-30), 3.4028234663852886e38);
  h.c = __uint_as_float(__float_as_uint((float)h.scale) - 1);
  h.lo = fmaxf((float)(h.scale - (double)h.c), __uint_as_float(1));
  return h;
}

// 2^x, x <= 0 or NaN: 2^k e^(r ln 2), |r| <= 1/2, the exponential's series to
// the tenth power (2e-13 relative).
__device__ __forceinline__ double exp2_f64(double x) {
  const double k = __builtin_rint(x), t = (x - k) * 0.6931471805599453;
  double p = 1.0 / 3628800;
  p = __builtin_fma(p, t, 1.0 / 362880);
  p = __builtin_fma(p, t, 1.0 / 40320);
  p = __builtin_fma(p, t, 1.0 / 5040);
  p = __builtin_fma(p, t, 1.0 / 720);
  p = __builtin_fma(p, t, 1.0 / 120);
  p = __builtin_fma(p, t, 1.0 / 24);
  p = __builtin_fma(p, t, 1.0 / 6);
  p = __builtin_fma(p, t, 0.5);
  p = __builtin_fma(p, t, 1.0);
  p = __builtin_fma(p, t, 1.0);
  return x < -1000.0 ? 0.0 : __builtin_ldexp(p, (int)k);
}

// Sums and minima over the wave, in every lane, and the inclusive running sum:
// lane swaps and DPP moves, an LDS permute is ten times as long.
__device__ __forceinline__ double pair_of(uint32_t lo, uint32_t hi) { return __longlong_as_double((long long)((uint64_t)hi << 32 | lo)); }
template <class F>
__device__ __forceinline__ double moved(double v, F f) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  return pair_of(f((uint32_t)u), f((uint32_t)(u >> 32)));
}
__device__ __forceinline__ double wave_sum(double v) {
  v += moved(v, [](uint32_t u) { return spk::lane_xor32_u(u); });
  v += moved(v, [](uint32_t u) { return spk::lane_xor16_u(u); });
  v += moved(v, [](uint32_t u) { return spk::row_ror_u<8>(u); });
  v += moved(v, [](uint32_t u) { return spk::row_ror_u<4>(u); });
  v += moved(v, [](uint32_t u) { return spk::row_ror_u<2>(u); });
  v += moved(v, [](uint32_t u) { return spk::row_ror_u<1>(u); });
  return v;
}
__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
  v = min(v, spk::lane_xor32_u(v));
  v = min(v, spk::lane_xor16_u(v));
  v = min(v, spk::row_ror_u<8>(v));
  v = min(v, spk::row_ror_u<4>(v));
  v = min(v, spk::row_ror_u<2>(v));
  return min(v, spk::row_ror_u<1>(v));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double from_below(double v) {  // +0 where nothing comes
  return moved(v, [](uint32_t u) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, CTRL, ROWS, 0xF, false); });
}
__device__ __forceinline__ double wave_scan(double v) {
  v += from_below<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v += from_below<0x112, 0xF>(v);
  v += from_below<0x114, 0xF>(v);
  v += from_below<0x118, 0xF>(v);
  v += from_below<0x142, 0xA>(v);  // lane 15 of a row to the next row
  v += from_below<0x143, 0xC>(v);  // lane 31 to the upper half
  return v;
}

// grid (parts, total_tokens, sides); block 256
template <class T>
__global__ __launch_bounds__(256) void verify_stats_kernel(Verify a) {
  constexpr int VE = 16 / sizeof(T);
  __shared__ Stat red[4];
  const int t = blockIdx.y, side = blockIdx.z;
  const int lane = threadIdx.x & 63;
  const int s = spk_paged::seq_of_token(a.cu, a.num_seqs, t, lane);
  if (s >= a.num_seqs || (side && t + 1 >= a.cu[s + 1])) return;  // no row of a sequence, or nothing was drafted after it
  const Heat heat = heat_of(a, s);
  const int c0 = blockIdx.x * a.part_len, n = min(a.part_len, a.vocab - c0);
  const T* row = static_cast<const T*>(side ? a.draft : a.target) + t * (side ? a.draft_stride : a.target_stride) + c0;
  const int head = min(n, (int)(((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16) / sizeof(T)));
  const int vecs = (n - head) / VE, tail = n - head - vecs * VE;

  float m = -INFINITY;
  int arg = -1;
  double sum = 0.0;
  auto shrink = [&](float from, float to) {  // of a sum whose maximum was `from`
    const float d = from - to;
    return (double)__builtin_amdgcn_exp2f(__builtin_fmaf(d, heat.lo, d * heat.c));
  };
  // W runs of `count` entries, at first, first + apart, ...: one look at the
  // maximum for all, an fp32 sum of each
  auto take = [&](const float* x, int W, int count, int first, int apart) __attribute__((always_inline)) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < W * count; ++i) top = fmaxf(top, x[i]);
    if (top > m) {
      if (m != -INFINITY) sum *= shrink(m, top);
      m = top;
#pragma unroll
      for (int w = W - 1; w >= 0; --w)
#pragma unroll
        for (int i = count - 1; i >= 0; --i)
          if (x[w * count + i] == top) arg = first + w * apart + i;
    }
    const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      float part = 0.0f;
#pragma unroll
      for (int i = 0; i < count; ++i) {
        const float d = x[w * count + i] - base;
        part += __builtin_amdgcn_exp2f(__builtin_fmaf(d, heat.lo, d * heat.c));
      }
      sum += (double)part;
    }
  };
  if ((int)threadIdx.x < head) {
    const float x[1] = {(float)row[threadIdx.x]};
    take(x, 1, 1, c0 + threadIdx.x, 0);
  }
  const uint4* from = reinterpret_cast<const uint4*>(row + head);
  auto widen = [&](uint4 u, float* x) __attribute__((always_inline)) {
    T e[VE];
    __builtin_memcpy(e, &u, 16);
#pragma unroll
    for (int i = 0; i < VE; ++i) x[i] = (float)e[i];
  };
  int v = threadIdx.x;
  constexpr int W = 4;
  for (; v + 768 < vecs; v += 1024) {  // four loads under way
    const uint4 u[4] = {from[v], from[v + 256], from[v + 512], from[v + 768]};
#pragma unroll
    for (int w = 0; w < 4; w += W) {
      float x[W * VE];
#pragma unroll
      for (int i = 0; i < W; ++i) widen(u[w + i], x + i * VE);
      take(x, W, VE, c0 + head + (v + 256 * w) * VE, 256 * VE);
    }
  }
  for (; v < vecs; v += 256) {
    float x[VE];
    widen(from[v], x);
    take(x, 1, VE, c0 + head + v * VE, 0);
  }
  if ((int)threadIdx.x < tail) {
    const float x[1] = {(float)row[n - tail + threadIdx.x]};
    take(x, 1, 1, c0 + n - tail + threadIdx.x, 0);
  }
  {
    const float top = spk::wave_max(m);
    if (m != top && m != -INFINITY) sum *= shrink(m, top);
    sum = wave_sum(sum);
    arg = (int)wave_min(m == top ? (uint32_t)arg : ~0u);
    m = top;
  }
  auto join = [&](float om, int oa, double os) {
    if (om > m)
      sum = (m == -INFINITY ? sum : sum * shrink(m, om)) + os;
    else if (m > om)
      sum += om == -INFINITY ? os : os * shrink(om, m);
    else
      sum += os;
    if (better(m, arg, om, oa)) arg = oa;
    m = fmaxf(m, om);
  };
  if (lane == 0) red[threadIdx.x >> 6] = {m, arg, sum};
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w) join(red[w].max, red[w].arg, red[w].sum);
    a.stats[((int64_t)side * a.total + t) * a.parts + blockIdx.x] = {m, arg, sum};
  }
}

// log x: the fp32 logarithm of the mantissa and one Newton step (1e-14).
__device__ __forceinline__ double log_f64(double x) {
  const double m = __builtin_amdgcn_frexp_mant(x), near = (double)__builtin_amdgcn_logf((float)m);
  const double y = near + (m * exp2_f64(-near) - 1.0) * 1.4426950408889634 + (double)__builtin_amdgcn_frexp_exp(x);
  return x == 0.0 ? -__builtin_inf() : x < __builtin_inf() ? y * 0.6931471805599453 : x;
}

// A lane's part of a row's statistics, and the row's from all lanes' parts, in
// every lane of the wave.
__device__ __forceinline__ Stat part_of(const Verify& a, int side, int t, int lane) {
  Stat r{-INFINITY, -1, 0.0};
  if (lane < a.parts) r = a.stats[((int64_t)side * a.total + t) * a.parts + lane];
  return r;
}
__device__ __forceinline__ Stat joined(const Stat& r, const Heat& heat) {
  const float m = spk::wave_max(r.max);
  const double sum = r.max == -INFINITY || r.max == m ? r.sum : r.sum * exp2_f64(((double)r.max - (double)m) * heat.scale);
  return {m, (int)wave_min(r.max == m ? (uint32_t)r.arg : ~0u), wave_sum(sum)};
}

// What entry x of a row counts: 2^((x - max) scale) / sum of logits, itself of
// probabilities; and its logarithm, without the exponential's underflow.
__device__ __forceinline__ double chance(bool probs, float x, double max, double sum, const Heat& heat) {
  return probs ? (double)x : exp2_f64(((double)x - max) * heat.scale) / sum;
}
__device__ __forceinline__ float log_chance(bool probs, float x, double max, double sum, const Heat& heat) {
  return (float)(probs ? log_f64((double)x) : ((double)x - max) * heat.scale * 0.6931471805599453 - log_f64(sum));
}

// The same for many entries of a row: with k the integer next to 32 (x - max)
// scale, 2^(k / 32) / sum from a table of 32 (each in LDS banks of its own) and
// the rest's exponential as its series to the fifth power (2e-15 relative; the
// table's is exp2_f64's).
template <class T>
struct Dist {
  const T* row;
  const double* table;
  double max, scale;
  bool probs;
  __device__ __forceinline__ void set(const Verify& a, const T* r, double m, const Heat& heat, const double* t) {
    row = r;
    table = t;
    probs = a.probs;
    max = m;
    scale = 32.0 * heat.scale;
  }
  __device__ __forceinline__ double of(float x) const {
    if (probs) return (double)x;
    constexpr double kWhole = 6755399441055744.0;  // 1.5 2^52: a sum's low word is the integer next to the other
    constexpr double w = 0.6931471805599453 / 32;
    const double e = fmax(((double)x - max) * scale, -1048576.0), y = e + kWhole, t = e - (y - kWhole);
    const int k = (int)(uint32_t)(uint64_t)__double_as_longlong(y);
    double p = w * w * w * w * w / 120;
    p = __builtin_fma(p, t, w * w * w * w / 24);
    p = __builtin_fma(p, t, w * w * w / 6);
    p = __builtin_fma(p, t, w * w / 2);
    p = __builtin_fma(p, t, w);
    p = __builtin_fma(p, t, 1.0);
    return __builtin_ldexp(table[k & 31] * p, k >> 5);
  }
};

struct Span {
  int first, rows;
};
__device__ __forceinline__ Span span_of(const Verify& a, int s) {
  const int first = min(max(a.cu[s], 0), a.total);
  return {first, min(max(a.cu[s + 1], first), a.total) - first};
}

// What a row leaves for token i: the residual where a draft `d` was refused
// there (d < 0: the row itself).
template <class T>
struct Rest {
  Dist<T> p, q;
  bool drafted;  // q is there
  int d;
  __device__ __forceinline__ void of(int i, float x, float y, double* rest, double* base) const {
    const double u = p.of(x);
    *base = u;
    if (d < 0) {
      *rest = u;
    } else if (drafted) {
      const double v = u - q.of(y);
      *rest = v > 0.0 || v != v ? v : 0.0;
    } else {
      *rest = i == d ? 0.0 : u;
    }
  }
};

// By all threads of a workgroup, which meet in it; `table` is in LDS.
template <class T>
__device__ __forceinline__ Rest<T> rest_of(const Verify& a, const Heat& heat, const Left& l, double* table) {
  Rest<T> r;
  r.drafted = l.refused >= 0 && a.draft;
  r.p.set(a, static_cast<const T*>(a.target) + l.row * a.target_stride, l.p_max, heat, table);
  r.q.set(a, r.drafted ? static_cast<const T*>(a.draft) + l.row * a.draft_stride : r.p.row, l.q_max, heat, table + 32);
  r.d = l.refused;
  if (threadIdx.x < 64) {
    const double sum = threadIdx.x < 32 ? l.p_sum : l.q_sum;
    // a row without weight is no distribution
    table[threadIdx.x] = sum > 0.0 ? 2.0 * exp2_f64((threadIdx.x & 31) / 32.0 - 1.0) / sum : __builtin_nan("");
  }
  __syncthreads();
  return r;
}

// body(j, entry of p, entry of q) for a thread's N entries, entry j of each
// at(j).  All are loaded first, without a branch, so that they are under way
// together; the loop stays one: straight code for 16 entries takes as long with
// half as many registers again.
template <class T, int N, class At, class Body>
__device__ __forceinline__ void entries(const Verify& a, const Rest<T>& r, At at, Body body) {
  constexpr int M = N < 4 ? N : 4;
  T px[N], qx[N];
#pragma unroll
  for (int j = 0; j < N; ++j) px[j] = r.p.row[min(at(j), a.vocab - 1)];
#pragma unroll
  for (int j = 0; j < N; ++j) qx[j] = r.q.row[min(at(j), a.vocab - 1)];
#pragma unroll 1
  for (int j0 = 0; j0 < N; j0 += M) {
#pragma unroll
    for (int j = 0; j < M; ++j) {
      double x, y;
      r.of(at(j0 + j), (float)px[j], (float)qx[j], &x, &y);
      const bool there = at(j0 + j) < a.vocab;
      body(j, there ? x : 0.0, there ? y : 0.0);
    }
#pragma unroll
    for (int j = 0; j + M < N; ++j) {
      px[j] = px[j + M];
      qx[j] = qx[j + M];
    }
  }
}

// Adds v and w over the workgroup's waves.
__device__ __forceinline__ void block_sums(double* v, double* w, double (*red)[16], int waves) {
  const int lane = threadIdx.x & 63;
  *v = wave_sum(*v);
  *w = wave_sum(*w);
  if (lane == 0) {
    red[0][threadIdx.x >> 6] = *v;
    red[1][threadIdx.x >> 6] = *w;
  }
  __syncthreads();
  *v = wave_sum(lane < waves ? red[0][lane] : 0.0);
  *w = wave_sum(lane < waves ? red[1][lane] : 0.0);
}

// grid (pieces of 256 N entries, num_seqs); block 256.  Loads go out as soon as
// their address is known, each row's before anything is computed: the steps to
// the residual (lengths, tokens and statistics, the drafts' entries, the row)
// are latencies in a row, half of a workgroup's time.
template <class T, int N>
__global__ __launch_bounds__(256) void verify_accept_kernel(Verify a) {
  __shared__ int stop_at;
  __shared__ Left left_of;
  __shared__ double red[2][16], table[64];
  const int s = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool lead = blockIdx.x == 0;
  const Span sp = span_of(a, s);
  const Heat heat = heat_of(a, s);
  if (lead && threadIdx.x == 0 && a.total && (sp.rows == 0 || heat.greedy)) a.left[s].row = -1;
  if (sp.rows == 0) {
    if (lead && threadIdx.x == 0) {
      a.accepted[s] = 0;
      if (a.context_out) a.context_out[s] = a.context[s];
    }
    return;
  }
  if (heat.greedy && !lead) return;
  if (threadIdx.x == 0) stop_at = INT32_MAX;
  __syncthreads();
  const T *target = static_cast<const T*>(a.target), *draft = static_cast<const T*>(a.draft);
  // a wave's rows up to its first refusal, as which the last row counts
  int stop = INT32_MAX;
  Left mine;
  for (int i = wave; i < sp.rows; i += 4) {
    const int t = sp.first + i;
    const bool last = i == sp.rows - 1;
    const int token = a.tokens[last ? t : t + 1];
    const bool known = !last && (uint32_t)token < (uint32_t)a.vocab;
    const int d = known ? token : 0;
    const float u = a.u_accept[t];
    Stat ps{}, qs{};
    if (!a.probs) {
      ps = part_of(a, 0, t, lane);
      if (draft) qs = part_of(a, 1, t, lane);
    }
    const float x = (float)target[t * a.target_stride + d], y = draft ? (float)draft[t * a.draft_stride + d] : 0.0f;
    if (!a.probs) {
      ps = joined(ps, heat);
      if (draft) qs = joined(qs, heat);
    }
    bool yes;
    if (heat.greedy)
      yes = known && ps.arg == d;
    else
      yes = known && (double)u * (draft ? chance(a.probs, y, (double)qs.max, qs.sum, heat) : 1.0) <
                         chance(a.probs, x, (double)ps.max, ps.sum, heat);
    const bool stops = !yes;
    const int drawn = stops && heat.greedy ? ps.arg : stops ? -1 : d;
    if (lead && (!stops || heat.greedy)) {  // right unless a row before it stops
      const float at = stops && drawn >= 0 ? (float)target[t * a.target_stride + drawn] : x;
      if (lane == 0) {
        a.out[t] = drawn;
        if (a.logprobs) a.logprobs[t] = drawn < 0 ? 0.0f : log_chance(a.probs, at, (double)ps.max, ps.sum, heat);
      }
    }
    if (stops) {
      stop = i;
      mine = {(double)ps.max, ps.sum, (double)qs.max, qs.sum, t, last ? -1 : known ? d : INT32_MAX};
      break;
    }
  }
  if (lane == 0 && stop != INT32_MAX) atomicMin(&stop_at, stop);
  __syncthreads();
  const bool first_stop = stop == stop_at;
  if (first_stop && lane == 0) left_of = mine;
  stop = stop_at;
  if (lead) {
    for (int i = wave; i < sp.rows; i += 4) {
      const int t = sp.first + i;
      if (i > stop && lane == 0) {
        a.out[t] = -1;
        if (a.logprobs) a.logprobs[t] = 0.0f;
      }
    }
    if (threadIdx.x == 0) {
      a.accepted[s] = stop;
      if (a.context_out) a.context_out[s] = a.context[s] - (sp.rows - 1 - stop);
    }
  }
  if (heat.greedy) return;
  __syncthreads();
  const Left l = left_of;
  if (lead && threadIdx.x == 0) a.left[s] = l;
  const Rest<T> rest = rest_of<T>(a, heat, l, table);
  double left = 0.0, all = 0.0;
  const int first = blockIdx.x * (256 * N) + threadIdx.x;
  entries<T, N>(a, rest, [&](int j) { return first + 256 * j; }, [&](int, double x, double y) {
    left += x;
    all += y;
  });
  block_sums(&left, &all, red, 4);
  if (threadIdx.x == 0) {
    double* m = a.mass + ((int64_t)s * a.pieces + blockIdx.x) * 2;
    m[0] = left;
    m[1] = all;
  }
}

// Over a workgroup of 1024: the first thread at which `before` and the running
// sum of v pass x and that adds to it, else the last that adds; the sum before
// that thread; and the whole sum.  thread -1: none adds, passed false.
struct Hit {
  int thread;
  bool passed;
  double before, all;
};
struct HitSpace {
  double sums[16], before;
  int first[16], last[16];
};
__device__ __forceinline__ Hit find(double v, double before, double x, HitSpace& sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const double run = wave_scan(v);
  __syncthreads();
  if (lane == 63) sh.sums[wave] = run;
  __syncthreads();
  const double other = lane < 16 ? sh.sums[lane] : 0.0;
  const double sum = before + wave_sum(lane < wave ? other : 0.0) + run;
  const unsigned long long adds = __ballot(v > 0.0), past = __ballot(sum > x) & adds;
  if (lane == 0) {
    sh.first[wave] = past ? __ffsll(past) - 1 + 64 * wave : INT32_MAX;
    sh.last[wave] = adds ? 63 - __clzll(adds) + 64 * wave : -1;
  }
  __syncthreads();
  const int first = (int)wave_min(lane < 16 ? (uint32_t)sh.first[lane] : ~0u);
  const int last = (int)~wave_min(lane < 16 ? ~(uint32_t)(sh.last[lane] + 1) : ~0u) - 1;
  Hit h;
  h.passed = first != INT32_MAX;
  h.thread = h.passed ? first : last;
  if ((int)threadIdx.x == h.thread) sh.before = sum - v;
  __syncthreads();
  h.before = sh.before;
  h.all = wave_sum(other);
  return h;
}

// grid (num_seqs); block 1024.  The piece (of 1024 N entries) in which the
// running sum passes u * total, then N consecutive entries of it to a thread,
// then the entry.  Where
// rounding leaves the last sum short, the last entry with weight.
template <class T, int N>
__global__ __launch_bounds__(1024) void verify_draw_kernel(Verify a) {
  __shared__ double red[2][16], table[64];
  __shared__ HitSpace space;
  __shared__ int token_at;
  const int s = blockIdx.x, tid = threadIdx.x;
  const Left l = a.left[s];
  if (l.row < 0) return;
  const Heat heat = heat_of(a, s);
  const Rest<T> rest = rest_of<T>(a, heat, l, table);
  const double* m = a.mass + (int64_t)s * a.pieces * 2;
  const double u = (double)a.u_sample[s];
  double left = 0.0, base = 0.0;
  for (int i = tid; i < a.pieces; i += 1024) {
    left += m[2 * i];
    base += m[2 * i + 1];
  }
  block_sums(&left, &base, red, 16);
  const bool itself = !(left > 0.0);  // nothing left: the row itself
  const double total = itself ? base : left, x = u * total;
  if (tid == 0) token_at = -1;
  if (total > 0.0) {
    int piece = -1;
    double from = 0.0, before = 0.0;
    for (int i0 = 0; i0 < a.pieces; i0 += 1024) {
      const int i = i0 + tid;
      const Hit h = find(i < a.pieces ? m[2 * i + itself] : 0.0, before, x, space);
      if (h.thread >= 0) {
        piece = i0 + h.thread;
        from = h.before;
      }
      if (h.passed) break;
      before += h.all;
    }
    const int i0 = (piece * 1024 + tid) * N;
    double v[N], sum = 0.0;
    entries<T, N>(a, rest, [&](int j) { return i0 + j; }, [&](int j, double r, double b) {
      v[j] = itself ? b : r;
      sum += v[j];
    });
    const Hit h = find(sum, from, x, space);
    if (tid == h.thread) {
      double run = h.before;
      int first = -1, some = -1;
#pragma unroll
      for (int j = N - 1; j >= 0; --j)
        if (some < 0 && v[j] > 0.0) some = i0 + j;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        run += v[j];
        if (first < 0 && run > x && v[j] > 0.0) first = i0 + j;
      }
      token_at = first >= 0 ? first : some;
    }
  }
  __syncthreads();
  if (tid == 0) {
    const int token = token_at;
    a.out[l.row] = token;
    if (a.logprobs) a.logprobs[l.row] = token < 0 ? 0.0f : log_chance(a.probs, (float)rest.p.row[token], l.p_max, l.p_sum, heat);
  }
}

// Parts of a row's statistics: enough workgroups to fill the chip (2,048),
// parts of at least 2,048 entries, and a lane for each.  222 rows of 248,320
// entries and their drafts: 87 us with 5 to 9 parts, 91 with 4, 104 with 36.
int parts_of(int vocab, int rows) {
  const int64_t want = std::max<int64_t>(1, 2048 / std::max(1, rows));
  return (int)std::min<int64_t>(kMaxParts, std::max<int64_t>(1, std::min<int64_t>(want, ((int64_t)vocab + 2047) / 2048)));
}

// Entries of a residual piece: 1024 where pieces of 4096 leave CUs idle (one
// sequence of 248,320 entries, 4 drafts: 43 us from call to result, 47 in pieces
// of 4096), 4096 where there are enough (64 sequences of 2 to 6 rows: 82 us, 107
// in pieces of 1024; every workgroup finds the acceptances by itself).
int piece_of(int vocab, int num_seqs) { return (int64_t)num_seqs * ((vocab + 4095) / 4096) <= 512 ? 1024 : 4096; }
int pieces_of(int vocab, int num_seqs) {
  const int n = piece_of(vocab, num_seqs);
  return (vocab + n - 1) / n;
}

template <class T>
void launch(const Verify& a, hipStream_t s) {
  if (!a.probs)
    hipLaunchKernelGGL(verify_stats_kernel<T>, dim3(a.parts, a.total, a.draft ? 2 : 1), dim3(256), 0, s, a);
  const bool small = piece_of(a.vocab, a.num_seqs) == 1024;
  hipLaunchKernelGGL((small ? verify_accept_kernel<T, 4> : verify_accept_kernel<T, 16>), dim3(a.pieces, a.num_seqs), dim3(256),
                     0, s, a);
  if (a.total)
    hipLaunchKernelGGL((small ? verify_draw_kernel<T, 1> : verify_draw_kernel<T, 4>), dim3(a.num_seqs), dim3(1024), 0, s, a);
}

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

// Bytes of a call, and of the largest with no more entries, sequences and rows: a
// row has fewer parts the more rows there are, but all of them no more than the
// 2,048 that fill the chip or one each; and small pieces are chosen up to 512
// large ones, which are 2,048 small ones.
size_t workspace_of(int64_t stats, int64_t seqs, int64_t masses) {
  return up(sizeof(Stat) * 2 * (size_t)stats) + up(sizeof(Left) * (size_t)seqs) + sizeof(double) * 2 * (size_t)masses;
}
size_t workspace_of_call(int vocab, int seqs, int rows) {
  return workspace_of((int64_t)rows * parts_of(vocab, rows), seqs, (int64_t)seqs * pieces_of(vocab, seqs));
}
size_t workspace_bound(int vocab, int64_t seqs, int64_t rows) {
  const int64_t large = seqs * (((int64_t)vocab + 4095) / 4096), small = seqs * (((int64_t)vocab + 1023) / 1024);
  const int64_t parts = std::min<int64_t>(kMaxParts, ((int64_t)vocab + 2047) / 2048);
  return workspace_of(std::max(rows, std::min<int64_t>(2048, rows * parts)), seqs, std::max(large, std::min<int64_t>(2048, small)));
}

}  // namespace

extern "C" size_t spk_verify_drafts_workspace_size(int32_t vocab, int32_t num_seqs, int32_t total_tokens) {
  if (vocab <= 0 || num_seqs <= 0 || total_tokens <= 0) return 0;
  return workspace_bound(vocab, num_seqs, total_tokens);
}

extern "C" int spk_verify_drafts(const SpkVerifyArgs* p, spk_stream_t stream) {
  const char* who = "spk_verify_drafts";
  if (!p) return spk::fail(SPK_ERR_NULL, "%s: NULL args", who);
  if (p->kind != SPK_VERIFY_LOGITS && p->kind != SPK_VERIFY_PROBS) return spk::fail(SPK_ERR_ARG, "%s: kind %d", who, p->kind);
  if (p->dtype != SPK_F32 && p->dtype != SPK_F16 && p->dtype != SPK_BF16)
    return spk::fail(SPK_ERR_ARG, "%s: dtype %d", who, p->dtype);
  if (p->vocab <= 0 || p->vocab > INT32_MAX - 4096 || p->num_seqs < 0 || p->total_tokens < 0)
    return spk::fail(SPK_ERR_SHAPE, "%s: vocab %d num_seqs %d total_tokens %d", who, p->vocab, p->num_seqs, p->total_tokens);
  if (p->num_seqs > 65535 || p->total_tokens > 65535)
    return spk::fail(SPK_ERR_SHAPE, "%s: %d sequences, %d rows (65535 at most)", who, p->num_seqs, p->total_tokens);
  if (p->kind == SPK_VERIFY_PROBS && p->temperature)
    return spk::fail(SPK_ERR_ARG, "%s: probabilities take no temperature", who);
  if (p->context_out && !p->context_lens) return spk::fail(SPK_ERR_NULL, "%s: context_out without context_lens", who);
  if (p->num_seqs == 0) return SPK_OK;
  if (!p->cu_seqlens || !p->accepted) return spk::fail(SPK_ERR_NULL, "%s: cu_seqlens or accepted is NULL", who);
  if (p->total_tokens) {
    if (!p->tokens || !p->target || !p->u_accept || !p->u_sample || !p->out_tokens)
      return spk::fail(SPK_ERR_NULL, "%s: tokens, target, u_accept, u_sample or out_tokens is NULL", who);
    if (p->target_stride < p->vocab || (p->draft && p->draft_stride < p->vocab))
      return spk::fail(SPK_ERR_SHAPE, "%s: rows of %d entries at strides %lld, %lld", who, p->vocab,
                       (long long)p->target_stride, (long long)p->draft_stride);
    if (p->out_tokens == p->tokens) return spk::fail(SPK_ERR_ARG, "%s: out_tokens is tokens", who);
    const size_t size = p->dtype == SPK_F32 ? 4 : 2;
    if (!spk::aligned(p->target, size) || !spk::aligned(p->draft, size))
      return spk::fail(SPK_ERR_ALIGN, "%s: target and draft must be aligned to their type", who);
    const size_t need = workspace_of_call(p->vocab, p->num_seqs, p->total_tokens);
    if (!p->workspace || p->workspace_bytes < need || !spk::aligned(p->workspace, 256))
      return spk::fail(p->workspace ? SPK_ERR_ARG : SPK_ERR_NULL, "%s: workspace of %zu bytes, %zu needed (256-byte aligned)",
                       who, p->workspace ? p->workspace_bytes : (size_t)0, need);
  }
  // every workgroup of a sequence reads its inputs, and one writes
  const void* ins[] = {p->cu_seqlens, p->tokens, p->target, p->draft, p->temperature, p->u_accept, p->u_sample, p->context_lens};
  const void* outs[] = {p->out_tokens, p->accepted, p->logprobs, p->context_out};
  for (int i = 0; i < 4; ++i) {
    bool own = true;
    for (const void* in : ins) own = own && (outs[i] != in || (i == 3 && in == p->context_lens));
    for (int j = 0; j < i; ++j) own = own && outs[i] != outs[j];
    if (outs[i] && !own) return spk::fail(SPK_ERR_ARG, "%s: an output is an input or another output", who);
  }
  Verify a{};
  a.target = p->target;
  a.draft = p->draft;
  a.target_stride = p->target_stride;
  a.draft_stride = p->draft_stride;
  a.cu = p->cu_seqlens;
  a.tokens = p->tokens;
  a.context = p->context_lens;
  a.temperature = p->temperature;
  a.u_accept = p->u_accept;
  a.u_sample = p->u_sample;
  a.out = p->out_tokens;
  a.accepted = p->accepted;
  a.context_out = p->context_out;
  a.logprobs = p->logprobs;
  a.vocab = p->vocab;
  a.num_seqs = p->num_seqs;
  a.total = p->total_tokens;
  a.parts = parts_of(p->vocab, p->total_tokens);
  a.part_len = (p->vocab + a.parts - 1) / a.parts;
  a.parts = (p->vocab + a.part_len - 1) / a.part_len;
  a.pieces = p->total_tokens ? pieces_of(p->vocab, p->num_seqs) : 1;
  a.probs = p->kind == SPK_VERIFY_PROBS;
  a.stats = static_cast<Stat*>(p->workspace);
  const size_t stats = sizeof(Stat) * 2 * (size_t)p->total_tokens * parts_of(p->vocab, p->total_tokens);
  a.left = reinterpret_cast<Left*>(static_cast<char*>(p->workspace) + up(stats));
  a.mass = reinterpret_cast<double*>(reinterpret_cast<char*>(a.left) + up(sizeof(Left) * (size_t)p->num_seqs));
  hipStream_t s = spk::to_hip(stream);
  if (a.total == 0) a.probs = 1;  // no rows: the lengths alone
  if (p->dtype == SPK_F32)
    launch<float>(a, s);
  else if (p->dtype == SPK_F16)
    launch<half_t>(a, s);
  else
    launch<bf_t>(a, s);
  return spk::check_launch(who);
}
