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
// The outcome hangs on comparisons, so whatever enters one is fp64: products
// u q(d) of two values, the exponentials of the drawn row and the running sums.
// The rows' sums of exponentials are fp32 exponentials, each off by a few units
// in the last place but none in common (log2(e) / T enters as two floats), in
// fp64 sums of eight.
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
  double* mass;         // [num_seqs][pieces][2]: residual, target
  int32_t vocab, num_seqs, total, parts, part_len, pieces;
  int32_t probs;
};

struct Stat {
  float max;
  int32_t arg;  // lowest index of the maximum, -1 where nothing is larger than -inf
  double sum;
};

constexpr int kPiece = 4096;    // vocabulary entries of a residual piece
constexpr int kMaxParts = 64;   // of a row's statistics: one for each lane

__device__ __forceinline__ bool better(float m, int a, float om, int oa) {
  return om > m || (om == m && (uint32_t)oa < (uint32_t)a);  // -1 is the largest index
}

// log2(e) / T, also as two floats; greedy rows count at T = 1.  The second is
// larger than 0, so that a logit of -inf stays one.
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
  h.scale = 1.4426950408889634 / fmax((double)t, 1e-30);
  h.c = __uint_as_float(__float_as_uint((float)h.scale) - 1);
  h.lo = (float)(h.scale - (double)h.c);
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
  auto take = [&](const float* x, int count, int first) __attribute__((always_inline)) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < count; ++i) top = fmaxf(top, x[i]);
    if (top > m) {
      if (m != -INFINITY) sum *= shrink(m, top);
      m = top;
#pragma unroll
      for (int i = count - 1; i >= 0; --i)
        if (x[i] == top) arg = first + i;
    }
    const float base = m == -INFINITY ? 0.0f : m;
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < count; ++i) {
      const float d = x[i] - base;
      part += __builtin_amdgcn_exp2f(__builtin_fmaf(d, heat.lo, d * heat.c));
    }
    sum += (double)part;
  };
  if ((int)threadIdx.x < head) {
    const float x[1] = {(float)row[threadIdx.x]};
    take(x, 1, c0 + threadIdx.x);
  }
  for (int v = threadIdx.x; v < vecs; v += 256) {
    const uint4 u = *reinterpret_cast<const uint4*>(row + head + (int64_t)v * VE);
    T e[VE];
    __builtin_memcpy(e, &u, 16);
    float x[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) x[i] = (float)e[i];
    take(x, VE, c0 + head + v * VE);
  }
  if ((int)threadIdx.x < tail) {
    const float x[1] = {(float)row[n - tail + threadIdx.x]};
    take(x, 1, c0 + n - tail + threadIdx.x);
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
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) join(__shfl_xor(m, d), __shfl_xor(arg, d), __shfl_xor(sum, d));
  if (lane == 0) red[threadIdx.x >> 6] = {m, arg, sum};
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w) join(red[w].max, red[w].arg, red[w].sum);
    a.stats[((int64_t)side * a.total + t) * a.parts + blockIdx.x] = {m, arg, sum};
  }
}

// The statistics of a row from its parts; every lane of the wave returns them.
__device__ __forceinline__ Stat row_stat(const Verify& a, const Heat& heat, int side, int t, int lane) {
  Stat r{-INFINITY, -1, 0.0};
  if (lane < a.parts) r = a.stats[((int64_t)side * a.total + t) * a.parts + lane];
  const float m = spk::wave_max(r.max);
  double sum = r.max == -INFINITY || r.max == m ? r.sum : r.sum * exp2_f64(((double)r.max - (double)m) * heat.scale);
  uint32_t arg = r.max == m ? (uint32_t)r.arg : ~0u;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    sum += __shfl_xor(sum, d);
    arg = min(arg, (uint32_t)__shfl_xor((int)arg, d));
  }
  return {m, (int)arg, sum};
}

// A row's distribution: entries count as 2^((x - max) scale) / sum of logits, as
// they are of probabilities.
template <class T>
struct Dist {
  const T* row;
  double max, scale, inv, log_sum;
  bool probs;
  __device__ __forceinline__ void set(const Verify& a, const T* r, const Stat& st, const Heat& heat) {
    row = r;
    probs = a.probs;
    max = (double)st.max;
    scale = heat.scale;
    inv = 1.0 / st.sum;
    log_sum = st.sum;
  }
  __device__ __forceinline__ double of(float x) const {
    return probs ? (double)x : exp2_f64(((double)x - max) * scale) * inv;
  }
  __device__ __forceinline__ double at(int64_t i) const { return of((float)row[i]); }
  // without the exponential's underflow
  __device__ __forceinline__ float log_at(int64_t i) const {
    const double x = (double)(float)row[i];
    return (float)(probs ? log(x) : (x - max) * scale * 0.6931471805599453 - log(log_sum));
  }
};

struct Span {
  int first, rows;
};
__device__ __forceinline__ Span span_of(const Verify& a, int s) {
  const int first = min(max(a.cu[s], 0), a.total);
  return {first, min(max(a.cu[s + 1], first), a.total) - first};
}

// The draft after a row; one that is no token is none that occurs.
__device__ __forceinline__ int draft_of(const Verify& a, int row) {
  const int d = a.tokens[row + 1];
  return (uint32_t)d < (uint32_t)a.vocab ? d : INT32_MAX;
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

template <class T>
__device__ __forceinline__ Rest<T> rest_of(const Verify& a, const Heat& heat, int row, bool refused, int lane) {
  Rest<T> r;
  r.drafted = refused && a.draft;
  r.p.set(a, static_cast<const T*>(a.target) + row * a.target_stride,
          a.probs ? Stat{} : row_stat(a, heat, 0, row, lane), heat);
  r.q.set(a, r.drafted ? static_cast<const T*>(a.draft) + row * a.draft_stride : nullptr,
          r.drafted && !a.probs ? row_stat(a, heat, 1, row, lane) : Stat{}, heat);
  r.d = refused ? draft_of(a, row) : -1;
  return r;
}

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

// grid (pieces, num_seqs); block 256
template <class T>
__global__ __launch_bounds__(256) void verify_accept_kernel(Verify a) {
  __shared__ int stop_at;
  __shared__ double red[4];
  const int s = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool lead = blockIdx.x == 0;
  const Span sp = span_of(a, s);
  if (sp.rows == 0) {
    if (lead && threadIdx.x == 0) {
      a.accepted[s] = 0;
      if (a.context_out) a.context_out[s] = a.context[s];
    }
    return;
  }
  const Heat heat = heat_of(a, s);
  if (heat.greedy && !lead) return;
  if (threadIdx.x == 0) stop_at = sp.rows - 1;
  __syncthreads();
  for (int i = wave; i < sp.rows - 1; i += 4) {
    const int t = sp.first + i, d = a.tokens[t + 1];
    bool yes = (uint32_t)d < (uint32_t)a.vocab;
    if (yes) {
      const Stat ps = a.probs ? Stat{} : row_stat(a, heat, 0, t, lane);
      if (heat.greedy) {
        yes = ps.arg == d;
      } else {
        Dist<T> p, q;
        p.set(a, static_cast<const T*>(a.target) + t * a.target_stride, ps, heat);
        double qd = 1.0;
        if (a.draft) {
          q.set(a, static_cast<const T*>(a.draft) + t * a.draft_stride, a.probs ? Stat{} : row_stat(a, heat, 1, t, lane),
                heat);
          qd = q.at(d);
        }
        yes = (double)a.u_accept[t] * qd < p.at(d);
      }
    }
    if (!yes && lane == 0) atomicMin(&stop_at, i);
  }
  __syncthreads();
  const int stop = stop_at, row = sp.first + stop;

  if (lead) {
    for (int i = wave; i < sp.rows; i += 4) {
      const int t = sp.first + i;
      if (i == stop && !heat.greedy) continue;  // drawn by the next launch
      int token = i < stop ? a.tokens[t + 1] : -1;
      float logp = 0.0f;
      if (i <= stop) {
        const Stat st = a.probs ? Stat{} : row_stat(a, heat, 0, t, lane);
        if (i == stop) token = st.arg;
        if (token >= 0 && a.logprobs) {
          Dist<T> p;
          p.set(a, static_cast<const T*>(a.target) + t * a.target_stride, st, heat);
          logp = p.log_at(token);
        }
      }
      if (lane == 0) {
        a.out[t] = token;
        if (a.logprobs) a.logprobs[t] = logp;
      }
    }
    if (threadIdx.x == 0) {
      a.accepted[s] = stop;
      if (a.context_out) a.context_out[s] = a.context[s] - (sp.rows - 1 - stop);
    }
  }
  if (heat.greedy) return;

  const Rest<T> rest = rest_of<T>(a, heat, row, stop < sp.rows - 1, lane);
  double left = 0.0, all = 0.0;
  const int end = min(a.vocab, (int)(blockIdx.x + 1) * kPiece);
#pragma unroll 4
  for (int i = blockIdx.x * kPiece + threadIdx.x; i < end; i += 256) {
    double x, y;
    rest.of(i, (float)rest.p.row[i], rest.drafted ? (float)rest.q.row[i] : 0.0f, &x, &y);
    left += x;
    all += y;
  }
  left = block_sum(left, red);
  all = block_sum(all, red);
  if (threadIdx.x == 0) {
    double* m = a.mass + ((int64_t)s * a.pieces + blockIdx.x) * 2;
    m[0] = left;
    m[1] = all;
  }
}

// Inclusive running sum over the workgroup's 256 threads.
__device__ __forceinline__ double block_scan(double v, double* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  __syncthreads();
  if (lane == 63) red[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v += red[w];
  return v;
}

// grid (num_seqs); block 256.  The piece in which the running sum passes
// u * total, then 16 consecutive entries of it to a thread, then the entry.  Where
// rounding leaves the last sum short, the last entry with weight.
template <class T>
__global__ __launch_bounds__(256) void verify_draw_kernel(Verify a) {
  __shared__ double red[4];
  __shared__ double before_at;
  __shared__ int found, last, token_at;
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const Span sp = span_of(a, s);
  if (sp.rows == 0) return;
  const Heat heat = heat_of(a, s);
  if (heat.greedy) return;
  const double* m = a.mass + (int64_t)s * a.pieces * 2;
  double left = 0.0, base = 0.0;
  for (int i = tid; i < a.pieces; i += 256) {
    left += m[2 * i];
    base += m[2 * i + 1];
  }
  const int stop = min(max(a.accepted[s], 0), sp.rows - 1), row = sp.first + stop;
  const Rest<T> rest = rest_of<T>(a, heat, row, stop < sp.rows - 1, lane);
  left = block_sum(left, red);
  base = block_sum(base, red);
  const bool itself = !(left > 0.0);  // nothing left: the row itself
  const double total = itself ? base : left, x = (double)a.u_sample[s] * total;
  if (tid == 0) {
    found = INT32_MAX;
    last = -1;
    token_at = -1;
    before_at = 0.0;
  }
  __syncthreads();
  if (total > 0.0) {
    // the first piece past x: found by its index, and the running sum before it
    double before = 0.0;
    for (int i0 = 0; i0 < a.pieces; i0 += 256) {
      const int i = i0 + tid;
      const double v = i < a.pieces ? m[2 * i + itself] : 0.0, sum = before + block_scan(v, red);
      if (i < a.pieces && sum > x) atomicMin(&found, i);
      if (v > 0.0) atomicMax(&last, i);
      __syncthreads();
      const int here = found != INT32_MAX ? found : last;
      if (i == here) before_at = sum - v;
      before += red[0] + red[1] + red[2] + red[3];
      if (found != INT32_MAX) break;
      __syncthreads();
    }
    __syncthreads();
    const int piece = found != INT32_MAX ? found : last;
    const double from = before_at;
    __syncthreads();
    if (tid == 0) {
      found = INT32_MAX;
      last = -1;
    }
    constexpr int N = kPiece / 256;
    const int i0 = piece * kPiece + N * tid;
    double v[N], sum = 0.0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      v[j] = 0.0;
      if (i0 + j < a.vocab) {
        double r, b;
        rest.of(i0 + j, (float)rest.p.row[i0 + j], rest.drafted ? (float)rest.q.row[i0 + j] : 0.0f, &r, &b);
        v[j] = itself ? b : r;
      }
      sum += v[j];
    }
    double run = from + block_scan(sum, red) - sum;
    int first = INT32_MAX, some = -1;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      run += v[j];
      if (i0 + j < a.vocab && run > x) first = min(first, i0 + j);
      if (v[j] > 0.0) some = i0 + j;
    }
    if (first != INT32_MAX) atomicMin(&found, first);
    if (some >= 0) atomicMax(&last, some);
    __syncthreads();
    if (tid == 0) token_at = found != INT32_MAX ? found : last;
    __syncthreads();
  }
  if (tid == 0) {
    const int token = token_at;
    a.out[row] = token;
    if (a.logprobs) a.logprobs[row] = token < 0 ? 0.0f : rest.p.log_at(token);
  }
}

// Parts of a row's statistics: enough workgroups to fill the chip (2,048),
// parts of at least 2,048 entries, and a lane for each.
int parts_of(int vocab, int rows) {
  const int64_t want = std::max<int64_t>(1, 2048 / std::max(1, rows));
  return (int)std::min<int64_t>(kMaxParts, std::max<int64_t>(1, std::min<int64_t>(want, ((int64_t)vocab + 2047) / 2048)));
}

int pieces_of(int vocab) { return (vocab + kPiece - 1) / kPiece; }

template <class T>
void launch(const Verify& a, hipStream_t s) {
  if (!a.probs)
    hipLaunchKernelGGL(verify_stats_kernel<T>, dim3(a.parts, a.total, a.draft ? 2 : 1), dim3(256), 0, s, a);
  hipLaunchKernelGGL(verify_accept_kernel<T>, dim3(a.pieces, a.num_seqs), dim3(256), 0, s, a);
  hipLaunchKernelGGL(verify_draw_kernel<T>, dim3(a.num_seqs), dim3(256), 0, s, a);
}

}  // namespace

extern "C" size_t spk_verify_drafts_workspace_size(int32_t vocab, int32_t num_seqs, int32_t total_tokens) {
  if (vocab <= 0 || num_seqs <= 0 || total_tokens <= 0) return 0;
  const size_t stats = sizeof(Stat) * 2 * (size_t)total_tokens * parts_of(vocab, total_tokens);
  return ((stats + 255) & ~(size_t)255) + sizeof(double) * 2 * (size_t)num_seqs * pieces_of(vocab);
}

extern "C" int spk_verify_drafts(const SpkVerifyArgs* p, spk_stream_t stream) {
  const char* who = "spk_verify_drafts";
  if (!p) return spk::fail(SPK_ERR_NULL, "%s: NULL args", who);
  if (p->kind != SPK_VERIFY_LOGITS && p->kind != SPK_VERIFY_PROBS) return spk::fail(SPK_ERR_ARG, "%s: kind %d", who, p->kind);
  if (p->dtype != SPK_F32 && p->dtype != SPK_F16 && p->dtype != SPK_BF16)
    return spk::fail(SPK_ERR_ARG, "%s: dtype %d", who, p->dtype);
  if (p->vocab <= 0 || p->vocab > INT32_MAX - kPiece || p->num_seqs < 0 || p->total_tokens < 0)
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
    const size_t need = spk_verify_drafts_workspace_size(p->vocab, p->num_seqs, p->total_tokens);
    if (!p->workspace || p->workspace_bytes < need || !spk::aligned(p->workspace, 256))
      return spk::fail(p->workspace ? SPK_ERR_ARG : SPK_ERR_NULL, "%s: workspace of %zu bytes, %zu needed (256-byte aligned)",
                       who, p->workspace ? p->workspace_bytes : (size_t)0, need);
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
  a.pieces = p->total_tokens ? pieces_of(p->vocab) : 1;
  a.probs = p->kind == SPK_VERIFY_PROBS;
  a.stats = static_cast<Stat*>(p->workspace);
  const size_t stats = sizeof(Stat) * 2 * (size_t)p->total_tokens * parts_of(p->vocab, p->total_tokens);
  a.mass = reinterpret_cast<double*>(static_cast<char*>(p->workspace) + ((stats + 255) & ~(size_t)255));
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
