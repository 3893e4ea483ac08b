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
// The rows' sums of exponentials are fp32 exponentials with an exact argument
// (two-float product with log2(e) / T), added in fp64.
#include <algorithm>

#include "capi_common.hpp"
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

constexpr int kPiece = 4096;  // vocabulary entries of a residual piece

template <class T>
__device__ __forceinline__ float value(const T* p, int64_t i) {
  return (float)p[i];
}

__device__ __forceinline__ bool better(float m, int a, float om, int oa) {
  return om > m || (om == m && (uint32_t)oa < (uint32_t)a);  // -1 is the largest index
}

// log2(e) / T as two floats; greedy rows count at T = 1.
struct Heat {
  float c, lo, least;  // least: differences below it weigh nothing
  double inv;
  bool greedy;
};
__device__ __forceinline__ Heat heat_of(const Verify& a, int s) {
  float t = a.temperature && s < a.num_seqs ? a.temperature[s] : 1.0f;
  Heat h;
  h.greedy = !(t > 0.0f);
  if (h.greedy) t = 1.0f;
  const double c = 1.4426950408889634 / fmax((double)t, 1e-30);
  h.c = (float)c;
  h.lo = (float)(c - (double)h.c);
  h.least = -200.0f / h.c;
  h.inv = (double)t;
  return h;
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
  auto take = [&](const float* x, int count, int first) {
    float top = x[0];
    for (int i = 1; i < count; ++i) top = fmaxf(top, x[i]);
    if (top > m) {
      const float d = m - top;
      if (m != -INFINITY) sum *= (double)__builtin_amdgcn_exp2f(d < heat.least ? -200.0f : d * heat.c);
      m = top;
      for (int i = count - 1; i >= 0; --i)
        if (x[i] == top) arg = first + i;
    }
    const float base = m == -INFINITY ? 0.0f : m;
    float part = 0.0f;
    for (int i = 0; i < count; ++i) {
      float d = x[i] - base;
      d = d < heat.least ? heat.least : d;
      const float k = __builtin_rintf(d * heat.c);
      const float r = __builtin_fmaf(d, heat.lo, __builtin_fmaf(d, heat.c, -k));
      part += __builtin_ldexpf(__builtin_amdgcn_exp2f(r), (int)k);
    }
    sum += (double)part;
  };
  if ((int)threadIdx.x < head) {
    const float x[1] = {value(row, threadIdx.x)};
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
    const float x[1] = {value(row, n - tail + threadIdx.x)};
    take(x, 1, c0 + n - tail + threadIdx.x);
  }

  auto join = [&](float om, int oa, double os) {
    if (om > m) {
      const float d = m - om;
      sum = (m == -INFINITY ? sum : sum * (double)__builtin_amdgcn_exp2f(d < heat.least ? -200.0f : d * heat.c)) + os;
    } else if (m > om) {
      const float d = om - m;
      sum += om == -INFINITY ? os : os * (double)__builtin_amdgcn_exp2f(d < heat.least ? -200.0f : d * heat.c);
    } else {
      sum += os;
    }
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
  const Stat* p = a.stats + ((int64_t)side * a.total + t) * a.parts;
  float m = -INFINITY;
  for (int j = lane; j < a.parts; j += 64) m = fmaxf(m, p[j].max);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  double sum = 0.0;
  int arg = -1;
  for (int j = lane; j < a.parts; j += 64) {
    const Stat x = p[j];
    sum += x.max == -INFINITY || x.max == m ? x.sum : x.sum * exp(((double)x.max - (double)m) / heat.inv);
    if (x.max == m && (uint32_t)x.arg < (uint32_t)arg) arg = x.arg;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    sum += __shfl_xor(sum, d);
    const int o = __shfl_xor(arg, d);
    if ((uint32_t)o < (uint32_t)arg) arg = o;
  }
  r.max = m;
  r.arg = arg;
  r.sum = sum;
  return r;
}

// The probability of entry i of a row.
template <class T>
__device__ __forceinline__ double prob(const Verify& a, const T* row, int64_t i, const Stat& st, const Heat& heat) {
  const double x = (double)(float)row[i];
  return a.probs ? x : exp((x - (double)st.max) / heat.inv) / st.sum;
}

// Log of it, without the exponential's underflow.
template <class T>
__device__ __forceinline__ float log_prob(const Verify& a, const T* row, int64_t i, const Stat& st, const Heat& heat) {
  const double x = (double)(float)row[i];
  return (float)(a.probs ? log(x) : (x - (double)st.max) / heat.inv - log(st.sum));
}

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

// What row `t` leaves for token i: the residual where a draft `d` was refused
// there (d < 0: the row itself).
template <class T>
struct Rest {
  const T *p, *q;
  Stat ps, qs;
  Heat heat;
  int d;
  __device__ __forceinline__ void at(const Verify& a, int i, double* rest, double* base) const {
    const double x = prob(a, p, i, ps, heat);
    *base = x;
    if (d < 0) {
      *rest = x;
    } else if (q) {
      const double y = x - prob(a, q, i, qs, heat);
      *rest = y > 0.0 || y != y ? y : 0.0;
    } else {
      *rest = i == d ? 0.0 : x;
    }
  }
};

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
  if (threadIdx.x == 0) stop_at = sp.rows - 1;
  __syncthreads();
  for (int i = wave; i < sp.rows - 1; i += 4) {
    const int t = sp.first + i, d = a.tokens[t + 1];
    bool yes = (uint32_t)d < (uint32_t)a.vocab;
    if (yes) {
      const T* p = static_cast<const T*>(a.target) + t * a.target_stride;
      const T* q = static_cast<const T*>(a.draft) + t * a.draft_stride;
      const Stat ps = a.probs ? Stat{} : row_stat(a, heat, 0, t, lane);
      if (heat.greedy) {
        yes = ps.arg == d;
      } else {
        const Stat qs = a.probs || !a.draft ? Stat{} : row_stat(a, heat, 1, t, lane);
        const double qd = a.draft ? prob(a, q, d, qs, heat) : 1.0;
        yes = (double)a.u_accept[t] * qd < prob(a, p, d, ps, heat);
      }
    }
    if (!yes && lane == 0) atomicMin(&stop_at, i);
  }
  __syncthreads();
  const int stop = stop_at, row = sp.first + stop;
  const T* p = static_cast<const T*>(a.target) + row * a.target_stride;
  const Stat ps = a.probs ? Stat{} : row_stat(a, heat, 0, row, lane);

  if (lead) {
    for (int i = wave; i < sp.rows; i += 4) {
      const int t = sp.first + i;
      if (i < stop) {
        const int d = a.tokens[t + 1];
        const Stat st = a.probs || !a.logprobs ? Stat{} : row_stat(a, heat, 0, t, lane);
        if (lane == 0) {
          a.out[t] = d;
          if (a.logprobs) a.logprobs[t] = log_prob(a, static_cast<const T*>(a.target) + t * a.target_stride, d, st, heat);
        }
      } else if (lane == 0 && (i > stop || heat.greedy)) {
        const bool here = i == stop && ps.arg >= 0;
        a.out[t] = here ? ps.arg : -1;
        if (a.logprobs) a.logprobs[t] = here ? log_prob(a, p, ps.arg, ps, heat) : 0.0f;
      }
    }
    if (threadIdx.x == 0) {
      a.accepted[s] = stop;
      if (a.context_out) a.context_out[s] = a.context[s] - (sp.rows - 1 - stop);
    }
  }
  if (heat.greedy) return;

  Rest<T> rest;
  const bool refused = stop < sp.rows - 1;
  rest.p = p;
  rest.ps = ps;
  rest.q = refused && a.draft ? static_cast<const T*>(a.draft) + row * a.draft_stride : nullptr;
  rest.qs = rest.q && !a.probs ? row_stat(a, heat, 1, row, lane) : Stat{};
  rest.heat = heat;
  rest.d = refused ? draft_of(a, row) : -1;
  double left = 0.0, all = 0.0;
  const int end = min(a.vocab, (int)(blockIdx.x + 1) * kPiece);
  for (int i = blockIdx.x * kPiece + threadIdx.x; i < end; i += 256) {
    double x, y;
    rest.at(a, i, &x, &y);
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

// The first index i of 0 .. n-1 whose running sum from `before` on passes x,
// else the last with weight, else -1; `next`: the running sum before it.
// value(i) is asked by one wave, 64 at a time, in order.
template <class F>
__device__ __forceinline__ int first_past(int n, double before, double x, int lane, F value, double* next) {
  int last = -1;
  double last_sum = before;
  for (int i0 = 0; i0 < n; i0 += 64) {
    const double v = i0 + lane < n ? value(i0 + lane) : 0.0;
    double sum = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    const unsigned long long past = __ballot(i0 + lane < n && before + sum > x);
    const unsigned long long some = __ballot(v > 0.0);
    const double prior = before + (sum - v);
    if (past) {
      const int l = __ffsll(past) - 1;
      *next = __shfl(prior, l);
      return i0 + l;
    }
    if (some) {
      const int l = 63 - __clzll(some);
      last = i0 + l;
      last_sum = __shfl(prior, l);
    }
    before += __shfl(sum, 63);
  }
  *next = last_sum;
  return last;
}

// grid (num_seqs); block 64
template <class T>
__global__ __launch_bounds__(64) void verify_draw_kernel(Verify a) {
  const int s = blockIdx.x, lane = threadIdx.x;
  const Span sp = span_of(a, s);
  if (sp.rows == 0) return;
  const Heat heat = heat_of(a, s);
  if (heat.greedy) return;
  const int stop = min(max(a.accepted[s], 0), sp.rows - 1), row = sp.first + stop;
  const bool refused = stop < sp.rows - 1;
  Rest<T> rest;
  rest.p = static_cast<const T*>(a.target) + row * a.target_stride;
  rest.ps = a.probs ? Stat{} : row_stat(a, heat, 0, row, lane);
  rest.q = refused && a.draft ? static_cast<const T*>(a.draft) + row * a.draft_stride : nullptr;
  rest.qs = rest.q && !a.probs ? row_stat(a, heat, 1, row, lane) : Stat{};
  rest.heat = heat;
  rest.d = refused ? draft_of(a, row) : -1;
  const double* m = a.mass + (int64_t)s * a.pieces * 2;
  double total = 0.0, base = 0.0;
  for (int i = lane; i < a.pieces; i += 64) {
    total += m[2 * i];
    base += m[2 * i + 1];
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    total += __shfl_xor(total, d);
    base += __shfl_xor(base, d);
  }
  const int which = total > 0.0 ? 0 : 1;  // nothing left: the row itself
  if (which) total = base;
  int token = -1;
  if (total > 0.0) {
    const double x = (double)a.u_sample[s] * total;
    double before;
    const int piece = first_past(a.pieces, 0.0, x, lane, [&](int i) { return m[2 * i + which]; }, &before);
    if (piece >= 0) {
      const int i0 = piece * kPiece, n = min(kPiece, a.vocab - i0);
      const int i = first_past(n, before, x, lane,
                               [&](int j) {
                                 double r, b;
                                 rest.at(a, i0 + j, &r, &b);
                                 return which ? b : r;
                               },
                               &before);
      token = i < 0 ? -1 : i0 + i;
    }
  }
  if (lane == 0) {
    a.out[row] = token;
    if (a.logprobs) a.logprobs[row] = token < 0 ? 0.0f : log_prob(a, rest.p, token, rest.ps, heat);
  }
}

// Parts of a row's statistics: enough workgroups to fill the chip (2,048),
// pieces of at least 2,048 entries.
int parts_of(int vocab, int rows) {
  const int64_t want = std::max<int64_t>(1, 2048 / std::max(1, rows));
  return (int)std::max<int64_t>(1, std::min<int64_t>(want, (vocab + 2047) / 2048));
}

int pieces_of(int vocab) { return (vocab + kPiece - 1) / kPiece; }

template <class T>
void launch(const Verify& a, hipStream_t s) {
  if (!a.probs)
    hipLaunchKernelGGL(verify_stats_kernel<T>, dim3(a.parts, a.total, a.draft ? 2 : 1), dim3(256), 0, s, a);
  hipLaunchKernelGGL(verify_accept_kernel<T>, dim3(a.pieces, a.num_seqs), dim3(256), 0, s, a);
  hipLaunchKernelGGL(verify_draw_kernel<T>, dim3(a.num_seqs), dim3(64), 0, s, a);
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
