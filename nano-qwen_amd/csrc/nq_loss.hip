// What a language model is trained with, on its logits and on its tokens'
// log-probabilities: the log-probability of each label with its gradient, a
// preference loss over pairs of sequences and a clipped policy loss with a KL
// term, each with its gradient.
//
// No atomics: partial sums are stored and added in a fixed order by a later
// launch (or the same workgroup), so every call gives the same bits.

#include <math.h>

#include "nq_common.hpp"
#include "nq_internal.hpp"
#include "nq_loss.hpp"

namespace nq {

// ---------------------------------------------------------------------------
// Log-probabilities of labels.  z = logits / T, m = max z T, l = sum exp(z - m / T):
//   logprob = z[label] - log sum exp z = (x[label] - m) / T - log l,
// in one pass with a running maximum and sum per thread.  exp(z - m/T) is taken
// as 2^((x - m) c), c = log2(e) / T: the difference of two stored values first, so
// large logits lose nothing.  Rows start at any element (a vocabulary of odd size):
// the 16-byte loads ask for element alignment only.
struct TokenParams {
  const void* x;
  int64_t bs, rs;  // strides of the sequences and of their rows (elements)
  const int64_t* labels;
  float* logprobs;
  floatx2* stats;  // per row (m, l)
  floatx2* part;   // (rows, splits) partial (m, l)
  int64_t rows, S;
  int64_t row0;    // this launch's first row
  int V, splits;
  int64_t ignore;
  float c, inv_t;
};

constexpr int TOK_U = 2;  // vectors of 8 that a thread has in flight (1163 us with 4 where 2 take 1094)

template <typename T>
__device__ __forceinline__ const T* token_row(const TokenParams& p, int64_t row) {
  const int64_t b = row / p.S;
  return reinterpret_cast<const T*>(p.x) + b * p.bs + (row - b * p.S) * p.rs;
}

// What a row's statistics say of its label: NaN for a label outside the vocabulary.
template <typename T>
__device__ __forceinline__ float label_logprob(const TokenParams& p, const T* x, int64_t y, RowStat s) {
  if (y < 0 || y >= p.V) return __builtin_nanf("");
  return ((float)x[y] - s.m) * p.inv_t - logf(s.l);
}

// TEAM threads a row: a workgroup; a wave where the row is no more than 4 vectors a lane (65536
// rows of 1000 in bf16: 33 us for 78), or 16 where the rows fill the chip (16384 rows of 2500,
// 5000, 8000: 20, 29, 44 us for 31, 39, 49; of 16000 alike); with SPLIT, where the rows are few, a
// workgroup a slice of a row.  Bound by HBM.
// STREAM: logits of more bytes than the 256 MB cache holds are loaded past it: 1502 rows of
// 151936 bf16 logits 90 us without, 80 with (5.7 TB/s).  Smaller ones stay in it for the
// backward: 1026 rows of 50257 fp32, both, 112 us for 121.
template <typename T, int TEAM, bool SPLIT, bool STREAM>
__global__ __launch_bounds__(256) void token_logprobs_kernel(TokenParams p) {
  __shared__ RowStat red[4];
  const int tid = threadIdx.x % TEAM;
  int64_t row = (int64_t)blockIdx.x * (256 / TEAM) + threadIdx.x / TEAM;
  int slice = 0;
  if (SPLIT) {
    slice = (int)(row % p.splits);
    row /= p.splits;
  }
  row += p.row0;
  if (TEAM < 256 && row >= p.rows) return;
  const int64_t y = p.labels[row];
  if (y == p.ignore) {
    if (tid == 0 && slice == 0 && !SPLIT) {
      p.logprobs[row] = 0.f;
      p.stats[row] = floatx2{0.f, 1.f};
    }
    return;
  }
  const T* x = token_row<T>(p, row);
  const int nv = p.V / 8;
  int j = 0, j1 = nv;
  if (SPLIT) {
    const int per = (nv + p.splits - 1) / p.splits;
    j = slice * per < nv ? slice * per : nv;
    j1 = j + per < nv ? j + per : nv;
  }
  RowStat s{-INFINITY, 0.f};
  for (j += tid; j < j1; j += TEAM * TOK_U) {
    floatx8 v[TOK_U];
#pragma unroll
    for (int u = 0; u < TOK_U; ++u) {
      if (j + TEAM * u < j1) v[u] = load8_any<T, STREAM>(x + (int64_t)(j + TEAM * u) * 8);
      else v[u] = floatx8{} - INFINITY;
    }
    float m = s.m;
#pragma unroll
    for (int u = 0; u < TOK_U; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, v[u][e]);
    const float base = finite_max(m);
    float l = s.l * fast_exp2((s.m - base) * p.c);
#pragma unroll
    for (int u = 0; u < TOK_U; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) l += fast_exp2((v[u][e] - base) * p.c);
    s = RowStat{m, l};
  }
  if (slice == (SPLIT ? p.splits - 1 : 0) && tid < p.V % 8) {
    const float v = (float)x[nv * 8 + tid];
    s = join(s, RowStat{v, v == -INFINITY ? 0.f : v - v + 1.f}, p.c);  // NaN of NaN and +inf
  }
#pragma unroll
  for (int k = 32; k >= 1; k >>= 1) s = join(s, RowStat{__shfl_xor(s.m, k, 64), __shfl_xor(s.l, k, 64)}, p.c);
  if (TEAM == 256) {
    if ((tid & 63) == 0) red[tid >> 6] = s;
    __syncthreads();
  }
  if (tid == 0) {
    if (TEAM == 256) s = join(join(red[0], red[1], p.c), join(red[2], red[3], p.c), p.c);
    if (SPLIT) {
      p.part[row * p.splits + slice] = floatx2{s.m, s.l};
    } else {
      p.logprobs[row] = label_logprob<T>(p, x, y, s);
      p.stats[row] = floatx2{s.m, s.l};
    }
  }
}

// The slices' statistics of a row joined, a wave per row and a lane per slice.
template <typename T>
__global__ __launch_bounds__(256) void token_join_kernel(TokenParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.rows) return;
  const int64_t y = p.labels[row];
  if (y == p.ignore) {
    if (lane == 0) {
      p.logprobs[row] = 0.f;
      p.stats[row] = floatx2{0.f, 1.f};
    }
    return;
  }
  RowStat s{-INFINITY, 0.f};
  if (lane < p.splits) {
    const floatx2 v = p.part[row * p.splits + lane];
    s = RowStat{v[0], v[1]};
  }
#pragma unroll
  for (int k = 32; k >= 1; k >>= 1) s = join(s, RowStat{__shfl_xor(s.m, k, 64), __shfl_xor(s.l, k, 64)}, p.c);
  if (lane == 0) {
    p.logprobs[row] = label_logprob<T>(p, token_row<T>(p, row), y, s);
    p.stats[row] = floatx2{s.m, s.l};
  }
}

// d logits = dy (1[v = label] - p) / T, p = 2^((x - m) c) / l; zero in ignored rows
// (which are not read), NaN where the label is outside the vocabulary.  Bound by HBM:
// the logits in, their gradient out; a workgroup takes a slice of a row.  4 x 2048 rows of
// 151936 bf16, a quarter ignored, with the forward: 1163 us with plain stores and 4 vectors a
// thread, 1117 with streaming stores, 1050 with 2 vectors, 1019 with the forward's streaming
// loads (6.23 GB: 6.1 TB/s).
struct TokenBwdParams {
  TokenParams t;
  const float* dy;
  void* dx;  // (rows, V) contiguous
  int slices;
};

constexpr int TOK_SLICE = 256 * TOK_U;  // vectors of a workgroup

template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_bwd_kernel(TokenBwdParams q) {
  const TokenParams& p = q.t;
  const int tid = threadIdx.x;
  const unsigned at = blockIdx.x / q.slices;
  const int slice = (int)(blockIdx.x - at * q.slices);
  const int64_t row = p.row0 + at;
  const int64_t y = p.labels[row];
  const int nv = p.V / 8, j0 = slice * TOK_SLICE + tid;
  T* dx = reinterpret_cast<T*>(q.dx) + row * p.V;
  const bool tail = slice == q.slices - 1 && tid < p.V % 8;
  if (y == p.ignore) {
#pragma unroll
    for (int u = 0; u < TOK_U; ++u)
      if (j0 + 256 * u < nv) store8_stream<T>(dx + (int64_t)(j0 + 256 * u) * 8, floatx8{});
    if (tail) dx[nv * 8 + tid] = (T)0.f;
    return;
  }
  const T* x = token_row<T>(p, row);
  floatx8 v[TOK_U];
#pragma unroll
  for (int u = 0; u < TOK_U; ++u)
    if (j0 + 256 * u < nv) v[u] = load8_any<T>(x + (int64_t)(j0 + 256 * u) * 8);
  const floatx2 st = p.stats[row];
  const float g = (y < 0 || y >= p.V) ? __builtin_nanf("") : q.dy[row] * p.inv_t;
  const float k = -g / st[1];
#pragma unroll
  for (int u = 0; u < TOK_U; ++u) {
    const int j = j0 + 256 * u;
    if (j < nv) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = k * fast_exp2((v[u][e] - st[0]) * p.c);
        v[u][e] = (int64_t)j * 8 + e == y ? g + d : d;
      }
      store8_stream<T>(dx + (int64_t)j * 8, v[u]);
    }
  }
  if (tail) {
    const float d = k * fast_exp2(((float)x[nv * 8 + tid] - st[0]) * p.c);
    dx[nv * 8 + tid] = (T)(nv * 8 + tid == y ? g + d : d);
  }
}

// ---------------------------------------------------------------------------
// Sums over a team of threads: a wave, or a workgroup of 256 or 1024.
template <int TEAM>
__device__ __forceinline__ double team_sum(double v, double* lds) {
#pragma unroll
  for (int k = 32; k >= 1; k >>= 1) v += __shfl_xor(v, k, 64);
  if (TEAM == 64) return v;
  __syncthreads();  // the buffer's readers of the sum before
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double sum = 0;
#pragma unroll
  for (int w = 0; w < TEAM / 64; ++w) sum += lds[w];
  return sum;
}

// Sequences of a call: the last launches' threads step over them by 256 in an int.
constexpr int MOST_SEQUENCES = 1 << 30;

// Where a launch of one workgroup does the whole forward: at most this many sequences,
// a wave each, of at most this many tokens.
constexpr int ONE_ROWS = 16, ONE_TOKENS = 1024;

// ---------------------------------------------------------------------------
// Preference loss over pairs.  d = sum over a sequence's kept tokens of lp - ref (or
// their mean), h = beta (d_chosen - d_rejected), each pair's loss
//   sigmoid  -(1 - e) log s(h) - e log s(-h),  slope d loss / d d_chosen = beta (e - s(-h))
//   hinge    max(0, 1 - h),                    slope -beta where h < 1
//   ipo      (d_chosen - d_rejected - 1 / (2 beta))^2
// and their mean.  The sums cancel to a small difference of large ones and are held in
// 64 bits.  A workgroup (or, for few short pairs, a wave) takes a pair; bound by the
// launches for all but the largest batches.
struct PrefSide {
  const float* lp;
  const float* ref;
  const unsigned char* mask;
  int64_t lp_rs, ref_rs, mask_rs, S;
  float* reward;  // (B)
  float* coef;    // (B): d loss / d lp of a kept token
  float* grad;    // backward: (B, S) contiguous
};
struct PrefParams {
  PrefSide side[2];
  int B, kind, average;
  double beta, smoothing;
  float* loss;
  double* pair_loss;   // (B)
  const float* gout;   // backward: d / d loss
  int64_t blocks0;     // backward: workgroups of side 0
  int64_t first;       // this launch's first pair, or workgroup of the backward
};

template <int TEAM>
__device__ __forceinline__ double pref_pair(const PrefParams& p, int b, int t, double* lds) {
  double d[2], len[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const PrefSide& s = p.side[i];
    double sum = 0, n = 0;
#pragma unroll 4
    for (int64_t k = t; k < s.S; k += TEAM) {
      if (!s.mask || s.mask[b * s.mask_rs + k]) {
        const double v = s.lp[b * s.lp_rs + k];
        sum += s.ref ? v - (double)s.ref[b * s.ref_rs + k] : v;
        n += 1;
      }
    }
    d[i] = team_sum<TEAM>(sum, lds);
    len[i] = 1;
    if (p.average) {
      const double total = team_sum<TEAM>(n, lds);
      len[i] = total > 1 ? total : 1;
      d[i] /= len[i];
    }
  }
  const double diff = d[0] - d[1], h = p.beta * diff;
  double loss, slope;
  if (p.kind == NQ_PREF_SIGMOID) {
    // -log s(h) is log(1 + e^-|h|), which does not overflow, and -h where h < 0; -log s(-h) the
    // same and h where h > 0: each side weighed by itself, as infinities of both would cancel
    const double away = h < 0 ? -(1 - p.smoothing) * h : p.smoothing != 0 ? p.smoothing * h : 0;
    loss = log1p(exp(-fabs(h))) + away;
    slope = p.beta * (p.smoothing - 1 / (1 + exp(h)));
  } else if (p.kind == NQ_PREF_HINGE) {
    loss = h >= 1 ? 0 : 1 - h;  // NaN stays
    slope = h >= 1 ? 0 : h < 1 ? -p.beta : h;
  } else {
    const double e = diff - 0.5 / p.beta;
    loss = e * e;
    slope = 2 * e;
  }
  if (t == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      p.side[i].reward[b] = (float)(p.beta * d[i]);
      p.side[i].coef[b] = (float)((i ? -slope : slope) / (len[i] * p.B));
    }
  }
  return loss;
}

template <int TEAM>
__global__ __launch_bounds__(TEAM) void pref_pairs_kernel(PrefParams p) {
  __shared__ double lds[TEAM / 64];
  const int b = (int)(p.first + blockIdx.x);
  const double loss = pref_pair<TEAM>(p, b, threadIdx.x, lds);
  if (threadIdx.x == 0) p.pair_loss[b] = loss;
}

__global__ __launch_bounds__(256) void pref_mean_kernel(PrefParams p) {
  __shared__ double lds[4];
  double sum = 0;
  for (int b = threadIdx.x; b < p.B; b += 256) sum += p.pair_loss[b];
  sum = team_sum<256>(sum, lds);
  if (threadIdx.x == 0) *p.loss = (float)(sum / p.B);
}

__global__ __launch_bounds__(1024) void pref_one_kernel(PrefParams p) {
  __shared__ double lds[ONE_ROWS];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (wave < p.B) {
    const double loss = pref_pair<64>(p, wave, lane, nullptr);
    if (lane == 0) lds[wave] = loss;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0;
    for (int b = 0; b < p.B; ++b) sum += lds[b];
    *p.loss = (float)(sum / p.B);
  }
}

// d loss / d lp: the pair's coefficient in kept tokens.  A thread per 4 tokens.
__global__ __launch_bounds__(256) void pref_bwd_kernel(PrefParams p) {
  const int64_t block = p.first + blockIdx.x;
  const bool second = block >= p.blocks0;
  const PrefSide& s = p.side[second];
  const int64_t n = (int64_t)p.B * s.S;
  const int64_t i0 = (block - (second ? p.blocks0 : 0)) * 1024 + threadIdx.x;
  const float gout = *p.gout;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t i = i0 + 256 * u;
    if (i < n) {
      const int64_t b = i / s.S, k = i - b * s.S;
      s.grad[i] = !s.mask || s.mask[b * s.mask_rs + k] ? gout * s.coef[b] : 0.f;
    }
  }
}

// ---------------------------------------------------------------------------
// Clipped policy loss with a KL term.  Per kept token, with d = lp - old, r = e^d,
// q = ref - lp:
//   term = -min(r A, clip(r, 1 - low, 1 + high) A) + kl_coef (e^q - q - 1)
//   d term / d lp = -r A (0 where the clip decides) + kl_coef (1 - e^q)
// and the mean over all kept tokens, or over the sequences of each one's mean.  The
// clip decides where A > 0 and d > log(1 + high), or A < 0 and d < log(1 - low): d is the
// 64-bit difference, so that a token next to a border falls on its side.  Terms in 32
// bits, sums in 64.
struct PolicyParams {
  const float *lp, *old, *ref, *adv;
  const unsigned char* mask;
  int64_t lp_rs, old_rs, ref_rs, adv_rs, mask_rs;
  int adv_per_token, B, mean_of_means, segs;
  int64_t S, seg_len;
  int64_t first;      // this launch's first sequence, or workgroup of the backward
  float bound_hi, bound_lo, kl_coef;
  double log_hi, log_lo;
  float *loss, *kl, *clipped;
  float* weight;      // (B): a kept token's share of the loss
  double* part;       // (B, segs, 4): sums of term, kl, kept, clipped
  const float* gout;  // backward
  float* grad;        // (B, S) contiguous
};

// e^q - q - 1: below 1/2 its series, whose terms do not cancel (the first one left out
// is under 2^-30 of the sum).
__device__ __forceinline__ float exp_excess(float q) {
  if (fabsf(q) >= 0.5f) return expf(q) - q - 1.f;
  float s = 1.f / 3628800.f;
  s = __builtin_fmaf(s, q, 1.f / 362880.f);
  s = __builtin_fmaf(s, q, 1.f / 40320.f);
  s = __builtin_fmaf(s, q, 1.f / 5040.f);
  s = __builtin_fmaf(s, q, 1.f / 720.f);
  s = __builtin_fmaf(s, q, 1.f / 120.f);
  s = __builtin_fmaf(s, q, 1.f / 24.f);
  s = __builtin_fmaf(s, q, 1.f / 6.f);
  s = __builtin_fmaf(s, q, 0.5f);
  return s * q * q;
}

struct PolicyToken {
  float term, kl, grad;
  bool cut;
};

__device__ __forceinline__ PolicyToken policy_token(const PolicyParams& p, float lp, float old, float ref, float a) {
  PolicyToken o;
  const double d = (double)lp - (double)old;
  const float r = expf((float)d);
  const bool hi = a > 0 && d > p.log_hi, lo = a < 0 && d < p.log_lo;
  o.cut = hi || lo;
  // no advantage, no term, also where the ratio overflows (an infinity times zero); NaN stays
  const float ra = a == 0.f && d == d ? 0.f : r * a;
  o.term = hi ? -(p.bound_hi * a) : lo ? -(p.bound_lo * a) : -ra;
  o.grad = o.cut ? 0.f : -ra;
  o.kl = 0.f;
  if (p.ref) {
    const float q = (float)((double)ref - (double)lp);
    o.kl = exp_excess(q);
    if (p.kl_coef != 0.f) {
      o.term += p.kl_coef * o.kl;
      o.grad -= p.kl_coef * expm1f(q);
    }
  }
  return o;
}

__device__ __forceinline__ float policy_adv(const PolicyParams& p, int64_t b, int64_t k) {
  return p.adv[b * p.adv_rs + (p.adv_per_token ? k : 0)];
}

struct PolicySums {
  double term, kl, kept, cut;
};

template <int TEAM>
__device__ __forceinline__ PolicySums policy_sums(const PolicyParams& p, int b, int64_t k0, int64_t k1, int t,
                                                  double* lds) {
  PolicySums s{0, 0, 0, 0};
  int kept = 0, cut = 0;
#pragma unroll 4
  for (int64_t k = k0 + t; k < k1; k += TEAM) {
    if (!p.mask || p.mask[b * p.mask_rs + k]) {
      const PolicyToken o = policy_token(p, p.lp[b * p.lp_rs + k], p.old[b * p.old_rs + k],
                                         p.ref ? p.ref[b * p.ref_rs + k] : 0.f, policy_adv(p, b, k));
      s.term += o.term;
      s.kl += o.kl;
      kept += 1;
      cut += o.cut;
    }
  }
  s.term = team_sum<TEAM>(s.term, lds);
  s.kl = team_sum<TEAM>(s.kl, lds);
  s.kept = team_sum<TEAM>((double)kept, lds);
  s.cut = team_sum<TEAM>((double)cut, lds);
  return s;
}

// Workgroup = a segment of a sequence.
__global__ __launch_bounds__(256) void policy_sums_kernel(PolicyParams p) {
  __shared__ double lds[4];
  const int at = blockIdx.x / p.segs, seg = blockIdx.x - at * p.segs, b = (int)(p.first + at);
  const int64_t k0 = seg * p.seg_len, k1 = k0 + p.seg_len < p.S ? k0 + p.seg_len : p.S;
  const PolicySums s = policy_sums<256>(p, b, k0, k1, threadIdx.x, lds);
  if (threadIdx.x == 0) {
    double* o = p.part + ((int64_t)b * p.segs + seg) * 4;
    o[0] = s.term, o[1] = s.kl, o[2] = s.kept, o[3] = s.cut;
  }
}

// From the sequences' sums to the loss: one workgroup, thread b holds sequences b, b + N, ...
template <int N, typename Row>
__device__ __forceinline__ void policy_finish(const PolicyParams& p, Row row) {
  __shared__ double red[N / 64][4];
  PolicySums t{0, 0, 0, 0};
  for (int b = threadIdx.x; b < p.B; b += N) {
    const PolicySums s = row(b);
    t.term += p.mean_of_means ? (s.kept > 0 ? s.term / s.kept : 0) : s.term;
    t.kl += s.kl;
    t.kept += s.kept;
    t.cut += s.cut;
    if (p.mean_of_means) p.weight[b] = s.kept > 0 ? (float)(1 / (s.kept * p.B)) : 0.f;
  }
  const double v[4] = {t.term, t.kl, t.kept, t.cut};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double w = team_sum<64>(v[i], nullptr);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][i] = w;
  }
  __syncthreads();
  double sum[4] = {0, 0, 0, 0};
  for (int w = 0; w < N / 64; ++w)
    for (int i = 0; i < 4; ++i) sum[i] += red[w][i];
  const double n = sum[2] > 0 ? sum[2] : 1;
  if (threadIdx.x == 0) {
    *p.loss = (float)(sum[0] / (p.mean_of_means ? (double)p.B : n));
    *p.kl = (float)(sum[1] / n);
    *p.clipped = (float)(sum[3] / n);
  }
  if (!p.mean_of_means)
    for (int b = threadIdx.x; b < p.B; b += N) p.weight[b] = (float)(1 / n);
}

__global__ __launch_bounds__(256) void policy_finish_kernel(PolicyParams p) {
  policy_finish<256>(p, [&](int b) {
    PolicySums s{0, 0, 0, 0};
    for (int i = 0; i < p.segs; ++i) {
      const double* o = p.part + ((int64_t)b * p.segs + i) * 4;
      s.term += o[0], s.kl += o[1], s.kept += o[2], s.cut += o[3];
    }
    return s;
  });
}

__global__ __launch_bounds__(1024) void policy_one_kernel(PolicyParams p) {
  __shared__ PolicySums rows[ONE_ROWS];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (wave < p.B) {
    const PolicySums s = policy_sums<64>(p, wave, 0, p.S, lane, nullptr);
    if (lane == 0) rows[wave] = s;
  }
  __syncthreads();
  policy_finish<1024>(p, [&](int b) { return rows[b]; });
}

__global__ __launch_bounds__(256) void policy_bwd_kernel(PolicyParams p) {
  const int64_t n = (int64_t)p.B * p.S;
  const int64_t i0 = (p.first + blockIdx.x) * 1024 + threadIdx.x;
  const float gout = *p.gout;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t i = i0 + 256 * u;
    if (i < n) {
      const int64_t b = i / p.S, k = i - b * p.S;
      float g = 0.f;
      if (!p.mask || p.mask[b * p.mask_rs + k])
        g = gout * p.weight[b] *
            policy_token(p, p.lp[b * p.lp_rs + k], p.old[b * p.old_rs + k], p.ref ? p.ref[b * p.ref_rs + k] : 0.f,
                         policy_adv(p, b, k)).grad;
      p.grad[i] = g;
    }
  }
}

}  // namespace nq

using namespace nq;

static bool aligned_to(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// A launch has fewer than 2^32 threads: n groups of `each` workgroups of `threads`, in as many launches
// as that takes, launch(first group, workgroups).
template <typename F>
static void in_launches(int64_t n, int64_t each, int threads, F launch) {
  const int64_t most = (int64_t)UINT32_MAX / threads / each;
  for (int64_t first = 0; first < n; first += most)
    launch(first, dim3((unsigned)((n - first < most ? n - first : most) * each)));
}

// ------------------------------------------------------------------ token log-probabilities

// Slices of a row: as many workgroups as two rounds of the chip hold, each slice at least
// one turn of the loop, a lane of the join for each.
static int token_splits(int64_t rows, int V) {
  const int64_t want = (2048 + rows - 1) / rows;
  const int64_t most = (V / 8 + 256 * TOK_U - 1) / (256 * TOK_U);
  int64_t s = want < most ? want : most;
  if (s > 64) s = 64;
  return s < 1 ? 1 : (int)s;
}

extern "C" int64_t nq_token_logprobs_workspace_bytes(int64_t rows, int V) {
  if (rows <= 0 || V <= 0) return 0;
  const int s = token_splits(rows, V);
  return s > 1 ? rows * s * (int64_t)sizeof(floatx2) : 0;
}

static int token_check(const void* logits, const int64_t* labels, const void* stats, int64_t B, int64_t S, int V,
                       int64_t bs, int64_t rs, int dtype, float temperature) {
  if (!nq_dtype_ok(dtype)) return nq_fail(NQ_ERR_UNSUPPORTED, "dtype must be NQ_DTYPE_BF16 or NQ_DTYPE_F32");
  if (B <= 0 || S <= 0 || V <= 0)
    return nq_fail(NQ_ERR_INVALID, "sizes must be positive (B=%lld S=%lld V=%d)", (long long)B, (long long)S, V);
  if (bs < 0 || rs < 0) return nq_fail(NQ_ERR_INVALID, "strides must not be negative");
  if (B > INT32_MAX / S) return nq_fail(NQ_ERR_UNSUPPORTED, "too many rows for one launch");
  if (!logits || !labels || !stats) return nq_fail(NQ_ERR_INVALID, "logits, labels and stats are required");
  if (!aligned_to(logits, nq_dtype_size(dtype)) || !aligned_to(labels, 8) || !aligned_to(stats, 8))
    return nq_fail(NQ_ERR_INVALID, "logits, labels and stats must be aligned to their elements");
  const float inv = 1.f / temperature;
  if (!(temperature > 0.f) || !isfinite(temperature) || !isfinite(inv * kLog2e))
    return nq_fail(NQ_ERR_INVALID, "the temperature must be positive and finite, and so must its reciprocal");
  return NQ_OK;
}

template <typename T, bool STREAM>
static void launch_tokens(TokenParams p, hipStream_t st) {
  const dim3 block(256);
  if (p.splits > 1) {
    const dim3 waves((unsigned)((p.rows + 3) / 4)), grid((unsigned)(p.rows * p.splits));
    hipLaunchKernelGGL((token_logprobs_kernel<T, 256, true, STREAM>), grid, block, 0, st, p);
    hipLaunchKernelGGL((token_join_kernel<T>), waves, block, 0, st, p);
  } else if (p.V / 8 <= (p.rows >= 2048 ? 1024 : 256)) {
    in_launches((p.rows + 3) / 4, 1, 256, [&](int64_t first, dim3 grid) {
      p.row0 = first * 4;
      hipLaunchKernelGGL((token_logprobs_kernel<T, 64, false, STREAM>), grid, block, 0, st, p);
    });
  } else {
    in_launches(p.rows, 1, 256, [&](int64_t first, dim3 grid) {
      p.row0 = first;
      hipLaunchKernelGGL((token_logprobs_kernel<T, 256, false, STREAM>), grid, block, 0, st, p);
    });
  }
}

extern "C" int nq_token_logprobs(const void* logits, int64_t batch_stride, int64_t row_stride, const int64_t* labels,
                                 float* logprobs, float* stats, void* workspace, int64_t workspace_bytes, int64_t B,
                                 int64_t S, int V, int dtype, float temperature, int64_t ignore_index, void* stream) {
  nq_clear_error();
  if (int rc = token_check(logits, labels, stats, B, S, V, batch_stride, row_stride, dtype, temperature)) return rc;
  if (!logprobs || !aligned_to(logprobs, 4)) return nq_fail(NQ_ERR_INVALID, "logprobs is required, aligned to fp32");
  const int64_t rows = B * S, need = nq_token_logprobs_workspace_bytes(rows, V);
  if (need && (!workspace || workspace_bytes < need || !aligned_to(workspace, 8)))
    return nq_fail(NQ_ERR_WORKSPACE, "workspace too small or not 8-byte aligned: %lld bytes, need %lld",
                   (long long)workspace_bytes, (long long)need);
  const float inv = 1.f / temperature;
  const int splits = token_splits(rows, V);
  if (rows * splits > INT32_MAX) return nq_fail(NQ_ERR_UNSUPPORTED, "too many rows for one launch");
  TokenParams p{logits, batch_stride, row_stride, labels, logprobs, reinterpret_cast<floatx2*>(stats),
                reinterpret_cast<floatx2*>(workspace), rows, S, 0, V, splits, ignore_index, inv * kLog2e, inv};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool b16 = dtype == NQ_DTYPE_BF16;
  const bool past = rows * V * (b16 ? 2 : 4) > ((int64_t)256 << 20);
  if (b16) past ? launch_tokens<bf16, true>(p, st) : launch_tokens<bf16, false>(p, st);
  else past ? launch_tokens<float, true>(p, st) : launch_tokens<float, false>(p, st);
  return nq_check_launch(hipGetLastError());
}

extern "C" int nq_token_logprobs_bwd(const void* logits, int64_t batch_stride, int64_t row_stride,
                                     const int64_t* labels, const float* stats, const float* dlogprobs, void* dlogits,
                                     int64_t B, int64_t S, int V, int dtype, float temperature, int64_t ignore_index,
                                     void* stream) {
  nq_clear_error();
  if (int rc = token_check(logits, labels, stats, B, S, V, batch_stride, row_stride, dtype, temperature)) return rc;
  if (!dlogprobs || !dlogits || !aligned_to(dlogprobs, 4) || !aligned_to(dlogits, nq_dtype_size(dtype)))
    return nq_fail(NQ_ERR_INVALID, "dlogprobs and dlogits are required, aligned to their elements");
  const float inv = 1.f / temperature;
  const int64_t rows = B * S;
  const int slices = (V / 8 + TOK_SLICE - 1) / TOK_SLICE > 0 ? (V / 8 + TOK_SLICE - 1) / TOK_SLICE : 1;
  if (rows * slices > INT32_MAX) return nq_fail(NQ_ERR_UNSUPPORTED, "too many rows for one launch");
  TokenBwdParams q{{logits, batch_stride, row_stride, labels, nullptr,
                    reinterpret_cast<floatx2*>(const_cast<float*>(stats)), nullptr, rows, S, 0, V, 1, ignore_index,
                    inv * kLog2e, inv},
                   dlogprobs, dlogits, slices};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  in_launches(rows, slices, 256, [&](int64_t first, dim3 grid) {
    q.t.row0 = first;
    if (dtype == NQ_DTYPE_BF16) hipLaunchKernelGGL((token_logprobs_bwd_kernel<bf16>), grid, dim3(256), 0, st, q);
    else hipLaunchKernelGGL((token_logprobs_bwd_kernel<float>), grid, dim3(256), 0, st, q);
  });
  return nq_check_launch(hipGetLastError());
}

// ------------------------------------------------------------------ preference loss

extern "C" int64_t nq_preference_loss_workspace_bytes(int B) {
  return B > 0 ? (int64_t)B * (int64_t)sizeof(double) : 0;
}

static int pref_check(int B, int64_t Sc, int64_t Sr, const float* coef) {
  if (B <= 0 || Sc < 0 || Sr < 0)
    return nq_fail(NQ_ERR_INVALID, "B must be positive and the lengths not negative (B=%d Sc=%lld Sr=%lld)", B,
                   (long long)Sc, (long long)Sr);
  if (B > MOST_SEQUENCES) return nq_fail(NQ_ERR_UNSUPPORTED, "at most 2^30 sequences in one call, got %d", B);
  if (Sc > ((int64_t)1 << 40) / B || Sr > ((int64_t)1 << 40) / B)
    return nq_fail(NQ_ERR_UNSUPPORTED, "too many tokens for one launch");
  if (!coef || !aligned_to(coef, 4)) return nq_fail(NQ_ERR_INVALID, "coef is required, aligned to fp32");
  return NQ_OK;
}

extern "C" int nq_preference_loss(const float* chosen, int64_t chosen_stride, const float* rejected,
                                  int64_t rejected_stride, const float* ref_chosen, int64_t ref_chosen_stride,
                                  const float* ref_rejected, int64_t ref_rejected_stride, const uint8_t* chosen_mask,
                                  int64_t chosen_mask_stride, const uint8_t* rejected_mask,
                                  int64_t rejected_mask_stride, float* loss, float* chosen_reward,
                                  float* rejected_reward, float* coef, void* workspace, int64_t workspace_bytes, int B,
                                  int64_t Sc, int64_t Sr, int kind, double beta, double label_smoothing, int average,
                                  void* stream) {
  nq_clear_error();
  if (int rc = pref_check(B, Sc, Sr, coef)) return rc;
  if (kind != NQ_PREF_SIGMOID && kind != NQ_PREF_HINGE && kind != NQ_PREF_IPO)
    return nq_fail(NQ_ERR_UNSUPPORTED, "unknown kind %d", kind);
  if (!(beta > 0) || !isfinite(beta)) return nq_fail(NQ_ERR_INVALID, "beta must be positive and finite");
  if (!(label_smoothing >= 0 && label_smoothing < 0.5) || (label_smoothing != 0 && kind != NQ_PREF_SIGMOID))
    return nq_fail(NQ_ERR_INVALID, "label_smoothing is for the sigmoid loss, from 0 to under 1/2");
  if ((Sc && !chosen) || (Sr && !rejected) || !loss || !chosen_reward || !rejected_reward)
    return nq_fail(NQ_ERR_INVALID, "chosen, rejected, loss and the rewards are required");
  const bool one = B <= ONE_ROWS && Sc <= ONE_TOKENS && Sr <= ONE_TOKENS;
  if (!one && (!workspace || !aligned_to(workspace, 8) || workspace_bytes < nq_preference_loss_workspace_bytes(B)))
    return nq_fail(NQ_ERR_WORKSPACE, "workspace too small or not 8-byte aligned: %lld bytes, need %lld",
                   (long long)workspace_bytes, (long long)nq_preference_loss_workspace_bytes(B));
  PrefParams p{{{chosen, ref_chosen, chosen_mask, chosen_stride, ref_chosen_stride, chosen_mask_stride, Sc,
                 chosen_reward, coef, nullptr},
                {rejected, ref_rejected, rejected_mask, rejected_stride, ref_rejected_stride, rejected_mask_stride, Sr,
                 rejected_reward, coef + B, nullptr}},
               B, kind, average != 0, beta, label_smoothing, loss, reinterpret_cast<double*>(workspace), nullptr, 0, 0};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (one) {
    hipLaunchKernelGGL(pref_one_kernel, dim3(1), dim3(1024), 0, st, p);
  } else {
    // 256 pairs of 4096 tokens: 10.5 us with 1024 threads a pair for 15.5 with 256
    const bool longer = Sc > ONE_TOKENS || Sr > ONE_TOKENS;
    in_launches(B, 1, longer ? 1024 : 256, [&](int64_t first, dim3 grid) {
      p.first = first;
      if (longer) hipLaunchKernelGGL((pref_pairs_kernel<1024>), grid, dim3(1024), 0, st, p);
      else hipLaunchKernelGGL((pref_pairs_kernel<256>), grid, dim3(256), 0, st, p);
    });
    hipLaunchKernelGGL(pref_mean_kernel, dim3(1), dim3(256), 0, st, p);
  }
  return nq_check_launch(hipGetLastError());
}

extern "C" int nq_preference_loss_bwd(const float* coef, const float* dloss, const uint8_t* chosen_mask,
                                      int64_t chosen_mask_stride, const uint8_t* rejected_mask,
                                      int64_t rejected_mask_stride, float* dchosen, float* drejected, int B,
                                      int64_t Sc, int64_t Sr, void* stream) {
  nq_clear_error();
  if (int rc = pref_check(B, Sc, Sr, coef)) return rc;
  if (!dloss) return nq_fail(NQ_ERR_INVALID, "dloss is required");
  PrefParams p{};
  p.B = B;
  p.gout = dloss;
  float* grads[2] = {dchosen, drejected};
  const uint8_t* masks[2] = {chosen_mask, rejected_mask};
  const int64_t strides[2] = {chosen_mask_stride, rejected_mask_stride}, lens[2] = {Sc, Sr};
  int64_t blocks[2];
  for (int i = 0; i < 2; ++i) {  // a side without an output is left out
    p.side[i].grad = grads[i];
    p.side[i].mask = masks[i];
    p.side[i].mask_rs = strides[i];
    p.side[i].S = grads[i] ? lens[i] : 0;
    p.side[i].coef = const_cast<float*>(coef) + (int64_t)i * B;
    blocks[i] = (p.side[i].S * B + 1023) / 1024;
  }
  p.blocks0 = blocks[0];
  if (blocks[0] + blocks[1] == 0) return NQ_OK;
  if (blocks[0] + blocks[1] > INT32_MAX) return nq_fail(NQ_ERR_UNSUPPORTED, "too many tokens for one launch");
  in_launches(blocks[0] + blocks[1], 1, 256, [&](int64_t first, dim3 grid) {
    p.first = first;
    hipLaunchKernelGGL(pref_bwd_kernel, grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream), p);
  });
  return nq_check_launch(hipGetLastError());
}

// ------------------------------------------------------------------ policy loss

// Segments of a sequence: workgroups for two rounds of the chip, each at least 8 tokens a thread.
static int policy_segs(int B, int64_t S) {
  const int64_t want = (2048 + B - 1) / B, most = (S + 2047) / 2048;
  const int64_t s = want < most ? want : most;
  return s < 1 ? 1 : (int)s;
}

extern "C" int64_t nq_policy_loss_workspace_bytes(int B, int64_t S) {
  return B > 0 && S >= 0 ? (int64_t)B * policy_segs(B, S) * 4 * (int64_t)sizeof(double) : 0;
}

static int policy_params(PolicyParams* p, const float* logprobs, int64_t lp_rs, const float* old, int64_t old_rs,
                         const float* ref, int64_t ref_rs, const float* adv, int64_t adv_rs, int adv_per_token,
                         const uint8_t* mask, int64_t mask_rs, float* weight, int B, int64_t S, double clip_low,
                         double clip_high, double kl_coef) {
  if (B <= 0 || S < 0) return nq_fail(NQ_ERR_INVALID, "B must be positive and S not negative (B=%d S=%lld)", B, (long long)S);
  if (B > MOST_SEQUENCES) return nq_fail(NQ_ERR_UNSUPPORTED, "at most 2^30 sequences in one call, got %d", B);
  if (S > ((int64_t)1 << 40) / B) return nq_fail(NQ_ERR_UNSUPPORTED, "too many tokens for one launch");
  if ((S && (!logprobs || !old)) || (!adv && (S || !adv_per_token)) || !weight)
    return nq_fail(NQ_ERR_INVALID, "logprobs, old logprobs, advantages and weight are required");
  if (!(clip_low >= 0 && clip_low <= 1) || !(clip_high >= 0) || !isfinite(clip_high) || !isfinite(kl_coef))
    return nq_fail(NQ_ERR_INVALID, "clip_low must lie in [0, 1], clip_high be at least 0, and both and kl_coef finite");
  if (S && kl_coef != 0 && !ref) return nq_fail(NQ_ERR_INVALID, "a KL term needs the reference's logprobs");
  *p = PolicyParams{};
  p->lp = logprobs, p->old = old, p->ref = ref, p->adv = adv, p->mask = mask;
  p->lp_rs = lp_rs, p->old_rs = old_rs, p->ref_rs = ref_rs, p->adv_rs = adv_rs, p->mask_rs = mask_rs;
  p->adv_per_token = adv_per_token != 0, p->B = B, p->S = S;
  p->bound_hi = (float)(1 + clip_high), p->bound_lo = (float)(1 - clip_low), p->kl_coef = (float)kl_coef;
  p->log_hi = log1p(clip_high), p->log_lo = log1p(-clip_low);
  p->weight = weight;
  return NQ_OK;
}

extern "C" int nq_policy_loss(const float* logprobs, int64_t logprobs_stride, const float* old_logprobs,
                              int64_t old_stride, const float* ref_logprobs, int64_t ref_stride,
                              const float* advantages, int64_t advantages_stride, int advantages_per_token,
                              const uint8_t* mask, int64_t mask_stride, float* loss, float* kl, float* clipped,
                              float* weight, void* workspace, int64_t workspace_bytes, int B, int64_t S,
                              double clip_low, double clip_high, double kl_coef, int mean_of_means, void* stream) {
  nq_clear_error();
  PolicyParams p;
  if (int rc = policy_params(&p, logprobs, logprobs_stride, old_logprobs, old_stride, ref_logprobs, ref_stride,
                             advantages, advantages_stride, advantages_per_token, mask, mask_stride, weight, B, S,
                             clip_low, clip_high, kl_coef))
    return rc;
  if (!loss || !kl || !clipped) return nq_fail(NQ_ERR_INVALID, "loss, kl and clipped are required");
  p.loss = loss, p.kl = kl, p.clipped = clipped, p.mean_of_means = mean_of_means != 0;
  p.segs = policy_segs(B, S);
  p.seg_len = (S + p.segs - 1) / p.segs;
  p.part = reinterpret_cast<double*>(workspace);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (B <= ONE_ROWS && S <= ONE_TOKENS) {
    hipLaunchKernelGGL(policy_one_kernel, dim3(1), dim3(1024), 0, st, p);
    return nq_check_launch(hipGetLastError());
  }
  if (!workspace || !aligned_to(workspace, 8) || workspace_bytes < nq_policy_loss_workspace_bytes(B, S))
    return nq_fail(NQ_ERR_WORKSPACE, "workspace too small or not 8-byte aligned: %lld bytes, need %lld",
                   (long long)workspace_bytes, (long long)nq_policy_loss_workspace_bytes(B, S));
  if ((int64_t)B * p.segs > INT32_MAX) return nq_fail(NQ_ERR_UNSUPPORTED, "too many sequences for one launch");
  in_launches(B, p.segs, 256, [&](int64_t first, dim3 grid) {
    p.first = first;
    hipLaunchKernelGGL(policy_sums_kernel, grid, dim3(256), 0, st, p);
  });
  hipLaunchKernelGGL(policy_finish_kernel, dim3(1), dim3(256), 0, st, p);
  return nq_check_launch(hipGetLastError());
}

extern "C" int nq_policy_loss_bwd(const float* logprobs, int64_t logprobs_stride, const float* old_logprobs,
                                  int64_t old_stride, const float* ref_logprobs, int64_t ref_stride,
                                  const float* advantages, int64_t advantages_stride, int advantages_per_token,
                                  const uint8_t* mask, int64_t mask_stride, const float* weight, const float* dloss,
                                  float* dlogprobs, int B, int64_t S, double clip_low, double clip_high,
                                  double kl_coef, void* stream) {
  nq_clear_error();
  PolicyParams p;
  if (int rc = policy_params(&p, logprobs, logprobs_stride, old_logprobs, old_stride, ref_logprobs, ref_stride,
                             advantages, advantages_stride, advantages_per_token, mask, mask_stride,
                             const_cast<float*>(weight), B, S, clip_low, clip_high, kl_coef))
    return rc;
  if (!dloss || (S && !dlogprobs)) return nq_fail(NQ_ERR_INVALID, "dloss and dlogprobs are required");
  if (S == 0) return NQ_OK;
  p.gout = dloss, p.grad = dlogprobs;
  const int64_t blocks = ((int64_t)B * S + 1023) / 1024;
  if (blocks > INT32_MAX) return nq_fail(NQ_ERR_UNSUPPORTED, "too many tokens for one launch");
  in_launches(blocks, 1, 256, [&](int64_t first, dim3 grid) {
    p.first = first;
    hipLaunchKernelGGL(policy_bwd_kernel, grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream), p);
  });
  return nq_check_launch(hipGetLastError());
}
