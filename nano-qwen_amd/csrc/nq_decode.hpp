// What the decode kernels share: their parameters, the schedule of waves over
// (sequence, kv head) rows, the LDS tile of a step and the merge of partials.
#pragma once

#include <type_traits>

#include "nq_common.hpp"

namespace nq {

constexpr int DC_THREADS = 256;  // four independent waves
constexpr int DC_WAVES = DC_THREADS / 64;
constexpr int DC_STEP = 32;      // keys per wave step
constexpr int DC_WG_PER_CU = 1;  // resident workgroups per CU for the persistent grid
constexpr int DC_MAX_WAVES = 1024;  // persistent grid cap: 256 CUs x 1 workgroup x 4 waves
constexpr int DC_MERGE_MAX_THREADS = 1024;
constexpr int DC_MERGE_WIDE_PARTIALS = 16;  // launched waves per row from which a row's merge takes 1024 threads

struct DecodeParams {
  const void* q;
  int64_t qsb, qsh;
  // dense: (batch, kv head, row) strides of a (B, Hkv, T, D) cache;
  // paged: (page, kv head, row) strides of a (pages, Hkv, page_size, D) pool
  void* kc;
  int64_t ksb, ksh, kst;
  void* vc;
  int64_t vsb, vsh, vst;
  const int32_t* lens;
  void* o;
  int64_t osb, osh;
  float* ws_o;   // (slots, 16, D) unnormalised partial outputs
  float* ws_ml;  // (slots, 16, 2) running max (log2 units) and sum
  int32_t* ws_rw;  // (rows, 2) first and last wave that covered each row
  const float* qw;  // bf16 when q16
  int q16, k16;
  float eps;
  const float* cos_tab;
  const float* sin_tab;
  int max_pos;
  const int32_t* q_pos;
  int q_pos0;
  int B, Hq, Hkv, G, NG, max_len;
  int rows_per_batch;  // Hkv * NG
  int hs;              // the merge's heads per slice: 2^hs >= min(G, 16)
  int nwaves;          // waves launched
  int span;            // steps per wave; 0 = split N evenly over nwaves
  float scale_log2;
  int append;          // 1: a new key per batch row is appended (see kn)
  // paged: block table (row b at bt + b * bts) and rows per page (a multiple
  // of DC_STEP)
  const int32_t* bt;
  int64_t bts;
  int page;
  // fused append: the new token's raw K (normed with kw, rotated) and V go to
  // row lens[b] of the cache and are attended
  const void* kn;
  int64_t knsb, knsh;
  const void* vn;
  int64_t vnsb, vnsh;
  const float* kw;
  int32_t* lens_out;  // lens[b] + 1 after an append (never aliases lens)
  float* lse;  // (B, Hq) natural log-sum-exp of the scaled scores, or null
};

// LDS tile of DC_STEP rows (keys) x D bf16, 16-byte chunks XOR-swizzled per row.
template <int D>
struct DcTile {
  static constexpr int RB = 2 * D;                 // bytes per row
  static constexpr int CPR = D / 8;                // 16-byte chunks per row
  static constexpr int RPB = 256 / RB;             // rows per 256-byte bank row
  static constexpr int BYTES = DC_STEP * RB;       // one K or V tile
  static constexpr int RPI = 64 / CPR;             // rows per 64-lane load
  static constexpr int LOADS = DC_STEP / RPI;      // 16-byte pieces per lane per tile
  // K: a ds_read_b128 of one chunk from 16 consecutive rows hits 16 distinct
  // 16-byte bank groups.
  __device__ static int kswz(int row) { return (row / RPB) % CPR; }
  // V: a transpose read of 32 bytes from 8 consecutive rows hits 8 distinct
  // 32-byte bank groups.
  __device__ static int vswz(int row) { return ((row / RPB) % (CPR / 2)) * 2; }
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Natural log-sum-exp of a row with maximum m (log2 units) and sum l.
__device__ __forceinline__ float row_lse(float m, float l) { return (m + __builtin_amdgcn_logf(l)) * kLn2; }

// ---------------------------------------------------------------- schedule
// Keys attended by batch row b (the appended key included), or -1 for a row
// whose length lies outside [0, max_len - append]: such a row attends
// nothing, appends nothing and its output is NaN (a cache row past max_len is
// not the caller's to give).
__device__ __forceinline__ int batch_len(const DecodeParams& p, int b) {
  if (!p.lens) return p.max_len;
  const int l = p.lens[b];
  return (l < 0 || l > p.max_len - p.append) ? -1 : l + p.append;
}
// Steps of each of its rows.  COST: what the start of a row counts for in the split, in
// steps; those come first, and hold no keys.
template <int COST = 0>
__device__ __forceinline__ int batch_steps(const DecodeParams& p, int b) {
  const int len = batch_len(p, b);
  return len > 0 ? (len + DC_STEP - 1) / DC_STEP + COST : 0;
}
__device__ __forceinline__ int64_t wave_sum_i64(int64_t v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
  return v;
}
__device__ __forceinline__ int64_t lane_value_i64(int64_t v, int src) {
  const int lo = __builtin_amdgcn_readlane((int)(uint32_t)(uint64_t)v, src);
  const int hi = __builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)v >> 32), src);
  return (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}

// Total number of steps N over all rows (same value in every lane).
template <int COST = 0>
__device__ inline int64_t total_steps(const DecodeParams& p, int lane) {
  int64_t acc = 0;
  for (int base = 0; base < p.B; base += 64) {
    const int b = base + lane;
    if (b < p.B) acc += batch_steps<COST>(p, b);
  }
  return wave_sum_i64(acc) * p.rows_per_batch;
}

// The batch whose rows hold global step q (q < N), and the steps before it.
template <int COST = 0>
__device__ inline void find_batch(const DecodeParams& p, int lane, int64_t q, int& b_out, int64_t& before) {
  int64_t run = 0;
  for (int base = 0; base < p.B; base += 64) {
    const int b = base + lane;
    const int64_t v = b < p.B ? (int64_t)batch_steps<COST>(p, b) * p.rows_per_batch : 0;
    int64_t incl = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t t = __shfl_up(incl, off, 64);
      if (lane >= off) incl += t;
    }
    const int64_t excl = run + incl - v;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(v > 0 && excl <= q && q < excl + v);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      b_out = base + src;
      before = lane_value_i64(excl, src);
      return;
    }
    run += lane_value_i64(incl, 63);
  }
  b_out = p.B - 1;  // not reached for q < N
  before = run;
}

// Effective number of waves of the balanced split (never more than N).
__device__ __forceinline__ int64_t waves_used(const DecodeParams& p, int64_t N) {
  return p.span > 0 ? (N + p.span - 1) / p.span : min((int64_t)p.nwaves, N);
}
// The persistent split weights the waves by the XCD they run on (workgroup i
// runs on XCD i mod 8): a wave on an odd XCD takes DC_ODD_W / DC_EVEN_W of the
// steps of one on an even XCD.  Timestamps per wave on MI355X put the odd XCDs'
// waves 12-15% behind the even ones' over the same number of steps, whichever
// rows they stream (their share of the memory system is smaller), so an even
// split left the even XCDs idle for the last tenth of the kernel.
constexpr int DC_EVEN_W = 25, DC_ODD_W = 22;
// Total weight of waves [0, w).
__device__ __forceinline__ int64_t split_weight(int64_t w) {
  constexpr int GW = DC_WAVES * 8;  // the waves of one workgroup on each XCD
  const int64_t rounds = w / GW;
  const int k = (int)(w % GW), g = k / DC_WAVES, r = k % DC_WAVES;
  return rounds * (DC_WAVES * 4) * (DC_EVEN_W + DC_ODD_W) +
         ((int64_t)((g + 1) / 2) * DC_EVEN_W + (int64_t)(g / 2) * DC_ODD_W) * DC_WAVES +
         (int64_t)r * ((g & 1) ? DC_ODD_W : DC_EVEN_W);
}
// First global step of wave w (the chunked form: span steps per wave).  The
// weighted split applies when it still gives every wave at least one step (a
// wave with none would leave a gap in a row's run of partials); otherwise the
// steps are split evenly.
__device__ __forceinline__ int64_t wave_begin(const DecodeParams& p, int64_t N, int64_t We, int64_t w) {
  if (p.span > 0) return min(N, w * p.span);
  const int64_t total = split_weight(We);
  return N * DC_ODD_W >= total ? split_weight(w) * N / total : w * N / We;
}

// A wave's walk over its range of steps, one row segment at a time, for the fp32 and
// 4-bit stream kernels.  (The bf16 one keeps the same walk in its own variables: through
// this struct it ran 1.2% slower at B64, 64/4 heads, up to 32768 keys.)
template <int COST = 0>
struct Walk {
  int64_t q, q1;      // the range's next step and its end
  int b, j, ls, nb;   // batch, row within it, first step within the row, steps of a row
  int lens_lane;      // lens of up to 64 batch rows, one per lane: no memory round trip at a row boundary
  bool lens_in_reg;

  __device__ __forceinline__ int len_of(const DecodeParams& p, int bb) const {
    return lens_in_reg ? __builtin_amdgcn_readlane(lens_lane, bb) : uniform(batch_len(p, bb));
  }
  __device__ __forceinline__ int steps_of(const DecodeParams& p, int bb) const {
    const int l = len_of(p, bb);
    return l > 0 ? (l + DC_STEP - 1) / DC_STEP + COST : 0;
  }
  // false: wave w has no steps.  EVEN: ranges of one size, whichever XCD they run on, and of 8
  // steps at least, or of sqrt(steps of a row / 2) where that is more: what a wave saves by a
  // shorter range the merge, a workgroup a row, then takes for more partials.
  template <bool EVEN = false>
  __device__ __forceinline__ bool start(const DecodeParams& p, int lane, int64_t w) {
    const int64_t N = lane_value_i64(total_steps<COST>(p, lane), 0);
    if (N == 0) return false;
    int64_t We;
    if constexpr (EVEN) {
      const float row = (float)N / ((float)p.B * (float)p.rows_per_batch);
      We = max(min((int64_t)p.nwaves, N / max(8, (int)__builtin_sqrtf(0.5f * row))), (int64_t)1);
    } else {
      We = waves_used(p, N);
    }
    if (w >= We) return false;
    q = EVEN ? w * N / We : wave_begin(p, N, We, w);
    q1 = EVEN ? (w + 1) * N / We : wave_begin(p, N, We, w + 1);
    if (q >= q1) return false;
    lens_in_reg = p.B <= 64;
    lens_lane = lens_in_reg && lane < p.B ? batch_len(p, lane) : 0;
    int64_t before;
    find_batch<COST>(p, lane, q, b, before);
    nb = steps_of(p, b);
    j = (int)((q - before) / nb);
    ls = (int)((q - before) % nb);
    return true;
  }
  // past a segment of nseg steps; false at the end of the range
  __device__ __forceinline__ bool next(const DecodeParams& p, int nseg) {
    q += nseg;
    if (q >= q1) return false;
    ls = 0;
    if (++j == p.rows_per_batch) {
      j = 0;
      do nb = steps_of(p, ++b); while (nb == 0 && b + 1 < p.B);  // q < q1: a batch with keys follows
    }
    return true;
  }
};

// One workgroup per row (batch, kv head, head group): combines the partials
// of the waves that covered the row, or writes zeros for a row without keys.
// 16 threads hold a head (D/16 consecutive dims each); the workgroup's threads
// make up slices of the row's 2^p.hs heads, and slice i takes partials i,
// i + slices, ...: the partials' round trips to memory overlap, and the slices
// meet in LDS, each thread then adding them for two output dims.  Latency-bound
// (a few MB in all).  With one slice of 16 heads, B1 32/8 heads with 1500 keys
// (48 partials a row, 4 heads) took 11.5 us; 16 slices of 4 heads take 5.0 us.
template <int D, typename T>
__global__ void __launch_bounds__(DC_MERGE_MAX_THREADS) decode_merge_kernel(DecodeParams p) {
  constexpr int DPT = D / 16;  // dims per thread (8, 4 or 2)
  extern __shared__ float merge_lds[];
  const int64_t r = blockIdx.x;
  const int b = (int)(r / p.rows_per_batch), j = (int)(r % p.rows_per_batch);
  const int kvh = j / p.NG, hg = j % p.NG;
  const int heads = 1 << p.hs, slots = blockDim.x >> 4, slices = slots >> p.hs;
  const int slot = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * DPT;
  const int hq = slot & (heads - 1), slice = slot >> p.hs;
  const int nh = min(heads, p.G - hg * 16);  // valid heads of the group
  // the row's first and last covering wave, read through the scalar path
  // alongside lens[b] (a row without keys never uses them)
  const int64_t wf = ld_uniform(p.ws_rw, r * 2), wl = ld_uniform(p.ws_rw, r * 2 + 1);
  const int len = uniform(batch_len(p, b));
  if (p.lens_out && j == 0 && threadIdx.x == 0) p.lens_out[b] = len < 0 ? p.lens[b] : p.lens[b] + 1;
  T* out = reinterpret_cast<T*>(p.o) + b * p.osb + (int64_t)(kvh * p.G + hg * 16) * p.osh;
  float* lse = p.lse ? p.lse + (int64_t)b * p.Hq + kvh * p.G + hg * 16 : nullptr;
  if (len <= 0) {  // no keys: zeros; a length out of range: NaN
    const float f = len < 0 ? __builtin_nanf("") : 0.f;
    for (int t = threadIdx.x; t < nh * (D / 2); t += blockDim.x)
      store2<T>(out + (t / (D / 2)) * p.osh + (t % (D / 2)) * 2, f, f);
    if (lse && threadIdx.x < (unsigned)nh) lse[threadIdx.x] = len < 0 ? f : -INFINITY;
    return;
  }
  if (wf == wl) return;  // one wave covered the row and wrote it
  const int ns = (int)(wl - wf + 1);
  // one pass with a running max, so every partial's (m, l) and outputs are
  // loaded together (a partial whose scores are all -inf has m = -inf and l = 0)
  float M = -INFINITY, wsum = 0.f;
  float acc[DPT];
#pragma unroll
  for (int e = 0; e < DPT; ++e) acc[e] = 0.f;
  const float* ml = p.ws_ml + ((wf + r) * 16 + hq) * 2;
  const float* po = p.ws_o + ((wf + r) * 16 + hq) * D + d0;
  auto add = [&](int first, auto stride) {
#pragma unroll 4
    for (int i = first; i < ns; i += stride) {
      const floatx2 m_l = *reinterpret_cast<const floatx2*>(ml + i * 32);
      float o[DPT];
      if constexpr (DPT == 2) {
        const floatx2 o2 = *reinterpret_cast<const floatx2*>(po + (int64_t)i * 16 * D);
        o[0] = o2[0];
        o[1] = o2[1];
      } else {
#pragma unroll
        for (int e = 0; e < DPT; e += 4) {
          const floatx4 o4 = *reinterpret_cast<const floatx4*>(po + (int64_t)i * 16 * D + e);
#pragma unroll
          for (int k = 0; k < 4; ++k) o[e + k] = o4[k];
        }
      }
      const float Mn = fmaxf(M, m_l[0]);
      const float Mu = Mn > -INFINITY ? Mn : 0.f;
      const float a = fast_exp2(M - Mu);  // 0 for the first partial
      const float sc = fast_exp2(m_l[0] - Mu);
      wsum = wsum * a + m_l[1] * sc;
#pragma unroll
      for (int e = 0; e < DPT; ++e) acc[e] = acc[e] * a + o[e] * sc;
      M = Mn;
    }
  };
  if (slices == 1) {
    if (hq >= nh) return;
    add(0, std::integral_constant<int, 1>{});
    const float inv = 1.0f / wsum;
    if (lse && d0 == 0) lse[hq] = row_lse(M, wsum);
    T* orow = out + hq * p.osh + d0;
    if constexpr (DPT == 8) {
      store8<T>(orow, floatx8{acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv,
                              acc[4] * inv, acc[5] * inv, acc[6] * inv, acc[7] * inv});
    } else if constexpr (DPT == 4) {
      store4<T>(orow, floatx4{acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv});
    } else {
      store2<T>(orow, acc[0] * inv, acc[1] * inv);
    }
    return;
  }
  if (hq < nh) add(slice, slices);
  // slot (slice, head): D sums, then its max and weight (a slice without
  // partials: M = -inf, weight 0)
  float* mine = merge_lds + slot * (D + 2);
#pragma unroll
  for (int e = 0; e < DPT; e += 2) *reinterpret_cast<floatx2*>(mine + d0 + e) = floatx2{acc[e], acc[e + 1]};
  if (d0 == 0) *reinterpret_cast<floatx2*>(mine + D) = floatx2{M, wsum};
  __syncthreads();
  const int used = min(slices, ns);  // slices that hold partials
  for (int t = threadIdx.x; t < nh * (D / 2); t += blockDim.x) {
    const int h = t / (D / 2), d = (t % (D / 2)) * 2;
    const float* s0 = merge_lds + h * (D + 2);
    const int step = heads * (D + 2);
    float top = s0[D];
    for (int i = 1; i < used; ++i) top = fmaxf(top, s0[i * step + D]);
    float sum = 0.f, a0 = 0.f, a1 = 0.f;
    for (int i = 0; i < used; ++i) {
      const float* si = s0 + i * step;
      const float f = fast_exp2(si[D] - top);
      sum = __builtin_fmaf(si[D + 1], f, sum);
      a0 = __builtin_fmaf(si[d], f, a0);
      a1 = __builtin_fmaf(si[d + 1], f, a1);
    }
    const float inv = 1.0f / sum;
    if (lse && d == 0) lse[h] = row_lse(top, sum);
    store2<T>(out + h * p.osh + d, a0 * inv, a1 * inv);
  }
}

}  // namespace nq
