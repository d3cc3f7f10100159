// Eviction from a paged KV cache by accumulated attention weight, for gfx950: the weight
// each cached key got, the keys worth keeping, and their rows moved to other pages.  No
// counterpart in the reference, whose cache (model/attention.py:24-46) only grows.

#include <type_traits>

#include "nq_common.hpp"
#include "nq_internal.hpp"
#include "nq_kv4.hpp"

namespace nq {

// ---------------------------------------------------------------- key weights
//   w[b, h, t] (+)= sum over the G query heads of kv head h and the S queries that see
//   key t of exp(scale q . k_t - lse),
// the columns of the attention's probabilities, which a flash attention never forms: its
// log-sum-exp gives them from q and K alone.  The product is taken as S = Q K^T, so a
// lane holds one key and four (query, head) rows, and the sum over rows stays in it until
// the end; K stays in registers while the rows pass.  Rows run r = s G + g.
struct KeyWeightParams {
  const bf16* q;
  int64_t qsb, qsh, qss;
  const void* pool;       // 4-bit pages (strides in bytes) or bf16 ones (elements)
  int64_t psb, psh, pss;  // page, head and (bf16) row strides
  int npages;
  const int32_t* bt;
  int64_t bts;
  Divider page;
  const int32_t* lens;
  const float* lse;  // (B, Hq, S)
  float* w;
  int64_t wsb, wsh;
  int add;           // add to w, else write it
  int B, Hq, Hkv, S, max_len, causal;
  Divider G;
  float scale_log2;
  Divider range;           // keys of a workgroup
  int same;                // workgroups of each chunk, 0: as many as it has ranges
  int chunks, chunk_rows;  // rows of a workgroup: chunks > 1 write partial sums
  float* part;             // (chunks, B, Hkv, max_len)
};

// The elements that lane slot grp holds of operand i, in eights: q's must be K's.  4-bit rows:
// D/4 consecutive ones, as the decode's (one load, one scale); bf16 rows: as they lie, 64
// consecutive bytes of a row to four lanes.
template <int D, bool FOUR>
__device__ __forceinline__ constexpr int eight_of(int grp, int i) {
  return FOUR ? grp * (D / 32) + i : i * 4 + grp;
}

// 32 keys, as operands of the product (lane: key c16 of each 16, slot grp).  ONCE: read once,
// past the caches.
template <int D, bool FOUR, bool ONCE> struct Keys32 {
  static constexpr int NDQ = D / 32;
  typedef uint32_t codes_t __attribute__((ext_vector_type(NDQ)));
  codes_t c[2];
  uint32_t e[2];
  bf16x8 k[2][FOUR ? 1 : NDQ];
  template <typename V>
  __device__ __forceinline__ static V fetch(const void* src) {
    if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const V*>(src));
    else return *reinterpret_cast<const V*>(src);
  }
  __device__ __forceinline__ void load(const KeyWeightParams& p, int pid, int kvh, int rel, int c16, int grp) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int row = rel + t * 16 + c16;
      if constexpr (FOUR) {
        using F = Kv4<D>;
        const unsigned char* rec = reinterpret_cast<const unsigned char*>(p.pool) + pid * p.psb + kvh * p.psh;
        c[t] = fetch<codes_t>(rec + row * F::CB + grp * (D / 8));
        e[t] = rec[F::k_scales(p.page.d) + row * F::SB + grp * (D / 4) / 32];
      } else {
        const bf16* src = reinterpret_cast<const bf16*>(p.pool) + pid * p.psb + kvh * p.psh + row * p.pss;
#pragma unroll
        for (int i = 0; i < NDQ; ++i) k[t][i] = fetch<bf16x8>(src + eight_of<D, FOUR>(grp, i) * 8);
      }
    }
  }
  __device__ __forceinline__ bf16x8 operand(int t, int i) const {
    if constexpr (FOUR) return kv4_bf16x8(c[t][i], kv4_scale(e[t]));
    else return k[t][i];
  }
};

// i of n, turned by `by`.
__device__ __forceinline__ uint32_t turned(uint32_t i, uint32_t n, uint32_t by) {
  i += by % n;
  return i < n ? i : i - n;
}

// Where a wave's keys lie: a lane holds the page of the 32 keys from `first` on, which never
// cross one, and their first row there; past the last key its 32 again.  lost: the pages
// that are none of the pool's, a bit a lane.
struct KeyPages {
  int pid, rel;
  uint64_t lost;
  __device__ __forceinline__ void load(const KeyWeightParams& p, int b, int first, int len) {
    first = min(first, (len - 1) & ~31);
    const int page = p.page.div(first, rel);
    pid = p.bt[b * p.bts + page];
  }
  __device__ __forceinline__ void check(const KeyWeightParams& p) {  // waits for the load
    const bool bad = (uint32_t)pid >= (uint32_t)p.npages;
    lost = __builtin_amdgcn_ballot_w64(bad);
    if (bad) pid = 0;
  }
};

// A row's lse: -inf for rows past the last.
__device__ __forceinline__ float row_lse_of(const KeyWeightParams& p, int b, int kvh, int r, int R) {
  int g;
  const int s = p.G.div(min(r, R - 1), g);
  const float v = p.lse[((int64_t)b * p.Hq + kvh * p.G.d + g) * p.S + s];
  return r >= R ? -INFINITY : v;
}
// What it adds to the row's scores, in log2 units: -inf (no weight) for a query that sees no key.
// The product is rounded to fp32: 2^-24 |lse| of a weight, as much as by the rounding of lse itself.
__device__ __forceinline__ float row_offset(float lse) { return lse == -INFINITY ? lse : -lse * kLog2e; }

// Four values' sums over the wave's four groups of 16 lanes: group g gets that of value g.
// (The swaps exchange odd groups of the first with even ones of the second, halves likewise.)
__device__ __forceinline__ float group_sums(const float (&v)[4]) {
  float y[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), false, false);
    y[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(y[0]), __float_as_uint(y[1]), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---- up to 16 rows (a decode step): every key's score in one MFMA tile.  HBM-bound: K read
// once.  A wave takes 64 keys at a time, of 4-bit pages two to four such runs, the next one
// on its way; of bf16 pages one.  4-bit codes are read past the caches (cached, 64 sequences
// of 32768 keys and 4 heads took 119 us for 110); bf16 rows are not, two loads sharing each
// line (past the caches 241 us for 212 at 1024 to 32768 keys).  64 sequences of as many 4-bit
// keys (64/4 heads, 291 MB): 61 us, 4.8 TB/s; with a part of 128 keys a wave, all of its
// loads at once, 73.
template <int D, bool FOUR, bool ADD>
__global__ void __launch_bounds__(256) key_weights_step_kernel(KeyWeightParams p) {
  constexpr int NDQ = D / 32;
  constexpr int RUN = 64;  // keys
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, grp = lane >> 4;
  const int b = blockIdx.z, kvh = blockIdx.y;
  // Turned by the head: the XCD of a workgroup goes by blockIdx.x where the grid is a multiple
  // of 8 wide, and only some sequences have last keys (not turned: 88 us for 69).
  const uint32_t x = turned(blockIdx.x, gridDim.x, (uint32_t)b * (uint32_t)p.Hkv + (uint32_t)kvh);
  const int span = p.range.d, k0 = (int)(x * 4 + wave) * span;
  if (k0 >= p.max_len) return;
  const int len = ld_uniform(p.lens, b);
  float* w = p.w + b * p.wsb + kvh * p.wsh;
  const bool bad_len = len < 0 || len > p.max_len;
  const int runs = bad_len || k0 >= len ? 0 : (min(len - k0, span) + RUN - 1) / RUN;
  if (!ADD)  // what the runs do not reach
    for (int t = k0 + runs * RUN + lane; t < min(k0 + span, p.max_len); t += 64) w[t] = bad_len ? __builtin_nanf("") : 0.f;
  if (runs == 0) return;
  // what does not hang on the block table is on its way before it is waited for
  KeyPages at;
  at.load(p, b, k0 + min(lane, span / 32 - 1) * 32, len);
  const int R = p.S * p.G.d;
  int g;
  const int s = p.G.div(min(c16, R - 1), g);
  const bf16* qrow = p.q + b * p.qsb + (int64_t)(kvh * p.G.d + g) * p.qsh + s * p.qss;
  bf16x8 q[NDQ];
#pragma unroll
  for (int i = 0; i < NDQ; ++i) q[i] = Vec8<bf16>::load_bf16(qrow + eight_of<D, FOUR>(grp, i) * 8);
  const float own = row_lse_of(p, b, kvh, c16, R);
  float off[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) off[e] = row_lse_of(p, b, kvh, grp * 4 + e, R);
  at.check(p);
  struct Run {
    Keys32<D, FOUR, FOUR> k[2];
    float old;  // the weights so far
  };
  auto load = [&](Run& x, int i) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
      x.k[u].load(p, __builtin_amdgcn_readlane(at.pid, 2 * i + u), kvh, __builtin_amdgcn_readlane(at.rel, 2 * i + u), c16, grp);
    if constexpr (ADD) x.old = w[min(k0 + i * RUN + lane, len - 1)];
  };
  Run even, odd;
  load(even, 0);
  if constexpr (FOUR) load(odd, min(1, runs - 1));
  // a query that saw nothing adds nothing, whatever it holds
#pragma unroll
  for (int i = 0; i < NDQ; ++i) q[i] = own == -INFINITY ? bf16x8{} : q[i];
  int last[4];  // the last key that the row's query sees
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    off[e] = row_offset(off[e]);
    last[e] = p.causal ? len - p.S + p.G.div(grp * 4 + e) : 0x7fffffff;
  }
  auto weigh = [&](const Run& x, int i) {
    float sum[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      floatx4 sc = floatx4{};
#pragma unroll
      for (int d = 0; d < NDQ; ++d) sc = mfma16(q[d], x.k[t / 2].operand(t & 1, d), sc);
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[e] = fast_exp2(__builtin_fmaf(sc[e], p.scale_log2, off[e]));
      if (p.causal) {
        const int key = k0 + i * RUN + t * 16 + c16;
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[e] = key <= last[e] ? sc[e] : 0.f;
      }
      sum[t] = (sc[0] + sc[1]) + (sc[2] + sc[3]);
    }
    float mine = group_sums(sum);
    if (at.lost >> (2 * i + lane / 32) & 1) mine = __builtin_nanf("");
    const int t = k0 + i * RUN + lane;
    if (t < len) w[t] = ADD ? x.old + mine : mine;
    else if (!ADD && t < p.max_len) w[t] = 0.f;
  };
  if constexpr (!FOUR) {
    weigh(even, 0);
  } else {
    if (runs == 1) {
      weigh(even, 0);
      return;
    }
    int i = 0;
    for (; i + 3 < runs; i += 2) {
      weigh(even, i);
      load(even, i + 2);
      weigh(odd, i + 1);
      load(odd, i + 3);
    }
    weigh(even, i);
    if (i + 2 < runs) load(even, i + 2);
    weigh(odd, i + 1);
    if (i + 2 < runs) weigh(even, i + 2);
  }
}

// ---- more rows (prompts): a workgroup holds a chunk of up to 256 rows in LDS, read once, and
// its four waves pass their keys by it, 64 at a time, the next 64 on their way meanwhile.
// No wave waits for another after the chunk is staged.  Bound by the exponentials' side: 16
// rows and 64 keys take 16 x (4 + 8 + 4) cycles of scaling, exponential and sum, and the 16
// products hold up the vector unit for some 11 cycles each of their 16.  Chunks > 1 write
// partial sums that key_weights_sum_kernel adds, in order.
constexpr int KW_ROWS = 256;   // rows of a chunk
constexpr int KW_PASS = 256;   // keys that its waves take at a time

// Ranges of keys that a chunk has: up to the last that its last query sees in a sequence of
// max_len.  (In shorter ones it sees fewer; the workgroups past them find nothing to do.)
__host__ __device__ __forceinline__ int chunk_ranges(const KeyWeightParams& p, int chunk) {
  const int R = p.S * (int)p.G.d, end = R / KW_ROWS > chunk ? (chunk + 1) * KW_ROWS : R;
  const int seen = p.causal ? p.max_len - p.S + p.G.div(end - 1) + 1 : p.max_len;
  return seen > 0 ? p.range.div(seen + (int)p.range.d - 1) : 0;
}

template <int D, bool FOUR>
__global__ void __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(2)))
key_weights_kernel(KeyWeightParams p) {
  constexpr int NDQ = D / 32;
  constexpr int RB = 2 * D, CPR = D / 8, RPB = 256 / RB;  // bytes and 16-byte chunks of a row, rows of 256 bytes
  constexpr int PCS = KW_ROWS * CPR / 256;                // chunks a thread stages
  __shared__ __attribute__((aligned(16))) unsigned char qt[KW_ROWS * RB];
  __shared__ __attribute__((aligned(16))) float offs[KW_ROWS];
  __shared__ __attribute__((aligned(16))) int lasts[KW_ROWS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, grp = lane >> 4;
  const int b = blockIdx.z, kvh = blockIdx.y;
  // the workgroups of chunk 0, then those of chunk 1, ...: as many as each has ranges, or
  // (many chunks) as many as the last has.  Turned by the head or the chunk, as in the step
  // kernel: 16 sequences of up to 16384 4-bit keys, 64 queries, 32/8 heads take 97 us, not turned 135.
  int chunk = 0, at_range;
  if (p.same) {
    chunk = blockIdx.x / p.same;
    at_range = (int)turned(blockIdx.x % p.same, p.same, chunk);
  } else {
    at_range = (int)turned(blockIdx.x, gridDim.x, (uint32_t)b * (uint32_t)p.Hkv + (uint32_t)kvh);
    for (int n; chunk + 1 < p.chunks && at_range >= (n = chunk_ranges(p, chunk)); ++chunk) at_range -= n;
  }
  const int range0 = at_range * (int)p.range.d;
  const int len = ld_uniform(p.lens, b);
  const bool bad_len = len < 0 || len > p.max_len;
  const bool add = p.add && p.chunks == 1;
  float* w = p.chunks > 1 ? p.part + (((int64_t)chunk * p.B + b) * p.Hkv + kvh) * p.max_len
                          : p.w + b * p.wsb + kvh * p.wsh;
  const int R = p.S * p.G.d, r0 = chunk * p.chunk_rows, rows = min(R - r0, p.chunk_rows);
  const int hidden = p.causal ? len - p.S : 0x3fffffff;  // query s sees keys up to hidden + s
  const int kend = rows > 0 ? min(len, p.causal ? hidden + p.G.div(r0 + rows - 1) + 1 : len) : 0;
  if (bad_len || range0 >= kend) {  // no weight from this chunk
    if (!add)
      for (int t = range0 + threadIdx.x; t < min(range0 + (int)p.range.d, p.max_len); t += 256)
        w[t] = bad_len ? __builtin_nanf("") : 0.f;
    return;
  }
  // lane 2 i + u: half u of the wave's tile i, keys range0 + (4 i + wave) 64 + 32 u
  const int tiles = p.range.d / KW_PASS;
  KeyPages at;
  {
    const int l = min(lane, 2 * tiles - 1);
    at.load(p, b, range0 + ((l >> 1) * 4 + wave) * 64 + (l & 1) * 32, len);
    at.check(p);
  }
  Keys32<D, FOUR, false> keys[2];
  auto load_keys = [&](int i) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
      keys[u].load(p, __builtin_amdgcn_readlane(at.pid, 2 * i + u), kvh, __builtin_amdgcn_readlane(at.rel, 2 * i + u), c16,
                   grp);
  };
  load_keys(0);
  {
    // rows r0 + threadIdx.x / CPR + i STEP: the first by a division, each next by an addition
    constexpr int STEP = 256 / CPR;
    const int s0 = p.G.div(r0), qsh = (int)p.qsh, qss = (int)p.qss, G = (int)p.G.d;
    const bf16* src = p.q + b * p.qsb + (int64_t)kvh * G * p.qsh + s0 * p.qss;  // 32-bit offsets from here
    int g;
    const int s = p.G.div(r0 + threadIdx.x / CPR, g);
    int ds_g;
    const int ds_s = p.G.div(STEP, ds_g);
    const int step = ds_s * qss + ds_g * qsh, wrap = qss - G * qsh;
    int row = threadIdx.x / CPR, at_row = (s - s0) * qss + g * qsh + (threadIdx.x % CPR) * 8;
    unsigned char* dst = qt + row * RB + (((threadIdx.x % CPR) ^ ((row / RPB) % CPR)) << 4);
    static_assert(STEP % (RPB * CPR) == 0, "the swizzle repeats every step");
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      bf16x8 piece[PCS / 2];
#pragma unroll
      for (int i = 0; i < PCS / 2; ++i) {
        piece[i] = Vec8<bf16>::load_bf16(src + (row < rows ? at_row : 0));
        row += STEP;
        g += ds_g;
        at_row += step + (g >= G ? wrap : 0);
        g -= g >= G ? G : 0;
      }
#pragma unroll
      for (int i = 0; i < PCS / 2; ++i)
        *reinterpret_cast<bf16x8*>(dst + (half * (PCS / 2) + i) * STEP * RB) = piece[i];
    }
    offs[threadIdx.x] = row_offset(row_lse_of(p, b, kvh, r0 + threadIdx.x, r0 + rows));
    lasts[threadIdx.x] = hidden + p.G.div(r0 + threadIdx.x);
  }
  __syncthreads();
  // a query that saw nothing adds nothing, whatever it holds (NaN behind a padded sequence)
  if (offs[threadIdx.x] == -INFINITY)
#pragma unroll
    for (int i = 0; i < CPR; ++i) *reinterpret_cast<bf16x8*>(qt + threadIdx.x * RB + i * 16) = bf16x8{};
  __syncthreads();
  const int n = (rows + 15) / 16;
  int qoff[NDQ];  // this lane's operands of 16 rows (the swizzle repeats every 16)
#pragma unroll
  for (int d = 0; d < NDQ; ++d) qoff[d] = c16 * RB + ((eight_of<D, FOUR>(grp, d) ^ ((c16 / RPB) % CPR)) << 4);

#pragma unroll 1
  for (int i = 0; i < tiles; ++i) {
    const int k0 = range0 + (i * 4 + wave) * 64;
    if (k0 >= p.max_len) break;
    bf16x8 k[4][NDQ];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int d = 0; d < NDQ; ++d) k[t][d] = keys[t / 2].operand(t & 1, d);
    if (i + 1 < tiles) load_keys(i + 1);
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    auto pass = [&](int from, int to, auto masked) {
      for (int rt = from; rt < to; ++rt) {
        bf16x8 q[NDQ];
#pragma unroll
        for (int d = 0; d < NDQ; ++d) q[d] = *reinterpret_cast<const bf16x8*>(qt + rt * 16 * RB + qoff[d]);
        floatx4 sc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) sc[t] = floatx4{};
#pragma unroll
        for (int d = 0; d < NDQ; ++d)
#pragma unroll
          for (int t = 0; t < 4; ++t) sc[t] = mfma16(q[d], k[t][d], sc[t]);
        const floatx4 off = *reinterpret_cast<const floatx4*>(&offs[rt * 16 + grp * 4]);
        int last[4];
        if constexpr (decltype(masked)::value) {
#pragma unroll
          for (int e = 0; e < 4; ++e) last[e] = lasts[rt * 16 + grp * 4 + e];
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float pe = fast_exp2(__builtin_fmaf(sc[t][e], p.scale_log2, off[e]));
            if constexpr (decltype(masked)::value) acc[t] += k0 + t * 16 + c16 <= last[e] ? pe : 0.f;
            else acc[t] += pe;
          }
      }
    };
    // rows before `seen` see none of these keys, rows from `all` on see all of them
    const int64_t G = p.G.d;
    const int seen = p.causal ? (int)min(max((int64_t)(k0 - hidden) * G - r0, (int64_t)0), (int64_t)rows) / 16 : 0;
    const int all =
        p.causal ? ((int)min(max((int64_t)(k0 + 63 - hidden) * G - r0, (int64_t)0), (int64_t)(rows + 15)) + 15) / 16 : 0;
    if (k0 < kend) {
      pass(seen, min(all, n), std::true_type{});
      pass(max(all, 0), n, std::false_type{});
    }
    float mine = group_sums(acc);
    if (at.lost >> (2 * i + lane / 32) & 1) mine = __builtin_nanf("");
    const int t = k0 + lane;
    if (t < len) w[t] = add ? w[t] + mine : mine;
    else if (!add && t < p.max_len) w[t] = 0.f;
  }
}

// The chunks' partial sums, added in order: of the chunks whose ranges reach the key.
__global__ void __launch_bounds__(256) key_weights_sum_kernel(KeyWeightParams p) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  const int b = blockIdx.z, kvh = blockIdx.y;
  if (t >= p.max_len) return;
  const int range = p.range.div(t);
  int c = 0;  // the first chunk that reaches the key (ranges grow with the chunk)
  for (int hi = p.chunks; c < hi;) {
    const int mid = (c + hi) / 2;
    if (chunk_ranges(p, mid) <= range) c = mid + 1;
    else hi = mid;
  }
  const float* src = p.part + ((int64_t)b * p.Hkv + kvh) * p.max_len + t;
  const int64_t step = (int64_t)p.B * p.Hkv * p.max_len;
  float sum = 0.f;
#pragma unroll 4
  for (; c < p.chunks; ++c) sum += src[c * step];
  float* w = p.w + b * p.wsb + kvh * p.wsh + t;
  const int len = ld_uniform(p.lens, b);
  if (!p.add) *w = sum;
  else if (len <= p.max_len && t < len) *w += sum;
}

// Keys of a wave of the 4-bit step kernel, in runs of 64: two runs, and up to four where more
// than 8192 waves would have two.  64 sequences of 1024 to 32768 keys, 64/4 heads (with a
// fill of 10 us): four runs 68 us, eight 72, sixteen 77; 256 of up to 1024, 32/8 heads: two
// 28, four 23.
static int key_weight_span(const KeyWeightParams& p) {
  const int64_t runs = ((int64_t)p.max_len + 63) / 64 * p.B * p.Hkv / 8192;
  return 64 * (int)(runs < 2 ? 2 : (runs > 4 ? 4 : runs));
}

// Chunks of the rows.
static int key_weight_chunks(int64_t R) { return (int)((R + KW_ROWS - 1) / KW_ROWS); }

// Workgroups of a (sequence, kv head).
static int64_t key_weight_groups(const KeyWeightParams& p) {
  int64_t n = 0;
  for (int c = 0; c < p.chunks; ++c) n += chunk_ranges(p, c);
  return n;
}

// Keys of a workgroup: the fewest with which all of them are resident at once, two a CU
// (512 in all), so that none waits for another's end and each waits for its rows once; 1024
// where more are needed anyway, and 512 where the diagonal cuts most of them.  2 prompts of
// 2048, 16/8 heads, causal: 256 keys 48 us, 1024 45, the 768 chosen 38 (480 workgroups); also
// launched for the ranges that a chunk does not have, of which the XCDs get unequal shares,
// 56.  A prompt of 8192, 32/8 heads: 1024 keys 401 us, 512 349; without turning the ranges by
// the chunk 548.  2048 queries at the end of 32768 keys, 64/4 heads: 1024 keys 966 us, 512
// 1024.
constexpr int KW_FEW_CHUNKS = 64;
static int key_weight_range(KeyWeightParams p) {
  if (p.chunks <= KW_FEW_CHUNKS)
    for (int range = KW_PASS; range <= 2048; range += KW_PASS) {
      p.range = Divider(range);
      if (key_weight_groups(p) * p.B * p.Hkv <= 512) return range;
    }
  return p.causal && p.S > p.max_len / 2 ? 512 : 1024;
}

// ---------------------------------------------------------------- selection
// The rows that a (sequence, kv head) keeps: the first `first`, the last `recent`, and of
// the rows between them the `keep - first - recent` heaviest, equal weights by the lower
// index; in ascending order.  A workgroup of 16 waves per (sequence, head), each with a
// contiguous share of the weights, finds the smallest kept one by a radix select over its
// bits (11 + 11 + 10, a histogram in LDS for each), then each wave writes its kept rows:
// its place in the output follows from the counts of the waves before it.  The first 32
// weights of a lane (32768 in all) stay in registers; of longer rows the rest is read five
// times, from the cache.  Bound by its instructions, five passes over 32 weights a lane on one
// CU: 64 rows of 32768 take 22 us (8 MB; four copies of the histogram changed nothing).
struct SelectParams {
  const float* w;
  int64_t wsb, wsh;
  const int32_t* lens;
  int32_t* kept;  // (B, Hkv, keep)
  int Hkv, W, keep, recent, first;
};

constexpr int SEL_THREADS = 1024, SEL_WAVES = SEL_THREADS / 64, SEL_BINS = 2048, SEL_HELD = 32;

// Orders as the weights do: NaN above everything, -0 as +0.  0 is no weight's.
__device__ __forceinline__ uint32_t weight_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(SEL_THREADS) select_keys_kernel(SelectParams p) {
  __shared__ uint32_t hist[SEL_BINS];
  __shared__ uint32_t wave_a[SEL_WAVES], wave_b[SEL_WAVES];
  __shared__ uint32_t found[2];
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float* w = p.w + b * p.wsb + h * p.wsh;
  int32_t* kept = p.kept + (int64_t)blockIdx.x * p.keep;
  int n = ld_uniform(p.lens, b);
  if (n < 0 || n > p.W) n = 0;  // not a length: nothing is kept
  if (n <= p.keep) {
    for (int i = tid; i < p.keep; i += SEL_THREADS) kept[i] = i < n ? i : -1;
    return;
  }
  const int lo = p.first, hi = n - p.recent;
  uint32_t room = (uint32_t)(p.keep - p.first - p.recent);
  for (int i = tid; i < p.first; i += SEL_THREADS) kept[i] = i;
  for (int i = tid; i < p.recent; i += SEL_THREADS) kept[p.keep - p.recent + i] = hi + i;
  if (room == 0) return;

  const int rounds = (hi - lo + SEL_THREADS - 1) / SEL_THREADS;  // 64 weights each
  const int begin = min(lo + wave * rounds * 64, hi), end = min(begin + rounds * 64, hi);
  uint32_t held[SEL_HELD];
#pragma unroll
  for (int r = 0; r < SEL_HELD; ++r)
    if (r < rounds) held[r] = __float_as_uint(w[min(begin + r * 64 + lane, hi - 1)]);
#pragma unroll
  for (int r = 0; r < SEL_HELD; ++r) held[r] = begin + r * 64 + lane < end ? weight_key(__uint_as_float(held[r])) : 0u;
  // f(key, index) for the wave's share, in order, all lanes each time; key 0: past the share
  auto each = [&](auto&& f) {
#pragma unroll
    for (int r = 0; r < SEL_HELD; ++r)
      if (r < rounds) f(held[r], begin + r * 64 + lane);
    for (int r = SEL_HELD; r < rounds; ++r) {
      const int i = begin + r * 64 + lane;
      f(i < end ? weight_key(w[i]) : 0u, i);
    }
  };

  uint32_t prefix = 0;  // the bits of the smallest kept key found so far
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < SEL_BINS; i += SEL_THREADS) hist[i] = 0;
    __syncthreads();
    each([&](uint32_t key, int) {
      if (pass == 0 ? key != 0 : key >> (shift + bits) == prefix >> (shift + bits))
        atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1)], 1u);
    });
    __syncthreads();
    // counts from the top: thread t holds bins 2t and 2t + 1
    const uint32_t c0 = hist[2 * tid], c1 = hist[2 * tid + 1];
    uint32_t above = c0 + c1;  // inclusive suffix sum over the wave's lanes
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t v = __shfl_down(above, off, 64);
      if (lane + off < 64) above += v;
    }
    if (lane == 0) wave_a[wave] = above;
    __syncthreads();
    for (int i = wave + 1; i < SEL_WAVES; ++i) above += wave_a[i];
    const uint32_t over1 = above - c0 - c1, over0 = above - c0;  // keys in higher bins than 2t + 1, than 2t
    if (over1 < room && over1 + c1 >= room) {
      found[0] = 2 * tid + 1;
      found[1] = over1;
    } else if (over0 < room && over0 + c0 >= room) {
      found[0] = 2 * tid;
      found[1] = over0;
    }
    __syncthreads();
    prefix |= found[0] << shift;
    room -= found[1];
    __syncthreads();
  }
  // `room` of the keys equal to `prefix` are kept, the lowest indices
  uint32_t more = 0, same = 0;
  each([&](uint32_t key, int) {
    more += key > prefix;
    same += key == prefix;
  });
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    more += __shfl_xor(more, m, 64);
    same += __shfl_xor(same, m, 64);
  }
  if (lane == 0) {
    wave_a[wave] = more;
    wave_b[wave] = same;
  }
  __syncthreads();
  uint32_t at = p.first, ties = 0;  // rows kept and equal keys met before this wave's share
  for (int i = 0; i < wave; ++i) {
    at += wave_a[i];
    ties += wave_b[i];
  }
  at += min(ties, room);
  // set bits of lanes before this one
  auto rank_of = [](uint64_t m) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
  };
  each([&](uint32_t key, int i) {
    const uint64_t eq = __builtin_amdgcn_ballot_w64(key == prefix);
    bool take = key > prefix;
    if (eq) {
      take |= key == prefix && ties + rank_of(eq) < room;
      ties += __popcll(eq);
    }
    const uint64_t taken = __builtin_amdgcn_ballot_w64(take);
    const uint32_t to = at + rank_of(taken);
    if (take && to < (uint32_t)(p.keep - p.recent)) kept[to] = i;  // (weights that change meanwhile)
    at += __popcll(taken);
  });
}

// ---------------------------------------------------------------- moving rows
// Row kept[b, h, i] of a sequence's pages to row i of its new pages, for every part of a
// row (K and V rows; of 4-bit pages codes and scales), and its weight.  A workgroup moves
// 64 rows: their places are worked out once, in LDS, then each thread has all its pieces
// of a part in flight.  HBM-bound, each kept row read and written once, past the caches: 8
// x 8 heads, 8192 of 32768 bf16 rows (D = 128, K and V, 537 MB) take 104 us, as a contiguous
// copy of as much; through the caches 117.  As many 4-bit rows (143 MB): 42 us, 3.4 TB/s;
// through the caches 71.
struct RowPart {
  int64_t off;    // of the part within a page's head (bytes)
  int stride;     // between rows (bytes)
  int pool;        // which
  Divider pieces;  // pieces of a row's part
};
struct CompactParams {
  unsigned char* pool[2];
  int64_t psb[2], psh[2];  // page and head strides (bytes)
  RowPart part[4];
  int npages, cols, row_groups;
  Divider page;
  const int32_t *bt, *new_bt;
  int64_t bts, nbts;
  const int32_t* kept;
  const float* w;
  float* w_out;
  int64_t wsb, wsh;
  int Hkv, keep, W;
};

constexpr int CP_ROWS = 64;  // rows of a workgroup

// N pieces of a part that a thread has in flight.
template <typename T, int N> struct Moves {
  T v[N];
  unsigned char* dst[N];
  __device__ __forceinline__ void load(const CompactParams& p, const RowPart& q, int h, const int (*place)[4], int rows,
                                       int first) {
    unsigned char* pool = p.pool[q.pool] + h * p.psh[q.pool] + q.off;
    const int64_t psb = p.psb[q.pool];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int id = first + u * 256;
      dst[u] = nullptr;
      if (id >= rows * (int)q.pieces.d) continue;
      int piece;
      const int* at = place[q.pieces.div(id, piece)];
      if (at[0] < 0) continue;
      const int o = piece * (int)sizeof(T);
      v[u] = __builtin_nontemporal_load(reinterpret_cast<const T*>(pool + at[0] * psb + (int64_t)at[1] * q.stride + o));
      dst[u] = pool + at[2] * psb + (int64_t)at[3] * q.stride + o;
    }
  }
  __device__ __forceinline__ void store() {
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (dst[u]) __builtin_nontemporal_store(v[u], reinterpret_cast<T*>(dst[u]));
  }
};

// S: void for K and V pools, else a row's scales in 4-bit pages.
template <typename S>
__global__ void __launch_bounds__(256) compact_rows_kernel(CompactParams p) {
  __shared__ int place[CP_ROWS][4];  // page and row: from, to; page -1: nothing to move
  const int b = blockIdx.z, h = blockIdx.y;
  if ((int)blockIdx.x >= p.row_groups) {  // weights of the rows that are no more
    const int64_t t = (int64_t)((int)blockIdx.x - p.row_groups) * 256 + threadIdx.x + p.keep;
    if (t < p.W) p.w_out[b * p.wsb + h * p.wsh + t] = 0.f;
    return;
  }
  const int i0 = blockIdx.x * CP_ROWS, rows = min(CP_ROWS, p.keep - i0);
  if ((int)threadIdx.x < rows) {
    const int i = i0 + threadIdx.x;
    const int j = p.kept[((int64_t)b * p.Hkv + h) * p.keep + i];
    int from = -1, to = -1, fr = 0, tr = 0;
    if (j >= 0) {
      const int col = p.page.div(j, fr);
      if (col < p.cols) {
        from = p.bt[b * p.bts + col];
        to = p.new_bt[b * p.nbts + p.page.div(i, tr)];
      }
      if (p.w_out) p.w_out[b * p.wsb + h * p.wsh + i] = col < p.cols && j < p.W ? p.w[b * p.wsb + h * p.wsh + j] : 0.f;
    } else if (p.w_out) {
      p.w_out[b * p.wsb + h * p.wsh + i] = 0.f;
    }
    const bool real = (uint32_t)from < (uint32_t)p.npages && (uint32_t)to < (uint32_t)p.npages;
    place[threadIdx.x][0] = real ? from : -1;
    place[threadIdx.x][1] = fr;
    place[threadIdx.x][2] = to;
    place[threadIdx.x][3] = tr;
  }
  __syncthreads();
  // all loads before the stores: a store holds up what follows it for as long as a load
  if constexpr (std::is_void<S>::value) {
    for (int first = threadIdx.x; first < rows * (int)p.part[0].pieces.d; first += 256 * 4) {
      Moves<bf16x8, 4> k, v;
      k.load(p, p.part[0], h, place, rows, first);
      v.load(p, p.part[1], h, place, rows, first);
      k.store();
      v.store();
    }
  } else {  // 64 rows of at most 64 code bytes: a piece a thread
    Moves<bf16x8, 1> k, v;
    Moves<S, 1> ks, vs;
    k.load(p, p.part[0], h, place, rows, threadIdx.x);
    v.load(p, p.part[1], h, place, rows, threadIdx.x);
    ks.load(p, p.part[2], h, place, rows, threadIdx.x);
    vs.load(p, p.part[3], h, place, rows, threadIdx.x);
    k.store();
    v.store();
    ks.store();
    vs.store();
  }
}

}  // namespace nq

using namespace nq;

static int evict_check_table(const int32_t* bt, int64_t stride, int cols, int page_size, int num_pages) {
  if (!bt || cols <= 0 || stride < cols || num_pages <= 0)
    return nq_fail(NQ_ERR_INVALID, "a block table, its columns and pages are required, its rows at least bt_cols apart");
  if (page_size <= 0 || page_size % 32 || page_size > (1 << 20))
    return nq_fail(NQ_ERR_UNSUPPORTED, "page_size must be a multiple of 32 up to 2^20, got %d", page_size);
  return NQ_OK;
}

extern "C" int64_t nq_key_weights_workspace_bytes(int B, int Hq, int Hkv, int S, int max_len) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || S <= 0 || max_len <= 0 || Hq % Hkv) return 0;
  const int64_t R = (int64_t)S * (Hq / Hkv);
  const int64_t n = R <= 16 ? 1 : key_weight_chunks(R);
  return n > 1 ? n * B * Hkv * max_len * (int64_t)sizeof(float) : 0;
}

extern "C" int nq_key_weights(const void* q, const int64_t* q_strides, const void* k_pool,
                              const int64_t* pool_strides, int four_bit, int num_pages, const int32_t* block_table,
                              int64_t bt_stride, int bt_cols, int page_size, const int32_t* lens, const float* lse,
                              float* weights, const int64_t* weight_strides, int accumulate, void* workspace,
                              int64_t workspace_bytes, int B, int Hq, int Hkv,
                              int S, int D, int max_len, int causal, float sm_scale, void* stream) {
  nq_clear_error();
  if (!head_dim_ok(D)) return nq_fail(NQ_ERR_UNSUPPORTED, "head_dim must be 32, 64 or 128, got %d", D);
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || S <= 0 || max_len <= 0)
    return nq_fail(NQ_ERR_INVALID, "sizes must be positive (B=%d Hq=%d Hkv=%d S=%d max_len=%d)", B, Hq, Hkv, S, max_len);
  if (Hq % Hkv) return nq_fail(NQ_ERR_INVALID, "num_heads %d not divisible by num_kv_heads %d", Hq, Hkv);
  int rc = evict_check_table(block_table, bt_stride, bt_cols, page_size, num_pages);
  if (rc != NQ_OK) return rc;
  if (!q || !q_strides || !k_pool || !pool_strides || !lens || !lse || !weights || !weight_strides)
    return nq_fail(NQ_ERR_INVALID, "q, the pool, lens, lse, weights and their strides are required");
  if ((max_len + page_size - 1) / page_size > bt_cols)
    return nq_fail(NQ_ERR_INVALID, "the block table's %d columns hold fewer than max_len %d rows", bt_cols, max_len);
  if (!nq_aligned16(q) || !nq_aligned16(k_pool)) return nq_fail(NQ_ERR_INVALID, "q and the pool must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % 8) return nq_fail(NQ_ERR_INVALID, "q strides must be multiples of 16 bytes");
  // a chunk of 256 rows is addressed with 32-bit offsets
  if (q_strides[1] < 0 || q_strides[2] < 0 || q_strides[1] > (1 << 30) / (Hq / Hkv) || q_strides[2] > (1 << 30) / 257)
    return nq_fail(NQ_ERR_UNSUPPORTED, "q strides of 256 rows exceed 2^30 elements, or are negative");
  for (int i = 0; i < (four_bit ? 2 : 3); ++i)
    if (pool_strides[i] % (four_bit ? 16 : 8)) return nq_fail(NQ_ERR_INVALID, "pool strides must be multiples of 16 bytes");
  if (B > 65535 || Hkv > 65535 || (int64_t)S * (Hq / Hkv) > (1 << 24) || max_len > (1 << 30))
    return nq_fail(NQ_ERR_UNSUPPORTED, "at most 65535 sequences and kv heads, 2^24 query rows a kv head and 2^30 keys");
  KeyWeightParams p{};
  p.q = reinterpret_cast<const bf16*>(q); p.qsb = q_strides[0]; p.qsh = q_strides[1]; p.qss = q_strides[2];
  p.pool = k_pool; p.psb = pool_strides[0]; p.psh = pool_strides[1]; p.pss = four_bit ? 0 : pool_strides[2];
  p.npages = num_pages; p.bt = block_table; p.bts = bt_stride; p.page = Divider(page_size);
  p.lens = lens; p.lse = lse; p.w = weights; p.wsb = weight_strides[0]; p.wsh = weight_strides[1];
  p.add = accumulate != 0; p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.G = Divider(Hq / Hkv); p.S = S; p.max_len = max_len;
  p.causal = causal != 0 && S > 1;
  p.scale_log2 = (sm_scale > 0.f ? sm_scale : 1.0f / sqrtf((float)D)) * kLog2e;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t R = (int64_t)S * p.G.d;
  if (R <= 16) {
    p.range = Divider(four_bit ? key_weight_span(p) : 64);
    const int64_t keys = 4 * (int64_t)p.range.d;
    const dim3 grid((unsigned)((max_len + keys - 1) / keys), (unsigned)Hkv, (unsigned)B);
    return nq_check_launch(with_head_dim(D, [&](auto dc) {
      constexpr int DD = decltype(dc)::value;
      if (four_bit && p.add) hipLaunchKernelGGL((key_weights_step_kernel<DD, true, true>), grid, dim3(256), 0, st, p);
      else if (four_bit) hipLaunchKernelGGL((key_weights_step_kernel<DD, true, false>), grid, dim3(256), 0, st, p);
      else if (p.add) hipLaunchKernelGGL((key_weights_step_kernel<DD, false, true>), grid, dim3(256), 0, st, p);
      else hipLaunchKernelGGL((key_weights_step_kernel<DD, false, false>), grid, dim3(256), 0, st, p);
      return hipGetLastError();
    }));
  }
  p.chunks = key_weight_chunks(R);
  p.chunk_rows = KW_ROWS;
  if (p.chunks > 1) {
    const int64_t need = nq_key_weights_workspace_bytes(B, Hq, Hkv, S, max_len);
    if (!workspace || workspace_bytes < need || !nq_aligned16(workspace))
      return nq_fail(NQ_ERR_WORKSPACE, "an aligned workspace of %lld bytes is required, %lld given", (long long)need,
                     (long long)workspace_bytes);
    p.part = reinterpret_cast<float*>(workspace);
  }
  p.range = Divider(key_weight_range(p));
  if (p.chunks > KW_FEW_CHUNKS) p.same = p.range.div(max_len + (int)p.range.d - 1);
  const int64_t groups = p.same ? (int64_t)p.chunks * p.same : key_weight_groups(p);
  if (groups > 0xffffff) return nq_fail(NQ_ERR_UNSUPPORTED, "more query rows and keys than one launch takes");
  const dim3 grid((unsigned)groups, (unsigned)Hkv, (unsigned)B);
  hipError_t e = with_head_dim(D, [&](auto dc) {
    constexpr int DD = decltype(dc)::value;
    if (four_bit) hipLaunchKernelGGL((key_weights_kernel<DD, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((key_weights_kernel<DD, false>), grid, dim3(256), 0, st, p);
    return hipGetLastError();
  });
  if (e == hipSuccess && p.chunks > 1) {
    hipLaunchKernelGGL(key_weights_sum_kernel, dim3((unsigned)((max_len + 255) / 256), (unsigned)Hkv, (unsigned)B), dim3(256),
                       0, st, p);
    e = hipGetLastError();
  }
  return nq_check_launch(e);
}

extern "C" int nq_select_keys(const float* weights, const int64_t* weight_strides, const int32_t* lens, int32_t* kept,
                              int B, int Hkv, int width, int keep, int recent, int first, void* stream) {
  nq_clear_error();
  if (B <= 0 || Hkv <= 0 || width <= 0 || keep <= 0)
    return nq_fail(NQ_ERR_INVALID, "sizes must be positive (B=%d Hkv=%d width=%d keep=%d)", B, Hkv, width, keep);
  if (recent < 0 || first < 0 || (int64_t)recent + first > keep)
    return nq_fail(NQ_ERR_INVALID, "first %d and recent %d must fit keep %d", first, recent, keep);
  if (!weights || !weight_strides || !lens || !kept)
    return nq_fail(NQ_ERR_INVALID, "weights, their strides, lens and kept are required");
  if (width > (1 << 30) || keep > (1 << 30))  // indices, rounded up to a workgroup's rounds, are ints
    return nq_fail(NQ_ERR_UNSUPPORTED, "at most 2^30 weights and kept rows a head");
  if ((int64_t)B * Hkv * SEL_THREADS > 0xffffffffll)  // a launch has fewer than 2^32 threads
    return nq_fail(NQ_ERR_UNSUPPORTED, "more (sequence, kv head) rows than one launch takes");
  SelectParams p{weights, weight_strides[0], weight_strides[1], lens, kept, Hkv, width, keep, recent, first};
  hipLaunchKernelGGL(select_keys_kernel, dim3((unsigned)(B * Hkv)), dim3(SEL_THREADS), 0,
                     reinterpret_cast<hipStream_t>(stream), p);
  return nq_check_launch(hipGetLastError());
}

extern "C" int nq_kv_compact(void* k_pool, const int64_t* k_strides, void* v_pool, const int64_t* v_strides,
                             int row_bytes, int head_dim, int num_pages, const int32_t* block_table,
                             int64_t bt_stride, int bt_cols, const int32_t* new_table, int64_t new_stride,
                             int new_cols, int page_size, const int32_t* kept, const float* weights,
                             float* weights_out, const int64_t* weight_strides, int width, int B, int Hkv, int keep,
                             void* stream) {
  nq_clear_error();
  if (B <= 0 || Hkv <= 0 || keep <= 0) return nq_fail(NQ_ERR_INVALID, "sizes must be positive (B=%d Hkv=%d keep=%d)", B, Hkv, keep);
  if (B > 65535 || Hkv > 65535) return nq_fail(NQ_ERR_UNSUPPORTED, "at most 65535 sequences and kv heads");
  int rc = evict_check_table(block_table, bt_stride, bt_cols, page_size, num_pages);
  if (rc == NQ_OK) rc = evict_check_table(new_table, new_stride, new_cols, page_size, num_pages);
  if (rc != NQ_OK) return rc;
  if (new_table == block_table) return nq_fail(NQ_ERR_INVALID, "new_table must name other pages than block_table");
  if ((int64_t)new_cols * page_size < keep)
    return nq_fail(NQ_ERR_INVALID, "the new table's %d columns hold fewer than the %d kept rows", new_cols, keep);
  const bool four = v_pool == nullptr;
  if (!k_pool || !k_strides || !kept || (!four && !v_strides))
    return nq_fail(NQ_ERR_INVALID, "the pools, their strides and the kept rows are required");
  if ((weights == nullptr) != (weights_out == nullptr) || (weights && (!weight_strides || width < keep)))
    return nq_fail(NQ_ERR_INVALID, "weights, weights_out, their strides and a width of at least keep go together");
  if (weights && weights == weights_out) return nq_fail(NQ_ERR_INVALID, "weights_out must not be weights");
  CompactParams p{};
  if (four) {
    if (!head_dim_ok(head_dim)) return nq_fail(NQ_ERR_UNSUPPORTED, "head_dim must be 32, 64 or 128, got %d", head_dim);
    const int cb = head_dim / 2, sb = head_dim / 32;
    p.part[0] = RowPart{0, cb, 0, Divider(cb / 16)};
    p.part[1] = RowPart{(int64_t)page_size * cb, cb, 0, Divider(cb / 16)};
    p.part[2] = RowPart{(int64_t)page_size * 2 * cb, sb, 0, Divider(1)};
    p.part[3] = RowPart{(int64_t)page_size * (2 * cb + sb), sb, 0, Divider(1)};
  } else {
    if (row_bytes <= 0 || row_bytes % 16 || row_bytes > (1 << 20) || k_strides[2] < row_bytes || v_strides[2] < row_bytes ||
        k_strides[2] > (1 << 30) || v_strides[2] > (1 << 30))
      return nq_fail(NQ_ERR_INVALID, "rows must be multiples of 16 bytes that do not overlap, got %d", row_bytes);
    p.part[0] = RowPart{0, (int)k_strides[2], 0, Divider(row_bytes / 16)};
    p.part[1] = RowPart{0, (int)v_strides[2], 1, Divider(row_bytes / 16)};
    p.pool[1] = reinterpret_cast<unsigned char*>(v_pool); p.psb[1] = v_strides[0]; p.psh[1] = v_strides[1];
  }
  p.pool[0] = reinterpret_cast<unsigned char*>(k_pool); p.psb[0] = k_strides[0]; p.psh[0] = k_strides[1];
  for (int i = 0; i < (four ? 1 : 2); ++i) {
    if (!nq_aligned16(p.pool[i]) || p.psb[i] % 16 || p.psh[i] % 16 || (!four && (i ? v_strides : k_strides)[2] % 16))
      return nq_fail(NQ_ERR_INVALID, "the pools and their strides must be multiples of 16 bytes");
  }
  p.npages = num_pages; p.page = Divider(page_size); p.cols = bt_cols;
  p.bt = block_table; p.bts = bt_stride; p.new_bt = new_table; p.nbts = new_stride;
  p.kept = kept; p.w = weights; p.w_out = weights_out;
  if (weights) { p.wsb = weight_strides[0]; p.wsh = weight_strides[1]; }
  p.Hkv = Hkv; p.keep = keep; p.W = weights ? width : keep;
  p.row_groups = (keep + CP_ROWS - 1) / CP_ROWS;
  const int64_t groups = p.row_groups + ((int64_t)p.W - keep + 255) / 256;
  if (groups > 0xffffff) return nq_fail(NQ_ERR_UNSUPPORTED, "more kept rows than one launch takes");
  const dim3 grid((unsigned)groups, (unsigned)Hkv, (unsigned)B);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (!four) hipLaunchKernelGGL((compact_rows_kernel<void>), grid, dim3(256), 0, st, p);
  else if (head_dim == 128) hipLaunchKernelGGL((compact_rows_kernel<uint32_t>), grid, dim3(256), 0, st, p);
  else if (head_dim == 64) hipLaunchKernelGGL((compact_rows_kernel<uint16_t>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((compact_rows_kernel<unsigned char>), grid, dim3(256), 0, st, p);
  return nq_check_launch(hipGetLastError());
}
