// Rows into 4-bit pages, rows of 4-bit pages read back, and single-token attention
// over them, for gfx950.  The page format is nq_kv4.hpp's.  No counterpart in the
// reference, whose cache (model/attention.py:24-46) holds the model's type.

#include <type_traits>

#include "nq_common.hpp"
#include "nq_decode.hpp"
#include "nq_internal.hpp"
#include "nq_kv4.hpp"

namespace nq {

// ---------------------------------------------------------------- rows into pages
constexpr int64_t KV4_MOST_LANES = 0x7fffff00;  // of a launch in x

struct Kv4AppendParams {
  const void *k, *v, *q;
  int64_t ksb, ksh, kss, vsb, vsh, vss, qsb, qsh, qss;
  void* q_out;
  int64_t osb, osh, oss;
  unsigned char* pool;
  int64_t psb, psh;  // page and head strides (bytes)
  int npages;
  const int32_t* bt;
  int64_t bts;
  int64_t cap;  // rows that the block table maps
  int page;
  Divider by_S, by_HT, by_page;  // HT = Hq + 2 Hkv
  int B, S, Hq, Hkv;
  const void *qw, *kw;
  int q16, k16;
  float eps;
  const float *cos_tab, *sin_tab;
  int max_pos;
  const int32_t *pos, *pos_base, *pos_shift;
  int pos0;
  const int32_t* row_base;
  int row0;
  int32_t* lens_out;
};

// Largest magnitude's bits over groups of N = 2 or 4 lanes.
template <int N>
__device__ __forceinline__ uint32_t group_max_bits(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));  // quad xor 1
  if (N == 4) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));  // quad xor 2
  return v;
}

__device__ __forceinline__ uint32_t max_bits8(const floatx8& x) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
  return m;
}

// Codes of 8 elements, rounded to the nearest (halfway: the even code) and to +-6
// where beyond.
__device__ __forceinline__ uint32_t kv4_codes8(const floatx8& x, float scale) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], scale, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], scale, 3);
  return c;
}

// One row of k, v or q to D/16 lanes: lane `sub` holds elements [8 sub, +8) and
// [D/2 + 8 sub, +8), the layout of norm_row / rope_row, in which a block of 32 is
// four lanes' first or second chunk (D = 32: both chunks of two lanes).  K rows are
// normed and rotated in fp32 and rounded once, to their codes; q rows likewise, to
// q_out.  The tokens of a head are consecutive lanes, so a page's codes and scales are
// written in runs.  HBM-bound: each row read once, 17 D / 32 bytes written.  4 sequences,
// 2048 tokens, 8 heads of 128, K and V (42 MB): 10.4 us, 4.1 TB/s; with the heads of a
// token consecutive 9% more.  A single token of 64 sequences: 4.0 us, the launch and its
// dependent loads.
template <int D, typename T>
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4AppendParams p) {
  using L = Kv4<D>;
  constexpr int LPR = D / 16;
  const int64_t gl = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row64 = gl / LPR;
  const int sub = (int)(gl % LPR);
  if (row64 >= (int64_t)p.B * p.S * (p.Hq + 2 * p.Hkv)) return;  // whole groups of LPR lanes leave together
  int s, h;
  const int b = p.by_HT.div(p.by_S.div((int)row64, s), h);
  const int base = p.row_base ? p.row_base[b] : p.row0;
  const bool fits = base >= 0 && (int64_t)base + p.S <= p.cap;
  if (p.lens_out && h == 0 && s == 0 && sub == 0) p.lens_out[b] = fits ? base + p.S : base;
  const bool is_q = h < p.Hq, is_k = !is_q && h < p.Hq + p.Hkv;
  if (!is_q && !fits) return;
  const T* src;
  if (is_q) {
    src = reinterpret_cast<const T*>(p.q) + b * p.qsb + h * p.qsh + s * p.qss;
  } else if (is_k) {
    h -= p.Hq;
    src = reinterpret_cast<const T*>(p.k) + b * p.ksb + h * p.ksh + s * p.kss;
  } else {
    h -= p.Hq + p.Hkv;
    src = reinterpret_cast<const T*>(p.v) + b * p.vsb + h * p.vsh + s * p.vss;
  }
  floatx8 x1 = Vec8<T>::load_f32(src + sub * 8), x2 = Vec8<T>::load_f32(src + D / 2 + sub * 8);
  if (is_q || is_k) {
    const void* w = is_q ? p.qw : p.kw;
    if (w) {
      const int w16 = is_q ? p.q16 : p.k16;
      Weight8 a, c;
      a.load(w, w16, sub * 8);
      c.load(w, w16, D / 2 + sub * 8);
      norm_row<D>(x1, x2, a.value(w16), c.value(w16), p.eps);
    }
    if (p.cos_tab) {
      int at = row_position(p.pos, p.pos_base, p.pos0, b, s, p.S);
      if (p.pos_shift) at += p.pos_shift[b];
      at = table_row(at, p.max_pos);
      rope_row(x1, x2, load_tab8(p.cos_tab, at, D / 2, sub * 8), load_tab8(p.sin_tab, at, D / 2, sub * 8));
    }
  }
  if (is_q) {
    T* dst = reinterpret_cast<T*>(p.q_out) + b * p.osb + h * p.osh + s * p.oss;
    store8<T>(dst + sub * 8, x1);
    store8<T>(dst + D / 2 + sub * 8, x2);
    return;
  }
  uint32_t m1 = max_bits8(x1), m2 = max_bits8(x2);
  if (D == 32) m1 = m2 = max(m1, m2);
  constexpr int LPB = D == 32 ? 2 : 4;  // lanes of a block
  const uint32_t e1 = kv4_scale_byte(group_max_bits<LPB>(m1)), e2 = kv4_scale_byte(group_max_bits<LPB>(m2));
  int in;
  const int pid = p.bt[b * p.bts + p.by_page.div(base + s, in)];
  if ((uint32_t)pid >= (uint32_t)p.npages) return;  // not a page of the pool
  unsigned char* rec = p.pool + pid * p.psb + h * p.psh;
  unsigned char* codes = rec + (is_k ? 0 : L::v_codes(p.page)) + in * L::CB;
  unsigned char* scales = rec + (is_k ? L::k_scales(p.page) : L::v_scales(p.page)) + in * L::SB;
  *reinterpret_cast<uint32_t*>(codes + sub * 4) = kv4_codes8(x1, kv4_scale(e1 == 255 ? 127 : e1));
  *reinterpret_cast<uint32_t*>(codes + L::CB / 2 + sub * 4) = kv4_codes8(x2, kv4_scale(e2 == 255 ? 127 : e2));
  if (sub % LPB == 0) {
    scales[sub / LPB] = (unsigned char)e1;
    if (D > 32) scales[L::SB / 2 + sub / LPB] = (unsigned char)e2;
  }
}

// ---------------------------------------------------------------- rows read back
struct Kv4GatherParams {
  const unsigned char* pool;
  int64_t psb, psh;
  int npages;
  const int32_t* bt;
  int64_t bts;
  int64_t cap;
  int page;
  void *k, *v;
  int64_t ksb, ksh, kss, vsb, vsh, vss;
  Divider by_S, by_H, by_page;
  int B, S, Hkv;
  const int32_t* row_base;
  int row0;
};

// A row's 16 elements a lane, 8 of either half, so that each store of a wave fills whole
// lines; the rows of a head consecutive; the codes read past the caches, where the rows
// written lie for their reader.  HBM-bound by its writes: 8192 rows of 4 sequences and
// 8 heads of 128, K and V (170 MB), take 31 us, 5.5 TB/s.  With the append above, over
// changing pools, 46.4 us; 53.7 with 16 adjacent elements a lane, 47.9 with the codes
// cached.  A row without a page reads as NaN.
template <int D, typename T>
__global__ void __launch_bounds__(256) kv4_gather_kernel(Kv4GatherParams p) {
  using L = Kv4<D>;
  constexpr int LPR = D / 16;
  const int64_t gl = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row64 = gl / LPR;
  const int sub = (int)(gl % LPR);
  if (row64 >= (int64_t)p.B * p.S * p.Hkv) return;
  int s, h;
  const int b = p.by_H.div(p.by_S.div((int)row64, s), h);
  const bool is_v = blockIdx.y;
  const int64_t r = (int64_t)(p.row_base ? p.row_base[b] : p.row0) + s;
  T* dst = is_v ? reinterpret_cast<T*>(p.v) + b * p.vsb + h * p.vsh + s * p.vss
                : reinterpret_cast<T*>(p.k) + b * p.ksb + h * p.ksh + s * p.kss;
  uint32_t c[2] = {0, 0}, e[2] = {255, 255};
  if (r >= 0 && r < p.cap) {
    int in;
    const int pid = p.bt[b * p.bts + p.by_page.div((int)r, in)];
    if ((uint32_t)pid < (uint32_t)p.npages) {
      const unsigned char* rec = p.pool + pid * p.psb + h * p.psh;
      const unsigned char* codes = rec + (is_v ? L::v_codes(p.page) : 0) + in * L::CB + sub * 4;
      c[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(codes));
      c[1] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(codes + L::CB / 2));
      const unsigned char* scales = rec + (is_v ? L::v_scales(p.page) : L::k_scales(p.page)) + in * L::SB;
      e[0] = scales[sub / 4];
      e[1] = scales[(D / 2 + sub * 8) / 32];
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bf16x8 v = kv4_bf16x8(c[i], kv4_scale(e[i]));
    store8<T>(dst + sub * 8 + i * (D / 2), __builtin_convertvector(v, floatx8));
  }
}

// ---------------------------------------------------------------- decode
// o = softmax(scale q K^T) V over the keys [0, lens[b]) of each sequence.  Rows (sequence,
// kv head, up to 16 query heads) are cut into steps of 32 keys as in the bf16 decode
// (nq_decode.hip); a workgroup takes a contiguous range of a row's steps, each of its W waves
// every W-th step, and joins them in LDS.  Either a workgroup of eight waves takes a whole
// row and writes its output (few or short rows: one launch), or a persistent grid of
// workgroups of four shares the steps of all rows evenly, and partials meet in the bf16
// decode's merge.
//
// How a step's 32 keys reach the matrix cores:
//   K: a 16-key tile is one load per lane of D/4 consecutive elements of a row, in the
//     order in which the MFMA's k slots are taken (slot 8 g + j of MFMA i is element
//     g D/4 + 8 i + j, for q as well), and one scale byte, since those elements lie in
//     one block.  They become bf16 operands in registers, without LDS.
//   V: whole rows as they lie in the page; a lane's codes become bf16 in registers, go
//     to a wave-private LDS tile and come back transposed, as in the bf16 decode.
// Codes times a power of two are exact in bf16, so the products are those of a bf16
// cache that held the same values.  fp32 queries: q and the probabilities are split into
// three bf16 terms each (8 + 8 + 8 significant bits), three MFMAs in place of one.  bf16
// queries: the probabilities are rounded to bf16 for the second product, as in the bf16
// decode; outputs lie 1.9-2.0e-3 from 64 bits (2-norm), 1.6e-3 of it their own rounding.
//
// The running maximum is raised only for a score more than 2^8 above it: most steps then
// exchange nothing between lanes and rescale no output, and the sums, held in fp32, have
// room for the larger terms.
//
// HBM-bound: 17/16 D bytes a cached row and kv head.  64 sequences of 1024 to 32768 keys, 64/4
// heads, D = 128 (539 MB): 93 us, 5.8 TB/s, and 4.6 for the merge.  What remains is uneven
// ends: workgroups of equal ranges end between 64 and 94 us (a tenth by 70, nine by 89).
// Waves that each took a range of their own (2048 of them, and partials) took 107 with the
// merge; a whole row to a workgroup there 132, its rows differing in length.
// Loads of two steps in flight a wave; three or four gained nothing.
constexpr int KV4_ROW_WAVES = 8;          // of a workgroup that takes a row of its own
constexpr int KV4_WAVES = 4;              // of one of the persistent grid's
constexpr int KV4_PER_CU = 2;             // of which a CU holds this many
constexpr int KV4_MAX_GROUPS = 256 * KV4_PER_CU;
// What a row's start counts for in the split, in steps: its workgroup waits for block table,
// first codes and the join, about 4.5 us, in which the CU's other one goes on.  At 0, 64
// sequences of 1024 to 32768 keys (64/4 heads) took 105 us, at 24 99.
constexpr int KV4_ROW_COST = 24;
constexpr int KV4_DEPTH = 2;              // steps of a wave whose loads are in flight
constexpr float KV4_SLACK = 8.f;          // log2 of how far a score may exceed the running maximum

// One step's codes and scales as loaded.
template <int D> struct Kv4Step {
  static constexpr int KW = D / 32;                    // K dwords a lane and 16-key tile
  static constexpr int VB = D == 32 ? 8 : 16;          // V bytes a lane and load
  static constexpr int VL = D / 4 / VB;                // V loads a step
  uint32_t k[2][KW], ks[2];
  uint32_t v[VL][VB / 4], vs[VL];
};

template <int N>
__device__ __forceinline__ void kv4_load(uint32_t (&d)[N], BufRsrc r, int voff, int soff) {
  if constexpr (N == 4) {
    const auto w = __builtin_amdgcn_raw_buffer_load_b128(r, voff, soff, 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = w[i];
  } else if constexpr (N == 2) {
    const auto w = __builtin_amdgcn_raw_buffer_load_b64(r, voff, soff, 2);
    d[0] = w[0];
    d[1] = w[1];
  } else {
    d[0] = __builtin_amdgcn_raw_buffer_load_b32(r, voff, soff, 2);
  }
}

// x as the sum of NT bf16 vectors (NT = 1: x rounded).
template <int NT>
__device__ __forceinline__ void split_bf16(floatx8 x, bf16x8 (&out)[NT]) {
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    out[t] = to_bf16x8(x);
    if (t + 1 < NT) x -= __builtin_convertvector(out[t], floatx8);
  }
}

__device__ __forceinline__ float xor16_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor16_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

struct Kv4DecodeParams {
  DecodeParams d;  // kc: the pool; ksb, ksh: page and head strides in bytes; nwaves: workgroups
  int npages;
  uint32_t pu, magic;  // steps of a page, floor(2^32 / pu)
};

template <int D, typename T, bool ROWS, int W = ROWS ? KV4_ROW_WAVES : KV4_WAVES>
__global__ void __attribute__((amdgpu_flat_work_group_size(W * 64, W * 64), amdgpu_waves_per_eu(2)))
decode_kv4_kernel(Kv4DecodeParams pp) {
  const DecodeParams& p = pp.d;
  using F = Kv4<D>;
  using L = DcTile<D>;
  using Step = Kv4Step<D>;
  constexpr int NT = std::is_same<T, float>::value ? 3 : 1;
  constexpr int NDQ = D / 32, NDO = D / 16;
  static_assert(L::BYTES == 16 * D * 4, "a wave's V tile holds its outputs");
  __shared__ __attribute__((aligned(16))) unsigned char smem[W * L::BYTES];
  __shared__ floatx2 part_ml[W][16];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, grp = lane >> 4;
  Walk<ROWS ? 0 : KV4_ROW_COST> at;
  if constexpr (ROWS) {
    const int r = blockIdx.x;
    at.b = r / p.rows_per_batch;
    at.j = r % p.rows_per_batch;
    at.ls = 0;
    at.lens_in_reg = false;
    at.nb = batch_steps(p, at.b);
    at.q = 0;
    at.q1 = at.nb;
    if (at.nb == 0) {  // no keys: zeros; a length out of range: NaN
      const int kvh = at.j / p.NG, hg = at.j % p.NG, nh = min(16, p.G - hg * 16);
      const int len = batch_len(p, at.b);
      const float f = len < 0 ? __builtin_nanf("") : 0.f;
      const int head0 = kvh * p.G + hg * 16;
      T* out = reinterpret_cast<T*>(p.o) + at.b * p.osb + (int64_t)head0 * p.osh;
      for (int t = threadIdx.x; t < nh * (D / 2); t += (W * 64))
        store2<T>(out + (t / (D / 2)) * p.osh + (t % (D / 2)) * 2, f, f);
      if (p.lse && threadIdx.x < (unsigned)nh) p.lse[(int64_t)at.b * p.Hq + head0 + threadIdx.x] = len < 0 ? f : -INFINITY;
      return;
    }
  } else {
    // Even ranges: weighted as the bf16 decode's are, 64 sequences of up to 32768 keys took
    // 101 us, even 99.  (The wave of the walk is a workgroup here.)  Their least size: one
    // sequence of 10000 keys, 8/1 heads, took 26 us over 338 workgroups of a step, 13 over 42
    // of 8; of 32768, 64/4 heads, 29 over 512 and 20 over 190.
    if (!at.template start<true>(p, lane, blockIdx.x)) return;
  }
  unsigned char* vt = smem + wave * L::BYTES;

  // byte offsets within a step's codes and scales
  const int kvo = c16 * F::CB + grp * (D / 8), kso = c16 * F::SB + grp * (D / 4) / 32;
  const int vvo = lane * Step::VB, vso = lane * Step::VB / 16;
  // V pieces in the LDS tile: row and first 8-element chunk
  constexpr int LPV = F::CB / Step::VB;  // lanes of a row
  constexpr int CPP = Step::VB / 4;      // chunks of a piece
  const int vprow = lane / LPV, vpc = (lane % LPV) * CPP;
  int vwa[Step::VL][CPP];
#pragma unroll
  for (int i = 0; i < Step::VL; ++i)
#pragma unroll
    for (int c = 0; c < CPP; ++c) {
      const int row = i * (64 / LPV) + vprow;
      vwa[i][c] = row * L::RB + (((vpc + c) ^ L::vswz(row)) << 4);
    }
  const int jj = lane & 15;
  const int vrow = 4 * grp + (jj >> 2);
  const int voff = vrow * L::RB + ((L::vswz(vrow) >> 1) << 5) + (jj & 3) * 8;
  const int pbytes = p.page * F::RB, vbase = F::v_codes(p.page), ksbase = F::k_scales(p.page), vsbase = F::v_scales(p.page);
  // floor(n / pu): the product with floor(2^32 / pu) falls at most one short
  auto page_of = [&](uint32_t n) {
    uint32_t g = __umulhi(n, pp.magic);
    if (n - g * pp.pu >= pp.pu) ++g;
    return (int)g;
  };

  while (true) {
    // (said to be wave-uniform, which the buffer loads' scalar operands have to be)
    constexpr int COST = ROWS ? 0 : KV4_ROW_COST;
    const int span = uniform((int)min((int64_t)(at.nb - at.ls), at.q1 - at.q));
    const int b = uniform(at.b), nb = uniform(at.nb) - COST, j = uniform(at.j), start = uniform(at.ls) - COST;
    const int ls = max(start, 0), nseg = max(start + span, 0) - ls;
    if (nseg == 0) {  // a part of the row's start, which holds no keys
      if (!at.next(p, span)) break;
      continue;
    }
    const int len = at.len_of(p, b);
    const int kvh = j / p.NG, hg = j % p.NG;
    const bool whole = ls == 0 && nseg == nb;
    const int kend = min(len, (ls + nseg) * DC_STEP);
    const int mine = nseg > wave ? (nseg - wave + W - 1) / W : 0;  // steps ls + wave + W i

    // the pages of this wave's steps [wbase, wbase + 64), one per lane
    int wbase = 0, win = 0;
    bool lost = false;  // a page that is not in the pool: the row is NaN
    auto load_window = [&](int first) {
      wbase = first;
      win = first + lane < mine ? p.bt[b * p.bts + page_of(ls + wave + (first + lane) * W)] : 0;
      const bool bad = (uint32_t)win >= (uint32_t)pp.npages;
      lost |= wave_any(bad);
      if (bad) win = 0;
    };
    const unsigned char* heads = reinterpret_cast<const unsigned char*>(p.kc) + kvh * p.ksh;
    // Past the wave's last step the loads go out all the same, over no bytes: behind a
    // branch the compiler could not tell how many are in flight, and would wait for all
    // of them at every step.
    auto load = [&](Step& st, int i) {
      if (i - wbase >= 64) load_window(i);
      const int pid = __builtin_amdgcn_readlane(win, i - wbase);
      const uint32_t n = ls + wave + i * W;
      const int rel = (int)(n - uniform(page_of(n)) * pp.pu) * DC_STEP;
      const BufRsrc rs = make_rsrc(heads + pid * p.ksb, i < mine ? (uint32_t)pbytes : 0u);
      const int kc = rel * F::CB, ks = ksbase + rel * F::SB;
      const int vc = vbase + rel * F::CB, vs = vsbase + rel * F::SB;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        kv4_load(st.k[t], rs, kvo, kc + t * 16 * F::CB);
        st.ks[t] = __builtin_amdgcn_raw_buffer_load_b8(rs, kso, ks + t * 16 * F::SB, 2);
      }
#pragma unroll
      for (int l = 0; l < Step::VL; ++l) {
        kv4_load(st.v[l], rs, vvo, vc + l * 64 * Step::VB);
        st.vs[l] = __builtin_amdgcn_raw_buffer_load_b8(rs, vso, vs + l * 4 * Step::VB, 2);
      }
    };

    float m_i = -INFINITY, l_i = 0.f;
    floatx4 oacc[NDO];
#pragma unroll
    for (int dd = 0; dd < NDO; ++dd) oacc[dd] = floatx4{};
    const int gh = hg * 16 + c16;
    const bool hvalid = gh < p.G;

    if (mine > 0) {
      load_window(0);
      // ---- the query: lane (head c16, slot grp) holds elements grp D/4 + 8 i + j
      const T* qrow =
          reinterpret_cast<const T*>(p.q) + b * p.qsb + (kvh * p.G + (hvalid ? gh : 0)) * p.qsh + grp * (D / 4);
      floatx8 x[NDQ];
#pragma unroll
      for (int i = 0; i < NDQ; ++i) x[i] = Vec8<T>::load_f32(qrow + i * 8);
      Step st[KV4_DEPTH];
#pragma unroll
      for (int u = 0; u < KV4_DEPTH; ++u) load(st[u], u);
      bf16x8 qop[NDQ][NT];
#pragma unroll
      for (int i = 0; i < NDQ; ++i) split_bf16<NT>(hvalid ? x[i] : floatx8{}, qop[i]);

      auto step = [&](Step& st, int i) {
        const int k0 = (ls + wave + i * W) * DC_STEP;
        if (k0 + DC_STEP > kend) {  // value rows past the last key as zeros, whatever they hold
#pragma unroll
          for (int l = 0; l < Step::VL; ++l)
            if (k0 + l * (64 / LPV) + vprow >= kend) {
              st.vs[l] = 127;
#pragma unroll
              for (int c = 0; c < CPP; ++c) st.v[l][c] = 0;
            }
        }
        floatx4 sc[2] = {floatx4{}, floatx4{}};
#pragma unroll
        for (int d = 0; d < NDQ; ++d)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const bf16x8 a = kv4_bf16x8(st.k[t][d], kv4_scale(st.ks[t]));
#pragma unroll
            for (int n = NT - 1; n >= 0; --n) sc[t] = mfma16(a, qop[d][n], sc[t]);
          }
        // V to the LDS tile (in-order within the wave: the previous step's reads of the
        // tile have been served), and back transposed; the reads are issued together,
        // and the softmax runs while they are served
#pragma unroll
        for (int l = 0; l < Step::VL; ++l) {
          const float scale = kv4_scale(st.vs[l]);
#pragma unroll
          for (int c = 0; c < CPP; ++c)
            *reinterpret_cast<bf16x8*>(vt + vwa[l][c]) = kv4_bf16x8(st.v[l][c], scale);
        }
        load(st, i + KV4_DEPTH);
        bf16x8 vop[NDO];
#pragma unroll
        for (int dd = 0; dd < NDO; ++dd) {
          const unsigned char* src = vt + (voff ^ (dd << 5));
          vop[dd] = lds_read_tr8(reinterpret_cast<const bf16*>(src), reinterpret_cast<const bf16*>(src + 16 * L::RB));
        }
        __builtin_amdgcn_sched_barrier(0);
        if (k0 + DC_STEP > kend) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (k0 + t * 16 + grp * 4 + e >= kend) sc[t][e] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[t][e]);
        mx *= p.scale_log2;
        if (wave_any(mx > m_i + KV4_SLACK)) {
          const float m_new = fmaxf(m_i, xor32_max(xor16_max(mx)));
          const float alpha = m_new > -INFINITY ? fast_exp2(m_i - m_new) : 1.f;
          l_i *= alpha;
#pragma unroll
          for (int dd = 0; dd < NDO; ++dd) oacc[dd] *= alpha;
          m_i = m_new;
        }
        // without a finite score so far the row keeps m = -inf and exponentiates against 0
        const float m_use = m_i > -INFINITY ? m_i : 0.f;
        floatx8 pf;
        float rs = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float pe = fast_exp2(__builtin_fmaf(sc[t][e], p.scale_log2, -m_use));
            pf[t * 4 + e] = pe;
            rs += pe;
          }
        bf16x8 pop[NT];
        split_bf16<NT>(pf, pop);
        l_i += rs;
#pragma unroll
        for (int dd = 0; dd < NDO; ++dd)
#pragma unroll
          for (int n = NT - 1; n >= 0; --n) oacc[dd] = mfma16(vop[dd], pop[n], oacc[dd]);
      };
      int i = 0;
      for (; i + KV4_DEPTH <= mine; i += KV4_DEPTH)
#pragma unroll
        for (int u = 0; u < KV4_DEPTH; ++u) step(st[u], i + u);
#pragma unroll
      for (int u = 0; u < KV4_DEPTH - 1; ++u)
        if (i + u < mine) step(st[u], i + u);
    }

    // ---- the waves' parts meet in LDS: maxima and sums first, then each wave's outputs,
    // brought to the common maximum, in its own V tile
    l_i = xor32_sum(xor16_sum(l_i));
    if (lost) l_i = __builtin_nanf("");
    if (grp == 0) part_ml[wave][c16] = floatx2{m_i, l_i};
    __syncthreads();
    const int used = min(nseg, W);  // waves that took steps
    float M = -INFINITY;
    for (int i = 0; i < used; ++i) M = fmaxf(M, part_ml[i][c16][0]);
    const float f = M > -INFINITY ? fast_exp2(m_i - M) : 1.f;
    if (wave < used) {
#pragma unroll
      for (int dd = 0; dd < NDO; ++dd)
        *reinterpret_cast<floatx4*>(vt + c16 * (D * 4) + (((dd * 4 + grp) ^ (c16 & (D / 4 - 1))) << 4)) = oacc[dd] * f;
    }
    __syncthreads();
    const int64_t r = ((int64_t)b * p.Hkv + kvh) * p.NG + hg;
    const int64_t slot = blockIdx.x + r;
    if (!ROWS && threadIdx.x == 0) {
      if (ls == 0) p.ws_rw[r * 2] = (int32_t)blockIdx.x;
      if (ls + nseg == nb) p.ws_rw[r * 2 + 1] = (int32_t)blockIdx.x;
    }
    for (int t = threadIdx.x; t < 16 * (D / 4); t += (W * 64)) {
      const int h = t / (D / 4), c = t % (D / 4);
      if (hg * 16 + h >= p.G) continue;
      float top = -INFINITY, sum = 0.f;
      for (int i = 0; i < used; ++i) top = fmaxf(top, part_ml[i][h][0]);
      floatx4 acc = floatx4{};
      for (int i = 0; i < used; ++i) {
        const floatx2 ml = part_ml[i][h];
        sum = __builtin_fmaf(ml[1], top > -INFINITY ? fast_exp2(ml[0] - top) : 1.f, sum);
        acc += *reinterpret_cast<const floatx4*>(smem + i * L::BYTES + h * (D * 4) + ((c ^ (h & (D / 4 - 1))) << 4));
      }
      if (ROWS || whole) {
        const int head = kvh * p.G + hg * 16 + h;
        store4<T>(reinterpret_cast<T*>(p.o) + b * p.osb + (int64_t)head * p.osh + c * 4, acc * (1.0f / sum));
        if (p.lse && c == 0) p.lse[(int64_t)b * p.Hq + head] = row_lse(top, sum);
      } else {
        *reinterpret_cast<floatx4*>(p.ws_o + (slot * 16 + h) * D + c * 4) = acc;
        if (c == 0) *reinterpret_cast<floatx2*>(p.ws_ml + (slot * 16 + h) * 2) = floatx2{top, sum};
      }
    }
    if (ROWS || !at.next(p, span)) break;
    __syncthreads();  // the tiles and sums are read; the next segment may write them
  }
}

// Whether each row goes to a workgroup of its own.  Its eight waves take about KV4_STEP_US
// for a step each; the shared form takes KV4_SHARE_US more, for the schedule, the
// partials' way to memory and the merge's launch.  Rows of one launch differ in length, and
// the host knows no more than the longest: the shared work is taken as half of it.
constexpr float KV4_STEP_US = 0.9f, KV4_SHARE_US = 7.f;
static bool kv4_whole_rows(int64_t rows, int max_len, int cus) {
  const int64_t turns = ((int64_t)max_len + DC_STEP * KV4_ROW_WAVES - 1) / (DC_STEP * KV4_ROW_WAVES);
  const float own = (float)((rows + cus - 1) / cus) * turns * KV4_STEP_US;
  const float shared = 0.5f * (float)rows * turns / cus * KV4_STEP_US + KV4_SHARE_US;
  return own <= shared;
}

// CUs of the current device (256 where there is none).
static int kv4_cus() {
  static int known[64];
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  cus = __atomic_load_n(&known[dev], __ATOMIC_RELAXED);
  if (cus == 0) {
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) return 256;
    __atomic_store_n(&known[dev], cus, __ATOMIC_RELAXED);
  }
  return cus;
}

// Partial slots and the rows' covering workgroups; whole rows need none.
static int64_t kv4_workspace(int B, int Hq, int Hkv, int D, int max_len) {
  const int64_t rows = (int64_t)B * Hkv * ((Hq / Hkv + 15) / 16);
  if (kv4_whole_rows(rows, max_len, kv4_cus())) return 0;
  return (KV4_MAX_GROUPS + rows) * 16 * (D + 2) * (int64_t)sizeof(float) + rows * 2 * (int64_t)sizeof(int32_t);
}

template <int D, typename T>
static hipError_t launch_decode_kv4(Kv4DecodeParams pp, hipStream_t st) {
  DecodeParams& p = pp.d;
  const int cus = kv4_cus();
  const int64_t rows = (int64_t)p.B * p.rows_per_batch;
  if (kv4_whole_rows(rows, p.max_len, cus)) {
    hipLaunchKernelGGL((decode_kv4_kernel<D, T, true>), dim3((unsigned)rows), dim3(KV4_ROW_WAVES * 64), 0, st, pp);
    return hipGetLastError();
  }
  const int groups = cus * KV4_PER_CU < KV4_MAX_GROUPS ? cus * KV4_PER_CU : KV4_MAX_GROUPS;
  p.nwaves = groups;
  hipLaunchKernelGGL((decode_kv4_kernel<D, T, false>), dim3((unsigned)groups), dim3(KV4_WAVES * 64), 0, st, pp);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int threads = rows * DC_MERGE_WIDE_PARTIALS <= groups ? DC_MERGE_MAX_THREADS : DC_THREADS;
  hipLaunchKernelGGL((decode_merge_kernel<D, T>), dim3((unsigned)rows), dim3(threads),
                     (threads / 16) * (D + 2) * sizeof(float), st, p);
  return hipGetLastError();
}

// ---------------------------------------------------------------- host checks
// What every entry over 4-bit pages checks of them.
static int kv4_check_pages(const void* pool, const int64_t* pool_strides, int num_pages, const int32_t* block_table,
                           int64_t bt_stride, int bt_cols, int page_size, int Hkv, int D) {
  if (!head_dim_ok(D)) return nq_fail(NQ_ERR_UNSUPPORTED, "head_dim must be 32, 64 or 128, got %d", D);
  if (!pool || !pool_strides || !block_table) return nq_fail(NQ_ERR_INVALID, "a pool, its strides and a block table are required");
  if (page_size <= 0 || page_size % DC_STEP || page_size > (1 << 20))
    return nq_fail(NQ_ERR_UNSUPPORTED, "page_size must be a multiple of %d up to 2^20, got %d", DC_STEP, page_size);
  if (num_pages <= 0 || bt_cols <= 0 || bt_stride < bt_cols)
    return nq_fail(NQ_ERR_INVALID, "num_pages and bt_cols must be positive and rows of the table at least bt_cols apart");
  const int64_t rec = (int64_t)page_size * 17 * D / 16;
  if (!nq_aligned16(pool) || pool_strides[0] % 16 || pool_strides[1] % 16)
    return nq_fail(NQ_ERR_INVALID, "the pool and its strides must be multiples of 16 bytes");
  if (pool_strides[1] < rec && Hkv > 1) return nq_fail(NQ_ERR_INVALID, "the pool's heads must not overlap");
  return NQ_OK;
}

static int kv4_check_strides(const char* name, const void* t, const int64_t* st, int esz) {
  if (!st) return nq_fail(NQ_ERR_INVALID, "%s needs its strides", name);
  if (!nq_aligned16(t)) return nq_fail(NQ_ERR_INVALID, "%s must be 16-byte aligned", name);
  for (int i = 0; i < 3; ++i)
    if ((st[i] * esz) % 16) return nq_fail(NQ_ERR_INVALID, "%s strides must be multiples of 16 bytes", name);
  return NQ_OK;
}

}  // namespace nq

using namespace nq;

extern "C" int nq_kv4_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                             const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides,
                             void* pool, const int64_t* pool_strides, int num_pages, const int32_t* block_table,
                             int64_t bt_stride, int bt_cols, int page_size, int B, int S, int Hq, int Hkv, int D,
                             int dtype, const void* q_weight, const void* k_weight, float eps, const float* cos_tab,
                             const float* sin_tab, int max_pos, const int32_t* pos, const int32_t* pos_base,
                             const int32_t* pos_shift, int pos0, const int32_t* row_base, int row0,
                             int32_t* lens_out, void* stream) {
  nq_clear_error();
  Kv4AppendParams p{};
  const int dt = nq_take_weight_flags(dtype, &p.q16, &p.k16);
  if (!nq_dtype_ok(dt) || ((p.q16 || p.k16) && dt != NQ_DTYPE_BF16))
    return nq_fail(NQ_ERR_UNSUPPORTED, "unknown dtype code %d", dtype);
  if (B <= 0 || S <= 0 || Hkv <= 0 || Hq < 0)
    return nq_fail(NQ_ERR_INVALID, "sizes must be positive (B=%d S=%d Hkv=%d Hq=%d)", B, S, Hkv, Hq);
  int rc = kv4_check_pages(pool, pool_strides, num_pages, block_table, bt_stride, bt_cols, page_size, Hkv, D);
  if (rc != NQ_OK) return rc;
  if (!k || !v) return nq_fail(NQ_ERR_INVALID, "k and v are required");
  if ((Hq > 0) != (q != nullptr) || (q != nullptr) != (q_out != nullptr))
    return nq_fail(NQ_ERR_INVALID, "q, q_out and Hq > 0 go together");
  const int esz = nq_dtype_size(dt);
  if ((rc = kv4_check_strides("k", k, k_strides, esz)) || (rc = kv4_check_strides("v", v, v_strides, esz))) return rc;
  if (q && ((rc = kv4_check_strides("q", q, q_strides, esz)) || (rc = kv4_check_strides("q_out", q_out, q_out_strides, esz))))
    return rc;
  if ((cos_tab == nullptr) != (sin_tab == nullptr) || (cos_tab && max_pos <= 0))
    return nq_fail(NQ_ERR_INVALID, "cos and sin tables go together, with max_pos > 0");
  if (!nq_aligned16(q_weight) || !nq_aligned16(k_weight) || !nq_aligned16(cos_tab) || !nq_aligned16(sin_tab))
    return nq_fail(NQ_ERR_INVALID, "norm weights and tables must be 16-byte aligned");
  const uintptr_t out = reinterpret_cast<uintptr_t>(lens_out), lens_bytes = (uintptr_t)B * sizeof(int32_t);
  for (const int32_t* in : {row_base, pos_base, pos_shift})  // each read by all of a sequence's rows
    if (lens_out && in && reinterpret_cast<uintptr_t>(in) < out + lens_bytes && out < reinterpret_cast<uintptr_t>(in) + lens_bytes)
      return nq_fail(NQ_ERR_INVALID, "lens_out must not alias row_base, pos_base or pos_shift");
  const int64_t rows = (int64_t)B * S * ((int64_t)Hq + 2 * (int64_t)Hkv);
  if (rows * (D / 16) > KV4_MOST_LANES) return nq_fail(NQ_ERR_UNSUPPORTED, "too many rows for one call");
  p.k = k; p.ksb = k_strides[0]; p.ksh = k_strides[1]; p.kss = k_strides[2];
  p.v = v; p.vsb = v_strides[0]; p.vsh = v_strides[1]; p.vss = v_strides[2];
  if (q) {
    p.q = q; p.qsb = q_strides[0]; p.qsh = q_strides[1]; p.qss = q_strides[2];
    p.q_out = q_out; p.osb = q_out_strides[0]; p.osh = q_out_strides[1]; p.oss = q_out_strides[2];
  }
  p.pool = reinterpret_cast<unsigned char*>(pool); p.psb = pool_strides[0]; p.psh = pool_strides[1];
  p.npages = num_pages; p.bt = block_table; p.bts = bt_stride; p.page = page_size;
  p.cap = (int64_t)bt_cols * page_size;
  if (p.cap > 0x7fffffff) p.cap = 0x7fffffff;
  p.by_S = Divider(S); p.by_HT = Divider(Hq + 2 * Hkv); p.by_page = Divider(page_size);
  p.B = B; p.S = S; p.Hq = Hq; p.Hkv = Hkv; p.qw = q_weight; p.kw = k_weight; p.eps = eps;
  p.cos_tab = cos_tab; p.sin_tab = sin_tab; p.max_pos = max_pos;
  p.pos = pos; p.pos_base = pos_base; p.pos_shift = pos_shift; p.pos0 = pos0;
  p.row_base = row_base; p.row0 = row0; p.lens_out = lens_out;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return nq_check_launch(with_head_dim(D, [&](auto dc) {
    constexpr int DD = decltype(dc)::value;
    const int64_t blocks = (rows * (DD / 16) + 255) / 256;
    if (dt == NQ_DTYPE_BF16)
      hipLaunchKernelGGL((kv4_append_kernel<DD, bf16>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL((kv4_append_kernel<DD, float>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    return hipGetLastError();
  }));
}

extern "C" int nq_kv4_gather(const void* pool, const int64_t* pool_strides, int num_pages, const int32_t* block_table,
                             int64_t bt_stride, int bt_cols, int page_size, void* k, const int64_t* k_strides,
                             void* v, const int64_t* v_strides, int B, int S, int Hkv, int D, int dtype,
                             const int32_t* row_base, int row0, void* stream) {
  nq_clear_error();
  if (!nq_dtype_ok(dtype)) return nq_fail(NQ_ERR_UNSUPPORTED, "unknown dtype code %d", dtype);
  if (B <= 0 || S <= 0 || Hkv <= 0)
    return nq_fail(NQ_ERR_INVALID, "sizes must be positive (B=%d S=%d Hkv=%d)", B, S, Hkv);
  int rc = kv4_check_pages(pool, pool_strides, num_pages, block_table, bt_stride, bt_cols, page_size, Hkv, D);
  if (rc != NQ_OK) return rc;
  if (!k || !v) return nq_fail(NQ_ERR_INVALID, "k and v are required");
  const int esz = nq_dtype_size(dtype);
  if ((rc = kv4_check_strides("k", k, k_strides, esz)) || (rc = kv4_check_strides("v", v, v_strides, esz))) return rc;
  const int64_t rows = (int64_t)B * S * Hkv;
  if (rows * (D / 16) > KV4_MOST_LANES) return nq_fail(NQ_ERR_UNSUPPORTED, "too many rows for one call");
  Kv4GatherParams p{};
  p.pool = reinterpret_cast<const unsigned char*>(pool); p.psb = pool_strides[0]; p.psh = pool_strides[1];
  p.npages = num_pages; p.bt = block_table; p.bts = bt_stride; p.page = page_size;
  p.cap = (int64_t)bt_cols * page_size;
  if (p.cap > 0x7fffffff) p.cap = 0x7fffffff;
  p.k = k; p.ksb = k_strides[0]; p.ksh = k_strides[1]; p.kss = k_strides[2];
  p.v = v; p.vsb = v_strides[0]; p.vsh = v_strides[1]; p.vss = v_strides[2];
  p.by_S = Divider(S); p.by_H = Divider(Hkv); p.by_page = Divider(page_size);
  p.B = B; p.S = S; p.Hkv = Hkv; p.row_base = row_base; p.row0 = row0;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return nq_check_launch(with_head_dim(D, [&](auto dc) {
    constexpr int DD = decltype(dc)::value;
    const dim3 grid((unsigned)((rows * (DD / 16) + 255) / 256), 2);
    if (dtype == NQ_DTYPE_BF16)
      hipLaunchKernelGGL((kv4_gather_kernel<DD, bf16>), grid, dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL((kv4_gather_kernel<DD, float>), grid, dim3(256), 0, st, p);
    return hipGetLastError();
  }));
}

extern "C" int64_t nq_attn_decode_kv4_workspace_bytes(int B, int Hq, int Hkv, int D, int max_len) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || max_len <= 0 || Hq % Hkv) return 0;
  return kv4_workspace(B, Hq, Hkv, D, max_len);
}

extern "C" int nq_attn_decode_kv4(const void* q, const int64_t* q_strides, const void* pool,
                                  const int64_t* pool_strides, int num_pages, const int32_t* block_table,
                                  int64_t bt_stride, int bt_cols, int page_size, const int32_t* lens, void* o,
                                  const int64_t* o_strides, float* lse, void* workspace, int64_t workspace_bytes,
                                  int B, int Hq, int Hkv, int D, int max_len, int dtype, float sm_scale,
                                  void* stream) {
  nq_clear_error();
  if (!nq_dtype_ok(dtype)) return nq_fail(NQ_ERR_UNSUPPORTED, "unknown dtype code %d", dtype);
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || max_len <= 0)
    return nq_fail(NQ_ERR_INVALID, "sizes must be positive (B=%d Hq=%d Hkv=%d max_len=%d)", B, Hq, Hkv, max_len);
  if (Hq % Hkv) return nq_fail(NQ_ERR_INVALID, "num_heads %d not divisible by num_kv_heads %d", Hq, Hkv);
  int rc = kv4_check_pages(pool, pool_strides, num_pages, block_table, bt_stride, bt_cols, page_size, Hkv, D);
  if (rc != NQ_OK) return rc;
  if (!q || !o || !q_strides || !o_strides || !lens)
    return nq_fail(NQ_ERR_INVALID, "q, o, their strides and lens are required");
  if (!nq_aligned16(q) || !nq_aligned16(o)) return nq_fail(NQ_ERR_INVALID, "q and o must be 16-byte aligned");
  const int esz = nq_dtype_size(dtype);
  for (int i = 0; i < 2; ++i)
    if ((q_strides[i] * esz) % 16 || (o_strides[i] * esz) % 16)
      return nq_fail(NQ_ERR_INVALID, "q and o strides must be multiples of 16 bytes");
  if ((max_len + page_size - 1) / page_size > bt_cols)
    return nq_fail(NQ_ERR_INVALID, "the block table's %d columns hold fewer than max_len %d rows", bt_cols, max_len);
  if (max_len > (1 << 30))  // keys, rounded up to whole steps, are ints
    return nq_fail(NQ_ERR_UNSUPPORTED, "at most 2^30 keys, got max_len %d", max_len);
  const int NG = (Hq / Hkv + 15) / 16;
  if ((int64_t)B * Hkv * NG * DC_MERGE_MAX_THREADS > 0xffffffffll)  // a launch has fewer than 2^32 threads
    return nq_fail(NQ_ERR_UNSUPPORTED, "more (sequence, kv head) rows than one launch takes");
  const int64_t need = kv4_workspace(B, Hq, Hkv, D, max_len);
  if (need && (!workspace || workspace_bytes < need || !nq_aligned16(workspace)))
    return nq_fail(NQ_ERR_WORKSPACE, "an aligned workspace of %lld bytes is required, %lld given", (long long)need,
                   (long long)workspace_bytes);
  Kv4DecodeParams pp{};
  DecodeParams& p = pp.d;
  p.q = q; p.qsb = q_strides[0]; p.qsh = q_strides[1];
  p.kc = const_cast<void*>(pool); p.ksb = pool_strides[0]; p.ksh = pool_strides[1];
  p.lens = lens; p.o = o; p.osb = o_strides[0]; p.osh = o_strides[1]; p.lse = lse;
  p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.NG = NG; p.max_len = max_len;
  p.rows_per_batch = Hkv * NG;
  while ((1 << p.hs) < (p.G < 16 ? p.G : 16)) ++p.hs;
  const int64_t slots = KV4_MAX_GROUPS + (int64_t)B * p.rows_per_batch;
  p.ws_o = reinterpret_cast<float*>(workspace);
  p.ws_ml = p.ws_o + slots * 16 * D;
  p.ws_rw = reinterpret_cast<int32_t*>(p.ws_ml + slots * 16 * 2);
  p.scale_log2 = (sm_scale > 0.f ? sm_scale : 1.0f / sqrtf((float)D)) * kLog2e;
  p.bt = block_table; p.bts = bt_stride; p.page = page_size;
  pp.npages = num_pages;
  pp.pu = (uint32_t)(page_size / DC_STEP);
  pp.magic = pp.pu == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / pp.pu);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return nq_check_launch(with_head_dim(D, [&](auto dc) {
    return dtype == NQ_DTYPE_BF16 ? launch_decode_kv4<decltype(dc)::value, bf16>(pp, st)
                                  : launch_decode_kv4<decltype(dc)::value, float>(pp, st);
  }));
}
