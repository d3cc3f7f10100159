// Log-probabilities of labels straight from a model's last hidden states and its LM head,
// and their gradients: z = h w^T / T without the (tokens x vocabulary) logits in memory.
//
//   forward    z tile by tile; each tile leaves its rows' maximum and sum of exponentials
//              (and the label's logit), which a second launch joins:
//              logprob = (z[label] - m) / T - log l
//   backward   dz = dy (1[v = label] - softmax) / T, formed again from the statistics a
//              range of the vocabulary at a time, in bf16; dh += dz w and dw = dz^T h
//
// Four products of 2 tokens vocabulary width operations each, all on one core: bf16 MFMA
// with fp32 accumulation over tiles of 256 x 256 (or 64 tokens, where there are few).  dz
// is rounded to bf16 once, as the matrix cores need it: half a step, 2^-8 of a value at
// most, independent from term to term.  Ignored rows are left out first: the kept rows are
// gathered to the front, and the products run over those.

#include <math.h>

#include "nq_common.hpp"
#include "nq_internal.hpp"
#include "nq_loss.hpp"

namespace nq {

constexpr int HD_BM = 256;  // a tile's extent on the MFMA's row axis
constexpr int HD_BK = 64;   // depth of a step
constexpr int HD_WAVES = 8;
constexpr int HD_PREP = 64;  // rows of a gathering workgroup

// ---------------------------------------------------------------------------
// The kept rows, in order: pos[row] = its place among them (-1: ignored), index the
// reverse, hc their hidden states.  A workgroup counts the kept rows before its own 64 (the
// labels are small and in L2) rather than wait for another launch.
struct HeadRows {
  const bf16* hidden;
  int64_t bs, rs, S;
  const int64_t* labels;
  int64_t rows, ignore;
  int H, V;
  int* count;
  int* pos;       // (rows)
  int* index;     // (rows)
  int* target;    // (rows) the kept rows' labels, -1 outside the vocabulary
  bf16* hc;       // (rows, H)
  // forward
  float* logprobs;
  floatx2* stats;
  float* zlabel;  // (rows) by place
  // backward
  const float* dy;
  floatx4* coef;  // (rows) by place: m, -g / l, g = dy / T
  float inv_t;
};

__global__ __launch_bounds__(256) void head_rows_kernel(HeadRows p) {
  __shared__ int before[4], own[HD_PREP];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r0 = (int64_t)blockIdx.x * HD_PREP;
  int n = 0;
  for (int64_t r = tid; r < r0; r += 256) n += p.labels[r] != p.ignore;
#pragma unroll
  for (int k = 32; k >= 1; k >>= 1) n += __shfl_xor(n, k, 64);
  if (lane == 0) before[wave] = n;
  __syncthreads();
  const int base = before[0] + before[1] + before[2] + before[3];
  if (wave == 0) {
    const int64_t r = r0 + lane;
    const int64_t y = r < p.rows ? p.labels[r] : p.ignore;
    const bool kept = y != p.ignore;
    const uint64_t ballot = __builtin_amdgcn_ballot_w64(kept);
    const int place = kept ? base + __popcll(ballot & ((1ull << lane) - 1)) : -1;
    own[lane] = place;
    if (r < p.rows) {
      p.pos[r] = place;
      const bool inside = y >= 0 && y < p.V;
      if (kept) {
        p.index[place] = (int)r;
        p.target[place] = inside ? (int)y : -1;
        if (p.zlabel) p.zlabel[place] = __builtin_nanf("");  // stays for a label outside the vocabulary
        if (p.dy) {
          const floatx2 st = p.stats[r];
          const float g = inside ? p.dy[r] * p.inv_t : __builtin_nanf("");
          p.coef[place] = floatx4{st[0], -g / st[1], g, 0.f};
        }
      } else if (p.logprobs) {
        p.logprobs[r] = 0.f;
        p.stats[r] = floatx2{0.f, 1.f};
      }
    }
    if (r0 + HD_PREP >= p.rows && lane == 0) *p.count = base + __popcll(ballot);
  }
  __syncthreads();
  const int ch = p.H / 8;
  for (int i = wave; i < HD_PREP && r0 + i < p.rows; i += 4) {
    const int place = own[i];
    if (place < 0) continue;
    const int64_t r = r0 + i, b = r / p.S;
    const bf16x8* src = reinterpret_cast<const bf16x8*>(p.hidden + b * p.bs + (r - b * p.S) * p.rs);
    bf16x8* dst = reinterpret_cast<bf16x8*>(p.hc + (int64_t)place * p.H);
    for (int c = lane; c < ch; c += 64) dst[c] = src[c];
  }
}

// ---------------------------------------------------------------------------
// One operand of a product, (extent x depth), staged in LDS a step of 64 deep at a time.
//   ROW   depth contiguous in memory: LDS rows of 128 bytes, an operand one 16-byte read.
//         16-byte chunk c of row r lies at c ^ (r / 2 % 8): 16 consecutive rows' reads
//         hit distinct banks.
//   !ROW  extent contiguous: LDS rows (one depth each) of 2 EXT bytes, transpose reads.
//         Chunk c of depth k lies at c ^ 4 (k % 4): the 4 depths of a read hit distinct
//         banks.
// HBM -> LDS without registers; what lies outside (rows past the extent, depths past the
// end) is out of the descriptor's range and arrives as zeros.
template <int EXT, bool ROW>
struct Stage {
  static constexpr int BYTES = EXT * HD_BK * 2;
  static constexpr int NI = BYTES / 1024 / HD_WAVES;  // loads of a wave per step
  static constexpr int LINE = ROW ? 128 : EXT * 2;    // bytes of an LDS row
  static constexpr int ROWS_PER = 1024 / LINE;
  const char* base;   // ROW: first row, else first depth
  uint32_t line;      // bytes of a row in memory
  uint32_t range;     // ROW: bytes from base to the end of the last row
  int64_t extent;     // !ROW: columns from base that exist (bytes), so that none past a line's end is read
  int depth;          // how many depths exist
  uint32_t off, chunk;

  // rows [e0, e0 + EXT) of `extent` rows of `ld` elements; depths [0, depth)
  __device__ __forceinline__ void init(const bf16* p, int64_t ld, int64_t e0, int64_t n, int depth_, int wave,
                                       int lane) {
    line = (uint32_t)(ld * 2);
    depth = depth_;
    const int r = wave * ROWS_PER + lane / (LINE / 16), pc = lane % (LINE / 16);
    if (ROW) {
      const int64_t left = n - e0;
      base = reinterpret_cast<const char*>(p + e0 * ld);
      range = left <= 0 ? 0 : (uint32_t)((left < EXT ? left : EXT) * (int64_t)line);
      chunk = (uint32_t)((pc ^ ((r >> 1) & 7)) * 8);  // first depth of the chunk
      off = (uint32_t)r * line + chunk * 2;
    } else {
      base = reinterpret_cast<const char*>(p + e0);
      extent = (n - e0) * 2;
      chunk = (uint32_t)((pc ^ ((r & 3) << 2)) * 16);  // byte of the chunk in its line
      off = (uint32_t)r * line + chunk;
    }
  }
  // the step at depth k0 into LDS at `tile`
  __device__ __forceinline__ void load(unsigned char* tile, int k0, int wave) const {
    constexpr uint32_t NONE = 0x80000000u;  // out of any range
    if (ROW) {
      const BufRsrc r = make_rsrc(base, range);
      const uint32_t o = k0 + (int)chunk < depth ? off + (uint32_t)k0 * 2 : NONE;
#pragma unroll
      for (int i = 0; i < NI; ++i)
        buffer_load_lds16(r, tile + (wave + HD_WAVES * i) * 1024, o + (o == NONE ? 0u : i * (HD_WAVES * ROWS_PER) * line), 0u);
    } else {
      const int left = depth - k0;
      const BufRsrc r = make_rsrc(base + (int64_t)k0 * line, (uint32_t)(left < HD_BK ? left : HD_BK) * line);
      const uint32_t o = (int64_t)chunk < extent ? off : NONE;
#pragma unroll
      for (int i = 0; i < NI; ++i)
        buffer_load_lds16(r, tile + (wave + HD_WAVES * i) * 1024, o + (o == NONE ? 0u : i * (HD_WAVES * ROWS_PER) * line), 0u);
    }
  }
};

// LDS addresses of a wave's operand (32-wide blocks t < NT from `e0`): one for each
// 16-depth kk (ROW) or each block (!ROW), the other index an immediate.
template <int EXT, bool ROW, int NT>
struct Reads {
  static constexpr int N = ROW ? 4 : NT;
  static constexpr int PER = ROW ? NT : 2 * NT;  // LDS reads of one depth of 16
  uint32_t a[N];
  __device__ __forceinline__ void init(uint32_t tile, int e0, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (ROW) {
        const int r = e0 + (lane & 31);
        a[i] = tile + r * 128 + ((((lane >> 5) + 2 * i) ^ ((r >> 1) & 7)) << 4);
      } else {
        const int g = lane >> 4, j = lane & 15;
        const int k = (g >> 1) * 8 + (j >> 2), col = (e0 + i * 32) * 2 + (g & 1) * 32 + (j & 3) * 8;
        a[i] = tile + k * (EXT * 2) + (col ^ ((j >> 2) << 6));
      }
    }
  }
  template <int KK>
  __device__ __forceinline__ void read(uint32_t buf, bf16x8 (&v)[NT]) const {
    if constexpr (ROW) {
      one<0, KK>(buf, v);
    } else {
      one<0, KK>(buf, v);
    }
  }
  template <int T, int KK>
  __device__ __forceinline__ void one(uint32_t buf, bf16x8 (&v)[NT]) const {
    if constexpr (T < NT) {
      if constexpr (ROW) {
        v[T] = lds_read_b128_nowait<T * 32 * 128>(a[KK] + buf);
      } else {
        typedef short shortx8 __attribute__((ext_vector_type(8)));
        constexpr int LINE = EXT * 2;
        const shortx4 lo = lds_read_tr4_nowait<KK * 16 * LINE>(a[T] + buf);
        const shortx4 hi = lds_read_tr4_nowait<KK * 16 * LINE + 4 * LINE>(a[T] + buf);
        const shortx8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        v[T] = __builtin_bit_cast(bf16x8, both);
      }
      one<T + 1, KK>(buf, v);
    }
  }
};

// How the eight waves share a tile of 256 x BN: each MT x NT blocks of 32 x 32.
template <int BN> struct Waves;
template <> struct Waves<256> { static constexpr int M = 2, N = 4, MT = 4, NT = 2; };
template <> struct Waves<64> { static constexpr int M = 8, N = 1, MT = 1, NT = 2; };

// acc[mt][nt] += the wave's blocks of A B^T over `depth`.  Two LDS buffers: the next step's
// loads are in flight while this step's 64 depths are multiplied, one barrier a step; the
// operands of the next 16 depths are read while these are multiplied.
template <int BN, bool AROW, bool BROW>
__device__ __forceinline__ void head_product(unsigned char* lds, const Stage<HD_BM, AROW>& sa,
                                             const Stage<BN, BROW>& sb, int depth, int wave, int lane,
                                             floatx16 (&acc)[Waves<BN>::MT][Waves<BN>::NT]) {
  using W = Waves<BN>;
  constexpr int AB = Stage<HD_BM, AROW>::BYTES, BUF = AB + Stage<BN, BROW>::BYTES;
  Reads<HD_BM, AROW, W::MT> ra;
  Reads<BN, BROW, W::NT> rb;
  ra.init(lds_addr(lds), (wave / W::N) * (W::MT * 32), lane);
  rb.init(lds_addr(lds + AB), (wave % W::N) * (W::NT * 32), lane);
  constexpr int PER = Reads<HD_BM, AROW, W::MT>::PER + Reads<BN, BROW, W::NT>::PER;
  const int steps = (depth + HD_BK - 1) / HD_BK;
  sa.load(lds, 0, wave);
  sb.load(lds + AB, 0, wave);
  for (int s = 0; s < steps; ++s) {
    const uint32_t buf = (s & 1) * BUF;
    wait_vmcnt0();
    __syncthreads();  // the step has landed, and the other buffer's readers are done
    __builtin_amdgcn_sched_barrier(0);
    if (s + 1 < steps) {
      sa.load(lds + (BUF - buf), (s + 1) * HD_BK, wave);
      sb.load(lds + (BUF - buf) + AB, (s + 1) * HD_BK, wave);
    }
    bf16x8 a[2][W::MT], b[2][W::NT];
    ra.template read<0>(buf, a[0]);
    rb.template read<0>(buf, b[0]);
    auto multiply = [&](int h) {
#pragma unroll
      for (int i = 0; i < W::MT; ++i)
#pragma unroll
        for (int j = 0; j < W::NT; ++j) acc[i][j] = mfma32(a[h][i], b[h][j], acc[i][j]);
    };
    ra.template read<1>(buf, a[1]);
    rb.template read<1>(buf, b[1]);
    lgkm_wait<PER>();
    multiply(0);
    ra.template read<2>(buf, a[0]);
    rb.template read<2>(buf, b[0]);
    lgkm_wait<PER>();
    multiply(1);
    ra.template read<3>(buf, a[1]);
    rb.template read<3>(buf, b[1]);
    lgkm_wait<PER>();
    multiply(0);
    lgkm_wait<0>();
    multiply(1);
  }
}

// Which tile a workgroup takes.  Workgroups go to the 8 XCDs in turn; each XCD gets a
// contiguous run of tiles, in groups of 8 row tiles over all column tiles, so that the 32
// that run at once on it share 8 + 4 operand tiles in its L2.
__device__ __forceinline__ bool head_tile(int id, int nm, int nn, int& tm, int& tn) {
  const int total = nm * nn, per = (total + 7) / 8;
  const int w = (id & 7) * per + (id >> 3);
  if ((id >> 3) >= per || w >= total) return false;
  const int group = w / (8 * nn), left = nm - group * 8, g = left < 8 ? left : 8;
  const int in = w - group * 8 * nn;
  tn = in / g;
  tm = group * 8 + in - tn * g;
  return true;
}
static int head_grid(int64_t nm, int64_t nn) { return (int)((nm * nn + 7) / 8 * 8); }

struct HeadParams {
  const bf16* hc;
  const bf16* w;
  int64_t rows;      // tokens in all, kept or not
  int V, H;
  const int* count;
  const int* target;
  float c;           // log2(e) / T
  floatx2* part;     // forward: (vocabulary tiles, rows) partial (m, l)
  float* zlabel;
  const floatx4* coef;  // backward
  bf16* dz;          // (rows, ldz): this range's v0 .. v0 + vc
  int64_t ldz;
  int v0, vc;
  bf16* dw;
  float* dh;         // (slabs, rows, H) fp32 partial sums
  int slabs, add;
};

// ---------------------------------------------------------------------------
// z = hc w^T, vocabulary on the row axis: a lane holds one token's 64 (or 16) vocabulary
// entries of each block, so their maximum and sum need no shuffles but one.  DZ: dz of a
// range of the vocabulary instead of the statistics.
template <int BN, bool DZ>
__global__ __launch_bounds__(512) void head_logits_kernel(HeadParams p) {
  using W = Waves<BN>;
  extern __shared__ __align__(1024) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int count = *p.count;
  int tm, tn;
  const int vc = DZ ? p.vc : p.V;
  if (!head_tile(blockIdx.x, (vc + HD_BM - 1) / HD_BM, (int)((p.rows + BN - 1) / BN), tm, tn)) return;
  const int n0 = tn * BN, v0 = (DZ ? p.v0 : 0) + tm * HD_BM;
  if (n0 >= count) return;
  const int vend = DZ ? p.v0 + p.vc : p.V;
  Stage<HD_BM, true> sa;
  Stage<BN, true> sb;
  sa.init(p.w, p.H, v0, vend, p.H, wave, lane);
  sb.init(p.hc, p.H, n0, count, p.H, wave, lane);
  floatx16 acc[W::MT][W::NT];
#pragma unroll
  for (int i = 0; i < W::MT; ++i)
#pragma unroll
    for (int j = 0; j < W::NT; ++j) acc[i][j] = floatx16{};
  head_product<BN, true, true>(lds, sa, sb, p.H, wave, lane, acc);

  const int wm = wave / W::N, wn = wave % W::N;
  const int vw = wm * (W::MT * 32) + (lane >> 5) * 4;  // the lane's first entry in the tile
  __syncthreads();                                     // the buffers' readers are done
#pragma unroll
  for (int j = 0; j < W::NT; ++j) {
    const int nl = wn * (W::NT * 32) + j * 32 + (lane & 31), n = n0 + nl;
    const int y = n < count ? p.target[n] : -1;
    const int at = y - v0 - vw;  // the label's entry relative to the lane's first
    if (!DZ) {
      if (wave_any(y >= 0 && at >= 0 && at < W::MT * 32 && !(at & 4))) {
#pragma unroll
        for (int i = 0; i < W::MT; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (y >= 0 && at == i * 32 + (e >> 2) * 8 + (e & 3)) p.zlabel[n] = acc[i][j][e];
      }
      if (v0 + HD_BM > p.V) {
#pragma unroll
        for (int i = 0; i < W::MT; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (v0 + vw + i * 32 + (e >> 2) * 8 + (e & 3) >= p.V) acc[i][j][e] = -INFINITY;
      }
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < W::MT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, acc[i][j][e]);
      m = xor32_max(m);
      const float base = finite_max(m);
      float l = 0.f;
#pragma unroll
      for (int i = 0; i < W::MT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) l += fast_exp2((acc[i][j][e] - base) * p.c);
      l = xor32_sum(l);
      if (lane < 32) reinterpret_cast<floatx2*>(lds)[wm * BN + nl] = floatx2{m, l};
    } else {
      const floatx4 k = n < count ? p.coef[n] : floatx4{};
#pragma unroll
      for (int i = 0; i < W::MT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int vl = vw + i * 32 + q * 8;  // 4 consecutive entries
          floatx4 d;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            d[e] = k[1] * fast_exp2((acc[i][j][q * 4 + e] - k[0]) * p.c);
            if (at == i * 32 + q * 8 + e && y >= 0) d[e] += k[2];
            if (v0 + vl + e >= vend) d[e] = 0.f;
          }
          store4<bf16>(reinterpret_cast<bf16*>(lds + nl * 512 + (((vl >> 3) ^ (nl & 31)) << 4) + (lane >> 5) * 8), d);
        }
    }
  }
  __syncthreads();
  if (!DZ) {
    for (int nl = threadIdx.x; nl < BN; nl += 512) {
      if (n0 + nl < count) {
        RowStat s{-INFINITY, 0.f};
#pragma unroll
        for (int i = 0; i < W::M; ++i) {
          const floatx2 v = reinterpret_cast<const floatx2*>(lds)[i * BN + nl];
          s = join(s, RowStat{v[0], v[1]}, p.c);
        }
        p.part[(int64_t)tm * p.rows + n0 + nl] = floatx2{s.m, s.l};
      }
    }
  } else {
    const int ch = threadIdx.x & 31;
    for (int nl = threadIdx.x >> 5; nl < BN; nl += 16) {
      const int64_t col = (int64_t)(v0 - p.v0) + ch * 8;
      if (n0 + nl < count && col < p.ldz)
        *reinterpret_cast<bf16x8*>(p.dz + (int64_t)(n0 + nl) * p.ldz + col) =
            *reinterpret_cast<const bf16x8*>(lds + nl * 512 + ((ch ^ (nl & 31)) << 4));
    }
  }
}

// The tiles' statistics of each kept row joined: 16 rows x 64 slots of tiles a workgroup.
struct HeadJoin {
  const floatx2* part;
  const float* zlabel;
  const int* count;
  const int* index;
  float* logprobs;
  floatx2* stats;
  int64_t rows;
  int tiles;
  float c, inv_t;
};

__global__ __launch_bounds__(1024) void head_join_kernel(HeadJoin p) {
  __shared__ RowStat red[64][17];
  const int r = threadIdx.x & 15, slot = threadIdx.x >> 4;
  const int count = *p.count;
  const int n0 = blockIdx.x * 16, n = n0 + r;
  if (n0 >= count) return;
  RowStat s{-INFINITY, 0.f};
  if (n < count) {
#pragma unroll 4
    for (int t = slot; t < p.tiles; t += 64) {
      const floatx2 v = p.part[(int64_t)t * p.rows + n];
      s = join(s, RowStat{v[0], v[1]}, p.c);
    }
  }
  red[slot][r] = s;
  __syncthreads();
  for (int k = 32; k >= 1; k >>= 1) {
    if (slot < k) red[slot][r] = join(red[slot][r], red[slot + k][r], p.c);
    __syncthreads();
  }
  if (slot == 0 && n < count) {
    s = red[0][r];
    const int row = p.index[n];
    p.logprobs[row] = (p.zlabel[n] - s.m) * p.inv_t - logf(s.l);
    p.stats[row] = floatx2{s.m, s.l};
  }
}

// dw[v][h] = sum over kept tokens of dz[n][v] hc[n][h], v0 <= v < v0 + vc: both operands have
// the depth (tokens) as their slow axis.  The tile goes out through LDS in whole lines.
__global__ __launch_bounds__(512) void head_dw_kernel(HeadParams p) {
  using W = Waves<256>;
  extern __shared__ __align__(1024) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int count = *p.count;
  int th, tv;
  if (!head_tile(blockIdx.x, (p.H + HD_BM - 1) / HD_BM, (p.vc + 255) / 256, th, tv)) return;
  const int h0 = th * HD_BM, v0 = tv * 256;
  Stage<HD_BM, false> sa;
  Stage<256, false> sb;
  sa.init(p.hc, p.H, h0, p.H, count, wave, lane);
  sb.init(p.dz, p.ldz, v0, p.ldz, count, wave, lane);
  floatx16 acc[W::MT][W::NT];
#pragma unroll
  for (int i = 0; i < W::MT; ++i)
#pragma unroll
    for (int j = 0; j < W::NT; ++j) acc[i][j] = floatx16{};
  if (count > 0) head_product<256, false, false>(lds, sa, sb, count, wave, lane, acc);
  const int wm = wave / W::N, wn = wave % W::N;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < W::NT; ++j) {
    const int vl = wn * 64 + j * 32 + (lane & 31);
#pragma unroll
    for (int i = 0; i < W::MT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int hl = wm * 128 + i * 32 + q * 8;
        const floatx4 d{acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]};
        store4<bf16>(reinterpret_cast<bf16*>(lds + vl * 512 + (((hl >> 3) ^ (vl & 31)) << 4) + (lane >> 5) * 8), d);
      }
  }
  __syncthreads();
  const int ch = threadIdx.x & 31;
  for (int vl = threadIdx.x >> 5; vl < 256; vl += 16) {
    const int v = v0 + vl, h = h0 + ch * 8;
    if (v < p.vc && h < p.H)
      *reinterpret_cast<bf16x8*>(p.dw + (int64_t)(p.v0 + v) * p.H + h) =
          *reinterpret_cast<const bf16x8*>(lds + vl * 512 + ((ch ^ (vl & 31)) << 4));
  }
}

// dh[n][h] (+)= sum over this range's v of dz[n][v] w[v][h], fp32.  The depth (vocabulary) is
// long and the tiles may be few: it is split over slabs, each with sums of its own, which
// the last launch adds in order.
template <int BN>
__global__ __launch_bounds__(512) void head_dh_kernel(HeadParams p) {
  using W = Waves<BN>;
  extern __shared__ __align__(1024) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int count = *p.count;
  const int nh = (p.H + HD_BM - 1) / HD_BM, nn = (int)((p.rows + BN - 1) / BN);
  int th, rest;
  if (!head_tile(blockIdx.x, nh, nn * p.slabs, th, rest)) return;
  const int slab = rest / nn, tn = rest - slab * nn;
  const int h0 = th * HD_BM, n0 = tn * BN;
  if (n0 >= count) return;
  const int per = ((p.vc + p.slabs - 1) / p.slabs + HD_BK - 1) / HD_BK * HD_BK;
  const int k0 = slab * per, depth = p.vc - k0 < per ? p.vc - k0 : per;
  floatx16 acc[W::MT][W::NT];
#pragma unroll
  for (int i = 0; i < W::MT; ++i)
#pragma unroll
    for (int j = 0; j < W::NT; ++j) acc[i][j] = floatx16{};
  if (depth > 0) {
    Stage<HD_BM, false> sa;
    Stage<BN, true> sb;
    sa.init(p.w + (int64_t)(p.v0 + k0) * p.H, p.H, h0, p.H, depth, wave, lane);
    sb.init(p.dz + k0, p.ldz, n0, count, depth, wave, lane);
    head_product<BN, false, true>(lds, sa, sb, depth, wave, lane, acc);
  } else if (p.add) {
    return;
  }
  const int wm = wave / W::N, wn = wave % W::N;
#pragma unroll
  for (int j = 0; j < W::NT; ++j) {
    const int n = n0 + wn * (W::NT * 32) + j * 32 + (lane & 31);
    if (n < count) {
#pragma unroll
      for (int i = 0; i < W::MT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int h = h0 + wm * (W::MT * 32) + i * 32 + q * 8 + (lane >> 5) * 4;
          if (h < p.H) {
            floatx4* o = reinterpret_cast<floatx4*>(p.dh + ((int64_t)slab * p.rows + n) * p.H + h);
            floatx4 d{acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]};
            if (p.add) d += *o;
            *o = d;
          }
        }
    }
  }
}

// dhidden: the slabs' sums, rounded, in the rows' own places; zeros in ignored rows.
__global__ __launch_bounds__(256) void head_dh_out_kernel(const float* dh, int slabs, int64_t rows, int H,
                                                          const int* pos, bf16* out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int ch = H / 8;
  if (i >= rows * ch) return;
  const int64_t row = i / ch;
  const int c = (int)(i - row * ch), place = pos[row];
  floatx8 s{};
  if (place >= 0) {
    const float* src = dh + (int64_t)place * H + c * 8;
    s = Vec8<float>::load_f32(src);
    for (int k = 1; k < slabs; ++k) s += Vec8<float>::load_f32(src + k * rows * H);
  }
  store8<bf16>(out + row * H + c * 8, s);
}

}  // namespace nq

using namespace nq;

static int64_t pad256(int64_t n) { return (n + 255) / 256 * 256; }

// Tokens of a tile.
static int head_bn(int64_t rows) { return rows <= 64 ? 64 : 256; }

// Where each piece of a workspace lies.
struct HeadSpace {
  int64_t count, pos, index, target, zlabel, coef, hc, part, dz, dh, total;
  int64_t ldz;
  int vc, slabs;
};

constexpr int64_t HD_DZ_BYTES = (int64_t)1 << 30;  // the largest range's dz

static HeadSpace head_space(int64_t rows, int V, int H, bool backward) {
  HeadSpace s{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += pad256(bytes);
    return here;
  };
  s.count = take(4);
  s.pos = take(rows * 4);
  s.index = take(rows * 4);
  s.target = take(rows * 4);
  s.hc = take(rows * H * 2);
  if (!backward) {
    s.zlabel = take(rows * 4);
    s.part = take(rows * ((V + HD_BM - 1) / HD_BM) * 8);
  } else {
    s.coef = take(rows * 16);
    // equal ranges of whole tiles
    const int64_t most = HD_DZ_BYTES / (rows * 2) / HD_BM * HD_BM;
    const int64_t vpad = pad256(V), step = most < HD_BM ? HD_BM : most;
    const int64_t ranges = (vpad + step - 1) / step;
    s.vc = (int)pad256((V + ranges - 1) / ranges);
    if (s.vc > V) s.vc = V;
    s.ldz = (s.vc + 7) / 8 * 8;
    const int bn = head_bn(rows);
    const int64_t tiles = ((rows + bn - 1) / bn) * ((H + HD_BM - 1) / HD_BM);
    int64_t slabs = 256 / tiles;
    const int64_t deep = (s.vc + 8 * HD_BK - 1) / (8 * HD_BK);  // at least 8 steps each
    if (slabs > deep) slabs = deep;
    s.slabs = slabs < 1 ? 1 : (int)slabs;
    s.dz = take(rows * s.ldz * 2);
    s.dh = take((int64_t)s.slabs * rows * H * 4);
  }
  s.total = at;
  return s;
}

static bool head_sizes_ok(int64_t rows, int V, int H) {
  return rows > 0 && rows <= (1 << 24) && V > 0 && V <= (1 << 24) && H > 0 && H % 8 == 0 && H <= (1 << 20);
}

extern "C" int64_t nq_linear_logprobs_workspace_bytes(int64_t rows, int V, int H) {
  return head_sizes_ok(rows, V, H) ? head_space(rows, V, H, false).total : 0;
}
extern "C" int64_t nq_linear_logprobs_bwd_workspace_bytes(int64_t rows, int V, int H) {
  return head_sizes_ok(rows, V, H) ? head_space(rows, V, H, true).total : 0;
}

static int head_check(const void* hidden, int64_t bs, int64_t rs, const void* weight, const int64_t* labels,
                      const void* stats, const void* workspace, int64_t workspace_bytes, int64_t B, int64_t S, int V,
                      int H, float temperature, bool backward) {
  if (B <= 0 || S <= 0 || V <= 0 || H <= 0)
    return nq_fail(NQ_ERR_INVALID, "sizes must be positive (B=%lld S=%lld V=%d H=%d)", (long long)B, (long long)S, V, H);
  if (H % 8) return nq_fail(NQ_ERR_UNSUPPORTED, "the width must be a multiple of 8, got %d", H);
  if (S > (1 << 24) || B > (1 << 24) / S || !head_sizes_ok(B * S, V, H))
    return nq_fail(NQ_ERR_UNSUPPORTED, "at most 2^24 rows and entries and a width of 2^20");
  if (!hidden || !weight || !labels || !stats)
    return nq_fail(NQ_ERR_INVALID, "hidden, weight, labels and stats are required");
  if (bs < 0 || rs < 0 || bs % 8 || rs % 8 || !nq_aligned16(hidden) || !nq_aligned16(weight))
    return nq_fail(NQ_ERR_INVALID, "rows of hidden and weight must be 16-byte aligned, strides not negative");
  if ((reinterpret_cast<uintptr_t>(labels) & 7u) || (reinterpret_cast<uintptr_t>(stats) & 7u))
    return nq_fail(NQ_ERR_INVALID, "labels and stats must be aligned to their elements");
  const float inv = 1.f / temperature;
  if (!(temperature > 0.f) || !isfinite(temperature) || !isfinite(inv * kLog2e))
    return nq_fail(NQ_ERR_INVALID, "the temperature must be positive and finite, and so must its reciprocal");
  const int64_t need = head_space(B * S, V, H, backward).total;
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return nq_fail(NQ_ERR_WORKSPACE, "workspace too small or not 256-byte aligned: %lld bytes, need %lld",
                   (long long)workspace_bytes, (long long)need);
  return NQ_OK;
}

// Dynamic LDS of a product: two buffers of both operands.
static constexpr int head_lds(int bn) { return 2 * (HD_BM + bn) * HD_BK * 2; }

// The attribute belongs to a kernel on a device; setting it is cheap and idempotent.
static int head_allow(const void* kernel, int bytes) {
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  return e == hipSuccess ? NQ_OK : nq_check_launch(e);
}

template <typename K>
static int head_launch(K kernel, int grid, int bn, hipStream_t st, const HeadParams& p) {
  if (int rc = head_allow(reinterpret_cast<const void*>(kernel), head_lds(bn))) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(512), head_lds(bn), st, p);
  return nq_check_launch(hipGetLastError());
}

extern "C" int nq_linear_logprobs(const void* hidden, int64_t batch_stride, int64_t row_stride, const void* weight,
                                  const int64_t* labels, float* logprobs, float* stats, void* workspace,
                                  int64_t workspace_bytes, int64_t B, int64_t S, int V, int H, float temperature,
                                  int64_t ignore_index, void* stream) {
  nq_clear_error();
  if (int rc = head_check(hidden, batch_stride, row_stride, weight, labels, stats, workspace, workspace_bytes, B, S, V,
                          H, temperature, false))
    return rc;
  if (!logprobs || (reinterpret_cast<uintptr_t>(logprobs) & 3u))
    return nq_fail(NQ_ERR_INVALID, "logprobs is required, aligned to fp32");
  const int64_t rows = B * S;
  const HeadSpace s = head_space(rows, V, H, false);
  char* ws = reinterpret_cast<char*>(workspace);
  const float inv = 1.f / temperature;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  HeadRows r{};
  r.hidden = reinterpret_cast<const bf16*>(hidden), r.bs = batch_stride, r.rs = row_stride, r.S = S;
  r.labels = labels, r.rows = rows, r.ignore = ignore_index, r.H = H, r.V = V;
  r.count = reinterpret_cast<int*>(ws + s.count), r.pos = reinterpret_cast<int*>(ws + s.pos);
  r.index = reinterpret_cast<int*>(ws + s.index), r.target = reinterpret_cast<int*>(ws + s.target);
  r.hc = reinterpret_cast<bf16*>(ws + s.hc);
  r.logprobs = logprobs, r.stats = reinterpret_cast<floatx2*>(stats), r.zlabel = reinterpret_cast<float*>(ws + s.zlabel);
  hipLaunchKernelGGL(head_rows_kernel, dim3((unsigned)((rows + HD_PREP - 1) / HD_PREP)), dim3(256), 0, st, r);
  HeadParams p{};
  p.hc = r.hc, p.w = reinterpret_cast<const bf16*>(weight), p.rows = rows, p.V = V, p.H = H;
  p.count = r.count, p.target = r.target, p.c = inv * kLog2e;
  p.part = reinterpret_cast<floatx2*>(ws + s.part), p.zlabel = r.zlabel;
  const int bn = head_bn(rows), tiles = (V + HD_BM - 1) / HD_BM;
  const int64_t nn = (rows + bn - 1) / bn;
  if (tiles * nn > INT32_MAX / 2) return nq_fail(NQ_ERR_UNSUPPORTED, "too many tiles for one launch");
  const int grid = head_grid(tiles, nn);
  if (int rc = bn == 64 ? head_launch(head_logits_kernel<64, false>, grid, bn, st, p)
                        : head_launch(head_logits_kernel<256, false>, grid, bn, st, p))
    return rc;
  HeadJoin j{p.part, p.zlabel, r.count, r.index, logprobs, r.stats, rows, tiles, p.c, inv};
  hipLaunchKernelGGL(head_join_kernel, dim3((unsigned)((rows + 15) / 16)), dim3(1024), 0, st, j);
  return nq_check_launch(hipGetLastError());
}

extern "C" int nq_linear_logprobs_bwd(const void* hidden, int64_t batch_stride, int64_t row_stride, const void* weight,
                                      const int64_t* labels, const float* stats, const float* dlogprobs,
                                      void* dhidden, void* dweight, void* workspace, int64_t workspace_bytes,
                                      int64_t B, int64_t S, int V, int H, float temperature, int64_t ignore_index,
                                      void* stream) {
  nq_clear_error();
  if (int rc = head_check(hidden, batch_stride, row_stride, weight, labels, stats, workspace, workspace_bytes, B, S, V,
                          H, temperature, true))
    return rc;
  if (!dlogprobs || (reinterpret_cast<uintptr_t>(dlogprobs) & 3u) || !nq_aligned16(dhidden) || !nq_aligned16(dweight))
    return nq_fail(NQ_ERR_INVALID, "dlogprobs is required, and gradients must be 16-byte aligned");
  if (!dhidden && !dweight) return NQ_OK;
  const int64_t rows = B * S;
  const HeadSpace s = head_space(rows, V, H, true);
  char* ws = reinterpret_cast<char*>(workspace);
  const float inv = 1.f / temperature;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  HeadRows r{};
  r.hidden = reinterpret_cast<const bf16*>(hidden), r.bs = batch_stride, r.rs = row_stride, r.S = S;
  r.labels = labels, r.rows = rows, r.ignore = ignore_index, r.H = H, r.V = V;
  r.count = reinterpret_cast<int*>(ws + s.count), r.pos = reinterpret_cast<int*>(ws + s.pos);
  r.index = reinterpret_cast<int*>(ws + s.index), r.target = reinterpret_cast<int*>(ws + s.target);
  r.hc = reinterpret_cast<bf16*>(ws + s.hc);
  r.stats = reinterpret_cast<floatx2*>(const_cast<float*>(stats)), r.dy = dlogprobs;
  r.coef = reinterpret_cast<floatx4*>(ws + s.coef), r.inv_t = inv;
  hipLaunchKernelGGL(head_rows_kernel, dim3((unsigned)((rows + HD_PREP - 1) / HD_PREP)), dim3(256), 0, st, r);
  HeadParams p{};
  p.hc = r.hc, p.w = reinterpret_cast<const bf16*>(weight), p.rows = rows, p.V = V, p.H = H;
  p.count = r.count, p.target = r.target, p.c = inv * kLog2e, p.coef = r.coef;
  p.dz = reinterpret_cast<bf16*>(ws + s.dz), p.ldz = s.ldz;
  p.dw = reinterpret_cast<bf16*>(dweight), p.dh = reinterpret_cast<float*>(ws + s.dh), p.slabs = s.slabs;
  const int bn = head_bn(rows), nh = (H + HD_BM - 1) / HD_BM;
  const int64_t nn = (rows + bn - 1) / bn;
  if (((int64_t)s.vc / 256 + 1) * (nn > nh ? nn : nh) > INT32_MAX / 2 || nn * s.slabs * nh > INT32_MAX / 2)
    return nq_fail(NQ_ERR_UNSUPPORTED, "too many tiles for one launch");
  for (int v0 = 0; v0 < V; v0 += s.vc) {
    p.v0 = v0, p.vc = V - v0 < s.vc ? V - v0 : s.vc, p.add = v0 > 0;
    const int nv = (p.vc + 255) / 256;
    int rc = bn == 64 ? head_launch(head_logits_kernel<64, true>, head_grid(nv, nn), bn, st, p)
                      : head_launch(head_logits_kernel<256, true>, head_grid(nv, nn), bn, st, p);
    if (!rc && dhidden)
      rc = bn == 64 ? head_launch(head_dh_kernel<64>, head_grid(nh, nn * s.slabs), bn, st, p)
                    : head_launch(head_dh_kernel<256>, head_grid(nh, nn * s.slabs), bn, st, p);
    if (!rc && dweight) rc = head_launch(head_dw_kernel, head_grid(nh, nv), 256, st, p);
    if (rc) return rc;
  }
  if (dhidden) {
    const int64_t n = rows * (H / 8);
    hipLaunchKernelGGL(head_dh_out_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p.dh, s.slabs, rows, H,
                       r.pos, reinterpret_cast<bf16*>(dhidden));
  }
  return nq_check_launch(hipGetLastError());
}
