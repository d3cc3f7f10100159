// Log-probabilities of labels straight from a model's last hidden states and its LM head,
// and their gradients: z = h w^T / T without the (tokens x vocabulary) logits in memory.
//
//   forward    z tile by tile; each tile leaves its rows' maximum and sum of exponentials
//              (and the label's logit), which a second launch joins:
//              logprob = (z[label] - m) / T - log l
//   backward   dz = dy (1[v = label] - softmax) / T in bf16, a range of the vocabulary at a
//              time, from the exponentials that the forward kept or from its product again;
//              dh += dz w and dw = dz^T h
//
// Three or four products of 2 tokens vocabulary width operations each, all on one core:
// bf16 MFMA with fp32 accumulation over tiles of 256 x 256 (or 64 tokens, where there are
// few).  dz is rounded to bf16 once, as the matrix cores need it, and so is a kept
// exponential: half a step, 2^-8 of a value at most, independent from term to term.  Ignored
// rows are left out first: the kept rows are gathered to the front, and the products run over
// those.
//
// Bound by the matrix cores at the clock that the power limit leaves them.  8192 x 2048 against
// 151936 entries: the forward, with what it keeps, 4.5 ms (1.14 PFLOP/s; a library product of
// its size alone 3.8), dz 0.9 (5.5 TB/s), dh 4.0 and dw 4.1 (library products 3.8 and 4.6).
// 4 x 1023 rows of 1024, a quarter ignored: 0.93 ms, 0.34, 0.84 and 0.84 (library 1.0, 1.2 and 1.1).

#include <math.h>

#include "nq_common.hpp"
#include "nq_internal.hpp"
#include "nq_loss.hpp"

namespace nq {

constexpr int HD_BK = 64;    // depth of a step
constexpr int HD_CUS = 256;

// A product's tile, BM (the MFMA's row axis) x BN, and how its waves share it: M x N of
// them, each MT x NT blocks of 32 x 32.  OUT: rows that a wave puts out at a time.
//   Wide  one workgroup a CU: 128 accumulator registers a lane, 128 KB of operands
//   Few   at most 64 tokens, bound by reading the weights: three workgroups a CU, so that
//         72 KB are in flight there (33 rows of 1024 against 151936 entries, 311 MB: 54 us,
//         60 with two)
struct Wide {
  static constexpr int BM = 256, BN = 256, M = 2, N = 4, MT = 4, NT = 2, PER_CU = 1, OUT = 32;
};
struct Few {
  static constexpr int BM = 128, BN = 64, M = 4, N = 1, MT = 1, NT = 2, PER_CU = 3, OUT = 16;
};
template <class C> constexpr int threads_of() { return C::M * C::N * 64; }

// The rows as the caller holds them; for at most 64 a workgroup finds the kept ones by itself.
struct HeadSource {
  const bf16* hidden;
  int64_t bs, rs, S;
  const int64_t* labels;
  int64_t rows, ignore;
  __device__ __forceinline__ const bf16* row(int64_t r) const {
    const int64_t b = r / S;
    return hidden + b * bs + (r - b * S) * rs;
  }
  // by one wave: index[place] of each kept row; how many there are
  __device__ __forceinline__ int few(int lane, int V, int* index, int* target) const {
    const int64_t y = lane < rows ? labels[lane] : ignore;
    const uint64_t kept = __builtin_amdgcn_ballot_w64(y != ignore);
    if (y != ignore) {
      const int place = __popcll(kept & ((1ull << lane) - 1));
      index[place] = lane;
      target[place] = y >= 0 && y < V ? (int)y : -1;
    }
    return __popcll(kept);
  }
};

// ---------------------------------------------------------------------------
// The kept rows, in order: pos[row] = its place among them (-1: ignored), index the
// reverse, hc their hidden states.  A workgroup counts the kept rows before its own (the
// labels are small and in L2) rather than wait for another launch: 16 rows each, or more
// where there would be over 2048 workgroups to read them.
struct HeadRows {
  HeadSource src;
  int64_t each;  // rows of a workgroup
  int H, V;
  int* count;
  int* pos;       // (rows)
  int* index;     // (rows)
  int* target;    // (rows) the kept rows' labels, -1 outside the vocabulary
  bf16* hc;       // (rows, H)
  // forward
  float* logprobs;
  floatx2* stats;
  // backward
  const float* dy;
  floatx4* coef;  // (rows) by place: m, -g / l, g = dy / T
  float inv_t;
};

__global__ __launch_bounds__(256) void head_rows_kernel(HeadRows p) {
  __shared__ int before[4], own[64], kept_here;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t first = (int64_t)blockIdx.x * p.each;
  const int64_t last = first + p.each < p.src.rows ? first + p.each : p.src.rows;
  int n = 0;
#pragma unroll 8
  for (int64_t r = tid; r < first; r += 256) n += p.src.labels[r] != p.src.ignore;
#pragma unroll
  for (int k = 32; k >= 1; k >>= 1) n += __shfl_xor(n, k, 64);
  if (lane == 0) before[wave] = n;
  __syncthreads();
  int base = before[0] + before[1] + before[2] + before[3];
  const int ch = p.H / 8;
  for (int64_t r0 = first; r0 < last; r0 += 64) {
    const int here = (int)(last - r0 < 64 ? last - r0 : 64);
    if (wave == 0) {
      const int64_t r = r0 + lane;
      const int64_t y = lane < here ? p.src.labels[r] : p.src.ignore;
      const bool kept = y != p.src.ignore;
      const uint64_t ballot = __builtin_amdgcn_ballot_w64(kept);
      const int place = kept ? base + __popcll(ballot & ((1ull << lane) - 1)) : -1;
      own[lane] = place;
      if (lane == 0) kept_here = __popcll(ballot);
      if (lane < here) {
        p.pos[r] = place;
        const bool inside = y >= 0 && y < p.V;
        if (kept) {
          p.index[place] = (int)r;
          p.target[place] = inside ? (int)y : -1;
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
    }
    __syncthreads();
    base += kept_here;
    for (int i = wave; i < here; i += 4) {
      const int place = own[i];
      if (place < 0) continue;
      const bf16x8* src = reinterpret_cast<const bf16x8*>(p.src.row(r0 + i));
      bf16x8* dst = reinterpret_cast<bf16x8*>(p.hc + (int64_t)place * p.H);
      for (int c = lane; c < ch; c += 64) dst[c] = src[c];
    }
    __syncthreads();  // own's readers are done
  }
  if (last == p.src.rows && tid == 0) *p.count = base;
}

// One operand of a product, (extent x depth), staged in LDS a step of 64 deep at a time.
//   ROW   depth contiguous in memory: LDS rows of 128 bytes, an operand one 16-byte read.
//         16-byte chunk c of row r lies at c ^ (r / 2 % 8): 16 consecutive rows' reads
//         hit distinct banks.
//   !ROW  extent contiguous: LDS rows (one depth each) of 2 EXT bytes, transpose reads.
//         Chunk c of depth k lies at c ^ 4 (k % 4): the 4 depths of a read hit distinct
//         banks.
// HBM -> LDS without registers; what lies outside (rows past the extent, depths past the
// end) is out of the descriptor's range and arrives as zeros.
template <int EXT, bool ROW, int WAVES, bool STREAM = false>
struct Stage {
  static constexpr int BYTES = EXT * HD_BK * 2;
  static constexpr int NI = BYTES / 1024 / WAVES;   // loads of a wave per step
  static constexpr int LINE = ROW ? 128 : EXT * 2;  // bytes of an LDS row
  static constexpr int ROWS_PER = 1024 / LINE;
  static_assert(BYTES % (1024 * WAVES) == 0 && (WAVES * ROWS_PER) % 16 == 0, "a wave's loads keep their swizzle");
  const char* base;  // ROW: first row, else first depth
  uint32_t line;     // bytes of a row in memory
  uint32_t range;    // ROW: bytes from base to the end of the last row; else of the columns that exist
  int depth;         // how many depths exist
  uint32_t off, chunk;

  __device__ __forceinline__ void lanes(int64_t ld, int wave, int lane) {
    line = (uint32_t)(ld * 2);
    const int r = wave * ROWS_PER + lane / (LINE / 16), pc = lane % (LINE / 16);
    chunk = ROW ? (uint32_t)((pc ^ ((r >> 1) & 7)) * 16) : (uint32_t)((pc ^ ((r & 3) << 2)) * 16);
    off = (uint32_t)r * line + chunk;
  }
  // extents [e0, e0 + EXT) of n, of depths [0, d)
  __device__ __forceinline__ void at(const bf16* p, int64_t e0, int64_t n, int d) {
    depth = d;
    const int64_t left = n - e0;
    if (ROW) {
      base = reinterpret_cast<const char*>(p) + e0 * line;
      range = left <= 0 ? 0 : (uint32_t)((left < EXT ? left : EXT) * (int64_t)line);
    } else {
      base = reinterpret_cast<const char*>(p + e0);
      range = left <= 0 ? 0 : (uint32_t)((left < EXT ? left : EXT) * 2);
    }
  }
  // the step at depth k0 into LDS at `tile`
  __device__ __forceinline__ void load(unsigned char* tile, int k0, int wave) const {
    constexpr uint32_t NONE = 0x80000000u;  // out of any range
    const int left = depth - k0;
    uint32_t o;
    BufRsrc r;
    if (ROW) {
      r = make_rsrc(base, range);
      o = (int)chunk < 2 * left ? off + (uint32_t)k0 * 2 : NONE;
    } else {
      r = make_rsrc(base + (int64_t)k0 * line, (uint32_t)(left < HD_BK ? left : HD_BK) * line);
      o = chunk < range ? off : NONE;
    }
    const uint32_t step = o == NONE ? 0u : WAVES * ROWS_PER * line;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if (STREAM) buffer_load_lds16_nt(r, tile + (wave + WAVES * i) * 1024, o + i * step, 0u);
      else buffer_load_lds16(r, tile + (wave + WAVES * i) * 1024, o + i * step, 0u);
    }
  }
};

// Stage<EXT, true> of rows that lie anywhere: their hidden states as the caller holds them.
// Rows past the count repeat the first (nothing is kept of them), and depths past the end its
// first chunk, against zeros of the other operand.
template <int EXT, int WAVES>
struct GatherStage {
  static constexpr int BYTES = EXT * HD_BK * 2, NI = BYTES / 1024 / WAVES;
  const char* row[NI];
  int depth;
  uint32_t chunk;
  // row_of(r): where row r begins
  template <typename F>
  __device__ __forceinline__ void at(F row_of, int d, int wave, int lane) {
    depth = d;
    const int r = wave * 8 + lane / 8;
    chunk = (uint32_t)(((lane % 8) ^ ((r >> 1) & 7)) * 16);
#pragma unroll
    for (int i = 0; i < NI; ++i) row[i] = reinterpret_cast<const char*>(row_of(r + WAVES * 8 * i));
  }
  __device__ __forceinline__ void load(unsigned char* tile, int k0, int wave) const {
    const int64_t o = (int)chunk < 2 * (depth - k0) ? (int64_t)k0 * 2 + chunk : 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) global_load_lds16(row[i] + o, tile + (wave + WAVES * i) * 1024);
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
  template <int KK, int T = 0>
  __device__ __forceinline__ void read(uint32_t buf, bf16x8 (&v)[NT]) const {
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
      read<KK, T + 1>(buf, v);
    }
  }
};

// A workgroup's stream of products.  Two LDS buffers: the next step's loads are in flight
// while a step's 64 depths are multiplied, one barrier a step, and the step after a tile's
// last is the next tile's first, so that its loads run under this tile's last products and
// its epilogue.  The operands of the next 16 depths are read while these are multiplied.
template <class C, bool AROW, bool BROW, bool GATHER = false, bool STREAM = false>
struct Product {
  static constexpr int WAVES = C::M * C::N;
  typedef Stage<C::BM, AROW, WAVES, STREAM> A;
  typedef std::conditional_t<GATHER, GatherStage<C::BN, WAVES>, Stage<C::BN, BROW, WAVES>> B;
  static_assert(BROW || !GATHER, "rows are gathered");
  static constexpr int BUF = A::BYTES + B::BYTES;
  static constexpr int NB = C::MT < 2 ? C::MT : 2, CH = NB * 4;  // an output line: blocks, 16-byte chunks
  static constexpr int OWN = C::OUT * CH * 16;  // bytes of a wave's own LDS,
  static constexpr int PRIVATE = 2 * BUF;       // after the buffers
  static constexpr int LDS = PRIVATE + WAVES * OWN;
  static_assert(LDS * C::PER_CU <= 160 * 1024, "LDS of a CU");
  typedef floatx16 Acc[C::MT][C::NT];
  unsigned char* lds;
  int wave, lane;
  uint32_t cur;  // byte offset of the buffer whose step comes next
  Reads<C::BM, AROW, C::MT> ra;
  Reads<C::BN, BROW, C::NT> rb;

  __device__ __forceinline__ void init(unsigned char* l, int w, int ln) {
    lds = l, wave = w, lane = ln, cur = 0;
    ra.init(lds_addr(l), (w / C::N) * (C::MT * 32), ln);
    rb.init(lds_addr(l + A::BYTES), (w % C::N) * (C::NT * 32), ln);
  }
  __device__ __forceinline__ void load(uint32_t buf, const A& a, const B& b, int k0) {
    a.load(lds + buf, k0, wave);
    b.load(lds + buf + A::BYTES, k0, wave);
  }
  // acc = the wave's blocks of A B^T; the first step is under way in the current buffer,
  // and the one of (na, nb) is afterwards, if there is another tile.
  __device__ __forceinline__ void run(const A& a, const B& b, bool more, const A& na, const B& nb, Acc& acc) {
#pragma unroll
    for (int i = 0; i < C::MT; ++i)
#pragma unroll
      for (int j = 0; j < C::NT; ++j) acc[i][j] = floatx16{};
    constexpr int PER = Reads<C::BM, AROW, C::MT>::PER + Reads<C::BN, BROW, C::NT>::PER;
    for (int k = 0; k < a.depth; k += HD_BK) {
      wait_vmcnt0();
      __builtin_amdgcn_s_barrier();  // the step has landed, and the other buffer's readers are done
      __builtin_amdgcn_sched_barrier(0);
      if (k + HD_BK < a.depth) load(BUF - cur, a, b, k + HD_BK);
      else if (more) load(BUF - cur, na, nb, 0);
      bf16x8 x[2][C::MT], y[2][C::NT];
      auto multiply = [&](int h) {
#pragma unroll
        for (int i = 0; i < C::MT; ++i)
#pragma unroll
          for (int j = 0; j < C::NT; ++j) acc[i][j] = mfma32(x[h][i], y[h][j], acc[i][j]);
      };
      ra.template read<0>(cur, x[0]);
      rb.template read<0>(cur, y[0]);
      ra.template read<1>(cur, x[1]);
      rb.template read<1>(cur, y[1]);
      lgkm_wait<PER>();
      multiply(0);
      ra.template read<2>(cur, x[0]);
      rb.template read<2>(cur, y[0]);
      lgkm_wait<PER>();
      multiply(1);
      ra.template read<3>(cur, x[1]);
      rb.template read<3>(cur, y[1]);
      lgkm_wait<PER>();
      multiply(0);
      lgkm_wait<0>();
      multiply(1);
      cur = BUF - cur;
    }
  }
  // The wave's rows (one per lane of its column blocks j) of value(j, i, q), four values of
  // row block i, to global rows of bf16 through the wave's own LDS: 16 bytes a lane in
  // lines of 128 (or 64) bytes.  at(r): row r's first element, or NULL; cols: how many
  // columns exist from there.
  template <typename V, typename At>
  __device__ __forceinline__ void store(V value, At at, int64_t cols) {
    unsigned char* own = lds + PRIVATE + wave * OWN;
    const int ch = lane % CH, mine = lane & 31;
#pragma unroll
    for (int j = 0; j < C::NT; ++j)
#pragma unroll
      for (int i2 = 0; i2 < C::MT; i2 += NB)
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += C::OUT) {
          if (C::OUT == 32 || mine / C::OUT == r0 / C::OUT) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
              for (int q = 0; q < 4; ++q)
                store4<bf16>(reinterpret_cast<bf16*>(own + (mine - r0) * (CH * 16) + (((i * 4 + q) ^ (mine % CH)) << 4) +
                                                     (lane >> 5) * 8),
                             value(j, i2 + i, q));
          }
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int r = 0; r < C::OUT; r += 64 / CH) {
            const int row = r + lane / CH;
            const bf16x8 v = *reinterpret_cast<const bf16x8*>(own + row * (CH * 16) + ((ch ^ ((r0 + row) % CH)) << 4));
            bf16* o = at(j * 32 + r0 + row);
            const int col = i2 * 32 + ch * 8;
            if (o && col < cols) *reinterpret_cast<bf16x8*>(o + col) = v;
          }
          __builtin_amdgcn_wave_barrier();
        }
  }
};

// The tiles of a workgroup.  Workgroups go to the 8 XCDs in turn; each XCD takes a contiguous
// run of tiles, in groups of 8 row tiles over all column tiles, so that the 32 that it works
// on at once share 8 + 4 operand tiles in its L2.
struct Tiles {
  int nm, nn, w, step, end;
  __device__ __forceinline__ Tiles(int nm_, int nn_) : nm(nm_), nn(nn_) {
    const int total = nm * nn, per = (total + 7) / 8, xcd = blockIdx.x & 7;
    w = xcd * per + (blockIdx.x >> 3);
    end = (xcd + 1) * per < total ? (xcd + 1) * per : total;
    step = gridDim.x >> 3;
  }
  __device__ __forceinline__ bool has(int ahead) const { return w + ahead * step < end; }
  __device__ __forceinline__ void get(int ahead, int& tm, int& tn) const {
    const int v = w + ahead * step;
    const int group = v / (8 * nn), left = nm - group * 8, g = left < 8 ? left : 8;
    const int in = v - group * 8 * nn;
    tn = in / g;
    tm = group * 8 + in - tn * g;
  }
};
template <class C>
static int head_grid(int64_t tiles) {
  const int64_t most = HD_CUS * C::PER_CU, n = (tiles + 7) / 8 * 8;
  return (int)(n < most ? n : most);
}

struct HeadParams {
  HeadSource src;
  const bf16* hc;
  const bf16* w;
  int64_t rows;  // tokens in all, kept or not
  int V, H;
  const int* count;
  const int* target;
  float c;       // log2(e) / T
  floatx2* part;  // forward: (vocabulary tiles, rows) partial (m, l)
  float* zlabel;
  bf16* exps;    // kept for the backward: (rows, ldv) 2^((z - m) c) of the m of their 128 entries
  float* exps_m;  // (groups of 128, rows)
  int64_t ldv;
  const floatx4* coef;  // backward
  bf16* dz;      // (rows, ldz): this range's v0 .. v0 + vc
  int64_t ldz;
  int v0, vc, vmax;  // vmax: the largest range
  bf16* dw;
  float* dh;     // fp32 partial sums, a slab after the other
  int add;
};

// ---------------------------------------------------------------------------
// z = hc w^T, vocabulary on the row axis: a lane holds one token's 64 (or 16) vocabulary
// entries of each block, so their maximum and sum need no shuffles but one.  KEEP: the
// exponentials too, for the backward; DZ: dz of a range of the vocabulary instead.
enum { STATS, KEEP, DZ };
template <class C, int MODE, bool GATHER = false, bool STREAM = false>
__global__ __launch_bounds__(threads_of<C>()) void head_logits_kernel(HeadParams p) {
  typedef Product<C, true, true, GATHER, STREAM> P;
  extern __shared__ __align__(1024) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int vend = MODE == DZ ? p.v0 + p.vc : p.V, vfirst = MODE == DZ ? p.v0 : 0;
  // GATHER: the kept rows and their labels in the waves' own LDS, where nothing else lies before
  // the first epilogue, and the labels in registers from there on
  int* few_index = reinterpret_cast<int*>(lds + P::PRIVATE);
  int count;
  if (GATHER) {
    count = p.src.few(lane, p.V, few_index + wave * 128, few_index + wave * 128 + 64);
    __builtin_amdgcn_wave_barrier();
  } else {
    count = __builtin_amdgcn_readfirstlane(*p.count);
  }
  Tiles t((vend - vfirst + C::BM - 1) / C::BM, (count + C::BN - 1) / C::BN);
  if (!t.has(0)) return;
  P prod;
  prod.init(lds, wave, lane);
  typename P::A a, na;
  typename P::B b, nb;
  a.lanes(p.H, wave, lane);
  na = a;
  int few_target[C::NT];
  if constexpr (GATHER) {
    const int* index = few_index + wave * 128;
    b.at([&](int r) { return p.src.row(index[r < count ? r : 0]); }, p.H, wave, lane);
#pragma unroll
    for (int j = 0; j < C::NT; ++j) {
      const int n = (wave % C::N) * (C::NT * 32) + j * 32 + (lane & 31);
      few_target[j] = n < count ? index[64 + n] : -1;
    }
  } else {
    b.lanes(p.H, wave, lane);
  }
  nb = b;
  int tm, tn, um = 0, un = 0;
  t.get(0, tm, tn);
  a.at(p.w, vfirst + tm * C::BM, vend, p.H);
  if constexpr (!GATHER) b.at(p.hc, tn * C::BN, count, p.H);
  prod.load(0, a, b, 0);
  const int wm = wave / C::N, wn = wave % C::N;
  const int vw = wm * (C::MT * 32) + (lane >> 5) * 4;  // the lane's first entry in the tile
  for (;;) {
    const bool more = t.has(1);
    if (more) {
      t.get(1, um, un);
      na.at(p.w, vfirst + um * C::BM, vend, p.H);
      if constexpr (!GATHER) nb.at(p.hc, un * C::BN, count, p.H);
    }
    typename P::Acc acc;
    prod.run(a, b, more, na, nb, acc);

    const int n0 = tn * C::BN, v0 = vfirst + tm * C::BM;
    if (MODE != DZ) {
      // a wave's statistics in its own LDS
      static_assert(C::NT * 32 * 8 <= P::OWN, "room for the waves' statistics");
      floatx2 st[C::NT];
#pragma unroll
      for (int j = 0; j < C::NT; ++j) {
        const int n = n0 + wn * (C::NT * 32) + j * 32 + (lane & 31);
        const int y = GATHER ? few_target[j] : n < count ? p.target[n] : -1;
        const int at = y - v0 - vw;  // the label's entry relative to the lane's first
        if (wave_any(y >= 0 && at >= 0 && at < C::MT * 32 && !(at & 4))) {
#pragma unroll
          for (int i = 0; i < C::MT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (y >= 0 && at == i * 32 + (e >> 2) * 8 + (e & 3)) p.zlabel[n] = acc[i][j][e];
        }
        if (v0 + C::BM > p.V) {
#pragma unroll
          for (int i = 0; i < C::MT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (v0 + vw + i * 32 + (e >> 2) * 8 + (e & 3) >= p.V) acc[i][j][e] = -INFINITY;
        }
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < C::MT; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) m = fmaxf(m, acc[i][j][e]);
        m = xor32_max(m);
        const float base = finite_max(m);
        float l = 0.f;
#pragma unroll
        for (int i = 0; i < C::MT; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float x = fast_exp2((acc[i][j][e] - base) * p.c);
            l += x;
            if (MODE == KEEP) acc[i][j][e] = x;
          }
        l = xor32_sum(l);
        st[j] = floatx2{m, l};
        if (MODE == KEEP && lane < 32 && n < count) p.exps_m[(int64_t)(tm * C::M + wm) * p.rows + n] = m;
      }
      if (MODE == KEEP) {
        static_assert(MODE != KEEP || C::MT * 32 == 128, "a maximum per 128 entries");
        const int64_t col0 = (int64_t)tm * C::BM + wm * (C::MT * 32);
        prod.store(
            [&](int j, int i, int q) {
              return floatx4{acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]};
            },
            [&](int r) {
              const int n = n0 + wn * (C::NT * 32) + r;
              return n < count ? p.exps + (int64_t)n * p.ldv + col0 : nullptr;
            },
            p.ldv - col0);
      }
#pragma unroll
      for (int j = 0; j < C::NT; ++j)
        if (lane < 32) reinterpret_cast<floatx2*>(lds + P::PRIVATE + wave * P::OWN)[j * 32 + lane] = st[j];
      __syncthreads();  // the next writes there follow the next tile's barriers
      for (int nl = threadIdx.x; nl < C::BN; nl += threads_of<C>()) {
        if (n0 + nl < count) {
          RowStat s{-INFINITY, 0.f};
#pragma unroll
          for (int i = 0; i < C::M; ++i) {
            const int w = i * C::N + nl / (C::NT * 32);
            const floatx2 v = reinterpret_cast<const floatx2*>(lds + P::PRIVATE + w * P::OWN)[nl % (C::NT * 32)];
            s = join(s, RowStat{v[0], v[1]}, p.c);
          }
          p.part[(int64_t)tm * p.rows + n0 + nl] = floatx2{s.m, s.l};
        }
      }
    } else {
      floatx4 k[C::NT];
      int at[C::NT];
#pragma unroll
      for (int j = 0; j < C::NT; ++j) {
        const int n = n0 + wn * (C::NT * 32) + j * 32 + (lane & 31);
        k[j] = n < count ? p.coef[n] : floatx4{};
        const int y = n < count ? p.target[n] : -1;
        at[j] = y < 0 ? -1 : y - v0 - vw;
      }
      const int64_t col0 = (int64_t)tm * C::BM + wm * (C::MT * 32);
      prod.store(
          [&](int j, int i, int q) {
            floatx4 d;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              d[e] = k[j][1] * fast_exp2((acc[i][j][q * 4 + e] - k[j][0]) * p.c);
              if (at[j] == i * 32 + q * 8 + e) d[e] += k[j][2];
              if (v0 + vw + i * 32 + q * 8 + e >= vend) d[e] = 0.f;
            }
            return d;
          },
          [&](int r) {
            const int n = n0 + wn * (C::NT * 32) + r;
            return n < count ? p.dz + (int64_t)n * p.ldz + col0 : nullptr;
          },
          p.ldz - col0);
    }
    if (!more) break;
    a = na, b = nb, tm = um, tn = un;
    t.w += t.step;
  }
}

// dz of a range from the exponentials that the forward kept: a pass over both, bound by HBM,
// in place of the range's product.  A kept exponential is half a step of bf16 off; the
// label's own, which the label's gradient is one less than, comes from its fp32 logit.
__global__ __launch_bounds__(256) void head_dz_kernel(HeadParams p) {
  const int count = *p.count;
  const unsigned across = (p.vc + 2047) / 2048, group = blockIdx.x / across;
  const int col = (int)((blockIdx.x - group * across) * 256 + threadIdx.x) * 8;
  if (col >= p.vc) return;
  const int v = p.v0 + col;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t n = (int64_t)group * 4 + u;
    if (n < count) {
      const floatx4 k = p.coef[n];
      const floatx8 x = Vec8<bf16>::load_f32(p.exps + n * p.ldv + v);
      const float f = k[1] * fast_exp2((p.exps_m[(int64_t)(v >> 7) * p.rows + n] - k[0]) * p.c);
      floatx8 d;
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = f * x[e];
      const int at = p.target[n] - v;
      if (at >= 0 && at < 8) {
        const float own = k[1] * fast_exp2((p.zlabel[n] - k[0]) * p.c) + k[2];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e == at) d[e] = own;
      }
      store8<bf16>(p.dz + n * p.ldz + col, d);
    }
  }
}

// The tiles' statistics of each kept row joined: R rows x 1024 / R slots of tiles a
// workgroup.  GATHER: the kept rows found as the products did.
struct HeadJoin {
  HeadSource src;
  const floatx2* part;
  const float* zlabel;  // written for every kept row whose label is in the vocabulary
  const int* count;
  const int* index;
  const int* target;
  float* logprobs;
  floatx2* stats;
  int V, tiles;
  float c, inv_t;
};

template <int R, bool GATHER>
__global__ __launch_bounds__(1024) void head_join_kernel(HeadJoin p) {
  constexpr int SLOTS = 1024 / R;
  __shared__ RowStat red[SLOTS][R + 1];
  __shared__ int few[128];
  __shared__ int few_count;
  const int r = threadIdx.x % R, slot = threadIdx.x / R;
  int count;
  if (GATHER) {
    if (threadIdx.x < 64) {
      const int lane = threadIdx.x, n = p.src.few(lane, p.V, few, few + 64);
      if (lane == 0) few_count = n;
      if (blockIdx.x == 0 && lane < p.src.rows && p.src.labels[lane] == p.src.ignore) {
        p.logprobs[lane] = 0.f;
        p.stats[lane] = floatx2{0.f, 1.f};
      }
    }
    __syncthreads();
    count = few_count;
  } else {
    count = *p.count;
  }
  const int n0 = blockIdx.x * R, n = n0 + r;
  if (n0 >= count) return;
  RowStat s{-INFINITY, 0.f};
  if (n < count) {
#pragma unroll 8
    for (int t = slot; t < p.tiles; t += SLOTS) {
      const floatx2 v = p.part[(int64_t)t * p.src.rows + n];
      s = join(s, RowStat{v[0], v[1]}, p.c);
    }
  }
  red[slot][r] = s;
  __syncthreads();
  for (int k = SLOTS / 2; k >= 1; k >>= 1) {
    if (slot < k) red[slot][r] = join(red[slot][r], red[slot + k][r], p.c);
    __syncthreads();
  }
  if (slot == 0 && n < count) {
    s = red[0][r];
    const int row = GATHER ? few[n] : p.index[n], y = GATHER ? few[64 + n] : p.target[n];
    p.logprobs[row] = y < 0 ? __builtin_nanf("") : (p.zlabel[n] - s.m) * p.inv_t - logf(s.l);
    p.stats[row] = floatx2{s.m, s.l};
  }
}

// dw[v][h] = sum over kept tokens of dz[n][v] hc[n][h], v0 <= v < v0 + vc: both operands have
// the depth (tokens) as their slow axis.
__global__ __launch_bounds__(threads_of<Wide>()) void head_dw_kernel(HeadParams p) {
  typedef Wide C;
  typedef Product<C, false, false> P;
  extern __shared__ __align__(1024) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int count = __builtin_amdgcn_readfirstlane(*p.count);
  Tiles t((p.H + C::BM - 1) / C::BM, (p.vc + C::BN - 1) / C::BN);
  if (!t.has(0)) return;
  P prod;
  prod.init(lds, wave, lane);
  P::A a, na;
  P::B b, nb;
  a.lanes(p.H, wave, lane);
  b.lanes(p.ldz, wave, lane);
  na = a, nb = b;
  int tm, tn, um = 0, un = 0;
  t.get(0, tm, tn);
  a.at(p.hc, tm * C::BM, p.H, count);
  b.at(p.dz, tn * C::BN, p.vc, count);
  if (count > 0) prod.load(0, a, b, 0);
  const int wm = wave / C::N, wn = wave % C::N;
  for (;;) {
    const bool more = t.has(1);
    if (more) {
      t.get(1, um, un);
      na.at(p.hc, um * C::BM, p.H, count);
      nb.at(p.dz, un * C::BN, p.vc, count);
    }
    P::Acc acc;
    prod.run(a, b, more, na, nb, acc);
    const int h0 = tm * C::BM + wm * (C::MT * 32), v0 = tn * C::BN + wn * (C::NT * 32);
    prod.store(
        [&](int j, int i, int q) {
          return floatx4{acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]};
        },
        [&](int r) { return v0 + r < p.vc ? p.dw + (int64_t)(p.v0 + v0 + r) * p.H + h0 : nullptr; }, p.H - h0);
    if (!more) break;
    a = na, b = nb, tm = um, tn = un;
    t.w += t.step;
  }
}

// The depth of dh's products (vocabulary) is long and its tiles may be few: it is split over
// slabs, each with sums of its own, which the last launch adds in order.  As many as fill
// the CUs' last round best, less a little for each one's sums.
__host__ __device__ __forceinline__ int head_slabs(int64_t tiles, int vmax) {
  const int64_t deep = (vmax + 8 * HD_BK - 1) / (8 * HD_BK);  // at least 8 steps each
  int64_t best = 1, most = 0, rounds_of = 1;  // whole numbers: every kernel finds the same
  for (int64_t s = 1; s <= 8; ++s) {
    const int64_t n = tiles * s, rounds = (n + HD_CUS - 1) / HD_CUS, use = n * (100 - s);
    if (s > 1 && n > 4 * HD_CUS) break;
    if (use * rounds_of > most * rounds) most = use, rounds_of = rounds, best = s;
  }
  if (tiles * 8 <= HD_CUS) best = HD_CUS / tiles;
  if (best > deep) best = deep;
  return best < 1 ? 1 : (int)best;
}

// dh[n][h] (+)= sum over this range's v of dz[n][v] w[v][h], fp32.
template <class C>
__global__ __launch_bounds__(threads_of<C>()) void head_dh_kernel(HeadParams p) {
  typedef Product<C, false, true> P;
  extern __shared__ __align__(1024) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int count = __builtin_amdgcn_readfirstlane(*p.count);
  const int nh = (p.H + C::BM - 1) / C::BM, nn = (count + C::BN - 1) / C::BN;
  if (nn == 0) return;
  const int slabs = head_slabs((int64_t)nh * nn, p.vmax);
  const int per = ((p.vc + slabs - 1) / slabs + HD_BK - 1) / HD_BK * HD_BK;
  Tiles t(nh, nn * slabs);
  if (!t.has(0)) return;
  P prod;
  prod.init(lds, wave, lane);
  typename P::A a, na;
  typename P::B b, nb;
  a.lanes(p.H, wave, lane);
  b.lanes(p.ldz, wave, lane);
  na = a, nb = b;
  auto place = [&](int th, int rest, typename P::A& x, typename P::B& y) {
    const int slab = rest / nn, tn = rest - slab * nn, k0 = slab * per;
    const int left = p.vc - k0, depth = left < 0 ? 0 : left < per ? left : per;
    x.at(p.w + (int64_t)(p.v0 + (depth ? k0 : 0)) * p.H, th * C::BM, p.H, depth);
    y.at(p.dz + (depth ? k0 : 0), tn * C::BN, count, depth);
  };
  int th, rest, uh = 0, us = 0;
  t.get(0, th, rest);
  place(th, rest, a, b);
  if (a.depth) prod.load(0, a, b, 0);
  const int wm = wave / C::N, wn = wave % C::N;
  for (;;) {
    const bool more = t.has(1);
    if (more) {
      t.get(1, uh, us);
      place(uh, us, na, nb);
    }
    typename P::Acc acc;
    prod.run(a, b, more && na.depth, na, nb, acc);
    if (!a.depth && more && na.depth) prod.load(prod.cur, na, nb, 0);  // nothing ran that would have begun it
    const int slab = rest / nn, tn = rest - slab * nn;
    if (a.depth || !p.add) {
#pragma unroll
      for (int j = 0; j < C::NT; ++j) {
        const int n = tn * C::BN + wn * (C::NT * 32) + j * 32 + (lane & 31);
        if (n < count) {
#pragma unroll
          for (int i = 0; i < C::MT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int h = th * C::BM + wm * (C::MT * 32) + i * 32 + q * 8 + (lane >> 5) * 4;
              if (h < p.H) {
                floatx4* o = reinterpret_cast<floatx4*>(p.dh + ((int64_t)slab * nn * C::BN + n) * p.H + h);
                floatx4 d{acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]};
                if (p.add) d += *o;
                *o = d;
              }
            }
        }
      }
    }
    if (!more) break;
    a = na, b = nb, th = uh, rest = us;
    t.w += t.step;
  }
}

// dhidden: the slabs' sums, rounded, in the rows' own places; zeros in ignored rows.
struct HeadOut {
  const float* dh;
  const int* count;
  const int* pos;
  bf16* out;
  int64_t rows;
  int H, bm, bn, vmax;
};
__global__ __launch_bounds__(256) void head_dh_out_kernel(HeadOut p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int ch = p.H / 8;
  if (i >= p.rows * ch) return;
  const int64_t row = i / ch;
  const int c = (int)(i - row * ch), place = p.pos[row];
  floatx8 s{};
  if (place >= 0) {
    const int nn = (*p.count + p.bn - 1) / p.bn;
    const int slabs = head_slabs((int64_t)((p.H + p.bm - 1) / p.bm) * nn, p.vmax);
    const int64_t stride = (int64_t)nn * p.bn * p.H;
    const float* src = p.dh + (int64_t)place * p.H + c * 8;
    s = Vec8<float>::load_f32(src);
    for (int k = 1; k < slabs; ++k) s += Vec8<float>::load_f32(src + k * stride);
  }
  store8<bf16>(p.out + row * p.H + c * 8, s);
}

}  // namespace nq

using namespace nq;

static int64_t pad256(int64_t n) { return (n + 255) / 256 * 256; }

// Which tile: Few reads the weights once for up to 64 tokens.
static bool head_few(int64_t rows) { return rows <= Few::BN; }

// Where each piece of a workspace lies.
struct HeadSpace {
  int64_t count, pos, index, target, zlabel, coef, hc, part, dz, dh, total;
  int64_t ldz;
  int vc;
};

// The largest range's dz; above 2^21 rows more, as a range has at least the 256 entries of a tile.
constexpr int64_t HD_DZ_BYTES = (int64_t)1 << 30;

// What a forward keeps for its backward: the labels' logits, the maxima of each 128 entries
// and the exponentials.  Up to 4 GiB (1.4% of the memory); beyond 64 rows, as a product of so few
// is bound by the weights' bytes, of which this would save one pass in four; and from a width of
// 256, below which the product takes less than the exponentials' bytes (forward and backward
// of 8192 rows against 151936 entries, kept and repeated: width 128 2978 and 2865 us, 256
// 3437 and 3552, 1024 7771 and 9441; 2048 rows 809 and 755, 910 and 918, 2030 and 2428).
struct HeadKept {
  int64_t zlabel, m, exps, total, ldv;
};
constexpr int64_t HD_KEPT_BYTES = (int64_t)4 << 30;

static HeadKept head_kept(int64_t rows, int V, int H) {
  HeadKept k{};
  k.ldv = (V + 7) / 8 * 8;
  k.m = pad256(rows * 4);
  k.exps = k.m + pad256(rows * ((V + 255) / 256 * 2) * 4);
  k.total = k.exps + pad256(rows * k.ldv * 2);
  if (head_few(rows) || H < 256 || k.total > HD_KEPT_BYTES) k.total = 0;
  return k;
}

static HeadSpace head_space(int64_t rows, int V, int H, bool backward) {
  HeadSpace s{};
  const int64_t bm = head_few(rows) ? Few::BM : Wide::BM, bn = head_few(rows) ? Few::BN : Wide::BN;
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
    s.part = take(rows * ((V + bm - 1) / bm) * 8);
  } else {
    s.coef = take(rows * 16);
    // ranges of whole tiles, as many as fill the CUs in whole rounds of dw's
    const int64_t nh = (H + 255) / 256, unit = (nh < HD_CUS ? HD_CUS / nh : 1) * 256;
    int64_t most = HD_DZ_BYTES / (rows * 2) / 256 * 256;
    most = most < 256 ? 256 : most < unit ? most : most / unit * unit;
    const int64_t ranges = (V + most - 1) / most, each = ((V + ranges - 1) / ranges + unit - 1) / unit * unit;
    if (each < most) most = each;
    s.vc = (int)(most < V ? most : V);
    s.ldz = (s.vc + 7) / 8 * 8;
    s.dz = take(rows * s.ldz * 2);
    // as many slabs as any number of kept rows takes
    const int64_t tiles = ((rows + bn - 1) / bn) * ((H + bm - 1) / bm);
    int64_t slots = 8 * tiles < HD_CUS ? HD_CUS : 8 * tiles;
    if (slots > 4 * HD_CUS) slots = 4 * HD_CUS;
    if (slots < tiles) slots = tiles;
    s.dh = take(slots * bm * bn * 4);
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
extern "C" int64_t nq_linear_logprobs_kept_bytes(int64_t rows, int V, int H) {
  return head_sizes_ok(rows, V, H) ? head_kept(rows, V, H).total : 0;
}
extern "C" int64_t nq_linear_logprobs_bwd_workspace_bytes(int64_t rows, int V, int H) {
  return head_sizes_ok(rows, V, H) ? head_space(rows, V, H, true).total : 0;
}

static int head_check(const void* hidden, int64_t bs, int64_t rs, const void* weight, const int64_t* labels,
                      const void* stats, const void* kept, int64_t kept_bytes, const void* workspace,
                      int64_t workspace_bytes, int64_t B, int64_t S, int V, int H, float temperature, bool backward) {
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
  const int64_t keeps = head_kept(B * S, V, H).total;
  if (kept && (!keeps || kept_bytes < keeps || (reinterpret_cast<uintptr_t>(kept) & 255u)))
    return nq_fail(NQ_ERR_WORKSPACE, "kept too small or not 256-byte aligned: %lld bytes, need %lld (0: none is kept)",
                   (long long)kept_bytes, (long long)keeps);
  const int64_t need = head_space(B * S, V, H, backward).total;
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return nq_fail(NQ_ERR_WORKSPACE, "workspace too small or not 256-byte aligned: %lld bytes, need %lld",
                   (long long)workspace_bytes, (long long)need);
  return NQ_OK;
}

static void head_kept_at(void* kept, HeadParams* p) {
  const HeadKept k = head_kept(p->rows, p->V, p->H);
  char* at = reinterpret_cast<char*>(kept);
  p->zlabel = reinterpret_cast<float*>(at + k.zlabel), p->exps_m = reinterpret_cast<float*>(at + k.m);
  p->exps = reinterpret_cast<bf16*>(at + k.exps), p->ldv = k.ldv;
}

// A launch with P's dynamic LDS (the attribute belongs to the kernel on the device; setting it
// again is cheap).
template <class P, typename K>
static int head_launch(K kernel, int grid, int threads, hipStream_t st, const HeadParams& p) {
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, P::LDS);
  if (e != hipSuccess) return nq_check_launch(e);
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3((unsigned)threads), P::LDS, st, p);
  return nq_check_launch(hipGetLastError());
}
static void launch_rows(HeadRows& r, hipStream_t st) {
  const int64_t rows = r.src.rows;
  r.each = rows <= 16 * 2048 ? 16 : ((rows + 2047) / 2048 + 63) / 64 * 64;
  hipLaunchKernelGGL(head_rows_kernel, dim3((unsigned)((rows + r.each - 1) / r.each)), dim3(256), 0, st, r);
}
template <class C, int MODE, bool GATHER = false, bool STREAM = false>
static int launch_logits(int64_t tiles, hipStream_t st, const HeadParams& p) {
  return head_launch<Product<C, true, true, GATHER, STREAM>>(head_logits_kernel<C, MODE, GATHER, STREAM>,
                                                             head_grid<C>(tiles), threads_of<C>(), st, p);
}
template <class C>
static int launch_dh(int64_t tiles, hipStream_t st, const HeadParams& p) {
  return head_launch<Product<C, false, true>>(head_dh_kernel<C>, head_grid<C>(tiles), threads_of<C>(), st, p);
}

extern "C" int nq_linear_logprobs(const void* hidden, int64_t batch_stride, int64_t row_stride, const void* weight,
                                  const int64_t* labels, float* logprobs, float* stats, void* kept,
                                  int64_t kept_bytes, void* workspace, int64_t workspace_bytes, int64_t B, int64_t S,
                                  int V, int H, float temperature, int64_t ignore_index, void* stream) {
  nq_clear_error();
  if (int rc = head_check(hidden, batch_stride, row_stride, weight, labels, stats, kept, kept_bytes, workspace,
                          workspace_bytes, B, S, V, H, temperature, false))
    return rc;
  if (!logprobs || (reinterpret_cast<uintptr_t>(logprobs) & 3u))
    return nq_fail(NQ_ERR_INVALID, "logprobs is required, aligned to fp32");
  const int64_t rows = B * S;
  const HeadSpace s = head_space(rows, V, H, false);
  char* ws = reinterpret_cast<char*>(workspace);
  const float inv = 1.f / temperature;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  HeadRows r{};
  r.src = HeadSource{reinterpret_cast<const bf16*>(hidden), batch_stride, row_stride, S, labels, rows, ignore_index};
  r.H = H, r.V = V;
  r.count = reinterpret_cast<int*>(ws + s.count), r.pos = reinterpret_cast<int*>(ws + s.pos);
  r.index = reinterpret_cast<int*>(ws + s.index), r.target = reinterpret_cast<int*>(ws + s.target);
  r.hc = reinterpret_cast<bf16*>(ws + s.hc);
  r.logprobs = logprobs, r.stats = reinterpret_cast<floatx2*>(stats);
  HeadParams p{};
  p.src = r.src, p.hc = r.hc, p.w = reinterpret_cast<const bf16*>(weight), p.rows = rows, p.V = V, p.H = H;
  p.count = r.count, p.target = r.target, p.c = inv * kLog2e;
  p.part = reinterpret_cast<floatx2*>(ws + s.part), p.zlabel = reinterpret_cast<float*>(ws + s.zlabel);
  if (kept) head_kept_at(kept, &p);
  const bool few = head_few(rows);
  const int bm = few ? Few::BM : Wide::BM, bn = few ? Few::BN : Wide::BN, tiles = (V + bm - 1) / bm;
  const int64_t all = tiles * ((rows + bn - 1) / bn);
  if (all > INT32_MAX / 2) return nq_fail(NQ_ERR_UNSUPPORTED, "too many tiles for one launch");
  const HeadJoin j{r.src, p.part, p.zlabel, r.count, r.index, r.target, logprobs, r.stats, V, tiles, p.c, inv};
  if (few) {
    // 33 rows of 1024 against 151936 entries: 69 us with the gathering launch, 60 without it, 54
    // with weights that the 256 MB cache cannot hold loaded past it
    const bool past = (int64_t)V * H * 2 > ((int64_t)256 << 20);
    if (int rc = past ? launch_logits<Few, STATS, true, true>(all, st, p) : launch_logits<Few, STATS, true>(all, st, p))
      return rc;
    hipLaunchKernelGGL((head_join_kernel<4, true>), dim3((unsigned)((rows + 3) / 4)), dim3(1024), 0, st, j);
  } else {
    launch_rows(r, st);
    if (int rc = kept ? launch_logits<Wide, KEEP>(all, st, p) : launch_logits<Wide, STATS>(all, st, p)) return rc;
    hipLaunchKernelGGL((head_join_kernel<16, false>), dim3((unsigned)((rows + 15) / 16)), dim3(1024), 0, st, j);
  }
  return nq_check_launch(hipGetLastError());
}

extern "C" int nq_linear_logprobs_bwd(const void* hidden, int64_t batch_stride, int64_t row_stride, const void* weight,
                                      const int64_t* labels, const float* stats, const void* kept,
                                      int64_t kept_bytes, const float* dlogprobs, void* dhidden, void* dweight,
                                      void* workspace, int64_t workspace_bytes, int64_t B, int64_t S, int V, int H,
                                      float temperature, int64_t ignore_index, void* stream) {
  nq_clear_error();
  if (int rc = head_check(hidden, batch_stride, row_stride, weight, labels, stats, kept, kept_bytes, workspace,
                          workspace_bytes, B, S, V, H, temperature, true))
    return rc;
  if (!dlogprobs || (reinterpret_cast<uintptr_t>(dlogprobs) & 3u) || !nq_aligned16(dhidden) || !nq_aligned16(dweight))
    return nq_fail(NQ_ERR_INVALID, "dlogprobs is required, and gradients must be 16-byte aligned");
  if (!dhidden && !dweight) return NQ_OK;
  const int64_t rows = B * S;
  const HeadSpace s = head_space(rows, V, H, true);
  const bool few = head_few(rows);
  const int bm = few ? Few::BM : Wide::BM, bn = few ? Few::BN : Wide::BN, nh = (H + bm - 1) / bm;
  const int64_t nn = (rows + bn - 1) / bn, nw = (H + Wide::BM - 1) / Wide::BM;
  if (((int64_t)s.vc / bm + 1) * nn > INT32_MAX / 2 || nn * nh * HD_CUS > INT32_MAX / 2 ||
      ((int64_t)s.vc / Wide::BN + 1) * nw > INT32_MAX / 2)
    return nq_fail(NQ_ERR_UNSUPPORTED, "too many tiles for one launch");
  if (dhidden && rows * (H / 8) > UINT32_MAX - 255)  // a launch has fewer than 2^32 threads
    return nq_fail(NQ_ERR_UNSUPPORTED, "too many elements of hidden states for one launch");
  char* ws = reinterpret_cast<char*>(workspace);
  const float inv = 1.f / temperature;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  HeadRows r{};
  r.src = HeadSource{reinterpret_cast<const bf16*>(hidden), batch_stride, row_stride, S, labels, rows, ignore_index};
  r.H = H, r.V = V;
  r.count = reinterpret_cast<int*>(ws + s.count), r.pos = reinterpret_cast<int*>(ws + s.pos);
  r.index = reinterpret_cast<int*>(ws + s.index), r.target = reinterpret_cast<int*>(ws + s.target);
  r.hc = reinterpret_cast<bf16*>(ws + s.hc);
  r.stats = reinterpret_cast<floatx2*>(const_cast<float*>(stats)), r.dy = dlogprobs;
  r.coef = reinterpret_cast<floatx4*>(ws + s.coef), r.inv_t = inv;
  launch_rows(r, st);
  HeadParams p{};
  p.hc = r.hc, p.w = reinterpret_cast<const bf16*>(weight), p.rows = rows, p.V = V, p.H = H;
  p.count = r.count, p.target = r.target, p.c = inv * kLog2e, p.coef = r.coef;
  p.dz = reinterpret_cast<bf16*>(ws + s.dz), p.ldz = s.ldz;
  if (kept) head_kept_at(const_cast<void*>(kept), &p);
  p.dw = reinterpret_cast<bf16*>(dweight), p.dh = reinterpret_cast<float*>(ws + s.dh), p.vmax = s.vc;
  for (int v0 = 0; v0 < V; v0 += s.vc) {
    p.v0 = v0, p.vc = V - v0 < s.vc ? V - v0 : s.vc, p.add = v0 > 0;
    const int64_t logits = (p.vc + bm - 1) / bm * nn;
    int rc = NQ_OK;
    if (kept) {
      // at most 2^31 kept values, 8192 a workgroup
      hipLaunchKernelGGL(head_dz_kernel, dim3((unsigned)((p.vc + 2047) / 2048 * ((rows + 3) / 4))), dim3(256), 0, st, p);
    } else {
      rc = few ? launch_logits<Few, DZ>(logits, st, p) : launch_logits<Wide, DZ>(logits, st, p);
    }
    // as many workgroups as the CUs hold: how many tiles there are goes by the kept rows
    if (!rc && dhidden) rc = few ? launch_dh<Few>(INT32_MAX / 2, st, p) : launch_dh<Wide>(INT32_MAX / 2, st, p);
    if (!rc && dweight) {
      const int64_t tiles = nw * ((p.vc + Wide::BN - 1) / Wide::BN);
      rc = head_launch<Product<Wide, false, false>>(head_dw_kernel, head_grid<Wide>(tiles), threads_of<Wide>(), st, p);
    }
    if (rc) return rc;
  }
  if (dhidden) {
    const HeadOut o{p.dh, r.count, r.pos, reinterpret_cast<bf16*>(dhidden), rows, H, bm, bn, s.vc};
    const int64_t n = rows * (H / 8);
    hipLaunchKernelGGL(head_dh_out_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, o);
  }
  return nq_check_launch(hipGetLastError());
}
