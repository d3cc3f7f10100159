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
// the end; K stays in registers while the rows pass.
struct KeyWeightParams {
  const bf16* q;
  int64_t qsb, qsh, qss;
  const void* pool;       // 4-bit pages (strides in bytes) or bf16 ones (elements)
  int64_t psb, psh, pss;  // page, head and (bf16) row strides
  int npages;
  const int32_t* bt;
  int64_t bts;
  int page;
  const int32_t* lens;
  const float* lse;  // (B, Hq, S)
  float* w;
  int64_t wsb, wsh;
  int add;           // add to w, else write it
  int Hq, Hkv, G, S, max_len, causal;
  float scale_log2;
};

constexpr int KW_KEYS = 64;              // keys of a wave
constexpr int KW_BLOCK = 4 * KW_KEYS;    // of a workgroup

template <int D, bool FOUR>
__global__ void __launch_bounds__(256) key_weights_kernel(KeyWeightParams p) {
  using F = Kv4<D>;
  constexpr int NDQ = D / 32;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, grp = lane >> 4;
  const int b = blockIdx.z, kvh = blockIdx.y;
  const int k0 = blockIdx.x * KW_BLOCK + wave * KW_KEYS;
  const int len = ld_uniform(p.lens, b);
  float* w = p.w + b * p.wsb + kvh * p.wsh;
  if (k0 >= p.max_len) return;
  const bool bad_len = len < 0 || len > p.max_len;
  if (bad_len || k0 >= len) {  // no keys here
    const int t = k0 + lane;
    if (!p.add && t < p.max_len) w[t] = bad_len ? __builtin_nanf("") : 0.f;
    return;
  }
  // K: lane (key c16, slot grp) holds elements grp D/4 + 8 i + j, as the decode
  bf16x8 k[KW_KEYS / 16][NDQ];
  bool lost[KW_KEYS / 32];
#pragma unroll
  for (int half = 0; half < KW_KEYS / 32; ++half) {
    const int first = k0 + half * 32;  // 32 keys never cross a page
    int pid = first < len ? ld_uniform(p.bt, b * p.bts + first / p.page) : 0;
    lost[half] = (uint32_t)pid >= (uint32_t)p.npages;
    if (lost[half]) pid = 0;
    const int rel = first % p.page;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int row = rel + t * 16 + c16;
      if constexpr (FOUR) {
        const unsigned char* rec = reinterpret_cast<const unsigned char*>(p.pool) + pid * p.psb + kvh * p.psh;
        const uint32_t* codes = reinterpret_cast<const uint32_t*>(rec + row * F::CB) + grp * NDQ;
        const float scale = kv4_scale(rec[F::k_scales(p.page) + row * F::SB + grp * (D / 4) / 32]);
#pragma unroll
        for (int i = 0; i < NDQ; ++i) k[half * 2 + t][i] = kv4_bf16x8(codes[i], scale);
      } else {
        const bf16* src = reinterpret_cast<const bf16*>(p.pool) + pid * p.psb + kvh * p.psh + row * p.pss + grp * (D / 4);
#pragma unroll
        for (int i = 0; i < NDQ; ++i) k[half * 2 + t][i] = Vec8<bf16>::load_bf16(src + i * 8);
      }
    }
  }
  const int R = p.S * p.G;
  const int hidden = p.causal ? len - p.S : 0x7fffffff;  // query s sees keys up to hidden + s
  int r0 = 0;
  if (p.causal && k0 > hidden) {
    const int64_t first = (int64_t)(k0 - hidden) * p.G;  // rows before it see none of the wave's keys
    r0 = (int)(first < R ? first : R) & ~15;
  }
  float acc[KW_KEYS / 16];
#pragma unroll
  for (int t = 0; t < KW_KEYS / 16; ++t) acc[t] = 0.f;
  for (; r0 < R; r0 += 16) {
    const int r = r0 + c16;
    const bool valid = r < R;
    const int s = (valid ? r : 0) / p.G, g = (valid ? r : 0) % p.G;
    const bf16* qrow = p.q + b * p.qsb + (int64_t)(kvh * p.G + g) * p.qsh + s * p.qss + grp * (D / 4);
    bf16x8 q[NDQ];
#pragma unroll
    for (int i = 0; i < NDQ; ++i) q[i] = Vec8<bf16>::load_bf16(qrow + i * 8);
    float off[4];
    int last[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int ri = r0 + grp * 4 + i, ok = ri < R;
      const int si = (ok ? ri : 0) / p.G, gi = (ok ? ri : 0) % p.G;
      const float v = p.lse[((int64_t)b * p.Hq + kvh * p.G + gi) * p.S + si];
      off[i] = !ok || v == -INFINITY ? INFINITY : v * kLog2e;  // a row without keys, or past the last: no weight
      last[i] = p.causal ? hidden + si : 0x7fffffff;
    }
#pragma unroll
    for (int t = 0; t < KW_KEYS / 16; ++t) {
      floatx4 sc = floatx4{};
#pragma unroll
      for (int i = 0; i < NDQ; ++i) sc = mfma16(q[i], k[t][i], sc);
      const int key = k0 + t * 16 + c16;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = fast_exp2(__builtin_fmaf(sc[i], p.scale_log2, -off[i]));
        acc[t] += key <= last[i] && off[i] != INFINITY ? e : 0.f;
      }
    }
  }
#pragma unroll
  for (int t = 0; t < KW_KEYS / 16; ++t) {
    acc[t] += shfl_xor_f(acc[t], 16);
    acc[t] = xor32_sum(acc[t]);
    if (lost[t / 2]) acc[t] = __builtin_nanf("");
  }
  const float mine = grp == 0 ? acc[0] : grp == 1 ? acc[1] : grp == 2 ? acc[2] : acc[3];
  const int t = k0 + lane;
  if (t < len) w[t] = p.add ? w[t] + mine : mine;
  else if (!p.add && t < p.max_len) w[t] = 0.f;
}

// ---------------------------------------------------------------- selection
// The rows that a (sequence, kv head) keeps: the first `first`, the last `recent`, and of
// the rows between them the `keep - first - recent` heaviest, equal weights by the lower
// index; in ascending order.  A workgroup of 16 waves per (sequence, head) finds the
// smallest kept weight by a radix select over its bits (11 + 11 + 10, a histogram in LDS
// for each), then writes the kept rows in order: each wave takes a contiguous share, and
// its place in the output follows from the counts of the waves before it.
struct SelectParams {
  const float* w;
  int64_t wsb, wsh;
  const int32_t* lens;
  int32_t* kept;  // (B, Hkv, keep)
  int Hkv, W, keep, recent, first;
};

constexpr int SEL_THREADS = 1024, SEL_WAVES = SEL_THREADS / 64, SEL_BINS = 2048;

// Orders as the weights do: NaN above everything, -0 as +0.
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
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* w = p.w + b * p.wsb + h * p.wsh;
  int32_t* kept = p.kept + (int64_t)blockIdx.x * p.keep;
  int n = p.lens[b];
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

  uint32_t prefix = 0;  // the bits of the smallest kept key found so far
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < SEL_BINS; i += SEL_THREADS) hist[i] = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += SEL_THREADS) {
      const uint32_t key = weight_key(w[i]);
      if (pass == 0 || key >> (shift + bits) == prefix >> (shift + bits))
        atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1)], 1u);
    }
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
  const int share = ((hi - lo + SEL_THREADS - 1) / SEL_THREADS) * 64;
  const int begin = min(lo + wave * share, hi), end = min(begin + share, hi);
  uint32_t more = 0, same = 0;
  for (int i = begin; i < end; i += 64) {
    const uint32_t key = i + lane < end ? weight_key(w[i + lane]) : 0;
    more += __popcll(__builtin_amdgcn_ballot_w64(i + lane < end && key > prefix));
    same += __popcll(__builtin_amdgcn_ballot_w64(i + lane < end && key == prefix));
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
  const uint64_t below = lane == 0 ? 0 : ~0ull >> (64 - lane);
  for (int i = begin; i < end; i += 64) {
    const bool in = i + lane < end;
    const uint32_t key = in ? weight_key(w[i + lane]) : 0;
    const uint64_t eq = __builtin_amdgcn_ballot_w64(in && key == prefix);
    const bool take = in && (key > prefix || (key == prefix && ties + __popcll(eq & below) < room));
    const uint64_t taken = __builtin_amdgcn_ballot_w64(take);
    const uint32_t to = at + __popcll(taken & below);
    if (take && to < (uint32_t)(p.keep - p.recent)) kept[to] = i + lane;  // (weights that change meanwhile)
    at += __popcll(taken);
    ties += __popcll(eq);
  }
}

// ---------------------------------------------------------------- moving rows
// Row kept[b, h, i] of a sequence's pages to row i of its new pages, for every part of a
// row (K and V rows; of 4-bit pages codes and scales), and its weight.  A thread per
// piece of a row; HBM-bound, each kept row read and written once.
struct RowPart {
  int64_t off;         // of the part within a page's head (bytes)
  int stride, bytes;   // between rows, of a row
  int pool;            // which pool
};
struct CompactParams {
  unsigned char* pool[2];
  int64_t psb[2], psh[2];  // page and head strides (bytes)
  RowPart part[4];
  int parts, unit[4], pieces[4];  // bytes of a piece, pieces of a row's part
  int per_row;                    // pieces of a row, the weight's included
  int npages, page, cols, new_cols;
  const int32_t *bt, *new_bt;
  int64_t bts, nbts;
  const int32_t* kept;
  const float* w;
  float* w_out;
  int64_t wsb, wsh;
  int Hkv, keep, W;
};

__global__ void __launch_bounds__(256) compact_rows_kernel(CompactParams p) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t moves = (int64_t)p.keep * p.per_row;
  if (id >= moves) {  // weights of the rows that are no more
    const int64_t t = id - moves + p.keep;
    if (p.w_out && t < p.W) p.w_out[b * p.wsb + h * p.wsh + t] = 0.f;
    return;
  }
  const int i = (int)(id / p.per_row);
  int piece = (int)(id % p.per_row);
  const int j = p.kept[((int64_t)b * p.Hkv + h) * p.keep + i];
  const bool real = j >= 0 && j < p.cols * (int64_t)p.page;
  int c = 0;
  while (c < p.parts && piece >= p.pieces[c]) piece -= p.pieces[c++];
  if (c == p.parts) {
    if (p.w_out) p.w_out[b * p.wsb + h * p.wsh + i] = real && j < p.W ? p.w[b * p.wsb + h * p.wsh + j] : 0.f;
    return;
  }
  if (!real) return;
  const int from = p.bt[b * p.bts + j / p.page], to = p.new_bt[b * p.nbts + i / p.page];
  if ((uint32_t)from >= (uint32_t)p.npages || (uint32_t)to >= (uint32_t)p.npages) return;  // not pages of the pool
  const RowPart& q = p.part[c];
  unsigned char* base = p.pool[q.pool] + h * p.psh[q.pool] + q.off;
  const int64_t at = (int64_t)piece * p.unit[c];
  const unsigned char* src = base + from * p.psb[q.pool] + (int64_t)(j % p.page) * q.stride + at;
  unsigned char* dst = base + to * p.psb[q.pool] + (int64_t)(i % p.page) * q.stride + at;
  switch (p.unit[c]) {
    case 16: *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src); break;
    case 4: *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(src); break;
    case 2: *reinterpret_cast<uint16_t*>(dst) = *reinterpret_cast<const uint16_t*>(src); break;
    default: *dst = *src;
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

extern "C" int nq_key_weights(const void* q, const int64_t* q_strides, const void* k_pool,
                              const int64_t* pool_strides, int four_bit, int num_pages, const int32_t* block_table,
                              int64_t bt_stride, int bt_cols, int page_size, const int32_t* lens, const float* lse,
                              float* weights, const int64_t* weight_strides, int accumulate, int B, int Hq, int Hkv,
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
  for (int i = 0; i < (four_bit ? 2 : 3); ++i)
    if (pool_strides[i] % (four_bit ? 16 : 8)) return nq_fail(NQ_ERR_INVALID, "pool strides must be multiples of 16 bytes");
  if (B > 65535 || Hkv > 65535 || (int64_t)S * (Hq / Hkv) > 0x3fffffff)
    return nq_fail(NQ_ERR_UNSUPPORTED, "at most 65535 sequences and kv heads and 2^30 query rows a kv head");
  KeyWeightParams p{};
  p.q = reinterpret_cast<const bf16*>(q); p.qsb = q_strides[0]; p.qsh = q_strides[1]; p.qss = q_strides[2];
  p.pool = k_pool; p.psb = pool_strides[0]; p.psh = pool_strides[1]; p.pss = four_bit ? 0 : pool_strides[2];
  p.npages = num_pages; p.bt = block_table; p.bts = bt_stride; p.page = page_size;
  p.lens = lens; p.lse = lse; p.w = weights; p.wsb = weight_strides[0]; p.wsh = weight_strides[1];
  p.add = accumulate != 0; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.S = S; p.max_len = max_len;
  p.causal = causal != 0 && S > 1;
  p.scale_log2 = (sm_scale > 0.f ? sm_scale : 1.0f / sqrtf((float)D)) * kLog2e;
  const dim3 grid((unsigned)((max_len + KW_BLOCK - 1) / KW_BLOCK), (unsigned)Hkv, (unsigned)B);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return nq_check_launch(with_head_dim(D, [&](auto dc) {
    constexpr int DD = decltype(dc)::value;
    if (four_bit) hipLaunchKernelGGL((key_weights_kernel<DD, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((key_weights_kernel<DD, false>), grid, dim3(256), 0, st, p);
    return hipGetLastError();
  }));
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
  if ((int64_t)B * Hkv > 0x7fffffff) return nq_fail(NQ_ERR_UNSUPPORTED, "more than 2^31 (sequence, kv head) rows");
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
    p.parts = 4;
    p.part[0] = RowPart{0, cb, cb, 0};
    p.part[1] = RowPart{(int64_t)page_size * cb, cb, cb, 0};
    p.part[2] = RowPart{(int64_t)page_size * 2 * cb, sb, sb, 0};
    p.part[3] = RowPart{(int64_t)page_size * (2 * cb + sb), sb, sb, 0};
  } else {
    if (row_bytes <= 0 || row_bytes % 16 || row_bytes > (1 << 20) || k_strides[2] < row_bytes || v_strides[2] < row_bytes ||
        k_strides[2] > (1 << 30) || v_strides[2] > (1 << 30))
      return nq_fail(NQ_ERR_INVALID, "rows must be multiples of 16 bytes that do not overlap, got %d", row_bytes);
    p.parts = 2;
    p.part[0] = RowPart{0, (int)k_strides[2], row_bytes, 0};
    p.part[1] = RowPart{0, (int)v_strides[2], row_bytes, 1};
    p.pool[1] = reinterpret_cast<unsigned char*>(v_pool); p.psb[1] = v_strides[0]; p.psh[1] = v_strides[1];
  }
  p.pool[0] = reinterpret_cast<unsigned char*>(k_pool); p.psb[0] = k_strides[0]; p.psh[0] = k_strides[1];
  for (int i = 0; i < (four ? 1 : 2); ++i) {
    if (!nq_aligned16(p.pool[i]) || p.psb[i] % 16 || p.psh[i] % 16 || (!four && (i ? v_strides : k_strides)[2] % 16))
      return nq_fail(NQ_ERR_INVALID, "the pools and their strides must be multiples of 16 bytes");
  }
  p.per_row = 1;
  for (int i = 0; i < p.parts; ++i) {
    const int n = p.part[i].bytes;
    p.unit[i] = n % 16 == 0 ? 16 : n % 4 == 0 ? 4 : n % 2 == 0 ? 2 : 1;
    p.pieces[i] = n / p.unit[i];
    p.per_row += p.pieces[i];
  }
  p.npages = num_pages; p.page = page_size; p.cols = bt_cols; p.new_cols = new_cols;
  p.bt = block_table; p.bts = bt_stride; p.new_bt = new_table; p.nbts = new_stride;
  p.kept = kept; p.w = weights; p.w_out = weights_out;
  if (weights) { p.wsb = weight_strides[0]; p.wsh = weight_strides[1]; }
  p.Hkv = Hkv; p.keep = keep; p.W = weights ? width : keep;
  const int64_t threads = (int64_t)keep * p.per_row + (p.W - keep);
  if (threads > 0xffffffffll) return nq_fail(NQ_ERR_UNSUPPORTED, "more kept rows than one launch moves");
  hipLaunchKernelGGL(compact_rows_kernel, dim3((unsigned)((threads + 255) / 256), (unsigned)Hkv, (unsigned)B), dim3(256),
                     0, reinterpret_cast<hipStream_t>(stream), p);
  return nq_check_launch(hipGetLastError());
}
