// Attention over the paged cache with a sliding window and visible first tokens (sinks), over 16-bit caches, 8-bit caches
// with one scale per tensor and 8-bit caches with a scale for each (block, kv head).
//   K cache [blocks, kv_heads, head/x, block_size, x] (x = 16 bytes of elements), V cache [blocks, kv_heads, head, block_size]
//
// Query row j of a sequence sits at position p = seq_len - query_len + j and sees token t where
//   t <= p  and  (no window, or t > p - window, or t < sinks);
// a row that sees nothing comes out as zeros.  Rows of several query heads that share a kv head are flattened into
// columns, (row, head) = (c / G, c % G): decode rows, drafts and prompts differ only in how many columns there are.
//
//   S^T = K Q^T, O^T = V^T P^T on the matrix cores, running maximum and sum per column.
//
// 8-bit codes become fp16 (every int8 and every e4m3 value is one) and are multiplied with fp16 queries: a bf16 query row is
// first brought to [2^13, 2^14) by a power of two, which keeps all 8 bits of every element within 2^-28 of the row's
// largest.  K's and V's block scales stay outside the products, for the 16 tokens of a lane group lie in one block.  K's is
// one factor per lane on the logits.  V's is taken relative to the largest V scale met so far (vref, rescaled like the running
// maximum), so that fp16 holds it: for decode rows one factor per lane on the probabilities; for prompts a power of two, exact
// on V's codes, and the rest in [1, 2), which goes into the exponent of the probabilities.  Where it is too small for that (the
// larger one may be of tokens that other rows see) it goes onto the products, in fp32, which holds scales 2^100 apart.  One scale
// for the whole cache goes into the softmax scale and into the result.  Scales are 0 or more, or NaN.
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace mi355q {

typedef __attribute__((ext_vector_type(2))) _Float16 wa_f16x2;

constexpr float WA_LOG2E = 1.44269504088896f;
// Probabilities are kept as 2^(x - m + 6): fp16 then resolves a probability down to 2^-30 of the largest, and the running
// maximum m may lag behind by up to 8 before the sums are rescaled (with a factor of up to 2 from V's scale, the largest
// value is 2^15).  The sums of weights are taken over the probabilities as they are rounded for the product with V: where a
// few tokens carry a row, their rounding cancels.
constexpr float WA_SHIFT = 6.0f, WA_LAG = 8.0f;

// The prompt kernel: 8 waves of 32 columns.
constexpr int WA_WAVES = 8, WA_FLASH_COLS = 32 * WA_WAVES;

struct WindowParams {
  uint16_t* out;
  const uint16_t* q;
  const unsigned char* kc;
  const unsigned char* vc;
  const float* ks;
  const float* vs;
  const int32_t* tables;
  const int32_t* seq_lens;
  const int32_t* starts;        // query_start_loc, or null: one row per sequence
  float* part_o;                // [rows, heads, splits, head] partial sums (`rows` as part_row counts them)
  float* part_ml;               // [rows, heads, splits, 2] their maxima (base 2) and sums
  int64_t out_stride, q_stride;
  int64_t block_stride, head_stride;   // bytes
  int64_t scale_block_stride, scale_head_stride;
  float scale;
  int num_seqs, num_rows, num_heads, num_kv_heads, group;
  int num_blocks, table_width;
  int out16;                    // output rows start on 16 bytes
  int bs, page_magic;
  int window, sinks;            // window 0: none
  int splits, split_tiles;      // the context in stretches of split_tiles 64-token tiles, at most `splits` of them
  int part_rows;                // decode rows: room for so many rows of a sequence (0: rows as they are numbered)
  int col_tiles;                // decode rows: column tiles of the longest query
  int longest_cols;             // columns of the longest query as the caller announced it (rows kernel: at most WA_ROWS_COLS); a
                                // longer query is served so far
  int lds_cols;                 // rows kernel: columns of a 16-column tile that any sequence has
  int min_cols, max_cols;       // sequences with fewer or more columns (rows x heads per kv head) are another launch's
};

__device__ inline int wa_page(int n, int magic) { return magic ? (int)__umulhi((unsigned)n, (unsigned)magic) : n; }

// a load whose address is the same for the whole wave and whose memory no store of the launch touches: scalar cache
template <typename T>
__device__ inline T sload(const T* p) {
  return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

// Prompt rows: column tile `slot` of the batch, counted over the sequences that have any (seq < 0: there are fewer).  The grid
// is as large as num_rows allows, not sequences times the longest: every wave counts for itself, a sequence per lane.
struct Slot { int seq, ct, start, qlen; };
template <int COLS>
__device__ inline Slot slot_of(const WindowParams& p, int slot) {
  const int lane = threadIdx.x & 63;
  auto first_row = [&](int s) { return p.starts ? p.starts[min(s, p.num_seqs)] : min(s, p.num_seqs); };
  int from = first_row(lane), to = first_row(lane + 1);
  for (int s0 = 0; s0 < p.num_seqs; s0 += 64) {
    const int start = from, qlen = to - from;
    if (s0 + 64 < p.num_seqs) from = first_row(s0 + 64 + lane), to = first_row(s0 + 65 + lane);   // on their way meanwhile
    const int cols = min(min(qlen, p.num_rows - start) * p.group, p.longest_cols);   // (the grid has room for no more than was announced)
    const int n = start < 0 || cols < p.min_cols ? 0 : (max(cols, 0) + COLS - 1) / COLS;
    int upto = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(upto, d, 64);
      upto += lane >= d ? x : 0;
    }
    const uint64_t past = __ballot(upto > slot);
    if (past) {
      const int l = __builtin_ctzll(past);
      const int end = __builtin_amdgcn_readlane(upto, l);
      // a sequence's last rows, which see most under the causal mask, first
      return {s0 + l, end - 1 - slot, __builtin_amdgcn_readlane(start, l), __builtin_amdgcn_readlane(qlen, l)};
    }
    slot -= __builtin_amdgcn_readlane(upto, 63);
  }
  return {-1, 0, 0, 0};
}

__device__ inline int64_t part_row(const WindowParams& p, int seq, int start, int row) {
  return p.part_rows ? (int64_t)seq * p.part_rows + (row - start) : row;
}

// what a sequence's rows [first column, last column] see: sink tokens [0, sink_end) and [low, end), 64 at a time
struct Span {
  int sink_end, low, end, sink_tiles, tiles;
  __device__ inline int base(int i) const { return i < sink_tiles ? 64 * i : low + 64 * (i - sink_tiles); }
  __device__ inline int limit(int i) const { return i < sink_tiles ? sink_end : end; }
};
__device__ inline Span span_of(const WindowParams& p, int pos_first, int pos_last) {
  Span s;
  s.end = min(pos_last + 1, p.table_width * p.bs);
  const int low = p.window ? max(0, pos_first - p.window + 1) : 0;
  s.low = min(low, max(s.end, 0)) & ~15;
  s.sink_end = min(p.sinks, s.low);
  s.sink_tiles = (s.sink_end + 63) >> 6;
  s.tiles = s.sink_tiles + (s.end > s.low ? (s.end - s.low + 63) >> 6 : 0);
  return s;
}

enum { KV16 = MI355Q_KV_16, KVF8 = MI355Q_KV_FP8, KVI8 = MI355Q_KV_INT8, KVF8_ONE = 3 };   // (3: one scale for the tensor)

// type of the products
template <typename DT, int KV>
struct MathOf { typedef FP16 T; };
template <typename DT>
struct MathOf<DT, KV16> { typedef DT T; };

// 4 codes -> 4 fp16
template <int KV>
__device__ inline u32x2 widen4(uint32_t w) {
  u32x2 r;
  if constexpr (KV == KVF8) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
  } else {
    // 0x6400 + u is the fp16 number 1024 + u: the code biased by 128 in the low byte, then 1152 taken off, exactly
    const uint32_t u = w ^ 0x80808080u;
    const wa_f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    r[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(wa_f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias);
    r[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(wa_f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias);
  }
  return r;
}
// half h (8 codes) of a 16-byte piece
template <int KV>
__device__ inline u32x4 widen8(u32x4 w, int h) {
  const u32x2 a = widen4<KV>(w[2 * h]), b = widen4<KV>(w[2 * h + 1]);
  return u32x4{a[0], a[1], b[0], b[1]};
}


typedef __attribute__((ext_vector_type(2))) _Float16 cvt_f16x2;
template <typename MT> __device__ inline uint32_t pack_p(float lo, float hi) { return pack2<MT>(lo, hi); }
template <> __device__ inline uint32_t pack_p<FP16>(float lo, float hi) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, cvt_f16x2)); }
// max over the four lanes that share a column
__device__ inline float group_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float group_sum(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// whether one of eight 16-bit values is an infinity or NaN
template <typename MT>
__device__ inline bool not_finite(u32x4 v) {
  const uint32_t e = MT::id == MI355Q_BF16 ? 0x7f80u : 0x7c00u;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; i++) bad |= (v[i] & e) == e || ((v[i] >> 16) & e) == e;
  return bad;
}
// c + the two 16-bit values of w
template <typename MT>
__device__ inline float add_pair(uint32_t w, float c);
template <>
__device__ inline float add_pair<BF16>(uint32_t w, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, BF16::ones), c, false);
}
template <>
__device__ inline float add_pair<FP16>(uint32_t w, float c) {
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(wa_f16x2, w), __builtin_bit_cast(wa_f16x2, FP16::ones), c, false);
}

// value n of eight (none: n outside 0 .. 7), or all of them, in lanes that are `here`; zeros elsewhere
template <typename MT>
__device__ inline u32x4 only(u32x4 v, bool here, int n, bool all = false) {
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] &= here ? (all ? ~0u : n == 2 * i ? 0xffffu : n == 2 * i + 1 ? 0xffff0000u : 0u) : 0u;
  return v;
}

// ---------------------------------------------------------------------------------------------------------------------
// Few columns (decode rows, drafts): one workgroup of NW waves per (sequence, 16 NCT columns, kv head, stretch of the context);
// the waves take the stretch's 64-token tiles in turn, each with a running softmax of its own, and meet once in LDS.
// Bound by HBM: K of the next tile is requested as soon as this tile's logits stand, V as soon as its products do, so a wave
// has half a tile to a whole one on the way at any time.  Pages and scales are looked up for 16 tiles at once, a 16-token
// stretch per lane.
//
// Token order inside a tile: row i of 16-row MFMA tile T is token 16 (i / 4) + 4 T + i % 4, so the 16 logits that a lane of
// group g = lane / 16 holds after S^T are tokens 16 g .. 16 g + 15: one block, one scale, and the B operand of O^T as
// they stand; V comes in its own order, 16 tokens of a head dim per lane.
//
// Probabilities are 2^(x - m + 15) here, times V's relative scale, which is at most 1: fp16 holds their products to 2^-25, which is 2^-24
// of a token's own V down to scales of 2^-16.  Tiles with smaller ones (but zeros) are taken up once more at the end, a lane group's
// tokens at a time, the scale put onto the sums of products in fp32 (half the blocks at 2^-30: 32 rows of 100 to 4037 tokens 33 -> 96 us).
//
// Measured, 32 heads over 8 kv heads of 128: 32 rows under a window of 4096 in bf16 83 us, 468.6 MB, 5.6 TB/s (a large read reaches 6.0;
// the matrix cores are busy 5 % of the time); 32 rows of 100 to 4095 tokens in int8 34 us, 138.3 MB, 4.1 TB/s, the longest sequence's
// workgroup ends last; two rows of 131072 and 50002 tokens, 64 heads, e4m3, 68.5 us and 4.8 us for the join, 371.3 MB, 5.1 TB/s; 16 drafts
// of five rows over 500 to 3500 tokens, int8, 23.0 and 4.2 us, 67.1 MB, 2.5 TB/s; one row of 1001 tokens 11 us, round trips.
// ---------------------------------------------------------------------------------------------------------------------
constexpr float WA_ROWS_SHIFT = 15.0f, WA_RLEAST = 0x1p-16f;

template <typename DT, int KV, int HEAD, int NCT, int NW>
__global__ __launch_bounds__(64 * NW, 2) void window_rows_kernel(const WindowParams p) {
  typedef typename MathOf<DT, KV>::T MT;
  constexpr int EB = KV == KV16 ? 2 : 1;
  constexpr int DS = HEAD / 32, DT16 = HEAD / 16;
  constexpr int KP = EB == 1 ? DS / 2 : DS;      // 16-byte pieces of K per lane and row tile
  constexpr int VP = EB == 1 ? 1 : 2;            // of V per lane and 16 head dims
  constexpr int LD = HEAD + 4, COLS = 16 * NCT;
  extern __shared__ __attribute__((aligned(16))) float acc[];   // [NW][columns of a 16-column tile][LD]
  __shared__ float stat[NW][2][COLS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;

  const int kvh = blockIdx.x % p.num_kv_heads;
  int b = blockIdx.x / p.num_kv_heads;
  const int seq = b % p.num_seqs;
  b /= p.num_seqs;
  const int split = b % p.splits, ct = b / p.splits;   // what few sequences have, stretches and column tiles, last
  const int G = p.group;

  const int start = p.starts ? sload(p.starts + seq) : seq;
  const int qlen = p.starts ? sload(p.starts + seq + 1) - start : 1;
  const int all = min(qlen, p.num_rows - start) * G, cols = min(all, p.longest_cols);   // (no more than the caller announced)
  if (start < 0 || ct * COLS >= cols || all > p.max_cols) return;
  const int seq_len = sload(p.seq_lens + seq);
  const int c0 = ct * COLS, c1 = min(c0 + COLS, cols) - 1;
  const int pos0 = seq_len - qlen + c0 / G, pos1 = seq_len - qlen + c1 / G;
  const Span span = span_of(p, pos0, pos1);
  // (a context longer than the caller's bound: the last stretch takes the rest)
  const int begin = split == 0 ? 0 : split * p.split_tiles;
  const int end = split == p.splits - 1 ? span.tiles : min(begin + p.split_tiles, span.tiles);
  if (split > 0 && begin >= end) return;      // nothing here; the merge knows how many stretches there are
  const bool whole = span.tiles <= p.split_tiles;

  // ---- this lane's query columns ------------------------------------------------------------------------------------
  u32x4 qf[NCT][DS];
  float qscale[NCT];
  int pos[NCT];
#pragma unroll
  for (int n = 0; n < NCT; n++) {
    const int c = min(c0 + 16 * n + col, c1);
    const int row = start + c / G, head = kvh * G + c % G;
    pos[n] = seq_len - qlen + c / G;
    qscale[n] = fabsf(p.scale) * WA_LOG2E;
    const uint16_t* qp = p.q + (int64_t)row * p.q_stride + (int64_t)head * HEAD;
#pragma unroll
    for (int ds = 0; ds < DS; ds++) {
      const int d0 = EB == 1 ? 16 * (4 * (ds >> 1) + g) + 8 * (ds & 1) : 32 * ds + 8 * g;
      qf[n][ds] = *reinterpret_cast<const u32x4*>(qp + d0);
    }
  }

  // ---- pages and scales of the wave's next 16 tiles, a stretch per lane -------------------------------------------------
  const int32_t* table = p.tables + (int64_t)seq * p.table_width;
  const int pieces = p.bs >> 4;
  const unsigned char* kc = p.kc + (int64_t)kvh * p.head_stride;
  const unsigned char* vc = p.vc + (int64_t)kvh * p.head_stride;
  const int wg_low = p.window ? pos0 - p.window + 1 : INT_MIN;
  int64_t at_k = 0, at_v = 0;
  float at_ks = 1.f, at_vs = 0.f;
  uint64_t at_ok = 0;
  auto look_up = [&](int first) {        // first: a tile of this wave
    const int tile = min(first + NW * (lane >> 2), end - 1), j = lane & 3;
    const int t = span.base(tile) + 16 * j, lim = span.limit(tile);
    const int n16 = min(t, (lim - 1) & ~15) >> 4;         // past the end: the last stretch again, masked
    const int pg = wa_page(n16, p.page_magic);
    const int blk = table[pg];
    const bool in = (unsigned)blk < (unsigned)p.num_blocks;
    const int64_t at = in ? blk : 0;
    const int off = (n16 - pg * pieces) * 16;
    at_k = at * p.block_stride + off * 16;
    at_v = at * p.block_stride + off * EB;
    // a stretch counts where some column sees some of it
    const bool ok = in && t < lim && (t + 16 > wg_low || t < p.sinks);
    at_ok = __ballot(ok);
    if constexpr (KV != KV16) {
      const int64_t si = at * p.scale_block_stride + kvh * p.scale_head_stride;
      at_ks = ok ? p.ks[si] : 1.f;
      at_vs = ok ? p.vs[si] : 0.f;
    }
  };
  auto from = [](int64_t v, int l) {
    return (int64_t)(((uint64_t)(uint32_t)__shfl((int)(v >> 32), l, 64) << 32) | (uint32_t)__shfl((int)v, l, 64));
  };

  const int klane = (g * p.bs + (col & 3)) * 16, vlane = col * p.bs * EB, kstep = 64 * p.bs, vstep = 16 * p.bs * EB;
  u32x4 kf[4][KP], vf[DT16][VP];
  auto load_k = [&](int i) {             // tile i of the 16
    const unsigned char* kp = kc + from(at_k, 4 * i + (col >> 2)) + klane;
#pragma unroll
    for (int s = 0; s < KP; s++) {
#pragma unroll
      for (int T = 0; T < 4; T++) kf[T][s] = *reinterpret_cast<const u32x4*>(kp + T * 64);
      kp += kstep;
    }
  };
  auto load_v = [&](int i) {
    const unsigned char* vp = vc + from(at_v, 4 * i + g) + vlane;
#pragma unroll
    for (int d = 0; d < DT16; d++) {
#pragma unroll
      for (int s = 0; s < VP; s++) vf[d][s] = *reinterpret_cast<const u32x4*>(vp + s * 16);
      vp += vstep;
    }
  };

  int tile = begin + wave, at = 0;       // `at`: the tile's place among the 16 looked up
  if (tile < end) {
    look_up(tile);
    load_k(0);
    load_v(0);
  }
  // (the queries were requested first and are turned to fp16 while the tiles are on their way)
#pragma unroll
  for (int n = 0; n < NCT; n++) {
    if constexpr (EB == 1 && DT::id == MI355Q_BF16) {
      float top = 0.f;
#pragma unroll
      for (int ds = 0; ds < DS; ds++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          top = fmaxf(top, fmaxf(fabsf(BF16::to_f32((uint16_t)qf[n][ds][e])), fabsf(BF16::to_f32((uint16_t)(qf[n][ds][e] >> 16)))));
      top = group_max(top);
      int ex = (int)(__float_as_uint(top) >> 23);            // biased exponent; 255: not finite, 0: zero or subnormal
      ex = ex == 255 ? 140 : max(ex, 20);
      const float up = __uint_as_float((uint32_t)(127 + 140 - ex) << 23);   // 2^(13 - exponent)
      qscale[n] *= __uint_as_float((uint32_t)(ex - 13) << 23);
#pragma unroll
      for (int ds = 0; ds < DS; ds++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          qf[n][ds][e] = pack2<FP16>(BF16::to_f32((uint16_t)qf[n][ds][e]) * up, BF16::to_f32((uint16_t)(qf[n][ds][e] >> 16)) * up);
    }
    if (p.scale < 0.f) {   // the factor of the exponent stays positive
#pragma unroll
      for (int ds = 0; ds < DS; ds++) qf[n][ds] ^= u32x4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
    }
  }

  f32x4 o[NCT][DT16];
  float m[NCT], l[NCT], vref = 0.f, vinv = 1.f;
#pragma unroll
  for (int n = 0; n < NCT; n++) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int d = 0; d < DT16; d++) o[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  auto fragment = [&](int d, int h) {
    if constexpr (EB == 1) return widen8<KV>(vf[d][0], h);
    else return vf[d][h];
  };
  auto logits = [&](f32x4 (&s)[NCT][4]) {
#pragma unroll
    for (int T = 0; T < 4; T++) {
#pragma unroll
      for (int n = 0; n < NCT; n++) s[n][T] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ds = 0; ds < DS; ds++) {
        u32x4 a;
        if constexpr (EB == 1) a = widen8<KV>(kf[T][ds >> 1], ds & 1);
        else a = kf[T][ds];
#pragma unroll
        for (int n = 0; n < NCT; n++) s[n][T] = mfma16<MT>(a, qf[n][ds], s[n][T]);
      }
    }
  };
  // bits of the 16 tokens from tg on that column n sees
  auto sees = [&](int n, int tg, int lim, bool ok) {
    auto below = [](int k) { return k <= 0 ? 0u : k >= 16 ? 0xffffu : (1u << k) - 1; };
    uint32_t bits = ok ? below(min(pos[n] + 1, lim) - tg) : 0u;
    if (p.window) bits &= ~below(pos[n] - p.window + 1 - tg) | below(p.sinks - tg);
    return bits;
  };
  // V's tokens that no column sees become zeros, whatever bytes their places hold; whether what is left has an infinity or NaN
  auto clear_v = [&](int tg, int lim, bool ok) {
    auto below = [](int k) { return k <= 0 ? 0u : k >= 16 ? 0xffffu : (1u << k) - 1; };
    uint32_t any = ok ? below(min(pos1 + 1, lim) - tg) : 0u;
    if (p.window) any &= ~below(wg_low - tg) | below(p.sinks - tg);
    u32x4 keep[VP];
#pragma unroll
    for (int s = 0; s < VP; s++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if constexpr (EB == 1) {
          const uint32_t k = any >> (4 * e);
          keep[s][e] = ((k & 1) | ((k & 2) << 7) | ((k & 4) << 14) | ((k & 8) << 21)) * 0xffu;
        } else {
          const uint32_t k = any >> (8 * s + 2 * e);
          keep[s][e] = (k & 1 ? 0xffffu : 0u) | (k & 2 ? 0xffff0000u : 0u);
        }
      }
    bool bad = false;
#pragma unroll
    for (int d = 0; d < DT16; d++)
#pragma unroll
      for (int s = 0; s < VP; s++) {
        vf[d][s] &= keep[s];
        asm volatile("" : "+v"(vf[d][s]));      // in place: no second copy of the tile in registers
        if constexpr (EB == 2) {
          bad |= not_finite<MT>(vf[d][s]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) bad |= (((vf[d][s][e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;   // e4m3: 0x7f, 0xff
        }
      }
    return bad;
  };

  // a tile left out: V holds an infinity or NaN that only some columns may see, or its scale would leave fp16 probabilities too few bits
  // (the reference may be of tokens that other columns see)
  bool left_out = false;
  // One tile.  INNER: every column sees every token of it, if its pages exist.
  auto step = [&](auto inner) {
    constexpr bool INNER = decltype(inner)::value;
    const int t0 = span.base(tile), lim = span.limit(tile), tg = t0 + 16 * g;
    const uint32_t ok_tile = (uint32_t)(at_ok >> (4 * at)) & 15;
    const bool ok = (ok_tile >> g) & 1;
    float ks = 1.f, vs = 1.f;
    if constexpr (KV != KV16) {
      ks = __shfl(at_ks, 4 * at + g, 64);
      vs = __shfl(at_vs, 4 * at + g, 64);
    }
    f32x4 s[NCT][4];
    logits(s);
    const bool more = tile + NW < end;
    if (more) {
      if (++at == 16) {
        look_up(tile + NW);
        at = 0;
      }
      if constexpr (INNER) load_k(at);   // (the masks of a partial tile need the registers)
    }

    // ---- running softmax -------------------------------------------------------------------------------------------
    float vtop = 0.f;
    if constexpr (KV != KV16) vtop = group_max(vs);
    float back = 1.f;                  // what a new reference for V's scales does to the sums
    if (KV != KV16 && __any(vtop > vref)) {
      const float next = fmaxf(2.f * vtop, 0x1p-125f);   // headroom of 2: the next slightly larger scale changes nothing; 1 / vref is finite
      back = vref / next;
      vref = next;
      vinv = 1.f / vref;
    }
    const float r = KV == KV16 || !ok ? 1.f : vs * vinv;
    // the sum of weights over what is rounded for the product, where V's scale leaves it its bits
    const bool rounded = KV == KV16 || __all(r >= 0x1p-10f);
    const float less = KV == KV16 ? 1.f : __builtin_amdgcn_rcpf(r);
    const bool apart = KV != KV16 && __any(r > 0.f && r < WA_RLEAST);
    left_out |= apart;
    const float rp = apart ? 0.f : r;
    u32x4 pf[NCT][2];
#pragma unroll
    for (int n = 0; n < NCT; n++) {
      float f = KV == KV16 ? qscale[n] : qscale[n] * ks;
      uint32_t seen = 0xffffu;
      float x[16], mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; i++) x[i] = s[n][i >> 2][i & 3];
      if constexpr (INNER) {
        if (ok_tile != 15 && !ok) {
          f = 1.f;
#pragma unroll
          for (int i = 0; i < 16; i++) x[i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) mx = fmaxf(mx, x[i]);
        mx *= f;
      } else {
        seen = sees(n, tg, lim, ok);
#pragma unroll
        for (int i = 0; i < 16; i++) {
          x[i] = (seen >> i) & 1 ? x[i] * f : -INFINITY;
          mx = fmaxf(mx, x[i]);
        }
      }
      mx = group_max(mx);
      if (__any(mx > m[n] || back != 1.f)) {
        const float mn = fmaxf(m[n], mx);
        const float a = m[n] == -INFINITY ? 0.f : exp2_fast(m[n] - mn);
        l[n] *= a;
#pragma unroll
        for (int d = 0; d < DT16; d++) o[n][d] *= a * back;
        m[n] = mn;
      }
      const float ms = (m[n] == -INFINITY ? 0.f : m[n]) - WA_ROWS_SHIFT;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i++) x[i] = exp2_fast(INNER ? __builtin_fmaf(x[i], f, -ms) : x[i] - ms);
      if (!rounded) {
#pragma unroll
        for (int i = 0; i < 16; i++) sum += x[i];
        l[n] += sum;
        sum = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; i++) {
        uint32_t w = KV == KV16 ? pack_p<MT>(x[2 * i], x[2 * i + 1]) : pack_p<MT>(x[2 * i] * rp, x[2 * i + 1] * rp);
        sum = add_pair<MT>(w, sum);
        // (a NaN scale reaches only the columns that see its tokens)
        if (!INNER && KV != KV16) w &= ((seen >> (2 * i)) & 1 ? 0xffffu : 0u) | ((seen >> (2 * i)) & 2 ? 0xffff0000u : 0u);
        pf[n][i >> 2][i & 3] = w;
      }
      if (rounded) l[n] = KV == KV16 ? l[n] + sum : __builtin_fmaf(sum, less, l[n]);
    }

    // ---- O^T += V^T P^T ----------------------------------------------------------------------------------------------
    bool bad = false;
    if constexpr (!INNER && KV != KVI8) {
      bad = __any(clear_v(tg, lim, ok));
      left_out |= bad;
    }
    if constexpr (INNER && KV != KVI8) {
      if (ok_tile != 15) {               // a page outside the cache: block 0 was fetched in its place, and 0 times its NaN is one
#pragma unroll
        for (int d = 0; d < DT16; d++)
#pragma unroll
          for (int h = 0; h < VP; h++)
#pragma unroll
            for (int e = 0; e < 4; e++) vf[d][h][e] = ok ? vf[d][h][e] : 0u;
      }
    }
    if (INNER || KV == KVI8 || !bad) {
#pragma unroll
      for (int d = 0; d < DT16; d++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const u32x4 v = fragment(d, h);
#pragma unroll
          for (int n = 0; n < NCT; n++) o[n][d] = mfma16<MT>(v, pf[n][h], o[n][d]);
        }
    }
    if (more) {
      if constexpr (!INNER) load_k(at);
      load_v(at);
    }
    tile += NW;
  };
  // the tiles that every column sees whole: past the sinks and the window's moving start, before the moving end
  {
    const int first = p.window ? span.sink_tiles + max(0, pos1 - p.window + 1 - span.low + 63) / 64 : span.sink_tiles;
    const int to = min(pos0, span.end - 1) - 63 - span.low;
    const int in0 = min(end, first), in1 = min(end, span.sink_tiles + (to < 0 ? 0 : to / 64 + 1));
    while (tile < in0) step(std::false_type());
    while (tile < in1) step(std::true_type());
    while (tile < end) step(std::false_type());

    // tiles left out: once more, one token at a time (a lane group's 16 where all are finite), added to the columns that see them.  Which
    // they were: the same reference, from the start
    if (__builtin_expect(left_out, false)) {
      float ref = 0.f, inv = 1.f;
      for (tile = begin + wave; tile < end; tile += NW) {
        look_up(tile);
        const bool ok = (at_ok >> g) & 1, inner = tile >= in0 && tile < in1;
        const float vs = KV == KV16 ? 1.f : __shfl(at_vs, g, 64);
        bool again = false;
        if constexpr (KV != KV16) {
          const float vtop = group_max(vs);
          if (__any(vtop > ref)) ref = fmaxf(2.f * vtop, 0x1p-125f), inv = 1.f / ref;
          const float r = ok ? vs * inv : 1.f;
          again = __any(r > 0.f && r < WA_RLEAST);
        }
        if (!again && (KV == KVI8 || inner)) continue;
        load_k(0);
        load_v(0);
        const int lim = span.limit(tile), tg = span.base(tile) + 16 * g;
        const bool bad = __any(clear_v(tg, lim, ok)) && KV != KVI8;
        if (!bad && !again) continue;
        const float ks = KV == KV16 ? 1.f : __shfl(at_ks, g, 64);
        uint32_t zero;
        auto fresh = [&]() { asm volatile("v_mov_b32 %0, 0" : "=v"(zero)); };   // keeps widened operands out of registers across loops
#pragma unroll
        for (int n = 0; n < NCT; n++) {
          fresh();
          const uint32_t seen = sees(n, tg, lim, ok);
          const float f = qscale[n] * ks, ms = (m[n] == -INFINITY ? 0.f : m[n]) - WA_ROWS_SHIFT;
          u32x4 pf[2];
#pragma unroll
          for (int T = 0; T < 4; T++) {
            f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ds = 0; ds < DS; ds++) {
              u32x4 a;
              if constexpr (EB == 1) a = widen8<KV>(kf[T][ds >> 1] ^ u32x4{zero, zero, zero, zero}, ds & 1);
              else a = kf[T][ds];
              s = mfma16<MT>(a, qf[n][ds], s);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const uint32_t bits = seen >> (4 * T + 2 * i);
              pf[T >> 1][2 * (T & 1) + i] = pack2<MT>(exp2_fast(s[2 * i] * f - ms), exp2_fast(s[2 * i + 1] * f - ms)) &
                                            ((bits & 1 ? 0xffffu : 0u) | (bits & 2 ? 0xffff0000u : 0u));
            }
          }
#pragma unroll 1
          for (int k = 0; k < 64; k += bad ? 1 : 16) {
            const int i = k & 15;
            const bool here = g == k >> 4;
            const float factor = KV == KV16 ? 1.f : __shfl(vs * vinv, k & 48, 64);
            const bool counts = __shfl((int)seen, (k & 48) + col, 64) & (bad ? 1 << i : 0xffff);
            fresh();
#pragma unroll
            for (int d = 0; d < DT16; d++) {
              f32x4 x = KV == KV16 ? o[n][d] : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int h = 0; h < 2; h++) {
                u32x4 v;
                if constexpr (EB == 1) v = widen8<KV>(vf[d][0] ^ u32x4{zero, zero, zero, zero}, h);
                else v = vf[d][h] ^ u32x4{zero, zero, zero, zero};
                x = mfma16<MT>(only<MT>(v, here, i - 8 * h, !bad), only<MT>(pf[h], here, i - 8 * h, !bad), x);
              }
              if constexpr (KV != KV16) {
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf(x[e], factor, o[n][d][e]);
              }
              if (counts) o[n][d] = x;
            }
          }
        }
      }
    }
  }

  // ---- the waves meet --------------------------------------------------------------------------------------------------
#pragma unroll
  for (int n = 0; n < NCT; n++) {
    l[n] = group_sum(l[n]);
    if (m[n] == -INFINITY && l[n] != 0.f) m[n] = 0.f;   // every logit was NaN: so is the result, and not a row that sees nothing
    if (g == 0) {
      stat[wave][0][16 * n + col] = m[n];
      stat[wave][1][16 * n + col] = l[n];
    }
  }
  __syncthreads();
  constexpr int PER = HEAD / 16;
  const int width = p.lds_cols;          // columns of a 16-column tile that exist in some workgroup
#pragma unroll
  for (int n = 0; n < NCT; n++) {
    if (c0 + 16 * n > c1) break;
    if (n > 0) __syncthreads();
    float mall = stat[0][0][16 * n + col];
#pragma unroll
    for (int w = 1; w < NW; w++) mall = fmaxf(mall, stat[w][0][16 * n + col]);
    float a = m[n] == -INFINITY ? 0.f : exp2_fast(m[n] - mall);
    if constexpr (KV != KV16) a *= vref;
    if (col < width) {
#pragma unroll
      for (int d = 0; d < DT16; d++) *reinterpret_cast<f32x4*>(&acc[(wave * width + col) * LD + 16 * d + 4 * g]) = o[n][d] * a;
    }
    __syncthreads();
    const int cc = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * PER, c = c0 + 16 * n + cc;
    if (cc >= 16 || c > c1) continue;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < NW; w++) top = fmaxf(top, stat[w][0][16 * n + cc]);
    f32x4 v[PER / 4];
#pragma unroll
    for (int i = 0; i < PER / 4; i++) v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; w++) {
      const float mw = stat[w][0][16 * n + cc];
      sum += mw == -INFINITY ? 0.f : stat[w][1][16 * n + cc] * exp2_fast(mw - top);
#pragma unroll
      for (int i = 0; i < PER / 4; i++) v[i] += *reinterpret_cast<const f32x4*>(&acc[(w * width + cc) * LD + d0 + 4 * i]);
    }
    const int orow = start + c / G, ohead = kvh * G + c % G;
    if (whole) {
      const float inv = top == -INFINITY ? 0.f : 1.f / sum;
      uint32_t* out = reinterpret_cast<uint32_t*>(p.out + (int64_t)orow * p.out_stride + (int64_t)ohead * HEAD + d0);
#pragma unroll
      for (int i = 0; i < PER / 2; i++) out[i] = top == -INFINITY ? 0u : pack2<DT>(v[i >> 1][2 * (i & 1)] * inv, v[i >> 1][2 * (i & 1) + 1] * inv);
    } else {
      const int64_t to = (part_row(p, seq, start, orow) * p.num_heads + ohead) * p.splits + split;
#pragma unroll
      for (int i = 0; i < PER / 4; i++) *reinterpret_cast<f32x4*>(p.part_o + to * HEAD + d0 + 4 * i) = v[i];
      if (d0 == 0) {
        p.part_ml[2 * to] = top;
        p.part_ml[2 * to + 1] = sum;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Many columns (prompt rows): one workgroup of NW waves per (sequence, 32 NW columns, kv head, stretch of the context), 32
// columns a wave.  The workgroup brings a 64-token tile of K and V into LDS once, as 16-bit MFMA operands in lane order (codes
// are widened on the way: once per workgroup instead of once per wave), two tiles deep: the codes of the tile after the next
// are on their way in registers while this one is worked on.
//
// v_mfma_f32_32x32x16.  Row r of a 32-token tile of S^T is token r with bits 2 and 3 exchanged: the 8 logits a lane then holds
// of each 16-token stretch are tokens 8 h .. 8 h + 7 of it (h = lane / 32), the B operand of O^T as they stand.  A stretch lies
// in one block, so K's scale is wave-uniform per 8 registers and joins the factor of the exponent.  V's scale is a power of two
// times a number in [1, 2): the power, relative to that of the largest scale met so far and with 2^7 in hand, goes into the
// widened codes, exactly (down to scales of 2^-22 of the largest for e4m3, whose codes have bits down to 2^-9, and 2^-31 for int8; below
// that onto the products of a stretch in fp32); the number goes into the exponent of the probabilities.
//
// Bound by the matrix cores and the exponentials in turn: a SIMD holds two waves of 128-wide heads, and while both are in their
// softmax no product runs.  8192 rows of 32 heads of 128 under a window of 4096, bf16: 431 to 475 us from card to card, 870 to 960
// TFLOP/s of what is visible (a large matrix product reaches 1190 to 1230); the matrix cores are busy 45 % of the cycles counted, the
// vector units 46 %, LDS conflicts are 3 %.  2048 rows over a context of 6144 and 700 of their own, int8, with a decode row's two launches
// 286 to 313 us, 780 to 855 TFLOP/s.  64-wide heads have room for two workgroups to a CU, and the exponentials weigh twice as much: five
// prompts of up to 2047 rows under a window of 512, e4m3 with one scale, 40 us behind each other (44 on an idle card), vector units
// busy 61 %, matrix cores 22.
// Slower at 8192 rows: four waves (489 us), the next tile's logits ahead of this one's softmax (795, registers spill), the
// halves of a workgroup in opposite phases over three buffers (578), higher priority for half the waves (449 against 448).
// ---------------------------------------------------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(16))) float f32x16;

template <typename MT>
__device__ inline f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c);
template <>
__device__ inline f32x16 mfma32<BF16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ inline f32x16 mfma32<FP16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// max / sum over the two lanes that share a column
__device__ inline float pair_max(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float pair_sum(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
constexpr float WA_VSHIFT = 128.0f;

template <typename DT, int KV, int HEAD, int NW>
__global__ __launch_bounds__(64 * NW, HEAD == 64 ? 4 : 2) void window_flash_kernel(const WindowParams p) {
  typedef typename MathOf<DT, KV>::T MT;
  constexpr bool SCALED = KV == KVF8 || KV == KVI8;      // a scale for each (block, kv head)
  constexpr int CODE = KV == KVF8_ONE ? KVF8 : KV;
  constexpr int EB = KV == KV16 ? 2 : 1, NT = 64 * NW, COLS = 32 * NW;
  constexpr int KS = HEAD / 16, DTL = HEAD / 32;
  constexpr int KBYTES = 64 * HEAD * 2, STAGE = 2 * KBYTES;
  constexpr int PIECES = 64 * HEAD * EB / 16;        // 16-byte pieces of K in a tile, and as many of V
  constexpr int PP = 2 * PIECES / NT;                // of both, per thread
  constexpr int OLD = HEAD + 8;                      // output rows in LDS, padded
  constexpr int LDS = 2 * STAGE > COLS * OLD * 2 ? 2 * STAGE : COLS * OLD * 2;
  static_assert(2 * PIECES % NT == 0, "pieces are shared out evenly");
  constexpr int CHUNK = 64;
  constexpr int SCALES = SCALED ? 4 * CHUNK : 4;
  struct Chunk {
    u32x4 at[4 * CHUNK];      // per stretch: block offset (64 bits), token offset in the block, tokens somebody sees
    float ks[SCALES];
    float vpow[SCALES], vlog[SCALES], vinv[SCALES];   // V's scale: 2^7 power / vref (1 where vfac has it), log2 and reciprocal of the rest
    float vfac[SCALES];       // the power where fp16 would not hold its products with the codes, else 1
    int ok[CHUNK];            // per tile: stretches whose page exists and that begin before the end; 16: some vfac is not 1
    int first;                // the first such tile of the chunk
    float vref;               // a power of two above every scale so far
  };
  __shared__ __attribute__((aligned(1024))) unsigned char lds[LDS];
  __shared__ __attribute__((aligned(16))) Chunk chunks[2];
  __shared__ int bad_tile[2];   // a tile (from 1) with a V that is not finite and that some columns see in part
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;

  const int kvh = blockIdx.x % p.num_kv_heads;
  int b = blockIdx.x / p.num_kv_heads;
  const int split = b % p.splits;
  const Slot slot = slot_of<COLS>(p, b / p.splits);
  if (slot.seq < 0) return;
  const int seq = slot.seq, ct = slot.ct, start = slot.start, qlen = slot.qlen;
  const int G = p.group;
  const int cols = min(min(qlen, p.num_rows - start) * G, p.longest_cols);
  const int seq_len = sload(p.seq_lens + seq);
  const int c0 = ct * COLS, c1 = min(c0 + COLS, cols) - 1;
  const int pos0 = seq_len - qlen + c0 / G, pos1 = seq_len - qlen + c1 / G;
  const Span span = span_of(p, pos0, pos1);
  const int begin = split == 0 ? 0 : split * p.split_tiles;
  const int end = split == p.splits - 1 ? span.tiles : min(begin + p.split_tiles, span.tiles);
  if (split > 0 && begin >= end) return;
  const bool whole = span.tiles <= p.split_tiles;
  const int wg_low = p.window ? pos0 - p.window + 1 : INT_MIN;    // below it, only sinks are seen

  // ---- this lane's query column ---------------------------------------------------------------------------------------
  const int wc0 = c0 + wave * 32, wc1 = min(wc0 + 32, cols) - 1;  // the wave's columns (none: wc0 > wc1)
  const int c = min(wc0 + col, c1);
  const int row = start + c / G, head = kvh * G + c % G;
  const int pos = seq_len - qlen + c / G;
  const int wpos0 = seq_len - qlen + min(wc0, c1) / G, wpos1 = seq_len - qlen + min(wc0 + 31, c1) / G;
  u32x4 qf[KS];
  float qscale = fabsf(p.scale) * WA_LOG2E;
  if constexpr (KV == KVF8_ONE) qscale *= *p.ks;
  {
    const uint16_t* qp = p.q + (int64_t)row * p.q_stride + (int64_t)head * HEAD + 8 * half;
#pragma unroll
    for (int s = 0; s < KS; s++) qf[s] = *reinterpret_cast<const u32x4*>(qp + 16 * s);
    if constexpr (EB == 1 && DT::id == MI355Q_BF16) {
      float top = 0.f;
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          top = fmaxf(top, fmaxf(fabsf(BF16::to_f32((uint16_t)qf[s][e])), fabsf(BF16::to_f32((uint16_t)(qf[s][e] >> 16)))));
      top = pair_max(top);
      int ex = (int)(__float_as_uint(top) >> 23);
      ex = ex == 255 ? 140 : max(ex, 20);
      const float up = __uint_as_float((uint32_t)(127 + 140 - ex) << 23);
      qscale *= __uint_as_float((uint32_t)(ex - 13) << 23);
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          qf[s][e] = pack2<FP16>(BF16::to_f32((uint16_t)qf[s][e]) * up, BF16::to_f32((uint16_t)(qf[s][e] >> 16)) * up);
    }
    if (p.scale < 0.f) {   // the factor of the exponent stays positive
#pragma unroll
      for (int s = 0; s < KS; s++) qf[s] ^= u32x4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
    }
  }

  const int32_t* table = p.tables + (int64_t)seq * p.table_width;
  const int blocks16 = p.bs >> 4;
  const unsigned char* kc = p.kc + (int64_t)kvh * p.head_stride;
  const unsigned char* vc = p.vc + (int64_t)kvh * p.head_stride;

  // the tiles that every column sees whole: past the sinks and the window's moving start, before the moving end (numbered from
  // `begin`, like every tile below)
  const int tiles = end - begin;
  int in0, in1;
  {
    const int first = p.window ? span.sink_tiles + max(0, pos1 - p.window + 1 - span.low + 63) / 64 : span.sink_tiles;
    const int to = min(pos0, span.end - 1) - 63 - span.low;
    in0 = max(0, min(tiles, first - begin));
    in1 = max(in0, min(tiles, span.sink_tiles + (to < 0 ? 0 : to / 64 + 1) - begin));
  }

  // ---- where the tiles lie -------------------------------------------------------------------------------------------------
  // Looked up CHUNK tiles at a time by one wave, a 16-token stretch per lane, into LDS (two chunks, so that the next one is
  // there before it is needed): the loop itself then has no page arithmetic, and V's scales have one reference per chunk.
  auto fill = [&](int first) {
    Chunk& ch = chunks[(first - begin) / CHUNK & 1];
    float v[CHUNK / 16], top = 0.f;
#pragma unroll
    for (int i = 0; i < CHUNK / 16; i++) {
      const int n = 64 * i + lane, j = n & 3, tile = min(first + (n >> 2), end - 1);
      const int t0 = span.base(tile), lim = span.limit(tile), t = t0 + 16 * j;
      const int n16 = min(t, (lim - 1) & ~15) >> 4;           // past the end: the last stretch again, masked
      const int pg = wa_page(n16, p.page_magic);
      const int blk = table[pg];
      const bool in = (unsigned)blk < (unsigned)p.num_blocks;
      const int64_t at = in ? blk : 0;
      // tokens that some column of the workgroup sees
      auto below = [&](int k) { return k <= 0 ? 0u : k >= 16 ? 0xffffu : (1u << k) - 1; };
      uint32_t seen = below(lim - t);
      if (p.window) seen &= ~below(wg_low - t) | below(p.sinks - t);
      if (!in) seen = 0;
      const uint64_t ok = __ballot(in && t < lim);
      v[i] = 0.f;
      if constexpr (SCALED) {
        const int64_t si = at * p.scale_block_stride + kvh * p.scale_head_stride;
        ch.ks[n] = in ? p.ks[si] : 1.f;
        v[i] = seen ? p.vs[si] : 0.f;
        top = fmaxf(top, v[i]);
      }
      const int64_t byte = at * p.block_stride;
      ch.at[n] = u32x4{(uint32_t)byte, (uint32_t)(byte >> 32), (uint32_t)((n16 - pg * blocks16) * 16), seen};
      if (j == 0) ch.ok[n >> 2] = (int)(ok >> (lane & ~3)) & 15;
    }
    if constexpr (SCALED) {
      top = wave_max(top);
      top = top > 0.f ? __uint_as_float((__float_as_uint(fminf(fmaxf(top, 0x1p-110f), 0x1p125f)) & 0x7f800000u) + 0x00800000u) : 0.f;
      if (first > begin) top = fmaxf(top, chunks[((first - begin) / CHUNK & 1) ^ 1].vref);   // never falls
      const float inv = top > 0.f ? WA_VSHIFT / top : 0.f;
      int where = INT_MAX;          // the first tile that has one
#pragma unroll
      for (int i = 0; i < CHUNK / 16; i++) {
        const int n = 64 * i + lane;
        const uint32_t bits = __float_as_uint(v[i]);
        const bool split = v[i] > 0x1p-100f && v[i] < INFINITY;      // (else as it is: zero, next to it, or a NaN that stays one)
        const float rest = split ? __uint_as_float((bits & 0x007fffffu) | 0x3f800000u) : 1.f;
        const float power = split ? __uint_as_float(bits & 0x7f800000u) * inv : v[i] * inv + (v[i] - v[i]);
        const bool apart = power > 0.f && power < (KV == KVI8 ? 0x1p-24f : 0x1p-15f);   // products with codes of 2^-24 at least
        ch.vpow[n] = apart ? 1.f : power;
        ch.vfac[n] = apart ? power : 1.f;
        const uint64_t some = __ballot(apart);
        if ((lane & 3) == 0 && ((some >> lane) & 15)) ch.ok[n >> 2] |= 16;
        if (some) where = min(where, first - begin + 16 * i + (__builtin_ctzll(some) >> 2));
        ch.vlog[n] = __builtin_amdgcn_logf(rest);
        ch.vinv[n] = 1.f / rest;
      }
      if (lane == 0) ch.vref = top, ch.first = where;
    }
  };

  // ---- a tile on its way -------------------------------------------------------------------------------------------------
  // A wave fetches PP groups of 64 pieces, all of one 16-token stretch jw: the address is one scalar base and offsets that
  // never change.  K group: 16 tokens x 4 chunks of 16 bytes; V group: 64 head dims (8-bit), or 32 x 2 halves.
  u32x4 piece[PP];
  constexpr int GROUPS = PIECES / 64, GPJ = GROUPS / 4, KPP = PP > 1 ? PP / 2 : 1;
  const bool fetches_k = PP > 1 || wave < NW / 2;       // (PP 1: half the waves fetch K, half V)
  const int g0 = PP > 1 ? wave * KPP : wave % (NW / 2); // the wave's first K group and first V group
  const int jw = g0 / GPJ;
  static_assert(PP == 1 || GPJ % KPP == 0, "a wave's groups lie in one stretch");
  int koff[KPP], voff[KPP];
#pragma unroll
  for (int i = 0; i < KPP; i++) {
    const int q = (g0 + i) % GPJ;
    koff[i] = ((q * 4 + (lane >> 4)) * p.bs + (lane & 15)) * 16;
    voff[i] = (EB == 1 ? q * 64 + lane : q * 32 + col) * p.bs * EB + (EB == 2 ? 16 * half : 0);
  }
  auto chunk_of = [&](int n) -> Chunk& { return chunks[n / CHUNK & 1]; };   // n: tile - begin
  auto request = [&](int n) {
    const u32x4 e = chunk_of(n).at[n % CHUNK * 4 + jw];
    const uint32_t lo = __builtin_amdgcn_readfirstlane(e[0]), hi = __builtin_amdgcn_readfirstlane(e[1]);
    const uint32_t off = __builtin_amdgcn_readfirstlane(e[2]);
    const int64_t at = (int64_t)((uint64_t)hi << 32 | lo);
    const unsigned char* kb = kc + at + off * 16;
    const unsigned char* vb = vc + at + off * EB;
    if constexpr (PP > 1) {
#pragma unroll
      for (int i = 0; i < KPP; i++) {
        piece[i] = *reinterpret_cast<const u32x4*>(kb + (unsigned)koff[i]);
        piece[KPP + i] = *reinterpret_cast<const u32x4*>(vb + (unsigned)voff[i]);
      }
    } else {
      piece[0] = *reinterpret_cast<const u32x4*>((fetches_k ? kb : vb) + (unsigned)(fetches_k ? koff[0] : voff[0]));
    }
  };
  // the requested tile into LDS, as operands
  const int rho = ((lane & 3) | ((lane & 4) << 1) | ((lane & 8) >> 1)) + 16 * (jw & 1);   // K row of this lane's token
  auto deliver = [&](int n) {
    unsigned char* to = lds + (n & 1) * STAGE;
    auto put_k = [&](int i, u32x4 w) {
      const int ch = (g0 + i) % GPJ * 4 + (lane >> 4);      // 16-byte chunk of the head
      if constexpr (EB == 1) {
        unsigned char* at = to + (((jw >> 1) * KS + ch) * 64 + rho) * 16;
        *reinterpret_cast<u32x4*>(at) = widen8<CODE>(w, 0);
        *reinterpret_cast<u32x4*>(at + 512) = widen8<CODE>(w, 1);
      } else {
        *reinterpret_cast<u32x4*>(to + (((jw >> 1) * KS + (ch >> 1)) * 64 + (ch & 1) * 32 + rho) * 16) = w;
      }
    };
    auto put_v = [&](int i, u32x4 w) {
      const int d = (g0 + i) % GPJ * (EB == 1 ? 64 : 32) + (EB == 1 ? lane : col);
      unsigned char* at = to + KBYTES + (((d >> 5) * 4 + jw) * 64 + (d & 31)) * 16;
      const int e0 = n % CHUNK * 4 + jw;
      // tokens that no column of the workgroup sees are zeros in V, whatever their places hold
      const uint32_t seen = __builtin_amdgcn_readfirstlane(chunk_of(n).at[e0][3]);
      u32x4 v[EB == 1 ? 2 : 1];
      if constexpr (EB == 1) {
        v[0] = widen8<CODE>(w, 0);
        v[1] = widen8<CODE>(w, 1);
        if constexpr (SCALED) {
          const _Float16 r16 = (_Float16)chunk_of(n).vpow[e0];
          const wa_f16x2 rr = {r16, r16};
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const uint32_t x = v[h][e];   // (a bit cast of the vector element itself would take element 0)
              v[h][e] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(wa_f16x2, x) * rr);
            }
        }
      } else {
        v[0] = w;
      }
      if (seen != 0xffffu) {
#pragma unroll
        for (int h = 0; h < (EB == 1 ? 2 : 1); h++) {
          const uint32_t mask = EB == 1 ? seen >> (8 * h) : seen >> (8 * half);
#pragma unroll
          for (int e = 0; e < 4; e++) v[h][e] &= ((mask >> (2 * e)) & 1 ? 0xffffu : 0u) | ((mask >> (2 * e)) & 2 ? 0xffff0000u : 0u);
        }
      }
      if (n < in0 || n >= in1) {
        bool bad = not_finite<MT>(v[0]);
        if constexpr (EB == 1) bad |= not_finite<MT>(v[1]);
        if (__any(bad)) bad_tile[n & 1] = n + 1;
      }
      if constexpr (EB == 1) {
        *reinterpret_cast<u32x4*>(at) = v[0];
        *reinterpret_cast<u32x4*>(at + 512) = v[1];
      } else {
        *reinterpret_cast<u32x4*>(at + half * 512) = v[0];
      }
    };
    if constexpr (PP > 1) {
#pragma unroll
      for (int i = 0; i < KPP; i++) {
        put_k(i, piece[i]);
        put_v(i, piece[KPP + i]);
      }
    } else {
      if (fetches_k) put_k(0, piece[0]);
      else put_v(0, piece[0]);
    }
  };
  auto arrive = [&]() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  f32x16 o[DTL];
#pragma unroll
  for (int d = 0; d < DTL; d++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[d][e] = 0.f;
  float m = -INFINITY, l = 0.f, oref = 0.f;

  if (tiles > 0) {
    if (wave == 0) fill(begin);
    if (threadIdx.x < 2) bad_tile[threadIdx.x] = 0;
    arrive();
    request(0);
    deliver(0);
    if (tiles > 1) request(1);
  }

  // One tile.  INNER: every column of the workgroup sees every token of it, if its pages exist.
  auto step = [&](int n, auto inner) {
    constexpr bool INNER = decltype(inner)::value;
    arrive();               // the tile is in place for every wave, and the other buffer is free
    // the next chunk, half a chunk ahead: its slot's last reader was tile n - CHUNK / 2
    if (n % CHUNK == CHUNK / 2 && begin + n + CHUNK / 2 < end && wave == (n / CHUNK & (NW - 1))) fill(begin + n + CHUNK / 2);
    const unsigned char* st0 = lds + (n & 1) * STAGE + lane * 16;
    const Chunk& ch = chunk_of(n);
    const int t0 = INNER ? 0 : span.base(begin + n), lim = INNER ? 0 : span.limit(begin + n);
    const int state = __builtin_amdgcn_readfirstlane(ch.ok[n % CHUNK]), ok_tile = SCALED ? state & 15 : state;
    const bool apart = SCALED && state > 15;
    bool idle = wc0 > wc1;
    // does any of the wave's columns see any of it?
    if constexpr (!INNER) idle = idle || t0 > wpos1 || (p.window && t0 + 63 <= wpos0 - p.window && t0 >= p.sinks) || ok_tile == 0;

    f32x16 s[2];
    if (!idle) {
#pragma unroll
      for (int rt = 0; rt < 2; rt++) {
#pragma unroll
        for (int e = 0; e < 16; e++) s[rt][e] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; k++) s[rt] = mfma32<MT>(*reinterpret_cast<const u32x4*>(st0 + (rt * KS + k) * 1024), qf[k], s[rt]);
      }
      // operand reads ahead of the products: six, or three in the 128 registers that 64-wide heads leave (five prompts under a
      // window of 512: 48.5 us, with four or six of them 51)
      constexpr int AHEAD = HEAD == 64 ? 3 : 6;
      __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
      for (int k = 0; k < 2 * KS - AHEAD; k++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
    }
    float f[4];
    if constexpr (!SCALED) {
#pragma unroll
      for (int j = 0; j < 4; j++) f[j] = qscale;
    } else {
      const f32x4 ks = *reinterpret_cast<const f32x4*>(&ch.ks[n % CHUNK * 4]);
#pragma unroll
      for (int j = 0; j < 4; j++) f[j] = qscale * ks[j];
    }
    if (n + 1 < tiles) {
      deliver(n + 1);
      if (n + 2 < tiles) request(n + 2);
    }
    if (idle) return;

    // ---- running softmax ----------------------------------------------------------------------------------------------
    if constexpr (!INNER) {
      // logits scaled here, so that what is masked is -inf whatever its scale
#pragma unroll
      for (int e = 0; e < 32; e++) s[e >> 4][e & 15] *= f[e >> 3];
      auto token = [](int e) { return 32 * (e >> 4) + 16 * ((e >> 3) & 1) + (e & 7); };   // less 8 half
      const int from = t0 + 8 * half;
      if (t0 + 63 > wpos0 || t0 + 64 > lim) {
        const int hi = min(pos, lim - 1) - from;
#pragma unroll
        for (int e = 0; e < 32; e++) s[e >> 4][e & 15] = token(e) <= hi ? s[e >> 4][e & 15] : -INFINITY;
      }
      if (p.window && t0 <= wpos1 - p.window) {
        const int lo = pos - p.window + 1 - from, sk = p.sinks - from;
#pragma unroll
        for (int e = 0; e < 32; e++) s[e >> 4][e & 15] = token(e) >= lo || token(e) < sk ? s[e >> 4][e & 15] : -INFINITY;
      }
    }
    if (ok_tile != 15) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if ((ok_tile >> j) & 1) continue;
        f[j] = 1.f;
#pragma unroll
        for (int e = 0; e < 8; e++) s[j >> 1][8 * (j & 1) + e] = -INFINITY;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      float a = s[j >> 1][8 * (j & 1)];
#pragma unroll
      for (int e = 1; e < 8; e++) a = fmaxf(a, s[j >> 1][8 * (j & 1) + e]);
      mx = fmaxf(mx, INNER ? a * f[j] : a);
    }
    mx = pair_max(mx);
    const float vref_tile = SCALED ? ch.vref : 0.f;
    if (__any(mx > m + WA_LAG) || (SCALED && __any(vref_tile > oref))) {
      const float mn = mx > m + WA_LAG ? mx : m;
      float a = m == -INFINITY ? 0.f : exp2_fast(m - mn);
      l *= a;
      if constexpr (SCALED) {
        if (vref_tile > oref) a *= oref / vref_tile, oref = vref_tile;
      }
#pragma unroll
      for (int d = 0; d < DTL; d++) o[d] *= a;
      m = mn;
    }
    const float ms = (m == -INFINITY ? 0.f : m) - WA_SHIFT;
    f32x4 plus = {-ms, -ms, -ms, -ms}, less = {1.f, 1.f, 1.f, 1.f};
    if constexpr (SCALED) {
      plus += *reinterpret_cast<const f32x4*>(&ch.vlog[n % CHUNK * 4]);
      less = *reinterpret_cast<const f32x4*>(&ch.vinv[n % CHUNK * 4]);
    }
    u32x4 pf[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float x = s[j >> 1][8 * (j & 1) + e];
        s[j >> 1][8 * (j & 1) + e] = exp2_fast(INNER ? __builtin_fmaf(x, f[j], plus[j]) : x + plus[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        pf[j][e] = pack_p<MT>(s[j >> 1][8 * (j & 1) + 2 * e], s[j >> 1][8 * (j & 1) + 2 * e + 1]);
        sum = add_pair<MT>(pf[j][e], sum);
      }
      l = SCALED ? __builtin_fmaf(sum, less[j], l) : l + sum;
    }

    // ---- O^T += V^T P^T -------------------------------------------------------------------------------------------------
    const unsigned char* vt = st0 + KBYTES;
    const bool bad = !INNER && __builtin_amdgcn_readfirstlane(bad_tile[n & 1]) == n + 1;
    if (!INNER && __builtin_expect(bad || apart, false)) {
      // an infinity or NaN that some columns may see and others must not: one token at a time, added where it is seen.  Scales too far
      // apart for fp16: one stretch at a time, scaled in fp32.
#pragma unroll 1
      for (int k = 0; k < 64; k += bad ? 1 : 16) {
        const int st = k >> 4, i = k & 7, t = t0 + k;
        const bool here = !bad || half == ((k >> 3) & 1);
        const bool counts = !bad || (t < lim && t <= pos && (!p.window || t > pos - p.window || t < p.sinks) && ((ok_tile >> st) & 1));
        const u32x4 pb = only<MT>(st == 0 ? pf[0] : st == 1 ? pf[1] : st == 2 ? pf[2] : pf[3], here, i, !bad);
#pragma unroll
        for (int d = 0; d < DTL; d++) {
          const u32x4 a = only<MT>(*reinterpret_cast<const u32x4*>(vt + (d * 4 + st) * 1024), here, i, !bad);
          f32x16 r;
          if constexpr (SCALED) {
            r = mfma32<MT>(a, pb, f32x16{});
            const float factor = ch.vfac[n % CHUNK * 4 + st];
#pragma unroll
            for (int e = 0; e < 16; e++) r[e] = __builtin_fmaf(r[e], factor, o[d][e]);
          } else {
            r = mfma32<MT>(a, pb, o[d]);
          }
#pragma unroll
          for (int e = 0; e < 16; e++) o[d][e] = counts ? r[e] : o[d][e];
        }
      }
    } else {
#pragma unroll
      for (int d = 0; d < DTL; d++)
#pragma unroll
        for (int st = 0; st < 4; st++) o[d] = mfma32<MT>(*reinterpret_cast<const u32x4*>(vt + (d * 4 + st) * 1024), pf[st], o[d]);
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 1);
#pragma unroll
      for (int k = 0; k < 4 * DTL - 4; k++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 4, 1);
    }
  };
  // Where the run of unmasked tiles that n begins ends: a tile of scales too far apart goes through the masked step.  Asked once for
  // each chunk, which is 0 to 2 % slower than not at all; asked at each tile 1 to 6 %, and the products in an unmasked step of their own 10 %.
  // (2048 rows whose V scales are in part 2^-40 of the others: 80 -> 144 us.)
  auto stop = [&](int n) {
    return !SCALED ? in1 : min(min(in1, n - n % CHUNK + CHUNK), __builtin_amdgcn_readfirstlane(chunk_of(n).first));
  };
  int n = 0;
  if constexpr (HEAD == 64 || KV == KV16) {
    // the masked step stands once in the code: 35 KB instead of 45, and short walks are bound by fetching it (five prompts under a
    // window of 512 47.7 -> 44.4 us, 8192 rows in bf16 444 -> 440).  With codes of 128-wide heads the compiler then finds worse
    // registers: 2048 rows over 6144 296 -> 330 us.
    while (n < tiles) {
      const int to = stop(n);
      for (; n >= in0 && n < to; n++) step(n, std::true_type());
      if (n < tiles) step(n++, std::false_type());
    }
  } else {
    for (; n < in0; n++) step(n, std::false_type());
    for (int to; n < in1 && (to = stop(n)) > n;)
      for (; n < to; n++) step(n, std::true_type());
    for (; n < tiles; n++) step(n, std::false_type());
  }

  // ---- out ----------------------------------------------------------------------------------------------------------------
  l = pair_sum(l);
  if (m == -INFINITY && l != 0.f) m = 0.f;   // every logit was NaN: so is the result, and not a row that sees nothing
  const float unit = SCALED ? oref / WA_VSHIFT : KV == KVF8_ONE ? *p.vs : 1.f;
  if (whole) {
    arrive();               // the last tile has been read by every wave: LDS takes the output rows
    const float inv = m == -INFINITY ? 0.f : unit / l;
    uint16_t* mine = reinterpret_cast<uint16_t*>(lds) + (wave * 32 + col) * OLD;
#pragma unroll
    for (int d = 0; d < DTL; d++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        u32x2 w;
        w[0] = m == -INFINITY ? 0u : pack2<DT>(o[d][4 * q] * inv, o[d][4 * q + 1] * inv);
        w[1] = m == -INFINITY ? 0u : pack2<DT>(o[d][4 * q + 2] * inv, o[d][4 * q + 3] * inv);
        *reinterpret_cast<u32x2*>(mine + 32 * d + 8 * q + 4 * half) = w;
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // a wave reads back only what it wrote
    constexpr int LPR = HEAD / 8;                        // lanes per row, 16 bytes each
#pragma unroll
    for (int i = 0; i < 32 / (64 / LPR); i++) {
      const int r = i * (64 / LPR) + lane / LPR, d = lane % LPR * 8;
      const int cc = wc0 + r;
      if (cc > wc1) continue;
      const u32x4 w = *reinterpret_cast<const u32x4*>(reinterpret_cast<uint16_t*>(lds) + (wave * 32 + r) * OLD + d);
      uint16_t* to = p.out + (int64_t)(start + cc / G) * p.out_stride + (int64_t)(kvh * G + cc % G) * HEAD + d;
      if (p.out16) *reinterpret_cast<u32x4*>(to) = w;
      else
#pragma unroll
        for (int e = 0; e < 4; e++) reinterpret_cast<uint32_t*>(to)[e] = w[e];
    }
  } else if (wc0 + col <= wc1) {
    const int64_t at = (part_row(p, seq, start, row) * p.num_heads + head) * p.splits + split;
    float* to = p.part_o + at * HEAD + 4 * half;
#pragma unroll
    for (int d = 0; d < DTL; d++)
#pragma unroll
      for (int q = 0; q < 4; q++)
        *reinterpret_cast<f32x4*>(to + 32 * d + 8 * q) =
            f32x4{o[d][4 * q] * unit, o[d][4 * q + 1] * unit, o[d][4 * q + 2] * unit, o[d][4 * q + 3] * unit};
    if (half == 0) {
      p.part_ml[2 * at] = m;
      p.part_ml[2 * at + 1] = l;
    }
  }
}

// Joins the stretches of a long context: one wave per column (query row and head).  COLS: columns of a workgroup of the
// launch before, whose span decides how many stretches there are and which row they belong to.
template <typename DT, int HEAD, int COLS>
__global__ __launch_bounds__(256) void window_merge_kernel(const WindowParams p) {
  constexpr bool FLASH = COLS == WA_FLASH_COLS;
  constexpr int PER = HEAD / 64;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int b = blockIdx.x, c, kvh, seq, start, qlen;
  if (FLASH) {
    c = b % (COLS / 4) * 4 + wave;
    b /= COLS / 4;
    kvh = b % p.num_kv_heads;
    const Slot slot = slot_of<COLS>(p, b / p.num_kv_heads);
    if (slot.seq < 0) return;
    seq = slot.seq, start = slot.start, qlen = slot.qlen;
    c += slot.ct * COLS;
  } else {
    const int per_seq = p.col_tiles * COLS / 4;
    c = (b % per_seq) * 4 + wave;
    b /= per_seq;
    kvh = b % p.num_kv_heads, seq = b / p.num_kv_heads;
    start = p.starts ? sload(p.starts + seq) : seq;
    qlen = p.starts ? sload(p.starts + seq + 1) - start : 1;
  }
  const int all = min(qlen, p.num_rows - start) * p.group, cols = min(all, p.longest_cols);
  if (start < 0 || c >= cols || all > p.max_cols) return;
  const int seq_len = sload(p.seq_lens + seq);
  const int c0 = c / COLS * COLS, c1 = min(c0 + COLS, cols) - 1;
  const Span span = span_of(p, seq_len - qlen + c0 / p.group, seq_len - qlen + c1 / p.group);
  if (span.tiles <= p.split_tiles) return;    // written by its only workgroup
  const int n = min(p.splits, (span.tiles + p.split_tiles - 1) / p.split_tiles);
  const int row = start + c / p.group, head = kvh * p.group + c % p.group;
  const int64_t at = (part_row(p, seq, start, row) * p.num_heads + head) * p.splits;
  const float* ml = p.part_ml + 2 * at;
  const float* po = p.part_o + at * HEAD + lane * PER;
  float top = -INFINITY;
  for (int i = lane; i < n; i += 64) top = fmaxf(top, ml[2 * i]);
  top = wave_max(top);
  float sum = 0.f, v[PER];
#pragma unroll
  for (int j = 0; j < PER; j++) v[j] = 0.f;
#pragma unroll 4
  for (int i = 0; i < n; i++) {
    const float mi = ml[2 * i];
    const float w = mi == -INFINITY ? 0.f : exp2_fast(mi - top);
    sum += ml[2 * i + 1] * w;
#pragma unroll
    for (int j = 0; j < PER; j++) {
      const float x = po[(int64_t)i * HEAD + j] * w;
      v[j] += mi == -INFINITY ? 0.f : x;   // (a stretch of which nothing is seen, whatever its scales)
    }
  }
  uint16_t* out = p.out + (int64_t)row * p.out_stride + (int64_t)head * HEAD + lane * PER;
#pragma unroll
  for (int j = 0; j < PER; j++) out[j] = top == -INFINITY ? 0 : DT::from_f32(v[j] / sum);
}

// ---------------------------------------------------------------------------------------------------------------------
// how a call is cut: host side, from what the caller bounds
// ---------------------------------------------------------------------------------------------------------------------
struct WindowPart { int cols, waves, col_tiles, splits, split_tiles; };   // col_tiles: of a sequence (rows), of the batch (flash)
struct WindowPlan {
  WindowPart rows, flash;       // col_tiles 0: not launched
  bool all_flash;               // sequences of few rows too
  int row_cols;                 // sequences of more columns are prompts
};

// columns (rows x heads per kv head) up to which a sequence is served 16 or 32 at a time
constexpr int WA_ROWS_COLS = 64;

// 64-token tiles that `cols` columns see at most: the window of their first row, their own rows, an unaligned start, the sinks
static int64_t window_tiles(int cols, int G, int max_seq_len, int window, int sinks) {
  int64_t tiles = ((int64_t)max_seq_len + 63) / 64;
  if (window)
    tiles = std::min(tiles + 1, ((int64_t)std::min(window, max_seq_len) + (cols + G - 1) / G + 15 + 63) / 64 +
                                    ((int64_t)std::min(sinks, max_seq_len) + 63) / 64);
  return std::max<int64_t>(tiles, 1);
}
static void window_cut(WindowPart& w, int64_t tiles, int64_t want, int least_tiles) {
  w.split_tiles = (int)std::max<int64_t>(least_tiles, (tiles + want - 1) / want);
  w.splits = (int)((tiles + w.split_tiles - 1) / w.split_tiles);
}

static WindowPlan window_plan(int num_seqs, int num_rows, int num_heads, int num_kv_heads, int kv_type, int max_query_len, int max_seq_len,
                              int window, int sinks) {
  WindowPlan w{};
  const int G = num_heads / num_kv_heads;
  const int64_t cols = (int64_t)max_query_len * G;
  const bool prompts = cols > WA_ROWS_COLS;
  const int64_t flash_tiles = window_tiles(WA_FLASH_COLS, G, max_seq_len, window, sinks);
  // Next to prompts the decode kernel takes rows of up to 16 columns, which is one query each, and drafts go with the prompts:
  // 200 decode rows and a prompt of 1800 354 -> 265 us, 64 drafts of five rows and one of 1500 204 -> 183.  Not over contexts
  // past 8192, which a workgroup of the prompt kernel walks whole (one draft at 30000 679 us, with the decode kernel 149).
  w.row_cols = prompts && flash_tiles <= 128 ? 16 : WA_ROWS_COLS;
  // Decode rows between prompts have the decode kernel, unless they are few and no context is longer than 32 tiles: workgroups
  // of the prompt kernel then walk them while the prompts' own run, which costs less than a launch (five sequences under a
  // window of 512 50 us, apart 57; eight decode rows and two prompts 45 and 54; but 30 rows and a prompt 44 and 43, 100 rows 57 and
  // 40, 200 rows of 1500 tokens 202 and 109).  And the bounds may say that every sequence has max_query_len rows.
  w.all_flash = prompts && ((flash_tiles <= 32 && (int64_t)num_seqs * num_kv_heads <= 128) || (int64_t)num_seqs * max_query_len == num_rows);
  if (!w.all_flash) {
    const int64_t mine = std::min<int64_t>(cols, w.row_cols);
    // 32 columns to a workgroup read a draft's K and V once instead of twice; a 16-bit tile leaves no registers for it, and next to
    // prompts most sequences have one row
    w.rows.cols = !prompts && mine > 16 && kv_type != MI355Q_KV_16 ? 32 : 16;
    w.rows.col_tiles = (int)((mine + w.rows.cols - 1) / w.rows.cols);
    const int64_t tiles = window_tiles(w.rows.cols, G, max_seq_len, window, sinks);
    const int64_t groups = (int64_t)num_seqs * num_kv_heads * w.rows.col_tiles;
    w.rows.waves = groups <= 256 || w.rows.cols == 32 ? 8 : 4;
    // One workgroup to a CU is what up to 64 of them are cut into.  More (9 sequences of 8 kv heads) fill the chip by
    // themselves, but lengths differ: contexts are cut into stretches of 4096 tokens and more, 32 at
    // most, and fewer of more sequences (their sums take room).  Against no cut: one context of
    // 131072 among 31 of 2000 701 -> 171 us, 16 / 32 / 64 contexts spread from 1000 to 30000 132 -> 125, 258 -> 228, 465 -> 427,
    // 32 of 16384 each 201 -> 211; contexts up to 4096 under a bound of 131072 70 -> 76 (156 with a sequence's stretches
    // side by side in the grid).  What is shorter than two stretches stays whole: 64 contexts up to 4096 in four stretches took 84 us,
    // whole 71; 32 decode rows under a window of 4096 in two 91, whole 84.
    const int64_t stretches = groups <= 64 ? 256 / groups : std::max<int64_t>(256 / groups, std::clamp<int64_t>(std::min(tiles / 64, 16384 / groups), 1, 32));
    // A stretch has a tile for each wave at least, and two for each stay whole: the join is a launch of 4 us.  One sequence, in a
    // graph: 1000 tokens whole 11.1 us, in two 11.9; 2000 whole 15.7, in four 11.8; 4000 in four 13.9, in eight 12.2; 8000 15.8 and 14.0.
    // (Calls one by one from Python are bound by the host, and the join is a second launch there: 2000 tokens whole 20 us, in four 24.)
    window_cut(w.rows, tiles, stretches, (tiles <= 2 * w.rows.waves ? 2 : 1) * w.rows.waves);
  }
  if (prompts) {
    // Column tiles of the whole batch at most.  (Sequences times the longest one's tiles were 445 us for 200 decode rows and
    // a prompt of 1800, against 354.)
    const int64_t all = (int64_t)num_rows * G, least = w.all_flash ? 1 : w.row_cols + 1;
    const int64_t tiles = std::min(num_seqs * ((cols + WA_FLASH_COLS - 1) / WA_FLASH_COLS), all / WA_FLASH_COLS + std::min<int64_t>(num_seqs, all / least));
    if (tiles > 0) {              // (0: fewer rows than a prompt has)
      w.flash.cols = WA_FLASH_COLS;
      w.flash.waves = WA_WAVES;
      w.flash.col_tiles = (int)tiles;
      window_cut(w.flash, flash_tiles, std::max<int64_t>(1, (256 + num_kv_heads * tiles - 1) / (num_kv_heads * tiles)), 16);
    }
  }
  return w;
}

// a launch has fewer than 2^32 threads (taken apart by divisions: the products may pass 64 bits)
static bool window_fits(const WindowPlan& w, int num_seqs, int num_kv_heads) {
  auto fits = [&](const WindowPart& a, int64_t tiles) {
    const int64_t most = ((int64_t)1 << 32) - 1, of_tile = std::max<int64_t>((int64_t)a.splits * 64 * a.waves, a.splits > 1 ? a.cols / 4 * 256 : 0);
    return !a.col_tiles || tiles <= most / num_kv_heads / a.col_tiles / of_tile;
  };
  return fits(w.rows, num_seqs) && fits(w.flash, 1);
}

// Partial sums of decode rows: room for so many rows of a sequence, or (0) for the rows as they are numbered, if that is less.
static int window_part_rows(const WindowPlan& w, int num_seqs, int num_rows, int max_query_len, int G) {
  const int64_t of_seq = (std::min<int64_t>((int64_t)max_query_len * G, w.row_cols) + G - 1) / G;
  return num_seqs * of_seq < num_rows ? (int)of_seq : 0;
}

// floats of the partial sums' outputs, of one head dim (maxima and sums follow); the two kinds of row take turns with them
static int64_t window_partials(const WindowPlan& w, int num_seqs, int num_rows, int num_heads, int num_kv_heads, int max_query_len) {
  const int of_seq = window_part_rows(w, num_seqs, num_rows, max_query_len, num_heads / num_kv_heads);
  const int64_t rows = w.rows.splits > 1 ? (of_seq ? (int64_t)num_seqs * of_seq : num_rows) * w.rows.splits : 0;
  const int64_t flash = w.flash.splits > 1 ? (int64_t)num_rows * w.flash.splits : 0;
  return std::max(rows, flash) * num_heads;
}

template <typename DT, int KV, int HEAD>
static int launch_window(WindowParams p, const WindowPlan& w, int part_rows, hipStream_t s) {
  auto tiles = [&](const WindowPart& a) { return (int64_t)(&a == &w.rows ? p.num_seqs : 1) * p.num_kv_heads * a.col_tiles; };
  auto groups = [&](const WindowPart& a) { return tiles(a) * a.splits; };
  auto merges = [&](const WindowPart& a) { return tiles(a) * (a.cols / 4); };
  const int announced = p.longest_cols;
  for (int kind = 0; kind < 2; kind++) {
    const WindowPart& a = kind ? w.flash : w.rows;
    if (!a.col_tiles) continue;
    p.col_tiles = a.col_tiles, p.splits = a.splits;
    p.split_tiles = a.splits == 1 ? INT_MAX : a.split_tiles;
    p.part_rows = kind ? 0 : part_rows;
    p.min_cols = kind && !w.all_flash ? w.row_cols + 1 : 0;
    p.max_cols = kind || !w.flash.col_tiles ? INT_MAX : w.row_cols;
    p.longest_cols = kind ? announced : std::min(announced, w.row_cols);
    p.lds_cols = std::min(16, p.longest_cols);
    const dim3 grid((unsigned)groups(a)), wg(64 * a.waves);
    const size_t lds = (size_t)a.waves * p.lds_cols * (HEAD + 4) * sizeof(float);
    if (kind) {
      // One scale for the whole cache goes into the logits' factor and the result's: no scales are read, no codes multiplied.
      // Prompts of 2047 rows and less on 64-wide heads behind a window of 512: 57.1 us as block scales, 47.0 us so.
      if (KV == KVF8 && p.scale_block_stride == 0 && p.scale_head_stride == 0)
        hipLaunchKernelGGL((window_flash_kernel<DT, KV == KVF8 ? KVF8_ONE : KV, HEAD, WA_WAVES>), grid, wg, 0, s, p);
      else
        hipLaunchKernelGGL((window_flash_kernel<DT, KV, HEAD, WA_WAVES>), grid, wg, 0, s, p);
    } else if (a.cols == 32) {
      if constexpr (KV != KV16) hipLaunchKernelGGL((window_rows_kernel<DT, KV, HEAD, 2, 8>), grid, wg, lds, s, p);
    } else if (a.waves == 8) {
      hipLaunchKernelGGL((window_rows_kernel<DT, KV, HEAD, 1, 8>), grid, wg, lds, s, p);
    } else {
      hipLaunchKernelGGL((window_rows_kernel<DT, KV, HEAD, 1, 4>), grid, wg, lds, s, p);
    }
    if (int e = check_launch("paged_window_attention")) return e;
    if (a.splits > 1) {
      const dim3 joins((unsigned)merges(a));
      if (kind) hipLaunchKernelGGL((window_merge_kernel<DT, HEAD, WA_FLASH_COLS>), joins, dim3(256), 0, s, p);
      else if (a.cols == 32) hipLaunchKernelGGL((window_merge_kernel<DT, HEAD, 32>), joins, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((window_merge_kernel<DT, HEAD, 16>), joins, dim3(256), 0, s, p);
      if (int e = check_launch("paged_window_attention")) return e;
    }
  }
  return MI355Q_OK;
}

}  // namespace mi355q

using namespace mi355q;

static bool heads_fit(int num_heads, int num_kv_heads) {
  return num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0 && num_heads / num_kv_heads <= 16;
}

extern "C" size_t mi355q_paged_window_attention_workspace_bytes(int num_seqs, int num_rows, int num_heads, int num_kv_heads, int head_size,
                                                                int max_query_len, int max_seq_len, int window, int sinks, int kv_type) {
  // (bounds that the attention itself refuses need no scratch; the plan divides by the heads to a kv head)
  if (num_seqs <= 0 || num_rows <= 0 || !heads_fit(num_heads, num_kv_heads) || max_query_len <= 0 || max_seq_len <= 0 || window < 0 || sinks < 0)
    return 0;
  const WindowPlan w = window_plan(num_seqs, num_rows, num_heads, num_kv_heads, kv_type, max_query_len, max_seq_len, window, sinks);
  if (!window_fits(w, num_seqs, num_kv_heads)) return 0;
  return (size_t)window_partials(w, num_seqs, num_rows, num_heads, num_kv_heads, max_query_len) * (head_size + 2) * sizeof(float);
}

extern "C" int mi355q_paged_window_attention(void* out, int64_t out_stride, const void* query, int64_t q_stride, const void* key_cache,
                                             const void* value_cache, int64_t kv_block_stride, int64_t kv_head_stride, int num_blocks,
                                             int num_rows, int num_seqs, int num_heads, int num_kv_heads, int head_size, float scale,
                                             const int32_t* block_tables, int max_blocks_per_seq, const int32_t* seq_lens,
                                             const int32_t* query_start_loc, int max_query_len, int block_size, int max_seq_len,
                                             int window, int sinks, int dtype, int kv_type, const float* k_scale, const float* v_scale,
                                             int64_t scale_block_stride, int64_t scale_head_stride, void* workspace,
                                             size_t workspace_bytes, mi355q_stream_t stream) {
  MI355Q_REQUIRE(dtype == MI355Q_BF16 || dtype == MI355Q_FP16, "paged_window_attention: dtype must be bf16 or fp16");
  MI355Q_REQUIRE(kv_type == MI355Q_KV_16 || kv_type == MI355Q_KV_FP8 || kv_type == MI355Q_KV_INT8, "paged_window_attention: bad cache type %d", kv_type);
  MI355Q_REQUIRE(num_seqs >= 0 && num_rows >= 0, "paged_window_attention: bad sizes");
  if (num_seqs == 0 || num_rows == 0) return MI355Q_OK;
  MI355Q_REQUIRE(out && query && key_cache && value_cache && block_tables && seq_lens, "paged_window_attention: null pointer");
  MI355Q_REQUIRE(kv_type == MI355Q_KV_16 || (k_scale && v_scale), "paged_window_attention: an 8-bit cache needs k_scale / v_scale");
  MI355Q_REQUIRE(head_size == 64 || head_size == 128, "paged_window_attention: head_size %d (64 or 128)", head_size);
  MI355Q_REQUIRE(heads_fit(num_heads, num_kv_heads),
                 "paged_window_attention: %d query heads over %d kv heads (1 to 16 to each)", num_heads, num_kv_heads);
  MI355Q_REQUIRE(block_size >= 16 && block_size <= 256 && block_size % 16 == 0, "paged_window_attention: block size %d (a multiple of 16 up to 256)", block_size);
  MI355Q_REQUIRE(num_blocks > 0 && max_blocks_per_seq > 0 && (int64_t)max_blocks_per_seq * block_size < (int64_t)1 << 30,
                 "paged_window_attention: bad block table");
  MI355Q_REQUIRE(max_query_len > 0 && max_seq_len > 0 && window >= 0 && sinks >= 0, "paged_window_attention: negative or zero length");
  MI355Q_REQUIRE(query_start_loc || num_seqs <= num_rows, "paged_window_attention: %d rows for %d sequences", num_rows, num_seqs);
  const int eb = kv_type == MI355Q_KV_16 ? 2 : 1;
  const int64_t page = (int64_t)head_size * block_size;
  MI355Q_REQUIRE(kv_head_stride >= page && kv_block_stride >= page && kv_head_stride * eb % 16 == 0 && kv_block_stride * eb % 16 == 0,
                 "paged_window_attention: cache strides");
  MI355Q_REQUIRE((((uintptr_t)key_cache | (uintptr_t)value_cache | (uintptr_t)query) & 15) == 0 && q_stride % 8 == 0,
                 "paged_window_attention: caches and query rows must be 16-byte aligned");
  MI355Q_REQUIRE(((uintptr_t)out & 3) == 0 && out_stride % 2 == 0, "paged_window_attention: output rows must be 4-byte aligned");
  const WindowPlan w = window_plan(num_seqs, num_rows, num_heads, num_kv_heads, kv_type, max_query_len, max_seq_len, window, sinks);
  MI355Q_REQUIRE(window_fits(w, num_seqs, num_kv_heads), "paged_window_attention: too many workgroups");
  const int64_t partials = window_partials(w, num_seqs, num_rows, num_heads, num_kv_heads, max_query_len);
  const size_t need = (size_t)partials * (head_size + 2) * sizeof(float);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(MI355Q_ENOSPACE, "paged_window_attention: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, need);
  MI355Q_REQUIRE(!need || ((uintptr_t)workspace & 15) == 0, "paged_window_attention: workspace must be 16-byte aligned");
  WindowParams p{};
  p.out = (uint16_t*)out;
  p.q = (const uint16_t*)query;
  p.kc = (const unsigned char*)key_cache;
  p.vc = (const unsigned char*)value_cache;
  p.ks = k_scale, p.vs = v_scale;
  p.tables = block_tables, p.seq_lens = seq_lens, p.starts = query_start_loc;
  p.part_o = (float*)workspace;
  p.part_ml = (float*)workspace + partials * head_size;
  p.out_stride = out_stride, p.q_stride = q_stride;
  p.block_stride = kv_block_stride * eb, p.head_stride = kv_head_stride * eb;
  p.scale_block_stride = scale_block_stride, p.scale_head_stride = scale_head_stride;
  p.scale = scale;
  p.num_seqs = num_seqs, p.num_rows = num_rows, p.num_heads = num_heads, p.num_kv_heads = num_kv_heads, p.group = num_heads / num_kv_heads;
  p.num_blocks = num_blocks, p.table_width = max_blocks_per_seq;
  p.bs = block_size;
  const int pieces = block_size / 16;
  p.page_magic = pieces == 1 ? 0 : (int)(((1ull << 32) + pieces - 1) / pieces);
  p.window = std::min(window, 1 << 30), p.sinks = sinks;
  const int part_rows = window_part_rows(w, num_seqs, num_rows, max_query_len, p.group);
  p.longest_cols = (int)std::min<int64_t>((int64_t)max_query_len * p.group, INT_MAX);
  p.out16 = ((uintptr_t)out & 15) == 0 && out_stride % 8 == 0;
  hipStream_t s = (hipStream_t)stream;
#define BY_KV(DT, HD)                                                                                                     \
  (kv_type == MI355Q_KV_16 ? launch_window<DT, KV16, HD>(p, w, part_rows, s)                                                        \
                           : kv_type == MI355Q_KV_FP8 ? launch_window<DT, KVF8, HD>(p, w, part_rows, s) : launch_window<DT, KVI8, HD>(p, w, part_rows, s))
  if (dtype == MI355Q_BF16) return head_size == 128 ? BY_KV(BF16, 128) : BY_KV(BF16, 64);
  return head_size == 128 ? BY_KV(FP16, 128) : BY_KV(FP16, 64);
#undef BY_KV
}
