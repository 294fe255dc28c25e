// Append to a paged KV cache held in 8 bits with one fp32 scale for each (block of tokens, kv head) of K and of V,
// the position rotation applied on the way.
//   K cache [blocks, kv_heads, head/16, block_size, 16], V cache [blocks, kv_heads, head, block_size] (bytes),
//   scales [blocks, kv_heads]; a code c stands for c * scale (int8, |c| <= 127, or e4m3fn).
//
// For a block b and head h that a call writes, with first = the smallest offset written:
//   s_old = first > 0 ? scale[b, h] : 0          offset 0 restarts a block: what it held before is void
//   s_new = max(s_old, max |x| * (1 / QMAX))     over the call's tokens in b
//   codes at offsets < first become round(c * (s_old / s_new)) where s_new > s_old
//   new codes are round(x / s_new), 0 where s_new is 0; other offsets keep their bytes.
// A run of tokens that skipped or repeated slots stretch over more than 64 positions (a lane each) is appended 64 positions at a
// time, as so many calls would: each stretch is a call's tokens in what is said above.
// A value that is not finite makes its block's scale NaN: reads of the block are NaN until it is restarted.
//
// The tokens of one block follow one another in slot_mapping (tokens without a slot may stand between them), so a block's
// work belongs to the wave of the run's first token: the largest magnitude is known before anything is encoded, no
// atomics, no second launch, and the result does not depend on any order of execution.
//
// Bound by HBM for prompts: 8192 tokens of 32 query and 8 kv heads of 128, int8, 186.8 MB in 38 to 40 us, 4.7 to 4.9 TB/s, where two
// batches take turns, 45 us, 4.2 TB/s, over eight, of which the caches hold nothing (a large copy reaches 5.15).  A decode step is a
// chain of round trips: slots, then rows, angles, scales and the block, then the stores: 6 to 7 us for one token, 6.5 to 8 for 64; 508
// tokens with half of a 64-wide head rotated 9.6.
#include "common.h"

// one rounding per operation: the results equal a sequence of separate fp32 multiplications and additions
#pragma clang fp contract(off)

namespace mi355q {

struct AppendParams {
  const int64_t* positions;
  const uint16_t* q;
  uint16_t* q_out;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_stride, q_out_stride, k_stride, v_stride;
  int num_tokens, num_heads, num_kv_heads;
  const void* cos_sin;
  int cos_dtype, rot, max_pos, is_neox;
  int rot_mode;           // ROT_*
  int aligned;            // every row of q, q_out, k and v starts on 16 bytes
  unsigned char* kc;
  unsigned char* vc;
  int64_t block_stride;   // bytes from block to block (both caches)
  float* ks;
  float* vs;
  int64_t scale_block_stride, scale_head_stride;
  const int64_t* slots;
  int num_slots;          // blocks * block size: slots outside [0, num_slots) are skipped
  int bs, page_magic;     // block of slot s = page_of(s / 16)
  int kv_groups;          // workgroups that append; the rest rotate the query
  int tokens_per_wave;    // token positions an appending wave looks at
};

// ROT_HALVES / ROT_PAIRS: NeoX / GPT-J pairing where runs of 16 elements turn as a whole and the angles can be loaded as
// vectors; ROT_ANY: every other even number of rotated elements, element by element
enum { ROT_NONE = 0, ROT_HALVES = 1, ROT_PAIRS = 2, ROT_ANY = 3 };

// n / d for n * d < 2^32 with magic = ceil(2^32 / d); magic 0 stands for d = 1
__device__ inline int page_of(int n, int magic) { return magic ? (int)__umulhi((unsigned)n, (unsigned)magic) : n; }

struct Row16 { u32x4 a, b; };   // 16 consecutive 16-bit elements

__device__ inline Row16 load16(const uint16_t* p, bool aligned) {
  Row16 r;
  if (aligned) {
    r.a = reinterpret_cast<const u32x4*>(p)[0];
    r.b = reinterpret_cast<const u32x4*>(p)[1];
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      r.a[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
      r.b[i] = (uint32_t)p[8 + 2 * i] | ((uint32_t)p[9 + 2 * i] << 16);
    }
  }
  return r;
}
__device__ inline void store16(uint16_t* p, const Row16& r, bool aligned) {
  if (aligned) {
    reinterpret_cast<u32x4*>(p)[0] = r.a;
    reinterpret_cast<u32x4*>(p)[1] = r.b;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      p[2 * i] = (uint16_t)r.a[i], p[2 * i + 1] = (uint16_t)(r.a[i] >> 16);
      p[8 + 2 * i] = (uint16_t)r.b[i], p[9 + 2 * i] = (uint16_t)(r.b[i] >> 16);
    }
  }
}
template <typename DT>
__device__ inline float elem(const Row16& x, int i) {
  const uint32_t w = i < 8 ? x.a[i >> 1] : x.b[(i - 8) >> 1];
  return DT::to_f32((uint16_t)((i & 1) ? w >> 16 : w & 0xffff));
}
template <typename DT>
__device__ inline void put2(Row16& r, int i, float lo, float hi) {
  const uint32_t w = pack2<DT>(lo, hi);
  if (i < 8) r.a[i >> 1] = w;
  else r.b[(i - 8) >> 1] = w;
}
__device__ inline float table_at(const void* c, int64_t i, int dtype) {
  if (dtype == MI355Q_FP32) return reinterpret_cast<const float*>(c)[i];
  const uint16_t h = reinterpret_cast<const uint16_t*>(c)[i];
  return dtype == MI355Q_BF16 ? BF16::to_f32(h) : FP16::to_f32(h);
}
template <int N>
__device__ inline void load_table(float* out, const void* c, int64_t i, int dtype) {
  if (dtype == MI355Q_FP32) {
#pragma unroll
    for (int j = 0; j < N / 4; j++) {
      const f32x4 v = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(c) + i)[j];
#pragma unroll
      for (int k = 0; k < 4; k++) out[4 * j + k] = v[k];
    }
  } else {
#pragma unroll
    for (int j = 0; j < N / 8; j++) {
      const u32x4 v = reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(c) + i)[j];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const uint16_t lo = (uint16_t)v[k], hi = (uint16_t)(v[k] >> 16);
        out[8 * j + 2 * k] = dtype == MI355Q_BF16 ? BF16::to_f32(lo) : FP16::to_f32(lo);
        out[8 * j + 2 * k + 1] = dtype == MI355Q_BF16 ? BF16::to_f32(hi) : FP16::to_f32(hi);
      }
    }
  }
}

// cos and sin of 16 elements from d0 on (halves), or of the 8 pairs they form
struct Angles { float c[16], s[16]; };

// row of the table for token t; a position outside of it is brought to its ends
__device__ inline int position(const AppendParams& p, int t) {
  const int64_t pos = p.positions[t];
  return pos < 0 ? 0 : pos >= p.max_pos ? p.max_pos - 1 : (int)pos;
}
__device__ inline void load_angles(Angles& a, const AppendParams& p, int pos, int d0) {
  const int e = p.rot / 2;
  const int64_t row = (int64_t)pos * p.rot;
  if (p.rot_mode == ROT_HALVES) {
    const int j = d0 < e ? d0 : d0 - e;
    load_table<16>(a.c, p.cos_sin, row + j, p.cos_dtype);
    load_table<16>(a.s, p.cos_sin, row + e + j, p.cos_dtype);
  } else {
    load_table<8>(a.c, p.cos_sin, row + d0 / 2, p.cos_dtype);
    load_table<8>(a.s, p.cos_sin, row + e + d0 / 2, p.cos_dtype);
  }
}

// 16 elements x of a head from d0 on, turned and rounded to the model's type; y: their partners under ROT_HALVES
template <typename DT>
__device__ inline Row16 rotate16(const Row16& x, const Row16& y, const Angles& a, bool halves, bool first) {
  Row16 r;
  if (halves) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float s0 = first ? -a.s[i] : a.s[i], s1 = first ? -a.s[i + 1] : a.s[i + 1];
      put2<DT>(r, i, elem<DT>(x, i) * a.c[i] + elem<DT>(y, i) * s0, elem<DT>(x, i + 1) * a.c[i + 1] + elem<DT>(y, i + 1) * s1);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float u = elem<DT>(x, i), w = elem<DT>(x, i + 1), c = a.c[i / 2], s = a.s[i / 2];
      put2<DT>(r, i, u * c - w * s, w * c + u * s);
    }
  }
  return r;
}

// ROT_ANY: elements d0 .. d0 + 15 of the head at x
template <typename DT>
__device__ inline Row16 rotate16_any(const uint16_t* x, int d0, const AppendParams& p, int pos) {
  const int e = p.rot / 2;
  const int64_t row = (int64_t)pos * p.rot;
  Row16 r;
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    float z[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int d = d0 + i + j;
      z[j] = DT::to_f32(x[d]);
      if (d < p.rot) {
        const int at = p.is_neox ? (d < e ? d : d - e) : d >> 1;
        const bool first = p.is_neox ? d < e : !(d & 1);
        const int other = p.is_neox ? (first ? d + e : d - e) : d ^ 1;
        const float c = table_at(p.cos_sin, row + at, p.cos_dtype);
        const float s = table_at(p.cos_sin, row + e + at, p.cos_dtype);
        z[j] = z[j] * c + DT::to_f32(x[other]) * (first ? -s : s);
      }
    }
    put2<DT>(r, i, z[0], z[1]);
    __builtin_amdgcn_sched_barrier(0);   // a pair at a time: the rare form must not set the kernel's registers
  }
  return r;
}

// 8 pairs (x, y) held as packed 16-bit values turned by their angles
template <typename DT>
__device__ inline void rotate8(u32x4& x, u32x4& y, const u32x4 c, const u32x4 s) {
  auto lo = [](uint32_t w) { return DT::to_f32((uint16_t)w); };
  auto hi = [](uint32_t w) { return DT::to_f32((uint16_t)(w >> 16)); };
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float x0 = lo(x[e]), x1 = hi(x[e]), y0 = lo(y[e]), y1 = hi(y[e]), c0 = lo(c[e]), c1 = hi(c[e]), s0 = lo(s[e]), s1 = hi(s[e]);
    x[e] = pack2<DT>(x0 * c0 - y0 * s0, x1 * c1 - y1 * s1);
    y[e] = pack2<DT>(y0 * c0 + x0 * s0, y1 * c1 + x1 * s1);
  }
}

// largest magnitude of 16 elements as the low 15 bits of the 16-bit type: ordered like the values, infinities and NaN on top
__device__ inline uint32_t top_bits(const Row16& x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    m = max(m, max(x.a[i] & 0x7fffu, (x.a[i] >> 16) & 0x7fffu));
    m = max(m, max(x.b[i] & 0x7fffu, (x.b[i] >> 16) & 0x7fffu));
  }
  return m;
}
__device__ inline uint32_t wave_umax(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true));
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(r[0], r[1]);
}
// the scale that holds a largest magnitude given by its bits; NaN where it is not finite
template <typename DT>
__device__ inline float scale_of(uint32_t bits, float qmax) {
  const uint32_t inf = DT::id == MI355Q_BF16 ? 0x7f80u : 0x7c00u;
  return bits >= inf ? __builtin_nanf("") : DT::to_f32((uint16_t)bits) * (1.0f / qmax);
}

// four quotients as codes.  int8: 1.5 * 2^23 + x holds x, rounded to the nearest integer (ties to even), in its low bits
template <bool INT8>
__device__ inline uint32_t encode4(float a, float b, float c, float d) {
  if constexpr (INT8) {
    auto bits = [](float v) { return __float_as_uint(v + 12582912.0f); };
    const uint32_t lo = __builtin_amdgcn_perm(bits(b), bits(a), 0x0c0c0400u), hi = __builtin_amdgcn_perm(bits(d), bits(c), 0x04000c0cu);
    return lo | hi;
  } else {
    auto cut = [](float v) { return __builtin_fminf(__builtin_fmaxf(v, -448.0f), 448.0f); };
    const int r = __builtin_amdgcn_cvt_pk_fp8_f32(cut(a), cut(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(cut(c), cut(d), r, true);
  }
}

// Division by a block's scale: with the reciprocal y of s, q = x y and q + (x - q s) y (both fused) is the correctly rounded
// quotient (Markstein 1990; for the one mantissa of all ones it may be a neighbour), three instructions instead of a
// dozen.  x and s are brought to the middle of the range first, by a power of two: 1 / s is finite, nothing underflows.
struct Divisor {
  float s, y, up;
  __device__ inline explicit Divisor(float scale) {
    up = scale < 0x1p-60f ? 0x1p90f : scale > 0x1p60f ? 0x1p-64f : 1.f;
    s = scale * up;
    y = scale > 0.f ? 1.f / s : 0.f;   // (0: every value is 0; NaN: a value was not finite; the codes are 0 in both)
  }
  __device__ inline float quotient(float x) const {
    x *= up;
    const float q = x * y;
    return __builtin_fmaf(__builtin_fmaf(-q, s, x), y, q);
  }
};
template <typename DT, bool INT8>
__device__ inline u32x4 encode16(const Row16& x, const Divisor& d) {
  u32x4 r = {0, 0, 0, 0};
  if (d.y != 0.f) {
#pragma unroll
    for (int i = 0; i < 4; i++)
      r[i] = encode4<INT8>(d.quotient(elem<DT>(x, 4 * i)), d.quotient(elem<DT>(x, 4 * i + 1)), d.quotient(elem<DT>(x, 4 * i + 2)),
                           d.quotient(elem<DT>(x, 4 * i + 3)));
  }
  return r;
}
template <bool INT8>
__device__ inline u32x4 rescale16(u32x4 w, float ratio) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    float f[4];
    if constexpr (INT8) {
#pragma unroll
      for (int j = 0; j < 4; j++) f[j] = (float)(int)(signed char)(w[i] >> (8 * j));
    } else {
      const f32x2 lo = fp8x2_to_f32(w[i], false), hi = fp8x2_to_f32(w[i], true);
      f[0] = lo[0], f[1] = lo[1], f[2] = hi[0], f[3] = hi[1];
    }
    w[i] = encode4<INT8>(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
  }
  return w;
}
// byte mask of a 16-byte piece from a 16-bit mask
__device__ inline u32x4 byte_mask(uint32_t m) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t n = (m >> (4 * i)) & 0xf;
    r[i] = ((n & 1) | ((n & 2) << 7) | ((n & 4) << 14) | ((n & 8) << 21)) * 0xffu;
  }
  return r;
}

// One wave appends tokens t + i of one kv head for the bits i of `here`, all in block `blk`; lane i holds token t + i's
// offset there and its row of the angles' table.  A token takes HEAD / 16 lanes of 16 elements, 64 / (HEAD / 16) tokens a pass;
// the first two passes stay in registers between the search for the largest magnitude and the encoding (a 16-token block
// of 128-wide heads is two), later ones are read again.  K codes go out as the cache's own 16-byte pieces; V codes are
// turned in LDS, so that the cache takes 16 tokens of a head dim at once.  What the block held (needed where the scale
// grows, and around the new tokens of V) is requested together with the new rows: a decode step is three round trips.
// FORM_WHOLE: NeoX pairing over the whole head, 16-bit angles of the model's type, aligned rows; FORM_NONE: no rotation, aligned
// rows -- nearly every call, in kernels that the general form's code (60 KB) does not weigh on.  Over eight batches in turn, in a graph,
// general form and this: 8192 prompt tokens of 32 + 8 heads 89 and 45 us, without rotation 61 and 46; one token 7.8 and 5.8, 6.4 and 5.6.
// Under FORM_WHOLE a lane holds 8 elements of K and their 8 partners.
// FORM_PART: the other rotations that turn runs of 16, aligned rows: half of each head in pairs 81 and 75 us, in halves 89 and 81, 64
// decode tokens 8.2 and 6.9, 8.5 and 7.1: the query has one pass on its way where FORM_WHOLE has four, and in halves every run is
// read once more for its partners.  (One batch again and again 62 us and, for 64 tokens, 7.8; with registers for three workgroups to
// a CU instead of two, as the two forms above have, 59 and 9.8.)
enum { FORM_ANY = 0, FORM_WHOLE = 1, FORM_NONE = 2, FORM_PART = 3 };
template <typename DT, bool INT8, int HEAD, int FORM>
__device__ __forceinline__ void append_run(const AppendParams& p, int t, uint64_t here, int blk, int offset, int pos, int h,
                                           unsigned char* stage, int lane) {
  constexpr int LPT = HEAD / 16, TPP = 64 / LPT, HELD = 2, OLD = 2;
  constexpr float QMAX = INT8 ? 127.0f : 448.0f;
  const int chunk = lane % LPT, sub = lane / LPT, d0 = chunk * 16;
  const bool turns = (p.rot_mode == ROT_HALVES || p.rot_mode == ROT_PAIRS) && d0 < p.rot;
  const bool halves = p.rot_mode == ROT_HALVES, first_half = d0 < p.rot / 2;
  const int partner = turns && halves ? (first_half ? p.rot / 2 : -(p.rot / 2)) : 0;

  // which tokens stand: of several for one slot the last; and the offsets they take
  const int lead = __builtin_ctzll(here), n = 64 - __builtin_clzll(here);
  bool dead = !((here >> lane) & 1);
  int first = __builtin_amdgcn_readlane(offset, lead);
  uint64_t taken;
  const int next = __shfl_down(offset, 1, 64);
  if (lead == 0 && (here & (here + 1)) == 0 && __ballot(lane + 1 < n && next != offset + 1) == 0) {
    taken = (n == 64 ? ~0ull : (1ull << n) - 1) << first;
  } else {
    taken = 0;
    for (int j = lead; j < n; j++) {
      if (!((here >> j) & 1)) continue;
      const int oj = __shfl(offset, j, 64);
      taken |= 1ull << oj;
      dead |= lane < j && oj == offset;
    }
    first = __builtin_ctzll(taken);
  }
  const uint64_t stand = ~__ballot(dead);

  const int passes = (n + TPP - 1) / TPP, per_row = p.bs >> 4;
  float* const ks = p.ks + blk * p.scale_block_stride + h * p.scale_head_stride;
  float* const vs = p.vs + blk * p.scale_block_stride + h * p.scale_head_stride;
  unsigned char* const kb = p.kc + blk * p.block_stride + (int64_t)h * HEAD * p.bs;
  unsigned char* const vb = p.vc + blk * p.block_stride + (int64_t)h * HEAD * p.bs;

  auto load = [&](int i, Row16& k, Row16& v) {
    const int j = min(i, n - 1);
    const int64_t row = t + j;
    const uint16_t* kr = p.k + row * p.k_stride + (int64_t)h * HEAD;
    const int at = __shfl(pos, j, 64);
    v = load16(p.v + row * p.v_stride + (int64_t)h * HEAD + d0, FORM != FORM_ANY || p.aligned);
    if constexpr (FORM == FORM_NONE) {
      k = load16(kr + d0, true);
    } else if constexpr (FORM == FORM_WHOLE) {
      const uint16_t* angle = reinterpret_cast<const uint16_t*>(p.cos_sin) + (int64_t)at * HEAD + 8 * chunk;
      k.a = *reinterpret_cast<const u32x4*>(kr + 8 * chunk);
      k.b = *reinterpret_cast<const u32x4*>(kr + HEAD / 2 + 8 * chunk);
      rotate8<DT>(k.a, k.b, *reinterpret_cast<const u32x4*>(angle), *reinterpret_cast<const u32x4*>(angle + HEAD / 2));
    } else if (FORM == FORM_ANY && p.rot_mode == ROT_ANY) {
      k = rotate16_any<DT>(kr, d0, p, at);
    } else {
      k = load16(kr + d0, FORM != FORM_ANY || p.aligned);
      if (turns) {
        Angles a;
        load_angles(a, p, at, d0);
        const Row16 other = halves ? load16(kr + d0 + partner, FORM != FORM_ANY || p.aligned) : k;
        k = rotate16<DT>(k, other, a, halves, first_half);
      }
    }
  };
  auto stands = [&](int i) { return i < 64 && ((stand >> i) & 1); };

  // what the block holds, the first OLD pieces of a lane; the scales it is held under
  u32x4 k_old[OLD], v_old[OLD];
  float ks_old = 0.f, vs_old = 0.f;
  auto kept = [&](int i) { return i < LPT * p.bs && i % p.bs < first; };                        // a K piece of an earlier token
  auto touched = [&](int i, uint32_t& fresh, int& before) {                                      // a V piece with new or earlier tokens
    const int g = i % per_row;
    fresh = (uint32_t)(taken >> (16 * g)) & 0xffffu;
    before = min(max(first - 16 * g, 0), 16);
    return i < HEAD * per_row;
  };
  if (first > 0) {
    ks_old = *ks;
    vs_old = *vs;
#pragma unroll
    for (int j = 0; j < OLD; j++)
      if (kept(lane + 64 * j)) k_old[j] = reinterpret_cast<const u32x4*>(kb)[lane + 64 * j];
  }
#pragma unroll
  for (int j = 0; j < OLD; j++) {
    uint32_t fresh;
    int before;
    if (touched(lane + 64 * j, fresh, before) && fresh != 0xffffu && (fresh || before)) v_old[j] = reinterpret_cast<const u32x4*>(vb)[lane + 64 * j];
  }

  Row16 k[HELD], v[HELD];
  uint32_t ktop = 0, vtop = 0;
  auto consider = [&](int i, const Row16& a, const Row16& b) {
    if (stands(i)) {
      ktop = max(ktop, top_bits(a));
      vtop = max(vtop, top_bits(b));
    }
  };
#pragma unroll
  for (int s = 0; s < HELD; s++)
    if (s < passes) load(s * TPP + sub, k[s], v[s]);
#pragma unroll
  for (int s = 0; s < HELD; s++)
    if (s < passes) consider(s * TPP + sub, k[s], v[s]);
  for (int s = HELD; s < passes; s++) {
    Row16 a, b;
    load(s * TPP + sub, a, b);
    consider(s * TPP + sub, a, b);
  }
  const float kn = scale_of<DT>(wave_umax(ktop), QMAX), vn = scale_of<DT>(wave_umax(vtop), QMAX);
  const float ks_new = kn > ks_old || kn != kn ? kn : ks_old, vs_new = vn > vs_old || vn != vn ? vn : vs_old;
  const bool kgrow = ks_new > ks_old, vgrow = vs_new > vs_old;
  const Divisor kdiv(ks_new), vdiv(vs_new);

  auto put = [&](int i, const Row16& a, const Row16& b) {
    const int o = __shfl(offset, min(i, 63), 64);
    if (!stands(i)) return;
    const u32x4 kk = encode16<DT, INT8>(a, kdiv);
    if constexpr (FORM == FORM_WHOLE) {
      unsigned char* to = kb + ((chunk >> 1) * p.bs + o) * 16 + 8 * (chunk & 1);
      *reinterpret_cast<u32x2*>(to) = u32x2{kk[0], kk[1]};
      *reinterpret_cast<u32x2*>(to + LPT / 2 * p.bs * 16) = u32x2{kk[2], kk[3]};
    } else {
      *reinterpret_cast<u32x4*>(kb + (chunk * p.bs + o) * 16) = kk;
    }
    const u32x4 c = encode16<DT, INT8>(b, vdiv);
#pragma unroll
    for (int j = 0; j < 16; j++) stage[(d0 + j) * p.bs + o] = (unsigned char)(c[j >> 2] >> (8 * (j & 3)));
  };
#pragma unroll
  for (int s = 0; s < HELD; s++)
    if (s < passes) put(s * TPP + sub, k[s], v[s]);
  for (int s = HELD; s < passes; s++) {
    Row16 a, b;
    load(s * TPP + sub, a, b);
    put(s * TPP + sub, a, b);
  }

  // earlier tokens of the block under a larger scale
  if (kgrow && first > 0) {
    const float ratio = ks_old / ks_new;
#pragma unroll
    for (int j = 0; j < OLD; j++)
      if (kept(lane + 64 * j)) reinterpret_cast<u32x4*>(kb)[lane + 64 * j] = rescale16<INT8>(k_old[j], ratio);
    for (int i = lane + 64 * OLD; i < LPT * p.bs; i += 64) {
      u32x4* at = reinterpret_cast<u32x4*>(kb) + i;
      if (kept(i)) *at = rescale16<INT8>(*at, ratio);
    }
  }
  const float ratio = vgrow && first > 0 ? vs_old / vs_new : 1.f;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the wave's LDS writes are in place for its other lanes
  auto merge = [&](int i, u32x4 old, uint32_t fresh, int before) {
    const u32x4 staged = reinterpret_cast<const u32x4*>(stage)[i];
    u32x4 r = staged;
    if (fresh != 0xffffu) {
      const bool again = vgrow && before > 0;
      const u32x4 keep = again ? byte_mask((1u << before) - 1) : u32x4{0, 0, 0, 0}, mine = byte_mask(fresh);
      const u32x4 less = again ? rescale16<INT8>(old, ratio) : old;
#pragma unroll
      for (int j = 0; j < 4; j++) r[j] = (staged[j] & mine[j]) | (less[j] & keep[j] & ~mine[j]) | (old[j] & ~keep[j] & ~mine[j]);
    }
    reinterpret_cast<u32x4*>(vb)[i] = r;
  };
  uint32_t fresh;
  int before;
#pragma unroll
  for (int j = 0; j < OLD; j++)
    if (touched(lane + 64 * j, fresh, before) && (fresh || (vgrow && before > 0))) merge(lane + 64 * j, v_old[j], fresh, before);
  for (int i = lane + 64 * OLD; touched(i, fresh, before); i += 64)
    if (fresh || (vgrow && before > 0)) merge(i, fresh != 0xffffu ? reinterpret_cast<const u32x4*>(vb)[i] : u32x4{0, 0, 0, 0}, fresh, before);
  if (lane == 0) {
    *ks = ks_new;
    *vs = vs_new;
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// The query of one token by one wave, 64 / (HEAD / 16) heads a pass: the general form, 16 elements of a head per lane.
template <typename DT, int HEAD, int FORM>
__device__ inline void rotate_query(const AppendParams& p, int t, int lane) {
  constexpr int LPT = HEAD / 16, TPP = 64 / LPT;
  const int chunk = lane % LPT, sub = lane / LPT, d0 = chunk * 16;
  const bool turns = (p.rot_mode == ROT_HALVES || p.rot_mode == ROT_PAIRS) && d0 < p.rot;
  const bool halves = p.rot_mode == ROT_HALVES, first_half = d0 < p.rot / 2;
  const int partner = turns && halves ? (first_half ? p.rot / 2 : -(p.rot / 2)) : 0;
  const bool aligned = FORM != FORM_ANY || p.aligned;
  const uint16_t* q = p.q + (int64_t)t * p.q_stride;
  uint16_t* out = p.q_out + (int64_t)t * p.q_out_stride;
  const int pos = p.rot_mode == ROT_NONE ? 0 : position(p, t);
  Angles a;
  if (turns) load_angles(a, p, pos, d0);
  for (int h0 = 0; h0 < p.num_heads; h0 += TPP) {
    const int h = min(h0 + sub, p.num_heads - 1);
    const uint16_t* x = q + (int64_t)h * HEAD;
    Row16 r;
    if (FORM == FORM_ANY && p.rot_mode == ROT_ANY) {
      r = rotate16_any<DT>(x, d0, p, pos);
    } else {
      r = load16(x + d0, aligned);
      if (turns) {
        const Row16 other = halves ? load16(x + d0 + partner, aligned) : r;
        r = rotate16<DT>(r, other, a, halves, first_half);
      }
    }
    // (in place, a lane's partner has been read by now: the store needs what the same instructions loaded)
    if (h0 + sub < p.num_heads) store16(out + (int64_t)h * HEAD + d0, r, aligned);
  }
}

template <int HEAD>
__device__ inline void copy_query(const AppendParams& p, int t, int lane) {
  const u32x4* q = reinterpret_cast<const u32x4*>(p.q + (int64_t)t * p.q_stride);
  u32x4* out = reinterpret_cast<u32x4*>(p.q_out + (int64_t)t * p.q_out_stride);
  for (int i = lane; i < p.num_heads * (HEAD / 8); i += 64) out[i] = q[i];
}

// The same for FORM_WHOLE: nothing is read twice, and four passes (32 heads of 128) are requested before the first is turned: the
// loop is bound by HBM, not by its round trips.
template <typename DT, int HEAD>
__device__ inline void rotate_query_whole(const AppendParams& p, int t, int lane) {
  constexpr int LPT = HEAD / 16, TPP = 64 / LPT, DEEP = 4, E = HEAD / 2;
  const int i0 = lane % LPT * 8, sub = lane / LPT;
  const uint16_t* q = p.q + (int64_t)t * p.q_stride + i0;
  uint16_t* out = p.q_out + (int64_t)t * p.q_out_stride + i0;
  const uint16_t* angle = reinterpret_cast<const uint16_t*>(p.cos_sin) + (int64_t)position(p, t) * HEAD + i0;
  u32x4 x[DEEP], y[DEEP], c, s;
  for (int h0 = 0; h0 < p.num_heads; h0 += DEEP * TPP) {
#pragma unroll
    for (int j = 0; j < DEEP; j++) {
      const int64_t at = (int64_t)min(h0 + j * TPP + sub, p.num_heads - 1) * HEAD;
      x[j] = *reinterpret_cast<const u32x4*>(q + at);
      y[j] = *reinterpret_cast<const u32x4*>(q + at + E);
    }
    if (h0 == 0) {
      c = *reinterpret_cast<const u32x4*>(angle);
      s = *reinterpret_cast<const u32x4*>(angle + E);
    }
#pragma unroll
    for (int j = 0; j < DEEP; j++) {
      const int h = h0 + j * TPP + sub;
      rotate8<DT>(x[j], y[j], c, s);
      if (h < p.num_heads) {
        *reinterpret_cast<u32x4*>(out + (int64_t)h * HEAD) = x[j];
        *reinterpret_cast<u32x4*>(out + (int64_t)h * HEAD + E) = y[j];
      }
    }
  }
}

template <typename DT, bool INT8, int HEAD, int FORM>
__global__ __launch_bounds__(256, FORM == FORM_ANY || FORM == FORM_PART ? 2 : 3) void rope_and_cache_blocks_kernel(const AppendParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char stage[];   // [4 waves][HEAD][block size]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  if ((int)blockIdx.x >= p.kv_groups) {
    const int t = ((int)blockIdx.x - p.kv_groups) * 4 + wave;
    if (t < p.num_tokens) {
      if constexpr (FORM == FORM_WHOLE) rotate_query_whole<DT, HEAD>(p, t, lane);
      else if constexpr (FORM == FORM_NONE) copy_query<HEAD>(p, t, lane);
      else rotate_query<DT, HEAD, FORM>(p, t, lane);
    }
    return;
  }

  // ---- keys and values: one wave per kv head and stretch of token positions, the runs that begin there ----------------
  const int unit = (int)blockIdx.x * 4 + wave;
  const int h = unit % p.num_kv_heads;
  const int t0 = unit / p.num_kv_heads * p.tokens_per_wave;
  if (t0 >= p.num_tokens) return;
  auto block_at = [&](int t, int& slot) {   // block of token t, -1 where it has none
    slot = -1;
    if (t < 0 || t >= p.num_tokens) return -1;
    const int64_t s = p.slots[t];
    if (s < 0 || s >= p.num_slots) return -1;
    slot = (int)s;
    return page_of(slot >> 4, p.page_magic);
  };
  // the first token from t on that has a slot, and its block (num_tokens, -1: none); 512 positions a step
  auto next_token = [&](int t, int& b) {
    for (; t < p.num_tokens; t += 512) {
      int s, at[8];
#pragma unroll
      for (int j = 0; j < 8; j++) at[j] = block_at(t + 64 * j + lane, s);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const uint64_t some = __ballot(at[j] >= 0);
        if (some) {
          const int i = __builtin_ctzll(some);
          b = __builtin_amdgcn_readlane(at[j], i);
          return t + 64 * j + i;
        }
      }
    }
    b = -1;
    return p.num_tokens;
  };
  // the block of the last token before t that has a slot, -1: none
  auto block_before = [&](int t) {
    for (t -= 512; t > -512; t -= 512) {
      int s, at[8];
#pragma unroll
      for (int j = 0; j < 8; j++) at[j] = block_at(t + 64 * j + lane, s);
#pragma unroll
      for (int j = 7; j >= 0; j--) {
        const uint64_t some = __ballot(at[j] >= 0);
        if (some) return __builtin_amdgcn_readlane(at[j], 63 - __builtin_clzll(some));
      }
    }
    return -1;
  };
  // Lane i looks at token t0 - 1 + i: whether a run begins at one of the wave's positions, and (all but always) the whole of it.
  int slot;
  const int tl = t0 - 1 + lane, blk = block_at(tl, slot);
  const bool rotates = FORM == FORM_WHOLE || FORM == FORM_PART || (FORM == FORM_ANY && p.rot_mode != ROT_NONE);
  const int pos = rotates && tl >= 0 && tl < p.num_tokens ? position(p, tl) : 0;
  const int before = __shfl_up(blk, 1, 64);
  uint64_t heads = __ballot(lane > 0 && lane <= p.tokens_per_wave && blk >= 0 && blk != before);
  while (heads) {
    const int i = __builtin_ctzll(heads);
    heads &= heads - 1;
    const int b = __builtin_amdgcn_readlane(blk, i);
    int t = t0 - 1 + i;
    if (t > 0 && __builtin_amdgcn_readlane(before, i) < 0 && block_before(t) == b) continue;   // a run goes on behind a gap
    // the run, a token per lane; one that does not end in sight is looked up again, 64 positions (at most) a stretch
    const uint64_t others = __ballot(lane > i && blk >= 0 && blk != b);
    bool in_sight = others || t0 + 63 >= p.num_tokens;
    for (;;) {
      int s, ps, bt;
      if (in_sight) {
        const int from = min(lane + i, 63);
        s = __shfl(slot, from, 64), ps = __shfl(pos, from, 64), bt = __shfl(blk, from, 64);
        if (lane + i > 63) bt = -1;
      } else {
        bt = block_at(t + lane, s);
        ps = rotates && t + lane < p.num_tokens ? position(p, t + lane) : 0;
      }
      const uint64_t end = __ballot(bt >= 0 && bt != b);
      const uint64_t here = __ballot(bt == b) & (end ? (1ull << __builtin_ctzll(end)) - 1 : ~0ull);
      append_run<DT, INT8, HEAD, FORM>(p, t, here, b, s - b * p.bs, ps, h, stage + wave * HEAD * p.bs, lane);
      if (in_sight || end || t + 64 >= p.num_tokens) break;
      int bn;
      t = next_token(t + 64, bn);
      if (bn != b) break;
      __threadfence_block();
    }
  }
}

}  // namespace mi355q

using namespace mi355q;

extern "C" int mi355q_rope_and_cache_blocks(const int64_t* positions, const void* query, int64_t query_stride, void* query_out,
                                            int64_t query_out_stride, const void* key, int64_t key_stride, const void* value,
                                            int64_t value_stride, int head_size, int num_heads, int num_kv_heads,
                                            const void* cos_sin_cache, int rot_dim, int max_position, int cos_dtype, int is_neox,
                                            void* key_cache, void* value_cache, int num_blocks, int block_size,
                                            int64_t block_stride, float* k_scales, float* v_scales, int64_t scale_block_stride,
                                            int64_t scale_head_stride, const int64_t* slot_mapping, int num_tokens, int dtype,
                                            int code_type, mi355q_stream_t stream) {
  MI355Q_REQUIRE(dtype == MI355Q_BF16 || dtype == MI355Q_FP16, "rope_and_cache_blocks: dtype must be bf16 or fp16");
  MI355Q_REQUIRE(code_type == MI355Q_KV_INT8 || code_type == MI355Q_KV_FP8, "rope_and_cache_blocks: codes are int8 or e4m3");
  MI355Q_REQUIRE(head_size == 64 || head_size == 128, "rope_and_cache_blocks: head_size %d (64 or 128)", head_size);
  MI355Q_REQUIRE(num_tokens >= 0 && num_heads >= 0 && num_kv_heads > 0, "rope_and_cache_blocks: bad sizes");
  if (num_tokens == 0) return MI355Q_OK;
  MI355Q_REQUIRE(key && value && key_cache && value_cache && k_scales && v_scales && slot_mapping, "rope_and_cache_blocks: null pointer");
  MI355Q_REQUIRE(num_heads == 0 || (query && query_out), "rope_and_cache_blocks: null pointer");
  MI355Q_REQUIRE(block_size >= 16 && block_size <= 64 && block_size % 16 == 0, "rope_and_cache_blocks: block size %d (16, 32, 48 or 64)", block_size);
  MI355Q_REQUIRE(num_blocks > 0 && (int64_t)num_blocks * block_size < (int64_t)1 << 31, "rope_and_cache_blocks: %d blocks of %d tokens", num_blocks, block_size);
  MI355Q_REQUIRE(block_stride >= (int64_t)num_kv_heads * head_size * block_size && block_stride % 16 == 0,
                 "rope_and_cache_blocks: block stride %lld", (long long)block_stride);
  MI355Q_REQUIRE(((uintptr_t)key_cache | (uintptr_t)value_cache) % 16 == 0, "rope_and_cache_blocks: caches must be 16-byte aligned");
  MI355Q_REQUIRE(rot_dim >= 0 && rot_dim % 2 == 0 && rot_dim <= head_size, "rope_and_cache_blocks: rot_dim %d vs head_size %d", rot_dim, head_size);
  if (rot_dim) {
    MI355Q_REQUIRE(positions && cos_sin_cache && max_position > 0, "rope_and_cache_blocks: rotation needs positions and a cos/sin table");
    MI355Q_REQUIRE(cos_dtype >= MI355Q_BF16 && cos_dtype <= MI355Q_FP32, "rope_and_cache_blocks: bad cos/sin dtype");
  }
  AppendParams p{};
  p.positions = positions;
  p.q = (const uint16_t*)query;
  p.q_out = (uint16_t*)query_out;
  p.k = (const uint16_t*)key;
  p.v = (const uint16_t*)value;
  p.q_stride = query_stride, p.q_out_stride = query_out_stride, p.k_stride = key_stride, p.v_stride = value_stride;
  p.num_tokens = num_tokens, p.num_heads = num_heads, p.num_kv_heads = num_kv_heads;
  p.cos_sin = cos_sin_cache;
  p.cos_dtype = cos_dtype, p.rot = rot_dim, p.max_pos = max_position, p.is_neox = is_neox;
  auto off16 = [](const void* a, int64_t stride) { return ((uintptr_t)a & 15) || (stride & 7); };
  p.aligned = !(off16(key, key_stride) || off16(value, value_stride) ||
                (num_heads && (off16(query, query_stride) || off16(query_out, query_out_stride))));
  const bool table16 = cos_sin_cache && ((uintptr_t)cos_sin_cache & 15) == 0;
  p.rot_mode = !rot_dim ? ROT_NONE : !table16 ? ROT_ANY : is_neox && rot_dim % 32 == 0 ? ROT_HALVES : !is_neox && rot_dim % 16 == 0 ? ROT_PAIRS : ROT_ANY;
  p.kc = (unsigned char*)key_cache;
  p.vc = (unsigned char*)value_cache;
  p.block_stride = block_stride;
  p.ks = k_scales, p.vs = v_scales;
  p.scale_block_stride = scale_block_stride, p.scale_head_stride = scale_head_stride;
  p.slots = slot_mapping;
  p.num_slots = num_blocks * block_size;
  p.bs = block_size;
  const int pieces = block_size / 16;
  p.page_magic = pieces == 1 ? 0 : (int)(((1ull << 32) + pieces - 1) / pieces);
  // a wave looks at one position where a step holds few tokens (every one begins a run of its own), at 8 where they come
  // as prompts: most positions then continue a run, and waves that find nothing to begin are pure dispatch.  The slots are on the
  // device, so the number of tokens has to tell.  One position and eight, int8, 32 + 8 heads of 128, in a graph: decode rows 64 6.4 and
  // 32.5 us, 512 12.3 and 27.7, 1024 21.8 and 30.3, 2048 38.0 and 36.6; a prompt of 64 6.4 and 6.3, 512 12.9 and 7.0, 1024 21.4 and
  // 8.1, 8192 144 and 36.6.  (A decode batch of 600 rows pays 14 us for what a prompt of that length gains 7.)
  p.tokens_per_wave = num_tokens <= 512 ? 1 : 8;
  const int64_t units = ((int64_t)num_tokens + p.tokens_per_wave - 1) / p.tokens_per_wave * num_kv_heads;
  const int64_t kv_groups = (units + 3) / 4;
  const int q_groups = num_heads ? (int)(((int64_t)num_tokens + 3) / 4) : 0;
  MI355Q_REQUIRE(kv_groups + q_groups < (int64_t)1 << 24, "rope_and_cache_blocks: %d tokens are too many for a launch", num_tokens);
  p.kv_groups = (int)kv_groups;
  const size_t lds = (size_t)4 * head_size * block_size;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid(p.kv_groups + q_groups), wg(256);
  const bool i8 = code_type == MI355Q_KV_INT8;
  const bool whole = p.rot_mode == ROT_HALVES && rot_dim == head_size && p.aligned && cos_dtype == dtype;
  const bool none = p.rot_mode == ROT_NONE && p.aligned, part = (p.rot_mode == ROT_HALVES || p.rot_mode == ROT_PAIRS) && p.aligned;
#define LAUNCH(DT, I8, HD, FM) hipLaunchKernelGGL((rope_and_cache_blocks_kernel<DT, I8, HD, FM>), grid, wg, lds, s, p)
#define BY_FORM(DT, I8, HD)                      \
  do {                                           \
    if (whole) LAUNCH(DT, I8, HD, FORM_WHOLE);   \
    else if (none) LAUNCH(DT, I8, HD, FORM_NONE); \
    else if (part) LAUNCH(DT, I8, HD, FORM_PART); \
    else LAUNCH(DT, I8, HD, FORM_ANY);           \
  } while (0)
#define BY_HEAD(DT, I8)                          \
  do {                                           \
    if (head_size == 128) BY_FORM(DT, I8, 128);  \
    else BY_FORM(DT, I8, 64);                    \
  } while (0)
  if (dtype == MI355Q_BF16) {
    if (i8) BY_HEAD(BF16, true);
    else BY_HEAD(BF16, false);
  } else {
    if (i8) BY_HEAD(FP16, true);
    else BY_HEAD(FP16, false);
  }
#undef BY_HEAD
#undef BY_FORM
#undef LAUNCH
  return check_launch("rope_and_cache_blocks_kernel");
}
