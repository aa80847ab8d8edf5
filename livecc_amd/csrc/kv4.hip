// A KV cache held in 4 bits: the pass that fills it (RMS norms of queries and keys per head, M-RoPE, append; also into the bf16 cache), its
// read-back, and the attention of single tokens and of chunks over it.
//
// Format.  32 channels of one token and KV head share a power of two: value = code * 2^(e - 127), code one of +-{0 .5 1 1.5 2 3 4 6} in 4 bits, e one
// byte (4.25 bits a value against 16).  These are the fp4 / scale operands of gfx950's conversions (v_cvt_scalef32_pk_fp4_bf16 and
// v_cvt_scalef32_pk_bf16_fp4: two values an instruction, nearest with ties to the even code, 6 beyond; compared with the definition on every finite bf16 input and
// every code and scale), and every value is exact in bf16, so the attention is that of a bf16 cache holding those values.
//   e: the smallest with max |x| <= 7 * 2^(e - 127).  Up to 7 the nearest code is 6, at most one step (2) away, as far as any code of the
//   next scale would be; so a smaller scale never costs the largest value more and serves the others twice as finely.  In bits of a bf16
//   magnitude: ((bits + 0x1f) >> 7) - 2, clamped to 2 .. 252: values are never subnormal, never overflow.  A group that holds an infinity or a NaN has
//   e = 255 and reads as NaN (what the conversion gives, too).
// Layout of a slot: [layer][K codes | V codes | K scales | V scales] bytes (kernels.h: Kv4Layout):
//   K codes  [head][position][64]: a token's 128 channels in order.  A lane of the decode kernel loads 16 bytes = one group of one key and one scale byte.
//   V codes  [head][position / 32][g 4][i 16][t 4][e 8]: position 8 g + e of the block, channels 32 t + i (low half) and 32 t + 16 + i.  The two
//     values of a byte are of one token (tokens never share a byte: appends need no read-modify-write, two streams' appends no order) and one scale, and
//     a lane's 32 bytes (g, i) are its operand of the eight 16x16x32 products over the block.
//   K scales [head][position][4], V scales [head][position / 32][g 4][t 4][e 8].
#include <algorithm>
#include <type_traits>
#include <utility>

#include "common.h"
#include "kernels.h"

namespace lcc {

typedef __attribute__((ext_vector_type(16))) float f32x16;

template <class F, int... I>
LCC_DEVICE void unrolled_of(F&& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, class F>
LCC_DEVICE void unrolled(F&& f) { unrolled_of(f, std::make_integer_sequence<int, N>{}); }      // f(0) .. f(N - 1), the index a constant

LCC_DEVICE f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
LCC_DEVICE int swap23(int i) { return (i & ~12) | ((i & 4) << 1) | ((i & 8) >> 1); }
LCC_DEVICE float xor32_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
LCC_DEVICE float xor32_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

LCC_DEVICE float xor16_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
LCC_DEVICE float xor16_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// byte SEL of `w` -> its two values under `scale`, of which the conversion reads the exponent field alone: the mantissa and sign may hold anything
template <int SEL>
LCC_DEVICE unsigned fp4_pair(unsigned w, unsigned scale) { return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, __uint_as_float(scale), SEL)); }
// scale byte SEL of `w` in the exponent field
template <int SEL>
LCC_DEVICE unsigned scale_of(unsigned w) { return SEL < 3 ? w << (23 - 8 * SEL) : w >> 1; }
// a word of K codes -> eight channels
LCC_DEVICE u32x4 fp4_word(unsigned w, unsigned scale) { return (u32x4){fp4_pair<0>(w, scale), fp4_pair<1>(w, scale), fp4_pair<2>(w, scale), fp4_pair<3>(w, scale)}; }

// ------------------------------------------------------------------------------------------------------------------------------
// Norm, rotation, append: every head row of a token is read once and written once (queries as bf16, keys and values into the cache).
// Bound: up to some 400 rows the trips to a row, its place and the cache (2.7 us for a row of 28 / 4 heads, 4.6 us for 386; into 4 bits 4.5 us for eight rows of 12 / 2, whose arena's address is
// loaded behind the norm); 9,048 rows 33 to 36 us for 169 MB, 4,076 rows of 64 / 8 heads into 4 bits 31 to 33 us for 155 MB, 4.7-5.1 TB/s, where a copy of the same bytes takes 34 and 31: the vector work (the norm and eight roundings a pair, some 350 instructions a wave, 25 us by
// themselves) hides behind the memory as long as all loads of a lane are in flight before the first wait (one after the other: 3 us more) and V is stored by whole octets.  Blocks that stay
// and fetch their next item ahead were no faster, nor four heads a lane group behind one load of the tables; sums in 32 bits would save nothing.
// ------------------------------------------------------------------------------------------------------------------------------
// scale byte of a group whose largest bf16 magnitude has the bits `a`
LCC_DEVICE int kv4_exponent(int a) {
  const int e = ((a + 0x1f) >> 7) - 2;
  return a >= 0x7f80 ? 255 : e < 2 ? 2 : e > 252 ? 252 : e;
}
// eight bf16 (in pairs) -> a word of codes
LCC_DEVICE unsigned fp4_of(const u32x4& x, int e) {
  if (e == 255) return 0u;
  const float s = __uint_as_float((unsigned)e << 23);
  unsigned w = 0;
  const unsigned a = x[0], b = x[1], c = x[2], d = x[3];        // by value: hipcc's bit_cast of a vector's element reads the first element
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, a), s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, b), s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, c), s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, d), s, 3);
  return w;
}
LCC_DEVICE int max_bits(const u32x4& x) {
  int a = 0;
#pragma unroll
  for (int d = 0; d < 4; ++d) { const int lo = x[d] & 0x7fff, hi = x[d] >> 16 & 0x7fff; a = max(a, max(lo, hi)); }
  return a;
}
// lane ^ X of 32: on the LDS crossbar, whose pattern is a constant (a lane's address would be vector work, which large calls have no room for; moves of the vector unit: 45.5 -> 47.4 us
// for 9,048 rows)
template <int X> LCC_DEVICE int lane_xor(int x) { return __builtin_amdgcn_ds_swizzle(x, X << 10 | 0x1f); }
template <int X> LCC_DEVICE double lane_xor(double x) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = lane_xor<X>((int)(unsigned)u), hi = lane_xor<X>((int)(unsigned)(u >> 32));
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
// over the four lanes that hold a group
LCC_DEVICE int max4(int a) {
  a = max(a, lane_xor<1>(a));
  return max(a, lane_xor<2>(a));
}

// A lane's 16 channels of a head (c0 .. + 7, c0 + 64 .. + 71) of a row: bf16, or bf16(sum of the slabs + bias).  rows * heads fits 31 bits.
LCC_DEVICE void row16(const QkNormArgs& a, int s, int head, int c0, float (&x1)[8], float (&x2)[8]) {
  const int heads = a.n_q_heads + 2 * a.n_kv_heads;
  if (a.partial == nullptr) {
    const bf16_t* p = a.qkv + ((size_t)(unsigned)(s * heads + head) << 7) + c0;
    const u32x4 y1 = ld16(p), y2 = ld16(p + 64);
#pragma unroll
    for (int d = 0; d < 4; ++d) { x1[2 * d] = lo2f(y1[d]); x1[2 * d + 1] = hi2f(y1[d]); x2[2 * d] = lo2f(y2[d]); x2[2 * d + 1] = hi2f(y2[d]); }
    return;
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float(&v)[8] = half ? x2 : x1;
    const int col = head * 128 + c0 + half * 64;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    for (int sp = 0; sp < a.nsplit; ++sp) {
      const float* p = a.partial + ((size_t)sp * a.rows + s) * heads * 128 + col;
      const f32x4 x = *reinterpret_cast<const f32x4*>(p), y = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] += x[e]; v[4 + e] += y[e]; }
    }
    const u32x4 b = a.bias != nullptr ? ld16(a.bias + col) : (u32x4){0, 0, 0, 0};
#pragma unroll
    for (int d = 0; d < 4; ++d) { v[2 * d] = rbf(v[2 * d] + lo2f(b[d])); v[2 * d + 1] = rbf(v[2 * d + 1] + hi2f(b[d])); }
  }
}

// RMS norm of a head's 128 channels over its eight lanes, with the model's rounding points: bf16(w bf16(x r)).  The mean square and its root are formed in 64
// bits and r is rounded once: keys are quantised behind this, and codes must not depend on the order of a sum.
LCC_DEVICE void head_norm(float (&x1)[8], float (&x2)[8], const u32x4& w1, const u32x4& w2, float eps) {
  double ss = 0.0;
#pragma unroll
  for (int e = 0; e < 8; ++e) { ss = fma((double)x1[e], (double)x1[e], ss); ss = fma((double)x2[e], (double)x2[e], ss); }
  ss += lane_xor<1>(ss);
  ss += lane_xor<2>(ss);
  ss += lane_xor<4>(ss);
  const double m = ss * (1.0 / 128) + (double)eps;
  double r = __builtin_amdgcn_rsq(m);
  if (m < __builtin_inf()) r = fma(0.5 * r, fma(-m * r, r, 1.0), r);        // the unit's result is good to about 2^-28; one step squares that
  const float rf = (float)r;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    float *a = x1 + 2 * d, *b = x2 + 2 * d;
    a[0] *= rf; a[1] *= rf; b[0] *= rf; b[1] *= rf;
    rbf2(a[0], a[1]); rbf2(b[0], b[1]);
    a[0] *= lo2f(w1[d]); a[1] *= hi2f(w1[d]); b[0] *= lo2f(w2[d]); b[1] *= hi2f(w2[d]);
    rbf2(a[0], a[1]); rbf2(b[0], b[1]);
  }
}

// From so many rows on V goes by windows.  Without / with them, us a call:
//   chunks        64 rows       128           386           1,131           single tokens of as many streams (no octet among them)   64            128           600
//   28 / 4, bf16  3.8 / 3.4     4.0 / 3.6     5.4 / 4.2     10.9 / 7.2                                                               3.8 / 5.1     4.3 / 5.6     9.0 / 9.3
//   28 / 4, 4 b.  4.1 / 4.0     4.1 / 4.1     5.0 / 4.6     8.8 / 7.3                                                                4.1 / 4.8     4.1 / 4.9     6.0 / 6.7
//   64 / 8, bf16  3.7 / 3.7     4.5 / 3.9     8.2 / 6.3     15.7 / 11.8                                                              3.8 / 5.6     5.2 / 6.7     13.8 / 14.2
//   64 / 8, 4 b.  3.4 / 4.1     3.9 / 4.3     6.1 / 6.6     11.7 / 11.7                                                              3.3 / 4.9     3.9 / 5.5     8.4 / 10.0
// Below 128 rows a chunk gains 0.4 us at most and a batch of single tokens loses 0.7 to 1.8; decode batches are of that size, larger calls are mostly chunks.
constexpr int KV4_WINDOW_ROWS = 128;
// Where a row's keys and values go: its slot and position, slot -1 for a row of no stream or no position.
LCC_DEVICE void row_place(const QkNormArgs& a, int s, int& slot, int& pos) {
  slot = a.tok_stream[s];
  pos = -1;
  if (slot >= 0 && slot < a.n_slots) pos = a.tok_pos != nullptr ? a.tok_pos[s] : a.kv_len[slot];
  if (pos < 0 || pos >= a.lmax) slot = -1;
}
// The lane's V codes: channels i and 16 + i of a group lie two lanes apart, so of four lanes the lower pair takes the lower group's bytes (r1: group j / 4), the
// upper pair the upper group's (2 + j / 4): bytes i = 8 (j & 1) .. + 7 of group t, e its scale
LCC_DEVICE void v_codes(const u32x4& r1, const u32x4& r2, int j, u32x2& bytes, int& t, int& e) {
  const int e1 = kv4_exponent(max4(max_bits(r1))), e2 = kv4_exponent(max4(max_bits(r2)));
  const unsigned w1 = fp4_of(r1, e1), w2 = fp4_of(r2, e2);
  const bool up = (j & 2) != 0;
  const unsigned mine = up ? w2 : w1, other = lane_xor<2>((int)(up ? w1 : w2)), lo = up ? other : mine, hi = up ? mine : other;
  t = up ? 2 + (j >> 2) : j >> 2;
  e = up ? e2 : e1;
#pragma unroll
  for (int d = 0; d < 2; ++d) {                       // nibbles 4 d .. 4 d + 3 of either word, spread to bytes
    const unsigned a = lo >> (16 * d) & 0xffffu, b = hi >> (16 * d) & 0xffffu;
    const unsigned x = (a | a << 8) & 0x00ff00ffu, y = (b | b << 8) & 0x00ff00ffu;
    bytes[d] = ((x | x << 4) & 0x0f0f0f0fu) | ((y | y << 4) & 0x0f0f0f0fu) << 4;
  }
}
// 16 channels of a row: a lane's r1, r2
LCC_DEVICE void row_pairs(const QkNormArgs& a, int s, int head, int c0, u32x4& r1, u32x4& r2) {
  float x1[8], x2[8];
  row16(a, s, head, c0, x1, x2);
#pragma unroll
  for (int d = 0; d < 4; ++d) { r1[d] = pack2(x1[2 * d], x1[2 * d + 1]); r2[d] = pack2(x2[2 * d], x2[2 * d + 1]); }
}

// V of 32 consecutive rows of a KV head, a block: V lies position-innermost, so rows are turned in LDS.  Eight rows that are the eight positions of an aligned octet of one stream are one
// store of a channel (16 bytes of bf16; 4 bits: 8 of a byte): the block in whose window they begin takes the rows behind its window along and writes them all.  Rows of no such octet (ends
// of a chunk, single tokens) are stored one by one, rows of an octet that began before the window not at all.
constexpr int KV4_V_ROWS = 39;                                              // a window and what an octet may take behind it
template <bool KV4> constexpr int KV4_V_PITCH = KV4 ? 68 : 260;             // bytes of a row: 64 code bytes [t][i] and 4 scales, or 128 bf16 (+ 4: rows on other banks)
template <bool KV4>
LCC_DEVICE void append_v_window(const QkNormArgs& a, int h, int r0, unsigned char* lds) {
  constexpr int PITCH = KV4_V_PITCH<KV4>;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = tid & 7, head = a.n_q_heads + a.n_kv_heads + h;
  u32x4 r1, r2;
  row_pairs(a, min(r0 + (tid >> 3), a.rows - 1), head, j * 8, r1, r2);
  auto stage = [&](int row) {
    unsigned char* at = lds + row * PITCH;
    if (KV4) {
      u32x2 w; int t, e;
      v_codes(r1, r2, j, w, t, e);
      *reinterpret_cast<unsigned*>(at + t * 16 + (j & 1) * 8) = w[0];
      *reinterpret_cast<unsigned*>(at + t * 16 + (j & 1) * 8 + 4) = w[1];
      if ((j & 1) == 0) at[64 + t] = (unsigned char)e;
    } else {
#pragma unroll
      for (int d = 0; d < 4; ++d) { *reinterpret_cast<unsigned*>(at + j * 16 + 4 * d) = r1[d]; *reinterpret_cast<unsigned*>(at + 128 + j * 16 + 4 * d) = r2[d]; }
    }
  };
  // lane i has row r0 - 7 + i: 46 rows, those of every octet that reaches into the window
  int slot = -1, pos = 0;
  const int mine = r0 - 7 + lane;
  if (lane < 46 && mine >= 0 && mine < a.rows) row_place(a, mine, slot, pos);
  const unsigned long long arena = slot >= 0 ? (unsigned long long)a.kv_base[slot] : 0;
  const int before = __shfl_up(slot, 1, 64), pos_before = __shfl_up(pos, 1, 64);
  const unsigned long long next = __ballot(lane > 0 && slot >= 0 && slot == before && pos == pos_before + 1);       // rows that continue the one before
  const int first = lane - (pos & 7);                                       // of the row's octet
  const bool whole = slot >= 0 && first >= 0 && ((next >> (max(first, 0) + 1)) & 0x7f) == 0x7f, window = lane >= 7 && lane < 39;
  unsigned long long octets = __ballot(window && whole && first == lane), singles = __ballot(window && slot >= 0 && !whole);
  stage(tid >> 3);
  if ((octets >> 32) != 0 && tid < 56) {                                    // the last octet ends behind the window
    row_pairs(a, min(r0 + 32 + (tid >> 3), a.rows - 1), head, j * 8, r1, r2);
    stage(32 + (tid >> 3));
  }
  __syncthreads();
  const Kv4Layout lay{a.n_kv_heads, a.lmax};
  const size_t kv = (size_t)a.n_kv_heads * a.lmax * 128;
  auto base_of = [&](int o) -> uint8_t* {                                   // of lane o's row
    uint8_t* at = (uint8_t*)((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(arena >> 32), o) << 32 | (unsigned)__builtin_amdgcn_readlane((int)(unsigned)arena, o));
    return KV4 ? at + (size_t)a.layer * lay.layer_bytes() : (uint8_t*)((bf16_t*)at + ((size_t)a.layer * 2 + 1) * kv + (size_t)h * a.lmax * 128);
  };
  auto place4 = [&](uint8_t* base, int ps, int b) -> uint8_t* {             // byte b of a row: codes (t, i), from 64 on scales
    return b < 64 ? base + lay.v_codes(h) + (size_t)(ps >> 5) * 2048 + ((ps & 31) >> 3) * 512 + (b & 15) * 32 + (b >> 4) * 8 + (ps & 7)
                  : base + lay.v_scales(h) + (size_t)(ps >> 5) * 128 + ((ps & 31) >> 3) * 32 + (b - 64) * 8 + (ps & 7);
  };
  auto place16 = [&](uint8_t* base, int ps, int c) { return (bf16_t*)base + ((size_t)(ps >> 5) * 128 + c) * 32 + (ps & 31); };
  // up to four octets, a wave each; singles in turn
  for (int i = 0; i < wave; ++i) { octets &= octets - 1; singles &= singles - 1; }
  if (octets != 0) {
    const int o = __builtin_ctzll(octets), ps = __builtin_amdgcn_readlane(pos, o);
    uint8_t* base = base_of(o);
    const unsigned char* at = lds + (o - 7) * PITCH;
    if (KV4) {
#pragma unroll
      for (int b = lane; b < 68; b += 64) {                                 // a byte of the rows
        u32x2 w = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e >> 2] |= (unsigned)at[e * PITCH + b] << (8 * (e & 3));
        st8(place4(base, ps, b), w);
      }
    } else {                                                                // a pair of channels
      u32x4 lo, hi;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const unsigned x = *reinterpret_cast<const unsigned*>(at + 2 * d * PITCH + lane * 4), y = *reinterpret_cast<const unsigned*>(at + (2 * d + 1) * PITCH + lane * 4);
        lo[d] = __builtin_amdgcn_perm(y, x, 0x05040100u); hi[d] = __builtin_amdgcn_perm(y, x, 0x07060302u);
      }
      bf16_t* dst = place16(base, ps, lane * 2);
      st16(dst, lo); st16(dst + 32, hi);
    }
  }
  while (singles != 0) {
    const int o = __builtin_ctzll(singles), ps = __builtin_amdgcn_readlane(pos, o);
    uint8_t* base = base_of(o);
    const unsigned char* at = lds + (o - 7) * PITCH;
    if (KV4) {
      for (int b = lane; b < 68; b += 64) *place4(base, ps, b) = at[b];
    } else {
      const unsigned x = *reinterpret_cast<const unsigned*>(at + lane * 4);
      bf16_t* dst = place16(base, ps, lane * 2);
      dst[0] = (bf16_t)x; dst[32] = (bf16_t)(x >> 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) singles &= singles - 1;
  }
}

// Eight lanes a (row, head), lane j with channels 8 j .. + 7 and 64 + 8 j .. + 7: the rotation's pairs and, four lanes each, two groups of the 4-bit format
// (2 exchanges a group, 3 for the norm).  WINDOWS: every v_every-th block takes V of a window of rows, the others queries and keys.
template <bool KV4, bool WINDOWS>
__global__ __launch_bounds__(256) void qk_norm_rope_append_kernel(QkNormArgs a, int v_blocks, int v_every) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[WINDOWS ? KV4_V_ROWS * KV4_V_PITCH<KV4> : 16];
  int block = (int)blockIdx.x;
  if (WINDOWS) {
    const int w = block / v_every;
    if (w < v_blocks && block == w * v_every) {
      const int wins = v_blocks / a.n_kv_heads, h = w / wins;
      append_v_window<KV4>(a, h, (w - h * wins) * 32, lds);
      return;
    }
    block -= min(w + 1, v_blocks);
  }
  const int per_row = a.n_q_heads + (WINDOWS ? 1 : 2) * a.n_kv_heads;
  // (row, head) of the lane's item 32 block + tid / 8: divided once a block; a row of 32 heads and more ends at most once in a block
  int s = (block * 32) / per_row, head = block * 32 - s * per_row + (int)(threadIdx.x >> 3);
  if (per_row >= 32) {
    if (head >= per_row) { head -= per_row; ++s; }
  } else {
    const int more = head / per_row;
    head -= more * per_row; s += more;
  }
  if (s >= a.rows) return;                                                  // whole groups of eight lanes
  const int j = threadIdx.x & 7, c0 = j * 8, kind = head < a.n_q_heads ? 0 : head < a.n_q_heads + a.n_kv_heads ? 1 : 2;
  const int h = kind == 0 ? head : head - a.n_q_heads - (kind - 1) * a.n_kv_heads;
  int slot = 0, pos = 0;
  u32x4 r1, r2;
  if (kind < 2) {
    // all loads ahead of the first wait
    const bf16_t* w = kind ? a.k_norm : a.q_norm;
    const u32x4 cq = ld16(a.cos + (size_t)s * 64 + c0), sq = ld16(a.sin + (size_t)s * 64 + c0);
    u32x4 w1 = {0, 0, 0, 0}, w2 = w1;
    if (w != nullptr) { w1 = ld16(w + c0); w2 = ld16(w + c0 + 64); }
    float x1[8], x2[8];
    asm volatile("" ::: "memory");
    row16(a, s, head, c0, x1, x2);
    if (kind > 0) row_place(a, s, slot, pos);
    if (w != nullptr) head_norm(x1, x2, w1, w2, a.eps);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      float p[4], q[4];                                                     // the four products of channels 2 d, 2 d + 1 and their partners, rounded
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const float c = z ? hi2f(cq[d]) : lo2f(cq[d]), sn = z ? hi2f(sq[d]) : lo2f(sq[d]), u = x1[2 * d + z], v = x2[2 * d + z];
        p[z] = u * c; p[2 + z] = -v * sn;
        q[z] = v * c; q[2 + z] = u * sn;
      }
      rbf2(p[0], p[1]); rbf2(p[2], p[3]); rbf2(q[0], q[1]); rbf2(q[2], q[3]);
      r1[d] = pack2(p[0] + p[2], p[1] + p[3]); r2[d] = pack2(q[0] + q[2], q[1] + q[3]);
    }
    if (kind == 0) {
      bf16_t* q = a.q_out + ((size_t)(unsigned)(s * a.n_q_heads + h) << 7) + c0;
      st16(q, r1); st16(q + 64, r2);
      return;
    }
  } else {
    row_pairs(a, s, head, c0, r1, r2);
    row_place(a, s, slot, pos);
  }
  if (slot < 0) return;
  if (!KV4) {
    bf16_t* base = (bf16_t*)a.kv_base[slot] + ((size_t)(a.layer * 2 + kind - 1) * a.n_kv_heads + h) * a.lmax * 128;
    if (kind == 1) {
      bf16_t* k = base + (size_t)pos * 128 + c0;
      st16(k, r1); st16(k + 64, r2);
    } else {
      bf16_t* v = base + ((size_t)(pos >> 5) * 128 + c0) * 32 + (pos & 31);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e * 32] = (bf16_t)((e & 1) ? r1[e >> 1] >> 16 : r1[e >> 1]);
        v[(64 + e) * 32] = (bf16_t)((e & 1) ? r2[e >> 1] >> 16 : r2[e >> 1]);
      }
    }
    return;
  }
  const Kv4Layout lay{a.n_kv_heads, a.lmax};
  uint8_t* base = (uint8_t*)a.kv_base[slot] + (size_t)a.layer * lay.layer_bytes();
  if (kind == 1) {
    const int e1 = kv4_exponent(max4(max_bits(r1))), e2 = kv4_exponent(max4(max_bits(r2)));       // groups j / 4 and 2 + j / 4
    unsigned* k = (unsigned*)(base + lay.k_codes(h) + (size_t)pos * 64);
    k[j] = fp4_of(r1, e1); k[8 + j] = fp4_of(r2, e2);
    if ((j & 3) == 0) {
      uint8_t* sc = base + lay.k_scales(h) + (size_t)pos * 4;
      sc[j >> 2] = (uint8_t)e1; sc[2 + (j >> 2)] = (uint8_t)e2;
    }
  } else {
    u32x2 b; int t, e;
    v_codes(r1, r2, j, b, t, e);
    uint8_t* v = base + lay.v_codes(h) + (size_t)(pos >> 5) * 2048 + ((pos & 31) >> 3) * 512 + (j & 1) * 256 + t * 8 + (pos & 7);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i * 32] = (uint8_t)(b[i >> 2] >> (8 * (i & 3)));
    if ((j & 1) == 0) base[lay.v_scales(h) + (size_t)(pos >> 5) * 128 + ((pos & 31) >> 3) * 32 + t * 8 + (pos & 7)] = (uint8_t)e;
  }
}

static int qk_norm_check(const QkNormArgs& a) {
  if (int rc = Kv4Args{a.kv_base, a.n_slots, a.n_layers, a.n_kv_heads, a.lmax, a.layer}.check()) return rc;
  if (a.rows < 0 || a.n_q_heads < 0 || a.n_q_heads > 65535) return LCC_ERR_SHAPE;
  if (a.partial != nullptr && (a.nsplit < 1 || a.nsplit > 8)) return LCC_ERR_SHAPE;
  if (!(a.eps > 0.f) && (a.q_norm != nullptr || a.k_norm != nullptr)) return LCC_ERR_ARG;
  return 0;
}
int qk_norm_rope_append(const QkNormArgs& a, bool kv4, hipStream_t st) {
  if (int rc = qk_norm_check(a)) return rc;
  if (a.rows == 0) return 0;
  const bool windows = a.rows >= KV4_WINDOW_ROWS;
  const int64_t items = (int64_t)a.rows * (a.n_q_heads + (windows ? 1 : 2) * a.n_kv_heads), blocks = (items + 31) / 32;
  const int64_t v_blocks = windows ? ((int64_t)a.rows + 31) / 32 * a.n_kv_heads : 0;
  if (blocks + v_blocks >= 1 << 24) return LCC_ERR_SHAPE;                    // a launch has fewer than 2^32 threads
  const dim3 grid((unsigned)(blocks + v_blocks));
  const int every = windows ? (int)(((blocks + v_blocks) / v_blocks - 1) | 1) : 1;         // V blocks among the others, an odd number apart: blocks go round the eight XCDs
  if (windows && kv4) qk_norm_rope_append_kernel<true, true><<<grid, dim3(256), 0, st>>>(a, (int)v_blocks, every);
  else if (windows) qk_norm_rope_append_kernel<false, true><<<grid, dim3(256), 0, st>>>(a, (int)v_blocks, every);
  else if (kv4) qk_norm_rope_append_kernel<true, false><<<grid, dim3(256), 0, st>>>(a, 0, 1);
  else qk_norm_rope_append_kernel<false, false><<<grid, dim3(256), 0, st>>>(a, 0, 1);
  return 0;
}

// ------------------------------------------------------------------------------------------------------------------------------
// Read-back: row s = (slot, position) -> its keys and values [heads][128] in bf16; a row of no stream or position: zeros.  Eight lanes a (row, head), 16 channels
// each; rows run innermost, so that the bytes of V a wave gathers lie side by side where rows are neighbours (heads innermost: 1.3 us more).  4,076 rows of 8 heads 6.6 to 7.4 us for 21 MB,
// 3 TB/s.  Bound: a lane waits for its row's place, and behind it for eight single bytes of V, 32 bytes apart.
// ------------------------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4Args a, const int32_t* __restrict__ tok_stream, const int32_t* __restrict__ tok_pos,
                                                       bf16_t* __restrict__ k_out, bf16_t* __restrict__ v_out, int rows) {
  const int item = blockIdx.x * 32 + (threadIdx.x >> 3);
  if (item >= rows * a.n_kv_heads) return;                                  // below 2^29
  const int h = item / rows, s = item - h * rows, j = threadIdx.x & 7;
  const int slot = tok_stream[s], pos = tok_pos[s];
  // K: channels 16 j .. + 15.  V: bytes i = 8 z .. + 7 of group t, that is channels 32 t + 8 z .. + 7 and 32 t + 16 + 8 z .. + 7
  const int t = j >> 1, z = j & 1;
  const size_t at = ((size_t)s * a.n_kv_heads + h) * 128;
  bf16_t *ko = k_out + at + j * 16, *vo = v_out + at + t * 32 + z * 8;
  u32x4 k0 = {0, 0, 0, 0}, k1 = k0, v0 = k0, v1 = k0;
  if (slot >= 0 && slot < a.n_slots && pos >= 0 && pos < a.lmax) {
    const Kv4Layout lay{a.n_kv_heads, a.lmax};
    const uint8_t* base = (const uint8_t*)a.kv_base[slot] + (size_t)a.layer * lay.layer_bytes();
    const u32x2 kc = ld8(base + lay.k_codes(h) + (size_t)pos * 64 + j * 8);
    const unsigned ks = (unsigned)base[lay.k_scales(h) + (size_t)pos * 4 + t] << 23;
    const int g = (pos & 31) >> 3, e = pos & 7;
    const uint8_t* vc = base + lay.v_codes(h) + (size_t)(pos >> 5) * 2048 + g * 512 + z * 256 + t * 8 + e;
    const unsigned vs = (unsigned)base[lay.v_scales(h) + (size_t)(pos >> 5) * 128 + g * 32 + t * 8 + e] << 23;
    unsigned lo = 0, hi = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) { const unsigned b = vc[i * 32]; lo |= (b & 15u) << (4 * i); hi |= (b >> 4) << (4 * i); }
    k0 = fp4_word(kc[0], ks); k1 = fp4_word(kc[1], ks);
    v0 = fp4_word(lo, vs); v1 = fp4_word(hi, vs);
  }
  st16(ko, k0); st16(ko + 8, k1); st16(vo, v0); st16(vo + 16, v1);
}
int kv4_read(const Kv4Args& a, const int32_t* tok_stream, const int32_t* tok_pos, bf16_t* k, bf16_t* v, int rows, hipStream_t st) {
  if (int rc = a.check()) return rc;
  if (rows < 0) return LCC_ERR_SHAPE;
  if (rows == 0) return 0;
  const int64_t blocks = ((int64_t)rows * a.n_kv_heads + 31) / 32;
  if (blocks >= 1 << 24) return LCC_ERR_SHAPE;
  kv4_read_kernel<<<dim3((unsigned)blocks), dim3(256), 0, st>>>(a, tok_stream, tok_pos, k, v, rows);
  return 0;
}

// ------------------------------------------------------------------------------------------------------------------------------
// Decode attention: one row per stream.  Block = (KV head, row, key split), its waves take the split's 32-key blocks in turn; a wave's 16 columns are the query
// heads of the KV head.  S^T = K Q^T: operand A is 16 keys x 32 channels, a lane's 16 bytes of codes (one group of one key) its share of all four steps -- the
// channels of step s are 8 s .. 8 s + 7 of each group, for Q alike.  Rows of the two key tiles are dealt so that a lane's eight scores are of the keys
// 8 g .. 8 g + 7, which are the slots of its P operand: O^T += V^T P^T takes the probabilities from the softmax' registers and V's bytes as they lie.
// The loads of a wave's next block go into the registers that the products have just left, K's first, so that either is waited for by a count while the other is in flight; 126
// registers, 16 waves a unit (a second set of them: spills at that occupancy, and no gain at half of it).
// Bound: 64 rows of 2,200 to 6,000 keys (28 / 4 heads) 32 us for 139 MB, 4.3 TB/s where a read stream reaches 6.0 (38 us where other data has passed the 256 MB cache in between); the
// arithmetic alone takes 25 us.  One row of 32,768 keys (64 / 8 heads, 32 splits) 9.8 us for 36 MB, of which some 4 are the launch and the first trip.
// The same kernel takes tiles of a few rows of a chunk (CHUNK): its columns are then (row, head) pairs.
// ------------------------------------------------------------------------------------------------------------------------------
// Scores are sums of products q k; a weight is 2^(KV4_SCALE (score - m)), the difference formed before it is scaled: m scaled by itself is off by half a step, which is more than 2^7 powers of
// two from scores of 2^35 on.  What a softmax subtracts, m, lies KV4_SLACK (8 powers of two) above the highest score at which it last moved, and moves when a score passes it, not at every new maximum: sums and
// products scale alike, and bf16's and fp32's relative steps are the same at 2^-8.  Where it does not move, eight (chunks: 64) multiplications of O a block fall away.  Weights are never
// above one, so that a product p V leaves fp32's range only where the sum of the values does.
constexpr float KV4_SCALE = 1.4426950408889634 / 11.313708498984761, KV4_SLACK = 8.f / KV4_SCALE;       // log2(e) / sqrt(128)
// Weights of keys are formed from KV4_SCALE score - (KV4_SCALE m) in one operation where |KV4_SCALE m| is at most this: its rounding is then 2^-13 powers of two at most, a thirtieth of the weight's to
// bf16.  Beyond, their scores become differences first, a wave at a time (always: eight chunks of ~340 rows 242 -> 251 us, 64 rows of 2,200 to 6,000 keys 32.3 -> 32.6).
constexpr float KV4_FUSED = 4096.f;
LCC_DEVICE float kv4_weight(float score, float m) { return __builtin_amdgcn_exp2f((score - m) * KV4_SCALE); }
struct Kv4Tile { u32x4 k[2], v[2], s[2]; unsigned ks[2]; };       // what a wave loads of a 32-key block: codes of two key tiles, of V, V's scales, K's
struct Kv4Head { const uint8_t *kc, *vc, *ks, *vs; };              // a head's regions, wave-uniform: a lane's part of the addresses is 32 bits that never change
LCC_DEVICE void kv4_load_k(Kv4Tile& t, const Kv4Head& h, int blk, unsigned key, unsigned g) {
  const uint8_t *kc = h.kc + (size_t)blk * 2048, *ks = h.ks + (size_t)blk * 128;
#pragma unroll
  for (unsigned T = 0; T < 2; ++T) {
    t.k[T] = ld16(kc + (key * 64 + g * 16 + T * 256));
    t.ks[T] = ks[key * 4 + g + T * 16];
  }
}
LCC_DEVICE void kv4_load_v(Kv4Tile& t, const Kv4Head& h, int blk, unsigned li, unsigned g) {
  const uint8_t *vc = h.vc + (size_t)blk * 2048, *vs = h.vs + (size_t)blk * 128;
  t.v[0] = ld16(vc + (g * 512 + li * 32)); t.v[1] = ld16(vc + (g * 512 + li * 32 + 16));
  t.s[0] = ld16(vs + g * 32); t.s[1] = ld16(vs + (g * 32 + 16));
}

// What the columns are: rows of a decode step (row b alone, its slot's length), or (CHUNK) a tile of a few rows of a stream.
struct Kv4Rows { const int32_t* slot; const int32_t* kv_len; const int32_t* q0; const int32_t* nq; const int32_t* pos0; int tile_rows, n_rows; };

template <int NW, bool CHUNK>
__global__ __launch_bounds__(NW * 64, 4) void attn_rows_kv4_kernel(Kv4Args a, Kv4Rows rows, const bf16_t* __restrict__ q, int n_q_heads, int nsplit, float* __restrict__ ws_o,
                                                                   float* __restrict__ ws_ml, bf16_t* __restrict__ out) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  float (*mo)[16][132] = reinterpret_cast<float (*)[16][132]>(lds);
  __shared__ float mm[NW][16], ml[NW][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, g = lane >> 4;
  const int split = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, G = n_q_heads / a.n_kv_heads;
  const int slot = rows.slot[b];
  const bool live = slot >= 0 && slot < a.n_slots;
  const int q0 = CHUNK ? rows.q0[b] : b, nq = CHUNK ? min(min(rows.nq[b], rows.tile_rows), rows.n_rows - q0) : 1;
  if (CHUNK && (q0 < 0 || nq <= 0)) return;
  const int pos0 = !live ? -1 : CHUNK ? min(rows.pos0[b], a.lmax) : min(rows.kv_len[slot], a.lmax - 1);       // of the first row
  const int n = live ? max(0, min(pos0 + nq, a.lmax)) : 0;                  // keys (a position below zero: none)
  const int nblk = (n + 31) >> 5, per = (nblk + nsplit - 1) / nsplit, b0 = split * per, b1 = min(nblk, b0 + per);
  const int r = CHUNK ? li / G : 0, lim = live ? pos0 + min(r, nq - 1) : -1;                                  // the column's row and the last key it sees

  f32x4 o[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) o[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  int blk = b0 + wave;
  if (blk < b1) {
    const Kv4Layout lay{a.n_kv_heads, a.lmax};
    const uint8_t* base = (const uint8_t*)a.kv_base[slot] + (size_t)a.layer * lay.layer_bytes();
    const Kv4Head head{base + lay.k_codes(hk), base + lay.v_codes(hk), base + lay.k_scales(hk), base + lay.v_scales(hk)};
    const unsigned key = 8 * (li >> 2) + (li & 3);
    u32x4 qf[4];
    const bf16_t* qp = q + ((size_t)(q0 + min(r, nq - 1)) * n_q_heads + hk * G + (CHUNK ? li - r * G : min(li, G - 1))) * 128 + g * 32;
#pragma unroll
    for (int s = 0; s < 4; ++s) qf[s] = ld16(qp + 8 * s);
    Kv4Tile cur;
    kv4_load_k(cur, head, blk, key, g);
    asm volatile("" ::: "memory");             // in the loop's order, so that its waits hold for the first turn, too
    kv4_load_v(cur, head, blk, li, g);
    asm volatile("" ::: "memory");
    for (; blk < b1; blk += NW) {
      const int nb = blk + NW < b1 ? blk + NW : blk;                        // behind the last: the same again, so that a wait can count what is in flight
      f32x4 sc[2];
#pragma unroll
      for (int T = 0; T < 2; ++T) {
        sc[T] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 4; ++s) sc[T] = mfma16(as_bf16x8(fp4_word(cur.k[T][s], cur.ks[T] << 23)), as_bf16x8(qf[s]), sc[T]);
      }
      kv4_load_k(cur, head, nb, key, g);                                    // into the registers that the products have left
      bool nan[4] = {false, false, false, false};                           // CHUNK: the column sees a V of this group that is NaN
      if (blk * 32 + 31 > pos0) {                                           // some column does not see all of the block: scores of its hidden keys to -inf
        const int key0 = blk * 32 + 8 * g, left = n - key0;                 // of this lane's octet; keys that exist
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[T][e] = key0 + 4 * T + e <= lim ? sc[T][e] : -INFINITY;
        // V of no key to zero (0 * NaN), and NaN values that a row before theirs must not meet: zero here, put behind the products into the columns that see them
        const unsigned long long keep = left >= 8 ? ~0ull : left <= 0 ? 0ull : (1ull << (8 * left)) - 1;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const unsigned w = cur.s[t >> 1][2 * (t & 1) + z] & (unsigned)(keep >> (32 * z));
            if (CHUNK) {
              const unsigned bad = ((w & 0x7f7f7f7fu) + 0x03030303u) & w & 0x80808080u;      // bytes of 253 and more
              const int seen = lim - key0 - 4 * z;                          // bytes 0 .. seen
              nan[t] |= (bad & (seen >= 3 ? ~0u : seen < 0 ? 0u : (256u << (8 * seen)) - 1)) != 0;
              cur.s[t >> 1][2 * (t & 1) + z] = w & ~((bad >> 7) * 255u);
            } else cur.s[t >> 1][2 * (t & 1) + z] = w;
          }
        if (CHUNK) {
#pragma unroll
          for (int t = 0; t < 4; ++t) {                                     // over the four octets
            int any = nan[t];
            any |= __shfl_xor(any, 16, 64);
            any |= __shfl_xor(any, 32, 64);
            nan[t] = any != 0;
          }
        }
      }
      float top = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(sc[0][0], sc[0][1]), __builtin_fmaxf(sc[0][2], sc[0][3])),
                                  __builtin_fmaxf(__builtin_fmaxf(sc[1][0], sc[1][1]), __builtin_fmaxf(sc[1][2], sc[1][3])));
      top = xor32_max(xor16_max(top));
      if (__any(top > m)) {
        const float mn = top > m ? top + KV4_SLACK : m, f = kv4_weight(m, mn == -INFINITY ? 0.f : mn);
        l *= f;
#pragma unroll
        for (int t = 0; t < 8; ++t) o[t] *= f;
        m = mn;
      }
      const float mu = m == -INFINITY ? 0.f : m;                            // a column that has seen no key, or scores of -inf alone
      float p[8], ms = mu * KV4_SCALE;
      if (__any(__builtin_fabsf(ms) > KV4_FUSED)) { sc[0] -= mu; sc[1] -= mu; ms = 0.f; }
#pragma unroll
      for (int e = 0; e < 8; ++e) { p[e] = __builtin_amdgcn_exp2f(fmaf(sc[e >> 2][e & 3], KV4_SCALE, -ms)); l += p[e]; }
      // The products take probabilities in bf16, as the bf16 cache's attention does (l sums them unrounded):
      // each off by half a step at most, 2^-8 of itself, and so the result by 2^-8 of the weighted mean of |V|.
      // A converted byte is a pair (channel i, channel 16 + i) of one key, two slots of the operand: against (p, 0) it is channel i's product, against (0, p) the other's.
      u32x4 pl[2], ph[2];
#pragma unroll
      for (int e = 0; e < 8; ++e) { pl[e >> 2][e & 3] = pack2(p[e], 0.f); ph[e >> 2][e & 3] = pl[e >> 2][e & 3] << 16; }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const unsigned w = cur.v[t >> 1][2 * (t & 1) + z], sw = cur.s[t >> 1][2 * (t & 1) + z];
          const bf16x8 v = as_bf16x8((u32x4){fp4_pair<0>(w, scale_of<0>(sw)), fp4_pair<1>(w, scale_of<1>(sw)), fp4_pair<2>(w, scale_of<2>(sw)), fp4_pair<3>(w, scale_of<3>(sw))});
          o[2 * t] = mfma16(v, as_bf16x8(pl[z]), o[2 * t]);
          o[2 * t + 1] = mfma16(v, as_bf16x8(ph[z]), o[2 * t + 1]);
        }
      if (CHUNK) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (nan[t]) { o[2 * t] = (f32x4){NAN, NAN, NAN, NAN}; o[2 * t + 1] = o[2 * t]; }
      }
      kv4_load_v(cur, head, nb, li, g);
      asm volatile("" ::: "memory");           // hipcc would move the loads to the head of the next turn, in front of their wait
    }
    l = xor32_sum(xor16_sum(l));
  }
  // the waves' parts, joined in LDS: column li, channels 16 t + 4 g .. + 3
#pragma unroll
  for (int t = 0; t < 8; ++t) *reinterpret_cast<f32x4*>(&mo[wave][li][16 * t + 4 * g]) = o[t];
  if (g == 0) { mm[wave][li] = m; ml[wave][li] = l; }
  __syncthreads();
  for (int i = threadIdx.x; i < nq * G * 32; i += NW * 64) {
    const int h = i >> 5, c = (i & 31) * 4;                                  // column, channel
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = __builtin_fmaxf(M, mm[w][h]);
    const float mu = M == -INFINITY ? 0.f : M;
    f32x4 acc = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = kv4_weight(mm[w][h], mu);
      L += f * ml[w][h];
      acc += f * *reinterpret_cast<const f32x4*>(&mo[w][h][c]);
    }
    const int rr = CHUNK ? h / G : 0;
    const size_t row = (size_t)(q0 + rr) * n_q_heads + hk * G + (h - rr * G);
    if (nsplit == 1) {
      const float r = L == 0.f ? 0.f : 1.f / L;
      st8(out + row * 128 + c, (u32x2){pack2(acc[0] * r, acc[1] * r), pack2(acc[2] * r, acc[3] * r)});
    } else {
      *reinterpret_cast<f32x4*>(ws_o + (row * nsplit + split) * 128 + c) = acc;
      if (c == 0) { ws_ml[(row * nsplit + split) * 2] = M; ws_ml[(row * nsplit + split) * 2 + 1] = L; }
    }
  }
}

// Joins the key splits of a (row, head): sums weighted by their m's distance from the highest, one rounding.  A half-wave reads a split's 128 channels at a time; W waves share a (row, head).
// blockIdx.y: a tile, or (tiles null) a row.  All loads of a (row, head) are in flight before the first weight is known; a trip's time otherwise: 32 splits of 64 heads 3.5 us,
// 64 of 17 rows x 28 4.3 us (15.8 MB), five of 386 rows x 28 7.7 us (28 MB, 3.7 TB/s).  In one wave (W = 1) to 8 splits, in four beyond: those have more to load than registers.
template <int W>
__global__ __launch_bounds__(256) void kv4_combine_kernel(const float* __restrict__ ws_o, const float* __restrict__ ws_ml, bf16_t* __restrict__ out,
                                                          const int32_t* __restrict__ tile_q0, const int32_t* __restrict__ tile_nq, int tile_rows, int n_rows, int n_q_heads,
                                                          int nsplit) {
  __shared__ f32x4 so[W][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, c = lane & 31;
  const int item = W == 1 ? blockIdx.x * 4 + wave : blockIdx.x, b = blockIdx.y, q0 = tile_q0 ? tile_q0[b] : b;
  if (q0 < 0 || item >= min(tile_q0 ? min(tile_nq[b], tile_rows) : 1, n_rows - q0) * n_q_heads) return;       // whole waves; W > 1: whole blocks
  const size_t row = (size_t)q0 * n_q_heads + item;
  const float* ml = ws_ml + row * nsplit * 2;
  const float* o = ws_o + row * nsplit * 128 + c * 4;
  constexpr int N = W == 1 ? 4 : 8;                                          // a half-wave's share of 8 or 64 splits, all in flight before the weights are formed
  const int s0 = wave * (W == 1 ? 0 : 2) + half;
  f32x4 v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = s0 + 2 * W * i;
    v[i] = s < nsplit ? *reinterpret_cast<const f32x4*>(o + (size_t)s * 128) : (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  const float m = lane < nsplit ? ml[lane * 2] : -INFINITY, l = lane < nsplit ? ml[lane * 2 + 1] : 0.f;
  const float M = wave_max(m), w = kv4_weight(m, M == -INFINITY ? 0.f : M);
  const float L = wave_sum(w * l);
  f32x4 acc = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = s0 + 2 * W * i;
    const float f = __shfl(w, s & 63, 64);
    if (s < nsplit) acc += f * v[i];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = xor32_sum(acc[e]);
  if (W > 1) {
    if (half == 0) so[wave][c] = acc;
    __syncthreads();
    if (wave != 0) return;
    acc = so[0][c];
#pragma unroll
    for (int i = 1; i < W; ++i) acc += so[i][c];
  }
  const float r = L == 0.f ? 0.f : 1.f / L;
  if (half == 0) st8(out + row * 128 + c * 4, (u32x2){pack2(acc[0] * r, acc[1] * r), pack2(acc[2] * r, acc[3] * r)});
}
static void kv4_combine(const float* ws_o, const float* ws_ml, bf16_t* out, const int32_t* tile_q0, const int32_t* tile_nq, int n_tiles, int tile_rows, int n_rows,
                        int n_q_heads, int nsplit, hipStream_t st) {
  const unsigned items = (unsigned)tile_rows * n_q_heads;                   // up to 256 * 65535
  if (nsplit <= 8) kv4_combine_kernel<1><<<dim3((items + 3) / 4, n_tiles), dim3(256), 0, st>>>(ws_o, ws_ml, out, tile_q0, tile_nq, tile_rows, n_rows, n_q_heads, nsplit);
  else kv4_combine_kernel<4><<<dim3(items, n_tiles), dim3(256), 0, st>>>(ws_o, ws_ml, out, tile_q0, tile_nq, tile_rows, n_rows, n_q_heads, nsplit);
}

// Key splits of a decode step, by its blocks without any (rows x KV heads; a unit takes one well) and the 32-key blocks of its longest row.  Measured (us, lengths spread over a quarter or fifth):
//   Up to 32 key blocks: none, one launch.  28 / 4 heads, one row of 300 keys 5.0, in eight 6.3; of 1,000 7.7 / 6.8, which a second launch's issue takes back.
//   Up to 32 blocks: a block for every unit.  One row of 32,000 keys 16 / 64 splits 16.6 / 10.2, 8 rows of 6,144 4 / 8 / 16 splits 13.7 / 11.1 / 12.0.
//   Up to 64: as many, from 64 key blocks on: 16 rows of 1,100 keys 1 / 4 splits 7.6 / 8.4, of 2,400 12.8 / 10.3; eight from 192 on: of 6,144 14.4 / 14.6, of 16,000 33.5 / 28.7.
//   More: eight, from 96 key blocks on, where the blocks leave a fifth of the units or more idle in their last round: 40 rows of 2,400 keys 1 / 2 / 8 splits 13.6 / 16.5 / 16.6, of 6,144
//   34.0 / 36.2 / 30.1; 24 rows of 2,400 13.0 / 12.7 / 12.7, of 6,144 26.2 / 20.4 / 18.0; 48 of 16,000 88.6 / 90.6 / 74.9; 80 of 6,000 65.4 / 59.7 / 53.7.  Where the round is full, from 320 on:
//   64 rows of 6,144 keys 1 / 6 splits 45.2 / 44.9, 56 rows 41.1 / 40.3, 128 rows of 6,000 1 / 8 splits 83.8 / 84.1, of 12,000 161.3 / 160.0, with lengths over two thirds 128.8 / 124.9.
// One count serves all rows of a launch, so a long row among short ones is split as if all were long: 32,000 keys alone 9.8 us (64 splits), beside 7 rows of 500 23.8 (eight; 32 splits would
// take 12.9), beside 63 26.6 (16: 22.8); 9,000 keys alone 7.9, beside 63 rows of 500 35.9 (unsplit; eight: 15.4).
int kv4_decode_splits(const int32_t* n_keys, int n, int n_kv_heads) {
  long most = 1;
  for (int i = 0; i < n; ++i) most = n_keys[i] > most ? n_keys[i] : most;
  const long keys = (most + 31) / 32, base = (long)(n > 0 ? n : 1) * n_kv_heads, units = (256 + base - 1) / base, rounds = (base + 255) / 256;
  if (keys <= 32 || (base > 32 && keys < 64) || (base > 64 && (keys < 96 || (base * 5 > rounds * 256 * 4 && keys < 320)))) return 1;
  const long k = base > 64 || (base > 32 && keys >= 192) ? 8 : units;
  return (int)std::max(std::min(k, std::min(keys / 4, 64L)), 1L);
}

// eight waves where a block has all keys, four where they are split: 16 waves a unit in either case once there are blocks enough
template <bool CHUNK>
static void attn_rows_launch(const Kv4Args& a, const Kv4Rows& rows, int n, const bf16_t* q, int n_q_heads, int nsplit, float* ws_o, float* ws_ml, bf16_t* out, hipStream_t st) {
  static DeviceOnce once;
  constexpr int part = 16 * 132 * 4;                                        // LDS of a wave's result
  if (auto turn = once.first()) (void)hipFuncSetAttribute((const void*)attn_rows_kv4_kernel<8, CHUNK>, hipFuncAttributeMaxDynamicSharedMemorySize, 8 * part);
  const dim3 grid(nsplit, a.n_kv_heads, n);
  if (nsplit == 1) attn_rows_kv4_kernel<8, CHUNK><<<grid, dim3(512), 8 * part, st>>>(a, rows, q, n_q_heads, nsplit, ws_o, ws_ml, out);
  else attn_rows_kv4_kernel<4, CHUNK><<<grid, dim3(256), 4 * part, st>>>(a, rows, q, n_q_heads, nsplit, ws_o, ws_ml, out);
}

int attn_decode_kv4(const Kv4Args& a, const bf16_t* q, const int32_t* slots, const int32_t* kv_len, int rows, int n_q_heads, int nsplit, float* ws_o, float* ws_ml,
                    bf16_t* out, hipStream_t st) {
  if (int rc = a.check()) return rc;
  if (rows < 0 || rows > 65535 || n_q_heads < 1 || n_q_heads % a.n_kv_heads || n_q_heads / a.n_kv_heads > 16 || nsplit < 1 || nsplit > 64) return LCC_ERR_SHAPE;
  if ((int64_t)rows * n_q_heads > 0x7fffffff) return LCC_ERR_SHAPE;
  if (nsplit > 1 && (ws_o == nullptr || ws_ml == nullptr)) return LCC_ERR_ARG;
  if (rows == 0) return 0;
  attn_rows_launch<false>(a, Kv4Rows{slots, kv_len, nullptr, nullptr, nullptr, 1, rows}, rows, q, n_q_heads, nsplit, ws_o, ws_ml, out, st);
  if (nsplit > 1) kv4_combine(ws_o, ws_ml, out, nullptr, nullptr, rows, 1, rows, n_q_heads, nsplit, st);
  return 0;
}

// ------------------------------------------------------------------------------------------------------------------------------
// Attention of chunks: tiles of up to 256 / G consecutive new rows of one stream, their (row, head) pairs the 8 x 32 columns of a block's waves.  The
// block turns 64 keys at a time into bf16 in LDS (each thread eight bytes of K and of V) and every wave multiplies them: S^T = K Q^T and
// O^T += V^T P^T on 32x32x16, K's rows read in the order (bits 2 and 3 swapped) that leaves a lane the scores of the keys its P operand wants.
// Conversion once a block and stage is what LDS is for: 8 KB of codes become 32 KB that all waves read, in images whose 16-byte chunks are permuted so that neither the reads (16 lanes at
// a time) nor the writes (8) meet in a bank (no conflicts counted).
// Eight chunks of ~340 rows on ~5,000 keys 242 to 252 us, 0.83-0.87 PFLOP/s where a large matrix product reaches 1.4 (the bf16 cache's attention takes 262 for them): of a wave's 64-key stage
// 1,024 clocks are matrix instructions and some 950 vector ones (conversion, softmax), and the counters show that the two waves of a SIMD overlap them by little (matrix units busy half of the
// time).  Other orders of the stage, pinned or with
// priorities, were no faster (159 -> 170 us for 386 rows unsplit); products in the 4-bit type itself, with queries in parts of 8 bits, sum to 2^-13.5 only and were not taken.
// Few rows: 17 rows of 28 / 4 heads on 26,800 keys 21 us, a third of it the 64 splits' partials (15.8 MB).
// ------------------------------------------------------------------------------------------------------------------------------
constexpr int KV4_STAGE = 64, KV4_KB = KV4_STAGE * 256, KV4_VB = 128 * KV4_STAGE * 2, KV4_LDS = 2 * (KV4_KB + KV4_VB);
template <int U> struct Kv4Stage { u32x2 k[U], v[U], s[U]; unsigned ks[U]; };

template <int NW>
__global__ __launch_bounds__(NW * 64, 2) void attn_chunk_kv4_kernel(Kv4Args a, const bf16_t* __restrict__ q, bf16_t* __restrict__ out, const int32_t* __restrict__ tile_stream,
                                                                      const int32_t* __restrict__ tile_q0, const int32_t* __restrict__ tile_nq,
                                                                      const int32_t* __restrict__ tile_pos0, int n_q_heads, int tile_rows, int nsplit, int n_rows,
                                                                      float* __restrict__ ws_o, float* __restrict__ ws_ml) {
  constexpr int U = 8 / NW;                                                 // units of 8 bytes of K and of V that a thread stages
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  __shared__ unsigned long long bad[4][4];                                  // keys of a stage, by group, whose V is NaN (stages with masked scores)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, hh = lane >> 5, G = n_q_heads / a.n_kv_heads;
  const int hk = blockIdx.x, tile = blockIdx.y, split = blockIdx.z;
  const int slot = tile_stream[tile], q0 = tile_q0[tile], pos0 = min(tile_pos0[tile], a.lmax);
  const bool live = slot >= 0 && slot < a.n_slots;
  const int nq = min(min(tile_nq[tile], tile_rows), n_rows - q0);
  if (q0 < 0 || nq <= 0) return;
  const int nk = live ? max(0, min(pos0 + nq, a.lmax)) : 0;                 // keys of the tile
  const int nst = (nk + KV4_STAGE - 1) / KV4_STAGE, per = (nst + nsplit - 1) / nsplit, s0 = split * per, s1 = min(nst, s0 + per);
  const int c = wave * 32 + col, r = c / G, h = c - r * G;
  const bool valid = r < nq;
  const int lim = live ? min(pos0 + min(r, nq - 1), a.lmax - 1) : -1;       // last key this column sees: an arena may end inside a stage, whose other keys are none

  u32x4 qf[8];
  const bf16_t* qp = q + ((size_t)(q0 + min(r, nq - 1)) * n_q_heads + hk * G + h) * 128 + hh * 8;
#pragma unroll
  for (int s = 0; s < 8; ++s) qf[s] = ld16(qp + 16 * s);
  f32x16 o[4];
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m = -INFINITY, l = 0.f;

  if (s0 < s1) {
    const Kv4Layout lay{a.n_kv_heads, a.lmax};
    const uint8_t* base = (const uint8_t*)a.kv_base[slot] + (size_t)a.layer * lay.layer_bytes();
    const uint8_t *kc = base + lay.k_codes(hk), *vc = base + lay.v_codes(hk), *ksc = base + lay.k_scales(hk), *vsc = base + lay.v_scales(hk);
    const int t = threadIdx.x, last_blk = a.lmax / 32 - 1;
    // Unit u of a thread: eight bytes of K (16 channels of a key) and of V (channels i, 16 + i of an octet of keys), number t + 64 NW u of the stage's two blocks of 256;
    // the block is the same for a wave.  Behind the arena: its last block again (masked).
    auto block_of = [&](int st, int u) { return (size_t)min(st * 2 + ((wave + u * NW) >> 2), last_blk); };
    const unsigned unit = t & 255, s_off = ((t >> 6) & 3) * 32 + (t & 3) * 8;
    auto fetch_k = [&](Kv4Stage<U>& x, int st) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x.k[u] = ld8(kc + block_of(st, u) * 2048 + unit * 8);
        x.ks[u] = (ksc + block_of(st, u) * 128)[unit >> 1];
      }
    };
    auto fetch_v = [&](Kv4Stage<U>& x, int st) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x.v[u] = ld8(vc + block_of(st, u) * 2048 + unit * 8);
        x.s[u] = ld8(vsc + block_of(st, u) * 128 + s_off);
      }
    };
    auto masked = [&](int st) { return st * KV4_STAGE + KV4_STAGE - 1 > pos0; };          // some row does not see all of the stage
    const bool k_swap = (t & 4) != 0;
    const unsigned kw_off = (t >> 3) * 256 + (((2 * (t & 7) + k_swap) ^ ((t >> 3) & 15)) << 4), vw_ch = (t & 3) * 32 + ((t >> 2) & 15);
    const unsigned vw_off = 2 * KV4_KB + vw_ch * 128 + (((t >> 6) ^ ((vw_ch >> 1) & 7) ^ (vw_ch & 1) ^ ((t & 3) << 1)) << 4);
    auto put_k = [&](auto W, const Kv4Stage<U>& x, int st) {               // word W of the units
      constexpr int w = decltype(W)::value;
#pragma unroll
      for (int u = 0; u < U; ++u)                                           // unit t + 256: 32 keys on
        *reinterpret_cast<u32x4*>(lds + ((kw_off + (st & 1) * KV4_KB) ^ (w << 4)) + u * 8192) = fp4_word(k_swap ? x.k[u][1 - w] : x.k[u][w], x.ks[u] << 23);
    };
    auto put_v = [&](int u, const unsigned (&cv)[8], int st) {             // a unit's converted bytes; unit t + 256: four octets on
      unsigned char* at = lds + ((vw_off + (st & 1) * KV4_VB) ^ (u << 6));
      u32x4 v;
#pragma unroll
      for (int d = 0; d < 4; ++d) v[d] = __builtin_amdgcn_perm(cv[2 * d + 1], cv[2 * d], 0x05040100u);
      *reinterpret_cast<u32x4*>(at) = v;
#pragma unroll
      for (int d = 0; d < 4; ++d) v[d] = __builtin_amdgcn_perm(cv[2 * d + 1], cv[2 * d], 0x07060302u);
      *reinterpret_cast<u32x4*>(at + 2048) = v;
    };
    // What a row does not see must not reach it through 0 * NaN: values behind the last key become zeros, and NaN values zeros that are put into the rows that
    // see them behind the product
    auto hide = [&](Kv4Stage<U>& x, int st) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int key = ((t >> 6) + u * NW) * 8, left = nk - st * KV4_STAGE - key;         // of the stage: block, octet; keys of the octet that exist
        const unsigned long long keep = left >= 8 ? ~0ull : left <= 0 ? 0ull : (1ull << (8 * left)) - 1;
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const unsigned w = x.s[u][d] & (unsigned)(keep >> (32 * d));
          const unsigned nan = ((w & 0x7f7f7f7fu) + 0x03030303u) & w & 0x80808080u;        // bytes of 253 and more
          x.s[u][d] = w & ~((nan >> 7) * 255u);
          if (nan && ((t >> 2) & 15) == 0)
            atomicOr(&bad[st & 3][t & 3], (unsigned long long)((nan >> 7 & 1u) | (nan >> 14 & 2u) | (nan >> 21 & 4u) | (nan >> 28 & 8u)) << (key + 4 * d));
        }
      }
    };
    f32x16 sc[2];
    bf16x8 pf[4];
    float back = 1.f;
    // operand of product i of a turn: V^T of stage st - 1 (i < 16: 16 keys i / 4, channels 32 (i mod 4) ..), K of stage st + 1 (key tile (i - 16) / 8, channels 16 (i mod 8) ..)
    const unsigned v_off = 2 * KV4_KB + col * 128 + ((hh ^ ((col >> 1) & 7) ^ (col & 1)) << 4), k_row = swap23(col), k_off = k_row * 256 + ((hh ^ (k_row & 15)) << 4);
    auto operand = [&](auto I, int st) -> u32x4 {
      constexpr int i = decltype(I)::value;
      if constexpr (i < 16) return *reinterpret_cast<const u32x4*>(lds + ((v_off + ((st + 1) & 1) * KV4_VB) ^ (((i >> 2) ^ (i & 3)) << 5)) + (i & 3) * 4096);
      else return *reinterpret_cast<const u32x4*>(lds + ((k_off + ((st + 1) & 1) * KV4_KB) ^ ((i & 7) << 5)) + ((i - 16) >> 3) * 8192);
    };
    auto product = [&](auto I, const u32x4& x) {
      constexpr int i = decltype(I)::value;
      if constexpr (i < 16) o[i & 3] = mfma32(as_bf16x8(x), pf[i >> 2], o[i & 3]);
      else {
        constexpr int T = (i - 16) >> 3;
        if constexpr ((i & 7) == 0) {
#pragma unroll
          for (int z = 0; z < 16; ++z) sc[T][z] = 0.f;
        }
        sc[T] = mfma32(as_bf16x8(x), as_bf16x8(qf[i & 7]), sc[T]);
      }
    };
    // NaN values of a stage into the rows that see them
    auto put_nan = [&](int st) {
      const int seen = lim - st * KV4_STAGE;                                // keys 0 .. seen of the stage
      const unsigned long long mine = seen >= 63 ? ~0ull : seen < 0 ? 0ull : (2ull << seen) - 1;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const bool put = (bad[st & 3][d] & mine) != 0;
        if (__any(put)) {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[d][i] = put ? __builtin_nanf("") : o[d][i];
        }
      }
    };

    Kv4Stage<U> x;
    const int top_st = s1 - 1;
    if (t < 16) bad[t >> 2][t & 3] = 0ull;
    const std::integral_constant<int, 0> first; const std::integral_constant<int, 1> second;
    {                                                                       // all in flight at once
      Kv4Stage<U> y, z;
      fetch_k(y, s0);
      fetch_k(z, min(s0 + 1, top_st));
      fetch_k(x, min(s0 + 2, top_st));
      fetch_v(x, s0);
      put_k(first, y, s0); put_k(second, y, s0);
      put_k(first, z, s0 + 1); put_k(second, z, s0 + 1);
    }
    for (int i = t; i < KV4_VB / 16; i += NW * 64)                          // the stage before the first
      *reinterpret_cast<u32x4*>(lds + 2 * KV4_KB + ((s0 + 1) & 1) * KV4_VB + i * 16) = (u32x4){0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < 4; ++u) pf[u] = as_bf16x8((u32x4){0, 0, 0, 0});
    __syncthreads();
    unrolled<16>([&](auto I) { const std::integral_constant<int, 16 + decltype(I)::value> J; product(J, operand(J, s0 - 1)); });
    __syncthreads();                                                        // K of the first stage is read before its slot is filled again
    // A turn: the softmax of stage st beside the products that do not wait for it, P V of the stage before and K Q^T of the one behind; K of st + 2 and V of
    // st go to LDS, those of the turn behind are fetched.
    for (int st = s0; st < s1; ++st) {
      if (masked(st)) {
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[T][i] = st * KV4_STAGE + T * 32 + (i >> 3) * 16 + hh * 8 + (i & 7) <= lim ? sc[T][i] : -INFINITY;
        hide(x, st);
        if (st - 2 >= s0 && masked(st - 2)) put_nan(st - 2);                // O holds the stages up to that one
      }
      if (__any(back != 1.f)) {                                             // the maximum has moved in the turn before: O is one stage behind
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] *= back;
      }
      if (t < 4) bad[(st + 1) & 3][t] = 0ull;                               // last read a turn ago, next written a turn on
      // 32 products, their operands read four ahead, and the vector work dealt out between them
      u32x4 fr[5], pn[4];
      unsigned cv[8];
      float t0 = 0.f, t1 = 0.f, mu = 0.f, ms = 0.f, f = 1.f;
      unrolled<4>([&](auto I) { fr[decltype(I)::value] = operand(I, st); });
      unrolled<32>([&](auto I) {
        constexpr int i = decltype(I)::value;
        if constexpr (i + 4 < 32) fr[(i + 4) % 5] = operand(std::integral_constant<int, i + 4>{}, st);
        product(I, fr[i % 5]);
        if constexpr (i < 2) {
          float& tt = i == 0 ? t0 : t1;
          tt = sc[i][0];
#pragma unroll
          for (int z = 1; z < 16; ++z) tt = __builtin_fmaxf(tt, sc[i][z]);
        } else if constexpr (i == 2) {
          const float top = xor32_max(__builtin_fmaxf(t0, t1));
          const float mn = top > m ? top + KV4_SLACK : m;
          mu = mn == -INFINITY ? 0.f : mn;
          f = kv4_weight(m, mu);
          m = mn;
          l *= f;
          ms = mu * KV4_SCALE;
          if (__any(__builtin_fabsf(ms) > KV4_FUSED)) {
#pragma unroll
            for (int z = 0; z < 32; ++z) sc[z >> 4][z & 15] -= mu;
            ms = 0.f;
          }
        } else if constexpr (i < 19) {                                      // two probabilities: the first tile's before its scores are overwritten, the second's too
          constexpr int k = i - 3;
          const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[k >> 3][(2 * k) & 15], KV4_SCALE, -ms)), p1 = __builtin_amdgcn_exp2f(fmaf(sc[k >> 3][(2 * k + 1) & 15], KV4_SCALE, -ms));
          l += p0 + p1;
          pn[k >> 2][k & 3] = pack2(p0, p1);
        } else if constexpr (i < 19 + 2 * U) {                              // V a unit at a time: converted, put
          constexpr int u = (i - 19) >> 1;
          if constexpr (((i - 19) & 1) == 0) {
#pragma unroll
            for (int d = 0; d < 2; ++d) {
              cv[4 * d] = fp4_pair<0>(x.v[u][d], scale_of<0>(x.s[u][d])); cv[4 * d + 1] = fp4_pair<1>(x.v[u][d], scale_of<1>(x.s[u][d]));
              cv[4 * d + 2] = fp4_pair<2>(x.v[u][d], scale_of<2>(x.s[u][d])); cv[4 * d + 3] = fp4_pair<3>(x.v[u][d], scale_of<3>(x.s[u][d]));
            }
          } else put_v(u, cv, st);
        } else if constexpr (i >= 23 && i < 25) put_k(std::integral_constant<int, i - 23>{}, x, st + 2);
        else if constexpr (i == 25) fetch_k(x, min(st + 3, top_st));
        else if constexpr (i == 27) fetch_v(x, min(st + 1, top_st));
      });
#pragma unroll
      for (int u = 0; u < 4; ++u) pf[u] = as_bf16x8(pn[u]);
      back = f;
      __syncthreads();
    }
    if (top_st - 1 >= s0 && masked(top_st - 1)) put_nan(top_st - 1);
#pragma unroll
    for (int d = 0; d < 4; ++d) o[d] *= back;
    unrolled<16>([&](auto I) { product(I, operand(I, top_st + 1)); });
    if (masked(top_st)) put_nan(top_st);
    l = xor32_sum(l);
  }
  // The result goes through LDS, a wave by itself, 32 columns x 64 channels at a time (16-byte chunks permuted by the column): a store is then of four columns' 256 bytes.
  // Straight from the registers, 32 bytes of a column at a time, the partials of 17 rows in 64 splits took 9 us of 21.
  const float f = nsplit > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
  const int mine = valid ? (q0 + r) * n_q_heads + hk * G + h : -1;
  if (nsplit > 1 && valid && hh == 0) { ws_ml[((size_t)mine * nsplit + split) * 2] = m; ws_ml[((size_t)mine * nsplit + split) * 2 + 1] = l; }
  __syncthreads();                                                          // every wave has read its operands
  unsigned char* tr = lds + wave * 8192;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int d = 0; d < 2; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x16& v = o[2 * half + d];
        *reinterpret_cast<f32x4*>(tr + col * 256 + (((d * 8 + 2 * i + hh) ^ (col & 15)) << 4)) = (f32x4){v[4 * i] * f, v[4 * i + 1] * f, v[4 * i + 2] * f, v[4 * i + 3] * f};
      }
    wave_lds_order();
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int cc = it * 4 + (lane >> 4), row = __shfl(mine, cc, 64), ch = half * 64 + (lane & 15) * 4;
      const f32x4 v = *reinterpret_cast<const f32x4*>(tr + cc * 256 + (((lane & 15) ^ (cc & 15)) << 4));
      if (row < 0) continue;
      if (nsplit > 1) *reinterpret_cast<f32x4*>(ws_o + ((size_t)row * nsplit + split) * 128 + ch) = v;
      else st8(out + (size_t)row * 128 + ch, (u32x2){pack2(v[0], v[1]), pack2(v[2], v[3])});
    }
    wave_lds_order();
  }
}

// Tile height -- which of the three kernels -- and key splits, by a cost in us.  All: 4 for the launch and the way to the first key; splits another launch (3) and their
// partials, 1,040 bytes a row, head and split written and read at 4.5 TB/s.
//   16 columns (attn_rows_kv4_kernel): a wave's 32-key block takes 1.1 when waves are few and 0.75 of a SIMD's time when they are many, a block of eight waves 1.7
//   besides.
//   128 or 256 columns (attn_chunk_kv4_kernel of four waves, two blocks a unit, or eight): a stage of 64 keys 1.6 (four waves: alone on a unit 1.2, two blocks 1.8), 3
//   stages for a block's prologue and result and 3 for the masked end; blocks that all run at once take as long as the longest, more of them (longest first) the mean
//   and half of one.
// Measured, 16 / 128 columns (us): 28 / 4 heads on 26,000 keys 2 rows 11.8 / 20.3, 8 rows 17.3 / 23.5, 12 rows 22.5 / 25.3, 18 rows 29.6 / 27.2; 18 rows on 500 keys of
// 64 / 8 heads 7.9 / 15.8; 8 x 18 rows on 3,000 keys 30.3 / 27.7.  128 / 256 columns: 8 x ~340 rows on ~5,000 keys 266 / 263, 386 rows on 6,100 60 / 56.
int kv4_prefill_plan(const int32_t* n_new, const int32_t* past, int n, int n_q_heads, int n_kv_heads, int cus, int* tile_rows, int* nsplit) {
  if (n < 0 || n_q_heads < 1 || n_kv_heads < 1 || n_q_heads % n_kv_heads || n_q_heads / n_kv_heads > 16 || cus < 1) return LCC_ERR_SHAPE;
  const int G = n_q_heads / n_kv_heads;
  long rows = 0;
  for (int i = 0; i < n; ++i) {
    if (n_new[i] < 0 || past[i] < 0) return LCC_ERR_SHAPE;
    rows += n_new[i];
  }
  const float join = rows * (float)n_q_heads * (1040.f / 4.5e6f);
  float best = 1e30f;
  *tile_rows = 256 / G; *nsplit = 1;
  for (const int columns : {16, 128, 256}) {
    const int height = columns / G, keys = columns == 16 ? 32 : KV4_STAGE;
    long tiles = 0, total = 0, longest = 0;                                 // stages (blocks of 32 keys) of a KV head
    for (int i = 0; i < n; ++i) {
      const long count = ((long)n_new[i] + height - 1) / height;
      tiles += count;
      for (long z = 0; z < std::min(count, 64L); ++z) {                     // of many tiles 64 spread over the stream stand for all
        const long t = count <= 64 ? z : z * count / 64, st = (past[i] + std::min<long>(n_new[i], (t + 1) * height) + keys - 1) / keys;
        total += count <= 64 ? st : st * count / 64;
        longest = std::max(longest, st);
      }
    }
    if (tiles > 65535) continue;
    for (int k = 1; k <= 64 && k <= std::max(1L, longest / 4); ++k) {
      const float blocks = (float)tiles * n_kv_heads * k, work = (float)total * n_kv_heads;
      float cost = 4.f + (k > 1 ? 3.f + join * k : 0.f);
      if (columns == 16) {
        const float one = 1.1f * (float)((longest + (k == 1 ? 8 : 4) * k - 1) / ((k == 1 ? 8 : 4) * k)), all = work * 0.75f / (4.f * cus);
        cost += std::max(one, all + (blocks > cus ? 0.5f * one + (k == 1 ? 1.7f : 0.85f) * (blocks / cus - 1.f) : 0.f));
      } else {
        const float slots = (float)cus * (columns == 128 ? 2 : 1), block = (float)longest / k + 6.f;
        cost += blocks <= slots ? (columns == 256 ? 1.6f : blocks <= cus ? 1.2f : 1.8f) * block
                                : (columns == 256 ? 1.6f : 1.5f) * ((work + 3.f * blocks + 3.f * tiles * n_kv_heads) / slots + 0.5f * block);
      }
      if (cost < best) { best = cost; *tile_rows = height; *nsplit = k; }
    }
  }
  return 0;
}

int attn_prefill_kv4(const Kv4Args& a, const bf16_t* q, bf16_t* out, const int32_t* tile_stream, const int32_t* tile_q0, const int32_t* tile_nq, const int32_t* tile_pos0,
                     int n_tiles, int n_q_heads, int tile_rows, int nsplit, int n_rows, float* ws_o, float* ws_ml, hipStream_t st) {
  if (int rc = a.check()) return rc;
  if (n_tiles < 0 || n_tiles > 65535 || n_rows < 0 || n_q_heads < 1 || n_q_heads % a.n_kv_heads || n_q_heads / a.n_kv_heads > 16 || nsplit < 1 || nsplit > 64)
    return LCC_ERR_SHAPE;
  if (tile_rows < 1 || tile_rows > 256 / (n_q_heads / a.n_kv_heads) || (int64_t)n_rows * n_q_heads > 0x7fffffff) return LCC_ERR_SHAPE;
  if (nsplit > 1 && (ws_o == nullptr || ws_ml == nullptr)) return LCC_ERR_ARG;
  if (n_tiles == 0 || n_rows == 0) return 0;
  static DeviceOnce once;
  if (auto turn = once.first()) {
    (void)hipFuncSetAttribute((const void*)attn_chunk_kv4_kernel<8>, hipFuncAttributeMaxDynamicSharedMemorySize, KV4_LDS);
    (void)hipFuncSetAttribute((const void*)attn_chunk_kv4_kernel<4>, hipFuncAttributeMaxDynamicSharedMemorySize, KV4_LDS);
  }
  const dim3 grid(a.n_kv_heads, n_tiles, nsplit);
  if (tile_rows * (n_q_heads / a.n_kv_heads) <= 16)
    attn_rows_launch<true>(a, Kv4Rows{tile_stream, nullptr, tile_q0, tile_nq, tile_pos0, tile_rows, n_rows}, n_tiles, q, n_q_heads, nsplit, ws_o, ws_ml, out, st);
  else if (tile_rows * (n_q_heads / a.n_kv_heads) > 128)
    attn_chunk_kv4_kernel<8><<<grid, dim3(512), KV4_LDS, st>>>(a, q, out, tile_stream, tile_q0, tile_nq, tile_pos0, n_q_heads, tile_rows, nsplit, n_rows, ws_o, ws_ml);
  else
    attn_chunk_kv4_kernel<4><<<grid, dim3(256), KV4_LDS, st>>>(a, q, out, tile_stream, tile_q0, tile_nq, tile_pos0, n_q_heads, tile_rows, nsplit, n_rows, ws_o, ws_ml);
  if (nsplit > 1) kv4_combine(ws_o, ws_ml, out, tile_q0, tile_nq, n_tiles, tile_rows, n_rows, n_q_heads, nsplit, st);
  return 0;
}

}  // namespace lcc
