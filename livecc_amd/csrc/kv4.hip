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
#include "common.h"
#include "kernels.h"

namespace lcc {

typedef __attribute__((ext_vector_type(16))) float f32x16;

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

// byte SEL of `w` -> its two values under `scale`, of which the conversion reads the exponent field alone: the mantissa and sign may hold anything
template <int SEL>
LCC_DEVICE unsigned fp4_pair(unsigned w, unsigned scale) { return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, __uint_as_float(scale), SEL)); }
// scale byte SEL of `w` in the exponent field
template <int SEL>
LCC_DEVICE unsigned scale_of(unsigned w) { return SEL < 3 ? w << (23 - 8 * SEL) : w >> 1; }
// a word of K codes -> eight channels
LCC_DEVICE u32x4 fp4_word(unsigned w, unsigned scale) { return (u32x4){fp4_pair<0>(w, scale), fp4_pair<1>(w, scale), fp4_pair<2>(w, scale), fp4_pair<3>(w, scale)}; }
// eight V bytes (keys 0..7 of an octet) and their eight scale bytes -> the octet's values of channel i (lo) and i + 16 (hi)
LCC_DEVICE void fp4_octet(u32x2 w, u32x2 s, u32x4& lo, u32x4& hi) {
  unsigned c[8];
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    c[4 * d] = fp4_pair<0>(w[d], scale_of<0>(s[d])); c[4 * d + 1] = fp4_pair<1>(w[d], scale_of<1>(s[d]));
    c[4 * d + 2] = fp4_pair<2>(w[d], scale_of<2>(s[d])); c[4 * d + 3] = fp4_pair<3>(w[d], scale_of<3>(s[d]));
  }
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    lo[d] = __builtin_amdgcn_perm(c[2 * d + 1], c[2 * d], 0x05040100u);
    hi[d] = __builtin_amdgcn_perm(c[2 * d + 1], c[2 * d], 0x07060302u);
  }
}

// ------------------------------------------------------------------------------------------------------------------------------
// Norm, rotation, append.
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
// over the four lanes that hold a group
LCC_DEVICE int max4(int a) {
  a = max(a, __shfl_xor(a, 1, 64));
  return max(a, __shfl_xor(a, 2, 64));
}

// eight channels of a row: bf16, or bf16(sum of the slabs + bias)
LCC_DEVICE void row8(const QkNormArgs& a, int s, int col, float* v) {
  const int ld = (a.n_q_heads + 2 * a.n_kv_heads) * 128;
  if (a.partial == nullptr) {
    const u32x4 x = ld16(a.qkv + (size_t)s * ld + col);
#pragma unroll
    for (int d = 0; d < 4; ++d) { v[2 * d] = lo2f(x[d]); v[2 * d + 1] = hi2f(x[d]); }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
  for (int sp = 0; sp < a.nsplit; ++sp) {
    const float* p = a.partial + ((size_t)sp * a.rows + s) * ld + col;
    const f32x4 x = *reinterpret_cast<const f32x4*>(p), y = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] += x[e]; v[4 + e] += y[e]; }
  }
  const u32x4 b = a.bias != nullptr ? ld16(a.bias + col) : (u32x4){0, 0, 0, 0};
#pragma unroll
  for (int d = 0; d < 4; ++d) { v[2 * d] = rbf(v[2 * d] + lo2f(b[d])); v[2 * d + 1] = rbf(v[2 * d + 1] + hi2f(b[d])); }
}

// RMS norm of a head's 128 channels over its eight lanes, with the model's rounding points: bf16(w bf16(x r)).  The mean square and its root are formed in 64
// bits and r is rounded once: keys are quantised behind this, and codes must not depend on the order of a sum.
LCC_DEVICE void head_norm(float (&x1)[8], float (&x2)[8], const bf16_t* w, int c0, float eps) {
  double ss = 0.0;
#pragma unroll
  for (int e = 0; e < 8; ++e) { ss = fma((double)x1[e], (double)x1[e], ss); ss = fma((double)x2[e], (double)x2[e], ss); }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) ss += __shfl_xor(ss, o, 64);
  const double m = ss * (1.0 / 128) + (double)eps;
  double r = __builtin_amdgcn_rsq(m);
  if (m < __builtin_inf()) r = fma(0.5 * r, fma(-m * r, r, 1.0), r);        // the unit's result is good to about 2^-28; one step squares that
  const float rf = (float)r;
  const u32x4 w1 = ld16(w + c0), w2 = ld16(w + c0 + 64);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a = (e & 1) ? hi2f(w1[e >> 1]) : lo2f(w1[e >> 1]), b = (e & 1) ? hi2f(w2[e >> 1]) : lo2f(w2[e >> 1]);
    x1[e] = rbf(a * rbf(x1[e] * rf));
    x2[e] = rbf(b * rbf(x2[e] * rf));
  }
}

// Eight lanes a (row, head): lane j holds channels 8 j .. + 7 and 64 + 8 j .. + 7, the rotation's pairs and, four lanes each, two groups of the 4-bit
// format (2 shuffles a group, 3 for the norm).
template <bool KV4>
__global__ __launch_bounds__(256) void qk_norm_rope_append_kernel(QkNormArgs a) {
  const int per_row = a.n_q_heads + 2 * a.n_kv_heads;
  const int64_t item = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
  if (item >= (int64_t)a.rows * per_row) return;                            // whole groups of eight lanes
  const int s = (int)(item / per_row), head = (int)(item - (int64_t)s * per_row), j = threadIdx.x & 7, c0 = j * 8;
  const int kind = head < a.n_q_heads ? 0 : head < a.n_q_heads + a.n_kv_heads ? 1 : 2, h = kind == 0 ? head : (head - a.n_q_heads) - (kind - 1) * a.n_kv_heads;
  float x1[8], x2[8];
  row8(a, s, head * 128 + c0, x1);
  row8(a, s, head * 128 + 64 + c0, x2);
  u32x4 r1, r2;
  if (kind < 2) {
    const bf16_t* w = kind == 0 ? a.q_norm : a.k_norm;
    if (w != nullptr) head_norm(x1, x2, w, c0, a.eps);
    const u32x4 cq = ld16(a.cos + (size_t)s * 64 + c0), sq = ld16(a.sin + (size_t)s * 64 + c0);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      float o1[2], o2[2];
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const float c = z ? hi2f(cq[d]) : lo2f(cq[d]), sv = z ? hi2f(sq[d]) : lo2f(sq[d]), u = x1[2 * d + z], v = x2[2 * d + z];
        o1[z] = rbf(u * c) + rbf(-v * sv);
        o2[z] = rbf(v * c) + rbf(u * sv);
      }
      r1[d] = pack2(o1[0], o1[1]); r2[d] = pack2(o2[0], o2[1]);
    }
    if (kind == 0) {
      bf16_t* q = a.q_out + ((size_t)s * a.n_q_heads + h) * 128 + c0;
      st16(q, r1); st16(q + 64, r2);
      return;
    }
  } else {
#pragma unroll
    for (int d = 0; d < 4; ++d) { r1[d] = pack2(x1[2 * d], x1[2 * d + 1]); r2[d] = pack2(x2[2 * d], x2[2 * d + 1]); }
  }
  const int slot = a.tok_stream[s];
  if (slot < 0 || slot >= a.n_slots) return;                                // a row of no stream
  const int pos = a.tok_pos != nullptr ? a.tok_pos[s] : a.kv_len[slot];
  if (pos < 0 || pos >= a.lmax) return;
  if (!KV4) {
    const size_t kv = (size_t)a.n_kv_heads * a.lmax * 128;
    bf16_t* base = (bf16_t*)a.kv_base[slot] + (size_t)a.layer * 2 * kv;
    if (kind == 1) {
      bf16_t* k = base + ((size_t)h * a.lmax + pos) * 128 + c0;
      st16(k, r1); st16(k + 64, r2);
    } else {
      bf16_t* v = base + kv + (size_t)h * a.lmax * 128 + ((size_t)(pos >> 5) * 128 + c0) * 32 + (pos & 31);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e * 32] = (bf16_t)((e & 1) ? r1[e >> 1] >> 16 : r1[e >> 1]);
        v[(64 + e) * 32] = (bf16_t)((e & 1) ? r2[e >> 1] >> 16 : r2[e >> 1]);
      }
    }
  } else {
    const Kv4Layout lay{a.n_kv_heads, a.lmax};
    uint8_t* base = (uint8_t*)a.kv_base[slot] + (size_t)a.layer * lay.layer_bytes();
    const int e1 = kv4_exponent(max4(max_bits(r1))), e2 = kv4_exponent(max4(max_bits(r2)));       // groups j / 4 and 2 + j / 4
    const unsigned w1 = fp4_of(r1, e1), w2 = fp4_of(r2, e2);
    if (kind == 1) {
      unsigned* k = (unsigned*)(base + lay.k_codes(h) + (size_t)pos * 64);
      k[j] = w1; k[8 + j] = w2;
      if ((j & 3) == 0) {
        uint8_t* sc = base + lay.k_scales(h) + (size_t)pos * 4;
        sc[j >> 2] = (uint8_t)e1; sc[2 + (j >> 2)] = (uint8_t)e2;
      }
    } else {
      // channels i and 16 + i of a group lie two lanes apart: the lower pair of lanes takes the lower group's bytes, the upper pair the upper group's
      const bool up = (j & 2) != 0;
      const unsigned mine = up ? w2 : w1, other = __shfl_xor(up ? w1 : w2, 2, 64);
      const unsigned lo = up ? other : mine, hi = up ? mine : other;
      const int t = up ? 2 + (j >> 2) : j >> 2;
      uint8_t* v = base + lay.v_codes(h) + (size_t)(pos >> 5) * 2048 + ((pos & 31) >> 3) * 512 + (j & 1) * 256 + t * 8 + (pos & 7);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e * 32] = (uint8_t)((lo >> (4 * e) & 15) | (hi >> (4 * e) & 15) << 4);
      if ((j & 1) == 0) base[lay.v_scales(h) + (size_t)(pos >> 5) * 128 + ((pos & 31) >> 3) * 32 + t * 8 + (pos & 7)] = (uint8_t)(up ? e2 : e1);
    }
  }
}

static int qk_norm_check(const QkNormArgs& a) {
  if (a.rows < 0 || a.n_q_heads < 0 || a.n_kv_heads < 1 || a.lmax < 32 || (a.lmax & 31) || a.n_layers < 1 || a.layer < 0 || a.layer >= a.n_layers || a.n_slots < 0)
    return LCC_ERR_SHAPE;
  if (a.partial != nullptr && (a.nsplit < 1 || a.nsplit > 8)) return LCC_ERR_SHAPE;
  if (!(a.eps > 0.f) && (a.q_norm != nullptr || a.k_norm != nullptr)) return LCC_ERR_ARG;
  return 0;
}
int qk_norm_rope_append(const QkNormArgs& a, bool kv4, hipStream_t st) {
  if (int rc = qk_norm_check(a)) return rc;
  if (a.rows == 0) return 0;
  const int64_t blocks = ((int64_t)a.rows * (a.n_q_heads + 2 * a.n_kv_heads) + 31) / 32;
  if (blocks > 0x7fffffff) return LCC_ERR_SHAPE;
  if (kv4) qk_norm_rope_append_kernel<true><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(a);
  else qk_norm_rope_append_kernel<false><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(a);
  return 0;
}

// ------------------------------------------------------------------------------------------------------------------------------
// Read-back: row s = (slot, position) -> its keys and values [heads][128] in bf16; a row of no stream or position: zeros.  Eight lanes a (row, head), 16 channels
// each.
// ------------------------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4Args a, const int32_t* __restrict__ tok_stream, const int32_t* __restrict__ tok_pos,
                                                       bf16_t* __restrict__ k_out, bf16_t* __restrict__ v_out, int rows) {
  const int64_t item = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
  if (item >= (int64_t)rows * a.n_kv_heads) return;
  const int s = (int)(item / a.n_kv_heads), h = (int)(item - (int64_t)s * a.n_kv_heads), j = threadIdx.x & 7;
  const int slot = tok_stream[s], pos = tok_pos[s];
  bf16_t *ko = k_out + (size_t)item * 128 + j * 16, *vo = v_out + (size_t)item * 128 + j * 16;
  u32x4 k0 = {0, 0, 0, 0}, k1 = k0, v0 = k0, v1 = k0;
  if (slot >= 0 && slot < a.n_slots && pos >= 0 && pos < a.lmax) {
    const Kv4Layout lay{a.n_kv_heads, a.lmax};
    const uint8_t* base = (const uint8_t*)a.kv_base[slot] + (size_t)a.layer * lay.layer_bytes();
    const u32x2 kc = ld8(base + lay.k_codes(h) + (size_t)pos * 64 + j * 8);
    const unsigned ks = (unsigned)base[lay.k_scales(h) + (size_t)pos * 4 + (j >> 1)] << 23;
    k0 = fp4_word(kc[0], ks); k1 = fp4_word(kc[1], ks);
    const int t = j >> 1, sh = (j & 1) * 4, g = (pos & 31) >> 3, e = pos & 7;
    const uint8_t* vc = base + lay.v_codes(h) + (size_t)(pos >> 5) * 2048 + g * 512 + t * 8 + e;
    const unsigned vs = (unsigned)base[lay.v_scales(h) + (size_t)(pos >> 5) * 128 + g * 32 + t * 8 + e] << 23;
    unsigned w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i >> 3] |= (unsigned)(vc[i * 32] >> sh & 15) << (4 * (i & 7));
    v0 = fp4_word(w[0], vs); v1 = fp4_word(w[1], vs);
  }
  st16(ko, k0); st16(ko + 8, k1); st16(vo, v0); st16(vo + 8, v1);
}
int kv4_read(const Kv4Args& a, const int32_t* tok_stream, const int32_t* tok_pos, bf16_t* k, bf16_t* v, int rows, hipStream_t st) {
  if (int rc = a.check()) return rc;
  if (rows < 0) return LCC_ERR_SHAPE;
  if (rows == 0) return 0;
  const int64_t blocks = ((int64_t)rows * a.n_kv_heads + 31) / 32;
  if (blocks > 0x7fffffff) return LCC_ERR_SHAPE;
  kv4_read_kernel<<<dim3((unsigned)blocks), dim3(256), 0, st>>>(a, tok_stream, tok_pos, k, v, rows);
  return 0;
}

// ------------------------------------------------------------------------------------------------------------------------------
// Decode attention: one row per stream.  Block = (KV head, row, key split), its waves take the split's 32-key blocks in turn; a wave's 16 columns are the query
// heads of the KV head.  S^T = K Q^T: operand A is 16 keys x 32 channels, a lane's 16 bytes of codes (one group of one key) its share of all four steps -- the
// channels of step s are 8 s .. 8 s + 7 of each group, for Q alike.  Rows of the two key tiles are dealt so that a lane's eight scores are of the keys
// 8 g .. 8 g + 7, which are the slots of its P operand: O^T += V^T P^T takes the probabilities from the softmax' registers and V's bytes as they lie.
// ------------------------------------------------------------------------------------------------------------------------------
struct Kv4Tile { u32x4 k[2], v[2], s[2]; unsigned ks[2]; };       // what a wave loads of a 32-key block: codes of two key tiles, of V, V's scales, K's
LCC_DEVICE void kv4_load(Kv4Tile& t, const uint8_t* kc, const uint8_t* vc, const uint8_t* ks, const uint8_t* vs, int blk, int li, int g) {
  const int key = 8 * (li >> 2) + (li & 3);
#pragma unroll
  for (int T = 0; T < 2; ++T) {
    t.k[T] = ld16(kc + ((size_t)blk * 32 + key + 4 * T) * 64 + g * 16);
    t.ks[T] = ks[((size_t)blk * 32 + key + 4 * T) * 4 + g];
  }
  const uint8_t* v = vc + (size_t)blk * 2048 + g * 512 + li * 32;
  const uint8_t* s = vs + (size_t)blk * 128 + g * 32;
  t.v[0] = ld16(v); t.v[1] = ld16(v + 16); t.s[0] = ld16(s); t.s[1] = ld16(s + 16);
}

template <int NW>
__global__ __launch_bounds__(NW * 64, 2) void attn_decode_kv4_kernel(Kv4Args a, const bf16_t* __restrict__ q, const int32_t* __restrict__ slots,
                                                                     const int32_t* __restrict__ kv_len, int n_q_heads, int nsplit,
                                                                     float* __restrict__ ws_o, float* __restrict__ ws_ml, bf16_t* __restrict__ out, float scale_log2e) {
  __shared__ float mo[NW][16][132];
  __shared__ float mm[NW][16], ml[NW][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4;
  const int split = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, G = n_q_heads / a.n_kv_heads;
  const int slot = slots[b];
  const bool live = slot >= 0 && slot < a.n_slots;
  const int n = live ? max(0, min(kv_len[slot], a.lmax - 1) + 1) : 0;       // keys (a length below zero: none)
  const int nblk = (n + 31) >> 5, per = (nblk + nsplit - 1) / nsplit, b0 = split * per, b1 = min(nblk, b0 + per);

  f32x4 o[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) o[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;                                             // m in units of log2
  int blk = b0 + wave;
  if (blk < b1) {
    const Kv4Layout lay{a.n_kv_heads, a.lmax};
    const uint8_t* base = (const uint8_t*)a.kv_base[slot] + (size_t)a.layer * lay.layer_bytes();
    const uint8_t *kc = base + lay.k_codes(hk), *vc = base + lay.v_codes(hk), *ks = base + lay.k_scales(hk), *vs = base + lay.v_scales(hk);
    u32x4 qf[4];
    const bf16_t* qp = q + ((size_t)b * n_q_heads + hk * G + min(li, G - 1)) * 128 + g * 32;
#pragma unroll
    for (int s = 0; s < 4; ++s) qf[s] = ld16(qp + 8 * s);
    Kv4Tile cur, nxt;
    kv4_load(cur, kc, vc, ks, vs, blk, li, g);
    for (; blk < b1; blk += NW) {
      if (blk + NW < b1) kv4_load(nxt, kc, vc, ks, vs, blk + NW, li, g);
      f32x4 sc[2];
#pragma unroll
      for (int T = 0; T < 2; ++T) {
        sc[T] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 4; ++s) sc[T] = mfma16(as_bf16x8(fp4_word(cur.k[T][s], cur.ks[T] << 23)), as_bf16x8(qf[s]), sc[T]);
      }
      const int left = n - blk * 32 - 8 * g;                                // keys of this lane's octet that exist
      if (n - blk * 32 < 32) {                                              // the last block: scores of no key to -inf, V there to zero (0 * NaN)
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[T][r] = 4 * T + r < left ? sc[T][r] : -INFINITY;
        const unsigned long long keep = left >= 8 ? ~0ull : left <= 0 ? 0ull : (1ull << (8 * left)) - 1;
#pragma unroll
        for (int t = 0; t < 2; ++t) { cur.s[t][0] &= (unsigned)keep; cur.s[t][1] &= (unsigned)(keep >> 32); cur.s[t][2] &= (unsigned)keep; cur.s[t][3] &= (unsigned)(keep >> 32); }
      }
      float top = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(sc[0][0], sc[0][1]), __builtin_fmaxf(sc[0][2], sc[0][3])),
                                  __builtin_fmaxf(__builtin_fmaxf(sc[1][0], sc[1][1]), __builtin_fmaxf(sc[1][2], sc[1][3])));
      top = __builtin_fmaxf(top, __shfl_xor(top, 16, 64));
      top = xor32_max(top);
      const float mn = __builtin_fmaxf(m, top * scale_log2e), mu = mn == -INFINITY ? 0.f : mn;
      if (__any(mn > m)) {
        const float f = __builtin_amdgcn_exp2f(m - mu);
        l *= f;
#pragma unroll
        for (int t = 0; t < 8; ++t) o[t] *= f;
        m = mn;
      }
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) { p[e] = __builtin_amdgcn_exp2f(fmaf(sc[e >> 2][e & 3], scale_log2e, -mu)); l += p[e]; }
      const bf16x8 pf = as_bf16x8((u32x4){pack2(p[0], p[1]), pack2(p[2], p[3]), pack2(p[4], p[5]), pack2(p[6], p[7])});
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        u32x4 lo, hi;
        fp4_octet((u32x2){cur.v[t >> 1][2 * (t & 1)], cur.v[t >> 1][2 * (t & 1) + 1]}, (u32x2){cur.s[t >> 1][2 * (t & 1)], cur.s[t >> 1][2 * (t & 1) + 1]}, lo, hi);
        o[2 * t] = mfma16(as_bf16x8(lo), pf, o[2 * t]);
        o[2 * t + 1] = mfma16(as_bf16x8(hi), pf, o[2 * t + 1]);
      }
      cur = nxt;
    }
    l += __shfl_xor(l, 16, 64);
    l = xor32_sum(l);
  }
  // the waves' parts, joined in LDS: column li, channels 16 t + 4 g .. + 3
#pragma unroll
  for (int t = 0; t < 8; ++t) *reinterpret_cast<f32x4*>(&mo[wave][li][16 * t + 4 * g]) = o[t];
  if (g == 0) { mm[wave][li] = m; ml[wave][li] = l; }
  __syncthreads();
  for (int i = threadIdx.x; i < G * 32; i += NW * 64) {
    const int h = i >> 5, c = (i & 31) * 4;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = __builtin_fmaxf(M, mm[w][h]);
    const float mu = M == -INFINITY ? 0.f : M;
    f32x4 acc = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(mm[w][h] - mu);
      L += f * ml[w][h];
      acc += f * *reinterpret_cast<const f32x4*>(&mo[w][h][c]);
    }
    const size_t row = (size_t)b * n_q_heads + hk * G + h;
    if (nsplit == 1) {
      const float r = L == 0.f ? 0.f : 1.f / L;
      st8(out + row * 128 + c, (u32x2){pack2(acc[0] * r, acc[1] * r), pack2(acc[2] * r, acc[3] * r)});
    } else {
      *reinterpret_cast<f32x4*>(ws_o + (row * nsplit + split) * 128 + c) = acc;
      if (c == 0) { ws_ml[(row * nsplit + split) * 2] = M; ws_ml[(row * nsplit + split) * 2 + 1] = L; }
    }
  }
}

// Joins the key splits of a (row, head): sums weighted by 2^(m - max), one rounding.
__global__ __launch_bounds__(256) void kv4_combine_kernel(const float* __restrict__ ws_o, const float* __restrict__ ws_ml, bf16_t* __restrict__ out, int nsplit) {
  __shared__ f32x4 so[8][32];
  __shared__ float sl[8];
  const size_t row = (size_t)blockIdx.x;
  const int grp = threadIdx.x >> 5, c = threadIdx.x & 31;
  float M = -INFINITY;
  for (int s = 0; s < nsplit; ++s) M = __builtin_fmaxf(M, ws_ml[(row * nsplit + s) * 2]);
  const float mu = M == -INFINITY ? 0.f : M;
  f32x4 acc = (f32x4){0.f, 0.f, 0.f, 0.f};
  float L = 0.f;
  for (int s = grp; s < nsplit; s += 8) {
    const float f = __builtin_amdgcn_exp2f(ws_ml[(row * nsplit + s) * 2] - mu);
    L += f * ws_ml[(row * nsplit + s) * 2 + 1];
    acc += f * *reinterpret_cast<const f32x4*>(ws_o + (row * nsplit + s) * 128 + c * 4);
  }
  so[grp][c] = acc;
  if (c == 0) sl[grp] = L;
  __syncthreads();
  if (grp != 0) return;
  for (int i = 1; i < 8; ++i) { acc += so[i][c]; L += sl[i]; }
  const float r = L == 0.f ? 0.f : 1.f / L;
  st8(out + row * 128 + c * 4, (u32x2){pack2(acc[0] * r, acc[1] * r), pack2(acc[2] * r, acc[3] * r)});
}

int kv4_decode_splits(const int32_t* n_keys, int n, int n_kv_heads) {
  long most = 1;
  for (int i = 0; i < n; ++i) most = n_keys[i] > most ? n_keys[i] : most;
  const long blocks = (most + 31) / 32, base = (long)(n > 0 ? n : 1) * n_kv_heads;
  long k = (512 + base - 1) / base;
  if (k > (blocks + 7) / 8) k = (blocks + 7) / 8;
  return (int)(k < 1 ? 1 : k > 64 ? 64 : k);
}

int attn_decode_kv4(const Kv4Args& a, const bf16_t* q, const int32_t* slots, const int32_t* kv_len, int rows, int n_q_heads, int nsplit, float* ws_o, float* ws_ml,
                    bf16_t* out, hipStream_t st) {
  if (int rc = a.check()) return rc;
  if (rows < 0 || rows > 65535 || n_q_heads < 1 || n_q_heads % a.n_kv_heads || n_q_heads / a.n_kv_heads > 16 || nsplit < 1 || nsplit > 64 || a.n_kv_heads > 65535)
    return LCC_ERR_SHAPE;
  if (nsplit > 1 && (ws_o == nullptr || ws_ml == nullptr)) return LCC_ERR_ARG;
  if (rows == 0) return 0;
  attn_decode_kv4_kernel<4><<<dim3(nsplit, a.n_kv_heads, rows), dim3(256), 0, st>>>(a, q, slots, kv_len, n_q_heads, nsplit, ws_o, ws_ml, out, 1.4426950408889634f / sqrtf(128.f));
  if (nsplit > 1) kv4_combine_kernel<<<dim3((unsigned)(rows * n_q_heads)), dim3(256), 0, st>>>(ws_o, ws_ml, out, nsplit);
  return 0;
}

// ------------------------------------------------------------------------------------------------------------------------------
// Attention of chunks: tiles of up to 256 / G consecutive new rows of one stream, their (row, head) pairs the 8 x 32 columns of a block's waves.  The
// block turns 64 keys at a time into bf16 in LDS (each thread eight bytes of K and of V) and every wave multiplies them: S^T = K Q^T and
// O^T += V^T P^T on 32x32x16, K's rows read in the order (bits 2 and 3 swapped) that leaves a lane the scores of the keys its P operand wants.
// ------------------------------------------------------------------------------------------------------------------------------
constexpr int KV4_STAGE = 64, KV4_KB = KV4_STAGE * 256, KV4_VB = 128 * KV4_STAGE * 2, KV4_LDS = 2 * (KV4_KB + KV4_VB);
struct Kv4Stage { u32x2 k, v, s; unsigned ks; };

__global__ __launch_bounds__(512, 2) void attn_prefill_kv4_kernel(Kv4Args a, const bf16_t* __restrict__ q, bf16_t* __restrict__ out, const int32_t* __restrict__ tile_stream,
                                                                  const int32_t* __restrict__ tile_q0, const int32_t* __restrict__ tile_nq,
                                                                  const int32_t* __restrict__ tile_pos0, int n_q_heads, int tile_rows, int nsplit, int n_rows,
                                                                  float* __restrict__ ws_o, float* __restrict__ ws_ml, float scale_log2e) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  __shared__ unsigned long long bad[3][4];                                  // keys of a stage, by group, whose V is NaN (stages with masked scores)
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
  const int lim = live ? pos0 + min(r, nq - 1) : -1;                        // last key this column sees
  const bool active = wave * 32 < nq * G;                                   // wave-uniform

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
    const int t = threadIdx.x, key = t >> 3, part = t & 7, vblk = t >> 8, vg = (t >> 6) & 3, vi = (t >> 2) & 15, vt = t & 3;
    auto fetch = [&](Kv4Stage& x, int st) {
      x.k = x.v = x.s = (u32x2){0u, 0u}; x.ks = 0u;
      if (st * KV4_STAGE + key < a.lmax) {
        x.k = ld8(kc + ((size_t)st * KV4_STAGE + key) * 64 + part * 8);
        x.ks = ksc[((size_t)st * KV4_STAGE + key) * 4 + (part >> 1)];
      }
      if (st * KV4_STAGE + vblk * 32 < a.lmax) {
        x.v = ld8(vc + ((size_t)st * 2 + vblk) * 2048 + (t & 255) * 8);
        x.s = ld8(vsc + ((size_t)st * 2 + vblk) * 128 + vg * 32 + vt * 8);
      }
    };
    auto masked = [&](int st) { return st * KV4_STAGE + KV4_STAGE - 1 > pos0; };          // some row does not see all of the stage
    auto stage = [&](Kv4Stage& x, int st) {
      unsigned char* kb = lds + (st & 1) * (KV4_KB + KV4_VB);
      unsigned char* vb = kb + KV4_KB;
      if (masked(st)) {
        // what a row does not see must not reach it through 0 * NaN: values behind the last key are zeros, and NaN values are zeros here and put into
        // the rows that see them behind the product
        const int k0 = st * KV4_STAGE + vblk * 32 + vg * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const unsigned byte = x.s[e >> 2] >> (8 * (e & 3)) & 255u;
          const bool nan = byte >= 253u;
          if (k0 + e >= nk || nan) x.s[e >> 2] &= ~(255u << (8 * (e & 3)));
          if (k0 + e < nk && nan && vi == 0) atomicOr(&bad[st % 3][vt], 1ull << (vblk * 32 + vg * 8 + e));
        }
      }
      const unsigned sc = x.ks << 23;
      *reinterpret_cast<u32x4*>(kb + key * 256 + (((2 * part) ^ (key & 15)) << 4)) = fp4_word(x.k[0], sc);
      *reinterpret_cast<u32x4*>(kb + key * 256 + (((2 * part + 1) ^ (key & 15)) << 4)) = fp4_word(x.k[1], sc);
      u32x4 lo, hi;
      fp4_octet(x.v, x.s, lo, hi);
      const int ch = vt * 32 + vi, chunk = vblk * 4 + vg;
      *reinterpret_cast<u32x4*>(vb + ch * 128 + ((chunk ^ ((ch >> 1) & 7)) << 4)) = lo;
      *reinterpret_cast<u32x4*>(vb + (ch + 16) * 128 + ((chunk ^ (((ch + 16) >> 1) & 7)) << 4)) = hi;
    };
    if (t < 12) bad[t >> 2][t & 3] = 0ull;
    __syncthreads();
    Kv4Stage x;
    fetch(x, s0);
    stage(x, s0);
    if (s0 + 1 < s1) fetch(x, s0 + 1);
    __syncthreads();
    const int krow = swap23(col);
    for (int st = s0; st < s1; ++st) {
      const unsigned char* kb = lds + (st & 1) * (KV4_KB + KV4_VB);
      const unsigned char* vb = kb + KV4_KB;
      if (t < 4) bad[(st + 2) % 3][t] = 0ull;                               // last read one stage ago, next written one stage on
      f32x16 sc[2];
      if (active) {
#pragma unroll
        for (int T = 0; T < 2; ++T) {
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[T][i] = 0.f;
          const int row = T * 32 + krow;
#pragma unroll
          for (int s = 0; s < 8; ++s)
            sc[T] = mfma32(as_bf16x8(*reinterpret_cast<const u32x4*>(kb + row * 256 + (((2 * s + hh) ^ (row & 15)) << 4))), as_bf16x8(qf[s]), sc[T]);
        }
      }
      if (st + 1 < s1) { stage(x, st + 1); if (st + 2 < s1) fetch(x, st + 2); }
      if (active) {
        if (masked(st)) {
#pragma unroll
          for (int T = 0; T < 2; ++T)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[T][i] = st * KV4_STAGE + T * 32 + (i >> 3) * 16 + hh * 8 + (i & 7) <= lim ? sc[T][i] : -INFINITY;
        }
        float top = sc[0][0];
#pragma unroll
        for (int i = 1; i < 32; ++i) top = __builtin_fmaxf(top, sc[i >> 4][i & 15]);
        top = xor32_max(top);
        const float mn = __builtin_fmaxf(m, top * scale_log2e), mu = mn == -INFINITY ? 0.f : mn;
        if (__any(mn > m)) {
          const float f = __builtin_amdgcn_exp2f(m - mu);
          l *= f;
#pragma unroll
          for (int d = 0; d < 4; ++d) o[d] *= f;
          m = mn;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) { p[e] = __builtin_amdgcn_exp2f(fmaf(sc[u >> 1][(u & 1) * 8 + e], scale_log2e, -mu)); l += p[e]; }
          const bf16x8 pf = as_bf16x8((u32x4){pack2(p[0], p[1]), pack2(p[2], p[3]), pack2(p[4], p[5]), pack2(p[6], p[7])});
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const int row = d * 32 + col;
            o[d] = mfma32(as_bf16x8(*reinterpret_cast<const u32x4*>(vb + row * 128 + (((2 * u + hh) ^ ((row >> 1) & 7)) << 4))), pf, o[d]);
          }
        }
        if (masked(st)) {
          const int seen = lim - st * KV4_STAGE;                            // keys 0 .. seen of the stage
          const unsigned long long mine = seen >= 63 ? ~0ull : seen < 0 ? 0ull : (2ull << seen) - 1;
#pragma unroll
          for (int d = 0; d < 4; ++d)
            if (bad[st % 3][d] & mine)
#pragma unroll
              for (int i = 0; i < 16; ++i) o[d][i] = __builtin_nanf("");
        }
      }
      __syncthreads();
    }
    l = xor32_sum(l);
  }
  if (!valid) return;
  const size_t row = (size_t)(q0 + r) * n_q_heads + hk * G + h;
  if (nsplit == 1) {
    const float f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        st8(out + row * 128 + d * 32 + 8 * i + 4 * hh, (u32x2){pack2(o[d][4 * i] * f, o[d][4 * i + 1] * f), pack2(o[d][4 * i + 2] * f, o[d][4 * i + 3] * f)});
  } else {
    float* w = ws_o + (row * nsplit + split) * 128;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<f32x4*>(w + d * 32 + 8 * i + 4 * hh) = (f32x4){o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
    if (hh == 0) { ws_ml[(row * nsplit + split) * 2] = m; ws_ml[(row * nsplit + split) * 2 + 1] = l; }
  }
}

int kv4_prefill_plan(const int32_t* n_new, const int32_t* past, int n, int n_q_heads, int n_kv_heads, int cus, int* tile_rows, int* nsplit) {
  if (n < 0 || n_q_heads < 1 || n_kv_heads < 1 || n_q_heads % n_kv_heads || n_q_heads / n_kv_heads > 16 || cus < 1) return LCC_ERR_SHAPE;
  const int rows = 256 / (n_q_heads / n_kv_heads);
  long tiles = 0, keys = 0;
  for (int i = 0; i < n; ++i) {
    if (n_new[i] < 0 || past[i] < 0) return LCC_ERR_SHAPE;
    tiles += (n_new[i] + rows - 1) / rows;
    if (n_new[i] > 0 && (long)past[i] + n_new[i] > keys) keys = (long)past[i] + n_new[i];
  }
  const long base = tiles * n_kv_heads, stages = (keys + KV4_STAGE - 1) / KV4_STAGE;
  *tile_rows = rows; *nsplit = 1;
  float best = 1e30f;
  for (int k = 1; k <= 32 && k <= (stages + 3) / 4; ++k) {
    const float cost = (float)((base * k + cus - 1) / cus) * ((float)stages / k + 3.f) + (k > 1 ? 4.f + 0.5f * k : 0.f);
    if (cost < best) { best = cost; *nsplit = k; }
  }
  return 0;
}

int attn_prefill_kv4(const Kv4Args& a, const bf16_t* q, bf16_t* out, const int32_t* tile_stream, const int32_t* tile_q0, const int32_t* tile_nq, const int32_t* tile_pos0,
                     int n_tiles, int n_q_heads, int tile_rows, int nsplit, int n_rows, float* ws_o, float* ws_ml, hipStream_t st) {
  if (int rc = a.check()) return rc;
  if (n_tiles < 0 || n_tiles > 65535 || n_rows < 0 || n_q_heads < 1 || n_q_heads % a.n_kv_heads || n_q_heads / a.n_kv_heads > 16 || nsplit < 1 || nsplit > 32)
    return LCC_ERR_SHAPE;
  if (tile_rows < 1 || tile_rows > 256 / (n_q_heads / a.n_kv_heads)) return LCC_ERR_SHAPE;
  if (nsplit > 1 && (ws_o == nullptr || ws_ml == nullptr)) return LCC_ERR_ARG;
  if (n_tiles == 0 || n_rows == 0) return 0;
  static DeviceOnce once;
  if (once.first()) (void)hipFuncSetAttribute((const void*)attn_prefill_kv4_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, KV4_LDS);
  attn_prefill_kv4_kernel<<<dim3(a.n_kv_heads, n_tiles, nsplit), dim3(512), KV4_LDS, st>>>(a, q, out, tile_stream, tile_q0, tile_nq, tile_pos0, n_q_heads, tile_rows,
                                                                                          nsplit, n_rows, ws_o, ws_ml, 1.4426950408889634f / sqrtf(128.f));
  if (nsplit > 1) kv4_combine_kernel<<<dim3((unsigned)n_rows * n_q_heads), dim3(256), 0, st>>>(ws_o, ws_ml, out, nsplit);
  return 0;
}

}  // namespace lcc
