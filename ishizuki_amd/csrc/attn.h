// What the attention kernels share: the 8-bit cache's geometry and codes, the call's rows, per-head
// norms and the position rotation.
#pragma once
#include <utility>

#include "common.h"

namespace attn {
// f(0) .. f(N - 1) with constants, for bodies too long for the unroller's limit.
template <class F, int... I>
DEV void unrolled(std::integer_sequence<int, I...>, F &&f) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
DEV void unrolled(F &&f) {
  unrolled(std::make_integer_sequence<int, N>{}, f);
}

constexpr int BLOCK = ISHZ_KV_BLOCK;  // tokens that share a scale, for each head

// The pool: codes of keys [blocks][heads][64][dim] and of values [blocks][heads][dim][64], their scales
// [blocks][heads]. Values stand with their tokens contiguous because P V contracts over tokens: a lane's
// 16-byte load is then a whole matrix operand, and neither keys nor values pass through LDS to be turned.
struct Pool {
  uint8_t *k, *v;
  float *ks, *vs;
  int blocks, heads, dim;
  // Offsets pass 32 bits in a long cache (64 heads * dim 128 * 64 tokens * 2^13 blocks = 2^32).
  DEV size_t tile(int block, int head) const { return ((size_t)block * heads + head) * (BLOCK * dim); }
  DEV size_t scale(int block, int head) const { return (size_t)block * heads + head; }
};

// The call's rows: sequence s has rows starts[s]..starts[s+1] of `rows` and lengths[s] tokens in the cache,
// those rows' own among them; its blocks are table[s * width ...]. Positions count from all lengths[s] tokens, also
// where the table is shorter: tokens past it are held nowhere, and those before stay where they are.
struct Rows {
  const int32_t *table, *lengths, *starts;
  int sequences, width, rows;
  DEV int first(int s) const { return min(max(starts[s], 0), rows); }
  DEV int count(int s) const { return max(min(starts[s + 1], rows) - first(s), 0); }
  DEV int length(int s) const { return max(lengths[s], 0); }
  DEV int held(int s) const { return min(length(s), width * BLOCK); }
  // The block that holds tokens 64 j.. of s, or -1: an entry outside the pool holds no tokens.
  DEV int block(int s, int j, int blocks) const {
    if (j < 0 || j >= width) return -1;
    const int b = table[(size_t)s * width + j];
    return b >= 0 && b < blocks ? b : -1;
  }
};

// ---------------------------------------------------------------- codes
template <int FMT>
constexpr float LIMIT = FMT == ISHZ_KV_INT8 ? 127.0f : 448.0f;

// Four codes as exact fp16 values. int8: offset by 128, each byte under the exponent byte of 1024 (0x64),
// minus 1152: one xor, two byte permutes, two packed subtractions. e4m3: two conversions of two.
template <int FMT>
DEV u2 decode4(uint32_t c) {
  if (FMT == ISHZ_KV_INT8) {
    c ^= 0x80808080u;
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    return u2{as_u32(as_h2(__builtin_amdgcn_perm(0x64646464u, c, 0x04010400u)) - off),
              as_u32(as_h2(__builtin_amdgcn_perm(0x64646464u, c, 0x04030402u)) - off)};
  }
  return u2{as_u32(__builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, false))),
            as_u32(__builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, true)))};
}
template <int FMT>
DEV h8 decode8(uint32_t lo, uint32_t hi) {
  const u2 a = decode4<FMT>(lo), b = decode4<FMT>(hi);
  return as_h8(u4{a.x, a.y, b.x, b.y});
}
// Four codes as fp32 values.
template <int FMT>
DEV f4 decode4f(uint32_t c) {
  if (FMT == ISHZ_KV_INT8)
    return f4{(float)(int8_t)c, (float)(int8_t)(c >> 8), (float)(int8_t)(c >> 16), (float)((int32_t)c >> 24)};
  return f4{__builtin_amdgcn_cvt_f32_fp8(c, 0), __builtin_amdgcn_cvt_f32_fp8(c, 1), __builtin_amdgcn_cvt_f32_fp8(c, 2),
            __builtin_amdgcn_cvt_f32_fp8(c, 3)};
}
// Four values, in units of the scale, as codes: the nearest, ties to even.
template <int FMT>
DEV uint32_t encode4(float a, float b, float c, float d) {
  const float m = LIMIT<FMT>;
  a = fminf(fmaxf(a, -m), m), b = fminf(fmaxf(b, -m), m), c = fminf(fmaxf(c, -m), m), d = fminf(fmaxf(d, -m), m);
  if (FMT == ISHZ_KV_INT8)
    return ((uint32_t)(int)rintf(a) & 255) | ((uint32_t)(int)rintf(b) & 255) << 8 | ((uint32_t)(int)rintf(c) & 255) << 16 |
           (uint32_t)(int)rintf(d) << 24;
  uint32_t r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// x / scale as a division rounds it, from up = 1 / scale: what the product leaves of x corrects it (two fused
// multiply-adds; the product alone is off by a step for a quarter of the values, which moves those at a border between
// codes). A zero keeps its sign. For scales below 2^-100, whose remainders leave fp32, to a step.
DEV float quotient(float x, float scale, float up) {
  const float q = x * up;
  return __builtin_fmaf(-__builtin_fmaf(q, scale, -x), up, q);
}

// ---------------------------------------------------------------- activations, eight at a time
template <int DT>
DEV void load8(const void *p, size_t i, float *o) {
  if (DT == ISHZ_DT_F32) {
    const f4 a = *(const f4 *)((const float *)p + i), b = *(const f4 *)((const float *)p + i + 4);
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = a[j], o[4 + j] = b[j];
  } else {
    const u4 v = *(const u4 *)((const uint16_t *)p + i);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      o[2 * j] = DT == ISHZ_DT_F16 ? h2f(v[j] & 0xffff) : __builtin_bit_cast(float, v[j] << 16);
      o[2 * j + 1] = DT == ISHZ_DT_F16 ? h2f(v[j] >> 16) : __builtin_bit_cast(float, v[j] & 0xffff0000u);
    }
  }
}
template <int DT>
DEV uint32_t narrow2(float a, float b) {
  if (DT == ISHZ_DT_F16) return (uint32_t)f2h(a) | (uint32_t)f2h(b) << 16;
  return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)b) << 16;
}
template <int DT, bool PAST = false>  // PAST: past the caches
DEV void store8(void *p, size_t i, const float *v) {
  const auto put = [&](u4 x, u4 *at) {
    if (PAST) __builtin_nontemporal_store(x, at);
    else *at = x;
  };
  if (DT == ISHZ_DT_F32) {
    put(__builtin_bit_cast(u4, (f4{v[0], v[1], v[2], v[3]})), (u4 *)((float *)p + i));
    put(__builtin_bit_cast(u4, (f4{v[4], v[5], v[6], v[7]})), (u4 *)((float *)p + i + 4));
  } else {
    put(u4{narrow2<DT>(v[0], v[1]), narrow2<DT>(v[2], v[3]), narrow2<DT>(v[4], v[5]), narrow2<DT>(v[6], v[7])}, (u4 *)((uint16_t *)p + i));
  }
}

// ---------------------------------------------------------------- norm and rotation of a head
// y = x * rsqrt(mean x^2 + eps) * w over the head, then the first `rot` values turned in pairs by their
// position's angle: (a, b) -> (a cos - b sin, b cos + a sin), pairs (i, i + rot/2) or, interleaved, (2i, 2i+1).
struct Turn {
  const int32_t *positions;
  const uint64_t *turns;  // [rot/2] turns a position, as fractions of 2^64
  int rot, interleaved;
  float factor;  // on both cosine and sine
};

// A lane holds two chunks of eight values of a head, chosen so that both values of every pair are its own:
// unit u of dim/16. Returns the chunks' first values.
DEV void unit_chunks(int u, int rot, bool interleaved, int *a, int *b) {
  if (interleaved || u >= rot / 16) *a = 16 * u, *b = 16 * u + 8;
  else *a = 8 * u, *b = rot / 2 + 8 * u;
}

// cos and sin of `phase` turns / 2^32. The angle never leaves the integers until it is within an eighth of a turn
// of a multiple of a quarter: a position's phase is the low 64 bits of position * turns, exact for any int32
// position, where an fp32 angle of position 10^6 is off by 0.06. Taylor series to 2^-25 on [-pi/4, pi/4].
DEV void cos_sin(uint32_t phase, float *c, float *s) {
  const uint32_t quarter = (phase + 0x20000000u) >> 30;
  const float t = (float)(int32_t)(phase - (quarter << 30)) * 1.46291807926715968e-9f;  // 2 pi / 2^32
  const float z = t * t;
  const float sn = t + t * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
  const float cs = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 - z * (1.0f / 3628800)))));
  const float x = quarter & 1 ? sn : cs, y = quarter & 1 ? cs : sn;
  *c = (quarter + 1) & 2 ? -x : x;
  *s = quarter & 2 ? -y : y;
}
DEV uint32_t phase_of(uint64_t turns, int32_t position) {
  return (uint32_t)(((uint64_t)(int64_t)position * turns) >> 32);
}
// The eight angles of unit u (u < rot / 16).
DEV void unit_angles(const Turn &t, int u, int32_t position, float *c, float *s) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    cos_sin(phase_of(t.turns[8 * u + i], position), c + i, s + i);
    c[i] *= t.factor, s[i] *= t.factor;
  }
}
// x: the unit's sixteen values, in place.
DEV void unit_turn(bool interleaved, const float *c, const float *s, float *x) {
  // values chosen, not places: a place chosen at run time would put x into memory
  float p[8], q[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float a0 = x[2 * i], a1 = x[i], b0 = x[2 * i + 1], b1 = x[8 + i];
    const float a = interleaved ? a0 : a1, b = interleaved ? b0 : b1;
    p[i] = a * c[i] - b * s[i], q[i] = b * c[i] + a * s[i];
  }
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const float y0 = i % 2 ? q[i / 2] : p[i / 2], y1 = i < 8 ? p[i % 8] : q[i % 8];
    x[i] = interleaved ? y0 : y1;
  }
}
// Sum over the head's U = dim / 16 lanes (4, 8 or 16).
template <int U>
DEV float head_sum(float v) {
  v += ISHZ_DPP(v, 0xB1);
  v += ISHZ_DPP(v, 0x4E);
  if (U >= 8) v += ISHZ_DPP(v, 0x141);
  if (U >= 16) v += ISHZ_DPP(v, 0x140);
  return v;
}
// Norms the unit's sixteen values in place; every lane of the head calls it. w: their weights.
template <int U>
DEV void unit_norm(float *x, const float *w, float eps) {
  float sum = 0;
#pragma unroll
  for (int i = 0; i < 16; i++) sum += x[i] * x[i];
  const float r = 1.0f / sqrtf(head_sum<U>(sum) * (1.0f / (16 * U)) + eps);
#pragma unroll
  for (int i = 0; i < 16; i++) x[i] *= r * w[i];
}

// ---------------------------------------------------------------- attention
struct Call {
  const void *q;
  int64_t row, head;  // strides in values
  void *out;          // [rows][heads][dim]
  int heads, group;   // q heads, and of them to a head of the cache
  float scale;        // of the logits, its magnitude times log2 e
  uint32_t sign;      // and its sign, of two fp16 values
  int causal, window;
  int splits;
  float *part;  // [splits][rows][heads][dim]: sums in units of their own maximum
  float2 *ml;   // [splits][rows][heads]: that maximum (of log2 weights) and the sum of weights
};

// A lane's values of a row of q, as matrix operands: dims 64 e + 16 quad .. + 15 for each e of D / 64; bf16 as fp16 with a
// power of two for the row (see act_prepare), which the returned factor of its logits holds. The scale's sign goes into the
// values (bf16: with that power), so that the factor is never below 0 and a row's largest product is its largest logit.
template <int D, int DT>
DEV float load_query(const Call &c, int64_t row, int head, int quad, h8 *q) {
  constexpr int C = D / 64;
  const size_t at = (size_t)(row * c.row + head * c.head) + 16 * quad;
  u4 v[2 * C];
#pragma unroll
  for (int e = 0; e < 2 * C; e++) v[e] = *(const u4 *)((const uint16_t *)c.q + at + 64 * (e / 2) + 8 * (e % 2));
  float scale = c.scale;
  if (DT == ISHZ_DT_BF16) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 2 * C; e++) m = bf16_absmax(v[e], m);
    const auto a = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = max((uint32_t)a[0], (uint32_t)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    const int x = bf16_row_exponent(max((uint32_t)b[0], (uint32_t)b[1]));
    const float down = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, ldexpf(1.0f, -x)) | (c.sign & 0x80000000u));
#pragma unroll
    for (int e = 0; e < 2 * C; e++) v[e] = bf16_to_half8(v[e], down);
    scale *= ldexpf(1.0f, x);
  }
#pragma unroll
  for (int e = 0; e < 2 * C; e++) q[e] = as_h8(DT == ISHZ_DT_BF16 ? v[e] : v[e] ^ c.sign);
  return scale;
}

// tile_kernel (attn_tile.hip) with 128 row_tiles packed rows to a workgroup (of heads of 256 128), `tiles` workgroups a sequence,
// head and split.
void launch_tile(const Call &c, const Pool &pool, const Rows &rows, int format, int dtype, int row_tiles, int tiles, uint32_t total,
                 hipStream_t st);

// What every call on the cache refuses (attn_cache.hip).
int check_pool(const void *k, const void *v, const float *ks, const float *vs, int format, int blocks, int heads, int dim);
int check_rows(const int32_t *table, const int32_t *lengths, const int32_t *starts, int sequences, int width, int rows);
int check_heads(const void *x, int dtype, int64_t row, int64_t head, const void *out);
}  // namespace attn
