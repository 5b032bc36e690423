// Around attention: per-head norms with the position rotation, and the 8-bit cache's writing and reading.
#include <algorithm>

#include "attn.h"

namespace attn {
// Heads of `rows` token rows: strides in values, the head's own values contiguous.
struct Heads {
  const void *x;
  int64_t row, head;
  int heads;
  const float *weight;  // of the norm, or null
  void *out;            // [rows][heads][dim], or null
};

// A unit's sixteen values as they are loaded.
template <int DT>
struct Raw {
  u4 v[DT == ISHZ_DT_F32 ? 4 : 2];
  DEV void load(const void *x, size_t at, int ca, int cb) {
    constexpr int H = DT == ISHZ_DT_F32 ? 2 : 1, Z = DT == ISHZ_DT_F32 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < H; i++) {
      v[i] = *(const u4 *)((const uint8_t *)x + (at + ca) * Z + 16 * i);
      v[H + i] = *(const u4 *)((const uint8_t *)x + (at + cb) * Z + 16 * i);
    }
  }
  DEV void widen(float *x) const {
    load8<DT>(v, 0, x);
    load8<DT>(v, 8, x + 8);
  }
};

// One wave's share of one row: part of `parts`, 64 / U heads at a time, over q's heads and then k's. Each value is read and
// written once, a unit of 16 a lane with both halves of its pairs in it, so that norm and rotation stay in registers; memory
// bounds it: 4096 rows of 28 heads of 256 in fp16 (117 MB) take 22.8 us, 5.1 TB/s. The next heads' values are on their way
// while these are worked on (24.4 us without that).
template <int DT, int U>
DEV void turn_row(const Heads &q, const Heads &k, const Turn &t, float eps, int row, int part, int parts) {
  constexpr int W = 64 / U;
  const int lane = threadIdx.x & 63, u = lane % U, gq = (q.heads + W - 1) / W, groups = gq + (k.heads + W - 1) / W;
  int ca, cb;
  unit_chunks(u, t.rot, t.interleaved, &ca, &cb);
  const auto load = [&](int g, Raw<DT> &x) {
    const Heads &y = g < gq ? q : k;
    const int h = min((g < gq ? g : g - gq) * W + lane / U, y.heads - 1);
    x.load(y.x, (size_t)(row * y.row + h * y.head), ca, cb);
  };
  if (part >= groups) return;
  Raw<DT> next;
  load(part, next);
  float c[8], s[8], w[16];
  if (u < t.rot / 16) unit_angles(t, u, t.positions[row], c, s);
  int held = -1;  // whose weight w is: 0 q's, 1 k's
  for (int g = part; g < groups; g += parts) {
    float x[16];
    next.widen(x);
    if (g + parts < groups) load(g + parts, next);
    const int whose = g >= gq;
    const Heads &y = whose ? k : q;
    if (whose != held && y.weight) {
#pragma unroll
      for (int i = 0; i < 16; i++) w[i] = y.weight[i < 8 ? ca + i : cb + i - 8];
    }
    held = whose;
    if (y.weight) unit_norm<U>(x, w, eps);
    if (u < t.rot / 16) unit_turn(t.interleaved, c, s, x);
    const int h = (whose ? g - gq : g) * W + lane / U;
    if (h < y.heads) {
      const size_t to = ((size_t)row * y.heads + h) * (16 * U);
      store8<DT>(y.out, to + ca, x);
      store8<DT>(y.out, to + cb, x + 8);
    }
  }
}

template <int DT, int U>
__global__ __launch_bounds__(256) void norm_rope_kernel(Heads q, Heads k, Turn t, float eps, int rows, int waves) {
  const int wave = wave_id(), row = blockIdx.x * (4 / waves) + wave / waves;
  if (row >= rows) return;
  turn_row<DT, U>(q, k, t, eps, row, blockIdx.y * waves + wave % waves, gridDim.y * waves);
}

// ---------------------------------------------------------------- writing
// A code of a block whose scale grew by 2^k.
template <int FMT>
DEV uint32_t regrow4(uint32_t c, float down) {
  const f4 v = decode4f<FMT>(c);
  return encode4<FMT>(v[0] * down, v[1] * down, v[2] * down, v[3] * down);
}

// The block's scale for new tokens of largest magnitude `most` (bits) from slot s0 on, and by which power of two its older
// codes go down. 2^-126 keeps it a normal number; a NaN or an infinity among the tokens makes it NaN, and so what is read
// of this block and head, rather than being dropped. A partly filled block keeps its scale, or grows it by the least power
// of two that holds the new tokens: its old codes are then rounded at most once for each doubling, and all those
// roundings together stay below one step.
template <int FMT>
DEV float next_scale(uint32_t most, int s0, float old, int *grow) {
  const float amax = __builtin_bit_cast(float, most);
  *grow = 0;
  if (most >= 0x7f800000u) return __builtin_nanf("");
  if (s0 == 0) return fmaxf(amax / LIMIT<FMT>, 0x1p-126f);
  const float scale = old < 0x1p-126f ? 0x1p-126f : old, held = LIMIT<FMT> * scale;
  if (!(amax > held)) return scale;
  int ea, eb;
  const float ma = frexpf(amax, &ea), mb = frexpf(held, &eb);
  *grow = ea - eb + (ma > mb);
  return ldexpf(scale, *grow);
}

// A workgroup per (sequence, block that its new rows reach, head, keys or values) owns that block's codes and scale, so
// the scale is the exact maximum over its new tokens without a second pass or atomics: the tokens stay in registers
// meanwhile. Of keys a thread has units of a token (the norm and the rotation go over the head); of values 4 tokens of 8
// dims, which are whole words of the block's rows of tokens: nothing is turned in LDS. Workgroups past those turn q's
// heads, `waves` waves a row. 8192 tokens of 8 heads of 128 in fp16 (50 MB) take 14.0 us, 3.6 TB/s, of which a launch and
// the waits, one after the other (lengths and table, values, the workgroup's maximum), are 5: one token of each of 16
// sequences takes 6.2.
template <int DT, int U, int FMT>
__global__ __launch_bounds__(256) void append_kernel(Heads k, Heads v, Heads q, Turn t, float eps, Pool pool, Rows rows,
                                                     int reach, int writers, int waves) {
  constexpr int D = 16 * U, N = U / 4, G = U <= 8 ? 1 : 2;
  __shared__ uint32_t scratch[4];
  const int tid = threadIdx.x;
  if ((int)blockIdx.x >= writers) {
    const int wave = wave_id(), row = (blockIdx.x - writers) * (4 / waves) + wave / waves;
    if (row < rows.rows) turn_row<DT, U>(q, Heads{}, t, eps, row, wave % waves, waves);
    return;
  }
  int id = blockIdx.x;
  const int head = id % pool.heads;
  id /= pool.heads;
  const bool values = id & 1;
  id >>= 1;
  const int j = id % reach, seq = id / reach;
  const int row0 = rows.first(seq), n = rows.count(seq), length = rows.length(seq), start = length - n;
  if (n == 0) return;
  const int jb = max(start, 0) / BLOCK + j;
  if (jb >= rows.width) return;  // past the table; below 2^31 tokens from here on
  const int lo = max(max(start, 0), jb * BLOCK), hi = min(length, jb * BLOCK + BLOCK);
  if (lo >= hi) return;
  const int block = rows.block(seq, jb, pool.blocks);
  if (block < 0) return;
  const int s0 = lo - jb * BLOCK, s1 = hi - jb * BLOCK, row_of = row0 + jb * BLOCK - start;  // of slot 0
  float *const scale_at = (values ? pool.vs : pool.ks) + pool.scale(block, head);
  const float old = *scale_at;
  uint8_t *const tile = (values ? pool.v : pool.k) + pool.tile(block, head);
  uint32_t most = 0;
  const auto larger = [&](float x) { most = max(most, __builtin_bit_cast(uint32_t, x) & 0x7fffffffu); };

  if (!values) {
    const int u = tid % U;
    int ca, cb;
    unit_chunks(u, t.rot, t.interleaved, &ca, &cb);
    float x[N][16], w[16];
    if (k.weight) {
#pragma unroll
      for (int i = 0; i < 16; i++) w[i] = k.weight[i < 8 ? ca + i : cb + i - 8];
    }
    Raw<DT> raw[N];
#pragma unroll
    for (int m = 0; m < N; m++)  // slots past the last read the last one's token again: whole heads take part in a norm
      raw[m].load(k.x, (size_t)((int64_t)(row_of + min(s0 + (tid + 256 * m) / U, s1 - 1)) * k.row + head * k.head), ca, cb);
    unrolled<N>([&](auto m) __attribute__((always_inline)) {
      if (256 * m / U >= s1 - s0) return;  // the same for the whole workgroup
      raw[m].widen(x[m]);
      if (k.weight) unit_norm<U>(x[m], w, eps);
      if (u < t.rot / 16) {
        float c[8], s[8];
        unit_angles(t, u, t.positions[row_of + min(s0 + (tid + 256 * m) / U, s1 - 1)], c, s);
        unit_turn(t.interleaved, c, s, x[m]);
      }
#pragma unroll
      for (int i = 0; i < 16; i++) larger(x[m][i]);
    });
    int grow;
    const float scale = next_scale<FMT>(block_absmax(most, scratch), s0, old, &grow), up = 1.0f / scale;
    if (tid == 0) *scale_at = scale;
#pragma unroll
    for (int m = 0; m < N; m++) {
      const int slot = s0 + (tid + 256 * m) / U;
      if (slot >= s1) continue;
      uint32_t code[4];
#pragma unroll
      for (int i = 0; i < 4; i++)
        code[i] = scale != scale ? 0 : encode4<FMT>(quotient(x[m][4 * i], scale, up), quotient(x[m][4 * i + 1], scale, up),
                                                    quotient(x[m][4 * i + 2], scale, up), quotient(x[m][4 * i + 3], scale, up));
      *(u2 *)(tile + slot * D + ca) = u2{code[0], code[1]};
      *(u2 *)(tile + slot * D + cb) = u2{code[2], code[3]};
    }
    if (grow > 0) {
      const float down = ldexpf(1.0f, -grow);
      for (int i = tid; i < s0 * D / 16; i += 256) {
        u4 o = *(u4 *)(tile + 16 * i);
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = regrow4<FMT>(o[e], down);
        *(u4 *)(tile + 16 * i) = o;
      }
    }
    return;
  }

  const int first = 4 * (tid % 16), dims = 8 * (tid / 16);  // this thread's slots and dims (of each 128)
  const bool mine = dims < D;
  float x[G][4][8];
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int slot = first + i;
      if (mine && slot >= s0 && slot < s1)
        load8<DT>(v.x, (size_t)((int64_t)(row_of + slot) * v.row + head * v.head) + dims + 128 * g, x[g][i]);
      else
#pragma unroll
        for (int e = 0; e < 8; e++) x[g][i][e] = 0;
    }
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) larger(x[g][i][e]);
  int grow;
  const float scale = next_scale<FMT>(block_absmax(most, scratch), s0, old, &grow), up = 1.0f / scale, down = ldexpf(1.0f, -grow);
  if (tid == 0) *scale_at = scale;
  // words that hold none of the new tokens are left alone, or lose steps where the scale grew
  if (!mine || first >= s1 || (first + 4 <= s0 && grow <= 0)) return;
  uint32_t fresh = 0;  // the bytes of new tokens
#pragma unroll
  for (int i = 0; i < 4; i++) fresh |= first + i >= s0 && first + i < s1 ? 255u << 8 * i : 0;
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      uint32_t *const at = (uint32_t *)(tile + (dims + 128 * g + e) * BLOCK + first);
      uint32_t code = scale != scale ? 0 : encode4<FMT>(quotient(x[g][0][e], scale, up), quotient(x[g][1][e], scale, up),
                                                        quotient(x[g][2][e], scale, up), quotient(x[g][3][e], scale, up));
      if (fresh != ~0u) {
        const uint32_t was = *at;
        // tokens past s1 in a word are none of the sequence's: what is made of them does not matter, but they stay
        uint32_t past = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) past |= first + i >= s1 ? 255u << 8 * i : 0;
        const uint32_t kept = grow > 0 ? (regrow4<FMT>(was, down) & ~past) | (was & past) : was;
        code = (code & fresh) | (kept & ~fresh);
      }
      *at = code;
    }
}

// ---------------------------------------------------------------- reading
// A workgroup per (sequence, block that holds some of its last `tail` tokens, head, keys or values). A thread has 8 dims of a
// token of keys at a time, 4 tokens of 8 dims of values: loads of words of the block's rows, stores of 16 bytes. What is
// written is seldom read soon: past the caches 55259 tokens of 8 heads of 128 take 79 us (4.8 TB/s, as fast as a large
// copy), through them 85.
template <int DT, int D, int FMT>
__global__ __launch_bounds__(256) void read_kernel(Pool pool, Rows rows, int tail, int reach, void *k_out, void *v_out) {
  constexpr int PER = D / 8, G = D == 256 ? 2 : 1;
  const int tid = threadIdx.x;
  int id = blockIdx.x;
  const int head = id % pool.heads;
  id /= pool.heads;
  const bool values = id & 1;
  id >>= 1;
  const int j = id % reach, seq = id / reach;
  const int p0 = rows.length(seq) - tail, to0 = j * BLOCK - (p0 & (BLOCK - 1));  // slot 0's place in the output
  const int s0 = max(-to0, 0), s1 = min(tail - to0, BLOCK);
  if (s0 >= s1) return;
  const int block = rows.block(seq, (p0 >> 6) + j, pool.blocks);
  const float scale = block < 0 ? 0.0f : (values ? pool.vs : pool.ks)[pool.scale(block, head)];
  const uint8_t *const tile = (values ? pool.v : pool.k) + pool.tile(max(block, 0), head);
  // of slot 0 and dim 0
  const int64_t at = (((int64_t)seq * tail + to0) * pool.heads + head) * D;
  const int64_t step = (int64_t)pool.heads * D;
  if (!values) {
    const int d = 8 * (tid % PER);
    u2 c[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; i++) {
      const int slot = tid / PER + i * (256 / PER);
      c[i] = block >= 0 && slot >= s0 && slot < s1 ? *(const u2 *)(tile + slot * D + d) : u2{0, 0};
    }
#pragma unroll
    for (int i = 0; i < D / 32; i++) {
      const int slot = tid / PER + i * (256 / PER);
      if (slot < s0 || slot >= s1) continue;
      const f4 a = decode4f<FMT>(c[i].x) * scale, b = decode4f<FMT>(c[i].y) * scale;
      const float o[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      store8<DT, true>(k_out, (size_t)(at + slot * step + d), o);
    }
    return;
  }
#pragma unroll
  for (int g = 0; g < G; g++) {
    const int d = 8 * (tid % PER), first = 4 * (tid / PER) + 32 * g;
    if (first >= BLOCK) return;
    uint32_t c[8];
#pragma unroll
    for (int e = 0; e < 8; e++) c[e] = block >= 0 ? *(const uint32_t *)(tile + (d + e) * BLOCK + first) : 0;
    f4 x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = decode4f<FMT>(c[e]) * scale;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int slot = first + i;
      if (slot < s0 || slot >= s1) continue;
      const float o[8] = {x[0][i], x[1][i], x[2][i], x[3][i], x[4][i], x[5][i], x[6][i], x[7][i]};
      store8<DT, true>(v_out, (size_t)(at + slot * step + d), o);
    }
  }
}

// ---------------------------------------------------------------- host side
// What every call on the cache refuses; 0 rows or sequences are no fault.
int check_pool(const void *k, const void *v, const float *ks, const float *vs, int format, int blocks, int heads, int dim) {
  if (format != ISHZ_KV_INT8 && format != ISHZ_KV_E4M3) return ishz::decline("the cache holds int8 or e4m3 codes");
  if (dim != 64 && dim != 128 && dim != 256) return ishz::decline("heads of 64, 128 or 256 values");
  if (blocks < 1 || heads < 1) return ishz::einval("a cache of no blocks or heads");
  if (!k || !v || !ks || !vs) return ishz::einval("null cache");
  if (((uintptr_t)k | (uintptr_t)v) & 15) return ishz::einval("cache codes must be 16-byte aligned");
  if (((uintptr_t)ks | (uintptr_t)vs) & 3) return ishz::einval("cache scales must be 4-byte aligned");
  return ISHZ_OK;
}
int check_rows(const int32_t *table, const int32_t *lengths, const int32_t *starts, int sequences, int width, int rows) {
  if (sequences < 0 || width < 0 || rows < 0) return ishz::einval("a negative count");
  if (sequences > 0 && (!lengths || !starts || (width > 0 && !table))) return ishz::einval("null table, lengths or starts");
  if (width > INT32_MAX / BLOCK) return ishz::decline("a table wider than 2^31 tokens");
  return ISHZ_OK;
}
int check_heads(const void *x, int dtype, int64_t row, int64_t head, const void *out) {
  if (!x) return ishz::einval("null activations");
  const int64_t step = dtype == ISHZ_DT_F32 ? 4 : 8;
  if (((uintptr_t)x & 15) || ((uintptr_t)out & 15) || row % step || head % step)
    return ishz::decline("rows and heads that do not start on 16 bytes");
  return ISHZ_OK;
}
int check_turn(const int32_t *positions, const uint64_t *turns, int rot, int dim, int rows) {
  if (rot < 0 || rot > dim || rot % 16) return ishz::decline("a rotation of a multiple of 16 values of the head");
  if (rot && rows && (!positions || !turns)) return ishz::einval("a rotation needs positions and turns");
  return ISHZ_OK;
}
}  // namespace attn

using namespace attn;

#define ISHZ_BY_DTYPE(dt, ...)                                    \
  switch (dt) {                                                   \
    case ISHZ_DT_F32: { constexpr int DT = ISHZ_DT_F32; __VA_ARGS__; } break;   \
    case ISHZ_DT_F16: { constexpr int DT = ISHZ_DT_F16; __VA_ARGS__; } break;   \
    default: { constexpr int DT = ISHZ_DT_BF16; __VA_ARGS__; } break;           \
  }
#define ISHZ_BY_DIM(dim, ...)                          \
  switch (dim) {                                       \
    case 64: { constexpr int U = 4; __VA_ARGS__; } break;   \
    case 128: { constexpr int U = 8; __VA_ARGS__; } break;  \
    default: { constexpr int U = 16; __VA_ARGS__; } break;  \
  }
#define ISHZ_BY_FORMAT(f, ...)                                             \
  if (f == ISHZ_KV_INT8) { constexpr int FMT = ISHZ_KV_INT8; __VA_ARGS__; } \
  else { constexpr int FMT = ISHZ_KV_E4M3; __VA_ARGS__; }

extern "C" int ishz_norm_rope(const void *q, int64_t q_row, int64_t q_head, int q_heads, const void *k, int64_t k_row,
                              int64_t k_head, int k_heads, int dtype, int rows, int dim, const int32_t *positions,
                              const uint64_t *turns, int rot, int interleaved, float factor, const float *q_weight,
                              const float *k_weight, float eps, void *q_out, void *k_out, ishz_stream_t stream) {
  if (dtype != ISHZ_DT_F32 && dtype != ISHZ_DT_F16 && dtype != ISHZ_DT_BF16) return ishz::decline("activations of fp32, fp16 or bf16");
  if (dim != 64 && dim != 128 && dim != 256) return ishz::decline("heads of 64, 128 or 256 values");
  if (rows < 0 || q_heads < 0 || k_heads < 0) return ishz::einval("a negative count");
  if (int rc = check_turn(positions, turns, rot, dim, rows)) return rc;
  const int64_t total = (int64_t)q_heads + k_heads;
  if (rows == 0 || total == 0) return ISHZ_OK;
  if (q_heads) {
    if (!q_out) return ishz::einval("null output");
    if (int rc = check_heads(q, dtype, q_row, q_head, q_out)) return rc;
  }
  if (k_heads) {
    if (!k_out) return ishz::einval("null output");
    if (int rc = check_heads(k, dtype, k_row, k_head, k_out)) return rc;
  }
  const Heads gq = {q, q_row, q_head, q_heads, q_weight, q_out}, gk = {k, k_row, k_head, k_heads, k_weight, k_out};
  const Turn t = {positions, turns, rot, interleaved, factor};
  const int per = 64 / (dim / 16);
  const int64_t groups = (total + per - 1) / per;
  // Rows that fill the chip with a wave each take one (its angles serve all its heads); fewer are spread over waves.
  const int waves = rows >= 2048 ? 1 : 4;
  const int64_t across = ((int64_t)rows + 4 / waves - 1) / (4 / waves);
  if (across > (1 << 24) - 1 || total > INT32_MAX - 64) return ishz::decline("more rows or heads than a launch holds");
  const dim3 grid((uint32_t)across, waves == 1 ? 1 : (uint32_t)std::min<int64_t>((groups + 3) / 4, UINT16_MAX));
  ISHZ_BY_DTYPE(dtype, ISHZ_BY_DIM(dim, hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_rope_kernel<DT, U>), grid, dim3(256), 0,
                                                           ishz::S(stream), gq, gk, t, eps, rows, waves)));
  ISHZ_LAUNCH_CHECK("norm and rotation launch");
  return ISHZ_OK;
}

extern "C" int ishz_kv_append(const void *k, int64_t k_row, int64_t k_head, const void *v, int64_t v_row, int64_t v_head,
                              int dtype, int rows, void *k_codes, void *v_codes, float *k_scale, float *v_scale, int format,
                              int blocks, int heads, int dim, const int32_t *table, int width, const int32_t *lengths,
                              const int32_t *starts, int sequences, int max_rows, const void *q, int64_t q_row,
                              int64_t q_head, int q_heads, const int32_t *positions, const uint64_t *turns, int rot,
                              int interleaved, float factor, const float *q_weight, const float *k_weight, float eps,
                              void *q_out, ishz_stream_t stream) {
  if (dtype != ISHZ_DT_F32 && dtype != ISHZ_DT_F16 && dtype != ISHZ_DT_BF16) return ishz::decline("activations of fp32, fp16 or bf16");
  if (int rc = check_pool(k_codes, v_codes, k_scale, v_scale, format, blocks, heads, dim)) return rc;
  if (int rc = check_rows(table, lengths, starts, sequences, width, rows)) return rc;
  if (int rc = check_turn(positions, turns, rot, dim, rows)) return rc;
  if (max_rows < 0 || q_heads < 0) return ishz::einval("a negative count");
  if (rows == 0) return ISHZ_OK;
  if (int rc = check_heads(k, dtype, k_row, k_head, nullptr)) return rc;
  if (int rc = check_heads(v, dtype, v_row, v_head, nullptr)) return rc;
  if (q_heads) {
    if (!q_out) return ishz::einval("null output");
    if (int rc = check_heads(q, dtype, q_row, q_head, q_out)) return rc;
  }
  // max_rows rows that start anywhere in a block reach this many.
  max_rows = std::min(max_rows, rows);
  const int64_t reach = max_rows > 0 ? ((int64_t)max_rows + BLOCK - 2) / BLOCK + 1 : 0;
  const int64_t writers = sequences * reach * 2 * heads, waves = rows >= 2048 ? 1 : 4;  // as for ishz_norm_rope
  const int64_t turners = q_heads ? (rows + 4 / waves - 1) / (4 / waves) : 0;
  if (writers + turners > (1 << 24) - 1) return ishz::decline("more blocks than a launch holds");
  if (writers + turners == 0) return ISHZ_OK;
  const Heads gk = {k, k_row, k_head, heads, k_weight, nullptr}, gv = {v, v_row, v_head, heads, nullptr, nullptr};
  const Heads gq = {q, q_row, q_head, q_heads, q_weight, q_out};
  const Turn t = {positions, turns, rot, interleaved, factor};
  const Pool pool = {(uint8_t *)k_codes, (uint8_t *)v_codes, k_scale, v_scale, blocks, heads, dim};
  const Rows r = {table, lengths, starts, sequences, width, rows};
  ISHZ_BY_FORMAT(format, ISHZ_BY_DTYPE(dtype, ISHZ_BY_DIM(dim, hipLaunchKernelGGL(
      HIP_KERNEL_NAME(append_kernel<DT, U, FMT>), dim3((uint32_t)(writers + turners)), dim3(256), 0, ishz::S(stream), gk, gv, gq,
      t, eps, pool, r, (int)reach, (int)writers, (int)waves))));
  ISHZ_LAUNCH_CHECK("cache append launch");
  return ISHZ_OK;
}

extern "C" int ishz_kv_read(const void *k_codes, const void *v_codes, const float *k_scale, const float *v_scale, int format,
                            int blocks, int heads, int dim, const int32_t *table, int width, const int32_t *lengths,
                            int sequences, int tail, int dtype, void *k_out, void *v_out, ishz_stream_t stream) {
  if (dtype != ISHZ_DT_F32 && dtype != ISHZ_DT_F16 && dtype != ISHZ_DT_BF16) return ishz::decline("outputs of fp32, fp16 or bf16");
  if (int rc = check_pool(k_codes, v_codes, k_scale, v_scale, format, blocks, heads, dim)) return rc;
  if (int rc = check_rows(table, lengths, lengths, sequences, width, 0)) return rc;
  if (tail < 0) return ishz::einval("a negative count");
  if (sequences == 0 || tail == 0) return ISHZ_OK;
  if (!k_out || !v_out || (((uintptr_t)k_out | (uintptr_t)v_out) & 15)) return ishz::einval("outputs must be 16-byte aligned");
  const int64_t reach = ((int64_t)tail + BLOCK - 2) / BLOCK + 1, total = (int64_t)sequences * reach * 2 * heads;
  if (total > (1 << 24) - 1) return ishz::decline("more blocks than a launch holds");
  const Pool pool = {(uint8_t *)k_codes, (uint8_t *)v_codes, (float *)k_scale, (float *)v_scale, blocks, heads, dim};
  const Rows r = {table, lengths, nullptr, sequences, width, 0};
  ISHZ_BY_FORMAT(format, ISHZ_BY_DTYPE(dtype, ISHZ_BY_DIM(dim, hipLaunchKernelGGL(
      HIP_KERNEL_NAME(read_kernel<DT, 16 * U, FMT>), dim3((uint32_t)total), dim3(256), 0, ishz::S(stream), pool, r, tail, (int)reach,
      k_out, v_out))));
  ISHZ_LAUNCH_CHECK("cache read launch");
  return ISHZ_OK;
}
