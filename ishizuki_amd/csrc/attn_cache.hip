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

// Loads unit u of head h of a row, normed and turned. c, s: the unit's angles (u < rot / 16).
template <int DT, int U>
DEV void load_unit(const Heads &g, const Turn &t, float eps, int row, int h, int u, const float *c, const float *s, float *x) {
  int ca, cb;
  unit_chunks(u, t.rot, t.interleaved, &ca, &cb);
  const size_t at = (size_t)(row * g.row + h * g.head);
  load8<DT>(g.x, at + ca, x);
  load8<DT>(g.x, at + cb, x + 8);
  if (g.weight) unit_norm<U>(x, g.weight, ca, cb, eps);
  if (u < t.rot / 16) unit_turn(t.interleaved, c, s, x);
}

// One wave's share of one row: part of `parts`, 64 / U heads at a time, over q's heads and then k's.
template <int DT, int U>
DEV void turn_row(const Heads &q, const Heads &k, const Turn &t, float eps, int row, int part, int parts) {
  constexpr int W = 64 / U;
  const int lane = threadIdx.x & 63, u = lane % U, total = q.heads + k.heads;
  float c[8], s[8];
  if (u < t.rot / 16) unit_angles(t, u, t.positions[row], c, s);
  int ca, cb;
  unit_chunks(u, t.rot, t.interleaved, &ca, &cb);
  for (int h0 = part * W; h0 < total; h0 += parts * W) {
    const int h = h0 + lane / U, hc = min(h, total - 1);
    const bool first = hc < q.heads;
    const Heads &g = first ? q : k;
    const int hh = first ? hc : hc - q.heads;
    float x[16];
    load_unit<DT, U>(g, t, eps, row, hh, u, c, s, x);
    if (h < total) {
      const size_t to = ((size_t)row * g.heads + hh) * (16 * U);
      store8<DT>(g.out, to + ca, x);
      store8<DT>(g.out, to + cb, x + 8);
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

// A workgroup per (sequence, block that its new rows reach, head, keys or values) owns that block's codes and
// scale, so the scale is the exact maximum over its new tokens without a second pass or atomics; workgroups past
// those turn q's heads, four rows each.
template <int DT, int U, int FMT>
__global__ __launch_bounds__(256) void append_kernel(Heads k, Heads v, Heads q, Turn t, float eps, Pool pool, Rows rows,
                                                     int reach, int writers) {
  constexpr int D = 16 * U, N = U / 4, PITCH = BLOCK + 16;
  __shared__ uint32_t scratch[4];
  __shared__ __attribute__((aligned(16))) uint8_t turned[D * PITCH];
  if ((int)blockIdx.x >= writers) {
    const int row = (blockIdx.x - writers) * 4 + wave_id();
    if (row < rows.rows) turn_row<DT, U>(q, Heads{}, t, eps, row, 0, 1);
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
  const int lo = max(max(start, 0), jb * BLOCK), hi = min(length, jb * BLOCK + BLOCK);
  if (lo >= hi) return;
  const int block = rows.block(seq, jb, pool.blocks);
  if (block < 0) return;
  const int s0 = lo - jb * BLOCK, s1 = hi - jb * BLOCK;
  const Heads &g = values ? v : k;
  const Turn none = {nullptr, nullptr, 0, 0, 1.0f};
  const Turn &turn = values ? none : t;

  float x[N][16];
  uint32_t most = 0;
#pragma unroll
  for (int m = 0; m < N; m++) {
    if (256 * m / U >= s1 - s0) break;
    const int unit = threadIdx.x + 256 * m, u = unit % U;
    const int row = row0 + lo - start + min(unit / U, s1 - s0 - 1);
    float c[8], s[8];
    if (u < turn.rot / 16) unit_angles(turn, u, turn.positions[row], c, s);
    load_unit<DT, U>(g, turn, eps, row, head, u, c, s, x[m]);
#pragma unroll
    for (int i = 0; i < 16; i++) most = max(most, __builtin_bit_cast(uint32_t, x[m][i]) & 0x7fffffffu);
  }
  float *const scale_at = (values ? pool.vs : pool.ks) + pool.scale(block, head);
  const float old = *scale_at;
  most = block_absmax(most, scratch);

  // The block's scale. 2^-126 keeps it a normal number; a NaN or an infinity among the tokens makes it NaN, and so
  // what is read of this block and head, rather than being dropped.
  const float amax = __builtin_bit_cast(float, most);
  float scale, down = 1.0f;
  int grow = 0;
  if (most >= 0x7f800000u) {
    scale = __builtin_nanf("");
  } else if (s0 == 0) {
    scale = fmaxf(amax / LIMIT<FMT>, 0x1p-126f);
  } else {
    // A partly filled block keeps its scale, or grows it by the least power of two that holds the new tokens: its old
    // codes are then rounded at most once for each doubling, and all those roundings together stay below one step.
    scale = old < 0x1p-126f ? 0x1p-126f : old;
    const float held = LIMIT<FMT> * scale;
    if (amax > held) {
      int ea, eb;
      const float ma = frexpf(amax, &ea), mb = frexpf(held, &eb);
      grow = ea - eb + (ma > mb);
      scale = ldexpf(scale, grow);
      down = ldexpf(1.0f, -grow);
    }
  }
  if (threadIdx.x == 0) *scale_at = scale;
  const float up = scale == scale ? 1.0f / scale : 0.0f;
  const bool dead = scale != scale;

  uint8_t *const tile = (values ? pool.v : pool.k) + pool.tile(block, head);
#pragma unroll
  for (int m = 0; m < N; m++) {
    const int unit = threadIdx.x + 256 * m, u = unit % U, slot = s0 + unit / U;
    if (slot >= s1) continue;
    int ca, cb;
    unit_chunks(u, turn.rot, turn.interleaved, &ca, &cb);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
      w[i] = dead ? 0 : encode4<FMT>(x[m][4 * i] * up, x[m][4 * i + 1] * up, x[m][4 * i + 2] * up, x[m][4 * i + 3] * up);
    if (!values) {
      *(u2 *)(tile + slot * D + ca) = u2{w[0], w[1]};
      *(u2 *)(tile + slot * D + cb) = u2{w[2], w[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++) turned[((i < 8 ? ca + i : cb + i - 8)) * PITCH + slot] = (uint8_t)(w[i / 4] >> 8 * (i % 4));
    }
  }
  if (!values) {
    if (grow > 0)
      for (int i = threadIdx.x; i < s0 * D / 16; i += 256) {
        u4 o = *(u4 *)(tile + 16 * i);
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = regrow4<FMT>(o[e], down);
        *(u4 *)(tile + 16 * i) = o;
      }
    return;
  }
  __syncthreads();
  if (s0 == 0 && s1 == BLOCK) {
    for (int i = threadIdx.x; i < D * 4; i += 256)
      *(u4 *)(tile + 16 * i) = *(const u4 *)(turned + i / 4 * PITCH + 16 * (i % 4));
    return;
  }
  // Four tokens of a value at a time, from the first that changes.
  const int w0 = grow > 0 ? 0 : s0 / 4, words = (s1 + 3) / 4 - w0;
  for (int i = threadIdx.x; i < D * words; i += 256) {
    const int d = i / words, w = w0 + i % words;
    uint32_t *const at = (uint32_t *)(tile + d * BLOCK + 4 * w);
    const uint32_t fresh = *(const uint32_t *)(turned + d * PITCH + 4 * w);
    if (4 * w >= s0 && 4 * w + 4 <= s1) {
      *at = fresh;
      continue;
    }
    const uint32_t was = *at, kept = grow > 0 ? regrow4<FMT>(was, down) : was;
    uint32_t o = 0;
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const int slot = 4 * w + b;
      o |= (slot < s0 ? kept : slot < s1 ? fresh : was) & (255u << 8 * b);
    }
    *at = o;
  }
}

// ---------------------------------------------------------------- reading
// A workgroup per (sequence, block that holds some of its last `tail` tokens, head, keys or values).
template <int DT, int FMT>
__global__ __launch_bounds__(256) void read_kernel(Pool pool, Rows rows, int tail, int reach, void *k_out, void *v_out) {
  __shared__ __attribute__((aligned(16))) uint8_t turned[BLOCK * (256 + 16)];
  const int D = pool.dim, pitch = D + 16;
  int id = blockIdx.x;
  const int head = id % pool.heads;
  id /= pool.heads;
  const bool values = id & 1;
  id >>= 1;
  const int j = id % reach, seq = id / reach;
  const int length = rows.length(seq), p0 = length - tail, jb = (p0 >> 6) + j;
  const int lo = max(p0, jb * BLOCK), hi = min(length, jb * BLOCK + BLOCK);
  if (lo >= hi) return;
  const int block = rows.block(seq, jb, pool.blocks);
  const float scale = block < 0 ? 0.0f : (values ? pool.vs : pool.ks)[pool.scale(block, head)];
  const uint8_t *const tile = (values ? pool.v : pool.k) + pool.tile(max(block, 0), head);
  if (values && block >= 0) {
    for (int i = threadIdx.x; i < D * 4; i += 256) {
      const u4 c = *(const u4 *)(tile + 16 * i);
#pragma unroll
      for (int e = 0; e < 16; e++) turned[(16 * (i % 4) + e) * pitch + i / 4] = (uint8_t)(c[e / 4] >> 8 * (e % 4));
    }
    __syncthreads();
  }
  void *const out = values ? v_out : k_out;
  const int per = D / 8;
  for (int i = threadIdx.x; i < (hi - lo) * per; i += 256) {
    const int p = lo + i / per, slot = p - jb * BLOCK, d = i % per * 8;
    float o[8] = {};
    if (block >= 0) {
      const u2 c = values ? *(const u2 *)(turned + slot * pitch + d) : *(const u2 *)(tile + slot * D + d);
      const f4 a = decode4f<FMT>(c.x), b = decode4f<FMT>(c.y);
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] = a[e] * scale, o[4 + e] = b[e] * scale;
    }
    store8<DT>(out, (((size_t)seq * tail + (p - p0)) * pool.heads + head) * D + d, o);
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
  const int total = q_heads + k_heads;
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
  const int per = 64 / (dim / 16), groups = (total + per - 1) / per;
  // Rows that fill the chip with a wave each take one (its angles serve all its heads); fewer are spread over waves.
  const int waves = rows >= 2048 ? 1 : 4;
  const dim3 grid((rows + 4 / waves - 1) / (4 / waves), waves == 1 ? 1 : (groups + 3) / 4);
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
  const int reach = max_rows > 0 ? (max_rows + BLOCK - 2) / BLOCK + 1 : 0;
  const int64_t writers = (int64_t)sequences * reach * 2 * heads, turners = q_heads ? (rows + 3) / 4 : 0;
  if (writers + turners > (1 << 24) - 1) return ishz::decline("more blocks than a launch holds");
  if (writers + turners == 0) return ISHZ_OK;
  const Heads gk = {k, k_row, k_head, heads, k_weight, nullptr}, gv = {v, v_row, v_head, heads, nullptr, nullptr};
  const Heads gq = {q, q_row, q_head, q_heads, q_weight, q_out};
  const Turn t = {positions, turns, rot, interleaved, factor};
  const Pool pool = {(uint8_t *)k_codes, (uint8_t *)v_codes, k_scale, v_scale, blocks, heads, dim};
  const Rows r = {table, lengths, starts, sequences, width, rows};
  ISHZ_BY_FORMAT(format, ISHZ_BY_DTYPE(dtype, ISHZ_BY_DIM(dim, hipLaunchKernelGGL(
      HIP_KERNEL_NAME(append_kernel<DT, U, FMT>), dim3((uint32_t)(writers + turners)), dim3(256), 0, ishz::S(stream), gk, gv, gq,
      t, eps, pool, r, reach, (int)writers))));
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
  ISHZ_BY_FORMAT(format, ISHZ_BY_DTYPE(dtype, hipLaunchKernelGGL(HIP_KERNEL_NAME(read_kernel<DT, FMT>), dim3((uint32_t)total),
                                                                 dim3(256), 0, ishz::S(stream), pool, r, tail, (int)reach,
                                                                 k_out, v_out)));
  ISHZ_LAUNCH_CHECK("cache read launch");
  return ISHZ_OK;
}
