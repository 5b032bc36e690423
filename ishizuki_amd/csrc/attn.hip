// Attention over the 8-bit cache.
#include <algorithm>

#include "attn.h"

namespace attn {
// ---------------------------------------------------------------- few rows: the cache streams past them
// The rows of a sequence and its q heads of one cache head are packed, 16 to a tile. A wave takes 64 tokens (one
// block) at a time, from memory straight into matrix operands:
//   S^T [64 tokens x 16 rows] = K Q^T: the operand's row r of tile t is token 16 (r / 4) + 4 t + r % 4, so that a lane
//   ends up with the weights of the 16 consecutive tokens 16 (lane / 16).. of row lane % 16;
//   O^T [dim x 16 rows] += V^T P^T: those 16 weights are two operands as they are, against 16 consecutive bytes of V^T.
// Neither codes nor weights pass through LDS, and each is read from memory once. The four waves of a workgroup take
// every fourth block and are joined in LDS; splits of a long cache are joined by join_kernel.
template <int D, int FMT, int DT, int RT>
__global__ __launch_bounds__(256) void stream_kernel(Call c, Pool pool, Rows rows, int tiles) {
  constexpr int C = D / 64, V = D / 16, PITCH = D + 4;
  __shared__ float joined[4 * 16 * PITCH];
  __shared__ float wave_m[4][16], wave_l[4][16];
  int id = blockIdx.x;
  const int kvh = id % pool.heads;
  id /= pool.heads;
  const int split = id % c.splits;
  id /= c.splits;
  const int tile = id % tiles, seq = id / tiles;
  const int row0 = rows.first(seq), n = rows.count(seq), length = rows.length(seq), base = length - n;
  const int packed = n * c.group, r0 = tile * (16 * RT);
  if (r0 >= packed) return;
  const int wave = wave_id(), lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;

  // the rows, and the tokens that each sees: begin[] .. end[] - 1
  h8 q[RT][2 * C];
  float scale[RT];
  int begin[RT], end[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int r = min(r0 + 16 * t + col, packed - 1), i = r / c.group;
    end[t] = c.causal ? base + i + 1 : length;
    begin[t] = c.window ? max(base + i + 1 - c.window, 0) : 0;
    scale[t] = load_query<D, DT>(c, row0 + i, kvh * c.group + r % c.group, quad, q[t]);
  }

  // blocks that some row sees; those that every row sees whole need no mask
  const int i0 = r0 / c.group, i1 = (min(r0 + 16 * RT, packed) - 1) / c.group;
  const int last = c.causal ? base + i1 + 1 : length, from = c.window ? max(base + i0 + 1 - c.window, 0) : 0;
  const int whole0 = c.window ? max(base + i1 + 1 - c.window, 0) : 0, whole1 = c.causal ? base + i0 + 1 : length;
  const int b0 = from / BLOCK, b1 = max((last + BLOCK - 1) / BLOCK, b0);
  const int each = (b1 - b0 + c.splits - 1) / c.splits;
  const int first = b0 + split * each, stop = min(first + each, b1);

  f4 o[RT][V];
  float m[RT], l[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    m[t] = -__builtin_inff(), l[t] = 0;
#pragma unroll
    for (int d = 0; d < V; d++) o[t][d] = f4{0, 0, 0, 0};
  }
  for (int b = first + wave; b < stop; b += 4) {
    const int block = __builtin_amdgcn_readfirstlane(rows.block(seq, b, pool.blocks));
    if (block < 0) continue;
    const uint8_t *const kt = pool.k + pool.tile(block, kvh), *const vt = pool.v + pool.tile(block, kvh);
    const float ks = pool.ks[pool.scale(block, kvh)], vs = pool.vs[pool.scale(block, kvh)];
    u4 kc[4][C], vc[V];
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
      for (int e = 0; e < C; e++)
        kc[t][e] = *(const u4 *)(kt + (16 * (col >> 2) + 4 * t + (col & 3)) * D + 64 * e + 16 * quad);
#pragma unroll
    for (int d = 0; d < V; d++) vc[d] = *(const u4 *)(vt + (16 * d + col) * BLOCK + 16 * quad);

    const int p0 = b * BLOCK, mine = p0 + 16 * quad;
    const bool whole = p0 >= whole0 && p0 + BLOCK <= whole1;
    h8 p[RT][2];
    float alpha[RT], vf[RT];
    f4 s[RT][4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
#pragma unroll
      for (int r = 0; r < RT; r++) s[r][t] = f4{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < C; e++) {
        const h8 a = decode8<FMT>(kc[t][e].x, kc[t][e].y), a2 = decode8<FMT>(kc[t][e].z, kc[t][e].w);
#pragma unroll
        for (int r = 0; r < RT; r++) s[r][t] = mfma32(a2, q[r][2 * e + 1], mfma32(a, q[r][2 * e], s[r][t]));
      }
    }
#pragma unroll
    for (int r = 0; r < RT; r++) {
      const float f = scale[r] * ks;
      vf[r] = vs;
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[r][t][i] *= f;
      if (!whole) {
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int at = mine + 4 * t + i;
            s[r][t][i] = at >= begin[r] && at < end[r] ? s[r][t][i] : -__builtin_inff();
          }
        // a row that sees none of the block takes nothing of it, whatever its scale is
        if (end[r] <= p0 || begin[r] >= p0 + BLOCK) vf[r] = 0;
      }
      float top = m[r];
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) top = fmaxf(top, s[r][t][i]);
      top = fmaxf(top, lane_xor16(top));
      top = fmaxf(top, lane_xor32(top));
      const float ref = top == -__builtin_inff() ? 0.0f : top;  // nothing seen so far: weights of 0, not of NaN
      alpha[r] = __builtin_amdgcn_exp2f(m[r] - ref);
      m[r] = top;
      float sum = 0;
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float w = __builtin_amdgcn_exp2f(s[r][t][i] - ref);
          sum += w;
          // Weights are rounded to fp16 for the matrix units: 2^-12 of each, the sums below stay in 32 bits.
          p[r][t / 2][4 * (t % 2) + i] = (_Float16)w;
        }
      l[r] = l[r] * alpha[r] + sum;
    }
    // past the sequence's end a block holds whatever was there: an e4m3 NaN times a weight of 0 must not count
    if (FMT == ISHZ_KV_E4M3 && p0 + BLOCK > length) {
#pragma unroll
      for (int d = 0; d < V; d++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int left = length - (mine + 4 * e);
          vc[d][e] &= left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << 8 * left) - 1;
        }
    }
#pragma unroll
    for (int d = 0; d < V; d++) {
      const h8 a = decode8<FMT>(vc[d].x, vc[d].y), a2 = decode8<FMT>(vc[d].z, vc[d].w);
#pragma unroll
      for (int r = 0; r < RT; r++) {
        const f4 x = mfma32(a2, p[r][1], mfma32(a, p[r][0], f4{0, 0, 0, 0}));
#pragma unroll
        for (int i = 0; i < 4; i++) o[r][d][i] = o[r][d][i] * alpha[r] + x[i] * vf[r];
      }
    }
  }

#pragma unroll
  for (int t = 0; t < RT; t++) {
    float sum = l[t];
    sum += lane_xor16(sum);
    sum += lane_xor32(sum);
    if (t) __syncthreads();
    if (quad == 0) wave_m[wave][col] = m[t], wave_l[wave][col] = sum;
#pragma unroll
    for (int d = 0; d < V; d++) *(f4 *)(joined + (wave * 16 + col) * PITCH + 16 * d + 4 * quad) = o[t][d];
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * (D / 8); x += 256) {
      const int rr = x / (D / 8), d = x % (D / 8) * 8, r = r0 + 16 * t + rr;
      if (r >= packed) continue;
      const float top = fmaxf(fmaxf(wave_m[0][rr], wave_m[1][rr]), fmaxf(wave_m[2][rr], wave_m[3][rr]));
      const float ref = top == -__builtin_inff() ? 0.0f : top;
      float acc[8] = {}, all = 0;
#pragma unroll
      for (int w = 0; w < 4; w++) {
        const float f = __builtin_amdgcn_exp2f(wave_m[w][rr] - ref);
        all += f * wave_l[w][rr];
        const f4 a = *(const f4 *)(joined + (w * 16 + rr) * PITCH + d), a2 = *(const f4 *)(joined + (w * 16 + rr) * PITCH + d + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] += f * a[i], acc[4 + i] += f * a2[i];
      }
      const size_t at = (size_t)(row0 + r / c.group) * c.heads + kvh * c.group + r % c.group;
      if (c.splits == 1) {
        const float inv = all == 0 ? 0.0f : 1.0f / all;
#pragma unroll
        for (int i = 0; i < 8; i++) acc[i] *= inv;
        store8<DT>(c.out, at * D + d, acc);
      } else {
        const size_t to = (size_t)split * rows.rows * c.heads + at;
        store8<ISHZ_DT_F32>(c.part, to * D + d, acc);
        if (d == 0) c.ml[to] = float2{top, all};
      }
    }
  }
}

// Joins the splits of a row and head: D / 8 lanes each.
template <int D, int DT>
__global__ __launch_bounds__(256) void join_kernel(Call c, const int32_t *starts, int sequences, int rows) {
  const size_t at = (size_t)blockIdx.x * (256 / (D / 8)) + threadIdx.x / (D / 8);
  const size_t total = (size_t)rows * c.heads;
  const int64_t row = at / c.heads;
  if (row >= rows || row < starts[0] || row >= starts[sequences]) return;
  const int d = threadIdx.x % (D / 8) * 8;
  float top = -__builtin_inff();
  for (int s = 0; s < c.splits; s++) top = fmaxf(top, c.ml[s * total + at].x);
  const float ref = top == -__builtin_inff() ? 0.0f : top;
  float acc[8] = {}, all = 0;
  for (int s = 0; s < c.splits; s++) {
    const float2 ml = c.ml[s * total + at];
    const float f = __builtin_amdgcn_exp2f(ml.x - ref);
    all += f * ml.y;
    float x[8];
    load8<ISHZ_DT_F32>(c.part, (s * total + at) * D + d, x);
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] += f * x[i];
  }
  const float inv = all == 0 ? 0.0f : 1.0f / all;
#pragma unroll
  for (int i = 0; i < 8; i++) acc[i] *= inv;
  store8<DT>(c.out, at * D + d, acc);
}

// How a call is divided: packed rows to a workgroup, and splits of the cache.
struct Plan {
  int row_tiles, tiles, splits;  // row_tiles 0: tile_kernel
};
static Plan plan(int q_heads, int heads, int dim, int sequences, int max_rows, int max_length) {
  Plan p;
  const int64_t packed = (int64_t)max_rows * (q_heads / heads);
  p.row_tiles = packed <= 16 ? 1 : packed <= 32 ? 2 : 0;
  const int per = p.row_tiles ? 16 * p.row_tiles : tile_rows(dim);
  p.tiles = (int)((packed + per - 1) / per);
  const int64_t groups = (int64_t)sequences * heads * p.tiles;
  const int64_t blocks = ((int64_t)max_length + BLOCK - 1) / BLOCK;
  const int64_t want = p.row_tiles ? 1024 : 512;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({(want + groups - 1) / std::max<int64_t>(groups, 1), (blocks + 3) / 4, 64}));
  if (!p.row_tiles && groups * 2 > want) p.splits = 1;
  return p;
}
}  // namespace attn

using namespace attn;

extern "C" size_t ishz_kv_attend_workspace_size(int rows, int q_heads, int heads, int dim, int sequences, int max_rows,
                                                int max_length) {
  if (rows < 1 || heads < 1 || q_heads < heads || sequences < 1 || max_rows < 1 || max_length < 1) return 0;
  const Plan p = plan(q_heads, heads, dim, sequences, std::min(max_rows, rows), max_length);
  return p.splits == 1 ? 0 : (size_t)p.splits * rows * q_heads * (dim + 2) * 4;
}

extern "C" int ishz_kv_attend(const void *q, int64_t q_row, int64_t q_head, int q_heads, int dtype, int rows,
                              const void *k_codes, const void *v_codes, const float *k_scale, const float *v_scale,
                              int format, int blocks, int heads, int dim, const int32_t *table, int width,
                              const int32_t *lengths, const int32_t *starts, int sequences, int max_rows, int max_length,
                              float scale, int causal, int window, void *out, void *workspace, size_t workspace_bytes,
                              ishz_stream_t stream) {
  if (dtype != ISHZ_DT_F16 && dtype != ISHZ_DT_BF16) return ishz::decline("queries of fp16 or bf16");
  if (int rc = check_pool(k_codes, v_codes, k_scale, v_scale, format, blocks, heads, dim)) return rc;
  if (int rc = check_rows(table, lengths, starts, sequences, width, rows)) return rc;
  if (max_rows < 0 || max_length < 0 || window < 0) return ishz::einval("a negative count");
  if (window && !causal) return ishz::einval("a window is of a causal call");
  if (q_heads < 1 || q_heads % heads) return ishz::einval("query heads must be a multiple of the cache's");
  if (rows == 0 || sequences == 0 || max_rows == 0) return ISHZ_OK;
  if (!out) return ishz::einval("null output");
  if (int rc = check_heads(q, dtype, q_row, q_head, out)) return rc;
  max_rows = std::min(max_rows, rows);
  const int group = q_heads / heads;
  if ((int64_t)max_rows * group > INT32_MAX - 64) return ishz::decline("more rows than a launch holds");
  const Plan p = plan(q_heads, heads, dim, sequences, max_rows, max_length);
  const size_t need = p.splits == 1 ? 0 : (size_t)p.splits * rows * q_heads * (dim + 2) * 4;
  if (workspace_bytes < need || (need && (!workspace || ((uintptr_t)workspace & 15)))) return ishz::einval("workspace too small");
  const int64_t total = (int64_t)sequences * heads * p.tiles * p.splits, joins = ((int64_t)rows * q_heads + 256 / (dim / 8) - 1) / (256 / (dim / 8));
  if (total > (1 << 24) - 1 || joins > (1 << 24) - 1) return ishz::decline("more rows than a launch holds");
  float *const part = (float *)workspace;
  const Call c = {q, q_row, q_head, out, q_heads, group, scale * 1.44269504088896341f, causal, window, p.splits, part,
                  (float2 *)(part + (need ? (size_t)p.splits * rows * q_heads * dim : 0))};
  const Pool pool = {(uint8_t *)k_codes, (uint8_t *)v_codes, (float *)k_scale, (float *)v_scale, blocks, heads, dim};
  const Rows r = {table, lengths, starts, sequences, width, rows};
#define ISHZ_STREAM(D, F, T, RT)                                                                                         \
  hipLaunchKernelGGL(HIP_KERNEL_NAME(stream_kernel<D, F, T, RT>), dim3((uint32_t)total), dim3(256), 0, ishz::S(stream), c, pool, r, \
                     p.tiles)
#define ISHZ_STREAM_RT(D, F, T) if (p.row_tiles == 1) ISHZ_STREAM(D, F, T, 1); else ISHZ_STREAM(D, F, T, 2)
#define ISHZ_STREAM_D(F, T)                          \
  if (dim == 64) { ISHZ_STREAM_RT(64, F, T); }       \
  else if (dim == 128) { ISHZ_STREAM_RT(128, F, T); } \
  else { ISHZ_STREAM_RT(256, F, T); }
  if (!p.row_tiles) launch_tile(c, pool, r, format, dtype, p.tiles, (uint32_t)total, ishz::S(stream));
  else if (format == ISHZ_KV_INT8) {
    if (dtype == ISHZ_DT_F16) { ISHZ_STREAM_D(ISHZ_KV_INT8, ISHZ_DT_F16); } else { ISHZ_STREAM_D(ISHZ_KV_INT8, ISHZ_DT_BF16); }
  } else {
    if (dtype == ISHZ_DT_F16) { ISHZ_STREAM_D(ISHZ_KV_E4M3, ISHZ_DT_F16); } else { ISHZ_STREAM_D(ISHZ_KV_E4M3, ISHZ_DT_BF16); }
  }
  ISHZ_LAUNCH_CHECK("attention launch");
  if (p.splits > 1) {
#define ISHZ_JOIN(D, T) hipLaunchKernelGGL(HIP_KERNEL_NAME(join_kernel<D, T>), dim3((uint32_t)joins), dim3(256), 0, ishz::S(stream), c, starts, sequences, rows)
#define ISHZ_JOIN_D(T) if (dim == 64) ISHZ_JOIN(64, T); else if (dim == 128) ISHZ_JOIN(128, T); else ISHZ_JOIN(256, T)
    if (dtype == ISHZ_DT_F16) { ISHZ_JOIN_D(ISHZ_DT_F16); } else { ISHZ_JOIN_D(ISHZ_DT_BF16); }
    ISHZ_LAUNCH_CHECK("attention join launch");
  }
  return ISHZ_OK;
}
