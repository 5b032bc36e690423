// Attention over the 8-bit cache.
#include <algorithm>
#include <cmath>

#include "attn.h"

namespace attn {
// ---------------------------------------------------------------- few rows: the cache streams past them
// The rows of a sequence and its q heads of one cache head are packed, 16 to a tile. A wave takes 64 tokens (one
// block) at a time, from memory straight into matrix operands:
//   S^T [64 tokens x 16 rows] = K Q^T: the operand's row r of tile t is token 16 (r / 4) + 4 t + r % 4, so that a lane
//   ends up with the weights of the 16 consecutive tokens 16 (lane / 16).. of row lane % 16;
//   O^T [dim x 16 rows] += V^T P^T: those 16 weights are two operands as they are, against 16 consecutive bytes of V^T.
// Neither codes nor weights pass through LDS, and each is read from memory once. The W waves of a workgroup take every
// W-th block and are joined in LDS; splits of a long cache are joined by join_kernel.
// Memory bounds it over long caches: 16 sequences of 12000 to 32768 tokens of 8 heads of 128 (731 MB) take 131 us and the
// join 4.8, 5.5 TB/s, where a kernel that only reads reaches 6.1. Vector operations are 35 % and matrix ones 7 % of the
// SIMDs' time. One token over 777 takes 9 to 10 us: a launch, three dependent reads (table, codes and scales) and the joining.
template <int D, int FMT, int DT, int RT, int W>
__global__ __launch_bounds__(64 * W) void stream_kernel(Call c, Pool pool, Rows rows, int tiles) {
  constexpr int C = D / 64, V = D / 16, PITCH = D + 4;
  extern __shared__ __attribute__((aligned(16))) float joined[];  // [W][16][PITCH]
  __shared__ float wave_m[W][16], wave_l[W][16];
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

  // blocks that some row sees; those that every row sees whole need no mask
  const int i0 = r0 / c.group, i1 = (min(r0 + 16 * RT, packed) - 1) / c.group;
  const int last = min(c.causal ? base + i1 + 1 : length, rows.held(seq)), from = c.window ? max(base + i0 + 1 - c.window, 0) : 0;
  const int whole0 = c.window ? max(base + i1 + 1 - c.window, 0) : 0, whole1 = c.causal ? base + i0 + 1 : length;
  const int b0 = from / BLOCK, b1 = max((last + BLOCK - 1) / BLOCK, b0);
  const int each = (b1 - b0 + c.splits - 1) / c.splits;
  const int first = b0 + split * each, stop = min(first + each, b1);

  int next = first + wave < stop ? rows.block(seq, first + wave, pool.blocks) : -1;
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

  f4 o[RT][V];
  float m[RT], l[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    m[t] = -__builtin_inff(), l[t] = 0;
#pragma unroll
    for (int d = 0; d < V; d++) o[t][d] = f4{0, 0, 0, 0};
  }
  for (int b = first + wave; b < stop; b += W) {
    const int block = __builtin_amdgcn_readfirstlane(next);
    next = b + W < stop ? rows.block(seq, b + W, pool.blocks) : -1;
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
          // Weights are rounded to fp16 for the matrix units: 2^-11 of each at most, the sums below stay in 32 bits.
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
    for (int x = threadIdx.x; x < 16 * (D / 8); x += 64 * W) {
      const int rr = x / (D / 8), d = x % (D / 8) * 8, r = r0 + 16 * t + rr;
      if (r >= packed) continue;
      float top = wave_m[0][rr];
#pragma unroll
      for (int w = 1; w < W; w++) top = fmaxf(top, wave_m[w][rr]);
      const float ref = top == -__builtin_inff() ? 0.0f : top;
      float acc[8] = {}, all = 0;
#pragma unroll
      for (int w = 0; w < W; w++) {
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

// Joins the splits of a row and head, a wave: lane s has split s's maximum and sum (64 splits at most), then each lane
// D / 64 of the values of all splits, eight of them on their way at a time.
template <int D, int DT>
__global__ __launch_bounds__(256) void join_kernel(Call c, const int32_t *starts, int sequences, int rows) {
  constexpr int N = D / 64;
  typedef float fn __attribute__((ext_vector_type(N)));
  const int lane = threadIdx.x & 63;
  const size_t at = (size_t)blockIdx.x * 4 + wave_id(), total = (size_t)rows * c.heads;
  const int64_t row = at / c.heads;
  if (row >= rows || row < starts[0] || row >= starts[sequences]) return;
  const float2 ml = lane < c.splits ? c.ml[lane * total + at] : float2{-__builtin_inff(), 0.0f};
  float top = ml.x;
  top = fmaxf(top, ISHZ_DPP(top, 0xB1));
  top = fmaxf(top, ISHZ_DPP(top, 0x4E));
  top = fmaxf(top, ISHZ_DPP(top, 0x141));
  top = fmaxf(top, ISHZ_DPP(top, 0x140));
  top = fmaxf(top, lane_xor16(top));
  top = fmaxf(top, lane_xor32(top));
  const float f = __builtin_amdgcn_exp2f(ml.x - (top == -__builtin_inff() ? 0.0f : top));
  const float all = group_sum<64>(f * ml.y);
  const float *const part = c.part + at * D + lane * N;
  float acc[N] = {};
  for (int s0 = 0; s0 < c.splits; s0 += 8) {
    fn x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = *(const fn *)(part + min(s0 + i, c.splits - 1) * total * D);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float by = s0 + i < c.splits ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), s0 + i)) : 0.0f;
#pragma unroll
      for (int e = 0; e < N; e++) acc[e] += by * x[i][e];
    }
  }
  const float inv = all == 0 ? 0.0f : 1.0f / all;
#pragma unroll
  for (int e = 0; e < N; e++) acc[e] *= inv;
  uint16_t *const out = (uint16_t *)c.out + at * D + lane * N;
  if constexpr (N == 1) *out = (uint16_t)narrow2<DT>(acc[0], 0.0f);
  else if constexpr (N == 2) *(uint32_t *)out = narrow2<DT>(acc[0], acc[1]);
  else *(u2 *)out = u2{narrow2<DT>(acc[0], acc[1]), narrow2<DT>(acc[2], acc[3])};
}

// How a call is divided: packed rows to a workgroup, and splits of the cache.
struct Plan {
  bool stream;  // stream_kernel, or tile_kernel
  int row_tiles, tiles, splits, waves;
};
static Plan plan(int q_heads, int heads, int dim, int sequences, int max_rows, int max_length, int window) {
  Plan p;
  const int64_t packed = (int64_t)max_rows * (q_heads / heads), blocks = ((int64_t)max_length + BLOCK - 1) / BLOCK;
  const int64_t pairs = std::max<int64_t>((int64_t)sequences * heads, 1);
  // Blocks that a workgroup's rows see: a window of 1000 over 32768 tokens is one row's 17 (9.0 us, 11.2 divided as 512).
  const int64_t span = window ? std::min(blocks, ((int64_t)window + std::min(max_rows, 256) + 62) / BLOCK + 1) : blocks;
  const auto tiles = [&](int per) { return (packed + per - 1) / per; };
  // Sixteen packed rows or fewer stream; of heads of 256, whose codes take most of the registers, only while a wave has
  // but a few blocks (64 blocks of 2 heads: 11.9 us, tiles 13.3; 256 of 32: 82 and 61). Up to 32 rows do of heads of 128
  // (four sequences of 8191 tokens, 8 heads: 23.8 us, tiles 31.8; of 64 21.3 and 18.5, of 256 38 and 24.5).
  p.stream = packed <= 16 ? dim < 256 || pairs * span < 1024 : packed <= 32 && dim == 128;
  p.waves = 4;
  int64_t splits;
  if (p.stream) {
    p.row_tiles = packed <= 16 ? 1 : 2;
    p.tiles = (int)tiles(16 * p.row_tiles);
    if (p.row_tiles == 1 && dim < 256 && span > 4 && span <= 16) {
      p.waves = 8;  // two blocks a wave and one launch (13 blocks: 9.6 us; four waves, four splits and their join: 10.1)
      splits = 1;
    } else {
      // Four workgroups a CU, and at most 32 blocks a wave's share of four, so that long sequences beside short ones end
      // sooner (16 sequences of 12000 to 32768 tokens, 8 heads: 138 us, 141 without; 60000 of one: 32.5). No more than 64
      // splits (below), so that fewer than 16 sequences and heads together fill less: one of one head a quarter of the CUs.
      splits = std::min(std::max((1024 + pairs - 1) / pairs, span / 32), (span + 3) / 4);
    }
  } else {
    // 256 rows a workgroup halve the decoding: for many of heads of 128 (4096 tokens of 32 heads over 8: 150 us, 128 rows
    // 185; of 64 114 and 118), or few rows over a long cache (512 over 16384: 148 and 158; of 64 108 and 134), of which they
    // see enough (700 rows of 32 heads over 8 in a window of 4500, 76 blocks: 90 and 98; of 64 69 and 74; of 3000, 52 blocks,
    // no difference; 3 x 1500 of 16 over 2 of 64 in one of 4096, 70 blocks: 195 and 153). Otherwise 128 rows end more evenly
    // (2048 tokens: 59 us, 72; of 64 42 and 53).
    const bool wide = packed > 128 && ((dim == 128 && pairs * tiles(256) >= 512) ||
                                       (dim < 256 && blocks >= 128 && span >= 72 && max_length >= 4 * (int64_t)max_rows));
    p.row_tiles = wide ? 2 : 1;
    p.tiles = (int)tiles(128 * p.row_tiles);
    // A workgroup a CU, two where a sequence's rows are one tile and the parts to join few (4 x 8 tokens over 8191 of 32
    // heads over 8 of 64: 18.5 us, 20.8 with one; 4 x 32 of 128 in a window of 4096: 26.8, two 31.5), and three blocks each
    // (16 tokens over 1500: 12.2 us, six 14.9). Where rows see nine blocks or fewer on average the join costs more than
    // that gives (16 tokens over 700: 12.9, unsplit 16.1; over 512 in two splits no gain; 700 among themselves 24 and 20).
    const int64_t mean = std::min(span, ((int64_t)max_length - max_rows / 2 + BLOCK - 1) / BLOCK);
    splits = 256 / std::max<int64_t>(pairs * p.tiles, 1);
    if (splits > 1 && splits <= 8 && dim < 256 && packed * dim <= 8192) splits *= 2;
    splits = mean < 9 ? 1 : std::min(splits, span / 3);
  }
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(splits, 64));  // a lane of join_kernel each
  // the workspace's size knows no window
  if (window) p.splits = std::min(p.splits, plan(q_heads, heads, dim, sequences, max_rows, max_length, 0).splits);
  return p;
}
}  // namespace attn

using namespace attn;

extern "C" size_t ishz_kv_attend_workspace_size(int rows, int q_heads, int heads, int dim, int sequences, int max_rows,
                                                int max_length) {
  if (rows < 1 || heads < 1 || q_heads < heads || sequences < 1 || max_rows < 1 || max_length < 1) return 0;
  const Plan p = plan(q_heads, heads, dim, sequences, std::min(max_rows, rows), max_length, 0);
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
  const Plan p = plan(q_heads, heads, dim, sequences, max_rows, max_length, window);
  const size_t need = p.splits == 1 ? 0 : (size_t)p.splits * rows * q_heads * (dim + 2) * 4;
  if (workspace_bytes < need || (need && (!workspace || ((uintptr_t)workspace & 15)))) return ishz::einval("workspace too small");
  const int64_t total = (int64_t)sequences * heads * p.tiles * p.splits, joins = ((int64_t)rows * q_heads + 3) / 4;
  // a launch holds fewer than 2^32 threads
  if (total * (p.stream ? 64 * p.waves : 512) > UINT32_MAX || joins > (1 << 24) - 1) return ishz::decline("more rows than a launch holds");
  float *const part = (float *)workspace;
  const Call c = {q, q_row, q_head, out, q_heads, group, std::fabs(scale) * 1.44269504088896341f,
                  std::signbit(scale) ? 0x80008000u : 0u, causal, window, p.splits, part,
                  (float2 *)(part + (need ? (size_t)p.splits * rows * q_heads * dim : 0))};
  const Pool pool = {(uint8_t *)k_codes, (uint8_t *)v_codes, (float *)k_scale, (float *)v_scale, blocks, heads, dim};
  const Rows r = {table, lengths, starts, sequences, width, rows};
#define ISHZ_STREAM(D, F, T, RT, W)                                                                                      \
  hipLaunchKernelGGL(HIP_KERNEL_NAME(stream_kernel<D, F, T, RT, W>), dim3((uint32_t)total), dim3(64 * W),                 \
                     W * 16 * (D + 4) * 4, ishz::S(stream), c, pool, r, p.tiles)
#define ISHZ_STREAM_D(F, T)                                            \
  if (dim == 64 && p.waves == 8) ISHZ_STREAM(64, F, T, 1, 8);          \
  else if (dim == 64) ISHZ_STREAM(64, F, T, 1, 4);                     \
  else if (dim == 256) ISHZ_STREAM(256, F, T, 1, 4);                   \
  else if (p.waves == 8) ISHZ_STREAM(128, F, T, 1, 8);                 \
  else if (p.row_tiles == 1) ISHZ_STREAM(128, F, T, 1, 4);             \
  else ISHZ_STREAM(128, F, T, 2, 4)
  if (!p.stream) launch_tile(c, pool, r, format, dtype, p.row_tiles, p.tiles, (uint32_t)total, ishz::S(stream));
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
