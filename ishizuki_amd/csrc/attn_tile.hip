// Attention over the 8-bit cache for many rows: prompts, drafted tokens of wide groups, cross attention.
#include "attn.h"

namespace attn {
// Eight waves of 16 RT packed rows (a sequence's rows and its q heads of one cache head) pass the cache's blocks together.
// Each block is decoded to fp16 once for all of them, into LDS in the order in which the matrix operands are read (a
// wave's 64 lanes read 1 KB in a row: 255 bytes a clock measured, rows of 272 bytes 128), two blocks deep: while one is
// worked on, the next one's codes are on their way in registers. As in stream_kernel S^T = K Q^T leaves a lane the
// weights of 16 consecutive tokens of a row, which are the operands of O^T += V^T P^T as they are.
//
// A row's sums stay in the units of a reference that is only moved when a logit passes it by 2^8 (weights stay below
// fp16's largest), and of a value scale `unit` that the scales of the blocks it sees are 1..255 of: log2 of that ratio is
// added to the block's logits, so that nothing but the matrix units touches the sums. A block outside 1..255 moves the
// unit, which stays above 2^-72 of the largest scale the row has seen (the sums' 2^45 then stay finite).
//
// Issue bounds it: 8192 tokens of 32 heads over 8 of 128, causal, take 526 to 546 us call after call (1010 to 1050 TFLOP/s),
// 4530 cycles a block of 256 rows at 2.35 GHz. Matrix units are busy for 42 % of the cycles and vector operations for 45 %
// (an exp2 takes two ordinary ones' cycles), in turn and hardly at once. By itself a call runs at 1.95 GHz and takes 620.
// The products alone, from registers, run at 1970 TFLOP/s on such values (1700 as 32x32x16), a library product of
// 8192 x 8192 x 8192 at 1250 to 1500. The time is within 4 % for 16 to 48 rows a wave, products of either shape, vector
// operations dealt between the products or not, and codes unpacked by a pass before.
template <int D, int FMT, int DT, int RT>
__global__ __launch_bounds__(512, RT == 1 && D <= 128 ? 4 : 2) void tile_kernel(Call c, Pool pool, Rows rows, int tiles) {
  constexpr int C = D / 64, V = D / 16;
  extern __shared__ h8 held[];  // [2][16 C operands][64]
  int id = blockIdx.x;
  const int kvh = id % pool.heads;
  id /= pool.heads;
  const int split = id % c.splits;
  id /= c.splits;
  // the last rows of a causal call see most and start first
  const int tile = tiles - 1 - id / rows.sequences, seq = id % rows.sequences;
  const int row0 = rows.first(seq), n = rows.count(seq), length = rows.length(seq), base = length - n;
  const int packed = n * c.group, r0 = tile * 128 * RT;
  if (r0 >= packed) return;
  const int wave = wave_id(), lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const int w0 = r0 + wave * (16 * RT);

  h8 q[RT][2 * C];
  float scale[RT];
  int end[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int r = min(w0 + 16 * t + col, packed - 1), i = r / c.group;
    end[t] = c.causal ? base + i + 1 : length;
    scale[t] = load_query<D, DT>(c, row0 + i, kvh * c.group + r % c.group, quad, q[t]);
  }
  const int window = c.window ? c.window : INT32_MAX;  // a row sees tokens end - window .. end - 1

  // blocks that some row of the workgroup sees, and the tokens that some, or all, of the wave's rows do
  const int i0 = r0 / c.group, i1 = (min(r0 + 128 * RT, packed) - 1) / c.group;
  const int last = min(c.causal ? base + i1 + 1 : length, rows.held(seq)), from = c.window ? max(base + i0 + 1 - c.window, 0) : 0;
  const int b0 = from / BLOCK, b1 = max((last + BLOCK - 1) / BLOCK, b0);
  const int each = (b1 - b0 + c.splits - 1) / c.splits;
  const int first = b0 + split * each, stop = min(first + each, b1);
  const int j0 = w0 / c.group, j1 = (min(w0 + 16 * RT, packed) - 1) / c.group;
  const int some0 = c.window ? max(base + j0 + 1 - c.window, 0) : 0;
  const int some1 = w0 >= packed ? 0 : c.causal ? base + j1 + 1 : length;
  const int whole0 = c.window ? max(base + j1 + 1 - c.window, 0) : 0, whole1 = c.causal ? base + j0 + 1 : length;

  // The operands of a block, 1 KB each: 8 C of K (tile t of the tokens, dims), then 8 C of V (dims, tokens). Waves 0..3
  // decode K's, 4..7 V's.
  u4 raw[C];
  const int part = wave & 3;
  const bool is_v = wave >> 2;
  const uint32_t from_at = is_v ? (16 * C * part + col) * BLOCK + 16 * quad : (16 * (col >> 2) + 4 * part + (col & 3)) * D + 16 * quad;
  const auto fetch = [&](int block) {
    const uint8_t *const x = (is_v ? pool.v : pool.k) + pool.tile(block, kvh) + from_at;
#pragma unroll
    for (int i = 0; i < C; i++) raw[i] = *(const u4 *)(x + (is_v ? 16 * BLOCK : 64) * i);
  };
  const auto put = [&](int b) {
    h8 *const to = held + ((b - first) & 1) * (16 * C * 64) + wave * (2 * C * 64) + lane;
    // past the sequence's end a block holds whatever was there: an e4m3 NaN times a weight of 0 must not count
    if (FMT == ISHZ_KV_E4M3 && is_v && b * BLOCK + BLOCK > length) {
#pragma unroll
      for (int i = 0; i < C; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int left = length - (b * BLOCK + 16 * quad + 4 * e);
          raw[i][e] &= left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << 8 * left) - 1;
        }
    }
#pragma unroll
    for (int i = 0; i < C; i++) {
      to[i * 128] = decode8<FMT>(raw[i].x, raw[i].y);
      to[i * 128 + 64] = decode8<FMT>(raw[i].z, raw[i].w);
    }
  };

  f4 o[RT][V];
  float m[RT], l[RT], unit[RT], inv[RT], largest[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    m[t] = -3e38f, l[t] = 0, unit[t] = 0x1p-100f, inv[t] = 0x1p100f, largest[t] = 0;
#pragma unroll
    for (int d = 0; d < V; d++) o[t][d] = f4{0, 0, 0, 0};
  }
  // The numbers and scales of 64 blocks from `from_b` on, a lane each: read one by one where they are needed, they would be
  // two dependent loads' latency in every step.
  int ids = -1, from_b = first;
  float kss = 0, vss = 0;
  const auto refill = [&](int b) {
    from_b = b;
    ids = b + lane < stop ? rows.block(seq, b + lane, pool.blocks) : -1;
  };
  const auto refill_scales = [&]() {
    const size_t x = pool.scale(max(ids, 0), kvh);
    const float v = pool.vs[x], none = v - v;
    // a value scale of no number makes the logits none, of the rows that see the block
    kss = ids < 0 ? 0.0f : pool.ks[x] + none;
    vss = ids < 0 || none != 0 ? -1.0f : fmaxf(v, 0x1p-126f);
  };
  const auto lane_value = [&](float v, int b) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), b - from_b));
  };
  const auto block_at = [&](int b) { return __builtin_amdgcn_readlane(ids, b - from_b); };
  refill(first);
  int block = first < stop ? block_at(first) : -1;
  if (block >= 0) fetch(block);
  refill_scales();
  if (block >= 0) put(first);
  __syncthreads();
  // Blocks b .. stop - 1; `apart`: what each brings is added in 32 bits. Without, a wave returns at the first block that needs
  // that, with its work on it still to be done.
  const auto pass = [&](auto apart, int b) {
    for (; b < stop; b++) {
      if (b - from_b > 62) refill(b), refill_scales();
      const int next = block_at(b + 1);
      if (next >= 0) fetch(next);
      const int p0 = b * BLOCK;
      if (block >= 0 && p0 < some1 && p0 + BLOCK > some0) {
        const float ks = lane_value(kss, b), vb = lane_value(vss, b);
        const h8 *const at = held + ((b - first) & 1) * (16 * C * 64) + lane;
        h8 a = at[0], a2 = at[64];
        f4 s[RT][4];
#pragma unroll
        for (int x = 0; x < 4 * C; x++) {
          const h8 y = at[(2 * x + 2) * 64], y2 = at[(2 * x + 3) * 64];
          __builtin_amdgcn_sched_barrier(0);
          const int t = x / C;
#pragma unroll
          for (int r = 0; r < RT; r++) s[r][t] = mfma32(a, q[r][2 * (x % C)], x % C ? s[r][t] : f4{0, 0, 0, 0});
#pragma unroll
          for (int r = 0; r < RT; r++) s[r][t] = mfma32(a2, q[r][2 * (x % C) + 1], s[r][t]);
          a = y, a2 = y2;
          __builtin_amdgcn_sched_barrier(0);
        }
        float f[RT], ratio[RT];
#pragma unroll
        for (int r = 0; r < RT; r++) f[r] = scale[r] * ks, ratio[r] = vb < 0 ? 1.0f : vb * inv[r];
        if (p0 < whole0 || p0 + BLOCK > whole1) {
#pragma unroll
          for (int r = 0; r < RT; r++) {
            const int before = end[r] - 1 - (p0 + 16 * quad);  // tokens between the lane's first and the row's last
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
              for (int i = 0; i < 4; i++)
                s[r][t][i] = before >= 4 * t + i && before - (4 * t + i) < window ? s[r][t][i] * f[r] : -__builtin_inff();
            f[r] = 1;
            if (end[r] <= p0 || end[r] - p0 >= (int64_t)window + BLOCK) ratio[r] = 1;  // sees none of the block
          }
        }
        float top[RT];
        bool move = false;
#pragma unroll
        for (int r = 0; r < RT; r++) {
          float x = s[r][0][0];
#pragma unroll
          for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) x = fmaxf(x, s[r][t][i]);
          top[r] = x * f[r];
          move |= top[r] > m[r] + 8.0f || ratio[r] > 255.0f || (ratio[r] < 1.0f && vb > 0x1p-120f);  // all zeros: moves nothing
        }
        bool below = false;
        if (__any(move)) {
#pragma unroll
          for (int r = 0; r < RT; r++) {
            float x = fmaxf(top[r], m[r]);
            x = fmaxf(x, lane_xor16(x));
            x = fmaxf(x, lane_xor32(x));
            float alpha = __builtin_amdgcn_exp2f(m[r] - x);
            m[r] = x;
            l[r] *= alpha;
            if (ratio[r] > 255.0f || (ratio[r] < 1.0f && vb > 0x1p-120f)) {
              largest[r] = fmaxf(fmaxf(largest[r], 256.0f * unit[r]), vb);
              const float to = fmaxf(fmaxf(vb * 0x1p-4f, 0x1p-72f * largest[r]), 0x1p-100f);
              alpha *= unit[r] / to;
              unit[r] = to, inv[r] = 1.0f / to, ratio[r] = vb * inv[r];
              below |= ratio[r] < 1.0f;
            }
#pragma unroll
            for (int d = 0; d < V; d++) {  // one after another: the compiler holds all of them twice otherwise
              f4 y = o[r][d] * alpha;
              asm volatile("" : "+v"(y));
              o[r][d] = y;
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        }
        if (!apart && __any(below)) return b;
        h8 p[RT][2];
#pragma unroll
        for (int r = 0; r < RT; r++) {
          const float part_of = apart ? 1.0f : fmaxf(ratio[r], 0x1p-64f), ref = __builtin_amdgcn_logf(part_of) - m[r];
          float sum = 0;
#pragma unroll
          for (int t = 0; t < 4; t++) {
            typedef float f2 __attribute__((ext_vector_type(2)));
            const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][t][0], f[r], ref));
            const float w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][t][1], f[r], ref));
            const float w2 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][t][2], f[r], ref));
            const float w3 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][t][3], f[r], ref));
            sum += (w0 + w1) + (w2 + w3);
            // Weights are rounded to fp16 for the matrix units: 2^-11 of each at most, the sums stay in 32 bits.
            const h2 lo = __builtin_convertvector((f2{w0, w1}), h2), hi = __builtin_convertvector((f2{w2, w3}), h2);
            p[r][t / 2][4 * (t % 2)] = lo.x, p[r][t / 2][4 * (t % 2) + 1] = lo.y;
            p[r][t / 2][4 * (t % 2) + 2] = hi.x, p[r][t / 2][4 * (t % 2) + 3] = hi.y;
          }
          l[r] += sum * __builtin_amdgcn_rcpf(part_of);
        }
#pragma unroll
        for (int d = 0; d < V; d++) {
          h8 y = a, y2 = a2;
          if (d + 1 < V) y = at[(8 * C + 2 * d + 2) * 64], y2 = at[(8 * C + 2 * d + 3) * 64];
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (apart) {
#pragma unroll
            for (int r = 0; r < RT; r++) o[r][d] += mfma32(a2, p[r][1], mfma32(a, p[r][0], f4{0, 0, 0, 0})) * ratio[r];
          } else {
#pragma unroll
            for (int r = 0; r < RT; r++) o[r][d] = mfma32(a, p[r][0], o[r][d]);
#pragma unroll
            for (int r = 0; r < RT; r++) o[r][d] = mfma32(a2, p[r][1], o[r][d]);
          }
          a = y, a2 = y2;
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (next >= 0) put(b + 1);
      block = next;
      __syncthreads();
    }
    return b;
  };
  const int rest = pass(std::false_type{}, first);
  if (rest < stop) pass(std::true_type{}, rest);

  // Out through LDS, a tile of the wave's at a time, so that rows are written whole.
  constexpr int PITCH = D + 8;
  uint16_t *const turned = (uint16_t *)held + wave * (16 * PITCH);
#pragma unroll
  for (int t = 0; t < RT; t++) {
    float sum = l[t];
    sum += lane_xor16(sum);
    sum += lane_xor32(sum);
    const float by = c.splits > 1 ? unit[t] : sum == 0 ? 0.0f : unit[t] / sum;
    const auto place = [&](int i) {  // of row i of the tile in out
      const int r = w0 + 16 * t + i;
      return (size_t)(row0 + r / c.group) * c.heads + kvh * c.group + r % c.group;
    };
    if (c.splits > 1) {
      if (w0 + 16 * t + col >= packed) continue;
      const size_t to = (size_t)split * rows.rows * c.heads + place(col);
#pragma unroll
      for (int d = 0; d < V; d++) *(f4 *)(c.part + to * D + 16 * d + 4 * quad) = o[t][d] * by;
      if (quad == 0) c.ml[to] = float2{m[t], sum};
      continue;
    }
#pragma unroll
    for (int d = 0; d < V; d++) {
      const f4 x = o[t][d] * by;
      *(u2 *)(turned + col * PITCH + 16 * d + 4 * quad) = u2{narrow2<DT>(x[0], x[1]), narrow2<DT>(x[2], x[3])};
    }
#pragma unroll
    for (int i = 0; i < D / 32; i++) {
      const int r = (64 * i + lane) / (D / 8), d = (64 * i + lane) % (D / 8) * 8;
      const u4 x = *(const u4 *)(turned + r * PITCH + d);
      if (w0 + 16 * t + r < packed) *(u4 *)((uint16_t *)c.out + place(r) * D + d) = x;
    }
  }
}

template <int D, int FMT, int DT, int RT>
static void launch(const Call &c, const Pool &pool, const Rows &rows, int tiles, uint32_t total, hipStream_t st) {
  hipLaunchKernelGGL(HIP_KERNEL_NAME(tile_kernel<D, FMT, DT, RT>), dim3(total), dim3(512), 2 * 16 * (D / 64) * 1024, st, c, pool, rows,
                     tiles);
}
void launch_tile(const Call &c, const Pool &pool, const Rows &rows, int format, int dtype, int row_tiles, int tiles, uint32_t total,
                 hipStream_t st) {
#define ISHZ_TILE_D(F, T)                                                                \
  if (pool.dim == 64 && row_tiles == 1) launch<64, F, T, 1>(c, pool, rows, tiles, total, st); \
  else if (pool.dim == 64) launch<64, F, T, 2>(c, pool, rows, tiles, total, st);          \
  else if (pool.dim == 256) launch<256, F, T, 1>(c, pool, rows, tiles, total, st);        \
  else if (row_tiles == 1) launch<128, F, T, 1>(c, pool, rows, tiles, total, st);         \
  else launch<128, F, T, 2>(c, pool, rows, tiles, total, st)
  if (format == ISHZ_KV_INT8) {
    if (dtype == ISHZ_DT_F16) { ISHZ_TILE_D(ISHZ_KV_INT8, ISHZ_DT_F16); } else { ISHZ_TILE_D(ISHZ_KV_INT8, ISHZ_DT_BF16); }
  } else {
    if (dtype == ISHZ_DT_F16) { ISHZ_TILE_D(ISHZ_KV_E4M3, ISHZ_DT_F16); } else { ISHZ_TILE_D(ISHZ_KV_E4M3, ISHZ_DT_BF16); }
  }
}
}  // namespace attn
