// Attention over the 8-bit block cache, for gfx950 (CDNA4): one new token of each
// sequence, or a chunk of them, against everything that the cache holds.
//
//   out[i] = sum_t softmax_t(scale q[i] . K[t]) V[t],  t <= position of row i
//
// with the keys and values that block_cache.hip stores: e4m3 codes and one scale a
// block and head, and the incomplete last block in 16 bits.
//
// Mapping.  The query heads of one key head and the chunk's tokens are the rows of
// one matrix; a wave holds TILES x 16 of them and walks over blocks of 64 tokens:
//   S^T = K Q^T    16 x 16 x 32 instructions with 16 tokens of K as rows
//   O^T += V^T P^T  the same with 16 features of V as rows
// In this orientation a lane holds the scores of ONE query row (l % 16) for 16
// tokens of a block, 16 (l / 16) .. + 15, so row sums and maxima are in-lane but for
// two exchanges, the weights are the second product's operand where they stand, and
// rescaling is one factor a lane.  K rows are dealt to the instruction's rows so
// that these 16 tokens are neighbours: the value codes, feature by feature in the
// cache, are then 16 bytes a lane, as the key codes are.  A wave loads its blocks
// straight into registers, the next one while it works on this one; nothing but the
// final merge goes through LDS.
//
// Precision.  Codes are exact in both types, so Q K^T takes them in the queries'
// type; the weights are fp16 (times 2^12, so that none above 2^-26 of the largest is
// subnormal), the scales, maxima, sums and outputs fp32.
//
// A long history is split over workgroups (and over the waves of one); a second
// launch merges their outputs with their maxima and sums.

#include <type_traits>

#include "decode_common.hpp"

namespace sah {
namespace {

constexpr float kWeightShift = 12.0f;  // log2 of what the weights are scaled by
constexpr int kUnits = 256;            // compute units

struct AttentionArgs {
  const void* query;
  void* output;  // [batch, seq, heads * D]
  const uint8_t* key_codes;
  const uint8_t* value_codes;
  const float* key_scales;
  const float* value_scales;
  const void* key_tail;
  const void* value_tail;
  const int32_t* table;
  const int32_t* starts;
  const int32_t* counts;
  float* partial;     // [batch, seq, heads, chunks, D]
  float* statistics;  // [batch, seq, heads, chunks, 2]: maximum, sum
  int64_t q_sb, q_sh, q_ss, o_sb, o_ss;
  int64_t blocks, max_blocks;
  int seq_len, heads, kv_heads, group;
  int chunks, chunk_blocks;
  uint32_t row_groups;
  float scale_log2;   // |scale| log2(e); log2(e) for a zero scale
  uint32_t sign;      // 0x80008000 where the scale is negative
  uint32_t keep;      // 0 for a zero scale: a zero query at scale 1
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The maximum over the four lanes l % 16 + {0, 16, 32, 48}.
__device__ __forceinline__ float quarters_max(float x) {
  typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
  const uint32_t a = __float_as_uint(x);
  const u32x2_t h = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane16_swap(a, a, false, false));
  const float y = fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
  const uint32_t c = __float_as_uint(y);
  const u32x2_t g = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(c, c, false, false));
  return fmaxf(__uint_as_float(g[0]), __uint_as_float(g[1]));
}
__device__ __forceinline__ float quarters_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Powers of two by their fp32 bits: 2^a / 2^b, 2^-126 where it is less.
__device__ __forceinline__ float power_ratio(int a_bits, int b_bits) {
  const int bits = 0x3f800000 + (a_bits - b_bits);
  return __int_as_float(bits < 0x00800000 ? 0x00800000 : bits);
}

// One block's codes of a wave: 16 bytes of a key row (value feature) a lane and tile.
template <int D>
struct KeyCodes {
  u32x4 part[4][D / 64];
};
template <int D>
struct ValueCodes {
  u32x4 part[D / 16];
};

template <typename T, int D, int TILES, int SPLIT, int ROWS>
__global__ __launch_bounds__(SPLIT * ROWS * 64) void cached_attention_kernel(const AttentionArgs a) {
  typedef typename Vec8<T>::type V8;
  constexpr int HALVES = D / 64;
  constexpr int FEATURES = D / 16;
  // One tile of rows waits for memory: keys and values of the next block are loaded
  // while this one is worked on.  More tiles work: the values come while the scores
  // are formed and the next keys during the rest, in half the registers.
  constexpr bool AHEAD = TILES == 1;
  // With more tiles the matrix cores add up the weights too (a row of ones).
  constexpr bool ONES = TILES > 1;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int column = lane & 15;    // query row of a tile; key row / value feature of an operand
  const int quarter = lane >> 4;
  const int split = wave % SPLIT;

  uint32_t at = blockIdx.x;
  const int chunk = (int)(at % (uint32_t)a.chunks);
  at /= (uint32_t)a.chunks;
  const uint32_t row_group = (at % a.row_groups) * ROWS + wave / SPLIT;
  at /= a.row_groups;
  const int h = (int)(at % (uint32_t)a.kv_heads);
  const int64_t b = at / (uint32_t)a.kv_heads;

  const int64_t start = a.starts[b];
  int count = a.counts != nullptr ? a.counts[b] : a.seq_len;
  if (count > a.seq_len) count = a.seq_len;
  if (start < 0 || count < 0) count = 0;
  // More tokens than the table can name: NaN.  Otherwise positions are below 2^31.
  const bool beyond = (start + count) / kBlockTokens > a.max_blocks;
  const int first_position = beyond ? 0 : (int)start;
  const int tail_block = beyond ? 0 : (int)((start + count) / kBlockTokens);

  // This lane's rows: token row / group of the chunk, query head h * group + row % group.
  const uint32_t first_row = row_group * (TILES * 16);  // rows are below 2^31
  int token[TILES], head[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const uint32_t row = first_row + t * 16 + column;
    token[t] = (int)(row / (uint32_t)a.group);
    head[t] = h * a.group + (int)(row - (uint32_t)token[t] * (uint32_t)a.group);
  }
  int last_position = -1, least_position = INT32_MAX;  // of the wave's rows
  {
    const int low = (int)(first_row / (uint32_t)a.group);
    const int high = (int)((first_row + TILES * 16 - 1) / (uint32_t)a.group);
    if (low < count) {
      least_position = first_position + low;
      last_position = first_position + (high < count ? high : count - 1);
    }
  }
  // Positions up to which a row sees; rows without a query see as far as the last.
  int sees[TILES];
  V8 q[TILES][HALVES][2];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const bool live = token[t] < count;
    sees[t] = live ? first_position + token[t] : last_position;
#pragma unroll
    for (int hh = 0; hh < HALVES; ++hh)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        u32x4 raw = {0u, 0u, 0u, 0u};
        if (live) {
          raw = load16(static_cast<const T*>(a.query) + b * a.q_sb + head[t] * a.q_sh + token[t] * a.q_ss +
                       hh * 64 + quarter * 16 + kk * 8);
          raw = (raw ^ a.sign) & a.keep;
        }
        q[t][hh][kk] = __builtin_bit_cast(V8, raw);
      }
  }

  // Blocks of this wave: the row group's, in chunks, the last chunk with the rest.
  const int all_blocks = last_position < 0 || beyond ? 0 : last_position / kBlockTokens + 1;
  const int64_t from64 = (int64_t)chunk * a.chunk_blocks;
  const int from = from64 < all_blocks ? (int)from64 : all_blocks;
  const int to = chunk == a.chunks - 1 || all_blocks - from < a.chunk_blocks ? all_blocks : from + a.chunk_blocks;
  const int coded_to = to < tail_block ? to : tail_block;

  // Outputs are held in units of a power of two, the largest value scale so far.
  f32x4 out[TILES][FEATURES];
  int unit = 0;  // its bits; 0 before the first block
  float most[TILES], sum[TILES];
  f32x4 sums[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    most[t] = -INFINITY;
    sum[t] = beyond && last_position >= 0 ? __builtin_nanf("") : 0.0f;
    sums[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int f = 0; f < FEATURES; ++f) out[t][f] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  }
  auto raise_unit = [&](int bits) {
    if (bits <= unit) return;
    if (unit != 0) {
      const float change = power_ratio(unit, bits);
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int f = 0; f < FEATURES; ++f) out[t][f] *= change;
    }
    unit = bits;
  };

  // The weights of a tile's row for one block, from its scores (16 tokens of the row
  // in this lane): the running maximum, sum and output are brought to it.
  auto softmax_step = [&](int t, f32x4 (&s)[4], float factor, int block, bool add) {
    if (block * kBlockTokens + (kBlockTokens - 1) > least_position) {
      const int open = sees[t] - block * kBlockTokens - quarter * 16;  // last visible of this lane's tokens
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i * 4 + j > open) s[i][j] = -INFINITY;
    }
    float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      top = fmaxf(fmaxf(top, s[i][0]), s[i][1]);
      top = fmaxf(fmaxf(top, s[i][2]), s[i][3]);
    }
    const float before = most[t];
    const float now = fmaxf(before, quarters_max(top) * factor);
    if (__any(now > before)) {
      // a row that has seen nothing yet has no output to rescale
      const float change = before == -INFINITY ? 0.0f : exp2_fast(before - now);
      sum[t] *= change;
      if (ONES) sums[t] *= change;
#pragma unroll
      for (int f = 0; f < FEATURES; ++f) out[t][f] *= change;
      most[t] = now;
    }
    const float shift = kWeightShift - (now == -INFINITY ? 0.0f : now);
    float lane_sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = exp2_fast(fmaf(s[i][j], factor, shift));
        if (add) lane_sum += s[i][j];
      }
    if (add) sum[t] += lane_sum;
  };

  auto load_keys = [&](KeyCodes<D>& c, int id) {
    const uint8_t* keys = a.key_codes + ((int64_t)id * a.kv_heads + h) * (kBlockTokens * D) + quarter * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int hh = 0; hh < HALVES; ++hh)
        c.part[i][hh] = load16(keys + ((column >> 2) * 16 + i * 4 + (column & 3)) * D + hh * 64);
  };
  auto load_values = [&](ValueCodes<D>& c, int id) {
    const uint8_t* values = a.value_codes + ((int64_t)id * a.kv_heads + h) * (kBlockTokens * D) + quarter * 16;
#pragma unroll
    for (int f = 0; f < FEATURES; ++f) c.part[f] = load16(values + (f * 16 + column) * kBlockTokens);
  };

  // A wave's blocks, 64 at a time: a lane each looks up the page and its scales.
  for (int base = from + split; base < coded_to; base += 64 * SPLIT) {
    int pages = -1;
    float key_scales = 0.0f, value_scales = 0.0f;
    const int mine = base + lane * SPLIT;
    if (mine < coded_to) {
      pages = a.table[b * a.max_blocks + mine];  // mine < tail_block <= max_blocks
      if (pages < 0 || pages >= a.blocks) pages = -1;
      if (pages >= 0) {
        key_scales = a.key_scales[(int64_t)pages * a.kv_heads + h];
        value_scales = a.value_scales[(int64_t)pages * a.kv_heads + h];
      }
    }
    const int left = (coded_to - base + SPLIT - 1) / SPLIT;
    const int count_here = left < 64 ? left : 64;
    KeyCodes<D> next_keys;
    ValueCodes<D> next_values;
    int page = __builtin_amdgcn_readlane(pages, 0);
    if (page >= 0) {
      load_keys(next_keys, page);
      if (AHEAD) load_values(next_values, page);
    }
    for (int i = 0; i < count_here; ++i) {
      const int block = base + i * SPLIT;
      const bool held = page >= 0;
      const int here = page;
      KeyCodes<D> keys = next_keys;
      ValueCodes<D> values;
      if (AHEAD) values = next_values;
      page = i + 1 < count_here ? __builtin_amdgcn_readlane(pages, i + 1) : -1;
      if (AHEAD && page >= 0) {
        load_keys(next_keys, page);
        load_values(next_values, page);
      }
      f32x4 s[TILES][4];
      if (held) {
        if (!AHEAD) load_values(values, here);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int hh = 0; hh < HALVES; ++hh)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
              const V8 k = e4m3_operand<T>(keys.part[r][hh][2 * kk], keys.part[r][hh][2 * kk + 1], 1.0f);
#pragma unroll
              for (int t = 0; t < TILES; ++t)
                s[t][r] = mfma16(k, q[t][hh][kk], hh + kk == 0 ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : s[t][r]);
            }
      }
      if (!AHEAD && page >= 0) load_keys(next_keys, page);
      if (!held) {  // a page outside the cache: every row that sees it answers NaN
#pragma unroll
        for (int t = 0; t < TILES; ++t)
          if (sees[t] >= block * kBlockTokens) sum[t] = __builtin_nanf("");
        continue;
      }
      // never 0, which would make NaN of a masked score
      const float factor = fmaxf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(key_scales), i)) * a.scale_log2,
                                 1.17549435e-38f);
      f16x8 p[TILES][2];
      if (!AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        softmax_step(t, s[t], factor, block, !ONES);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
          for (int e = 0; e < 8; ++e) p[t][k][e] = (f16)s[t][2 * k + e / 4][e % 4];
          if (ONES) {
            const f16 one = (f16)1.0f;
            sums[t] = mfma16((f16x8){one, one, one, one, one, one, one, one}, p[t][k], sums[t]);
          }
        }
      }
      if (!AHEAD) __builtin_amdgcn_sched_barrier(0);
      const int scale_bits = __builtin_amdgcn_readlane(__float_as_int(value_scales), i);
      raise_unit(scale_bits);
      const float ratio = power_ratio(scale_bits, unit);
      if (ratio >= 0x1p-15f) {  // codes times the ratio are exact in fp16
#pragma unroll
        for (int f = 0; f < FEATURES; ++f) {
          const f16x8 v0 = e4m3_operand<f16>(values.part[f][0], values.part[f][1], ratio);
          const f16x8 v1 = e4m3_operand<f16>(values.part[f][2], values.part[f][3], ratio);
#pragma unroll
          for (int t = 0; t < TILES; ++t) out[t][f] = mfma16(v1, p[t][1], mfma16(v0, p[t][0], out[t][f]));
        }
      } else {
#pragma unroll
        for (int f = 0; f < FEATURES; ++f) {
          const f16x8 v0 = e4m3_operand<f16>(values.part[f][0], values.part[f][1], 1.0f);
          const f16x8 v1 = e4m3_operand<f16>(values.part[f][2], values.part[f][3], 1.0f);
#pragma unroll
          for (int t = 0; t < TILES; ++t) {
            const f32x4 add = mfma16(v1, p[t][1], mfma16(v0, p[t][0], (f32x4){0.0f, 0.0f, 0.0f, 0.0f}));
#pragma unroll
            for (int j = 0; j < 4; ++j) out[t][f][j] = fmaf(add[j], ratio, out[t][f][j]);
          }
        }
      }
    }
  }

  // The incomplete block, in the tensors' own type: weights without the shift, in a
  // unit of at least 2^12 (the shift), so that large values do not overflow.
  if (tail_block >= from && tail_block < to && (tail_block - from) % SPLIT == split) {
    const int held = first_position + count - tail_block * kBlockTokens;  // tokens in it
    const int64_t tail_at = (b * a.kv_heads + h) * (int64_t)(kBlockTokens * D);
    const T* keys = static_cast<const T*>(a.key_tail) + tail_at + quarter * 16;
    const T* values = static_cast<const T*>(a.value_tail) + tail_at + quarter * 16;
    constexpr int SHIFT_BITS = (127 + (int)kWeightShift) << 23;
    raise_unit(SHIFT_BITS);
    const float ratio = power_ratio(SHIFT_BITS, unit);
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      if (t != 0) asm volatile("" ::: "memory");  // each tile loads its operands: kept, they would not fit
      f32x4 s[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int hh = 0; hh < HALVES; ++hh)
#pragma unroll
          for (int kk = 0; kk < 2; ++kk)
            s[i] = mfma16(*reinterpret_cast<const V8*>(
                              keys + ((column >> 2) * 16 + i * 4 + (column & 3)) * D + hh * 64 + kk * 8),
                          q[t][hh][kk], s[i]);
      }
      softmax_step(t, s, fmaxf(a.scale_log2, 1.17549435e-38f), tail_block, true);
      // bf16 weights keep 16 bits of precision as a sum of two; fp16 ones the shift
      constexpr bool WIDE = std::is_same<T, bf16>::value;
      V8 p[2], rest[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float w = s[2 * k + e / 4][e % 4] * (WIDE ? 0x1p-12f : 1.0f);
          p[k][e] = (T)w;
          rest[k][e] = (T)(w - (float)p[k][e]);
        }
#pragma unroll
      for (int f = 0; f < FEATURES; ++f) {
        f32x4 add = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          V8 v = *reinterpret_cast<const V8*>(values + (f * 16 + column) * kBlockTokens + k * 8);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (quarter * 16 + k * 8 + e >= held) v[e] = (T)0.0f;  // what stands behind the last token
          add = mfma16(v, p[k], add);
          if constexpr (WIDE) add = mfma16(v, rest[k], add);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) out[t][f][j] = fmaf(WIDE ? add[j] : add[j] * 0x1p-12f, ratio, out[t][f][j]);
      }
    }
  }

  // A row's sum over the four lanes that share it, and its output over the sum.
  const float unit_value = __int_as_float(unit);
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    sum[t] = quarters_sum(sum[t]);
    if (ONES) sum[t] += sums[t][0];
    const float inverse = sum[t] != 0.0f ? 1.0f / sum[t] : 0.0f;  // 0: a row that sees nothing here
#pragma unroll
    for (int f = 0; f < FEATURES; ++f)
#pragma unroll
      for (int j = 0; j < 4; ++j) out[t][f][j] = out[t][f][j] * inverse * unit_value;
  }

  // Merge of the waves that split the tokens, tile by tile: wave w's output weighs
  // sum_w 2^(most_w - top).
  if constexpr (SPLIT > 1) {
    constexpr int PITCH = D + 4;
    __shared__ float part[SPLIT * ROWS][16 * PITCH];
    __shared__ float stats[SPLIT * ROWS][16][2];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      if (t != 0) __syncthreads();
      if (quarter == 0) {
        stats[wave][column][0] = most[t];
        stats[wave][column][1] = sum[t];
      }
#pragma unroll
      for (int f = 0; f < FEATURES; ++f)
        *reinterpret_cast<f32x4*>(&part[wave][column * PITCH + f * 16 + quarter * 4]) = out[t][f];
      __syncthreads();
      // Each wave merges the tiles of features f % SPLIT == split of its rows.
      const int w0 = wave - split;
      float top = -INFINITY, total = 0.0f;
#pragma unroll
      for (int w = 0; w < SPLIT; ++w) top = fmaxf(top, stats[w0 + w][column][0]);
      const float base = top == -INFINITY ? 0.0f : top;
      float weight[SPLIT];
#pragma unroll
      for (int w = 0; w < SPLIT; ++w) {
        const float part_sum = stats[w0 + w][column][1];
        weight[w] = part_sum != 0.0f ? part_sum * exp2_fast(stats[w0 + w][column][0] - base) : 0.0f;
        total += weight[w];
      }
      most[t] = top;
      sum[t] = total;
      const float inverse = total != 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
      for (int f = 0; f < FEATURES; ++f) {
        if (f % SPLIT != split) continue;
        f32x4 merged = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < SPLIT; ++w) {
          const f32x4 v = *reinterpret_cast<const f32x4*>(&part[w0 + w][column * PITCH + f * 16 + quarter * 4]);
          const float share = weight[w] * inverse;
#pragma unroll
          for (int j = 0; j < 4; ++j) merged[j] = fmaf(v[j], share, merged[j]);
        }
        out[t][f] = merged;
      }
    }
  }

#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    if (token[t] >= a.seq_len) continue;
    const int64_t place = (b * a.seq_len + token[t]) * a.heads + head[t];
#pragma unroll
    for (int f = 0; f < FEATURES; ++f) {
      if (SPLIT > 1 && f % SPLIT != split) continue;
      if (a.chunks == 1) {
        T* o = static_cast<T*>(a.output) + b * a.o_sb + token[t] * a.o_ss + (int64_t)head[t] * D;
        typename Vec8<T>::half_type v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = token[t] < count ? (T)out[t][f][j] : (T)0.0f;  // rows without a query
        *reinterpret_cast<typename Vec8<T>::half_type*>(o + f * 16 + quarter * 4) = v;
      } else {
        *reinterpret_cast<f32x4*>(a.partial + (place * a.chunks + chunk) * D + f * 16 + quarter * 4) = out[t][f];
      }
    }
    if (a.chunks > 1 && split == 0 && quarter == 0) {
      float* statistics = a.statistics + (place * a.chunks + chunk) * 2;
      statistics[0] = most[t];
      statistics[1] = sum[t];
    }
  }
}

// Merge of the chunks, a wave a row: chunk c's output weighs sum_c 2^(most_c - top).
// A lane first looks at one chunk's statistics, then D / 4 lanes take a chunk's
// output each time, 256 / D chunks at once.
template <typename T, int D>
__global__ __launch_bounds__(256) void merge_kernel(const AttentionArgs a, int64_t rows) {
  constexpr int LANES = D / 4;
  constexpr int PARTS = 64 / LANES;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int feature = (lane % LANES) * 4;
  const int64_t token_row = row / a.heads;
  const int head = (int)(row - token_row * a.heads);
  const int64_t b = token_row / a.seq_len;
  const int64_t token = token_row - b * a.seq_len;
  const int count = a.counts != nullptr ? a.counts[b] : a.seq_len;
  const bool live = a.starts[b] >= 0 && token < count;

  f32x4 out = {0.0f, 0.0f, 0.0f, 0.0f};
  if (live) {
    const f32x2* statistics = reinterpret_cast<const f32x2*>(a.statistics) + row * a.chunks;
    const float* partial = a.partial + row * a.chunks * D + feature;
    float top = -INFINITY;
    for (int c = lane; c < a.chunks; c += 64) top = fmaxf(top, statistics[c][0]);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
    const float base = top == -INFINITY ? 0.0f : top;
    float total = 0.0f;
    for (int first = 0; first < a.chunks; first += 64) {
      float weight = 0.0f;
      if (first + lane < a.chunks) {
        const f32x2 s = statistics[first + lane];
        if (s[1] != 0.0f) weight = s[1] * exp2_fast(s[0] - base);  // 0: a chunk behind the row's last token
      }
      total += weight;
      const int here = a.chunks - first < 64 ? a.chunks - first : 64;
      for (int c = 0; c < here; c += 4 * PARTS) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int mine = c + u * PARTS + lane / LANES;
          const float w = __shfl(weight, mine);  // 0 behind the last chunk, whose output is then read again
          const int read = first + (mine < here ? mine : here - 1);
          const f32x4 v = *reinterpret_cast<const f32x4*>(partial + (int64_t)read * D);
#pragma unroll
          for (int j = 0; j < 4; ++j) out[j] = fmaf(v[j], w, out[j]);
        }
      }
    }
    total = wave_sum(total);
    const float inverse = total != 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
    for (int m = LANES; m < 64; m <<= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] += __shfl_xor(out[j], m);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] *= inverse;
  }
  if (lane >= LANES) return;
  typename Vec8<T>::half_type v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = (T)out[j];
  *reinterpret_cast<typename Vec8<T>::half_type*>(static_cast<T*>(a.output) + b * a.o_sb + token * a.o_ss +
                                                  (int64_t)head * D + feature) = v;
}

// How a call is laid out: row tiles of a wave, waves that split the tokens (the
// rest of a workgroup's four take other rows), workgroups of rows and chunks.
struct Layout {
  int tiles, split;
  int64_t row_groups;
  int chunks, chunk_blocks;
};

constexpr int kWaves = 4;

Layout layout_of(int64_t batch, int64_t seq_len, int64_t kv_heads, int64_t group, int64_t head_dim,
                 int64_t max_length) {
  Layout l{};
  const int64_t rows = seq_len * group;
  l.tiles = rows <= 16 ? 1 : 2;
  // waves that the registers leave room for, on all compute units
  const int64_t room = (int64_t)kUnits * 4 * (head_dim == 128 && l.tiles == 2 ? 1 : head_dim == 64 && l.tiles == 1 ? 3 : 2);
  const int64_t waves = batch * kv_heads * ceil_div(rows, 16 * l.tiles);
  const int64_t blocks = max_length / kBlockTokens + 1;
  l.split = waves >= room ? 1 : l.tiles == 1 && blocks <= 32 ? 8 : 4;
  if (l.tiles == 1 && l.split == 1) l.split = 4;
  l.row_groups = ceil_div(rows, (int64_t)16 * l.tiles * (l.split == 1 ? kWaves : 1));
  int64_t chunks = room / (waves * l.split);
  const int64_t most = ceil_div(blocks, 4 * l.split);
  if (chunks > most) chunks = most;
  if (chunks < 1) chunks = 1;
  l.chunk_blocks = (int)ceil_div(blocks, chunks);
  l.chunks = (int)ceil_div(blocks, l.chunk_blocks);
  return l;
}

template <typename T, int D>
int launch_attention(AttentionArgs& a, const Layout& l, int64_t batch, unsigned grid, hipStream_t stream) {
#define SAH_ATTENTION_CASE(TILES, SPLIT, ROWS)                                                               \
  if (l.tiles == TILES && l.split == SPLIT)                                                                  \
    hipLaunchKernelGGL((cached_attention_kernel<T, D, TILES, SPLIT, ROWS>), dim3(grid), dim3(SPLIT * ROWS * 64), 0, \
                       stream, a);
  SAH_ATTENTION_CASE(1, 4, 1)
  SAH_ATTENTION_CASE(1, 8, 1)
  SAH_ATTENTION_CASE(2, 4, 1)
  SAH_ATTENTION_CASE(2, 1, 4)
#undef SAH_ATTENTION_CASE
  int status = check_hip(hipGetLastError(), "cached attention launch");
  if (status != SAH_OK || l.chunks == 1) return status;
  const int64_t rows = batch * a.seq_len * a.heads;
  hipLaunchKernelGGL((merge_kernel<T, D>), dim3((unsigned)ceil_div(rows, 4)), dim3(256), 0, stream, a, rows);
  return check_hip(hipGetLastError(), "cached attention merge launch");
}

// Bytes of the chunks' outputs and statistics; the outputs come first.
size_t workspace_of(const Layout& l, int64_t batch, int64_t seq_len, int64_t heads, int64_t head_dim) {
  if (l.chunks == 1) return 0;
  return (size_t)(batch * seq_len * heads) * (size_t)l.chunks * (size_t)(head_dim + 2) * sizeof(float);
}

bool sizes_valid(int64_t batch, int64_t seq_len, int64_t heads, int64_t kv_heads, int64_t head_dim,
                 int64_t max_length) {
  return batch >= 0 && seq_len >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads <= 65536 &&
         (head_dim == 64 || head_dim == 128) && max_length >= 0 && max_length <= INT32_MAX && batch <= INT32_MAX &&
         seq_len <= (INT32_MAX - 256) / (heads / kv_heads) && (seq_len == 0 || batch <= ((int64_t)1 << 40) / (seq_len * heads));
}

}  // namespace
}  // namespace sah

using namespace sah;

extern "C" size_t sah_block_cache_attention_workspace_bytes(int64_t batch, int64_t seq_len, int64_t heads,
                                                            int64_t kv_heads, int64_t head_dim, int64_t max_length) {
  if (!sizes_valid(batch, seq_len, heads, kv_heads, head_dim, max_length) || batch == 0 || seq_len == 0) return 0;
  const Layout l = layout_of(batch, seq_len, kv_heads, heads / kv_heads, head_dim, max_length);
  return workspace_of(l, batch, seq_len, heads, head_dim);
}

extern "C" int sah_block_cache_attention(
    const void* query, const void* key_codes, const void* value_codes, const float* key_scales,
    const float* value_scales, const void* key_tail, const void* value_tail, const int32_t* block_table,
    const int32_t* starts, const int32_t* counts, void* output, int64_t batch, int64_t heads, int64_t kv_heads,
    int64_t seq_len, int64_t head_dim, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s,
    int64_t o_stride_b, int64_t o_stride_s, int64_t num_blocks, int64_t max_blocks, int64_t max_length, float scale,
    int dtype, void* workspace, size_t workspace_bytes, sah_stream_t stream) {
  const char* what = "sah_block_cache_attention";
  if (head_dim != 64 && head_dim != 128)
    return fail(SAH_ERR_UNSUPPORTED, "%s: head_dim %lld is not 64 or 128", what, (long long)head_dim);
  if (dtype != SAH_DTYPE_BF16 && dtype != SAH_DTYPE_F16)
    return fail(SAH_ERR_UNSUPPORTED, "%s: dtype %d is not bf16 or f16", what, dtype);
  if (!sizes_valid(batch, seq_len, heads, kv_heads, head_dim, max_length))
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: bad sizes (heads must be a multiple of kv_heads)", what);
  if (num_blocks < 0 || num_blocks > INT32_MAX || max_blocks < 0 || max_blocks > INT32_MAX / kBlockTokens)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: bad block count", what);
  const float scale_log2 = fabsf(scale) * 1.44269504f;
  if (!(scale_log2 < INFINITY)) return fail(SAH_ERR_INVALID_ARGUMENT, "%s: scale is not finite", what);
  if (batch == 0 || seq_len == 0) return SAH_OK;
  if (query == nullptr || output == nullptr || starts == nullptr || key_tail == nullptr || value_tail == nullptr ||
      (max_blocks != 0 && block_table == nullptr) ||
      (num_blocks != 0 && (key_codes == nullptr || value_codes == nullptr || key_scales == nullptr ||
                           value_scales == nullptr)))
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", what);
  const void* wide[] = {query, key_codes, value_codes, key_tail, value_tail, output, workspace};
  for (const void* p : wide)
    if (!aligned16(p)) return fail(SAH_ERR_INVALID_ARGUMENT, "%s: tensors must be 16-byte aligned", what);
  const void* words[] = {key_scales, value_scales, block_table, starts, counts};
  for (const void* p : words)
    if ((reinterpret_cast<uintptr_t>(p) & 3u) != 0)
      return fail(SAH_ERR_INVALID_ARGUMENT, "%s: scales, block table, starts and counts must be 4-byte aligned", what);
  const int64_t strides[] = {q_stride_b, q_stride_h, q_stride_s, o_stride_b, o_stride_s};
  for (int64_t v : strides)
    if (v % 8 != 0) return fail(SAH_ERR_INVALID_ARGUMENT, "%s: strides must be multiples of 8 elements", what);

  const Layout l = layout_of(batch, seq_len, kv_heads, heads / kv_heads, head_dim, max_length);
  const size_t need = workspace_of(l, batch, seq_len, heads, head_dim);
  if (need != 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(SAH_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  const int64_t units = batch * kv_heads;
  const int64_t most = (int64_t)(UINT32_MAX / 512);
  if (l.row_groups > most / l.chunks || units > most / (l.row_groups * l.chunks) ||
      batch * seq_len * heads > most * 8 - 8)
    return fail(SAH_ERR_UNSUPPORTED, "%s: too many rows for one launch", what);

  AttentionArgs a{};
  a.query = query;
  a.output = output;
  a.key_codes = static_cast<const uint8_t*>(key_codes);
  a.value_codes = static_cast<const uint8_t*>(value_codes);
  a.key_scales = key_scales;
  a.value_scales = value_scales;
  a.key_tail = key_tail;
  a.value_tail = value_tail;
  a.table = block_table;
  a.starts = starts;
  a.counts = counts;
  a.partial = static_cast<float*>(workspace);
  a.statistics = a.partial + (l.chunks == 1 ? 0 : batch * seq_len * heads * l.chunks * head_dim);
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.q_ss = q_stride_s;
  a.o_sb = o_stride_b;
  a.o_ss = o_stride_s;
  a.blocks = num_blocks;
  a.max_blocks = max_blocks;
  a.seq_len = (int)seq_len;
  a.heads = (int)heads;
  a.kv_heads = (int)kv_heads;
  a.group = (int)(heads / kv_heads);
  a.chunks = l.chunks;
  a.chunk_blocks = l.chunk_blocks;
  a.row_groups = (uint32_t)l.row_groups;
  a.sign = scale < 0.0f ? 0x80008000u : 0u;
  a.keep = scale == 0.0f ? 0u : ~0u;
  a.scale_log2 = scale == 0.0f ? 1.44269504f : scale_log2;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const unsigned grid = (unsigned)(units * l.row_groups * l.chunks);
  if (dtype == SAH_DTYPE_BF16)
    return head_dim == 64 ? launch_attention<bf16, 64>(a, l, batch, grid, s)
                          : launch_attention<bf16, 128>(a, l, batch, grid, s);
  return head_dim == 64 ? launch_attention<f16, 64>(a, l, batch, grid, s)
                        : launch_attention<f16, 128>(a, l, batch, grid, s);
}
