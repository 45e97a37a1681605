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

// One block's codes of a wave: 16 bytes of a key row (value feature) a lane and tile.
template <int D>
struct BlockCodes {
  u32x4 k[4][D / 64];
  u32x4 v[D / 16];
  float k_scale, v_scale;
  bool held;
};

template <typename T, int D, int TILES, int SPLIT, int ROWS>
__global__ __launch_bounds__(SPLIT * ROWS * 64) void cached_attention_kernel(const AttentionArgs a) {
  typedef typename Vec8<T>::type V8;
  constexpr int HALVES = D / 64;
  constexpr int FEATURES = D / 16;
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
  int64_t count = a.counts != nullptr ? (int64_t)a.counts[b] : (int64_t)a.seq_len;
  if (count > a.seq_len) count = a.seq_len;
  if (start < 0 || count < 0) count = 0;

  // This lane's rows: token row / group of the chunk, query head h * group + row % group.
  const uint32_t first_row = row_group * (TILES * 16);  // rows are below 2^31
  int64_t token[TILES];
  int head[TILES];
  int64_t last_position = -1, least_position = INT64_MAX;  // of the wave's rows
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const uint32_t row = first_row + t * 16 + column;
    const uint32_t i = row / (uint32_t)a.group;
    token[t] = i;
    head[t] = h * a.group + (int)(row - i * (uint32_t)a.group);
  }
  {
    const int64_t low = first_row / (uint32_t)a.group, high = (first_row + TILES * 16 - 1) / (uint32_t)a.group;
    if (low < count) {
      least_position = start + low;
      last_position = start + (high < count ? high : count - 1);
    }
  }
  // Positions up to which a row sees; rows without a query see as far as the last.
  int64_t sees[TILES];
  V8 q[TILES][HALVES][2];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const bool live = token[t] < count;
    sees[t] = live ? start + token[t] : last_position;
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
  const int64_t tail_block = (start + count) / kBlockTokens;
  const bool beyond = tail_block > a.max_blocks;  // more than the table can name
  const int64_t all_blocks = last_position < 0 || beyond ? 0 : last_position / kBlockTokens + 1;
  int64_t from = (int64_t)chunk * a.chunk_blocks;
  const int64_t to = chunk == a.chunks - 1 || from + a.chunk_blocks > all_blocks ? all_blocks : from + a.chunk_blocks;
  const int64_t coded_to = to < tail_block ? to : tail_block;

  f32x4 out[TILES][FEATURES];
  float most[TILES], sum[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    most[t] = -INFINITY;
    sum[t] = beyond && last_position >= 0 ? __builtin_nanf("") : 0.0f;
#pragma unroll
    for (int f = 0; f < FEATURES; ++f) out[t][f] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  }

  // The weights of a tile's row for one block, from its scores (16 tokens of the row
  // in this lane): the running maximum, sum and output are brought to it.
  auto softmax_step = [&](int t, f32x4 (&s)[4], float factor, int64_t block) {
    if (block * kBlockTokens + (kBlockTokens - 1) > least_position) {
      const int64_t open = sees[t] - block * kBlockTokens - quarter * 16;  // last visible of this lane's tokens
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i * 4 + j > open) s[i][j] = -INFINITY;
    }
    float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
#pragma unroll
    for (int i = 1; i < 4; ++i) top = fmaxf(top, fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3])));
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float before = most[t];
    const float now = fmaxf(before, top * factor);
    if (__any(now > before)) {
      // a row that has seen nothing yet has no output to rescale
      const float change = before == -INFINITY ? 0.0f : exp2_fast(before - now);
      sum[t] = sum[t] * change;
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
        lane_sum += s[i][j];
      }
    sum[t] += lane_sum;
  };

  auto load_block = [&](BlockCodes<D>& c, int64_t block) {
    const int64_t id = (int64_t)a.table[b * a.max_blocks + block];
    c.held = id >= 0 && id < a.blocks;  // block < tail_block <= max_blocks
    const int64_t entry = (c.held ? id : 0) * a.kv_heads + h;
    if (!c.held) return;
    const uint8_t* keys = a.key_codes + entry * (kBlockTokens * D) + quarter * 16;
    const uint8_t* values = a.value_codes + entry * (kBlockTokens * D) + quarter * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int hh = 0; hh < HALVES; ++hh)
        c.k[i][hh] = load16(keys + ((column >> 2) * 16 + i * 4 + (column & 3)) * D + hh * 64);
#pragma unroll
    for (int f = 0; f < FEATURES; ++f) c.v[f] = load16(values + (f * 16 + column) * kBlockTokens);
    c.k_scale = a.key_scales[entry];
    c.v_scale = a.value_scales[entry];
  };

  const int64_t first = from + split;
  BlockCodes<D> next;
  if (first < coded_to) load_block(next, first);
  for (int64_t block = first; block < coded_to; block += SPLIT) {
    const BlockCodes<D> c = next;
    if (block + SPLIT < coded_to) load_block(next, block + SPLIT);
    if (!c.held) {  // a page outside the cache: every row that sees it answers NaN
#pragma unroll
      for (int t = 0; t < TILES; ++t)
        if (sees[t] >= block * kBlockTokens) sum[t] = __builtin_nanf("");
      continue;
    }
    // never 0, which would make NaN of a masked score
    const float factor = fmaxf(c.k_scale * a.scale_log2, 1.17549435e-38f);
    f32x4 s[TILES][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int hh = 0; hh < HALVES; ++hh)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          const V8 k = e4m3_operand<T>(c.k[i][hh][2 * kk], c.k[i][hh][2 * kk + 1], 1.0f);
#pragma unroll
          for (int t = 0; t < TILES; ++t)
            s[t][i] = mfma16(k, q[t][hh][kk], hh + kk == 0 ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : s[t][i]);
        }
    }
    f16x8 p[TILES][2];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      softmax_step(t, s[t], factor, block);
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) p[t][k][e] = (f16)s[t][2 * k + e / 4][e % 4];
    }
#pragma unroll
    for (int f = 0; f < FEATURES; ++f) {
      const f16x8 v0 = e4m3_operand<f16>(c.v[f][0], c.v[f][1], 1.0f);
      const f16x8 v1 = e4m3_operand<f16>(c.v[f][2], c.v[f][3], 1.0f);
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        f32x4 sums = mfma16(v0, p[t][0], (f32x4){0.0f, 0.0f, 0.0f, 0.0f});
        sums = mfma16(v1, p[t][1], sums);
#pragma unroll
        for (int j = 0; j < 4; ++j) out[t][f][j] = fmaf(sums[j], c.v_scale, out[t][f][j]);
      }
    }
  }

  // The incomplete block, in the tensors' own type.
  if (tail_block >= from && tail_block < to && (tail_block - from) % SPLIT == split) {
    const int held = (int)(start + count - tail_block * kBlockTokens);  // tokens in it
    const int64_t tail_at = (b * a.kv_heads + h) * (int64_t)(kBlockTokens * D);
    const T* keys = static_cast<const T*>(a.key_tail) + tail_at + quarter * 16;
    const T* values = static_cast<const T*>(a.value_tail) + tail_at + quarter * 16;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
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
      softmax_step(t, s, fmaxf(a.scale_log2, 1.17549435e-38f), tail_block);
      // bf16 weights keep 16 bits of precision as a sum of two
      V8 p[2], rest[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float w = s[2 * k + e / 4][e % 4];
          p[k][e] = (T)w;
          rest[k][e] = (T)(w - (float)p[k][e]);
        }
#pragma unroll
      for (int f = 0; f < FEATURES; ++f)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          V8 v = *reinterpret_cast<const V8*>(values + (f * 16 + column) * kBlockTokens + k * 8);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (quarter * 16 + k * 8 + e >= held) v[e] = (T)0.0f;  // what stands behind the last token
          out[t][f] = mfma16(v, p[k], out[t][f]);
          if constexpr (std::is_same<T, bf16>::value) out[t][f] = mfma16(v, rest[k], out[t][f]);
        }
    }
  }

  // A row's sum over the four lanes that share it.
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    sum[t] += __shfl_xor(sum[t], 16);
    sum[t] += __shfl_xor(sum[t], 32);
  }

  // Merge of the waves that split the tokens, tile by tile.
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
      // Each wave merges the features FEATURES / SPLIT of its rows.
      const int w0 = wave - split;
      float top = -INFINITY, total = 0.0f;
#pragma unroll
      for (int w = 0; w < SPLIT; ++w) top = fmaxf(top, stats[w0 + w][column][0]);
      float weight[SPLIT];
#pragma unroll
      for (int w = 0; w < SPLIT; ++w) {
        weight[w] = top == -INFINITY ? 0.0f : exp2_fast(stats[w0 + w][column][0] - top);
        total += stats[w0 + w][column][1] * weight[w];
      }
      if (top == -INFINITY) {  // nothing seen, or pages outside the cache alone
#pragma unroll
        for (int w = 0; w < SPLIT; ++w) total += stats[w0 + w][column][1];
      }
      most[t] = top;
      sum[t] = total;
#pragma unroll
      for (int f = 0; f < FEATURES; ++f) {
        if (f % SPLIT != split) continue;
        f32x4 merged = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < SPLIT; ++w) {
          const f32x4 v = *reinterpret_cast<const f32x4*>(&part[w0 + w][column * PITCH + f * 16 + quarter * 4]);
#pragma unroll
          for (int j = 0; j < 4; ++j) merged[j] = fmaf(v[j], weight[w], merged[j]);
        }
        out[t][f] = merged;
      }
    }
  }

#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    if (token[t] >= a.seq_len) continue;
    if (a.chunks == 1) {
      // rows without a query and rows that see nothing are zeros
      const float inverse = token[t] < count && sum[t] != 0.0f ? 1.0f / sum[t] : 0.0f;
      T* o = static_cast<T*>(a.output) + b * a.o_sb + token[t] * a.o_ss + (int64_t)head[t] * D;
#pragma unroll
      for (int f = 0; f < FEATURES; ++f) {
        if (SPLIT > 1 && f % SPLIT != split) continue;
        typename Vec8<T>::half_type v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = token[t] < count ? (T)(out[t][f][j] * inverse) : (T)0.0f;
        *reinterpret_cast<typename Vec8<T>::half_type*>(o + f * 16 + quarter * 4) = v;
      }
    } else {
      const int64_t row = ((b * a.seq_len + token[t]) * a.heads + head[t]) * a.chunks + chunk;
#pragma unroll
      for (int f = 0; f < FEATURES; ++f) {
        if (SPLIT > 1 && f % SPLIT != split) continue;
        *reinterpret_cast<f32x4*>(a.partial + row * D + f * 16 + quarter * 4) = out[t][f];
      }
      if (split == 0 && quarter == 0) {
        a.statistics[row * 2] = most[t];
        a.statistics[row * 2 + 1] = sum[t];
      }
    }
  }
}

// Merge of the chunks: D / 4 lanes a row.
template <typename T, int D>
__global__ __launch_bounds__(256) void merge_kernel(const AttentionArgs a, int64_t rows) {
  constexpr int LANES = D / 4;
  const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (row >= rows) return;
  const int feature = (threadIdx.x % LANES) * 4;
  const int64_t token_row = row / a.heads;
  const int head = (int)(row - token_row * a.heads);
  const int64_t b = token_row / a.seq_len;
  const int64_t token = token_row - b * a.seq_len;
  const int64_t start = a.starts[b];
  const int64_t count = a.counts != nullptr ? (int64_t)a.counts[b] : (int64_t)a.seq_len;
  const bool live = start >= 0 && token < count;

  const float* statistics = a.statistics + row * a.chunks * 2;
  const float* partial = a.partial + row * a.chunks * D + feature;
  f32x4 out = {0.0f, 0.0f, 0.0f, 0.0f};
  if (live) {
    float top = -INFINITY, total = 0.0f;
    for (int c = 0; c < a.chunks; ++c) top = fmaxf(top, statistics[2 * c]);
    const float base = top == -INFINITY ? 0.0f : top;
    for (int c = 0; c < a.chunks; ++c) {
      const float sum = statistics[2 * c + 1];
      if (sum == 0.0f) continue;  // a chunk behind this row's last token
      const float weight = exp2_fast(statistics[2 * c] - base);
      total += sum * weight;
      const f32x4 v = *reinterpret_cast<const f32x4*>(partial + (int64_t)c * D);
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = fmaf(v[j], weight, out[j]);
    }
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] *= inverse;
  }
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
  const int most_tiles = head_dim == 64 ? 4 : 2;
  l.tiles = rows <= 16 ? 1 : rows <= 32 || most_tiles == 2 ? 2 : 4;
  l.split = rows <= 16 * l.tiles ? kWaves : 1;
  const int64_t rows_a_group = (int64_t)16 * l.tiles * (kWaves / l.split);
  l.row_groups = ceil_div(rows, rows_a_group);
  const int64_t blocks = max_length / kBlockTokens + 1;
  const int64_t units = batch * kv_heads * l.row_groups;
  // four workgroups a compute unit, of at least two blocks a wave
  int64_t chunks = ceil_div(4 * kUnits, units);
  const int64_t most = ceil_div(blocks, 2 * l.split);
  if (chunks > most) chunks = most;
  if (chunks < 1) chunks = 1;
  l.chunk_blocks = (int)ceil_div(blocks, chunks);
  l.chunks = (int)ceil_div(blocks, l.chunk_blocks);
  return l;
}

template <typename T, int D>
int launch_attention(AttentionArgs& a, const Layout& l, int64_t batch, unsigned grid, hipStream_t stream) {
#define SAH_ATTENTION_CASE(TILES, SPLIT)                                                                     \
  if (l.tiles == TILES && l.split == SPLIT)                                                                  \
    hipLaunchKernelGGL((cached_attention_kernel<T, D, TILES, SPLIT, kWaves / SPLIT>), dim3(grid),            \
                       dim3(kWaves * 64), 0, stream, a);
  SAH_ATTENTION_CASE(1, kWaves)
  SAH_ATTENTION_CASE(2, kWaves)
  SAH_ATTENTION_CASE(2, 1)
  if constexpr (D == 64) {
    SAH_ATTENTION_CASE(4, kWaves)
    SAH_ATTENTION_CASE(4, 1)
  }
#undef SAH_ATTENTION_CASE
  int status = check_hip(hipGetLastError(), "cached attention launch");
  if (status != SAH_OK || l.chunks == 1) return status;
  const int64_t rows = batch * a.seq_len * a.heads;
  hipLaunchKernelGGL((merge_kernel<T, D>), dim3((unsigned)ceil_div(rows, 256 / (D / 4))), dim3(256), 0, stream, a,
                     rows);
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
  const int64_t most = (int64_t)(UINT32_MAX / (kWaves * 64));
  if (l.row_groups > most / l.chunks || units > most / (l.row_groups * l.chunks) ||
      batch * seq_len * heads > most * 8)
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
