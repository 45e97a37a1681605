// Attention over the 8-bit block cache, for gfx950 (CDNA4): one new token of each
// sequence, or a chunk of them, against everything that the cache holds.
//
//   out[i] = sum_t softmax_t(scale q[i] . K[t]) V[t],  t <= position of row i
//
// with the keys and values that block_cache.hip stores: e4m3 codes and one scale a
// block and head, and the incomplete last block in 16 bits.
//
// Mapping.  The query heads of one key head and the chunk's tokens are the rows of
// one matrix; a wave holds 16 of them and walks over blocks of 64 tokens:
//   S^T = K Q^T    16 x 16 x 32 instructions with 16 tokens of K as rows
//   O^T += V^T P^T  the same with 16 features of V as rows
// In this orientation a lane holds the scores of ONE query row (l % 16) for 16
// tokens of a block, 16 (l / 16) .. + 15, so row sums and maxima are in-lane but for
// two exchanges, the weights are the second product's operand where they stand, and
// rescaling is one factor a lane.  K rows are dealt to the instruction's rows so
// that these 16 tokens are neighbours: the value codes, feature by feature in the
// cache, are then 16 bytes a lane, as the key codes are.  A wave loads its blocks
// straight into registers, the next block's keys and values as soon as this one's are
// used; nothing but the final merge goes through LDS.  Many rows (a chunk of tokens) go
// to a kernel of their own further down.
//
// Precision.  Codes are exact in both types, so Q K^T takes them in the queries'
// type; the weights are fp16 (times 2^11, so that none above 2^-25 of the largest is
// subnormal), the scales, maxima, sums and outputs fp32.  Here, and for the incomplete
// block, a weight is the sum of two 16-bit numbers, 22 bits (16 in bf16).  The kernel
// for chunks takes one of 11 bits for the coded blocks, and adds up what it takes: their
// errors, 2^-11 of a weight at most and of either sign, stay below a rounding of the
// output (fp16, 100 rows behind 3000 tokens, heads of 64: 2.17e-4 off in the root mean
// square, 2.10e-4 with the weights in fp32; bf16 1.647e-3, 1.646e-3), while two numbers
// cost it a third more time (2 x 512 rows behind 7680 tokens: heads of 64 58.6 / 80.6
// us, of 128 98 / 132) and this kernel 1 to 3% (64 x 2000 tokens 15.6 / 15.9 us, 32 x 100
// to 4095, heads of 128, 32.8 / 33.5).
//
// A long history is split over workgroups (and over the waves of one), which take its
// blocks in turn; a second launch merges their outputs with their maxima and sums.
//
// Bounds.  For a single token every feature of a held token is 2 bytes to read for
// 4 * group operations, so the codes' way from memory bounds it: 4 sequences of 90000
// to 100000 tokens, 16 heads of 64, 779 MB in 141 us, 5.5 TB/s (a copy moves 4.9), and
// 4.6 us for the merge of their parts.  32 sequences of 100 to 4095 tokens, 32 / 8 heads
// of 128 (138 MB), take 39 us, one of 777 tokens 8.1: there the longest wave's chain of
// loads bounds it.

#include <type_traits>

#include "decode_common.hpp"
#include "gemm_mainloop.hpp"

namespace sah {
namespace {

// Weights are 2^(score - base + kWeightShift); a row's base is raised to its maximum
// when that exceeds it by kWeightMargin, or in chunks when a weight leaves fp16's range
// (scores 5 above the base), so no weight is above 2^16.
constexpr float kWeightShift = 11.0f;
constexpr float kWeightMargin = 4.0f;
constexpr float kUnshift = 0x1p-11f;  // 2^-kWeightShift
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
  float* statistics;  // [batch, seq, heads, chunks, 2]: base, sum
  int64_t q_sb, q_sh, q_ss, o_sb, o_ss;
  int64_t blocks, max_blocks;
  int seq_len, heads, kv_heads, group;
  int chunks;
  uint32_t row_groups, batch;
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

// A wave's common value in a scalar register: a branch on it then is one, which the
// compiler does not see of what it divides or loads in vector registers.
__device__ __forceinline__ int common(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The maximum over lanes l and l ^ 32.
__device__ __forceinline__ float halves_max(float x) {
  const uint32_t a = __float_as_uint(x);
  const auto h = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  return fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
}

// Powers of two by their fp32 bits: 2^a / 2^b, 0 where it is below 2^-126.
__device__ __forceinline__ float power_ratio(int a_bits, int b_bits) {
  const int bits = (int)(0x3f800000u + (uint32_t)a_bits - (uint32_t)b_bits);  // used where a is at most b
  return __int_as_float(bits < 0x00800000 ? 0 : bits);
}

// A part's output that is weighed further: fp32's largest value where the type's largest
// ones were coded higher.  (A NaN row's weights are NaN, whatever its parts.)
__device__ __forceinline__ float finite_part(float x) {
  return __builtin_amdgcn_fmed3f(x, -3.40282347e38f, 3.40282347e38f);
}

// Whether any weight of an operand is not zero.
template <typename V8>
__device__ __forceinline__ bool any_weight(const V8 (&p)[2]) {
  const u32x4 bits = __builtin_bit_cast(u32x4, p[0]) | __builtin_bit_cast(u32x4, p[1]);
  return ((bits[0] | bits[1]) | (bits[2] | bits[3])) != 0;
}
template <typename V8>
__device__ __forceinline__ bool any_weight(const V8 (&p)[4]) {
  const u32x4 bits = (__builtin_bit_cast(u32x4, p[0]) | __builtin_bit_cast(u32x4, p[1])) |
                     (__builtin_bit_cast(u32x4, p[2]) | __builtin_bit_cast(u32x4, p[3]));
  return ((bits[0] | bits[1]) | (bits[2] | bits[3])) != 0;
}

// A row's outputs are held in a unit, the largest value scale so far of a block that it
// has weights in.  Rows of a wave share it (its bits; -1 where they do not), but a row
// that gives a block no weight, seen or not, does not follow it up by more than 2^60:
// what it holds would leave fp32.  What a row with a weight there loses is less than
// 2^-60 of the block's largest value.
constexpr int kUnitRise = 60 << 23;
__device__ __forceinline__ bool unit_rises(int unit, int bits, bool weighs) {
  return bits > unit && (unit == 0 || weighs || bits - unit <= kUnitRise);
}
__device__ __forceinline__ int common_unit(int unit) {
  const int first = common(unit);
  return __any(unit != first) ? -1 : first;
}

// How many of a sequence's `count` new rows see only blocks that its table has room for
// (the others answer NaN).  Their positions, and the tail's, are below 2^31.
__device__ __forceinline__ int rows_in_table(int64_t start, int count, int64_t max_blocks) {
  if ((start + count) / kBlockTokens <= max_blocks) return count;
  const int64_t room = max_blocks * kBlockTokens - start;  // below count
  return room < 0 ? 0 : (int)room;
}

template <typename T, int D, int SPLIT>
__global__ __launch_bounds__(SPLIT * 64) void cached_attention_kernel(const AttentionArgs a) {
  typedef typename Vec8<T>::type V8;
  constexpr int HALVES = D / 64;
  constexpr int FEATURES = D / 16;
  const int lane = threadIdx.x & 63;
  const int split = common(threadIdx.x >> 6);
  const int column = lane & 15;    // query row; key row / value feature of an operand
  const int quarter = lane >> 4;

  uint32_t at = blockIdx.x;
  const int chunk = common((int)(at % (uint32_t)a.chunks));
  at /= (uint32_t)a.chunks;
  const uint32_t group_row = (uint32_t)common((int)(at % a.row_groups)) * 16;
  at /= a.row_groups;
  const int h = common((int)(at % (uint32_t)a.kv_heads));
  const int64_t b = common((int)(at / (uint32_t)a.kv_heads));

  // The waves of all chunks take the blocks of a sequence in turn, whatever its length:
  // this one `first`, first + stride, ...  Their table entries are asked for before the
  // length is known; those behind the sequence's blocks are not used.
  const int first = chunk * SPLIT + split, stride = a.chunks * SPLIT;
  int first_pages = -1;
  if (first + (int64_t)lane * stride < a.max_blocks)
    first_pages = a.table[b * a.max_blocks + first + (int64_t)lane * stride];

  const int64_t start = common(a.starts[b]);
  int count = common(a.counts != nullptr ? a.counts[b] : a.seq_len);
  if (count > a.seq_len) count = a.seq_len;
  if (start < 0 || count < 0) count = 0;
  const int known = rows_in_table(start, count, a.max_blocks);
  const int first_position = known == 0 ? 0 : (int)start;
  const int tail_block = (first_position + known) / kBlockTokens;

  // This lane's row: token row / group of the chunk, query head h * group + row % group.
  const uint32_t row = group_row + column;
  const int token = (int)(row / (uint32_t)a.group);
  const int head = h * a.group + (int)(row - (uint32_t)token * (uint32_t)a.group);
  const bool live = token < count;
  const int last_position = first_position + known - 1;  // -1: no query
  // The position up to which the row sees; a row without a query sees as far as the last.
  const int sees = token < known ? first_position + token : last_position;
  V8 q[HALVES][2];
#pragma unroll
  for (int hh = 0; hh < HALVES; ++hh)
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      u32x4 raw = {0u, 0u, 0u, 0u};
      if (token < known) {
        raw = load16(static_cast<const T*>(a.query) + b * a.q_sb + head * a.q_sh + token * a.q_ss + hh * 64 +
                     quarter * 16 + kk * 8);
        raw = (raw ^ a.sign) & a.keep;
      }
      q[hh][kk] = __builtin_bit_cast(V8, raw);
    }

  const int all_blocks = known == 0 ? 0 : last_position / kBlockTokens + 1;
  const int coded_to = all_blocks < tail_block ? all_blocks : tail_block;

  f32x4 out[FEATURES];
  int unit = 0;  // the row's, 0 before the first block
  int wave_unit = 0;
  float most = -INFINITY;
  float sum = live && token >= known ? __builtin_nanf("") : 0.0f;
#pragma unroll
  for (int f = 0; f < FEATURES; ++f) out[f] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  auto raise_unit = [&](int bits, const auto& p) {
    if (bits <= wave_unit) return;
    if (wave_unit == 0 || (wave_unit > 0 && bits - wave_unit <= kUnitRise)) {  // every row follows
      if (wave_unit != 0) {
        const float change = power_ratio(wave_unit, bits);
#pragma unroll
        for (int f = 0; f < FEATURES; ++f) out[f] *= change;
      }
      unit = wave_unit = bits;
      return;
    }
    uint64_t weighs = __ballot(any_weight(p));
    weighs |= weighs >> 32;
    weighs |= weighs >> 16;
    const bool rises = unit_rises(unit, bits, (weighs >> column & 1) != 0);
    const float change = rises ? power_ratio(unit, bits) : 1.0f;  // of nothing, before the first block
#pragma unroll
    for (int f = 0; f < FEATURES; ++f) out[f] *= change;
    if (rises) unit = bits;
    wave_unit = common_unit(unit);
  };

  // The weights of the row for one block, from its scores (16 tokens of it in this
  // lane): the base, the sum and the output are brought to it.
  auto softmax_step = [&](f32x4 (&s)[4], float factor, int block) {
    if (block * kBlockTokens + (kBlockTokens - 1) > first_position) {
      const int open = sees - block * kBlockTokens - quarter * 16;  // last visible of this lane's tokens
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (r > open) s[r / 4][r % 4] = -INFINITY;
    }
    float top = fmaxf(s[0][0], s[0][1]);
#pragma unroll
    for (int r = 2; r < 16; r += 2) top = fmaxf(fmaxf(top, s[r / 4][r % 4]), s[r / 4][r % 4 + 1]);
    top = quarters_max(top) * factor;
    if (__any(top > most + kWeightMargin)) {
      const float now = fmaxf(most, top);
      // a row that has seen nothing yet has no output to rescale
      const float change = most == -INFINITY ? 0.0f : exp2_fast(most - now);
      sum *= change;
#pragma unroll
      for (int f = 0; f < FEATURES; ++f) out[f] *= change;
      most = now;
    }
    const float shift = kWeightShift - (most == -INFINITY ? 0.0f : most);
    float lane_sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r / 4][r % 4] = exp2_fast(fmaf(s[r / 4][r % 4], factor, shift));
      lane_sum += s[r / 4][r % 4];
    }
    sum += lane_sum;
  };

  // One block's codes: 16 bytes of a key row (value feature) a lane and tile.
  u32x4 keys[4][HALVES], values[FEATURES];
  auto load_keys = [&](int page) {
    const uint8_t* codes = a.key_codes + ((int64_t)page * a.kv_heads + h) * (kBlockTokens * D) + quarter * 16;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int hh = 0; hh < HALVES; ++hh)
        keys[r][hh] = load16(codes + ((column >> 2) * 16 + r * 4 + (column & 3)) * D + hh * 64);
  };
  auto load_values = [&](int page) {
    const uint8_t* codes = a.value_codes + ((int64_t)page * a.kv_heads + h) * (kBlockTokens * D) + quarter * 16;
#pragma unroll
    for (int f = 0; f < FEATURES; ++f) values[f] = load16(codes + (f * 16 + column) * kBlockTokens);
  };

  // A wave's blocks, 64 at a time: a lane each looks up the page and its scales.
  for (int base = first; base < coded_to; base += 64 * stride) {
    const int mine = base + lane * stride;
    int pages = first_pages;
    if (base != first && mine < coded_to) pages = a.table[b * a.max_blocks + mine];
    if (mine >= coded_to || pages < 0 || pages >= a.blocks) pages = -1;
    float key_scales = 0.0f, value_scales = 0.0f;
    if (pages >= 0) {
      key_scales = a.key_scales[(int64_t)pages * a.kv_heads + h];
      value_scales = a.value_scales[(int64_t)pages * a.kv_heads + h];
    }
    const int left = (coded_to - base + stride - 1) / stride;
    const int here = left < 64 ? left : 64;
    int page = __builtin_amdgcn_readlane(pages, 0);
    if (page >= 0) {
      load_keys(page);
      load_values(page);
    }
    for (int i = 0; i < here; ++i) {
      const int block = base + i * stride;
      const bool held = page >= 0;
      page = i + 1 < here ? __builtin_amdgcn_readlane(pages, i + 1) : -1;
      f32x4 s[4];
      if (held) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int hh = 0; hh < HALVES; ++hh)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
              s[r] = mfma16(e4m3_operand<T>(keys[r][hh][2 * kk], keys[r][hh][2 * kk + 1], 1.0f), q[hh][kk],
                            hh + kk == 0 ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : s[r]);
      }
      if (page >= 0) load_keys(page);
      if (held) {
        // never 0, which would make NaN of a masked score
        const float factor = fmaxf(
            __int_as_float(__builtin_amdgcn_readlane(__float_as_int(key_scales), i)) * a.scale_log2, 1.17549435e-38f);
        softmax_step(s, factor, block);
        f16x8 p[2], rest[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float w = s[2 * k + e / 4][e % 4];
            p[k][e] = (f16)w;
            rest[k][e] = (f16)(w - (float)p[k][e]);
          }
        const int scale_bits = __builtin_amdgcn_readlane(__float_as_int(value_scales), i);
        raise_unit(scale_bits, p);
        const float ratio = power_ratio(scale_bits, wave_unit);
        if (scale_bits <= wave_unit && ratio >= 0x1p-15f) {  // codes times the ratio are exact in fp16
#pragma unroll
          for (int f = 0; f < FEATURES; ++f) {
            const f16x8 v0 = e4m3_operand<f16>(values[f][0], values[f][1], ratio);
            const f16x8 v1 = e4m3_operand<f16>(values[f][2], values[f][3], ratio);
            out[f] = mfma16(v0, p[0], out[f]);
            out[f] = mfma16(v1, p[1], out[f]);
            out[f] = mfma16(v0, rest[0], out[f]);
            out[f] = mfma16(v1, rest[1], out[f]);
          }
        } else {
          const float to_unit = power_ratio(scale_bits, unit);
#pragma unroll
          for (int f = 0; f < FEATURES; ++f) {
            const f16x8 v0 = e4m3_operand<f16>(values[f][0], values[f][1], 1.0f);
            const f16x8 v1 = e4m3_operand<f16>(values[f][2], values[f][3], 1.0f);
            f32x4 add = mfma16(v0, p[0], (f32x4){0.0f, 0.0f, 0.0f, 0.0f});
            add = mfma16(v1, p[1], add);
            add = mfma16(v0, rest[0], add);
            add = mfma16(v1, rest[1], add);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[f][j] = fmaf(add[j], to_unit, out[f][j]);
          }
        }
      } else if (sees >= block * kBlockTokens) {  // a page outside the cache: NaN of every row that sees it
        sum = __builtin_nanf("");
      }
      if (page >= 0) load_values(page);
    }
  }

  // The incomplete block, in the tensors' own type: weights without the shift, in a
  // unit of at least 2^11 (the shift), so that large values do not overflow.
  if (tail_block < all_blocks && tail_block % stride == first) {
    const int held = first_position + known - tail_block * kBlockTokens;  // tokens in it
    const int64_t tail_at = (b * a.kv_heads + h) * (int64_t)(kBlockTokens * D);
    const T* tail_keys = static_cast<const T*>(a.key_tail) + tail_at + quarter * 16;
    const T* tail_values = static_cast<const T*>(a.value_tail) + tail_at + quarter * 16;
    constexpr int SHIFT_BITS = (127 + (int)kWeightShift) << 23;
    constexpr bool WIDE = std::is_same<T, bf16>::value;
    V8 v[FEATURES][2];
#pragma unroll
    for (int f = 0; f < FEATURES; ++f)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        v[f][k] = *reinterpret_cast<const V8*>(tail_values + (f * 16 + column) * kBlockTokens + k * 8);
    f32x4 s[4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int hh = 0; hh < HALVES; ++hh)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
          s[r] = mfma16(*reinterpret_cast<const V8*>(tail_keys + ((column >> 2) * 16 + r * 4 + (column & 3)) * D +
                                                     hh * 64 + kk * 8),
                        q[hh][kk], hh + kk == 0 ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : s[r]);
    asm volatile("" ::: "memory");  // the values are under way with the keys
    softmax_step(s, fmaxf(a.scale_log2, 1.17549435e-38f), tail_block);
    // weights as a sum of two; fp16 ones keep the shift
    V8 p[2], rest[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float w = s[2 * k + e / 4][e % 4] * (WIDE ? kUnshift : 1.0f);
        p[k][e] = (T)w;
        rest[k][e] = (T)(w - (float)p[k][e]);
      }
    raise_unit(SHIFT_BITS, p);
    const float ratio = power_ratio(SHIFT_BITS, unit);
#pragma unroll
    for (int f = 0; f < FEATURES; ++f) {
      f32x4 add = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (quarter * 16 + k * 8 + e >= held) v[f][k][e] = (T)0.0f;  // what stands behind the last token
        add = mfma16(v[f][k], p[k], add);
        add = mfma16(v[f][k], rest[k], add);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) out[f][j] = fmaf(WIDE ? add[j] : add[j] * kUnshift, ratio, out[f][j]);
    }
  }

  // The row's sum over the four lanes that share it, and its output over the sum.
  sum = quarters_sum(sum);
  const float inverse = sum != 0.0f ? 1.0f / sum : 0.0f;  // 0: a row that sees nothing here
  const float unit_value = __int_as_float(unit);

  // Merge of the waves: wave w's output weighs sum_w 2^(most_w - top).  Each wave merges
  // the tiles of 16 features f % SPLIT == split.
  constexpr int PITCH = D + 4;
  __shared__ __align__(16) float part[SPLIT][16 * PITCH];
  __shared__ float stats[SPLIT][16][2];
  if (quarter == 0) {
    stats[split][column][0] = most;
    stats[split][column][1] = sum;
  }
#pragma unroll
  for (int f = 0; f < FEATURES; ++f) {
#pragma unroll
    for (int j = 0; j < 4; ++j) out[f][j] = finite_part(out[f][j] * inverse * unit_value);
    *reinterpret_cast<f32x4*>(&part[split][column * PITCH + f * 16 + quarter * 4]) = out[f];
  }
  __syncthreads();
  if (token >= a.seq_len) return;
  float top = -INFINITY, total = 0.0f;
#pragma unroll
  for (int w = 0; w < SPLIT; ++w) top = fmaxf(top, stats[w][column][0]);
  const float base = top == -INFINITY ? 0.0f : top;
  float weight[SPLIT];
#pragma unroll
  for (int w = 0; w < SPLIT; ++w) {
    const float part_sum = stats[w][column][1];
    weight[w] = part_sum != 0.0f ? part_sum * exp2_fast(stats[w][column][0] - base) : 0.0f;
    total += weight[w];
  }
  const float share = total != 0.0f ? 1.0f / total : 0.0f;
  const int64_t place = ((b * a.seq_len + token) * a.heads + head) * a.chunks + chunk;
  for (int f = split; f < FEATURES; f += SPLIT) {
    f32x4 merged = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < SPLIT; ++w) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(&part[w][column * PITCH + f * 16 + quarter * 4]);
#pragma unroll
      for (int j = 0; j < 4; ++j) merged[j] = fmaf(v[j], weight[w] * share, merged[j]);
    }
    if (!live) merged = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    if (a.chunks == 1) {
      typename Vec8<T>::half_type v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = in_range<T>(merged[j]);
      *reinterpret_cast<typename Vec8<T>::half_type*>(static_cast<T*>(a.output) + b * a.o_sb + token * a.o_ss +
                                                      (int64_t)head * D + f * 16 + quarter * 4) = v;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) merged[j] = finite_part(merged[j]);
      *reinterpret_cast<f32x4*>(a.partial + place * D + f * 16 + quarter * 4) = merged;
    }
  }
  if (a.chunks > 1 && split == 0 && quarter == 0) {
    a.statistics[place * 2] = top;
    a.statistics[place * 2 + 1] = live ? total : 0.0f;
  }
}

// Attention of a chunk of new tokens: as above with 32 rows a wave, on 32 x 32 x 16
// products, which hold the scores of ONE query row (l % 32) for the 32 tokens
// 32 (l / 32) .. of a block in a lane.
//
// Many rows make it matrix work, and then the codes' way matters: read straight into
// the operands' order, every lane of a load touches another line.  So a block comes
// by direct-to-LDS loads of whole lines, one block ahead, and ROWS waves of other
// rows share it; 16-byte parts of a row change places by its number (key_turn,
// value_turn), so that the operands' reads of 8 and of 16 rows meet no bank twice.
// SPLIT groups of such waves take blocks in turn and merge in LDS at the end.
//
// The vector units bound it (busy 75% of the time, 32 weights and 64 conversions a
// lane and block; the matrix cores 25%, 16 instructions of 32 cycles), so with heads of
// 64 the products of the next block are issued beside this one's weights.  2 x 512
// tokens behind 7680, 16 / 4 heads: heads of 64 61 us, 33.3 GFLOP at 545 TFLOP/s; heads
// of 128 95 us, 700 TFLOP/s (107 with a row's maximum asked for in every block, which
// left too few registers).
template <int D>
__device__ __forceinline__ int key_turn(int t) {
  return D == 64 ? (((t >> 1) ^ (t >> 2)) & 1) | (((t >> 5) & 1) << 1)
                 : ((t ^ (t >> 2)) & 1) | (((t >> 1) & 1) << 1) | (((t >> 5) & 1) << 2);
}
__device__ __forceinline__ int value_turn(int d) { return (((d >> 1) ^ (d >> 3)) & 1) | (((d >> 2) & 1) << 1); }

template <typename T, int D, int SPLIT, int ROWS>
__global__ __launch_bounds__(SPLIT * ROWS * 64, 8 / (SPLIT * ROWS)) void chunk_attention_kernel(const AttentionArgs a) {
  typedef typename Vec8<T>::type V8;
  constexpr int WAVES = SPLIT * ROWS;
  constexpr int PAIRS = D / 32;      // 16-byte parts of a key row a lane
  constexpr int FEATURES = D / 32;   // tiles of 32 features
  constexpr int BYTES = kBlockTokens * D;  // of a block's keys, and of its values
  constexpr int LOADS = BYTES / 1024;      // wave loads of them
  constexpr int PITCH = 36;
  // Heads of 128 leave no registers for the scores of two blocks.  (The bound of 256
  // registers keeps two waves a SIMD.)
  constexpr bool AHEAD = D == 64;
  constexpr int TILES = D == 64 ? FEATURES : 1;  // that leave together
  static_assert(!AHEAD || 2 * PAIRS == 4, "a part of the next scores beside every eight weights");
  static_assert(LOADS % ROWS == 0, "every wave loads the same number of parts");
  union Shared {
    uint8_t block[SPLIT][4][BYTES];  // keys and values, twice
    float part[WAVES][TILES][32 * PITCH];
  };
  __shared__ __align__(16) Shared shared;
  __shared__ float stats[WAVES][32][2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int column = lane & 31;
  const int half = lane >> 5;
  const int split = wave / ROWS, row_wave = wave % ROWS;

  uint32_t at = blockIdx.x;
  // Key heads next to one another on the dies, so that each die's L2 keeps few of them.
  const int64_t b = common((int)(at % a.batch));
  at /= a.batch;
  const int h = common((int)(at % (uint32_t)a.kv_heads));
  at /= (uint32_t)a.kv_heads;
  const int chunk = common((int)(at % (uint32_t)a.chunks));
  const uint32_t group_row = (uint32_t)common((int)(at / (uint32_t)a.chunks)) * (ROWS * 32);  // rows are below 2^31

  // The queries and this wave's first table entries are asked for before its lengths
  // are known; those that do not count are not used.
  const uint32_t first_row = group_row + row_wave * 32;
  const uint32_t row = first_row + column;
  const int token = (int)(row / (uint32_t)a.group);
  V8 q[PAIRS][2];
  u32x4 loaded[PAIRS][2];
#pragma unroll
  for (int c = 0; c < PAIRS; ++c)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      loaded[c][e] = (u32x4){0u, 0u, 0u, 0u};
      if (token < a.seq_len) {
        const int head = h * a.group + (int)(row - (uint32_t)token * (uint32_t)a.group);
        loaded[c][e] = load16(static_cast<const T*>(a.query) + b * a.q_sb + head * a.q_sh + token * a.q_ss + c * 32 + half * 16 + e * 8);
      }
    }
  const int first_block = chunk * SPLIT + split, stride = a.chunks * SPLIT;
  int first_pages = -1;
  if (first_block + (int64_t)lane * stride < a.max_blocks)
    first_pages = a.table[b * a.max_blocks + first_block + (int64_t)lane * stride];

  const int64_t start = common(a.starts[b]);
  int count = common(a.counts != nullptr ? a.counts[b] : a.seq_len);
  if (count > a.seq_len) count = a.seq_len;
  if (start < 0 || count < 0) count = 0;
  const int known = rows_in_table(start, count, a.max_blocks);
  const int first_position = known == 0 ? 0 : (int)start;
  const int tail_block = (first_position + known) / kBlockTokens;

  // The last position that rows first .. first + rows - 1 see, -1 where none has a query.
  auto last_of = [&](uint32_t first, int rows) {
    const int low = common((int)(first / (uint32_t)a.group));
    const int high = common((int)((first + rows - 1) / (uint32_t)a.group));
    return low < known ? first_position + (high < known ? high : known - 1) : -1;
  };
  const int last_position = last_of(first_row, 32);
  const int group_last = last_of(group_row, ROWS * 32);
  const int least_position = first_position + common((int)(first_row / (uint32_t)a.group));
  const bool live = token < count;
  const int sees = token < known ? first_position + token : last_position;
#pragma unroll
  for (int c = 0; c < PAIRS; ++c)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const u32x4 raw = (loaded[c][e] ^ a.sign) & a.keep;
      q[c][e] = __builtin_bit_cast(V8, token < known ? raw : (u32x4){0u, 0u, 0u, 0u});
    }

  // The groups of all chunks take the blocks that the workgroup's rows see in turn; all
  // groups of a workgroup do as many turns, the last ones perhaps without a block.
  const int all_blocks = group_last < 0 ? 0 : group_last / kBlockTokens + 1;
  const int coded_to = all_blocks < tail_block ? all_blocks : tail_block;
  const int turns = coded_to > chunk * SPLIT ? (coded_to - chunk * SPLIT + stride - 1) / stride : 0;

  f32x16 out[FEATURES];
  int unit = 0, wave_unit = 0;
  float most = -INFINITY;
  float sum = live && token >= known ? __builtin_nanf("") : 0.0f;
#pragma unroll
  for (int f = 0; f < FEATURES; ++f) out[f] = (f32x16)(0.0f);
  auto raise_unit = [&](int bits, const auto& p) {
    if (bits <= wave_unit) return;
    if (wave_unit == 0 || (wave_unit > 0 && bits - wave_unit <= kUnitRise)) {  // every row follows
      if (wave_unit != 0) {
        const float change = power_ratio(wave_unit, bits);
#pragma unroll
        for (int f = 0; f < FEATURES; ++f) out[f] *= change;
      }
      unit = wave_unit = bits;
      return;
    }
    uint64_t weighs = __ballot(any_weight(p));
    weighs |= weighs >> 32;
    const bool rises = unit_rises(unit, bits, (weighs >> column & 1) != 0);
    const float change = rises ? power_ratio(unit, bits) : 1.0f;
#pragma unroll
    for (int f = 0; f < FEATURES; ++f) out[f] *= change;
    if (rises) unit = bits;
    wave_unit = common_unit(unit);
  };
  // The largest of a row's scores, times the factor (common to the lanes that share it).
  auto largest = [&](const f32x16 (&s)[2], float factor) {
    float top[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      top[k] = fmaxf(s[k / 2][k % 2 * 8], s[k / 2][k % 2 * 8 + 1]);
#pragma unroll
      for (int r = 2; r < 8; r += 2) top[k] = fmaxf(fmaxf(top[k], s[k / 2][k % 2 * 8 + r]), s[k / 2][k % 2 * 8 + r + 1]);
    }
    return halves_max(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]))) * factor;
  };
  auto hide = [&](f32x16 (&s)[2], int block) {  // what the row does not see
    const int open = sees - block * kBlockTokens - half * 32;
#pragma unroll
    for (int r = 0; r < 32; ++r)
      if (r > open) s[r / 16][r % 16] = -INFINITY;
  };
  auto raise_base = [&](float top) {
    const float now = fmaxf(most, top);
    const float change = most == -INFINITY ? 0.0f : exp2_fast(most - now);
    sum *= change;
#pragma unroll
    for (int f = 0; f < FEATURES; ++f) out[f] *= change;
    most = now;
  };
  auto shift_of = [&] { return kWeightShift - (most == -INFINITY ? 0.0f : most); };

  // This wave's part of the loads of a block's keys or values: slots of 16 bytes, its
  // lane's one each.
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)&shared.block[split][0][0];
  auto load_part = [&](int page, int buffer, auto of_values) {
    constexpr bool VALUES = decltype(of_values)::value;
    const uint8_t* codes = (VALUES ? a.value_codes : a.key_codes) + ((int64_t)page * a.kv_heads + h) * BYTES;
#pragma unroll
    for (int i = 0; i < LOADS / ROWS; ++i) {
      const int load = i * ROWS + row_wave;
      const int slot = load * 64 + lane;
      constexpr int PARTS = VALUES ? 4 : D / 16;  // of a row
      const int r = slot / PARTS, p = slot % PARTS;
      const int source = (r * PARTS + (p ^ (VALUES ? value_turn(r) : key_turn<D>(r)))) * 16;
      tile_dma16(codes, (uint32_t)source, lds + (buffer * 2 + VALUES) * BYTES + load * 1024);
    }
  };
  auto load_keys = [&](int page, int buffer) { load_part(page, buffer, std::false_type{}); };
  auto load_values = [&](int page, int buffer) { load_part(page, buffer, std::true_type{}); };

  // Scores of the block in a buffer, 32 tokens times 32 features at once.
  auto score_part = [&](f32x16 (&s)[2], int buffer, int part) {
    const int t = part / PAIRS, c = part % PAIRS;
    const int key = ((column >> 2) & 1) * 32 + t * 16 + (column >> 3) * 4 + (column & 3);
    const u32x4 raw = *reinterpret_cast<const u32x4*>(&shared.block[split][buffer * 2][0] + key * D +
                                                      ((c * 2 + half) ^ key_turn<D>(key)) * 16);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      s[t] = mfma32(e4m3_operand<T>(raw[2 * e], raw[2 * e + 1], 1.0f), q[c][e], c + e == 0 ? (f32x16)(0.0f) : s[t]);
  };
  auto score = [&](f32x16 (&s)[2], int buffer) {
#pragma unroll
    for (int part = 0; part < 2 * PAIRS; ++part) score_part(s, buffer, part);
  };
  // Eight weights of the lane in fp16, and their sum.
  auto weigh_part = [&](const f32x16 (&s)[2], int u, float factor, float shift, f16x8& p) {
    const f16x2 ones = {(f16)1.0f, (f16)1.0f};
    float added = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = (f16)exp2_fast(fmaf(s[u / 2][u % 2 * 8 + e], factor, shift));
#pragma unroll
    for (int e = 0; e < 8; e += 2) added = __builtin_amdgcn_fdot2((f16x2){p[e], p[e + 1]}, ones, added, false);
    return added;
  };
  auto value_operand = [&](int buffer, int f, int u, float scale) {
    const int d = f * 32 + column;
    const u32x2 raw = *reinterpret_cast<const u32x2*>(&shared.block[split][buffer * 2 + 1][0] + d * kBlockTokens +
                                                      ((half * 2 + u / 2) ^ value_turn(d)) * 16 + u % 2 * 8);
    return e4m3_operand<f16>(raw[0], raw[1], scale);
  };

  // The group's blocks, 64 at a time: a lane each looks up the page and its scales.  A
  // page outside the cache is loaded as the first one, and not used.
  int pages = -1;
  float key_scales = 0.0f, value_scales = 0.0f;
  auto look_up = [&](int first) {
    const int64_t mine = first_block + (int64_t)(first + lane) * stride;
    pages = first == 0 ? first_pages : -1;
    if (first != 0 && mine < coded_to) pages = a.table[b * a.max_blocks + mine];
    if (mine >= coded_to) pages = -1;
    if (pages < 0 || pages >= a.blocks) pages = -1;
    if (pages >= 0) {
      key_scales = a.key_scales[(int64_t)pages * a.kv_heads + h];
      value_scales = a.value_scales[(int64_t)pages * a.kv_heads + h];
    }
  };
  auto page_of = [&](int i) {
    const int page = __builtin_amdgcn_readlane(pages, i);
    return page < 0 ? 0 : page;
  };
  // Block i of this look-up, AHEAD: its scores in s; those of block i + 1 go to next
  // while this one's weights are formed and used.
  auto step = [&](int first, int i, int here, f32x16 (&s)[2], f32x16 (&next)[2]) {
    // Loads under way, in order: (keys i,) values i, keys i + 1, values i + 1.
    if (i + 1 < here)
      wait_loads<(AHEAD ? 1 : 2) * (LOADS / ROWS)>();
    else
      wait_loads<0>();
    if (AHEAD) wait_lds();  // keys i are read
    if (ROWS > 1) tile_barrier();  // every wave's part of the loads has come
    if (AHEAD && i + 2 < here) load_keys(page_of(i + 2), i & 1);
    if (!AHEAD) score(s, i & 1);
    const int block = first_block + (first + i) * stride;
    const bool held = __builtin_amdgcn_readlane(pages, i) >= 0;
    const bool seen = block < coded_to && block * kBlockTokens <= last_position;
    const bool whole = block * kBlockTokens + (kBlockTokens - 1) <= least_position;
    // never 0, which would make NaN of a masked score
    const float factor =
        fmaxf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(key_scales), i)) * a.scale_log2, 1.17549435e-38f);
    const int scale_bits = __builtin_amdgcn_readlane(__float_as_int(value_scales), i);
    const float ratio = power_ratio(scale_bits, wave_unit);
    f16x8 p[4];
    bool done = false;
    // Nearly all blocks: seen whole, no base or unit to raise, codes times the ratio of
    // scales exact in fp16.  The next block's products run beside the weights, and the
    // row's maximum is not asked for: a weight that left fp16's range is infinite, and so
    // is the sum.  Then the block is done again below.
    if (seen && held && whole && scale_bits <= wave_unit && ratio >= 0x1p-15f) {
      const float shift = shift_of();
      float added[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (AHEAD) score_part(next, (i + 1) & 1, u);
        added[u] = weigh_part(s, u, factor, shift, p[u]);
      }
      const float all = (added[0] + added[1]) + (added[2] + added[3]);
      if (!__any(!(all < INFINITY))) {
        sum += all;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int f = 0; f < FEATURES; ++f) out[f] = mfma32(value_operand(i & 1, f, u, ratio), p[u], out[f]);
        done = true;
      }
    } else if (AHEAD) {
      score(next, (i + 1) & 1);
    }
    if (!done && seen) {
      if (!held) {  // a page outside the cache
        if (sees >= block * kBlockTokens) sum = __builtin_nanf("");
      } else {
        if (!whole) hide(s, block);
        const float top = largest(s, factor);
        if (__any(top > most + kWeightMargin)) raise_base(top);
        const float shift = shift_of();
#pragma unroll
        for (int u = 0; u < 4; ++u) sum += weigh_part(s, u, factor, shift, p[u]);
        raise_unit(scale_bits, p);
        const float to_unit = power_ratio(scale_bits, unit);
#pragma unroll
        for (int f = 0; f < FEATURES; ++f) {
          f32x16 add = (f32x16)(0.0f);
#pragma unroll
          for (int u = 0; u < 4; ++u) add = mfma32(value_operand(i & 1, f, u, 1.0f), p[u], add);
#pragma unroll
          for (int r = 0; r < 16; ++r) out[f][r] = fmaf(add[r], to_unit, out[f][r]);
        }
      }
    }
    if (i + 2 < here) {
      wait_lds();
      if (ROWS > 1) tile_barrier();  // values i (and keys i) are read
      if (!AHEAD) load_keys(page_of(i + 2), i & 1);
      load_values(page_of(i + 2), i & 1);
    }
  };
  if (a.blocks == 0) {  // no cache to read
    if (first_block < coded_to && sees >= first_block * kBlockTokens) sum = __builtin_nanf("");
  } else {
    for (int first = 0; first < turns; first += 64) {
      look_up(first);
      const int here = turns - first < 64 ? turns - first : 64;
      if (first != 0) {  // the buffers' last blocks are read
        wait_lds();
        if (ROWS > 1) tile_barrier();
      }
      load_keys(page_of(0), 0);
      load_values(page_of(0), 0);
      if (here > 1) {
        load_keys(page_of(1), 1);
        load_values(page_of(1), 1);
        if (AHEAD) wait_loads<3 * (LOADS / ROWS)>();
      } else {
        wait_loads<0>();
      }
      f32x16 even[2], odd[2];
      if (AHEAD) {
        if (ROWS > 1) tile_barrier();
        score(even, 0);
      }
      for (int i = 0; i < here; i += 2) {
        step(first, i, here, even, odd);
        if (i + 1 < here) step(first, i + 1, here, odd, even);
      }
    }
  }

  // The incomplete block, as above.
  if (last_position >= tail_block * kBlockTokens && tail_block % stride == first_block) {
    const int held = first_position + known - tail_block * kBlockTokens;
    const int64_t tail_at = (b * a.kv_heads + h) * (int64_t)(kBlockTokens * D);
    const T* keys = static_cast<const T*>(a.key_tail) + tail_at + half * 16;
    const T* values = static_cast<const T*>(a.value_tail) + tail_at + half * 32;
    f32x16 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int key = ((column >> 2) & 1) * 32 + t * 16 + (column >> 3) * 4 + (column & 3);
#pragma unroll
      for (int c = 0; c < PAIRS; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          s[t] = mfma32(*reinterpret_cast<const V8*>(keys + key * D + c * 32 + e * 8), q[c][e],
                        c + e == 0 ? (f32x16)(0.0f) : s[t]);
    }
    constexpr int SHIFT_BITS = (127 + (int)kWeightShift) << 23;
    constexpr bool WIDE = std::is_same<T, bf16>::value;
    const float factor = fmaxf(a.scale_log2, 1.17549435e-38f);
    hide(s, tail_block);
    const float top = largest(s, factor);
    if (__any(top > most + kWeightMargin)) raise_base(top);
    const float shift = shift_of();
    V8 p[4], rest[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float weight = exp2_fast(fmaf(s[u / 2][u % 2 * 8 + e], factor, shift));
        sum += weight;
        const float w = weight * (WIDE ? kUnshift : 1.0f);
        p[u][e] = (T)w;
        rest[u][e] = (T)(w - (float)p[u][e]);
      }
    raise_unit(SHIFT_BITS, p);
    const float ratio = power_ratio(SHIFT_BITS, unit);
#pragma unroll
    for (int f = 0; f < FEATURES; ++f) {
      f32x16 add = (f32x16)(0.0f);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        V8 v = *reinterpret_cast<const V8*>(values + (f * 32 + column) * kBlockTokens + u * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (half * 32 + u * 8 + e >= held) v[e] = (T)0.0f;  // what stands behind the last token
        add = mfma32(v, p[u], add);
        add = mfma32(v, rest[u], add);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) out[f][r] = fmaf(WIDE ? add[r] : add[r] * kUnshift, ratio, out[f][r]);
    }
  }

  // Merge and store: the SPLIT waves of the same rows weigh their outputs by their share
  // of the row's sum, as above, and their sums leave in runs of 32 features.
  sum += __shfl_xor(sum, 32);
  if (half == 0) {
    stats[wave][column][0] = most;
    stats[wave][column][1] = sum;
  }
  __syncthreads();  // also: the blocks are read
  float top = -INFINITY, total = 0.0f;
#pragma unroll
  for (int w = 0; w < SPLIT; ++w) top = fmaxf(top, stats[w * ROWS + row_wave][column][0]);
  const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
  for (int w = 0; w < SPLIT; ++w) {
    const float part_sum = stats[w * ROWS + row_wave][column][1];
    total += part_sum != 0.0f ? part_sum * exp2_fast(stats[w * ROWS + row_wave][column][0] - base) : 0.0f;
  }
  const float share = sum != 0.0f && total != 0.0f ? exp2_fast(most - base) / total : 0.0f;
  const float unit_value = __int_as_float(unit);
  if (a.chunks > 1 && split == 0 && half == 0 && token < a.seq_len) {
    const int head = h * a.group + (int)(row - (uint32_t)token * (uint32_t)a.group);
    const int64_t place = ((b * a.seq_len + token) * a.heads + head) * a.chunks + chunk;
    *reinterpret_cast<f32x2*>(a.statistics + place * 2) = (f32x2){top, live ? total : 0.0f};
  }
  for (int pass = 0; pass < FEATURES / TILES; ++pass) {
    if (pass != 0) __syncthreads();  // the last tiles are read
#pragma unroll
    for (int f = 0; f < TILES; ++f)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = out[f][k * 4 + e];
#pragma unroll
          for (int g = 1; g < FEATURES / TILES; ++g) x = pass == g ? out[g * TILES + f][k * 4 + e] : x;
          v[e] = x * share * unit_value;
        }
        *reinterpret_cast<f32x4*>(&shared.part[wave][f][column * PITCH + k * 8 + half * 4]) = v;
      }
    __syncthreads();
#pragma unroll
    for (int i = split * 64 + lane; i < 32 * 8; i += SPLIT * 64) {
      const int r = i / 8, feature = i % 8 * 4;
      const uint32_t its_row = first_row + r;
      const int its_token = (int)(its_row / (uint32_t)a.group);
      const int head = h * a.group + (int)(its_row - (uint32_t)its_token * (uint32_t)a.group);
      if (its_token >= a.seq_len) continue;
#pragma unroll
      for (int f = 0; f < TILES; ++f) {
        f32x4 merged = {0.0f, 0.0f, 0.0f, 0.0f};
        if (its_token < count) {  // rows without a query stay zeros
#pragma unroll
          for (int w = 0; w < SPLIT; ++w)
            merged += *reinterpret_cast<const f32x4*>(&shared.part[w * ROWS + row_wave][f][r * PITCH + feature]);
        }
        const int at = (pass * TILES + f) * 32 + feature;
        if (a.chunks == 1) {
          typename Vec8<T>::half_type v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = in_range<T>(merged[e]);
          *reinterpret_cast<typename Vec8<T>::half_type*>(static_cast<T*>(a.output) + b * a.o_sb + its_token * a.o_ss +
                                                          (int64_t)head * D + at) = v;
        } else {
          const int64_t place = ((b * a.seq_len + its_token) * a.heads + head) * a.chunks + chunk;
#pragma unroll
          for (int e = 0; e < 4; ++e) merged[e] = finite_part(merged[e]);
          *reinterpret_cast<f32x4*>(a.partial + place * D + at) = merged;
        }
      }
    }
  }
}

// Merge of the chunks, a wave a row: chunk c's output weighs its share of the chunks'
// sum_c 2^(most_c - top).  A lane first looks at one chunk's statistics, then D / 4 lanes
// take a chunk's output each time, 256 / D chunks at once.
template <typename T, int D>
__global__ __launch_bounds__(256) void merge_kernel(const AttentionArgs a, int64_t rows) {
  constexpr int LANES = D / 4;
  constexpr int PARTS = 64 / LANES;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int feature = (lane % LANES) * 4;
  const f32x2* statistics = reinterpret_cast<const f32x2*>(a.statistics) + row * a.chunks;
  const float* partial = a.partial + row * a.chunks * D + feature;
  // (a sum of 0: a chunk behind the row's last token, or a row without a query)
  const f32x2 nothing = {-INFINITY, 0.0f};
  const f32x2 own = lane < a.chunks ? statistics[lane] : nothing;
  float top = own[0];
  for (int c = lane + 64; c < a.chunks; c += 64) top = fmaxf(top, statistics[c][0]);
  f32x4 out = {0.0f, 0.0f, 0.0f, 0.0f};
  auto weight_of = [&](f32x2 s) {
    return s[1] != 0.0f ? s[1] * exp2_fast(s[0] - (top == -INFINITY ? 0.0f : top)) : 0.0f;
  };
  float inverse = 0.0f;
  for (int first = 0; first < a.chunks; first += 64) {
    const int here = a.chunks - first < 64 ? a.chunks - first : 64;
    f32x4 v[4];
    auto load = [&](int c) {  // the parts' outputs do not wait for their weights
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int mine = c + u * PARTS + lane / LANES;
        v[u] = *reinterpret_cast<const f32x4*>(partial + (int64_t)(first + (mine < here ? mine : here - 1)) * D);
      }
    };
    load(0);
    if (first == 0) {
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
      float total = weight_of(own);
      for (int c = lane + 64; c < a.chunks; c += 64) total += weight_of(statistics[c]);
      total = wave_sum(total);
      inverse = total != 0.0f ? 1.0f / total : 0.0f;
    }
    const f32x2 s = first == 0 ? own : first + lane < a.chunks ? statistics[first + lane] : nothing;
    const float weight = weight_of(s) * inverse;
    for (int c = 0; c < here; c += 4 * PARTS) {
      if (c != 0) load(c);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float w = __shfl(weight, c + u * PARTS + lane / LANES);  // 0 behind the last chunk
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = fmaf(v[u][j], w, out[j]);
      }
    }
  }
#pragma unroll
  for (int m = LANES; m < 64; m <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] += __shfl_xor(out[j], m);
  if (lane >= LANES) return;
  const int64_t token_row = row / a.heads;
  const int head = (int)(row - token_row * a.heads);
  const int64_t b = token_row / a.seq_len;
  const int64_t token = token_row - b * a.seq_len;
  typename Vec8<T>::half_type v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = in_range<T>(out[j]);
  *reinterpret_cast<typename Vec8<T>::half_type*>(static_cast<T*>(a.output) + b * a.o_sb + token * a.o_ss +
                                                  (int64_t)head * D + feature) = v;
}

// How a call is laid out: rows of a wave (16, the decoding kernel, or 32, the chunk
// kernel), groups of waves that split the tokens of the same rows, waves of a group,
// workgroups of rows and chunks.
struct Layout {
  int wave_rows, split, rows;
  int64_t row_groups;
  int chunks;
};

Layout layout_of(int64_t batch, int64_t seq_len, int64_t kv_heads, int64_t group, int64_t head_dim,
                 int64_t max_length) {
  Layout l{};
  const int64_t rows = seq_len * group;
  const int64_t blocks = max_length / kBlockTokens + 1;
  l.rows = 1;
  // waves that the registers leave room for, on all compute units
  const int64_t few = (int64_t)kUnits * 4 * (head_dim == 64 ? 3 : 2), room = (int64_t)kUnits * 4 * 2;
  // A few groups of 16 rows, while eight waves of each fit the units, are done sooner by
  // the kernel without LDS on the blocks' way than by the one for chunks, which does more
  // rows a conversion (us, 16 / 32 rows a wave: 19 x 48 rows behind 2944 tokens, 4 key
  // heads of 128 30.7 / 41.4; 1 x 32 behind 629 9.5 / 13.8; 64 x 40 behind 1000, 8 heads
  // of 64 49 / 26).
  l.row_groups = ceil_div(rows, 16);
  l.wave_rows = rows <= 16 || (rows <= 64 && batch * kv_heads * l.row_groups * 8 <= few) ? 16 : 32;
  if (l.wave_rows == 16) {
    // The waves of a workgroup split the tokens, which leaves fewer parts to merge
    // through memory.  Eight of them do in one launch what four leave to a second one,
    // but leave registers unused with heads of 64 (tokens of a sequence, us with both
    // launches, eight / four: 64 x 2000 14.6 / 20.1, 64 x 8000 49.6 / 54.8; 8 x 20000
    // 28.4 / 25.2, 4 x 100000 160 / 142).  `blocks` counts the incomplete one: at a room of
    // 8192 tokens four begin (16 / 4 heads of 64: 1 x 8000 13.3 / 11.3, 32 x 2000 18.5 /
    // 13.8, 32 x 8000 35.7 / 28.5, 64 x 2000 14.7 / 22.1).
    l.split = blocks <= 128 ? 8 : 4;
    int64_t chunks = few / (batch * kv_heads * l.row_groups * l.split);
    // A part for every four blocks a wave, and one for what is left over: two from 33
    // blocks on, a room of 2048 tokens, where the second launch costs what it gives (us,
    // two parts / one, one sequence of 1500 / 2000 / 4000 tokens: 16 / 4 heads of 64 10.6 / 9.4,
    // 10.8 / 10.9, 13.6 / 16.5; 32 / 8 heads of 128 14.8 / 14.8, 14.9 / 17.6, 20.1 / 28.0).
    const int64_t most = ceil_div(blocks, 4 * l.split);
    if (chunks > most) chunks = most;
    l.chunks = chunks < 1 ? 1 : (int)chunks;
    return l;
  }
  // Heads of 128 have the registers for one block's scores only, and more to gain from
  // blocks shared by four waves of other rows (2 x 512 rows behind 7680 tokens, 16 / 4
  // heads: heads of 128 112 / 95 shared, heads of 64 62 / 68).
  const bool shared = head_dim == 128 && rows > 64;
  if (shared) l.rows = 4;
  l.row_groups = ceil_div(rows, (int64_t)32 * l.rows);
  const int64_t waves = batch * kv_heads * l.row_groups * l.rows;
  // Rows' waves split their tokens to fill the units, further over workgroups with a
  // second launch.  In blocks of 64 tokens, 2 us each: a wave's start and end cost six,
  // the second launch five and its parts' way through memory.  (24 x 479 rows behind 225
  // to 445, 8 heads of 64: one wave 46 us, four 64; 2 x 512 rows behind 7680 as above: two
  // waves and a second launch 72, four 62; 3 x 394, 12 / 1 heads of 128 behind 73 to 359:
  // one launch 28, two 33.)
  double least = INFINITY;
  for (int split = shared ? 2 : 4; split >= (head_dim == 128 && !shared ? 4 : 1); split /= 2) {
    int64_t most = room / (waves * split);
    if (most > ceil_div(blocks, 4 * split)) most = ceil_div(blocks, 4 * split);
    for (int second = 0; second < (most > 1 ? 2 : 1); ++second) {
      const int64_t chunks = second ? most : 1;
      const double parts = (double)split * (double)chunks, rounds = (double)waves * parts / (double)room;
      double cost = (rounds > 1.0 ? rounds : 1.0) * (6.0 + (double)blocks / parts);
      if (second) cost += 5.0 + (double)(batch * rows * kv_heads * chunks * head_dim) * 8.0 / 9.8e6;
      if (cost < least) {
        least = cost;
        l.split = split;
        l.chunks = (int)chunks;
      }
    }
  }
  return l;
}

template <typename T, int D>
int launch_attention(AttentionArgs& a, const Layout& l, int64_t batch, unsigned grid, hipStream_t stream) {
  const dim3 blocks(grid), threads((unsigned)(l.split * l.rows * 64));
  if (l.wave_rows == 16) {
    if (l.split == 8)
      hipLaunchKernelGGL((cached_attention_kernel<T, D, 8>), blocks, threads, 0, stream, a);
    else
      hipLaunchKernelGGL((cached_attention_kernel<T, D, 4>), blocks, threads, 0, stream, a);
  } else if constexpr (D == 64) {
    if (l.split == 1)
      hipLaunchKernelGGL((chunk_attention_kernel<T, D, 1, 1>), blocks, threads, 0, stream, a);
    else if (l.split == 2)
      hipLaunchKernelGGL((chunk_attention_kernel<T, D, 2, 1>), blocks, threads, 0, stream, a);
    else
      hipLaunchKernelGGL((chunk_attention_kernel<T, D, 4, 1>), blocks, threads, 0, stream, a);
  } else {
    if (l.rows == 1)
      hipLaunchKernelGGL((chunk_attention_kernel<T, D, 4, 1>), blocks, threads, 0, stream, a);
    else if (l.split == 2)
      hipLaunchKernelGGL((chunk_attention_kernel<T, D, 2, 4>), blocks, threads, 0, stream, a);
    else
      hipLaunchKernelGGL((chunk_attention_kernel<T, D, 1, 4>), blocks, threads, 0, stream, a);
  }
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
      (l.chunks > 1 && batch * seq_len * heads > most * 8 - 8))  // the merge, four rows a workgroup
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
  a.row_groups = (uint32_t)l.row_groups;
  a.batch = (uint32_t)batch;
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
