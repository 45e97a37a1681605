// Low-rank adapters of many requests beside a shared projection, for gfx950 (CDNA4).
//
//   y[b, s] = base[b, s] + scale_a (x[b, s] down_a^T) up_a^T,   a = index[b]
//
// Two products a token: h = down x (rank x in) and up h (out x rank), both with the
// adapter's weights as rows and 16 tokens as columns of 16 x 16 x 32 products.  A lane
// then holds, of its token's h, four numbers a tile of 16 rows; the rows of `down` are
// dealt to the tiles so that two tiles give a lane eight neighbouring ones, which is its
// part of the second product's operand: h never leaves its registers.  The rows of `up`
// are dealt so that a lane ends with 16 neighbouring outputs of its token.
//
// h is fp32.  It enters the second product as the sum of two 16-bit numbers, off by
// 2^-16 (bf16) or 2^-22 (fp16) of itself: one number's 2^-9 would be as much as the
// output's own rounding.  A token's h is taken in a power of two of its own, its largest
// below 2^15, so that fp16 reaches.
//
// Many tokens are bound by x, base and y: a wave does both products of its tokens (fused).
// Few tokens are bound by the adapters' bytes, and a wave a token would leave most of
// the chip idle: one launch shares `in` among workgroups and leaves partial sums of h,
// another adds them up in order and shares `out`.

#include <type_traits>

#include "decode_common.hpp"

namespace sah {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kGroup = 64;  // outputs of a wave at a time
constexpr int kMaxRank = 128;
constexpr int kFusedTiles = 2;  // tiles of 16 tokens of a workgroup that does both products

struct LowRankArgs {
  const void* x;
  const void* base;
  const void* down;        // [adapters, rank, in]
  const void* up;          // [adapters, out, rank]
  const float* scales;     // [adapters] or null
  const int32_t* ranks;    // [adapters] or null
  const int32_t* indices;  // [batch]
  const int32_t* counts;   // [batch] or null
  void* y;
  float* partial;          // [parts][tiles][tiles of rank][64][4]
  int64_t x_sb, x_ss, p_sb, p_ss, y_sb, y_ss;
  int64_t in, out, seq, adapters, rank;
  int64_t tiles_of_seq;    // of 16 (fused: 16 TT) tokens
  int64_t tiles;
  int parts, steps_of_part;
};

// What a sequence's adapter asks for; used == 0: none.
struct Adapter {
  int64_t index;
  int used;        // rows of down, a multiple of 8
  int64_t count;   // tokens that it is added to
};
__device__ __forceinline__ Adapter adapter_of(const LowRankArgs& a, int64_t b) {
  Adapter it{0, 0, 0};
  const int64_t index = a.indices[b];
  if (index < 0 || index >= a.adapters) return it;
  int64_t rank = a.rank;
  if (a.ranks != nullptr) {
    const int64_t asked = ((int64_t)a.ranks[index] + 7) / 8 * 8;
    rank = asked < rank ? asked : rank;
  }
  int64_t count = a.counts != nullptr ? (int64_t)a.counts[b] : a.seq;
  if (count > a.seq) count = a.seq;
  if (rank <= 0 || count <= 0) return it;
  it.index = index;
  it.used = (int)rank;
  it.count = count;
  return it;
}

// NP pairs of rank tiles; 0: a single tile.
template <int NP>
constexpr int kTiles = NP == 0 ? 1 : 2 * NP;

// Row of `down` at row m of tile t; rows from `used` on read row 0, and their h is
// taken as 0.
template <int NP>
__device__ __forceinline__ int down_row(int t, int m, int used) {
  const int row = NP == 0 ? m : 32 * (t / 2) + 8 * (m / 4) + 4 * (t & 1) + (m & 3);
  return row < used ? row : 0;
}
// h += down x over inputs [32 first, 32 last).  x: each tile's token row; w: each tile's
// row of down.
template <typename T, int NP, int TT, int UNROLL>
__device__ __forceinline__ void shrink(const T* const (&x)[TT], const T* const (&w)[kTiles<NP>], int64_t in,
                                       int64_t first, int64_t last, f32x4 (&h)[TT][kTiles<NP>]) {
  typedef typename Vec8<T>::type V8;
  constexpr int N = kTiles<NP>;
  const int quarter = (threadIdx.x & 63) >> 4;
  const int64_t whole = in / 32 < last ? in / 32 : last;  // steps without a ragged end
  int64_t step = first;
  for (; step + UNROLL <= whole; step += UNROLL) {
    V8 xs[UNROLL][TT], ws[UNROLL][N];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int64_t k = (step + u) * 32 + quarter * 8;
#pragma unroll
      for (int i = 0; i < TT; ++i) xs[u][i] = *reinterpret_cast<const V8*>(x[i] + k);
#pragma unroll
      for (int t = 0; t < N; ++t) ws[u][t] = *reinterpret_cast<const V8*>(w[t] + k);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int t = 0; t < N; ++t)
#pragma unroll
        for (int i = 0; i < TT; ++i) h[i][t] = mfma16(ws[u][t], xs[u][i], h[i][t]);
  }
  for (; step < last; ++step) {
    const int64_t k = step * 32 + quarter * 8;
    const bool there = k < in;
    V8 xs[TT];
#pragma unroll
    for (int i = 0; i < TT; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) xs[i][e] = (T)0.0f;
      if (there) xs[i] = *reinterpret_cast<const V8*>(x[i] + k);
    }
#pragma unroll
    for (int t = 0; t < N; ++t) {
      V8 ws;
#pragma unroll
      for (int e = 0; e < 8; ++e) ws[e] = (T)0.0f;
      if (there) ws = *reinterpret_cast<const V8*>(w[t] + k);
#pragma unroll
      for (int i = 0; i < TT; ++i) h[i][t] = mfma16(ws, xs[i], h[i][t]);
    }
  }
}

// A token's h, times 2^power, as the second product's operands.
template <typename T, int NP>
struct Hidden {
  typedef typename Vec8<T>::type V8;
  V8 high[NP == 0 ? 1 : NP];  // one tile: high and low in one operand
  V8 low[NP == 0 ? 1 : NP];
  int power;
};

template <typename T>
__device__ __forceinline__ void split_number(float v, T& high, T& low) {
  high = from_f32<T>(v);
  const float rest = v - to_f32(high);
  low = from_f32<T>(fabsf(to_f32(high)) < INFINITY ? rest : 0.0f);
}

template <typename T, int NP>
__device__ __forceinline__ Hidden<T, NP> make_hidden(const f32x4 (&h)[kTiles<NP>], int used) {
  constexpr int N = kTiles<NP>;
  const int quarter = (threadIdx.x & 63) >> 4;
  float v[N][4];
  float largest = 0.0f;
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = NP == 0 ? 4 * quarter + i : 32 * (t / 2) + 8 * quarter + 4 * (t & 1) + i;
      v[t][i] = row < used ? h[t][i] : 0.0f;
      largest = fmaxf(largest, fabsf(v[t][i]));
    }
  largest = fmaxf(largest, __shfl_xor(largest, 16));
  largest = fmaxf(largest, __shfl_xor(largest, 32));
  int power = 0;  // the largest comes to lie in [2^14, 2^15)
  if (largest > 0.0f && largest < INFINITY) power = 15 - __builtin_amdgcn_frexp_expf(largest);
  Hidden<T, NP> out;
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      T high, low;
      split_number<T>(ldexpf(v[t][i], power), high, low);
      if constexpr (NP == 0) {
        out.high[0][i] = high;
        out.high[0][4 + i] = low;
      } else {
        out.high[t / 2][4 * (t & 1) + i] = high;
        out.low[t / 2][4 * (t & 1) + i] = low;
      }
    }
  out.power = power;
  return out;
}

// What outputs [64 group, 64 group + 64) of a wave's tokens need: the rows of up, and
// base.  A lane's token is column lane % 16; its outputs 8 (lane / 16) + 0..7 of either
// half of the group, so that an access takes 64 bytes of a token.  Places outside the tensors read the nearest inside.
template <typename T, int NP, int TT>
struct Group {
  typedef typename Vec8<T>::type V8;
  typedef typename Vec8<T>::half_type V4;
  static constexpr int S = NP == 0 ? 1 : NP;
  V8 held[TT][2];
  V8 w[4][S];

  __device__ __forceinline__ void load(const T* up, int64_t rank, int64_t out, int used, int64_t group,
                                       const T* const (&base)[TT]) {
    const int lane = threadIdx.x & 63, quarter = lane >> 4, m = lane & 15;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int64_t asked = group * kGroup + 32 * p + 8 * quarter;
      const int64_t at = asked < out ? asked : out - 8;
#pragma unroll
      for (int i = 0; i < TT; ++i) held[i][p] = *reinterpret_cast<const V8*>(base[i] + at);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int64_t asked = group * kGroup + 32 * (t / 2) + 8 * (m / 4) + 4 * (t & 1) + (m & 3);
      const T* row = up + (asked < out ? asked : out - 1) * rank;
      if constexpr (NP == 0) {
        const V4 half = *reinterpret_cast<const V4*>(row + (4 * quarter < used ? 4 * quarter : 0));
        w[t][0] = __builtin_shufflevector(half, half, 0, 1, 2, 3, 0, 1, 2, 3);
      } else {
#pragma unroll
        for (int s = 0; s < NP; ++s) {
          const int at = 32 * s + 8 * quarter;
          w[t][s] = *reinterpret_cast<const V8*>(row + (at < used ? at : 0));
        }
      }
    }
  }

  // base + scale (up h).  Tokens that the adapter is not added to take base as it is,
  // tokens behind the sequence nothing.
  __device__ __forceinline__ void finish(int64_t out, int64_t group, float scale, const Hidden<T, NP> (&h)[TT],
                                         T* const (&y)[TT], const bool (&live)[TT], const bool (&added)[TT]) {
    const int quarter = (threadIdx.x & 63) >> 4;
    f32x4 sums[TT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < TT; ++i) sums[i][t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < TT; ++i) {
          if constexpr (NP != 0) sums[i][t] = mfma16(w[t][s], h[i].low[s], sums[i][t]);
          sums[i][t] = mfma16(w[t][s], h[i].high[s], sums[i][t]);
        }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int64_t at = group * kGroup + 32 * p + 8 * quarter;
#pragma unroll
      for (int i = 0; i < TT; ++i)
        if (live[i] && at < out) {
          V8 sum = held[i][p];
          if (added[i]) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              sum[e] = from_f32<T>(fmaf(scale, ldexpf(sums[i][2 * p + e / 4][e % 4], -h[i].power), to_f32(held[i][p][e])));
          }
          *reinterpret_cast<V8*>(y[i] + at) = sum;
        }
    }
  }
};

// Tokens without an adapter, groups first, first + step, ..: base as it is.
template <typename T, int TT, int DEEP>
__device__ __forceinline__ void copy_groups(int64_t out, int64_t first, int64_t groups, int64_t step,
                                            const T* const (&base)[TT], T* const (&y)[TT], const bool (&live)[TT]) {
  const int quarter = (threadIdx.x & 63) >> 4;
  for (int64_t g = first; g < groups; g += DEEP * step) {
    u32x4 held[DEEP][TT][2];
#pragma unroll
    for (int d = 0; d < DEEP; ++d)
#pragma unroll
      for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int64_t at = (g + d * step) * kGroup + 32 * p + 8 * quarter;
          held[d][i][p] = load16(base[i] + (at < out ? at : out - 8));
        }
#pragma unroll
    for (int d = 0; d < DEEP; ++d)
#pragma unroll
      for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int64_t at = (g + d * step) * kGroup + 32 * p + 8 * quarter;
          if (live[i] && at < out && y[i] != base[i]) store16(y[i] + at, held[d][i][p]);
        }
  }
}

template <typename T, int TT>
struct Tokens {
  const T* x[TT];
  const T* base[TT];
  T* y[TT];
  bool live[TT], added[TT];
};
// A lane's tokens `first` + 16 i + lane % 16 (behind the sequence: its last one, not live).
template <typename T, int TT>
__device__ __forceinline__ Tokens<T, TT> tokens_of(const LowRankArgs& a, int64_t b, int64_t first, int64_t count) {
  Tokens<T, TT> out;
#pragma unroll
  for (int i = 0; i < TT; ++i) {
    const int64_t token = first + 16 * i + (threadIdx.x & 15);
    const int64_t s = token < a.seq ? token : a.seq - 1;
    out.live[i] = token < a.seq;
    out.added[i] = token < count;
    out.x[i] = static_cast<const T*>(a.x) + b * a.x_sb + s * a.x_ss;
    out.base[i] = static_cast<const T*>(a.base) + b * a.p_sb + s * a.p_ss;
    out.y[i] = static_cast<T*>(a.y) + b * a.y_sb + s * a.y_ss;
  }
  return out;
}

// A workgroup takes 16 TT tokens.  Its waves share `in` for h, add their sums up in order
// through LDS, and share `out`, the next group's loads under way while one is worked on.
template <typename T, int NP, int TT>
__global__ __launch_bounds__(kThreads) void low_rank_fused_kernel(const LowRankArgs a) {
  constexpr int N = kTiles<NP>;
  __shared__ f32x4 sums[kWaves][TT * N][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tile = blockIdx.x;
  const int64_t b = tile / a.tiles_of_seq;
  const int64_t first = (tile - b * a.tiles_of_seq) * (16 * TT);
  const Adapter it = adapter_of(a, b);
  const Tokens<T, TT> tokens = tokens_of<T, TT>(a, b, first, it.count);
  const int64_t groups = (a.out + kGroup - 1) / kGroup;
  if (it.used == 0 || first >= it.count) {
    copy_groups<T, TT, 4>(a.out, wave, groups, kWaves, tokens.base, tokens.y, tokens.live);
    return;
  }
  const T* down = static_cast<const T*>(a.down) + it.index * a.rank * a.in;
  const T* w[N];
#pragma unroll
  for (int t = 0; t < N; ++t) w[t] = down + (int64_t)down_row<NP>(t, lane & 15, it.used) * a.in;
  f32x4 h[TT][N];
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int t = 0; t < N; ++t) h[i][t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  const int64_t steps = (a.in + 31) / 32, share = (steps + kWaves - 1) / kWaves;
  const int64_t to = (wave + 1) * share;
  shrink<T, NP, TT, (N + TT > 6 ? 2 : 4)>(tokens.x, w, a.in, wave * share, to < steps ? to : steps, h);
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int t = 0; t < N; ++t) sums[wave][i * N + t][lane] = h[i][t];
  __syncthreads();
  Hidden<T, NP> hidden[TT];
#pragma unroll
  for (int i = 0; i < TT; ++i) {
#pragma unroll
    for (int t = 0; t < N; ++t) {
      h[i][t] = sums[0][i * N + t][lane];
#pragma unroll
      for (int k = 1; k < kWaves; ++k) h[i][t] += sums[k][i * N + t][lane];
    }
    hidden[i] = make_hidden<T, NP>(h[i], it.used);
  }
  const float scale = a.scales != nullptr ? a.scales[it.index] : 1.0f;
  const T* up = static_cast<const T*>(a.up) + it.index * a.out * a.rank;
  Group<T, NP, TT> buffer[2];
  int64_t g = wave;
  if (g < groups) buffer[0].load(up, a.rank, a.out, it.used, g, tokens.base);
  while (g < groups) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (g >= groups) break;
      if (g + kWaves < groups) buffer[1 - k].load(up, a.rank, a.out, it.used, g + kWaves, tokens.base);
      buffer[k].finish(a.out, g, scale, hidden, tokens.y, tokens.live, tokens.added);
      g += kWaves;
    }
  }
}

// Partial sums of h: workgroup (tile, part) takes the part's steps, its waves in turn.
template <typename T, int NP>
__global__ __launch_bounds__(kThreads) void low_rank_shrink_kernel(const LowRankArgs a) {
  constexpr int N = kTiles<NP>;
  __shared__ f32x4 sums[kWaves - 1][N][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tile = blockIdx.x / (uint32_t)a.parts;
  const int part = (int)(blockIdx.x % (uint32_t)a.parts);
  const int64_t b = tile / a.tiles_of_seq;
  const int64_t first = (tile - b * a.tiles_of_seq) * 16;
  const Adapter it = adapter_of(a, b);
  if (it.used == 0 || first >= it.count) return;
  const Tokens<T, 1> tokens = tokens_of<T, 1>(a, b, first, it.count);
  const T* down = static_cast<const T*>(a.down) + it.index * a.rank * a.in;
  const T* w[N];
#pragma unroll
  for (int t = 0; t < N; ++t) w[t] = down + (int64_t)down_row<NP>(t, lane & 15, it.used) * a.in;
  f32x4 h[1][N];
#pragma unroll
  for (int t = 0; t < N; ++t) h[0][t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  const int64_t steps = (a.in + 31) / 32;
  const int64_t from = (int64_t)part * a.steps_of_part;
  const int64_t to = from + a.steps_of_part < steps ? from + a.steps_of_part : steps;
  const int64_t share = (to - from + kWaves - 1) / kWaves;
  const int64_t mine = from + wave * share;
  shrink<T, NP, 1, (N > 4 ? 2 : 4)>(tokens.x, w, a.in, mine, mine + share < to ? mine + share : to, h);
  if (wave != 0) {
#pragma unroll
    for (int t = 0; t < N; ++t) sums[wave - 1][t][lane] = h[0][t];
  }
  __syncthreads();
  if (wave != 0) return;
  f32x4* partial = reinterpret_cast<f32x4*>(a.partial) + ((int64_t)part * a.tiles + tile) * N * 64;
#pragma unroll
  for (int t = 0; t < N; ++t) {
    f32x4 sum = h[0][t];
#pragma unroll
    for (int k = 0; k < kWaves - 1; ++k) sum += sums[k][t][lane];
    partial[t * 64 + lane] = sum;
  }
}

template <typename T, int NP>
__global__ __launch_bounds__(kThreads) void low_rank_expand_kernel(const LowRankArgs a) {
  constexpr int N = kTiles<NP>;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t groups = (uint32_t)((a.out + kGroup - 1) / kGroup);
  const uint32_t workgroups = (groups + kWaves - 1) / kWaves;  // of a tile
  const int64_t tile = blockIdx.x / workgroups;
  const int64_t group = (int64_t)(blockIdx.x % workgroups) * kWaves + wave;
  if (group >= groups) return;
  const int64_t b = tile / a.tiles_of_seq;
  const int64_t first = (tile - b * a.tiles_of_seq) * 16;
  const Adapter it = adapter_of(a, b);
  const Tokens<T, 1> tokens = tokens_of<T, 1>(a, b, first, it.count);
  if (it.used == 0 || first >= it.count) {
    copy_groups<T, 1, 1>(a.out, group, group + 1, 1, tokens.base, tokens.y, tokens.live);
    return;
  }
  Group<T, NP, 1> data;
  data.load(static_cast<const T*>(a.up) + it.index * a.out * a.rank, a.rank, a.out, it.used, group, tokens.base);
  f32x4 h[N];
#pragma unroll
  for (int t = 0; t < N; ++t) h[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  if (tokens.added[0]) {
    const f32x4* partial = reinterpret_cast<const f32x4*>(a.partial) + tile * N * 64 + lane;
    // (of tiles that no row of down fills, what is read is not used)
#pragma unroll 4
    for (int p = 0; p < a.parts; ++p)
#pragma unroll
      for (int t = 0; t < N; ++t) h[t] += partial[(int64_t)p * a.tiles * N * 64 + t * 64];
  }
  const float scale = a.scales != nullptr ? a.scales[it.index] : 1.0f;
  const Hidden<T, NP> hidden[1] = {make_hidden<T, NP>(h, it.used)};
  data.finish(a.out, group, scale, hidden, tokens.y, tokens.live, tokens.added);
}

// How a call is launched.
struct Plan {
  bool fused;
  int tokens;              // of a tile
  int64_t tiles_of_seq, tiles;
  int parts, steps_of_part;
  int rank_tiles;
  size_t bytes;
};
constexpr int64_t kManyTiles = 1024;  // of 16 tokens: from here on one launch does both products

Plan plan_of(int64_t batch, int64_t seq, int64_t in, int64_t rank) {
  Plan p{};
  p.rank_tiles = rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8;
  p.tokens = 16;
  p.tiles_of_seq = ceil_div(seq, 16);
  p.tiles = batch * p.tiles_of_seq;
  p.fused = p.tiles >= kManyTiles;
  if (p.fused) {
    p.tokens = 16 * kFusedTiles;
    p.tiles_of_seq = ceil_div(seq, p.tokens);
    p.tiles = batch * p.tiles_of_seq;
    return p;
  }
  const int64_t steps = ceil_div(in, 32);
  int64_t parts = ceil_div(1024, p.tiles);
  const int64_t most = ceil_div(steps, 4 * kWaves);
  if (parts > most) parts = most;
  p.steps_of_part = (int)ceil_div(steps, parts);
  p.parts = (int)ceil_div(steps, p.steps_of_part);
  p.bytes = (size_t)(p.parts * p.tiles * p.rank_tiles) * 64 * sizeof(f32x4);
  return p;
}

template <typename T, int NP>
int launch(const LowRankArgs& a, const Plan& p, hipStream_t stream) {
  if (p.fused) {
    hipLaunchKernelGGL((low_rank_fused_kernel<T, NP, kFusedTiles>), dim3((unsigned)p.tiles), dim3(kThreads), 0, stream, a);
    return check_hip(hipGetLastError(), "low-rank adapters launch");
  }
  hipLaunchKernelGGL((low_rank_shrink_kernel<T, NP>), dim3((unsigned)(p.tiles * p.parts)), dim3(kThreads), 0, stream, a);
  const int status = check_hip(hipGetLastError(), "low-rank adapters launch");
  if (status != SAH_OK) return status;
  const int64_t workgroups = ceil_div(ceil_div(a.out, kGroup), kWaves);
  hipLaunchKernelGGL((low_rank_expand_kernel<T, NP>), dim3((unsigned)(p.tiles * workgroups)), dim3(kThreads), 0, stream,
                     a);
  return check_hip(hipGetLastError(), "low-rank adapters launch");
}

template <typename T>
int launch_rank(const LowRankArgs& a, const Plan& p, hipStream_t stream) {
  switch (p.rank_tiles) {
    case 1: return launch<T, 0>(a, p, stream);
    case 2: return launch<T, 1>(a, p, stream);
    case 4: return launch<T, 2>(a, p, stream);
    default: return launch<T, 4>(a, p, stream);
  }
}

bool sizes_ok(int64_t batch, int64_t seq, int64_t in, int64_t out, int64_t rank) {
  return batch >= 0 && batch <= INT32_MAX && seq >= 0 && seq <= INT32_MAX && in > 0 && in % 8 == 0 && in <= (1 << 24) &&
         out > 0 && out % 8 == 0 && out <= (1 << 24) && rank > 0 && rank % 8 == 0 && rank <= kMaxRank;
}

}  // namespace
}  // namespace sah

using namespace sah;

extern "C" size_t sah_low_rank_adapters_workspace_bytes(int64_t batch, int64_t seq_len, int64_t in_features,
                                                        int64_t out_features, int64_t rank) {
  if (!sizes_ok(batch, seq_len, in_features, out_features, rank) || batch == 0 || seq_len == 0) return 0;
  return plan_of(batch, seq_len, in_features, rank).bytes;
}

extern "C" int sah_low_rank_adapters(const void* x, const void* base, const void* down, const void* up,
                                     const float* scales, const int32_t* ranks, const int32_t* indices,
                                     const int32_t* counts, void* y, int64_t batch, int64_t seq_len,
                                     int64_t in_features, int64_t out_features, int64_t adapters, int64_t rank,
                                     int64_t x_stride_b, int64_t x_stride_s, int64_t base_stride_b,
                                     int64_t base_stride_s, int64_t y_stride_b, int64_t y_stride_s, int dtype,
                                     void* workspace, size_t workspace_bytes, sah_stream_t stream) {
  const char* what = "sah_low_rank_adapters";
  if (dtype != SAH_DTYPE_BF16 && dtype != SAH_DTYPE_F16)
    return fail(SAH_ERR_UNSUPPORTED, "%s: dtype %d is not bf16 or f16", what, dtype);
  if (batch < 0 || batch > INT32_MAX || seq_len < 0 || seq_len > INT32_MAX || in_features <= 0 || out_features <= 0 ||
      rank <= 0 || adapters < 0 || adapters > INT32_MAX)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: bad sizes", what);
  if (!sizes_ok(batch, seq_len, in_features, out_features, rank))
    return fail(SAH_ERR_UNSUPPORTED, "%s: in, out and rank must be multiples of 8, rank at most %d", what, kMaxRank);
  if (batch == 0 || seq_len == 0) return SAH_OK;
  if (x == nullptr || base == nullptr || y == nullptr || indices == nullptr ||
      (adapters != 0 && (down == nullptr || up == nullptr)))
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", what);
  const void* tensors[] = {x, base, down, up, y};
  for (const void* p : tensors)
    if (!aligned16(p)) return fail(SAH_ERR_INVALID_ARGUMENT, "%s: tensors must be 16-byte aligned", what);
  if (((reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(ranks) |
        reinterpret_cast<uintptr_t>(indices) | reinterpret_cast<uintptr_t>(counts)) & 3u) != 0)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: scales, ranks, indices and counts must be 4-byte aligned", what);
  const int64_t strides[] = {x_stride_b, x_stride_s, base_stride_b, base_stride_s, y_stride_b, y_stride_s};
  for (int64_t v : strides)
    if (v % 8 != 0) return fail(SAH_ERR_INVALID_ARGUMENT, "%s: strides must be multiples of 8 elements", what);
  // rows of y one after the other, whichever of the two axes is the outer one
  const bool apart =
      (seq_len == 1 && (batch == 1 || y_stride_b >= out_features)) ||
      (seq_len > 1 && batch == 1 && y_stride_s >= out_features) ||
      (seq_len > 1 && batch > 1 && y_stride_s >= out_features && y_stride_b >= (seq_len - 1) * y_stride_s + out_features) ||
      (seq_len > 1 && batch > 1 && y_stride_b >= out_features && y_stride_s >= (batch - 1) * y_stride_b + out_features);
  if (!apart) return fail(SAH_ERR_INVALID_ARGUMENT, "%s: rows of y overlap", what);
  const int64_t tiles = batch * ceil_div(seq_len, 16);
  const int64_t most = (int64_t)(UINT32_MAX / kThreads);
  if (tiles > most / ceil_div(out_features, kGroup))
    return fail(SAH_ERR_UNSUPPORTED, "%s: too many tokens for one launch", what);
  const Plan plan = plan_of(batch, seq_len, in_features, rank);
  if (plan.bytes != 0 && (workspace == nullptr || workspace_bytes < plan.bytes))
    return fail(SAH_ERR_WORKSPACE, "%s: workspace of %zu bytes, needs %zu", what, workspace == nullptr ? 0 : workspace_bytes,
                plan.bytes);
  if (plan.bytes != 0 && !aligned16(workspace))
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", what);
  LowRankArgs a{};
  a.x = x;
  a.base = base;
  a.down = down;
  a.up = up;
  a.scales = scales;
  a.ranks = ranks;
  a.indices = indices;
  a.counts = counts;
  a.y = y;
  a.partial = static_cast<float*>(workspace);
  a.x_sb = x_stride_b;
  a.x_ss = x_stride_s;
  a.p_sb = base_stride_b;
  a.p_ss = base_stride_s;
  a.y_sb = y_stride_b;
  a.y_ss = y_stride_s;
  a.in = in_features;
  a.out = out_features;
  a.seq = seq_len;
  a.adapters = adapters;
  a.rank = rank;
  a.tiles_of_seq = plan.tiles_of_seq;
  a.tiles = plan.tiles;
  a.parts = plan.parts;
  a.steps_of_part = plan.steps_of_part;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return dtype == SAH_DTYPE_BF16 ? launch_rank<bf16>(a, plan, s) : launch_rank<f16>(a, plan, s);
}
