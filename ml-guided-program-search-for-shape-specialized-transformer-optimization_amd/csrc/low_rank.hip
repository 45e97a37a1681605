// Low-rank adapters of many requests beside a shared projection, for gfx950 (CDNA4).
//
//   y[b, s] = base[b, s] + scale_a (x[b, s] down_a^T) up_a^T,   a = index[b]
//
// Two products a token, h = down x (rank x in) and up h (out x rank), on 16 x 16 x 32
// products whose operands hold 16 bytes of row lane % 16 a lane.  The rows of `down` are
// dealt to tiles of 16 so that two tiles leave a lane with eight neighbouring numbers of
// its token's h, which is its part of the second product's operand: h never leaves its
// registers.
//
// Memory is read in another order than the operands': four lanes in a row take 64 bytes of
// a row (the address units work on four lanes at a time, and in the operands' order, one
// row a lane, they were the bound: 91% busy).  Rows of x and `down` change places within
// four lanes in registers, rows of `up` through the wave's own part of LDS, and the second
// product's columns are outputs 4 n + t, so that 16 lanes take 128 bytes of base and y.
//
// h is fp32.  It enters the second product as the sum of three bf16 numbers, off by 2^-24
// of itself as fp32 is, or of two fp16 numbers, off by 2^-22: with one number its 2^-8 would
// be as much as the output's own rounding, and with two bf16 numbers some 0.2% of the
// outputs are rounded another way (34816 tokens 4096 -> 4096, rank 64, 208 us with three
// numbers, 204 with two, rank 128, 339 and 320).  A token's h is taken in a power of two of
// its own, its largest below 2^15, so that fp16 reaches.
//
// Few tokens are bound by the adapters' bytes and by latency, and a workgroup a token would
// leave most of the chip idle: one launch shares `in` among workgroups and leaves partial
// sums of h, another adds them up in order and shares `out`.  Many tokens are bound by x,
// base and y: a workgroup does both products of 32 tokens, and there is no workspace.  Nor
// is there for few tokens of short inputs, where latency and launches are all there is.
//   2 x 20001 tokens (ragged), 1024 -> 4096, rank 32 (697 MB, 142 us at a large copy's
//   rate): 139 us; some 10 more through the caches, 40 in the operands' order as well
//   64 tokens, 4096 -> 4096, an adapter each of rank 64 (33 MB, 7 us): 7.3 + 7.9 us
//   1 token, 1024 -> 4096, rank 16: 5.7 us

#include <type_traits>

#include "decode_common.hpp"

namespace sah {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kSlab = 128;  // inputs that a wave takes at a time
constexpr int kGroup = 64;  // outputs
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
  int64_t tiles_of_seq;    // of 16 (fused: 16 kFusedTiles) tokens
  int64_t tiles;
  int parts, slabs_of_part, groups_of_wave;
};

// What a sequence's adapter asks for; used == 0: none.
struct Adapter {
  int64_t index;
  int used;        // rows of down, a multiple of 8
  float scale;
  int64_t count;   // tokens that it is added to
};
__device__ __forceinline__ Adapter adapter_of(const LowRankArgs& a, int64_t b) {
  Adapter it{0, 0, 1.0f, 0};
  const int64_t index = a.indices[b];
  if (index < 0 || index >= a.adapters) return it;
  int64_t rank = a.rank;
  if (a.ranks != nullptr) {
    const int64_t asked = ((int64_t)a.ranks[index] + 7) / 8 * 8;
    rank = asked < rank ? asked : rank;
  }
  if (a.scales != nullptr) it.scale = a.scales[index];
  int64_t count = a.counts != nullptr ? (int64_t)a.counts[b] : a.seq;
  if (count > a.seq) count = a.seq;
  if (rank <= 0 || count <= 0) return it;
  it.index = index;
  it.used = (int)rank;
  it.count = count;
  return it;
}

// Lane l: quarter l / 16 of the operands' 16-byte parts, row (or column) l % 16; four by
// four of these are corner l % 16 / 4 and side l % 4.
__device__ __forceinline__ int quarter_of() { return (threadIdx.x & 63) >> 4; }
__device__ __forceinline__ int corner_of() { return (threadIdx.x & 15) >> 2; }
__device__ __forceinline__ int side_of() { return threadIdx.x & 3; }

// Rows of `down` in tiles of 16, S pairs of them: row m of tile t is row 32 (t / 2) + 8 (m /
// 4) + 4 (t % 2) + m % 4, so a lane's rows of a pair are 32 s + 8 quarter + 0..7.

// lane ^ 1 (0xB1) or lane ^ 2 (0x4E), of every lane: not for a branch that some take.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}

// Turns four registers' parts in four lanes: register j of lane i becomes register i of
// lane j.
template <typename V8>
__device__ __forceinline__ void turn_in_four(V8 (&v)[4]) {
  u32x4 r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = __builtin_bit_cast(u32x4, v[j]);
  const bool odd = (threadIdx.x & 1) != 0, high = (threadIdx.x & 2) != 0;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const uint32_t a = r[j][d], b = r[j + 1][d], other_a = dpp<0xB1>(a), other_b = dpp<0xB1>(b);
      r[j][d] = odd ? other_b : a;
      r[j + 1][d] = odd ? b : other_a;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t a = r[j][d], b = r[j + 2][d], other_a = dpp<0x4E>(a), other_b = dpp<0x4E>(b);
      r[j][d] = high ? other_b : a;
      r[j + 2][d] = high ? b : other_a;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = __builtin_bit_cast(V8, r[j]);
}

// h += down x over one slab of 128 inputs.  An access takes 256 bytes of four rows;
// turned, register i of a lane holds its row's inputs 32 quarter + 8 i + 0..7 of the slab,
// which is step i of the product.  x: the lane's rows 4 corner + 0..3 of each tile; w_first:
// its first row of down in each pair.
template <typename T, int S, int TT, bool WHOLE>
__device__ __forceinline__ void shrink_slab(const T* const (&x)[TT][4], const T* down, const int64_t (&w_first)[S],
                                            int64_t in, int64_t slab, f32x4 (&h)[TT][2 * S]) {
  typedef typename Vec8<T>::type V8;
  const int64_t at = slab * kSlab + 32 * quarter_of() + 8 * side_of();
  const bool there = WHOLE || at < in;
  const int64_t k = there ? at : 0;
  V8 xs[TT][4], ws[2 * S][4];
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) xs[i][j] = *reinterpret_cast<const V8*>(x[i][j] + k);
#pragma unroll
  for (int t = 0; t < 2 * S; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      ws[t][j] = *reinterpret_cast<const V8*>(down + (4 * (t & 1) + j) * in + (w_first[t / 2] + k));
  if constexpr (!WHOLE) {  // (both, as nothing times what is not there may be NaN)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) xs[i][j][e] = there ? xs[i][j][e] : (T)0.0f;
#pragma unroll
      for (int t = 0; t < 2 * S; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e) ws[t][j][e] = there ? ws[t][j][e] : (T)0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < TT; ++i) turn_in_four(xs[i]);
#pragma unroll
  for (int t = 0; t < 2 * S; ++t) {
    turn_in_four(ws[t]);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < TT; ++i) h[i][t] = mfma16(ws[t][j], xs[i][j], h[i][t]);
  }
}

// Slabs [first, last), the one that the inputs end in by itself.
template <typename T, int S, int TT>
__device__ __forceinline__ void shrink(const T* const (&x)[TT][4], const T* down, const int64_t (&w_first)[S], int64_t in,
                                       int64_t first, int64_t last, f32x4 (&h)[TT][2 * S]) {
  const int64_t whole = in / kSlab < last ? in / kSlab : last;
  int64_t slab = first;
#pragma unroll 1
  for (; slab < whole; ++slab) shrink_slab<T, S, TT, true>(x, down, w_first, in, slab, h);
  if (slab < last) shrink_slab<T, S, TT, false>(x, down, w_first, in, slab, h);
}

// A token's h, times 2^power, as the second product's operands, the largest part first;
// factor: scale / 2^power.
template <typename T, int S>
struct Hidden {
  static constexpr int PARTS = std::is_same<T, bf16>::value ? 3 : 2;
  typedef typename Vec8<T>::type V8;
  V8 part[PARTS][S];
  float factor;
};

template <int PARTS, typename T>
__device__ __forceinline__ void split_number(float v, T (&part)[PARTS]) {
  part[0] = from_f32<T>(v);
  float rest = fabsf(to_f32(part[0])) < INFINITY ? v - to_f32(part[0]) : 0.0f;
#pragma unroll
  for (int i = 1; i < PARTS; ++i) {
    part[i] = from_f32<T>(rest);
    rest -= to_f32(part[i]);
  }
}

template <typename T, int S>
__device__ __forceinline__ Hidden<T, S> make_hidden(const f32x4 (&h)[2 * S], int used, float scale) {
  float v[2 * S][4];
  float largest = 0.0f;
#pragma unroll
  for (int t = 0; t < 2 * S; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[t][i] = 32 * (t / 2) + 8 * quarter_of() < used ? h[t][i] : 0.0f;
      largest = fmaxf(largest, fabsf(v[t][i]));
    }
  largest = fmaxf(largest, __shfl_xor(largest, 16));
  largest = fmaxf(largest, __shfl_xor(largest, 32));
  if (largest == INFINITY) {  // (for a token's four lanes) it is so in any power, and the others keep theirs
    largest = 0.0f;
#pragma unroll
    for (int t = 0; t < 2 * S; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) largest = fmaxf(largest, fabsf(v[t][i]) < INFINITY ? fabsf(v[t][i]) : 0.0f);
    largest = fmaxf(largest, __shfl_xor(largest, 16));
    largest = fmaxf(largest, __shfl_xor(largest, 32));
  }
  // the largest comes to lie in [2^14, 2^15), where fp32 has room for scale / 2^power
  int power = 0;
  if (largest > 0.0f) power = 15 - __builtin_amdgcn_frexp_expf(largest);
  power = power < -100 ? -100 : power > 100 ? 100 : power;
  Hidden<T, S> out;
#pragma unroll
  for (int t = 0; t < 2 * S; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      T part[Hidden<T, S>::PARTS];
      split_number(ldexpf(v[t][i], power), part);
#pragma unroll
      for (int k = 0; k < Hidden<T, S>::PARTS; ++k) out.part[k][t / 2][4 * (t & 1) + i] = part[k];
    }
  out.factor = ldexpf(scale, -power);
  return out;
}

// A wave's tokens as the outputs have them: a lane's are 4 quarter + 0..3 of each tile.
template <typename T, int TT>
struct Tokens {
  const T* base[TT][4];
  T* y[TT][4];
  bool live[TT][4], added[TT][4];
  __device__ Tokens(const LowRankArgs& a, int64_t b, int64_t first, int64_t count) {
#pragma unroll
    for (int i = 0; i < TT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t token = first + 16 * i + 4 * quarter_of() + j;
        const int64_t s = token < a.seq ? token : a.seq - 1;
        live[i][j] = token < a.seq;
        added[i][j] = token < count;
        base[i][j] = static_cast<const T*>(a.base) + b * a.p_sb + s * a.p_ss;
        y[i][j] = static_cast<T*>(a.y) + b * a.y_sb + s * a.y_ss;
      }
  }
};
// The lane's rows of x, tokens 4 corner + 0..3 of each tile.
template <typename T, int TT>
__device__ __forceinline__ void rows_of_x(const LowRankArgs& a, int64_t b, int64_t first, const T* (&x)[TT][4]) {
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t token = first + 16 * i + 4 * corner_of() + j;
      x[i][j] = static_cast<const T*>(a.x) + b * a.x_sb + (token < a.seq ? token : a.seq - 1) * a.x_ss;
    }
}
// The lane's first row of down in each pair (rows from `used` on read the first ones, and
// their h is taken as 0).
template <int S>
__device__ __forceinline__ void rows_of_down(int used, int64_t in, int64_t (&first)[S]) {
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int row = 32 * s + 8 * corner_of();
    first[s] = (row < used ? row : 0) * in;
  }
}

// The wave's part of LDS for a group's rows of up: an operand tile of 1 KiB for each
// step s and t, the tiles 64 bytes apart from each other's banks.
template <int S>
struct UpStage {
  static constexpr int TILE = 1024 + 64;
  char bytes[4 * S * TILE];
};

// Four outputs of base or y, past the caches where PAST.
template <bool PAST, typename V4, typename T>
__device__ __forceinline__ V4 fetch(const T* p) {
  return PAST ? __builtin_nontemporal_load(reinterpret_cast<const V4*>(p)) : *reinterpret_cast<const V4*>(p);
}
template <bool PAST, typename V4, typename T>
__device__ __forceinline__ void put(T* p, V4 v) {
  if (PAST)
    __builtin_nontemporal_store(v, reinterpret_cast<V4*>(p));
  else
    *reinterpret_cast<V4*>(p) = v;
}

// What a group's outputs of a wave's tokens need: the 64 rows of up, and base.  Places
// behind `out` read the nearest inside.
template <typename T, int S, int TT, bool PAST = false>
struct Group {
  typedef typename Vec8<T>::type V8;
  typedef typename Vec8<T>::half_type V4;
  V4 held[TT][4];
  V8 w[S][4];  // 64 bytes of 16 rows each, in memory's order

  __device__ __forceinline__ void load(const T* up, int64_t rank, int64_t out, int used, int64_t group,
                                       const Tokens<T, TT>& tokens) {
    const int lane = threadIdx.x & 63;
    const int first = (int)group * kGroup, last = (int)out;
    const int asked = first + 4 * (lane & 15);
    const int column = asked < last ? asked : last - 4;
#pragma unroll
    for (int i = 0; i < TT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) held[i][j] = fetch<PAST, V4>(tokens.base[i][j] + column);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = first + 16 * r + lane / 4;
      const T* from = up + (row < last ? row : last - 1) * rank;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int chunk = 32 * s + 8 * (lane & 3);
        w[s][r] = *reinterpret_cast<const V8*>(from + (chunk < used ? chunk : 0));
      }
    }
  }

  static __device__ __forceinline__ char* place_of(UpStage<S>& lds, int s, int r) {
    const int lane = threadIdx.x & 63, row = 16 * r + lane / 4;
    return lds.bytes + (s * 4 + row % 4) * UpStage<S>::TILE + (row / 4) * 64 + (lane & 3) * 16;
  }

  // Zeros for the directions from `used` on, which no group's rows replace: h is 0 there, and
  // 0 times what load() reads in their place may be NaN.
  static __device__ __forceinline__ void clear(UpStage<S>& lds, int used) {
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (32 * s + 8 * side_of() >= used) {
#pragma unroll
        for (int r = 0; r < 4; ++r) store16(place_of(lds, s, r), (u32x4){0u, 0u, 0u, 0u});
      }
  }

  // Row 4 n + t of the group becomes row n of tile t.
  __device__ __forceinline__ void stage(UpStage<S>& lds, int used) const {
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (32 * s + 8 * side_of() < used) {
#pragma unroll
        for (int r = 0; r < 4; ++r) *reinterpret_cast<V8*>(place_of(lds, s, r)) = w[s][r];
      }
    // the wave's lanes read what the others wrote
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  static __device__ __forceinline__ void unstage() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // base + scale (up h).  Tokens that the adapter is not added to take base as it is,
  // tokens behind the sequence nothing.  The products with h's smaller parts come first: they
  // are NaN or infinite only with an infinite (or NaN) row of up, and then any number
  // will do beside those with the largest, whose infinity or NaN it is.
  static __device__ __forceinline__ void finish(const UpStage<S>& lds, const V4 (&base)[TT][4], int64_t out, int64_t group,
                                                const Hidden<T, S> (&h)[TT], const float (&factor)[TT][4],
                                                const Tokens<T, TT>& tokens) {
    const int lane = threadIdx.x & 63;
    f32x4 sums[TT][4];
    constexpr float kMost = 3.40282347e38f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      V8 tile[S];
#pragma unroll
      for (int i = 0; i < TT; ++i) sums[i][t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < S; ++s) {
        tile[s] = *reinterpret_cast<const V8*>(lds.bytes + (s * 4 + t) * UpStage<S>::TILE + (lane & 15) * 64 +
                                               (lane >> 4) * 16);
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
          for (int k = Hidden<T, S>::PARTS - 1; k > 0; --k) sums[i][t] = mfma16(h[i].part[k][s], tile[s], sums[i][t]);
      }
#pragma unroll
      for (int i = 0; i < TT; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[i][t][j] = __builtin_amdgcn_fmed3f(sums[i][t][j], -kMost, kMost);
#pragma unroll
        for (int s = 0; s < S; ++s) sums[i][t] = mfma16(h[i].part[0][s], tile[s], sums[i][t]);
      }
    }
    const int column = (int)group * kGroup + 4 * (lane & 15);
    if (column >= (int)out) return;
#pragma unroll
    for (int i = 0; i < TT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        V4 sum;
#pragma unroll
        for (int t = 0; t < 4; ++t) sum[t] = from_f32<T>(fmaf(factor[i][j], sums[i][t][j], to_f32(base[i][j][t])));
        if (tokens.live[i][j]) put<PAST>(tokens.y[i][j] + column, tokens.added[i][j] ? sum : base[i][j]);
      }
  }
};

// Groups first, first + step, .. of a wave's tokens, whose first one's loads are under way:
// a group's rows of up pass through LDS while the next one's loads begin.
template <typename T, int S, int TT, bool PAST>
__device__ __forceinline__ void expand(Group<T, S, TT, PAST>& data, UpStage<S>& lds, const T* up, int64_t rank, int64_t out,
                                       int used, int64_t first, int64_t groups, int64_t step,
                                       const Hidden<T, S> (&h)[TT], const Tokens<T, TT>& tokens) {
  float factor[TT][4];
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) factor[i][j] = __shfl(h[i].factor, 4 * quarter_of() + j);
  Group<T, S, TT, PAST>::clear(lds, used);
  for (int64_t g = first; g < groups; g += step) {
    typename Vec8<T>::half_type base[TT][4];
#pragma unroll
    for (int i = 0; i < TT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) base[i][j] = data.held[i][j];
    data.stage(lds, used);
    if (g + step >= groups) {
      Group<T, S, TT, PAST>::finish(lds, base, out, g, h, factor, tokens);
      break;
    }
    data.load(up, rank, out, used, g + step, tokens);
    Group<T, S, TT, PAST>::finish(lds, base, out, g, h, factor, tokens);
    Group<T, S, TT, PAST>::unstage();
  }
}

// Tokens without an adapter, groups first, first + step, ..: base as it is.
template <typename T, int TT, int DEEP, bool PAST>
__device__ __forceinline__ void copy_groups(int64_t out, int64_t first, int64_t groups, int64_t step,
                                            const Tokens<T, TT>& tokens) {
  typedef typename Vec8<T>::half_type V4;
  for (int64_t g = first; g < groups; g += DEEP * step) {
    V4 held[DEEP][TT][4];
#pragma unroll
    for (int d = 0; d < DEEP; ++d)
#pragma unroll
      for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t at = (g + d * step) * kGroup + 4 * (threadIdx.x & 15);
          held[d][i][j] = fetch<PAST, V4>(tokens.base[i][j] + (at < out ? at : out - 4));
        }
#pragma unroll
    for (int d = 0; d < DEEP; ++d)
#pragma unroll
      for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t at = (g + d * step) * kGroup + 4 * (threadIdx.x & 15);
          if (tokens.live[i][j] && g + d * step < groups && at < out && tokens.y[i][j] != tokens.base[i][j])
            put<PAST>(tokens.y[i][j] + at, held[d][i][j]);
        }
  }
}

// A workgroup takes 16 TT tokens and groups_of_wave groups of outputs a wave (all of them
// where tokens are many).  Its waves share `in` for h, add their sums up in order through
// LDS, and share the outputs.
// (Three waves a SIMD for ranks up to 32, two registers from the compiler's own choice: 2 x
// 20001 tokens of rank 32 139 us, with two waves 141.)
template <typename T, int S, int TT, bool PAST>
__global__ __launch_bounds__(kThreads, S == 1 ? 3 : 1) void low_rank_fused_kernel(const LowRankArgs a) {
  constexpr int N = 2 * S;
  __shared__ __align__(16) union {
    f32x4 sums[kWaves][TT * N][64];
    UpStage<S> up[kWaves];
  } lds;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t groups = (uint32_t)((a.out + kGroup - 1) / kGroup);
  const uint32_t portion = (uint32_t)a.groups_of_wave * kWaves;      // groups of a workgroup
  const uint32_t workgroups = (groups + portion - 1) / portion;      // of a tile
  const int64_t tile = blockIdx.x / workgroups;
  const int64_t from = (int64_t)(blockIdx.x % workgroups) * portion;
  const int64_t until = from + portion < groups ? from + portion : groups;
  const int64_t b = tile / a.tiles_of_seq;
  const int64_t first = (tile - b * a.tiles_of_seq) * (16 * TT);
  const Adapter it = adapter_of(a, b);
  if (it.used == 0 || first >= it.count) {
    const Tokens<T, TT> tokens(a, b, first, it.count);
    copy_groups<T, TT, 2, PAST>(a.out, from + wave, until, kWaves, tokens);
    return;
  }
  f32x4 h[TT][N];
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int t = 0; t < N; ++t) h[i][t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  {
    const T* x[TT][4];
    rows_of_x<T, TT>(a, b, first, x);
    int64_t w_first[S];
    rows_of_down<S>(it.used, a.in, w_first);
    const int64_t slabs = (a.in + kSlab - 1) / kSlab, share = (slabs + kWaves - 1) / kWaves;
    const int64_t to = (wave + 1) * share;
    shrink<T, S, TT>(x, static_cast<const T*>(a.down) + it.index * a.rank * a.in, w_first, a.in, wave * share,
                     to < slabs ? to : slabs, h);
  }
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int t = 0; t < N; ++t) lds.sums[wave][i * N + t][lane] = h[i][t];
  // the first group's loads pass the waves' meeting
  const Tokens<T, TT> tokens(a, b, first, it.count);
  const T* up = static_cast<const T*>(a.up) + it.index * a.out * a.rank;
  Group<T, S, TT, PAST> data;
  data.load(up, a.rank, a.out, it.used, from + wave < until ? from + wave : from, tokens);
  __syncthreads();
  Hidden<T, S> hidden[TT];
#pragma unroll
  for (int i = 0; i < TT; ++i) {
#pragma unroll
    for (int t = 0; t < N; ++t) {
      h[i][t] = lds.sums[0][i * N + t][lane];
#pragma unroll
      for (int k = 1; k < kWaves; ++k) h[i][t] += lds.sums[k][i * N + t][lane];
    }
    hidden[i] = make_hidden<T, S>(h[i], it.used, it.scale);
  }
  __syncthreads();
  expand<T, S, TT, PAST>(data, lds.up[wave], up, a.rank, a.out, it.used, from + wave, until, kWaves, hidden, tokens);
}

// Partial sums of h: workgroup (tile, part) takes the part's slabs, shared by its waves.
template <typename T, int S>
__global__ __launch_bounds__(kThreads) void low_rank_shrink_kernel(const LowRankArgs a) {
  constexpr int N = 2 * S;
  __shared__ f32x4 sums[kWaves - 1][N][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tile = blockIdx.x / (uint32_t)a.parts;
  const int part = (int)(blockIdx.x % (uint32_t)a.parts);
  const int64_t b = tile / a.tiles_of_seq;
  const int64_t first = (tile - b * a.tiles_of_seq) * 16;
  const Adapter it = adapter_of(a, b);
  if (it.used == 0 || first >= it.count) return;
  const T* x[1][4];
  rows_of_x<T, 1>(a, b, first, x);
  int64_t w_first[S];
  rows_of_down<S>(it.used, a.in, w_first);
  f32x4 h[1][N];
#pragma unroll
  for (int t = 0; t < N; ++t) h[0][t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  const int64_t slabs = (a.in + kSlab - 1) / kSlab;
  const int64_t from = (int64_t)part * a.slabs_of_part;
  const int64_t to = from + a.slabs_of_part < slabs ? from + a.slabs_of_part : slabs;
  const int64_t share = (to - from + kWaves - 1) / kWaves;
  const int64_t mine = from + wave * share;
  shrink<T, S, 1>(x, static_cast<const T*>(a.down) + it.index * a.rank * a.in, w_first, a.in, mine,
                  mine + share < to ? mine + share : to, h);
  if (wave != 0) {
#pragma unroll
    for (int t = 0; t < N; ++t) sums[wave - 1][t][lane] = h[0][t];
  }
  __syncthreads();
  if (wave != 0) return;
  f32x4* partial = reinterpret_cast<f32x4*>(a.partial) + ((int64_t)part * a.tiles + tile) * (N * 64) + lane;
#pragma unroll
  for (int t = 0; t < N; ++t) {
    f32x4 sum = h[0][t];
#pragma unroll
    for (int k = 0; k < kWaves - 1; ++k) sum += sums[k][t][lane];
    partial[t * 64] = sum;
  }
}

// The sums of h's parts and the outputs.  A workgroup's waves share the parts and add
// theirs up in order through LDS (each wave reading all of them: 64 tokens, 4096 -> 4096,
// rank 64, 12.7 us instead of 8.9, with a group a wave); a wave's groups lie a workgroup's waves apart.
template <typename T, int S>
__global__ __launch_bounds__(kThreads) void low_rank_expand_kernel(const LowRankArgs a) {
  constexpr int N = 2 * S;
  __shared__ __align__(16) union {
    f32x4 sums[kWaves][N][64];
    UpStage<S> up[kWaves];
  } lds;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t groups = (uint32_t)((a.out + kGroup - 1) / kGroup);
  const uint32_t share = (uint32_t)a.groups_of_wave * kWaves;  // groups of a workgroup
  const uint32_t workgroups = (groups + share - 1) / share;    // of a tile
  const int64_t tile = blockIdx.x / workgroups;
  const int64_t from = (int64_t)(blockIdx.x % workgroups) * share, mine = from + wave;
  const int64_t to = from + share < groups ? from + share : groups;
  const int64_t b = tile / a.tiles_of_seq;
  const int64_t first = (tile - b * a.tiles_of_seq) * 16;
  const Adapter it = adapter_of(a, b);
  const Tokens<T, 1> tokens(a, b, first, it.count);
  if (it.used == 0 || first >= it.count) {  // (the same for every wave)
    copy_groups<T, 1, 1, false>(a.out, mine, to, kWaves, tokens);
    return;
  }
  const T* up = static_cast<const T*>(a.up) + it.index * a.out * a.rank;
  // (the first group's loads before the parts', which they would wait for)
  Group<T, S, 1> data;
  data.load(up, a.rank, a.out, it.used, mine < to ? mine : from, tokens);
  f32x4 h[N];
#pragma unroll
  for (int t = 0; t < N; ++t) h[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  if (first + (lane & 15) < it.count) {
    const f32x4* partial = reinterpret_cast<const f32x4*>(a.partial) + tile * (N * 64) + lane;
    // (of rows that no row of down fills, what is read is not used)
    for (int p = a.parts > 1 ? wave : 0; p < a.parts; p += kWaves)
#pragma unroll
      for (int t = 0; t < N; ++t) h[t] += partial[(int64_t)p * a.tiles * (N * 64) + t * 64];
  }
  if (a.parts > 1) {  // the waves' shares of the parts, in order
#pragma unroll
    for (int t = 0; t < N; ++t) lds.sums[wave][t][lane] = h[t];
    __syncthreads();
#pragma unroll
    for (int t = 0; t < N; ++t) {
      h[t] = lds.sums[0][t][lane];
#pragma unroll
      for (int k = 1; k < kWaves; ++k) h[t] += lds.sums[k][t][lane];
    }
    __syncthreads();
  }
  const Hidden<T, S> hidden[1] = {make_hidden<T, S>(h, it.used, it.scale)};
  expand<T, S, 1, false>(data, lds.up[wave], up, a.rank, a.out, it.used, mine, to, kWaves, hidden, tokens);
}

// How a call is launched.
struct Plan {
  bool fused;
  bool past;               // base and y past the caches
  int tokens;              // of a tile
  int64_t tiles_of_seq, tiles;
  int parts, slabs_of_part, groups_of_wave;
  int rank_tiles;
  size_t bytes;
};
// Tiles of 16 tokens from which on one launch does both products.  4096 -> 4096, bf16, two
// launches / one, us: 8704 tokens of rank 16 63 / 63, of rank 64 84 / 80, of rank 128 121 /
// 134; 17408 tokens 103 / 94, 139 / 126 and 202 / 200; 34816 tokens 185 / 168, 255 / 207
// and 368 / 336.  Requests of up to a tile's tokens would leave the larger workgroups'
// places empty.
constexpr int64_t kManyTiles = 1024;
// Outputs (of 2 bytes) from which on base and y pass the caches: more than half of the 256 MB
// last-level cache, which the next operator could not find there anyway (2 x 20001
// tokens, 4096 outputs: 138 us instead of 149).
constexpr int64_t kPastOutputs = (int64_t)64 << 20;
// Few tokens of short inputs take one launch as well: a workgroup a tile and four groups of
// outputs, each with the first product to itself.  One / two launches, us: 1 and 8 tokens
// of 1024 inputs, rank 16, 5.4 / 3.3 + 3.9 and 5.8 / 3.8 + 4.2, rank 64 6.9 / 4.0 + 4.4 and
// 8.0 / 4.5 + 4.8; 7 tokens of 2048 inputs, rank 64, 10.0 / 5.0 + 4.8; and a launch is 3 us
// of the host's.  4096 inputs, 1 token of rank 64: 13.2 / 4.6 + 5.1.  More workgroups read
// `down` too often: 512 of rank 64 13.5 / 5.4 + 6.8, 4672 of rank 16 35 / 4.1 + 11.9.
constexpr int64_t kShortIn = 2048;
constexpr int64_t kFewWorkgroups = 256;

Plan plan_of(int64_t batch, int64_t seq, int64_t in, int64_t out, int64_t rank) {
  Plan p{};
  p.rank_tiles = rank <= 32 ? 2 : rank <= 64 ? 4 : 8;
  p.tokens = 16;
  p.tiles_of_seq = ceil_div(seq, 16);
  p.tiles = batch * p.tiles_of_seq;
  p.fused = p.tiles >= kManyTiles && seq > 16;
  if (p.fused) {
    p.tokens = 16 * kFusedTiles;
    p.tiles_of_seq = ceil_div(seq, p.tokens);
    p.tiles = batch * p.tiles_of_seq;
    p.groups_of_wave = (int)ceil_div(ceil_div(out, kGroup), kWaves);
    p.past = batch * seq * out > kPastOutputs;
    return p;
  }
  if (in <= kShortIn && p.tiles * ceil_div(ceil_div(out, kGroup), kWaves) <= kFewWorkgroups) {
    p.fused = true;
    p.groups_of_wave = 1;
    return p;
  }
  // Parts for a workgroup a unit, a slab a wave at least: every workgroup of the second
  // launch reads them all (64 tokens, 4096 -> 4096, rank 64: 18 us with 4, 20 with 8, 25
  // with 16, when every wave did).
  const int64_t slabs = ceil_div(in, kSlab);
  int64_t parts = ceil_div(256, p.tiles);
  const int64_t most = ceil_div(slabs, kWaves);
  if (parts > most) parts = most;
  p.slabs_of_part = (int)ceil_div(slabs, parts);
  p.parts = (int)ceil_div(slabs, p.slabs_of_part);
  // Several groups a wave, as long as that leaves waves for all units (64 tokens, 4096 ->
  // 4096, rank 64: the second launch 8.9 us with one, 7.6 with two, 8.8 with four; 16384
  // tokens, 4096 outputs, rank 64: 130 us with one, 105 with eight).
  const int64_t waves = p.tiles * ceil_div(out, kGroup);
  p.groups_of_wave = waves >= 8 * 4096 ? 8 : waves >= 4 * 4096 ? 4 : waves >= 4096 ? 2 : 1;
  p.bytes = (size_t)(p.parts * p.tiles * p.rank_tiles) * 64 * sizeof(f32x4);
  return p;
}

template <typename T, int S>
int launch(const LowRankArgs& a, const Plan& p, hipStream_t stream) {
  const int64_t workgroups = ceil_div(ceil_div(a.out, kGroup), kWaves * p.groups_of_wave);
  const dim3 grid((unsigned)(p.tiles * workgroups));
  if (p.fused) {
    if (p.tokens == 16)
      hipLaunchKernelGGL((low_rank_fused_kernel<T, S, 1, false>), grid, dim3(kThreads), 0, stream, a);
    else if (p.past)
      hipLaunchKernelGGL((low_rank_fused_kernel<T, S, kFusedTiles, true>), grid, dim3(kThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((low_rank_fused_kernel<T, S, kFusedTiles, false>), grid, dim3(kThreads), 0, stream, a);
    return check_hip(hipGetLastError(), "low-rank adapters launch");
  }
  hipLaunchKernelGGL((low_rank_shrink_kernel<T, S>), dim3((unsigned)(p.tiles * p.parts)), dim3(kThreads), 0, stream, a);
  const int status = check_hip(hipGetLastError(), "low-rank adapters launch");
  if (status != SAH_OK) return status;
  hipLaunchKernelGGL((low_rank_expand_kernel<T, S>), grid, dim3(kThreads), 0, stream, a);
  return check_hip(hipGetLastError(), "low-rank adapters launch");
}

template <typename T>
int launch_rank(const LowRankArgs& a, const Plan& p, hipStream_t stream) {
  switch (p.rank_tiles) {
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
  return plan_of(batch, seq_len, in_features, out_features, rank).bytes;
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
  const Plan plan = plan_of(batch, seq_len, in_features, out_features, rank);
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
  a.slabs_of_part = plan.slabs_of_part;
  a.groups_of_wave = plan.groups_of_wave;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return dtype == SAH_DTYPE_BF16 ? launch_rank<bf16>(a, plan, s) : launch_rank<f16>(a, plan, s);
}
