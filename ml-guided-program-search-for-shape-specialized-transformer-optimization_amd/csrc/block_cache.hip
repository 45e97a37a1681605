// Append to and read from the 8-bit block cache of keys and values, for gfx950
// (CDNA4).
//
// A sequence's tokens stand in blocks of 64.  A block that is complete holds e4m3
// codes, one scale for (block, head) for the keys and one for the values: the
// smallest power of two s (at least 2^-100) with max|x| / s <= 448, so x / s is
// exact and a code is off by at most half an e4m3 step; a block of zeros has s = 1.
// The block that is not complete yet stands in the tensors' own type in the
// sequence's tail and is coded once, when its last token comes: what the cache
// holds does not depend on the steps in which the tokens came, and a complete
// block never changes.
//
// Value codes stand feature by feature (64 tokens of a feature side by side), the
// order in which the attention's second product reads them.
//
// A token with a non-finite key or value takes a key of NaN and a value of zeros
// (and no part in the scales): every query that attends to it answers NaN, and a
// query that does not is not touched by it.

#include <type_traits>

#include "decode_common.hpp"

namespace sah {
namespace {

constexpr int kThreads = 256;

struct CacheArgs {
  uint8_t* key_codes;    // [blocks, heads, 64, D]
  uint8_t* value_codes;  // [blocks, heads, D, 64]
  float* key_scales;     // [blocks, heads]
  float* value_scales;
  void* key_tail;        // [batch, heads, 64, D]
  void* value_tail;      // [batch, heads, D, 64]
  const int32_t* table;  // [batch, max_blocks]
  int64_t blocks, max_blocks;
  int heads;
};

struct AppendArgs {
  CacheArgs cache;
  const void* key;
  const void* value;
  int64_t k_sb, k_sh, k_ss, v_sb, v_sh, v_ss;
  const int32_t* starts;
  const int32_t* counts;
  int seq_len;
  uint32_t span;  // blocks that seq_len tokens can touch
};

template <typename T>
__device__ __forceinline__ bool finite_value(T x) {
  return fabsf(to_f32(x)) < INFINITY;
}

// The power p of the scale 2^p of a block whose largest magnitude is `largest`
// (finite): largest = m 2^e with m in [1, 2) takes 2^(e - 8), or twice that where
// m > 1.75 (448 = 1.75 * 2^8).
__device__ __forceinline__ int scale_power(float largest) {
  if (largest == 0.0f) return 0;
  const uint32_t bits = __float_as_uint(largest);
  const int power = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return power < -100 ? -100 : power;
}
__device__ __forceinline__ float power_of_two(int p) { return __uint_as_float((uint32_t)(p + 127) << 23); }

__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  v = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
  return (uint32_t)v;
}

// HBM-bound on prompts: a token is read once, its codes written once, with all of a
// block's loads in flight before its largest magnitude is known.  Heads are dealt to
// neighbouring workgroups, so that a token's heads, neighbours in a packed projection,
// are read at the same time, and past the caches:
//   4 x 8001 tokens, 8 heads of 128, fp16 (197 MB): 41 us, 4.7 TB/s (48 through the
//   caches); 8 x 4001 tokens, 16 heads of 64: 43 us (66 block by block of a head)
//   33 x 1 token, 8 heads of 128: 3.3 us, 6.3 where a block is completed (8.6 with the
//   tail's values read token by token); 52 x 43 tokens: 16 us (25)
//
// One workgroup takes one block of (sequence, head): it codes the block if the
// append completes it, from the tail's old tokens and the new ones.  The first
// block's workgroup, the only one that reads the old tail, then also writes the new
// tail, so no workgroup writes what another one reads.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void block_append_kernel(const AppendArgs a) {
  typedef typename Vec8<T>::type V8;
  constexpr int LANES = D / 8;                 // of one token
  constexpr int TOKENS = kThreads / LANES;     // of one pass
  constexpr int PASSES = kBlockTokens / TOKENS;
  constexpr int ROW = kBlockTokens + 4;        // bytes of a feature in LDS: features on different banks
  __shared__ float largest_of[2][kThreads / 64];
  constexpr int WIDE_ROW = kBlockTokens + 1;   // values of a feature in LDS, an odd number
  __shared__ __align__(16) union {
    uint8_t codes[D * ROW];
    T values[D * WIDE_ROW];
  } turned;

  const uint32_t pair = blockIdx.x / (uint32_t)a.cache.heads;
  const int h = (int)(blockIdx.x - pair * (uint32_t)a.cache.heads);
  const uint32_t index = pair % a.span;
  const int64_t b = pair / a.span;
  const int tid = threadIdx.x;
  const int lane = tid & 63;

  const int64_t start = a.starts[b];
  int64_t count = a.counts != nullptr ? (int64_t)a.counts[b] : (int64_t)a.seq_len;
  if (count > a.seq_len) count = a.seq_len;
  if (start < 0 || count <= 0) return;
  const int64_t end = start + count;
  const int64_t first = start / kBlockTokens;
  const int64_t block = first + index;
  const bool complete = (block + 1) * kBlockTokens <= end;
  if (index != 0 && !complete) return;

  const int64_t id = complete && block < a.cache.max_blocks ? (int64_t)a.cache.table[b * a.cache.max_blocks + block] : -1;
  const bool held = id >= 0 && id < a.cache.blocks;  // a page outside the cache takes nothing
  const int feature = (tid & (LANES - 1)) * 8;
  const int token0 = tid / LANES;
  const T* key = static_cast<const T*>(a.key) + b * a.k_sb + h * a.k_sh + feature;
  const T* value = static_cast<const T*>(a.value) + b * a.v_sb + h * a.v_sh + feature;
  const int64_t tail_at = (b * a.cache.heads + h) * (int64_t)(kBlockTokens * D);
  T* key_tail = static_cast<T*>(a.cache.key_tail) + tail_at;
  T* value_tail = static_cast<T*>(a.cache.value_tail) + tail_at;

  // Whether any feature of this lane's token is not finite, in the key or the value.
  auto bad_token = [&](V8 k, V8 v) {
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) bad = bad || !finite_value<T>(k[e]) || !finite_value<T>(v[e]);
    const uint64_t any = __ballot(bad);
    return ((any >> (lane & ~(LANES - 1))) & ((1ull << LANES) - 1)) != 0;
  };

  if (complete) {
    V8 k[PASSES], v[PASSES];
    bool bad[PASSES];
    float k_largest = 0.0f, v_largest = 0.0f;
    if (index == 0 && start % kBlockTokens != 0) {  // the tail's values turn in LDS
      const int old = (int)(start % kBlockTokens);
#pragma unroll
      for (int i = tid; i < D * 8; i += kThreads) {
        const int slot = i % 8 * 8;
        if (slot >= old) continue;
        const V8 part = *reinterpret_cast<const V8*>(value_tail + i * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) turned.values[i / 8 * WIDE_ROW + slot + e] = part[e];
      }
      __syncthreads();
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int slot = token0 * PASSES + p;
      const int64_t position = block * kBlockTokens + slot;
      if (position < start) {  // index 0 only: an older token of this block
        k[p] = *reinterpret_cast<const V8*>(key_tail + slot * D + feature);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[p][e] = turned.values[(feature + e) * WIDE_ROW + slot];
      } else {
        const int64_t at = position - start;
        k[p] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(key + at * a.k_ss));
        v[p] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(value + at * a.v_ss));
      }
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      bad[p] = bad_token(k[p], v[p]);
      if (!bad[p]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          k_largest = fmaxf(k_largest, fabsf(to_f32(k[p][e])));
          v_largest = fmaxf(v_largest, fabsf(to_f32(v[p][e])));
        }
      }
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      k_largest = fmaxf(k_largest, __shfl_xor(k_largest, m));
      v_largest = fmaxf(v_largest, __shfl_xor(v_largest, m));
    }
    if (lane == 0) {
      largest_of[0][tid / 64] = k_largest;
      largest_of[1][tid / 64] = v_largest;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
      k_largest = fmaxf(k_largest, largest_of[0][w]);
      v_largest = fmaxf(v_largest, largest_of[1][w]);
    }
    const int k_power = scale_power(k_largest), v_power = scale_power(v_largest);
    const float k_inverse = power_of_two(-k_power), v_inverse = power_of_two(-v_power);
    const int64_t code_at = (id * a.cache.heads + h) * (int64_t)(kBlockTokens * D);
    u32x2 value_coded[PASSES];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int slot = token0 * PASSES + p;
      u32x2 coded = {0x7f7f7f7fu, 0x7f7f7f7fu};
      value_coded[p] = (u32x2){0u, 0u};
      if (!bad[p]) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = to_f32(k[p][e]) * k_inverse;
        coded = (u32x2){pack_e4m3(f[0], f[1], f[2], f[3]), pack_e4m3(f[4], f[5], f[6], f[7])};
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = to_f32(v[p][e]) * v_inverse;
        value_coded[p] = (u32x2){pack_e4m3(f[0], f[1], f[2], f[3]), pack_e4m3(f[4], f[5], f[6], f[7])};
      }
      if (held) *reinterpret_cast<u32x2*>(a.cache.key_codes + code_at + slot * D + feature) = coded;
    }
    // The values turn in LDS: a thread's PASSES neighbouring tokens leave together.
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t codes = 0;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) codes |= (value_coded[p][e / 4] >> (8 * (e % 4)) & 0xffu) << (8 * p);
      uint8_t* to = turned.codes + (feature + e) * ROW + token0 * PASSES;
      if constexpr (PASSES == 4)
        *reinterpret_cast<uint32_t*>(to) = codes;
      else
        *reinterpret_cast<uint16_t*>(to) = (uint16_t)codes;
    }
    __syncthreads();
    if (held) {
#pragma unroll
      for (int i = tid; i < D * 4; i += kThreads) {
        const uint32_t* from = reinterpret_cast<const uint32_t*>(turned.codes + (i / 4) * ROW + (i % 4) * 16);
        const u32x4 part = {from[0], from[1], from[2], from[3]};
        store16(a.cache.value_codes + code_at + i * 16, part);
      }
      if (tid == 0) {
        a.cache.key_scales[id * a.cache.heads + h] = power_of_two(k_power);
        a.cache.value_scales[id * a.cache.heads + h] = power_of_two(v_power);
      }
    }
  }

  // The tail: the new tokens of the last, incomplete block.  Every old token that
  // the block above needs is in registers (the barriers above).  Values of several
  // tokens turn in LDS too and leave a feature's tokens side by side.
  if (index != 0) return;
  const int64_t last = end / kBlockTokens * kBlockTokens;
  const int64_t from = start > last ? start : last;
  const bool several = end - from >= 8;
  if (several) __syncthreads();  // the codes above are read
  for (int64_t position = from + token0; position < end; position += TOKENS) {
    const int slot = (int)(position - last);
    const int64_t at = position - start;
    V8 k = *reinterpret_cast<const V8*>(key + at * a.k_ss);
    V8 v = *reinterpret_cast<const V8*>(value + at * a.v_ss);
    if (bad_token(k, v)) {  // asked of the lanes of one token, which are here together
#pragma unroll
      for (int e = 0; e < 8; ++e) k[e] = (T)__builtin_nanf(""), v[e] = (T)0.0f;
    }
    *reinterpret_cast<V8*>(key_tail + slot * D + feature) = k;
    if (several) {
#pragma unroll
      for (int e = 0; e < 8; ++e) turned.values[(feature + e) * WIDE_ROW + slot] = v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) value_tail[(feature + e) * kBlockTokens + slot] = v[e];
    }
  }
  if (!several) return;
  __syncthreads();
  const int slot = tid % kBlockTokens;
  if (slot < from - last || slot >= end - last) return;
#pragma unroll
  for (int d = tid / kBlockTokens; d < D; d += kThreads / kBlockTokens)
    value_tail[d * kBlockTokens + slot] = turned.values[d * WIDE_ROW + slot];
}

struct ReadArgs {
  CacheArgs cache;
  void* key;    // [batch, heads, tokens, D]
  void* value;
  const int32_t* firsts;
  const int32_t* lengths;
  int64_t tokens;
  uint32_t span;
};

// HBM-bound: codes are read once, 16-bit keys and values written once.  A workgroup
// takes one block of (sequence, head), whose values turn in LDS, a feature's tokens an
// odd number of places apart, on their way to the output's rows:
//   4 x 8001 tokens, 8 heads of 128, fp16 (197 MB): 39 us, 5.0 TB/s (41 with features
//   68 places apart); 64 x 64 tokens, 16 heads of 64: 8.4 us
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void block_read_kernel(const ReadArgs a) {
  typedef typename Vec8<T>::type V8;
  constexpr int LANES = D / 8;
  constexpr int TOKENS = kThreads / LANES;
  constexpr int PASSES = kBlockTokens / TOKENS;
  constexpr int ROW = kBlockTokens + 1;  // values of a feature in LDS
  __shared__ T turned[D * ROW];

  const uint32_t pair = blockIdx.x / (uint32_t)a.cache.heads;
  const int h = (int)(blockIdx.x - pair * (uint32_t)a.cache.heads);
  const uint32_t index = pair % a.span;
  const int64_t b = pair / a.span;
  const int tid = threadIdx.x;
  const int64_t first = a.firsts[b], length = a.lengths[b];
  // blocks from the one of `first` on, rounded down (also below zero)
  const int64_t block = (first >= 0 ? first : first - (kBlockTokens - 1)) / kBlockTokens + index;
  const int64_t offset = block * kBlockTokens - first;  // output row of the block's first token
  if (offset >= a.tokens) return;

  const bool is_tail = block >= 0 && block == length / kBlockTokens;
  const bool any = block >= 0 && block * kBlockTokens < length;
  int64_t id = -1;
  if (any && !is_tail && block < a.cache.max_blocks) id = a.cache.table[b * a.cache.max_blocks + block];
  const bool held = id >= 0 && id < a.cache.blocks;

  const int64_t code_at = ((held ? id : 0) * a.cache.heads + h) * (int64_t)(kBlockTokens * D);
  const int64_t tail_at = (b * a.cache.heads + h) * (int64_t)(kBlockTokens * D);
  const float nan = __builtin_nanf("");
  const float k_scale = held ? a.cache.key_scales[id * a.cache.heads + h] : nan;
  const float v_scale = held ? a.cache.value_scales[id * a.cache.heads + h] : nan;
  if (any) {  // values, feature by feature into LDS
    for (int i = tid; i < D * 8; i += kThreads) {
      const int feature = i / 8, slot = (i % 8) * 8;
      V8 v;
      if (is_tail) {
        v = *reinterpret_cast<const V8*>(static_cast<const T*>(a.cache.value_tail) + tail_at + feature * kBlockTokens + slot);
      } else {
        u32x2 raw = {0u, 0u};
        if (held) raw = *reinterpret_cast<const u32x2*>(a.cache.value_codes + code_at + feature * kBlockTokens + slot);
        const V8 codes = e4m3_operand<T>(raw[0], raw[1], 1.0f);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = in_range<T>(to_f32(codes[e]) * v_scale);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) turned[feature * ROW + slot + e] = v[e];
    }
  }
  __syncthreads();
  const int feature = (tid & (LANES - 1)) * 8;
  const int64_t out_at = (b * a.cache.heads + h) * a.tokens;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int slot = p * TOKENS + tid / LANES;
    const int64_t row = offset + slot;
    if (row < 0 || row >= a.tokens) continue;
    const bool live = any && block * kBlockTokens + slot < length;
    V8 k, v;
#pragma unroll
    for (int e = 0; e < 8; ++e) k[e] = v[e] = (T)0.0f;
    if (live) {
      if (is_tail) {
        k = *reinterpret_cast<const V8*>(static_cast<const T*>(a.cache.key_tail) + tail_at + slot * D + feature);
      } else {
        u32x2 raw = {0u, 0u};
        if (held) raw = *reinterpret_cast<const u32x2*>(a.cache.key_codes + code_at + slot * D + feature);
        const V8 codes = e4m3_operand<T>(raw[0], raw[1], 1.0f);
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] = in_range<T>(to_f32(codes[e]) * k_scale);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = turned[(feature + e) * ROW + slot];
    }
    *reinterpret_cast<V8*>(static_cast<T*>(a.key) + (out_at + row) * D + feature) = k;
    *reinterpret_cast<V8*>(static_cast<T*>(a.value) + (out_at + row) * D + feature) = v;
  }
}

template <typename T, int D>
int launch_append(const AppendArgs& a, unsigned grid, hipStream_t stream) {
  hipLaunchKernelGGL((block_append_kernel<T, D>), dim3(grid), dim3(kThreads), 0, stream, a);
  return check_hip(hipGetLastError(), "block cache append launch");
}
template <typename T, int D>
int launch_read(const ReadArgs& a, unsigned grid, hipStream_t stream) {
  hipLaunchKernelGGL((block_read_kernel<T, D>), dim3(grid), dim3(kThreads), 0, stream, a);
  return check_hip(hipGetLastError(), "block cache read launch");
}

int check_cache(const char* what, const CacheArgs& c, int64_t batch, int64_t kv_heads, int64_t head_dim, int dtype) {
  if (head_dim != 64 && head_dim != 128)
    return fail(SAH_ERR_UNSUPPORTED, "%s: head_dim %lld is not 64 or 128", what, (long long)head_dim);
  if (dtype != SAH_DTYPE_BF16 && dtype != SAH_DTYPE_F16)
    return fail(SAH_ERR_UNSUPPORTED, "%s: dtype %d is not bf16 or f16", what, dtype);
  if (batch < 0 || batch > INT32_MAX || kv_heads <= 0 || kv_heads > 65536 || c.blocks < 0 || c.blocks > INT32_MAX ||
      c.max_blocks < 0 || c.max_blocks > INT32_MAX / kBlockTokens)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: bad batch, head or block count", what);
  if (batch == 0) return SAH_OK;
  if (c.key_tail == nullptr || c.value_tail == nullptr || (c.max_blocks != 0 && c.table == nullptr) ||
      (c.blocks != 0 && (c.key_codes == nullptr || c.value_codes == nullptr || c.key_scales == nullptr ||
                         c.value_scales == nullptr)))
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: null cache pointer", what);
  if (!aligned16(c.key_tail) || !aligned16(c.value_tail) || !aligned16(c.key_codes) || !aligned16(c.value_codes))
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: codes and tails must be 16-byte aligned", what);
  const void* words[] = {c.key_scales, c.value_scales, c.table};
  for (const void* p : words)
    if ((reinterpret_cast<uintptr_t>(p) & 3u) != 0)
      return fail(SAH_ERR_INVALID_ARGUMENT, "%s: scales and block table must be 4-byte aligned", what);
  return SAH_OK;
}

// Workgroups of (sequence, head, block), or 0 where a launch cannot hold them.
unsigned grid_of(int64_t batch, int64_t heads, int64_t span) {
  const int64_t most = (int64_t)(UINT32_MAX / kThreads);
  if (span > most || batch * heads > most / span) return 0;
  return (unsigned)(batch * heads * span);
}

}  // namespace
}  // namespace sah

using namespace sah;

extern "C" int sah_block_cache_append(
    const void* key, const void* value, void* key_codes, void* value_codes, float* key_scales, float* value_scales,
    void* key_tail, void* value_tail, const int32_t* block_table, const int32_t* starts, const int32_t* counts,
    int64_t batch, int64_t kv_heads, int64_t seq_len, int64_t head_dim, int64_t k_stride_b, int64_t k_stride_h,
    int64_t k_stride_s, int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_s, int64_t num_blocks,
    int64_t max_blocks, int dtype, sah_stream_t stream) {
  AppendArgs a{};
  a.cache = {static_cast<uint8_t*>(key_codes), static_cast<uint8_t*>(value_codes), key_scales, value_scales,
             key_tail, value_tail, block_table, num_blocks, max_blocks, (int)kv_heads};
  const int status = check_cache("sah_block_cache_append", a.cache, batch, kv_heads, head_dim, dtype);
  if (status != SAH_OK) return status;
  if (seq_len < 0 || seq_len > INT32_MAX)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_block_cache_append: bad seq_len %lld", (long long)seq_len);
  if (batch == 0 || seq_len == 0) return SAH_OK;
  if (key == nullptr || value == nullptr || starts == nullptr)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_block_cache_append: null tensor pointer");
  if (!aligned16(key) || !aligned16(value))
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_block_cache_append: key and value must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(starts) & 3u) != 0 || (reinterpret_cast<uintptr_t>(counts) & 3u) != 0)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_block_cache_append: starts and counts must be 4-byte aligned");
  const int64_t strides[] = {k_stride_b, k_stride_h, k_stride_s, v_stride_b, v_stride_h, v_stride_s};
  for (int64_t v : strides)
    if (v % 8 != 0)
      return fail(SAH_ERR_INVALID_ARGUMENT, "sah_block_cache_append: strides must be multiples of 8 elements");
  a.key = key;
  a.value = value;
  a.k_sb = k_stride_b;
  a.k_sh = k_stride_h;
  a.k_ss = k_stride_s;
  a.v_sb = v_stride_b;
  a.v_sh = v_stride_h;
  a.v_ss = v_stride_s;
  a.starts = starts;
  a.counts = counts;
  a.seq_len = (int)seq_len;
  a.span = (uint32_t)((seq_len + kBlockTokens - 2) / kBlockTokens + 1);
  const unsigned grid = grid_of(batch, kv_heads, a.span);
  if (grid == 0) return fail(SAH_ERR_UNSUPPORTED, "sah_block_cache_append: too many blocks for one launch");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == SAH_DTYPE_BF16)
    return head_dim == 64 ? launch_append<bf16, 64>(a, grid, s) : launch_append<bf16, 128>(a, grid, s);
  return head_dim == 64 ? launch_append<f16, 64>(a, grid, s) : launch_append<f16, 128>(a, grid, s);
}

extern "C" int sah_block_cache_read(
    const void* key_codes, const void* value_codes, const float* key_scales, const float* value_scales,
    const void* key_tail, const void* value_tail, const int32_t* block_table, const int32_t* firsts,
    const int32_t* lengths, void* key, void* value, int64_t batch, int64_t kv_heads, int64_t tokens, int64_t head_dim,
    int64_t num_blocks, int64_t max_blocks, int dtype, sah_stream_t stream) {
  ReadArgs a{};
  a.cache = {static_cast<uint8_t*>(const_cast<void*>(key_codes)), static_cast<uint8_t*>(const_cast<void*>(value_codes)),
             const_cast<float*>(key_scales), const_cast<float*>(value_scales), const_cast<void*>(key_tail),
             const_cast<void*>(value_tail), block_table, num_blocks, max_blocks, (int)kv_heads};
  const int status = check_cache("sah_block_cache_read", a.cache, batch, kv_heads, head_dim, dtype);
  if (status != SAH_OK) return status;
  if (tokens < 0 || tokens > INT32_MAX)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_block_cache_read: bad token count %lld", (long long)tokens);
  if (batch == 0 || tokens == 0) return SAH_OK;
  if (key == nullptr || value == nullptr || firsts == nullptr || lengths == nullptr)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_block_cache_read: null tensor pointer");
  if (!aligned16(key) || !aligned16(value))
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_block_cache_read: key and value must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(firsts) & 3u) != 0 || (reinterpret_cast<uintptr_t>(lengths) & 3u) != 0)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_block_cache_read: firsts and lengths must be 4-byte aligned");
  a.key = key;
  a.value = value;
  a.firsts = firsts;
  a.lengths = lengths;
  a.tokens = tokens;
  a.span = (uint32_t)((tokens + kBlockTokens - 2) / kBlockTokens + 1);
  const unsigned grid = grid_of(batch, kv_heads, a.span);
  if (grid == 0) return fail(SAH_ERR_UNSUPPORTED, "sah_block_cache_read: too many blocks for one launch");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == SAH_DTYPE_BF16)
    return head_dim == 64 ? launch_read<bf16, 64>(a, grid, s) : launch_read<bf16, 128>(a, grid, s);
  return head_dim == 64 ? launch_read<f16, 64>(a, grid, s) : launch_read<f16, 128>(a, grid, s);
}
