// Norm of each query and key head and the position rotation in one pass, for
// gfx950 (CDNA4).
//
//   y = norm(x) * weight + bias        over the head's D features, fp32
//   out = y with its first r features turned by the angles of the position:
//         (a, b) -> (a cos - b sin, b cos + a sin), a = y[i], b = y[i + r/2]
//         (or neighbours, y[2i] and y[2i+1]), cos and sin from a table row
//
// HBM-bound: every element is read and written once, and a token's table row is
// small beside its heads.  D / 8 lanes hold a row of 8 features each, so a
// wavefront covers 512 / D rows an access; the rows of an access are neighbouring
// heads of one token (the packed projection's output is read in whole lines), and
// the wave goes over up to STEPS such groups with one read of the table row.  All its
// loads are issued before the first sum.
//   2 x 50001 tokens, 16 + 16 heads of 64, bf16 (846 MB): 206 us, 4.1 TB/s (228 with
//   cached loads and stores)
//   3 x 777 tokens, 12 + 4 heads of 128, fp32 (38 MB): 12.4 us; 1 token, 16 + 16 heads of
//   64, bf16: 3.3 us (4.8 with four groups of heads a wave)

#include <type_traits>

#include "sah_common.hpp"

namespace sah {
namespace {

constexpr int kWave = 64;
constexpr int kWaves = 4;

// 16 bytes, past the caches where STREAM.
template <bool STREAM>
__device__ __forceinline__ u32x4 fetch(const void* p) {
  return STREAM ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)) : load16(p);
}
template <bool STREAM>
__device__ __forceinline__ void put(void* p, u32x4 v) {
  if (STREAM)
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p));
  else
    store16(p, v);
}

template <bool STREAM, typename T>
__device__ __forceinline__ void load8(const T* p, float* out) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 a = __builtin_bit_cast(f32x4, fetch<STREAM>(p)), b = __builtin_bit_cast(f32x4, fetch<STREAM>(p + 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = a[i], out[i + 4] = b[i];
  } else {
    unpack8<T>(fetch<STREAM>(p), out);
  }
}

template <bool STREAM, typename T>
__device__ __forceinline__ void store8(T* p, const float* in) {
  if constexpr (sizeof(T) == 4) {
    put<STREAM>(p, __builtin_bit_cast(u32x4, (f32x4){in[0], in[1], in[2], in[3]}));
    put<STREAM>(p + 4, __builtin_bit_cast(u32x4, (f32x4){in[4], in[5], in[6], in[7]}));
  } else {
    put<STREAM>(p, pack8<T>(in));
  }
}

struct RotaryArgs {
  const void* query;
  const void* key;
  const void* weight[2];  // query's, key's
  const void* bias[2];
  const float* table;
  const int32_t* starts;
  void* query_out;
  void* key_out;
  int64_t q_sb, q_sh, q_ss, k_sb, k_sh, k_ss;
  int64_t table_rows;
  uint32_t tokens;  // batch * seq_len, below 2^31
  uint32_t first_token;
  int seq_len, heads, kv_heads;
  int rotary;
  int row_heads;  // heads beside each other in an access, a power of two
  int pairs, rms;
  float eps;
};

template <typename T, typename TP, int D, int STEPS, bool STREAM>
__global__ __launch_bounds__(kWaves * kWave) void qk_rotary_kernel(const RotaryArgs a) {
  constexpr int LANES = D / 8;            // of one row
  constexpr int ROWS = kWave / LANES;     // of one access
  const int lane = threadIdx.x & (kWave - 1);
  const int chunk = lane & (LANES - 1);   // features 8 chunk .. + 7
  const int row = lane / LANES;
  const uint32_t wave = blockIdx.x * kWaves + threadIdx.x / kWave;
  const int tokens_a_wave = ROWS / a.row_heads;
  const uint32_t token = a.first_token + wave * (uint32_t)tokens_a_wave + (uint32_t)(row / a.row_heads);
  const bool here = token < a.tokens;
  const uint32_t b = here ? token / (uint32_t)a.seq_len : 0;
  const uint32_t s = here ? token - b * (uint32_t)a.seq_len : 0;
  const int all = a.heads + a.kv_heads;
  const int first_head = (int)blockIdx.y * a.row_heads * STEPS + (row & (a.row_heads - 1));

  float x[STEPS][8];
#pragma unroll
  for (int u = 0; u < STEPS; ++u) {
    const int h = first_head + u * a.row_heads;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[u][e] = 0.0f;
    if (here && h < all) {
      const T* p = h < a.heads
                       ? static_cast<const T*>(a.query) + b * a.q_sb + h * a.q_sh + s * a.q_ss
                       : static_cast<const T*>(a.key) + b * a.k_sb + (h - a.heads) * a.k_sh + s * a.k_ss;
      load8<STREAM>(p + chunk * 8, x[u]);
    }
  }

  // The table row of this lane's features; a position that the table does not hold
  // makes NaN of the turned features.
  const int half = a.rotary >> 1;
  const bool turned = chunk * 8 < a.rotary;
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) cs[e] = 1.0f, sn[e] = 0.0f;
  if (here && turned) {
    const int64_t position = (a.starts != nullptr ? (int64_t)a.starts[b] : 0) + (int64_t)s;
    if (position >= 0 && position < a.table_rows) {
      const float* t = a.table + position * a.rotary;
      if (a.pairs) {  // features 8 chunk .. are pairs 4 chunk ..
        const f32x4 c4 = *reinterpret_cast<const f32x4*>(t + chunk * 4);
        const f32x4 s4 = *reinterpret_cast<const f32x4*>(t + half + chunk * 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) cs[e] = c4[e / 2], sn[e] = s4[e / 2];
      } else {
        const int at = chunk * 8 < half ? chunk * 8 : chunk * 8 - half;
        load8<false>(t + at, cs);
        load8<false>(t + half + at, sn);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) cs[e] = sn[e] = __builtin_nanf("");
    }
  }
  // a's side takes -sin
  const bool first_half = chunk * 8 < half;
  if (!a.pairs && first_half) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sn[e] = -sn[e];
  }
  const int partner = turned ? (first_half ? lane + half / 8 : lane - half / 8) : lane;

  float w[2][8], bias[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[k][e] = 1.0f, bias[k][e] = 0.0f;
    if (a.weight[k] != nullptr) load8<false>(static_cast<const TP*>(a.weight[k]) + chunk * 8, w[k]);
    if (a.bias[k] != nullptr) load8<false>(static_cast<const TP*>(a.bias[k]) + chunk * 8, bias[k]);
  }

#pragma unroll
  for (int u = 0; u < STEPS; ++u) {
    const int h = first_head + u * a.row_heads;
    const bool is_key = h >= a.heads;
    float mean = 0.0f;
    if (!a.rms) {
#pragma unroll
      for (int e = 0; e < 8; ++e) mean += x[u][e];
#pragma unroll
      for (int m = 1; m < LANES; m <<= 1) mean += __shfl_xor(mean, m);
      mean *= 1.0f / D;
    }
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = x[u][e] - mean;
      ss += d * d;
    }
#pragma unroll
    for (int m = 1; m < LANES; m <<= 1) ss += __shfl_xor(ss, m);
    const float rstd = rsqrtf(ss * (1.0f / D) + a.eps);
    float y[8], out[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      y[e] = (x[u][e] - mean) * rstd * (is_key ? w[1][e] : w[0][e]) + (is_key ? bias[1][e] : bias[0][e]);
    if (a.rotary == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = y[e];
    } else if (a.pairs) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        out[e] = y[e] * cs[e] - y[e + 1] * sn[e];
        out[e + 1] = y[e + 1] * cs[e] + y[e] * sn[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = __shfl(y[e], partner);
        out[e] = turned ? y[e] * cs[e] + other * sn[e] : y[e];
      }
    }
    if (here && h < all) {
      T* p = is_key ? static_cast<T*>(a.key_out) + ((int64_t)b * a.kv_heads + (h - a.heads)) * a.seq_len * D + (int64_t)s * D
                    : static_cast<T*>(a.query_out) + ((int64_t)b * a.heads + h) * a.seq_len * D + (int64_t)s * D;
      store8<STREAM>(p + chunk * 8, out);
    }
  }
}

template <typename T, typename TP, int D, int STEPS, bool STREAM>
int launch_steps(RotaryArgs a, int64_t tokens_a_block, hipStream_t stream) {
  const unsigned chunks = (unsigned)ceil_div(a.heads + a.kv_heads, (int64_t)a.row_heads * STEPS);
  // A grid holds fewer than 2^32 work items a dimension: more tokens go out as several launches.
  const int64_t per_launch = (int64_t)(UINT32_MAX / (kWaves * kWave)) * tokens_a_block;
  for (int64_t first = 0; first < (int64_t)a.tokens; first += per_launch) {
    const int64_t left = (int64_t)a.tokens - first;
    const int64_t count = left < per_launch ? left : per_launch;
    a.first_token = (uint32_t)first;
    hipLaunchKernelGGL((qk_rotary_kernel<T, TP, D, STEPS, STREAM>),
                       dim3((unsigned)ceil_div(count, tokens_a_block), chunks), dim3(kWaves * kWave), 0, stream, a);
    const int status = check_hip(hipGetLastError(), "query/key rotary kernel launch");
    if (status != SAH_OK) return status;
  }
  return SAH_OK;
}

// Groups of heads a wave: one where four would leave SIMDs of the 256 compute units
// without a wave (one read of the table row less against three passes in a row).
// Past the caches: outputs over half of the 256 MB last-level cache, which the next
// operator would not find there.
template <typename T, typename TP, int D>
int launch_rotary(RotaryArgs a, hipStream_t stream) {
  constexpr int ROWS = 512 / D;
  const int64_t all = a.heads + a.kv_heads;
  a.row_heads = 1;
  while (a.row_heads < ROWS && a.row_heads < all) a.row_heads *= 2;
  const int64_t tokens_a_block = (int64_t)kWaves * (ROWS / a.row_heads);
  const int64_t waves = ceil_div(a.tokens, ROWS / a.row_heads) * ceil_div(all, 4 * a.row_heads);
  if (waves < 1024) return launch_steps<T, TP, D, 1, false>(a, tokens_a_block, stream);
  return (int64_t)a.tokens * all * D * (int64_t)sizeof(T) > ((int64_t)128 << 20)
             ? launch_steps<T, TP, D, 4, true>(a, tokens_a_block, stream)
             : launch_steps<T, TP, D, 4, false>(a, tokens_a_block, stream);
}

template <typename T, typename TP>
int dispatch_dim(const RotaryArgs& a, int64_t dim, hipStream_t stream) {
  switch (dim) {
    case 64: return launch_rotary<T, TP, 64>(a, stream);
    case 128: return launch_rotary<T, TP, 128>(a, stream);
    default: return launch_rotary<T, TP, 256>(a, stream);
  }
}

}  // namespace
}  // namespace sah

using namespace sah;

extern "C" int sah_qk_norm_rotary(
    const void* query, const void* key, const void* query_weight, const void* query_bias,
    const void* key_weight, const void* key_bias, const float* table, const int32_t* starts,
    void* query_out, void* key_out, int64_t batch, int64_t seq_len, int64_t heads, int64_t kv_heads,
    int64_t head_dim, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s, int64_t k_stride_b,
    int64_t k_stride_h, int64_t k_stride_s, int64_t rotary_dim, int64_t table_rows, int interleaved,
    int norm_kind, float eps, int dtype, int param_dtype, sah_stream_t stream) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(SAH_ERR_UNSUPPORTED, "sah_qk_norm_rotary: head_dim %lld is not 64, 128 or 256", (long long)head_dim);
  if (dtype != SAH_DTYPE_F32 && dtype != SAH_DTYPE_F16 && dtype != SAH_DTYPE_BF16)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_qk_norm_rotary: unknown dtype code %d", dtype);
  if (param_dtype != SAH_DTYPE_F32 && param_dtype != dtype)
    return fail(SAH_ERR_UNSUPPORTED, "sah_qk_norm_rotary: param dtype must be f32 or the tensors' dtype");
  if (norm_kind != SAH_NORM_LAYER && norm_kind != SAH_NORM_RMS)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_qk_norm_rotary: unknown norm kind %d", norm_kind);
  if (!(eps >= 0.0f)) return fail(SAH_ERR_INVALID_ARGUMENT, "sah_qk_norm_rotary: eps must be >= 0");
  if (batch < 0 || seq_len < 0 || heads <= 0 || kv_heads <= 0 || heads > 65536 || kv_heads > 65536)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_qk_norm_rotary: bad batch, length or head count");
  if (batch > INT32_MAX || seq_len > INT32_MAX || (seq_len != 0 && batch > INT32_MAX / seq_len))
    return fail(SAH_ERR_UNSUPPORTED, "sah_qk_norm_rotary: batch * seq_len must be below 2^31");
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % (interleaved ? 8 : 16) != 0)
    return fail(SAH_ERR_UNSUPPORTED,
                "sah_qk_norm_rotary: rotary_dim %lld must be a multiple of %d up to head_dim",
                (long long)rotary_dim, interleaved ? 8 : 16);
  if (batch == 0 || seq_len == 0) return SAH_OK;
  if (query == nullptr || key == nullptr || query_out == nullptr || key_out == nullptr ||
      (rotary_dim != 0 && table == nullptr))
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_qk_norm_rotary: null tensor pointer");
  if (table_rows < 0) return fail(SAH_ERR_INVALID_ARGUMENT, "sah_qk_norm_rotary: negative table_rows");
  const void* wide[] = {query, key, query_weight, query_bias, key_weight, key_bias, table, query_out, key_out};
  for (const void* p : wide)
    if (!aligned16(p)) return fail(SAH_ERR_INVALID_ARGUMENT, "sah_qk_norm_rotary: tensors must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(starts) & 3u) != 0)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_qk_norm_rotary: starts must be 4-byte aligned");
  const int64_t unit = dtype == SAH_DTYPE_F32 ? 4 : 8;
  const int64_t strides[] = {q_stride_b, q_stride_h, q_stride_s, k_stride_b, k_stride_h, k_stride_s};
  for (int64_t v : strides)
    if (v % unit != 0)
      return fail(SAH_ERR_INVALID_ARGUMENT, "sah_qk_norm_rotary: strides must be multiples of 16 bytes");
  RotaryArgs a{};
  a.query = query;
  a.key = key;
  a.weight[0] = query_weight;
  a.weight[1] = key_weight;
  a.bias[0] = query_bias;
  a.bias[1] = key_bias;
  a.table = table;
  a.starts = starts;
  a.query_out = query_out;
  a.key_out = key_out;
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.q_ss = q_stride_s;
  a.k_sb = k_stride_b;
  a.k_sh = k_stride_h;
  a.k_ss = k_stride_s;
  a.table_rows = table_rows;
  a.tokens = (uint32_t)(batch * seq_len);
  a.seq_len = (int)seq_len;
  a.heads = (int)heads;
  a.kv_heads = (int)kv_heads;
  a.rotary = (int)rotary_dim;
  a.pairs = interleaved != 0;
  a.rms = norm_kind == SAH_NORM_RMS;
  a.eps = eps;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool f32_params = param_dtype == SAH_DTYPE_F32;
  if (dtype == SAH_DTYPE_F32) return dispatch_dim<float, float>(a, head_dim, s);
  if (dtype == SAH_DTYPE_BF16)
    return f32_params ? dispatch_dim<bf16, float>(a, head_dim, s) : dispatch_dim<bf16, bf16>(a, head_dim, s);
  return f32_params ? dispatch_dim<f16, float>(a, head_dim, s) : dispatch_dim<f16, f16>(a, head_dim, s);
}
