// Linear layer with 4-bit weights and group scales for few rows, for gfx950 (CDNA4).
//
//   y = act(x W^T + bias),  W[n][k] = scale[k / group][n] * code[n][k],  code -7 .. 7
//
// Bound by the codes: half a byte a weight, read once.  The rows are the columns of
// 16 x 16 x 32 products whose rows are 16 outputs, so up to 16 rows cost what one
// costs.  A word of eight codes is a lane's operand of one product; a lane's four
// words of a 16 x 128 tile stand side by side, so a wave reads 1 KiB an access.
//
// A code is a sign and three bits of magnitude.  As an e4m3 byte these four bits are
// sign * magnitude * 2^-9 (a subnormal, linear in the magnitude), which the
// conversion with a scale of 2^9 takes to the exact whole number in the operand's
// type.  The word holds the first four codes at bits 0-2 and 7 of its bytes and the
// other four the same way, turned left by four bits: one AND, one turn and AND, and
// four conversions of two make an operand of eight, with no offset to correct.
// Products and groups are summed in fp32, a group's sum is scaled by its scale there.
//
// Outputs are few, so a workgroup's waves split the inputs of 16 outputs and add
// their sums in LDS, in a fixed order.

#include <type_traits>

#include "decode_common.hpp"

namespace sah {
namespace {

constexpr int kUnitK = 128;  // inputs of a tile

struct LinearW4Args {
  const void* x;
  const uint32_t* codes;  // [out / 16, in / 128, 64, 4]
  const void* scales;     // [in / group, out]
  const void* bias;
  void* y;
  int64_t rows, x_stride, y_stride;
  int in_tiles, out_tiles;
  int gelu;
};

template <typename T>
__device__ __forceinline__ typename Vec8<T>::type code_operand(uint32_t word) {
  const uint32_t low = word & 0x87878787u;
  const uint32_t high = __builtin_rotateright32(word, 4) & 0x87878787u;
  return e4m3_operand<T>(low, high, 512.0f);
}

template <typename T, int GROUP, int TILES, int SPLIT>
__global__ __launch_bounds__(SPLIT * 64) void linear_w4_kernel(const LinearW4Args a) {
  typedef typename Vec8<T>::type V8;
  typedef typename Vec8<T>::half_type V4;
  constexpr int GROUPS = kUnitK / GROUP;
  constexpr int STEPS = GROUP / 32;  // products of a group
  __shared__ f32x4 part[SPLIT][TILES][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int column = lane & 15, quarter = lane >> 4;
  const uint32_t out_tile = blockIdx.x % (uint32_t)a.out_tiles;
  const int64_t first_row = (int64_t)(blockIdx.x / (uint32_t)a.out_tiles) * (TILES * 16);
  const int64_t out_features = (int64_t)a.out_tiles * 16;

  const u32x4* codes = reinterpret_cast<const u32x4*>(a.codes) + (int64_t)out_tile * a.in_tiles * 64 + lane;
  const T* scales = static_cast<const T*>(a.scales) + (int64_t)out_tile * 16 + quarter * 4;
  const T* x[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const int64_t row = first_row + t * 16 + column;  // columns without a row take the last one's
    x[t] = static_cast<const T*>(a.x) + (row < a.rows ? row : a.rows - 1) * a.x_stride + quarter * 8;
  }

  f32x4 sums[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) sums[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  for (int unit = wave; unit < a.in_tiles; unit += SPLIT) {
    const u32x4 words = codes[(int64_t)unit * 64];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const V4 scale = *reinterpret_cast<const V4*>(scales + ((int64_t)unit * GROUPS + g) * out_features);
      f32x4 group[TILES];
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const V8 w = code_operand<T>(words[g * STEPS + i]);
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          const V8 v = *reinterpret_cast<const V8*>(x[t] + (int64_t)unit * kUnitK + (g * STEPS + i) * 32);
          group[t] = mfma16(w, v, i == 0 ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : group[t]);
        }
      }
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[t][j] = fmaf(group[t][j], to_f32(scale[j]), sums[t][j]);
    }
  }
#pragma unroll
  for (int t = 0; t < TILES; ++t) part[wave][t][lane] = sums[t];
  __syncthreads();

  for (int t = wave; t < TILES; t += SPLIT) {
    const int64_t row = first_row + t * 16 + column;
    if (row >= a.rows) continue;
    f32x4 v = part[0][t][lane];
#pragma unroll
    for (int w = 1; w < SPLIT; ++w) {
      const f32x4 other = part[w][t][lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += other[j];
    }
    const int64_t n = (int64_t)out_tile * 16 + quarter * 4;
    if (a.bias != nullptr) {
      const V4 bias = *reinterpret_cast<const V4*>(static_cast<const T*>(a.bias) + n);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += to_f32(bias[j]);
    }
    V4 out;
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = from_f32<T>(a.gelu ? gelu_exact(v[j]) : v[j]);
    *reinterpret_cast<V4*>(static_cast<T*>(a.y) + row * a.y_stride + n) = out;
  }
}

template <typename T, int GROUP>
int launch_linear_w4(const LinearW4Args& a, hipStream_t stream) {
  const int tiles = a.rows <= 16 ? 1 : a.rows <= 32 ? 2 : 4;
  const int64_t grid = (int64_t)a.out_tiles * ceil_div(a.rows, 16 * tiles);
  constexpr int SPLIT = 8;
  if (grid > (int64_t)(UINT32_MAX / (SPLIT * 64)))
    return fail(SAH_ERR_UNSUPPORTED, "sah_linear_w4: too many rows for one launch");
  const dim3 blocks((unsigned)grid), threads(SPLIT * 64);
  if (tiles == 1)
    hipLaunchKernelGGL((linear_w4_kernel<T, GROUP, 1, SPLIT>), blocks, threads, 0, stream, a);
  else if (tiles == 2)
    hipLaunchKernelGGL((linear_w4_kernel<T, GROUP, 2, SPLIT>), blocks, threads, 0, stream, a);
  else
    hipLaunchKernelGGL((linear_w4_kernel<T, GROUP, 4, SPLIT>), blocks, threads, 0, stream, a);
  return check_hip(hipGetLastError(), "4-bit linear launch");
}

template <typename T>
int dispatch_group(const LinearW4Args& a, int64_t group, hipStream_t stream) {
  return group == 32 ? launch_linear_w4<T, 32>(a, stream)
         : group == 64 ? launch_linear_w4<T, 64>(a, stream)
                       : launch_linear_w4<T, 128>(a, stream);
}

}  // namespace
}  // namespace sah

using namespace sah;

extern "C" int sah_linear_w4(const void* x, const void* codes, const void* scales, const void* bias, void* y,
                             int64_t rows, int64_t in_features, int64_t out_features, int64_t group_size,
                             int64_t x_row_stride, int64_t y_row_stride, int dtype, int activation,
                             sah_stream_t stream) {
  if (dtype != SAH_DTYPE_BF16 && dtype != SAH_DTYPE_F16)
    return fail(SAH_ERR_UNSUPPORTED, "sah_linear_w4: dtype %d is not bf16 or f16", dtype);
  if (activation != SAH_ACTIVATION_NONE && activation != SAH_ACTIVATION_GELU_EXACT)
    return fail(SAH_ERR_UNSUPPORTED, "sah_linear_w4: unknown activation %d", activation);
  if (group_size != 32 && group_size != 64 && group_size != 128)
    return fail(SAH_ERR_UNSUPPORTED, "sah_linear_w4: group_size %lld is not 32, 64 or 128", (long long)group_size);
  if (rows < 0 || in_features <= 0 || out_features <= 0 || in_features > INT32_MAX || out_features > INT32_MAX ||
      rows > ((int64_t)1 << 40))
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_linear_w4: bad sizes");
  if (in_features % kUnitK != 0 || out_features % 16 != 0)
    return fail(SAH_ERR_UNSUPPORTED, "sah_linear_w4: in_features %lld must be a multiple of 128, out_features %lld of 16",
                (long long)in_features, (long long)out_features);
  if (rows == 0) return SAH_OK;
  if (x == nullptr || codes == nullptr || scales == nullptr || y == nullptr)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_linear_w4: null tensor pointer");
  if (!aligned16(x) || !aligned16(codes) || !aligned16(scales) || !aligned16(y) ||
      (reinterpret_cast<uintptr_t>(bias) & 7u) != 0)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_linear_w4: tensors must be 16-byte aligned, bias 8-byte");
  if (x_row_stride % 8 != 0 || y_row_stride % 8 != 0)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_linear_w4: row strides must be multiples of 8 elements");
  LinearW4Args a{};
  a.x = x;
  a.codes = static_cast<const uint32_t*>(codes);
  a.scales = scales;
  a.bias = bias;
  a.y = y;
  a.rows = rows;
  a.x_stride = x_row_stride;
  a.y_stride = y_row_stride;
  a.in_tiles = (int)(in_features / kUnitK);
  a.out_tiles = (int)(out_features / 16);
  a.gelu = activation == SAH_ACTIVATION_GELU_EXACT;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return dtype == SAH_DTYPE_BF16 ? dispatch_group<bf16>(a, group_size, s) : dispatch_group<f16>(a, group_size, s);
}
