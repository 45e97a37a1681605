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

// A workgroup takes OUTS x 16 outputs of TILES x 16 rows; its SPLIT waves share the
// inputs among them, a tile of 128 at a time, and load the next tile while they work
// on this one.  Rows of x are read in whole lines and pass through the wave's own
// part of LDS on their way to the operands (STAGED): a load straight in the operands'
// order touches a line a lane.  Few rows do without.
template <typename T, int GROUP, int TILES, int OUTS, int SPLIT, bool STAGED>
__global__ __launch_bounds__(SPLIT * 64) void linear_w4_kernel(const LinearW4Args a) {
  typedef typename Vec8<T>::type V8;
  typedef typename Vec8<T>::half_type V4;
  constexpr int GROUPS = kUnitK / GROUP;
  constexpr int STEPS = GROUP / 32;  // products of a group
  constexpr int PARTS = SPLIT < 4 ? SPLIT : 4;
  constexpr int PITCH = kUnitK + 8;  // values of a row in LDS: operands' rows fall on different banks
  constexpr int STAGE = STAGED ? TILES * 16 * PITCH : 8;
  union Shared {
    f32x4 part[PARTS][TILES * OUTS][64];
    T stage[SPLIT][STAGE];
  };
  __shared__ Shared shared;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int column = lane & 15, quarter = lane >> 4;
  const uint32_t out_groups = (uint32_t)a.out_tiles / OUTS;
  const uint32_t out_tile = blockIdx.x % out_groups * OUTS;
  const int64_t first_row = (int64_t)(blockIdx.x / out_groups) * (TILES * 16);
  const int64_t out_features = (int64_t)a.out_tiles * 16;

  const u32x4* codes = reinterpret_cast<const u32x4*>(a.codes) + (int64_t)out_tile * a.in_tiles * 64 + lane;
  const T* scales = static_cast<const T*>(a.scales) + (int64_t)out_tile * 16 + quarter * 4;
  // Places without a row take the last one's.
  constexpr int LOADS = STAGED ? TILES * 4 : TILES;
  const T* x[LOADS];
#pragma unroll
  for (int t = 0; t < LOADS; ++t) {
    const int64_t row = first_row + (STAGED ? t * 4 + lane / 16 : t * 16 + column);
    x[t] = static_cast<const T*>(a.x) + (row < a.rows ? row : a.rows - 1) * a.x_stride +
           (STAGED ? lane % 16 : quarter) * 8;
  }

  f32x4 sums[TILES][OUTS];
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int o = 0; o < OUTS; ++o) sums[t][o] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

  u32x4 next_codes[OUTS];
  V4 next_scales[OUTS][GROUPS];
  V8 next_x[TILES * 4];
  auto load = [&](int unit) {
#pragma unroll
    for (int o = 0; o < OUTS; ++o) {
      next_codes[o] = codes[((int64_t)o * a.in_tiles + unit) * 64];
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
        next_scales[o][g] = *reinterpret_cast<const V4*>(scales + ((int64_t)unit * GROUPS + g) * out_features + o * 16);
    }
#pragma unroll
    for (int i = 0; i < TILES * 4; ++i)
      next_x[i] = *reinterpret_cast<const V8*>(x[STAGED ? i : i / 4] + (int64_t)unit * kUnitK + (STAGED ? 0 : i % 4 * 32));
  };
  T* stage = shared.stage[wave];
  if (wave < a.in_tiles) load(wave);
  for (int unit = wave; unit < a.in_tiles; unit += SPLIT) {
    u32x4 words[OUTS];
    V4 scale[OUTS][GROUPS];
    V8 rows[STAGED ? 1 : TILES * 4];
#pragma unroll
    for (int o = 0; o < OUTS; ++o) {
      words[o] = next_codes[o];
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) scale[o][g] = next_scales[o][g];
    }
#pragma unroll
    for (int i = 0; i < TILES * 4; ++i) {
      if (STAGED)
        *reinterpret_cast<V8*>(stage + (i * 4 + lane / 16) * PITCH + lane % 16 * 8) = next_x[i];
      else
        rows[i] = next_x[i];
    }
    if (unit + SPLIT < a.in_tiles) load(unit + SPLIT);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      V8 operand[STEPS][TILES];
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int t = 0; t < TILES; ++t)
          operand[i][t] = STAGED ? *reinterpret_cast<const V8*>(stage + (t * 16 + column) * PITCH +
                                                                (g * STEPS + i) * 32 + quarter * 8)
                                 : rows[STAGED ? 0 : t * 4 + g * STEPS + i];
#pragma unroll
      for (int o = 0; o < OUTS; ++o) {
        f32x4 group[TILES];
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          const V8 w = code_operand<T>(words[o][g * STEPS + i]);
#pragma unroll
          for (int t = 0; t < TILES; ++t)
            group[t] = mfma16(w, operand[i][t], i == 0 ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : group[t]);
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) sums[t][o][j] = fmaf(group[t][j], to_f32(scale[o][g][j]), sums[t][o][j]);
      }
    }
  }
  __syncthreads();  // the sums take the stages' place

  // The waves' sums, in a fixed order: four waves at a time add theirs to those before.
#pragma unroll
  for (int turn = 0; turn < SPLIT / PARTS; ++turn) {
    if (turn != 0) __syncthreads();
    if (wave / PARTS == turn) {
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int o = 0; o < OUTS; ++o) {
          f32x4& place = shared.part[wave % PARTS][t * OUTS + o][lane];
          if (turn == 0) {
            place = sums[t][o];
          } else {
            const f32x4 before = place;
#pragma unroll
            for (int j = 0; j < 4; ++j) sums[t][o][j] += before[j];
            place = sums[t][o];
          }
        }
    }
  }
  __syncthreads();

  for (int i = wave; i < TILES * OUTS; i += SPLIT) {
    const int64_t row = first_row + i / OUTS * 16 + column;
    if (row >= a.rows) continue;
    f32x4 v = shared.part[0][i][lane];
#pragma unroll
    for (int w = 1; w < PARTS; ++w) {
      const f32x4 other = shared.part[w][i][lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += other[j];
    }
    const int64_t n = ((int64_t)out_tile + i % OUTS) * 16 + quarter * 4;
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

template <typename T, int GROUP, int TILES, int OUTS, int SPLIT, bool STAGED>
int launch_tiles(const LinearW4Args& a, hipStream_t stream) {
  const int64_t grid = (int64_t)(a.out_tiles / OUTS) * ceil_div(a.rows, 16 * TILES);
  if (grid > (int64_t)(UINT32_MAX / (SPLIT * 64)))
    return fail(SAH_ERR_UNSUPPORTED, "sah_linear_w4: too many rows for one launch");
  hipLaunchKernelGGL((linear_w4_kernel<T, GROUP, TILES, OUTS, SPLIT, STAGED>), dim3((unsigned)grid), dim3(SPLIT * 64),
                     0, stream, a);
  return check_hip(hipGetLastError(), "4-bit linear launch");
}

// Row tiles by the row count; 16-output tiles of a workgroup by how many there are:
// x is read anew by every workgroup, so as many outputs as still leave the compute
// units one each.  One row reads x in the operands' order (all its lanes read the
// same line).  Measured, us, OUTS 1 / 2 / 4 (SPLIT 8 up to 2, then 4):
//   16 rows  4096 ->  4096   5.5 /  5.9         64 rows  4096 ->  4096  11.5 / 12.9 / 16.1
//    8 rows  4096 ->  8192   7.8 /  6.5         64 rows  4096 ->  8192  23.0 / 13.0 / 16.5
//   16 rows  4096 -> 16384  14.7 / 11.3         64 rows  4096 -> 16384  42.7 / 24.1 / 21.0
//   32 rows  4096 ->  8192  12.4 /  9.1 / 11.0  32 rows  4096 -> 16384  21.6 / 14.4 / 12.5
// and without / with the stage: 1 row 4096 -> 4096 5.05 / 5.33, 13 rows 6.3 / 5.5.
template <typename T, int GROUP>
int launch_linear_w4(const LinearW4Args& a, hipStream_t stream) {
  const int64_t row_tiles = a.rows <= 16 ? 1 : a.rows <= 32 ? 2 : 4;
  const int64_t tiles = a.out_tiles * ceil_div(a.rows, 16 * row_tiles);
  const bool two = tiles >= 512 && a.out_tiles % 2 == 0;
  const bool four = tiles >= 1024 && a.out_tiles % 4 == 0;
  if (a.rows == 1)
    return two ? launch_tiles<T, GROUP, 1, 2, 8, false>(a, stream) : launch_tiles<T, GROUP, 1, 1, 8, false>(a, stream);
  if (row_tiles == 1)
    return two ? launch_tiles<T, GROUP, 1, 2, 8, true>(a, stream) : launch_tiles<T, GROUP, 1, 1, 8, true>(a, stream);
  if (row_tiles == 2)
    return four  ? launch_tiles<T, GROUP, 2, 4, 4, true>(a, stream)
           : two ? launch_tiles<T, GROUP, 2, 2, 8, true>(a, stream)
                 : launch_tiles<T, GROUP, 2, 1, 8, true>(a, stream);
  return four  ? launch_tiles<T, GROUP, 4, 4, 4, true>(a, stream)
         : two ? launch_tiles<T, GROUP, 4, 2, 4, true>(a, stream)
               : launch_tiles<T, GROUP, 4, 1, 8, true>(a, stream);
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
