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
// conversion with a scale of 1/2 takes to the code times 2^-10, exact in the operand's
// type; the outputs take the 2^10 back.  (A group of whole codes times the largest bf16
// values would leave fp32 where its scale brings it back in: 7 * 128 < 2^10.)  The word holds the first four codes at bits 0-2 and 7 of its bytes and the
// other four the same way, turned left by four bits: one AND, one turn and AND, and
// four conversions of two make an operand of eight, with no offset to correct.
// Products and groups are summed in fp32, a group's sum is scaled by its scale there.
//
// Outputs are few, so a workgroup's waves split the inputs of 16 outputs and add
// their sums in LDS, in a fixed order.

#include <type_traits>

#include "decode_common.hpp"
#include "gemm_mainloop.hpp"

namespace sah {
namespace {

constexpr int kUnitK = 128;  // inputs of a tile
constexpr int64_t kMaxRowStride = (int64_t)1 << 25;

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
  return e4m3_operand<T>(low, high, 0.5f);
}

// A workgroup takes OUTS x 16 outputs of TILES x 16 rows; its SPLIT waves share the
// inputs among them, a unit of 128 at a time, the next unit's codes, scales and rows of
// x under way while this one is worked on.  Rows pass through the wave's own part of
// LDS on their way to the operands (STAGED), by direct-to-LDS loads of whole lines: a
// load in the operands' order touches a line a lane.  One row does without.  16-byte
// parts of a row change places by its number, so that the 16 rows of an operand meet no
// bank twice.  A place in LDS is loaded anew when its operands are read, which are the
// unit's, or half of it where the sums leave no registers for more.
//
// Few rows are bound by the codes' latency and way from memory, many by the vector
// units (conversions and scales, 290 of them beside 64 matrix instructions a unit of
// 64 rows and 64 outputs) and the rows' way from L2, 512 KiB a workgroup.
template <typename T, int GROUP, int TILES, int OUTS, int SPLIT, bool STAGED>
__global__ __launch_bounds__(SPLIT * 64) void linear_w4_kernel(const LinearW4Args a) {
  typedef typename Vec8<T>::type V8;
  typedef typename Vec8<T>::half_type V4;
  constexpr int GROUPS = kUnitK / GROUP;
  constexpr int HALF = kUnitK / 2;                 // inputs that x comes in
  constexpr int RUN = GROUP < HALF ? GROUP : HALF;  // inputs summed before their scale
  constexpr int STEPS = RUN / 32;                  // products of a run
  constexpr int RUNS = HALF / RUN;
  constexpr int PARTS = SPLIT < 4 ? SPLIT : 4;
  constexpr bool WHOLE = TILES * OUTS <= 8;  // registers for a unit's operands at once
  constexpr int DMAS = TILES * 2;  // loads of 8 rows of a half
  union Shared {
    f32x4 part[PARTS][TILES * OUTS][64];
    T stage[STAGED ? SPLIT : 1][2][STAGED ? TILES * 16 * HALF : 8];
  };
  __shared__ __align__(16) Shared shared;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int column = lane & 15, quarter = lane >> 4;
  const uint32_t out_groups = (uint32_t)a.out_tiles / OUTS;
  const uint32_t out_tile = blockIdx.x % out_groups * OUTS;
  const int64_t first_row = (int64_t)(blockIdx.x / out_groups) * (TILES * 16);
  const int64_t out_features = (int64_t)a.out_tiles * 16;

  const u32x4* codes = reinterpret_cast<const u32x4*>(a.codes) + (int64_t)out_tile * a.in_tiles * 64 + lane;
  const T* scales = static_cast<const T*>(a.scales) + (int64_t)out_tile * 16 + quarter * 4;
  // Places without a row take the last one's.  Offsets are below 64 rows of at most 2^25.
  const T* x = static_cast<const T*>(a.x) + first_row * a.x_stride;
  uint32_t offset[DMAS];
#pragma unroll
  for (int i = 0; i < DMAS; ++i) {
    const int64_t row = i * 8 + lane / 8, last = a.rows - 1 - first_row;
    offset[i] = (uint32_t)((row < last ? row : last) * a.x_stride * 2) + ((lane ^ (lane >> 4) ^ (i % 2 * 4)) & 7) * 16;
  }
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) T*)&shared.stage[STAGED ? wave : 0][0][0];

  f32x4 sums[TILES][OUTS];
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int o = 0; o < OUTS; ++o) sums[t][o] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

  u32x4 words[2][OUTS];
  V4 scale[2][OUTS][GROUPS];
  V8 rows[STAGED ? 1 : 4];
  auto load_codes = [&](auto of_buffer, int unit) {
    constexpr int B = decltype(of_buffer)::value;
#pragma unroll
    for (int o = 0; o < OUTS; ++o) {
      words[B][o] = codes[((int64_t)o * a.in_tiles + unit) * 64];
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
        scale[B][o][g] = *reinterpret_cast<const V4*>(scales + ((int64_t)unit * GROUPS + g) * out_features + o * 16);
    }
  };
  auto load_x = [&](int half, int unit) {
    if constexpr (STAGED) {
#pragma unroll
      for (int i = 0; i < DMAS; ++i)
        tile_dma16(x + (int64_t)unit * kUnitK + half * HALF, offset[i], lds + half * (TILES * 16 * HALF * 2) + i * 1024);
    } else {
#pragma unroll
      for (int i = half * 2; i < half * 2 + 2; ++i)
        rows[i] = *reinterpret_cast<const V8*>(x + (int64_t)unit * kUnitK + i * 32 + quarter * 8);
    }
  };
  auto step = [&](int unit, auto of_buffer, auto has_next) {
    constexpr int B = decltype(of_buffer)::value;
    constexpr bool NEXT = decltype(has_next)::value;
    // All of the unit has come.  (The compiler, which does not count the direct loads,
    // would wait for the codes after some of the next unit's have been issued.)
    if (STAGED) wait_loads<0>();
#pragma unroll
    for (int o = 0; o < OUTS; ++o) {
      asm volatile("" : "+v"(words[B][o]));
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) asm volatile("" : "+v"(scale[B][o][g]));
    }
    V8 operand[4][TILES];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int i = half * 2; i < (WHOLE ? 4 - half * 2 : half * 2 + 2); ++i)
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          if constexpr (STAGED)
            operand[i][t] = *reinterpret_cast<const V8*>(&shared.stage[wave][i / 2][0] + (t * 16 + column) * HALF +
                                                         (((i % 2 * 4 + quarter) ^ (column >> 1)) & 7) * 8);
          else
            operand[i][t] = rows[i];
        }
      if (NEXT && !(WHOLE && half == 1)) {
        if (STAGED) wait_lds();
        load_x(half, unit + SPLIT);
        if (half == 0) load_codes(std::integral_constant<int, 1 - B>{}, unit + SPLIT);
        if (WHOLE) load_x(1, unit + SPLIT);
      }
#pragma unroll
      for (int o = 0; o < OUTS; ++o) {
#pragma unroll
        for (int r = 0; r < RUNS; ++r) {
          const int g = (half * HALF + r * RUN) / GROUP;
          f32x4 group[TILES];
#pragma unroll
          for (int i = 0; i < STEPS; ++i) {
            const V8 w = code_operand<T>(words[B][o][half * 2 + r * STEPS + i]);
#pragma unroll
            for (int t = 0; t < TILES; ++t)
              group[t] = mfma16(w, operand[half * 2 + r * STEPS + i][t], i == 0 ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : group[t]);
          }
#pragma unroll
          for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) sums[t][o][j] = fmaf(group[t][j], to_f32(scale[B][o][g][j]), sums[t][o][j]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  const std::integral_constant<int, 0> even{};
  const std::integral_constant<int, 1> odd{};
  int unit = wave;
  if (unit < a.in_tiles) {
    load_x(0, unit);
    load_codes(even, unit);
    load_x(1, unit);
  }
  for (; unit + 2 * SPLIT < a.in_tiles; unit += 2 * SPLIT) {
    step(unit, even, std::true_type{});
    step(unit + SPLIT, odd, std::true_type{});
  }
  if (unit + SPLIT < a.in_tiles) {
    step(unit, even, std::true_type{});
    step(unit + SPLIT, odd, std::false_type{});
  } else if (unit < a.in_tiles) {
    step(unit, even, std::false_type{});
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
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= 1024.0f;
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
// same line).  Measured, us, OUTS 1 / 2 / 4 as instantiated below, group 128, weights
// from memory:
//    1 row   4096 ->  4096   4.9 /  5.5 /  7.5    4096 -> 16384  13.1 / 10.7 / 10.0
//   16 rows  4096 ->  4096   5.6 /  6.2 /  8.0    4096 -> 16384  14.8 / 12.1 / 10.5
//   32 rows  4096 ->  8192  11.8 /  8.6 / 11.5    4096 -> 16384  21.2 / 14.8 / 13.1
//   64 rows  4096 ->  4096  10.7 / 11.4 / 14.2    4096 -> 16384  38.1 / 21.3 / 17.0
//   64 rows  4096 ->  8192  19.6 / 12.2 / 14.9
// (the last of 64 rows: 36 MB, 2.1 TB/s, 505 TFLOP/s), and 1 row 4096 -> 4096 without
// / with the stage 5.05 / 5.33, 13 rows 6.3 / 5.5.
template <typename T, int GROUP>
int launch_linear_w4(const LinearW4Args& a, hipStream_t stream) {
  const int64_t row_tiles = a.rows <= 16 ? 1 : a.rows <= 32 ? 2 : 4;
  const int64_t tiles = a.out_tiles * ceil_div(a.rows, 16 * row_tiles);
  const bool two = tiles >= 512 && a.out_tiles % 2 == 0;
  const bool four = tiles >= 1024 && a.out_tiles % 4 == 0;
  if (a.rows == 1)
    return four  ? launch_tiles<T, GROUP, 1, 4, 8, false>(a, stream)
           : two ? launch_tiles<T, GROUP, 1, 2, 8, false>(a, stream)
                 : launch_tiles<T, GROUP, 1, 1, 8, false>(a, stream);
  if (row_tiles == 1)
    return four  ? launch_tiles<T, GROUP, 1, 4, 8, true>(a, stream)
           : two ? launch_tiles<T, GROUP, 1, 2, 8, true>(a, stream)
                 : launch_tiles<T, GROUP, 1, 1, 8, true>(a, stream);
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
  if (rows > 1 && (x_row_stride < 0 || x_row_stride > kMaxRowStride))
    return fail(SAH_ERR_UNSUPPORTED, "sah_linear_w4: rows of x %lld elements apart", (long long)x_row_stride);
  if (x_row_stride % 8 != 0 || y_row_stride % 8 != 0)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_linear_w4: row strides must be multiples of 8 elements");
  if (rows > 1 && y_row_stride < out_features)
    return fail(SAH_ERR_INVALID_ARGUMENT, "sah_linear_w4: rows of y overlap (%lld elements apart)",
                (long long)y_row_stride);
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
