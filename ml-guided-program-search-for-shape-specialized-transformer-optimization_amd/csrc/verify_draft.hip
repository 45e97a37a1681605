// Verification of drafted tokens against the target's probabilities, for gfx950 (CDNA4).
//
// p_i = softmax(target row i / temperature), q_i = softmax(draft row i / temperature), or
// all of q_i at draft token x_i where the drafts have no probabilities.  Draft i stands
// where u_i q_i(x_i) < p_i(x_i) and every draft before it stands.  With j the first that
// does not, the next token is drawn from max(p_j - q_j, 0), or from p_j where all stand:
// the lowest v whose sum of weights up to v is above u times the sum of them all.  The
// tokens so chosen are distributed as if drawn from the target one by one.
//
// A token is chosen at a border between two, of which there are as many as tokens: sums
// wrong by 1e-7, as fp32 leaves them, choose another token once in 10^7 / vocabulary
// requests.  The choice here is that of exact arithmetic, but for borders closer than some
// 1e-14 of p's mass (an exponential of fp64 is off by 2^-51 and its exponent's rounding, some
// 1e-15; of the whole that max(p - q, 0) has, 1e-14 over how far p and q lie apart: 1e-8
// where they differ by 1e-6):
//   1. rows: a chunk of a row's largest logit and sum of exponentials, in fp32 (a row's
//      sum comes out right to kFastError).  The one pass over all logits, bound by them;
//   2. decide: p_i(x_i), q_i(x_i) from these; where the test's two sides lie within
//      that error, from sums in fp64.  j is known;
//   3. weigh: of row j alone, in fp64.  With e_p, e_q the exponentials and r = sum e_p /
//      sum e_q, the weights are in proportion to max(e_p - r e_q, 0).  r is known to
//      fp32's precision; a chunk adds up e_p, e_q, and both over the tokens S where
//      e_p > r e_q, and keeps how near e_p / e_q comes to r.  Its weight is then sum_S e_p
//      - r sum_S e_q for the r that the sums of all chunks give, unless a token changes
//      sides between the two;
//   4. pick: r, such chunks again (one in some thousand draws, or many where draft and
//      target are all but the same), the chunk in which the sum passes the border, the token.
//
// 64 requests, 7 drafts, 131072 tokens, bf16 (252 MB, 51 us at a large copy's rate): rows
// 53 us, decide 7, weigh 20, pick 5.4.  The draw's two parts in one launch, by the
// request's last workgroup, took 106 us instead of 27, as each of the 4096 releases its
// L2's lines.  All rows in fp64 took 126 us (some 80 with the exponential as it is now, 24
// instructions of four cycles a logit).  For one request (4 drafts, 32000 tokens) the parts
// are latencies, 4 + 11 us.

#include <type_traits>

#include "sah_common.hpp"

namespace sah {
namespace {

constexpr int kVec = 8;  // logits of one access
constexpr int kRowThreads = 256;
constexpr int kAccesses = 4;  // of a thread
constexpr int kRowChunk = kRowThreads * kVec * kAccesses;
constexpr int kDecideThreads = 1024;
constexpr int kPickThreads = 256;
constexpr int kPickChunk = kPickThreads * kVec;
constexpr int kMaxDrafts = 1024;
// Workgroups of the draw up to which each decides for itself, for a launch less: one request
// of 32000 tokens and 4 drafts 7.1 us instead of 4.6 + 4.0, 8 of 131072 tokens and 3 drafts
// (512) 8.9 instead of 6.0 + 5.2; 16 with 7 drafts (1024) 14.4 and 6.4 + 7.0.
constexpr int64_t kFewWorkgroups = 512;
// And up to which a request's last one also draws, for another: 16 11.4 us instead of 7.1 +
// 4.1, 125 9.4 instead of 5.5 + 3.7, 128 12.9 instead of 7.0 + 4.4, where a launch is 3 us
// of the host's; 256 15.6 instead of 7.2 + 4.5, 512 21 instead of 8.9 + 5.1, as each
// releases its L2's lines.  (A captured step has no such launch to save: it gains nothing
// and pays 1.5 us at 128.)
constexpr int64_t kFewestWorkgroups = 128;
enum { kDecided = 0, kDecides = 1, kDraws = 2 };
constexpr double kLog2e = 1.4426950408889634074;
// A row's sum in fp32, relative: an exponent |x| <= 64 (what lies below adds less than
// 2^-33) is off by its difference's, its factor's and its product's rounding, 3 * 64 *
// 2^-24 ln 2 = 8e-6; v_exp_f32 by 2^-22, 32 additions by 2e-6.  Two rows: 2^-15.
constexpr double kFastError = 1.0 / 32768.0;

struct RowPart {
  double sum;  // of exp2((l - top) c); NaN where a logit is NaN or +inf
  float top;   // the largest logit
  int32_t at;  // its lowest place (greedy requests)
};

// What the decision leaves for the draw, of one request.
struct Choice {
  int32_t row;      // the first draft that does not stand, or the number of drafts
  int32_t mode;     // how the next token is drawn
  float p_top, q_top;
  double ratio_log2;  // of sum e_p / sum e_q, about
  double c;         // log2(e) / temperature
  int32_t parted;   // workgroups of the request's draw that have left their sums
};
enum { kDone = 0, kFromTarget = 1, kWithout = 2, kResample = 3 };

struct Weights {
  double p, q;          // sums of e_p, e_q
  double p_over, q_over;  // where e_p > ratio e_q
  float near;             // the least distance of a token's e_p / e_q from ratio, in log2
};

struct VerifyArgs {
  const void* target;
  const void* draft;
  const int64_t* tokens;
  const float* uniforms;
  const int32_t* counts;
  const float* temperatures;
  int64_t* answer;
  int32_t* accepted;
  int64_t t_sb, t_ss, d_sb, d_ss;
  RowPart* parts;     // [batch][drafts + 1 (+ drafts)][row_chunks]
  Weights* weights;   // [batch][pick_chunks]
  Choice* choices;    // [batch]
  int batch, drafts, vocab, row_chunks, pick_chunks;
};

// 2^x for x <= 0, 0 from below the smallest number on (and for NaN, which no row that is
// drawn from has): x = n + f with |f| <= 1/2, and for 2^f the polynomial that meets it at
// the 11 Chebyshev points of that interval, off by 2^-51 of it.  Its coefficients stay in
// scalar registers, out of the compiler's sight: as literals each takes two moves beside
// the fma that adds it (weigh of 64 requests of 131072 tokens 25 us instead of 19.6).
struct Exp2 {
  double k[10];
  __device__ __forceinline__ Exp2()
      : k{0x1.e6063f7217bc6p-28, 0x1.b675bca4eeebbp-24, 0x1.62bfd47773353p-20, 0x1.ffcb54062e698p-17,
          0x1.430913096fd9fp-13, 0x1.5d87fe9d7a584p-10, 0x1.3b2ab6fba1ddap-7,  0x1.c6b08d703ce49p-5,
          0x1.ebfbdff82c598p-3,  0x1.62e42fefa3a19p-1} {
#pragma unroll
    for (int i = 0; i < 10; ++i) asm("" : "+s"(k[i]));
  }
  __device__ __forceinline__ double operator()(double x) const {
    x = fmax(x, -1100.0);
    const double n = __builtin_rint(x);
    const double f = x - n;
    double y = k[0];
#pragma unroll
    for (int i = 1; i < 10; ++i) y = fma(y, f, k[i]);
    return ldexp(fma(y, f, 1.0), (int)n);
  }
};
__device__ __forceinline__ double exponent_of(float logit, float top, double c) {
  return ((double)logit - (double)top) * c;
}

// log2(e) / temperature, and whether the request answers greedily instead (a temperature
// that is not above 0).  At least fp32's smallest normal number, for the rows' exponents:
// an infinite temperature keeps masked logits at weight 0, and only logits that lie 1e36 and
// more apart tell it, or one above 1.2e38, from 1.2e38.
__device__ __forceinline__ bool is_greedy(const VerifyArgs& a, int64_t b, double& c) {
  const float t = a.temperatures != nullptr ? a.temperatures[b] : 1.0f;
  if (!(t > 0.0f)) {
    c = kLog2e;
    return true;
  }
  c = kLog2e / (double)t;
  if (c < 0x1p-126) c = 0x1p-126;
  return false;
}

// Drafts of request b, or -1 where it takes no part.
__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int64_t b) {
  if (a.counts == nullptr) return a.drafts;
  const int count = a.counts[b];
  return count < 0 ? -1 : count < a.drafts ? count : a.drafts;
}

typedef uint32_t LooseWords __attribute__((ext_vector_type(4), aligned(2)));

// Logits [at, at + 8) of a row as fp32; -inf from the row's end on.  Rows start at any
// element.  ONCE: past the caches, which the pass over all rows would fill with what nothing
// reads again.  Rows of 64 requests in turn with other inputs 53 us instead of 56, weigh
// 20.1 instead of 19.5; of logits just written, 32 requests 25.4 instead of 26.2, 64 51 and
// 51, 128 97 instead of 115; of the same logits again and again 28.7 instead of 26.7, 52 instead
// of 47, 93 instead of 96.  At every size, without a border: logits that come from memory, or
// that the model has just written, are a program's case and gain or lose nothing, and
// smaller batches than these are bound by latency.
template <typename T, bool ONCE = false>
__device__ __forceinline__ void load_logits(const T* row, int64_t at, int64_t vocab, float* out) {
  if (at + kVec <= vocab) {
    T raw[kVec];
    if constexpr (ONCE) {
#pragma unroll
      for (int i = 0; i < (int)(sizeof(raw) / 16); ++i) {
        const LooseWords words = __builtin_nontemporal_load(reinterpret_cast<const LooseWords*>(row + at) + i);
        __builtin_memcpy(reinterpret_cast<char*>(raw) + 16 * i, &words, 16);
      }
    } else {
      __builtin_memcpy(raw, row + at, sizeof(raw));
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) out[e] = to_f32(raw[e]);
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) out[e] = at + e < vocab ? to_f32(row[at + e]) : -INFINITY;
  }
}

// Values of other lanes: within 16 by DPP (lane ^ 1, lane ^ 2, 7 - lane of 8, 15 - lane),
// which takes no trip through LDS; across 16 and 32 by the lane swaps, whose two results
// are the two partners of every lane.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __uint_as_float(dpp<CTRL>(__float_as_uint(v)));
}
template <int CTRL>
__device__ __forceinline__ int32_t dpp(int32_t v) {
  return (int32_t)dpp<CTRL>((uint32_t)v);
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
  const u32x2 w = __builtin_bit_cast(u32x2, v);
  return __builtin_bit_cast(double, (u32x2){dpp<CTRL>(w[0]), dpp<CTRL>(w[1])});
}
template <int LANES>
__device__ __forceinline__ void swap_lanes(uint32_t v, uint32_t& a, uint32_t& b) {
  const u32x2 r = LANES == 16 ? __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(v, v, false, false))
                              : __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(v, v, false, false));
  a = r[0];
  b = r[1];
}
template <int LANES>
__device__ __forceinline__ void swap_lanes(float v, float& a, float& b) {
  uint32_t x, y;
  swap_lanes<LANES>(__float_as_uint(v), x, y);
  a = __uint_as_float(x);
  b = __uint_as_float(y);
}
template <int LANES>
__device__ __forceinline__ void swap_lanes(int32_t v, int32_t& a, int32_t& b) {
  uint32_t x, y;
  swap_lanes<LANES>((uint32_t)v, x, y);
  a = (int32_t)x;
  b = (int32_t)y;
}
template <int LANES>
__device__ __forceinline__ void swap_lanes(double v, double& a, double& b) {
  const u32x2 w = __builtin_bit_cast(u32x2, v);
  u32x2 x, y;
  uint32_t x0, x1, y0, y1;
  swap_lanes<LANES>(w[0], x0, y0);
  swap_lanes<LANES>(w[1], x1, y1);
  x = (u32x2){x0, x1};
  y = (u32x2){y0, y1};
  a = __builtin_bit_cast(double, x);
  b = __builtin_bit_cast(double, y);
}
// op over the wave, in every lane.
template <typename V, typename Op>
__device__ __forceinline__ V wave_reduce(V v, Op op) {
  v = op(v, dpp<0xB1>(v));
  v = op(v, dpp<0x4E>(v));
  v = op(v, dpp<0x141>(v));
  v = op(v, dpp<0x140>(v));
  V a, b;
  swap_lanes<16>(v, a, b);
  v = op(a, b);
  swap_lanes<32>(v, a, b);
  return op(a, b);
}
template <typename V>
__device__ __forceinline__ V wave_add(V v) {
  return wave_reduce(v, [](V a, V b) { return a + b; });
}
__device__ __forceinline__ float wave_largest(float v) {
  return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ int32_t wave_lowest(int32_t v) {
  return wave_reduce(v, [](int32_t a, int32_t b) { return b < a ? b : a; });
}
// The sum over the lanes up to this one: within 16 by shifts, then the last lanes of the
// 16 and the 32 before.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_or_zero(double v) {
  const u32x2 w = __builtin_bit_cast(u32x2, v);
  const u32x2 r = {(uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[0], CTRL, ROWS, 0xF, false),
                   (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[1], CTRL, ROWS, 0xF, false)};
  return __builtin_bit_cast(double, r);
}
__device__ __forceinline__ double wave_up_to(double v) {
  v += dpp_or_zero<0x111, 0xF>(v);
  v += dpp_or_zero<0x112, 0xF>(v);
  v += dpp_or_zero<0x114, 0xF>(v);
  v += dpp_or_zero<0x118, 0xF>(v);
  v += dpp_or_zero<0x142, 0xA>(v);
  v += dpp_or_zero<0x143, 0xC>(v);
  return v;
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void verify_rows_kernel(const VerifyArgs a) {
  constexpr int WAVES = kRowThreads / 64;
  __shared__ float tops[WAVES];
  __shared__ float sums[WAVES];
  __shared__ int32_t places[WAVES];
  const int rows = a.drafts + 1 + (a.draft != nullptr ? a.drafts : 0);
  const uint32_t chunk = blockIdx.x % (uint32_t)a.row_chunks;
  const uint32_t request_row = blockIdx.x / (uint32_t)a.row_chunks;
  const int64_t b = request_row / (uint32_t)rows;
  const int r = (int)(request_row % (uint32_t)rows);
  const int tid = threadIdx.x, wave = tid >> 6;
  const int count = drafts_of(a, b);
  if (r == 0 && chunk == 0 && tid == 0) a.choices[b].parted = 0;
  const bool is_draft = r > a.drafts;
  if (is_draft ? r - a.drafts - 1 >= count : r > count) return;
  double factor;
  const bool greedy = is_greedy(a, b, factor);
  if (greedy && is_draft) return;  // a greedy request's draft stands by the target alone
  const T* row = is_draft ? static_cast<const T*>(a.draft) + b * a.d_sb + (r - a.drafts - 1) * a.d_ss
                          : static_cast<const T*>(a.target) + b * a.t_sb + r * a.t_ss;
  const int64_t first = (int64_t)chunk * kRowChunk + tid * kVec;
  float l[kAccesses][kVec];
#pragma unroll
  for (int i = 0; i < kAccesses; ++i) load_logits<T, true>(row, first + (int64_t)i * kRowThreads * kVec, a.vocab, l[i]);
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kAccesses; ++i)
#pragma unroll
    for (int e = 0; e < kVec; ++e) top = fmaxf(top, l[i][e]);
  top = wave_largest(top);
  if ((tid & 63) == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, tops[w]);
  // Differences of -inf from -inf would be NaN, which stands for a bad logit; from +inf
  // they are meant to be.
  const float base = top == -INFINITY ? 0.0f : top;
  const float c = fminf((float)factor, 3e38f);
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kAccesses; ++i)
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum += __builtin_amdgcn_exp2f((l[i][e] - base) * c);
  int32_t at = INT32_MAX;
  if (greedy) {
#pragma unroll
    for (int i = kAccesses - 1; i >= 0; --i)
#pragma unroll
      for (int e = kVec - 1; e >= 0; --e)
        if (l[i][e] == top) at = (int32_t)(first + (int64_t)i * kRowThreads * kVec + e);
    at = wave_lowest(at);
  }
  sum = wave_add(sum);
  if ((tid & 63) == 0) {
    sums[wave] = sum;
    places[wave] = at;
  }
  __syncthreads();
  if (tid == 0) {
    double total = (double)sum;
    for (int w = 1; w < WAVES; ++w) {
      total += (double)sums[w];
      at = places[w] < at ? places[w] : at;
    }
    RowPart* part = a.parts + (int64_t)request_row * a.row_chunks + chunk;
    part->sum = total;
    part->top = top;
    part->at = at;
  }
}

// A row's statistics from its chunks', by one wave.
struct RowSum {
  double sum;
  float top;
  int32_t at;
  __device__ bool there() const { return top > -INFINITY && top < INFINITY && sum == sum; }
};
__device__ __forceinline__ RowSum merge_row(const RowPart* parts, int chunks, double c, const Exp2& power) {
  const int lane = threadIdx.x & 63;
  RowPart part{0.0, -INFINITY, INT32_MAX};
  if (lane < chunks) part = parts[lane];
  float top = part.top;
  for (int i = lane + 64; i < chunks; i += 64) top = fmaxf(top, parts[i].top);
  top = wave_largest(top);
  double sum = 0.0;
  int32_t at = INT32_MAX;
  for (int i = lane; i < chunks; i += 64) {
    if (i != lane) part = parts[i];
    // (a sum that is NaN stays it)
    if (part.sum != 0.0) sum += part.sum * power(exponent_of(part.top, top, c));
    if (part.top == top && part.at < at) at = part.at;
  }
  return {wave_add(sum), top, wave_lowest(at)};
}

// What the threads of a workgroup that decides tell each other.
struct Seen {
  RowSum p, q;
  int32_t stands;  // 1: the draft stands, 0: it does not, -1: too near to say
  int32_t none;    // 1: no distribution to draw from
};
template <int THREADS>
struct DecideShared {
  Seen seen[THREADS / 64];
  double sums[THREADS / 64];
};

// A row's sum of exponentials in fp64, by the workgroup.
template <typename T, int THREADS>
__device__ double exact_sum(const T* row, float top, double c, int64_t vocab, const Exp2& power,
                            DecideShared<THREADS>& shared) {
  double sum = 0.0;
  for (int64_t at = (int64_t)threadIdx.x * kVec; at < vocab; at += THREADS * kVec) {
    float l[kVec];
    load_logits<T>(row, at, vocab, l);
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum += power(exponent_of(l[e], top, c));
  }
  sum = wave_add(sum);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) shared.sums[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < THREADS / 64; ++w) sum += shared.sums[w];
  return sum;
}

// Request b's decision by a workgroup, which leaves what it answers already where it
// `writes`.  A wave takes a row of the target, with the draft's beside it; as many rows at
// a time as there are waves, up to the first draft that does not stand.
template <typename T, int THREADS>
__device__ Choice decide(const VerifyArgs& a, int64_t b, bool writes, DecideShared<THREADS>& shared) {
  constexpr int WAVES = THREADS / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int count = drafts_of(a, b);
  int64_t* answer = a.answer + b * (a.drafts + 1);
  if (count < 0) {
    if (writes) {
      for (int i = tid; i <= a.drafts; i += THREADS) answer[i] = -1;
      if (tid == 0) a.accepted[b] = -1;
    }
    return {0, kDone, 0.0f, 0.0f, 0.0, 0.0, 0};
  }
  double c;
  const bool greedy = is_greedy(a, b, c);
  const bool sampled = a.draft != nullptr && !greedy;
  const int rows = a.drafts + 1 + (a.draft != nullptr ? a.drafts : 0);
  const RowPart* parts = a.parts + b * rows * a.row_chunks;
  const T* target = static_cast<const T*>(a.target) + b * a.t_sb;
  const T* draft = static_cast<const T*>(a.draft) + b * a.d_sb;
  const int64_t* tokens = a.tokens + b * a.drafts;
  const float* uniforms = a.uniforms + b * (a.drafts + 1);

  const Exp2 power;
  int j = -1;
  Seen found{};
  for (int first = 0; j < 0; first += WAVES) {
    const int i = first + wave;
    if (i <= count) {
      const int64_t token = i < count ? tokens[i] : -1;
      const bool known = token >= 0 && token < a.vocab;
      float p_logit = 0.0f, q_logit = 0.0f;
      if (known) p_logit = to_f32(target[i * a.t_ss + token]);
      if (known && sampled) q_logit = to_f32(draft[i * a.d_ss + token]);
      Seen mine{};
      mine.p = merge_row(parts + (int64_t)i * a.row_chunks, a.row_chunks, c, power);
      mine.q = {1.0, 0.0f, 0};
      if (sampled && i < count) mine.q = merge_row(parts + (int64_t)(a.drafts + 1 + i) * a.row_chunks, a.row_chunks, c, power);
      mine.none = mine.p.there() && mine.q.there() ? 0 : 1;
      if (mine.none == 0 && known) {
        if (greedy) {
          mine.stands = mine.p.at == token ? 1 : 0;
        } else {
          const double p = power(exponent_of(p_logit, mine.p.top, c)) / mine.p.sum;
          double q = (double)uniforms[i];
          if (sampled) q *= power(exponent_of(q_logit, mine.q.top, c)) / mine.q.sum;
          mine.stands = fabs(q - p) <= kFastError * p && p > 0.0 ? -1 : q < p ? 1 : 0;
        }
      }
      if (lane == 0) shared.seen[wave] = mine;
    }
    __syncthreads();
    for (int w = 0; w < WAVES && j < 0; ++w) {
      const int at = first + w;
      int stands = shared.seen[w].stands;
      if (stands < 0) {  // (the same for every thread)
        const int64_t token = tokens[at];
        const Seen& it = shared.seen[w];
        const T* p_row = target + at * a.t_ss;
        const double p =
            power(exponent_of(to_f32(p_row[token]), it.p.top, c)) / exact_sum<T>(p_row, it.p.top, c, a.vocab, power, shared);
        double q = (double)uniforms[at];
        if (sampled) {
          const T* q_row = draft + at * a.d_ss;
          q *= power(exponent_of(to_f32(q_row[token]), it.q.top, c)) / exact_sum<T>(q_row, it.q.top, c, a.vocab, power, shared);
        }
        stands = q < p ? 1 : 0;
      }
      if (stands == 0 || at == count) {
        j = at;
        found = shared.seen[w];
      }
    }
    __syncthreads();
  }

  const bool done = greedy || found.none != 0;
  if (writes) {
    for (int i = tid; i <= a.drafts; i += THREADS) {
      if (i < j)
        answer[i] = tokens[i];
      else if (i > j || done)  // answer[j] is the draw's otherwise
        answer[i] = i == j && found.none == 0 ? found.p.at : -1;
    }
    if (tid == 0) a.accepted[b] = j;
  }
  Choice choice{j, kDone, found.p.top, found.q.top, 0.0, c, 0};
  if (!done) choice.mode = j == count ? kFromTarget : sampled ? kResample : kWithout;
  if (choice.mode == kResample) choice.ratio_log2 = log2(found.p.sum / found.q.sum);
  return choice;
}

template <typename T>
__global__ __launch_bounds__(kDecideThreads) void verify_decide_kernel(const VerifyArgs a) {
  __shared__ DecideShared<kDecideThreads> shared;
  const Choice it = decide<T>(a, blockIdx.x, true, shared);
  if (threadIdx.x == 0) a.choices[blockIdx.x] = it;
}

// e_p and e_q of 8 tokens (e_q: 0 where it takes no part); zeros behind the row's end.
template <typename T>
struct Rows {
  const T* p_row;
  const T* q_row;
  int64_t drafted;  // the token that a certain draft takes out
  Exp2 power;
  __device__ Rows(const VerifyArgs& a, int64_t b, const Choice& it) {
    p_row = static_cast<const T*>(a.target) + b * a.t_sb + it.row * a.t_ss;
    q_row = static_cast<const T*>(a.draft) + b * a.d_sb + it.row * a.d_ss;
    drafted = it.mode == kWithout ? a.tokens[b * a.drafts + it.row] : -1;
  }
  // apart: log2 of e_p / e_q over ratio, +inf without a draft's row (NaN where both are 0)
  __device__ __forceinline__ void weigh(const VerifyArgs& a, const Choice& it, int64_t first, double* p, double* q,
                                        double* apart) const {
    float pl[kVec], ql[kVec];
    load_logits<T>(p_row, first, a.vocab, pl);
    if (it.mode == kResample) load_logits<T>(q_row, first, a.vocab, ql);
    if (it.mode == kResample) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const double x = exponent_of(pl[e], it.p_top, it.c), y = exponent_of(ql[e], it.q_top, it.c);
        p[e] = power(x);
        q[e] = power(y);
        apart[e] = x - y - it.ratio_log2;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        p[e] = power(exponent_of(first + e == drafted ? -INFINITY : pl[e], it.p_top, it.c));
        q[e] = 0.0;
        apart[e] = INFINITY;
      }
    }
  }
};

// The weights of 8 tokens with the ratio as it is, and their sum.
template <typename T>
__device__ __forceinline__ double weigh_exactly(const Rows<T>& rows, const VerifyArgs& a, const Choice& it, int64_t first,
                                                double ratio, double* p) {
  double q[kVec], apart[kVec], sum = 0.0;
  rows.weigh(a, it, first, p, q, apart);
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    p[e] -= ratio * q[e];
    p[e] = p[e] > 0.0 ? p[e] : 0.0;
    sum += p[e];
  }
  return sum;
}

// Request b's draw from its chunks' sums, by a workgroup.
template <typename T>
__device__ void pick(const VerifyArgs& a, int64_t b, const Choice& it) {
  constexpr int WAVES = kPickThreads / 64;
  __shared__ double sums[WAVES];
  __shared__ int32_t picks[WAVES], lasts[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Weights* weights = a.weights + b * a.pick_chunks;
  const Rows<T> rows(a, b, it);

  // Every wave for itself: the ratio, the whole, and the chunk in which the sum passes
  // u times the whole.
  double ratio = 0.0;
  if (it.mode == kResample) {
    double p = 0.0, q = 0.0;
    for (int i = lane; i < a.pick_chunks; i += 64) {
      p += weights[i].p;
      q += weights[i].q;
    }
    ratio = wave_add(p) / wave_add(q);
    // Chunks where a token may have changed sides, again (exponents are off by 2^-53 of
    // at most 1100 each, as far as they matter, and near by 2^-24 of itself).
    const double moved = fabs(log2(ratio) - it.ratio_log2) * 1.000001 + 1e-12;
    for (int at = 0; at < a.pick_chunks; at += 64) {
      uint64_t again = __ballot(at + lane < a.pick_chunks && weights[at + lane].near <= moved);
      while (again != 0) {  // (the same for every wave)
        const int i = at + __ffsll((unsigned long long)again) - 1;
        again &= again - 1;
        double p[kVec];
        const double up_to = wave_add(weigh_exactly<T>(rows, a, it, (int64_t)i * kPickChunk + tid * kVec, ratio, p));
        if (lane == 0) sums[wave] = up_to;
        __syncthreads();
        if (tid == 0) {
          double sum = 0.0;
          for (int w = 0; w < WAVES; ++w) sum += sums[w];
          weights[i].p_over = sum;
          weights[i].q_over = 0.0;
        }
        __syncthreads();
      }
    }
  }
  auto weight = [&](int i) {
    if (i >= a.pick_chunks) return 0.0;
    const double w = weights[i].p_over - ratio * weights[i].q_over;
    return w > 0.0 ? w : 0.0;
  };
  double whole = 0.0;
  for (int i = lane; i < a.pick_chunks; i += 64) whole += weight(i);
  whole = wave_add(whole);
  const double bound = (double)a.uniforms[b * (a.drafts + 1) + a.drafts] * whole;
  double before = 0.0, start = 0.0;
  int chosen = -1;
  for (int at = 0; at < a.pick_chunks; at += 64) {
    const double w = weight(at + lane);
    const double up_to = wave_up_to(w);
    const uint64_t some = __ballot(w > 0.0);
    const uint64_t above = __ballot(w > 0.0 && before + up_to > bound);
    if (some != 0) {  // (the last one with a weight, should none pass the border)
      const int k = above != 0 ? __ffsll((unsigned long long)above) - 1 : 63 - __clzll((long long)some);
      chosen = at + k;
      start = __shfl(before + (up_to - w), k);
    }
    if (above != 0) break;
    before += __shfl(up_to, 63);
  }
  int64_t* answer = a.answer + b * (a.drafts + 1) + it.row;
  if (chosen < 0) {  // nothing has a weight
    if (tid == 0) *answer = -1;
    return;
  }

  const int64_t first = (int64_t)chosen * kPickChunk + tid * kVec;
  double p[kVec];
  const double own = weigh_exactly<T>(rows, a, it, first, ratio, p);
  const double up_to = wave_up_to(own);
  if (lane == 63) sums[wave] = up_to;
  __syncthreads();
  double run = start + (up_to - own);
  for (int w = 0; w < wave; ++w) run += sums[w];
  int32_t found = INT32_MAX, last = -1;
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    run += p[e];
    if (p[e] > 0.0) {
      last = (int32_t)(first + e);
      if (run > bound && found == INT32_MAX) found = last;
    }
  }
  found = wave_lowest(found);
  last = -wave_lowest(-last);
  if (lane == 0) {
    picks[wave] = found;
    lasts[wave] = last;
  }
  __syncthreads();
  if (tid != 0) return;
  for (int w = 1; w < WAVES; ++w) {
    found = picks[w] < found ? picks[w] : found;
    last = lasts[w] > last ? lasts[w] : last;
  }
  *answer = found != INT32_MAX ? found : last;
}

template <typename T>
__global__ __launch_bounds__(kPickThreads) void verify_pick_kernel(const VerifyArgs a) {
  const Choice it = a.choices[blockIdx.x];
  if (it.mode != kDone) pick<T>(a, blockIdx.x, it);
}

// HOW: from kDecides on every workgroup decides for itself, and with kDraws a request's last
// one draws.
template <typename T, int HOW>
__global__ __launch_bounds__(kPickThreads) void verify_weigh_kernel(const VerifyArgs a) {
  constexpr int WAVES = kPickThreads / 64;
  __shared__ Weights waves[WAVES];
  const uint32_t chunk = blockIdx.x % (uint32_t)a.pick_chunks;
  const int64_t b = blockIdx.x / (uint32_t)a.pick_chunks;
  Choice it;
  if constexpr (HOW >= kDecides) {
    __shared__ DecideShared<kPickThreads> shared;
    it = decide<T>(a, b, chunk == 0, shared);
    if (HOW == kDecides && chunk == 0 && threadIdx.x == 0) a.choices[b] = it;
  } else {
    it = a.choices[b];
  }
  if (it.mode == kDone) return;
  const Rows<T> rows(a, b, it);
  double p[kVec], q[kVec], apart[kVec];
  rows.weigh(a, it, (int64_t)chunk * kPickChunk + threadIdx.x * kVec, p, q, apart);
  Weights sum{0.0, 0.0, 0.0, 0.0, INFINITY};
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    sum.p += p[e];
    sum.q += q[e];
    const bool over = apart[e] > 0.0;
    sum.p_over += over ? p[e] : 0.0;
    sum.q_over += over ? q[e] : 0.0;
    sum.near = fminf(sum.near, fabsf((float)apart[e]));
  }
  sum.p_over = wave_add(sum.p_over);
  if (it.mode == kResample) {
    sum.p = wave_add(sum.p);
    sum.q = wave_add(sum.q);
    sum.q_over = wave_add(sum.q_over);
    sum.near = wave_reduce(sum.near, [](float a, float b) { return fminf(a, b); });
  }
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < WAVES; ++w) {
      sum.p += waves[w].p;
      sum.q += waves[w].q;
      sum.p_over += waves[w].p_over;
      sum.q_over += waves[w].q_over;
      sum.near = fminf(sum.near, waves[w].near);
    }
    a.weights[b * a.pick_chunks + chunk] = sum;
  }
  if constexpr (HOW == kDraws) {
    __shared__ bool is_last;
    if (threadIdx.x == 0) {
      __threadfence();
      is_last = atomicAdd(&a.choices[b].parted, 1) == a.pick_chunks - 1;
    }
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    pick<T>(a, b, it);
  }
}

struct Layout {
  int64_t row_chunks, pick_chunks, rows;
  size_t weights, choices, bytes;
};
// Where the parts stand in the workspace; false for sizes that no launch takes.
bool lay_out(int64_t batch, int64_t drafts, int64_t vocab, bool sampled, Layout& out) {
  if (batch < 0 || drafts < 0 || drafts > kMaxDrafts || vocab <= 0 || vocab > INT32_MAX - kRowChunk) return false;
  out.row_chunks = ceil_div(vocab, kRowChunk);
  out.pick_chunks = ceil_div(vocab, kPickChunk);
  out.rows = drafts + 1 + (sampled ? drafts : 0);
  const int64_t most = (int64_t)(UINT32_MAX / kDecideThreads);
  if (batch > most / (out.rows * out.row_chunks) || batch > most / out.pick_chunks) return false;
  out.weights = (size_t)(batch * out.rows * out.row_chunks) * sizeof(RowPart);
  out.choices = out.weights + (size_t)(batch * out.pick_chunks) * sizeof(Weights);
  out.bytes = out.choices + (size_t)batch * sizeof(Choice);
  return true;
}

template <typename T>
int launch(const VerifyArgs& a, const Layout& layout, hipStream_t stream) {
  const unsigned batch = (unsigned)a.batch;
  hipLaunchKernelGGL(verify_rows_kernel<T>, dim3((unsigned)(batch * layout.rows * layout.row_chunks)),
                     dim3(kRowThreads), 0, stream, a);
  const int64_t weighing = batch * layout.pick_chunks;
  const dim3 grid((unsigned)weighing), threads(kPickThreads);
  if (weighing <= kFewestWorkgroups) {
    hipLaunchKernelGGL((verify_weigh_kernel<T, kDraws>), grid, threads, 0, stream, a);
    return check_hip(hipGetLastError(), "verify draft launch");
  }
  if (weighing <= kFewWorkgroups) {
    hipLaunchKernelGGL((verify_weigh_kernel<T, kDecides>), grid, threads, 0, stream, a);
  } else {
    hipLaunchKernelGGL(verify_decide_kernel<T>, dim3(batch), dim3(kDecideThreads), 0, stream, a);
    hipLaunchKernelGGL((verify_weigh_kernel<T, kDecided>), grid, threads, 0, stream, a);
  }
  hipLaunchKernelGGL(verify_pick_kernel<T>, dim3(batch), threads, 0, stream, a);
  return check_hip(hipGetLastError(), "verify draft launch");
}

}  // namespace
}  // namespace sah

using namespace sah;

extern "C" size_t sah_verify_draft_workspace_bytes(int64_t batch, int64_t drafts, int64_t vocab, int sampled) {
  Layout layout;
  return batch > 0 && lay_out(batch, drafts, vocab, sampled != 0, layout) ? layout.bytes : 0;
}

extern "C" int sah_verify_draft(const void* target, const void* draft, const int64_t* tokens, const float* uniforms,
                                const int32_t* counts, const float* temperatures, int64_t* answer, int32_t* accepted,
                                int64_t batch, int64_t drafts, int64_t vocab, int64_t target_stride_b,
                                int64_t target_stride_s, int64_t draft_stride_b, int64_t draft_stride_s, int dtype,
                                void* workspace, size_t workspace_bytes, sah_stream_t stream) {
  const char* what = "sah_verify_draft";
  if (dtype != SAH_DTYPE_BF16 && dtype != SAH_DTYPE_F16 && dtype != SAH_DTYPE_F32)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", what, dtype);
  if (batch < 0 || drafts < 0 || vocab <= 0)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: bad batch, draft or vocabulary size", what);
  Layout layout;
  if (!lay_out(batch, drafts, vocab, draft != nullptr && drafts != 0, layout))
    return fail(SAH_ERR_UNSUPPORTED, "%s: too many rows for one launch, or more than %d drafts", what, kMaxDrafts);
  if (batch == 0) return SAH_OK;
  if (target == nullptr || uniforms == nullptr || answer == nullptr || accepted == nullptr ||
      (drafts != 0 && tokens == nullptr))
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", what);
  const uintptr_t element = dtype == SAH_DTYPE_F32 ? 3u : 1u;
  if (((reinterpret_cast<uintptr_t>(target) | reinterpret_cast<uintptr_t>(draft)) & element) != 0 ||
      ((reinterpret_cast<uintptr_t>(tokens) | reinterpret_cast<uintptr_t>(answer)) & 7u) != 0 ||
      ((reinterpret_cast<uintptr_t>(uniforms) | reinterpret_cast<uintptr_t>(counts) |
        reinterpret_cast<uintptr_t>(temperatures) | reinterpret_cast<uintptr_t>(accepted)) & 3u) != 0)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: a tensor is not aligned to its elements", what);
  if (workspace == nullptr || workspace_bytes < layout.bytes)
    return fail(SAH_ERR_WORKSPACE, "%s: workspace of %zu bytes, needs %zu", what, workspace == nullptr ? 0 : workspace_bytes,
                layout.bytes);
  if (!aligned16(workspace)) return fail(SAH_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", what);
  VerifyArgs a{};
  a.target = target;
  a.draft = drafts != 0 ? draft : nullptr;
  a.tokens = tokens;
  a.uniforms = uniforms;
  a.counts = counts;
  a.temperatures = temperatures;
  a.answer = answer;
  a.accepted = accepted;
  a.t_sb = target_stride_b;
  a.t_ss = target_stride_s;
  a.d_sb = draft_stride_b;
  a.d_ss = draft_stride_s;
  char* space = static_cast<char*>(workspace);
  a.parts = reinterpret_cast<RowPart*>(space);
  a.weights = reinterpret_cast<Weights*>(space + layout.weights);
  a.choices = reinterpret_cast<Choice*>(space + layout.choices);
  a.batch = (int)batch;
  a.drafts = (int)drafts;
  a.vocab = (int)vocab;
  a.row_chunks = (int)layout.row_chunks;
  a.pick_chunks = (int)layout.pick_chunks;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == SAH_DTYPE_BF16) return launch<bf16>(a, layout, s);
  if (dtype == SAH_DTYPE_F16) return launch<f16>(a, layout, s);
  return launch<float>(a, layout, s);
}
