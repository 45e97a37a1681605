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
// requests.  Exponentials, sums and weights are fp64 (v_fma_f64 issues at fp32's rate
// here): the choice is that of exact arithmetic but for borders closer than 1e-15 or so
// of the whole.
//
// Bound by the logits, read once (rows that count alone), in three parts:
//   1. a workgroup's chunk of a row: largest logit, its place, sum of exponentials;
//   2. each chunk of the chosen row: every workgroup finds j by itself from the parts,
//      then the sum of its chunk's weights;
//   3. the workgroup of a request that comes last finds the chunk, then the token.

#include <type_traits>

#include "sah_common.hpp"

namespace sah {
namespace {

constexpr int kRowThreads = 256;
constexpr int kVec = 8;         // logits of one access
constexpr int kAccesses = 4;    // of a thread
constexpr int kChunk = kRowThreads * kVec * kAccesses;
constexpr int kPickThreads = kChunk / kVec;
constexpr int kMaxDrafts = 1024;
constexpr double kLog2e = 1.4426950408889634074;

struct RowPart {
  double sum;   // of exp2((l - top) c)
  float top;    // the largest logit; NaN where one is NaN
  int32_t at;   // its lowest place
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
  RowPart* parts;        // [batch][drafts + 1 (+ drafts)][chunks]
  double* weights;       // [batch][chunks]
  uint32_t* tickets;     // [batch]
  int batch, drafts, vocab, chunks;
};

// 2^x for x <= 0, 0 from below the smallest number on: x = n + f with |f| <= 1/2, and
// 2^f = e^(f ln 2) as its series, whose first term left out is (ln 2 / 2)^13 / 13!,
// below 2^-52.
__device__ __forceinline__ double exp2_upto0(double x) {
  x = x < -1100.0 ? -1100.0 : x;
  const double n = __builtin_rint(x);
  const double f = (x - n) * 0.69314718055994530942;
  double y = 1.0 / 479001600.0;
  y = fma(y, f, 1.0 / 39916800.0);
  y = fma(y, f, 1.0 / 3628800.0);
  y = fma(y, f, 1.0 / 362880.0);
  y = fma(y, f, 1.0 / 40320.0);
  y = fma(y, f, 1.0 / 5040.0);
  y = fma(y, f, 1.0 / 720.0);
  y = fma(y, f, 1.0 / 120.0);
  y = fma(y, f, 1.0 / 24.0);
  y = fma(y, f, 1.0 / 6.0);
  y = fma(y, f, 0.5);
  y = fma(y, f, 1.0);
  y = fma(y, f, 1.0);
  return ldexp(y, (int)n);
}

// log2(e) / temperature, and whether the request answers greedily instead (a temperature
// that is not above 0).  An infinite one keeps masked logits at weight 0.
__device__ __forceinline__ bool is_greedy(const VerifyArgs& a, int64_t b, double& c) {
  const float t = a.temperatures != nullptr ? a.temperatures[b] : 1.0f;
  if (!(t > 0.0f)) {
    c = kLog2e;
    return true;
  }
  c = kLog2e / (double)t;
  if (c < 1e-30) c = 1e-30;
  return false;
}

// Drafts of request b, or -1 where it takes no part.
__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int64_t b) {
  if (a.counts == nullptr) return a.drafts;
  const int count = a.counts[b];
  return count < 0 ? -1 : count < a.drafts ? count : a.drafts;
}

// Logits [at, at + 8) of a row as fp32; -inf from the row's end on.  Rows start at any
// element.
template <typename T>
__device__ __forceinline__ void load_logits(const T* row, int64_t at, int64_t vocab, float* out) {
  if (at + kVec <= vocab) {
    T raw[kVec];
    __builtin_memcpy(raw, row + at, sizeof(raw));
#pragma unroll
    for (int e = 0; e < kVec; ++e) out[e] = to_f32(raw[e]);
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) out[e] = at + e < vocab ? to_f32(row[at + e]) : -INFINITY;
  }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void verify_rows_kernel(const VerifyArgs a) {
  __shared__ float tops[kRowThreads / 64];
  __shared__ int32_t bads[kRowThreads / 64];
  __shared__ double totals[kRowThreads / 64];
  __shared__ int32_t places[kRowThreads / 64];
  const int rows = a.drafts + 1 + (a.draft != nullptr ? a.drafts : 0);
  const uint32_t chunk = blockIdx.x % (uint32_t)a.chunks;
  const uint32_t request_row = blockIdx.x / (uint32_t)a.chunks;
  const int64_t b = request_row / (uint32_t)rows;
  const int r = (int)(request_row % (uint32_t)rows);
  const int tid = threadIdx.x, wave = tid >> 6;
  if (r == 0 && chunk == 0 && tid == 0) a.tickets[b] = 0;
  const int count = drafts_of(a, b);
  const bool is_draft = r > a.drafts;
  if (is_draft ? r - a.drafts - 1 >= count : r > count) return;
  double c;
  const bool greedy = is_greedy(a, b, c);
  if (greedy && is_draft) return;  // a greedy request's draft stands by the target alone
  const T* row = is_draft ? static_cast<const T*>(a.draft) + b * a.d_sb + (r - a.drafts - 1) * a.d_ss
                          : static_cast<const T*>(a.target) + b * a.t_sb + r * a.t_ss;
  const int64_t first = (int64_t)chunk * kChunk + tid * kVec;
  float l[kAccesses][kVec];
#pragma unroll
  for (int i = 0; i < kAccesses; ++i) load_logits<T>(row, first + (int64_t)i * kRowThreads * kVec, a.vocab, l[i]);
  float top = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kAccesses; ++i)
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      top = fmaxf(top, l[i][e]);
      bad = bad || l[i][e] != l[i][e];
    }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const bool any_bad = __ballot(bad) != 0;
  if ((tid & 63) == 0) {
    tops[wave] = top;
    bads[wave] = any_bad ? 1 : 0;
  }
  __syncthreads();
  int32_t nan = 0;
#pragma unroll
  for (int w = 0; w < kRowThreads / 64; ++w) {
    top = fmaxf(top, tops[w]);
    nan |= bads[w];
  }
  double sum = 0.0;
  if (top > -INFINITY && top < INFINITY) {
    const double base = (double)top;
#pragma unroll
    for (int i = 0; i < kAccesses; ++i)
#pragma unroll
      for (int e = 0; e < kVec; ++e) sum += exp2_upto0(((double)l[i][e] - base) * c);
  }
  int32_t at = INT32_MAX;
  if (greedy) {
#pragma unroll
    for (int i = kAccesses - 1; i >= 0; --i)
#pragma unroll
      for (int e = kVec - 1; e >= 0; --e)
        if (l[i][e] == top) at = (int32_t)(first + (int64_t)i * kRowThreads * kVec + e);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int32_t other = __shfl_xor(at, d);
      at = other < at ? other : at;
    }
  }
  sum = wave_sum(sum);
  if ((tid & 63) == 0) {
    totals[wave] = sum;
    places[wave] = at;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kRowThreads / 64; ++w) {
      sum += totals[w];
      at = places[w] < at ? places[w] : at;
    }
    RowPart* part = a.parts + (int64_t)request_row * a.chunks + chunk;
    part->sum = sum;
    part->top = nan != 0 ? NAN : top;
    part->at = at;
  }
}

// A row's statistics from its chunks', by one wave: the largest logit (not finite: the
// row has no distribution), its place and the sum.
struct RowSum {
  double sum;
  float top;
  int32_t at;
};
__device__ __forceinline__ RowSum merge_row(const RowPart* parts, int chunks, double c) {
  const int lane = threadIdx.x & 63;
  float top = -INFINITY;
  bool bad = false;
  for (int i = lane; i < chunks; i += 64) {
    const float t = parts[i].top;
    bad = bad || t != t;
    top = fmaxf(top, t);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  if (__ballot(bad) != 0) top = NAN;
  double sum = 0.0;
  int32_t at = INT32_MAX;
  if (top > -INFINITY && top < INFINITY)
    for (int i = lane; i < chunks; i += 64) {
      const RowPart p = parts[i];
      if (p.top > -INFINITY) sum += p.sum * exp2_upto0(((double)p.top - (double)top) * c);
      if (p.top == top && p.at < at) at = p.at;
    }
  sum = wave_sum(sum);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t other = __shfl_xor(at, d);
    at = other < at ? other : at;
  }
  return {sum, top, at};
}

struct Chosen {
  int row;         // the first draft that does not stand, or the number of drafts
  int resample;    // 1: from max(p - q, 0)
  float p_top, q_top;
  double p_sum, q_sum;
  int32_t at;      // place of the largest logit of target's row
  int32_t none;    // 1: no distribution to draw from
};

template <typename T>
__global__ __launch_bounds__(kPickThreads) void verify_pick_kernel(const VerifyArgs a) {
  constexpr int WAVES = kPickThreads / 64;
  __shared__ Chosen found[WAVES];
  __shared__ double totals[WAVES];
  __shared__ int32_t is_last, chosen_chunk;
  __shared__ double border[2];
  const uint32_t chunk = blockIdx.x % (uint32_t)a.chunks;
  const int64_t b = blockIdx.x / (uint32_t)a.chunks;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int count = drafts_of(a, b);
  int64_t* answer = a.answer + b * (a.drafts + 1);
  if (count < 0) {
    if (chunk == 0) {
      for (int i = tid; i <= a.drafts; i += kPickThreads) answer[i] = -1;
      if (tid == 0) a.accepted[b] = -1;
    }
    return;
  }
  double c;
  const bool greedy = is_greedy(a, b, c);
  const bool sampled = a.draft != nullptr && !greedy;
  const int rows = a.drafts + 1 + (a.draft != nullptr ? a.drafts : 0);
  const RowPart* parts = a.parts + b * rows * a.chunks;
  const T* target = static_cast<const T*>(a.target) + b * a.t_sb;
  const T* draft = static_cast<const T*>(a.draft) + b * a.d_sb;

  // The waves take the rows in turn until one finds the first that does not stand; a
  // wave's own first is the lowest of its rows, and the lowest of them all is j.
  Chosen mine{count + 1, 0, 0.0f, 0.0f, 1.0, 1.0, 0, 0};
  for (int i = wave; i <= count; i += WAVES) {
    const RowSum p = merge_row(parts + (int64_t)i * a.chunks, a.chunks, c);
    const bool p_there = p.top > -INFINITY && p.top < INFINITY;
    RowSum q{1.0, 0.0f, 0};
    bool q_there = true;
    bool stands = false;
    if (i < count) {
      const int64_t token = a.tokens[b * a.drafts + i];
      const bool known = token >= 0 && token < a.vocab;
      if (sampled) {
        q = merge_row(parts + (int64_t)(a.drafts + 1 + i) * a.chunks, a.chunks, c);
        q_there = q.top > -INFINITY && q.top < INFINITY;
      }
      if (p_there && q_there && known) {
        if (greedy) {
          stands = p.at == token;
        } else {
          const double chance = exp2_upto0(((double)to_f32(target[i * a.t_ss + token]) - (double)p.top) * c) / p.sum;
          double other = 1.0;
          if (sampled) other = exp2_upto0(((double)to_f32(draft[i * a.d_ss + token]) - (double)q.top) * c) / q.sum;
          stands = (double)a.uniforms[b * (a.drafts + 1) + i] * other < chance;
        }
      }
    }
    if (!stands) {
      mine = {i, i < count ? 1 : 0, p.top, q.top, p.sum, q.sum, p.at, p_there && q_there ? 0 : 1};
      break;
    }
  }
  if (lane == 0) found[wave] = mine;
  __syncthreads();
  Chosen at = found[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w)
    if (found[w].row < at.row) at = found[w];
  const int j = at.row;

  auto write = [&](int64_t token) {  // by the workgroup's every thread
    for (int i = tid; i <= a.drafts; i += kPickThreads)
      answer[i] = i < j ? a.tokens[b * a.drafts + i] : i == j ? token : -1;
    if (tid == 0) a.accepted[b] = j;
  };
  if (greedy || at.none != 0) {
    if (chunk == 0) write(at.none != 0 ? -1 : at.at);
    return;
  }

  // The weights of 8 tokens; zeros behind the row's end.
  const bool resample = at.resample != 0;
  const int64_t drafted = resample ? a.tokens[b * a.drafts + j] : -1;
  const T* p_row = target + j * a.t_ss;
  const T* q_row = draft + j * a.d_ss;
  auto weigh = [&](int64_t first, double* w) {
    float l[kVec];
    load_logits<T>(p_row, first, a.vocab, l);
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      w[e] = exp2_upto0(((double)l[e] - (double)at.p_top) * c) / at.p_sum;
    if (!resample) return;
    if (sampled) {
      load_logits<T>(q_row, first, a.vocab, l);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const double less = w[e] - exp2_upto0(((double)l[e] - (double)at.q_top) * c) / at.q_sum;
        w[e] = less > 0.0 ? less : 0.0;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (first + e == drafted) w[e] = 0.0;
    }
  };

  double w[kVec];
  weigh((int64_t)chunk * kChunk + tid * kVec, w);
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < kVec; ++e) sum += w[e];
  sum = wave_sum(sum);
  if (lane == 0) totals[wave] = sum;
  __syncthreads();
  double* weights = a.weights + b * a.chunks;
  if (tid == 0) {
    double total = 0.0;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) total += totals[k];
    __hip_atomic_store(weights + chunk, total, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const uint32_t ticket = __hip_atomic_fetch_add(a.tickets + b, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    is_last = ticket + 1 == (uint32_t)a.chunks ? 1 : 0;
  }
  __syncthreads();
  if (is_last == 0) return;

  // The last workgroup: the chunk in which the sum passes u times the whole.
  if (wave == 0) {
    double whole = 0.0;
    for (int i = 0; i < a.chunks; i += 64) {
      const double v = i + lane < a.chunks
                           ? __hip_atomic_load(weights + i + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                           : 0.0;
      whole += wave_sum(v);
    }
    const double bound = (double)a.uniforms[b * (a.drafts + 1) + a.drafts] * whole;
    double before = 0.0, last_before = 0.0;
    int chosen = -1, last = -1;
    for (int i = 0; i < a.chunks && chosen < 0; i += 64) {
      const double v = i + lane < a.chunks
                           ? __hip_atomic_load(weights + i + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                           : 0.0;
      double up_to = v;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const double other = __shfl_up(up_to, d);
        if (lane >= d) up_to += other;
      }
      const uint64_t some = __ballot(v > 0.0);
      const uint64_t above = __ballot(v > 0.0 && before + up_to > bound);
      const double mine_before = before + (up_to - v);
      if (some != 0) {
        const int k = 63 - __clzll((long long)some);
        last = i + k;
        last_before = __shfl(mine_before, k);
      }
      if (above != 0) {
        const int k = __ffsll((unsigned long long)above) - 1;
        chosen = i + k;
        last_before = __shfl(mine_before, k);
      }
      before += __shfl(up_to, 63);
    }
    if (lane == 0) {
      chosen_chunk = chosen >= 0 ? chosen : last;  // (a border of rounding: the last weight)
      border[0] = last_before;
      border[1] = bound;
    }
  }
  __syncthreads();
  const int where = chosen_chunk;
  const double start = border[0], bound = border[1];
  if (where < 0) {  // the drafted token had all of the target's weight, and did not stand
    write(-1);
    return;
  }
  const int64_t first = (int64_t)where * kChunk + tid * kVec;
  weigh(first, w);
  double own_sum = 0.0;
#pragma unroll
  for (int e = 0; e < kVec; ++e) own_sum += w[e];
  double up_to = own_sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double other = __shfl_up(up_to, d);
    if (lane >= d) up_to += other;
  }
  __syncthreads();
  if (lane == 63) totals[wave] = up_to;
  __syncthreads();
  double run = start + (up_to - own_sum);
  for (int k = 0; k < wave; ++k) run += totals[k];
  int32_t pick = INT32_MAX, last = -1;
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    run += w[e];
    if (w[e] > 0.0) {
      last = (int32_t)(first + e);
      if (run > bound && pick == INT32_MAX) pick = last;
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t p = __shfl_xor(pick, d), q = __shfl_xor(last, d);
    pick = p < pick ? p : pick;
    last = q > last ? q : last;
  }
  __shared__ int32_t picks[WAVES], lasts[WAVES];
  if (lane == 0) {
    picks[wave] = pick;
    lasts[wave] = last;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < WAVES; ++k) {
    pick = picks[k] < pick ? picks[k] : pick;
    last = lasts[k] > last ? lasts[k] : last;
  }
  write(pick != INT32_MAX ? pick : last);
}

struct Layout {
  int64_t chunks, rows;
  size_t parts, weights, tickets, bytes;
};
// Where the parts stand in the workspace; false for sizes that no launch takes.
bool lay_out(int64_t batch, int64_t drafts, int64_t vocab, bool sampled, Layout& out) {
  if (batch < 0 || drafts < 0 || drafts > kMaxDrafts || vocab <= 0 || vocab > INT32_MAX - kChunk) return false;
  out.chunks = ceil_div(vocab, kChunk);
  out.rows = drafts + 1 + (sampled ? drafts : 0);
  const int64_t most = (int64_t)(UINT32_MAX / kPickThreads);
  if (batch > most / (out.rows * out.chunks)) return false;
  out.parts = 0;
  out.weights = (size_t)(batch * out.rows * out.chunks) * sizeof(RowPart);
  out.tickets = out.weights + (size_t)(batch * out.chunks) * sizeof(double);
  out.bytes = out.tickets + (size_t)batch * sizeof(uint32_t);
  return true;
}

template <typename T>
int launch(const VerifyArgs& a, const Layout& layout, hipStream_t stream) {
  hipLaunchKernelGGL(verify_rows_kernel<T>, dim3((unsigned)(a.batch * layout.rows * layout.chunks)), dim3(kRowThreads),
                     0, stream, a);
  const int status = check_hip(hipGetLastError(), "verify draft launch");
  if (status != SAH_OK) return status;
  hipLaunchKernelGGL(verify_pick_kernel<T>, dim3((unsigned)(a.batch * layout.chunks)), dim3(kPickThreads), 0, stream, a);
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
  a.parts = reinterpret_cast<RowPart*>(space + layout.parts);
  a.weights = reinterpret_cast<double*>(space + layout.weights);
  a.tickets = reinterpret_cast<uint32_t*>(space + layout.tickets);
  a.batch = (int)batch;
  a.drafts = (int)drafts;
  a.vocab = (int)vocab;
  a.chunks = (int)layout.chunks;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == SAH_DTYPE_BF16) return launch<bf16>(a, layout, s);
  if (dtype == SAH_DTYPE_F16) return launch<f16>(a, layout, s);
  return launch<float>(a, layout, s);
}
