// Book-keeping of the 8-bit block cache's places and the data that moves with it, for
// gfx950 (CDNA4).
//
// block_table [batch, max_blocks] names the place of each block of a sequence, holders
// [blocks] counts the entries that name a place; a place without holders is free.  A
// complete block is never written again, so sequences that go on from the same tokens
// share its place, and only the incomplete block, which stands in the tails, is copied.
//
// The book's kernels read and write some KB to some hundred KB: they are bound by the
// latency of one access after the other (some 1 us each from memory, 0.5 from L2) and a
// launch of 3 us on the host, which is why each call takes one launch wherever a workgroup
// or independent parts can do its work.  The kernels that move the cache's data are
// bound by its bytes.
//
// The whole numbers here are sums in any order (atomic counts) or follow from places in
// order (ranks by prefix sums), so a call's result does not depend on its schedule.

#include <type_traits>

#include "decode_common.hpp"

namespace sah {
namespace {

constexpr int kThreads = 256;
constexpr int kScanThreads = 1024;
constexpr int kPerThread = 16;  // places of one thread in a pass of a scan
constexpr int kScanTile = kScanThreads * kPerThread;

struct Pool {
  int32_t* table;    // [batch, max_blocks]
  int32_t* holders;  // [blocks]
  int64_t blocks;
  int batch, max_blocks;
};

__device__ __forceinline__ bool is_place(int64_t id, int64_t blocks) { return id >= 0 && id < blocks; }

// Sum of `value` over the threads before this one, and over all of them in `total`.
// `sums` may be written again once every thread is past the next barrier.
__device__ __forceinline__ int scan_threads(int value, int* sums, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int up_to = value;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int other = __shfl_up(up_to, d);
    if (lane >= d) up_to += other;
  }
  if (lane == 63) sums[wave] = up_to;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kScanThreads / 64; ++w) {
    const int s = sums[w];
    if (w < wave) before += s;
    total += s;
  }
  return before + up_to - value;
}

// Bit i: place first + i is there and has holders.
__device__ __forceinline__ uint32_t held_bits(const int32_t* holders, int64_t first, int64_t blocks) {
  int32_t count[kPerThread];
  if (first + kPerThread <= blocks) {
    __builtin_memcpy(count, holders + first, sizeof(count));
  } else {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) count[i] = first + i < blocks ? holders[first + i] : 0;
  }
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) bits |= (count[i] > 0 ? 1u : 0u) << i;
  return bits;
}
// The lowest n of a thread's kPerThread bits.
__device__ __forceinline__ uint32_t low_bits(int64_t n) {
  return n <= 0 ? 0u : n >= kPerThread ? (1u << kPerThread) - 1u : (1u << n) - 1u;
}

struct ReserveArgs {
  Pool pool;
  const int32_t* starts;
  const int32_t* counts;
  int32_t* missing;
  int32_t* offsets;  // workspace [batch]: places that the sequences before this one lack
  int32_t* free;     // workspace: the lowest free places
  int64_t tokens;
  int lanes;         // of one sequence: a power of two
};

// Every entry of [start / 64, (start + count) / 64) without a place takes one: the
// lowest free places, sequence by sequence and block by block.  One workgroup, as what
// a sequence lacks decides what the next ones get: in order, what each sequence lacks,
// its sums over the sequences before, that many free places, the entries.  The search
// ends with the last free place that is wanted; a thread reads 16 places in four accesses.
// 64 sequences of 8 tokens in a pool of 4032 places, or 32 of 777 in 6016: 6 us, four
// steps of accesses and barriers (a copy's time of what it reads would be 0.01); a pool
// without free places, which is searched whole, of 65536 11 us, of 262144 31.
__global__ __launch_bounds__(kScanThreads) void pool_reserve_kernel(const ReserveArgs a) {
  __shared__ int sums[2][kScanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int slot = tid & (a.lanes - 1);
  const int groups = kScanThreads / a.lanes;
  const uint64_t group_mask = (a.lanes == 64 ? ~0ull : (1ull << a.lanes) - 1) << (lane & ~(a.lanes - 1));
  const int64_t width = a.pool.max_blocks, blocks = a.pool.blocks;

  // The blocks [first, last) that sequence b's new tokens complete.
  auto span_of = [&](int b, int64_t& first, int64_t& last) {
    first = last = 0;
    if (b >= a.pool.batch) return;
    const int64_t start = a.starts[b];
    int64_t count = a.counts != nullptr ? (int64_t)a.counts[b] : a.tokens;
    if (count > a.tokens) count = a.tokens;
    if (start < 0 || count <= 0) return;
    first = start / kBlockTokens;
    last = (start + count) / kBlockTokens;
  };

  // A wave's lanes make the same rounds, so their votes are whole.
  for (int at = 0; at < a.pool.batch; at += groups) {
    const int b = at + tid / a.lanes;
    int64_t first, last;
    span_of(b, first, last);
    const int32_t* row = a.pool.table + (int64_t)b * width;
    const int64_t end = last < width ? last : width;
    int need = 0;
    for (int64_t j = first; __ballot(j < end) != 0; j += a.lanes) {
      const bool lacks = j + slot < end && !is_place(row[j + slot], blocks);
      need += __popcll(__ballot(lacks) & group_mask);
    }
    if (b < a.pool.batch && slot == 0) a.missing[b] = need;
  }
  __syncthreads();

  int wanted = 0;
  for (int at = 0; at < a.pool.batch; at += kScanThreads) {
    const int b = at + tid;
    int total;
    const int before = scan_threads(b < a.pool.batch ? a.missing[b] : 0, sums[(at / kScanThreads) & 1], total);
    if (b < a.pool.batch) a.offsets[b] = wanted + before;
    wanted += total;
  }
  __syncthreads();

  int found = 0;
  for (int64_t at = 0; at < blocks && found < wanted; at += kScanTile) {
    const int64_t first = at + (int64_t)tid * kPerThread;
    uint32_t open = ~held_bits(a.pool.holders, first, blocks) & low_bits(blocks - first);
    int total;
    int rank = found + scan_threads(__popc(open), sums[(at / kScanTile) & 1], total);
    while (open != 0 && rank < wanted) {
      a.free[rank++] = (int32_t)(first + __ffs((int)open) - 1);
      open &= open - 1;
    }
    found += total;
  }
  if (found > wanted) found = wanted;
  __syncthreads();

  for (int at = 0; at < a.pool.batch; at += groups) {
    const int b = at + tid / a.lanes;
    int64_t first, last;
    span_of(b, first, last);
    int32_t* row = a.pool.table + (int64_t)b * width;
    const int64_t end = last < width ? last : width;
    const int offset = b < a.pool.batch ? a.offsets[b] : 0;
    int rank = offset;
    for (int64_t j = first; __ballot(j < end) != 0; j += a.lanes) {
      const bool lacks = j + slot < end && !is_place(row[j + slot], blocks);
      const uint64_t votes = __ballot(lacks) & group_mask;
      const int mine = rank + __popcll(votes & ((1ull << lane) - 1));
      if (lacks && mine < found) {
        const int32_t place = a.free[mine];
        row[j + slot] = place;
        a.pool.holders[place] = 1;
      }
      rank += __popcll(votes);
    }
    if (b < a.pool.batch && slot == 0) {
      const int got = found <= offset ? 0 : found >= rank ? rank - offset : found - offset;
      // blocks behind the table's width have no entry to take a place
      const int64_t behind = last > width ? last - (first > width ? first : width) : 0;
      a.missing[b] = (int32_t)(rank - offset - got + behind);
    }
  }
}

// A thread an entry: 64 sequences of 63 blocks that end 8 tokens earlier, 2.5 us, 32 of 200
// that end 4000 earlier 2.8: a length, an entry, a count one after the other.
__global__ __launch_bounds__(kThreads) void pool_release_kernel(const Pool pool, const int32_t* lengths, uint32_t parts) {
  const int b = blockIdx.x / parts;
  const int64_t column = (int64_t)(blockIdx.x % parts) * kThreads + threadIdx.x;
  const int64_t length = lengths[b];
  if (length < 0 || column >= pool.max_blocks || column < length / kBlockTokens) return;
  int32_t* entry = pool.table + (int64_t)b * pool.max_blocks + column;
  const int32_t place = *entry;
  if (is_place(place, pool.blocks)) atomicSub(pool.holders + place, 1);
  if (place != -1) *entry = -1;
}

constexpr int kForkColumns = 16;  // of a workgroup: 64 bytes of each row
constexpr int kMaxForked = 1024;  // sequences, whose entries of these columns fill 64 KiB

// Sequence b goes on as a copy of sequence sources[b].  A column of the table is a
// problem of its own: a workgroup reads its columns of every sequence before it
// writes any of them, so sequences may change places.  64 sequences of 1563 blocks, half
// of them copies: 4 us, the table read once and the counts' atomics.
__global__ __launch_bounds__(kThreads) void pool_fork_kernel(const Pool pool, const int32_t* sources, const int32_t* lengths) {
  extern __shared__ int32_t before[];  // [batch][kForkColumns]
  const int64_t width = pool.max_blocks;
  const int column = threadIdx.x % kForkColumns;
  const int64_t at = (int64_t)blockIdx.x * kForkColumns + column;
  constexpr int ROWS = kThreads / kForkColumns;
  for (int b = threadIdx.x / kForkColumns; b < pool.batch; b += ROWS)
    before[b * kForkColumns + column] = at < width ? pool.table[b * width + at] : -1;
  __syncthreads();
  if (at >= width) return;
  for (int b = threadIdx.x / kForkColumns; b < pool.batch; b += ROWS) {
    const int source = sources[b];
    if (source < 0 || source >= pool.batch || source == b) continue;
    const int64_t length = lengths[source];
    const int32_t old = before[b * kForkColumns + column];
    // places behind the complete blocks are kept for the source's own next ones
    const int32_t fresh = length >= 0 && at < length / kBlockTokens ? before[source * kForkColumns + column] : -1;
    if (fresh == old) continue;
    if (is_place(old, pool.blocks)) atomicSub(pool.holders + old, 1);
    if (is_place(fresh, pool.blocks)) atomicAdd(pool.holders + fresh, 1);
    pool.table[b * width + at] = fresh;
  }
}

// Places and entries up to which one launch compacts a pool: 12.7 -> 8.4 us on the host,
// which is what a small pool's compaction takes (4128 of either: 9.3 us on the GPU in one
// launch, 8.6 + 4.6 in two; 16384 21 us).
constexpr int64_t kSmallPool = 16384;

struct CompactArgs {
  Pool pool;
  int32_t* origins;  // [blocks]
  int32_t* used;     // [1]
  int32_t* holes;    // workspace [blocks / 2 + 1]: free places below used, in order
  int32_t* movers;   // workspace [blocks / 2 + 1]: held places from used on, in order
  int32_t* ranks;    // workspace [blocks]: a mover's number, -1 of others from used on
  int32_t* moves;    // workspace [1]
};

constexpr int kApplyEntries = 4;  // of a thread in flight

// The entries take their places' new names, and each hole its mover's holders, by threads
// first, first + step, ...
__device__ __forceinline__ void compact_apply(const CompactArgs& a, int used, int moves, int64_t first, int64_t step) {
  for (int64_t i = first; i < moves; i += step) {
    const int32_t hole = a.holes[i], mover = a.movers[i];
    a.origins[hole] = mover;
    a.pool.holders[hole] = a.pool.holders[mover];
    a.pool.holders[mover] = 0;
  }
  // (four entries' accesses in flight together: 32 sequences of 129 blocks, by one
  // workgroup, the whole call a ninth less)
  const int64_t entries = (int64_t)a.pool.batch * a.pool.max_blocks;
  for (int64_t i = first; i < entries; i += kApplyEntries * step) {
    int32_t place[kApplyEntries], rank[kApplyEntries], hole[kApplyEntries];
#pragma unroll
    for (int e = 0; e < kApplyEntries; ++e) place[e] = a.pool.table[i + e * step < entries ? i + e * step : i];
#pragma unroll
    for (int e = 0; e < kApplyEntries; ++e) {
      const bool renamed = place[e] >= used && place[e] < a.pool.blocks;
      rank[e] = renamed ? a.ranks[place[e]] : -1;
    }
#pragma unroll
    for (int e = 0; e < kApplyEntries; ++e) hole[e] = rank[e] >= 0 ? a.holes[rank[e]] : -1;
#pragma unroll
    for (int e = 0; e < kApplyEntries; ++e)
      if (hole[e] >= 0 && i + e * step < entries) a.pool.table[i + e * step] = hole[e];
  }
}

// `used` places have holders.  The free ones below `used` are as many as the held
// ones from there on, and take their contents in order.  One workgroup counts, then
// lists both; of a small pool it does the rest too (APPLIES).  It reads the counts twice,
// 16384 places a pass: 65536 places 54 us with the second launch, 262144 202.
template <bool APPLIES>
__global__ __launch_bounds__(kScanThreads) void pool_compact_list_kernel(const CompactArgs a) {
  __shared__ int sums[2][kScanThreads / 64];
  const int64_t blocks = a.pool.blocks;
  const int tid = threadIdx.x;
  int mine = 0;
  for (int64_t at = 0; at < blocks; at += kScanTile)
    mine += __popc(held_bits(a.pool.holders, at + (int64_t)tid * kPerThread, blocks));
  int used;
  scan_threads(mine, sums[1], used);
  int holes = 0, movers = 0;
  for (int64_t at = 0; at < blocks; at += kScanTile) {
    const int64_t first = at + (int64_t)tid * kPerThread;
    const uint32_t there = low_bits(blocks - first);
    const uint32_t held = held_bits(a.pool.holders, first, blocks);
    const uint32_t low = low_bits(used - first);
    uint32_t open = there & ~held & low, move = held & ~low;
    // Both counts in one number: a pass has at most kScanTile of either, below 2^15.
    int total;
    const int before = scan_threads(__popc(open) | (__popc(move) << 16), sums[(at / kScanTile) & 1], total);
    int hole = holes + (before & 0xffff), mover = movers + (before >> 16);
    const uint32_t stays = there & ~open;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)
      if ((stays >> i) & 1u) a.origins[first + i] = -1;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)  // places that nothing should name
      if (((there & ~low & ~held) >> i) & 1u) a.ranks[first + i] = -1;
    while (open != 0) {
      a.holes[hole++] = (int32_t)(first + __ffs((int)open) - 1);
      open &= open - 1;
    }
    while (move != 0) {
      const int64_t place = first + __ffs((int)move) - 1;
      a.ranks[place] = mover;
      a.movers[mover++] = (int32_t)place;
      move &= move - 1;
    }
    holes += total & 0xffff;
    movers += total >> 16;
  }
  if (tid == 0) {
    *a.used = used;
    *a.moves = movers;
  }
  if constexpr (APPLIES) {
    __syncthreads();  // (after the last reads of holders, too)
    compact_apply(a, used, movers, tid, kScanThreads);
  }
}

__global__ __launch_bounds__(kThreads) void pool_compact_apply_kernel(const CompactArgs a) {
  compact_apply(a, *a.used, *a.moves, (int64_t)blockIdx.x * kThreads + threadIdx.x, (int64_t)gridDim.x * kThreads);
}

struct CopyArgs {
  uint8_t* codes[2];  // keys, values
  float* scales[2];
  const int32_t* origins;
  int64_t blocks;
  int64_t place_bytes;  // of a place's key codes, or value codes
  int64_t units;
  int parts;            // units of these
  int heads;
};

constexpr int kCopyLoads = 4;                          // 16-byte loads of a thread in flight
constexpr int kCopyPart = kThreads * 16 * kCopyLoads;  // bytes of a unit
constexpr int64_t kPastBytes = (int64_t)256 << 20;     // of a layer's codes: the last-level cache

__device__ __forceinline__ bool is_written(const CopyArgs& a, int64_t place) {
  const int64_t origin = a.origins[place];
  return is_place(origin, a.blocks) && origin != place;
}

// Place t takes what place origins[t] holds.  No place that is read is written: where
// an origin is itself written, the pair is left out.  Units of 16 KiB; a workgroup
// takes every gridDim-th, and looks 64 of them up at a time.  Bound by its bytes: 1000
// places of 16 heads of 64 (262 MB with the writes, 53 us at a large copy's rate) 57 us
// past the caches (PAST), 60.5 through them, where the cache's codes fill the last-level
// one.
template <bool PAST>
__global__ __launch_bounds__(kThreads) void cache_copy_kernel(const CopyArgs a) {
  const int lane = threadIdx.x & 63;
  const int units_of_place = 2 * a.parts;
  for (int64_t at = blockIdx.x; at < a.units; at += (int64_t)64 * gridDim.x) {
    const int64_t unit = at + (int64_t)lane * gridDim.x;
    bool takes = false;
    if (unit < a.units) {
      const int64_t target = unit / units_of_place;
      takes = is_written(a, target) && !is_written(a, a.origins[target]);
    }
    uint64_t votes = __ballot(takes);
    while (votes != 0) {
      const int64_t next = at + (int64_t)(__ffsll((unsigned long long)votes) - 1) * gridDim.x;
      votes &= votes - 1;
      const int64_t target = next / units_of_place;
      const int place_part = (int)(next - target * units_of_place);
      const int which = place_part / a.parts, part = place_part - which * a.parts;
      const int64_t origin = a.origins[target];
      const uint8_t* from = a.codes[which] + origin * a.place_bytes;
      uint8_t* to = a.codes[which] + target * a.place_bytes;
      const int64_t first = (int64_t)part * kCopyPart + threadIdx.x * 16;
      u32x4 data[kCopyLoads];
#pragma unroll
      for (int i = 0; i < kCopyLoads; ++i)
        if (first + i * kThreads * 16 < a.place_bytes) data[i] = PAST ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from + first + i * kThreads * 16))
                         : load16(from + first + i * kThreads * 16);
#pragma unroll
      for (int i = 0; i < kCopyLoads; ++i)
        if (first + i * kThreads * 16 < a.place_bytes) {
          if (PAST)
            __builtin_nontemporal_store(data[i], reinterpret_cast<u32x4*>(to + first + i * kThreads * 16));
          else
            store16(to + first + i * kThreads * 16, data[i]);
        }
      if (part == 0)
        for (int h = threadIdx.x; h < a.heads; h += kThreads)
          a.scales[which][target * a.heads + h] = a.scales[which][origin * a.heads + h];
    }
  }
}

// The tail of sequence sources[b] goes to sequence b.  A slice of the tails' bytes is a
// problem of its own: a workgroup has read its slice of every tail that it copies
// before it writes any.  The sequences that change are listed first, so that a thread's
// accesses are in flight together: 64 sequences, half of them copies, of 8 heads of 128 (17
// MB) 4 us, 9.9 with each sequence's source looked up on its way (5.2 with slices of 1 KiB).
constexpr int kForkLoads = 8;  // of a thread in flight

__global__ __launch_bounds__(kThreads) void cache_fork_kernel(char* key_tail, char* value_tail, const int32_t* sources,
                                                              int batch, int64_t tail_bytes, int slice_bytes) {
  extern __shared__ __align__(16) u32x4 held[];  // [changed][slice_bytes / 16]
  __shared__ int16_t targets[kMaxForked], origins[kMaxForked];
  __shared__ int changed;
  const int lanes = slice_bytes / 16;  // a power of two
  const uint32_t slices = (uint32_t)(tail_bytes / slice_bytes);
  char* tail = (blockIdx.x < slices ? key_tail : value_tail) + (int64_t)(blockIdx.x % slices) * slice_bytes;
  if (threadIdx.x < 64) {  // a wave lists them in order
    int count = 0;
    for (int at = 0; at < batch; at += 64) {
      const int b = at + threadIdx.x;
      const int source = b < batch ? sources[b] : -1;
      const bool changes = source >= 0 && source < batch && source != b;
      const uint64_t votes = __ballot(changes);
      if (changes) {
        const int place = count + __popcll(votes & ((1ull << threadIdx.x) - 1));
        targets[place] = (int16_t)b;
        origins[place] = (int16_t)source;
      }
      count += __popcll(votes);
    }
    if (threadIdx.x == 0) changed = count;
  }
  __syncthreads();
  const int parts = changed * lanes;
  for (int at = threadIdx.x; at < parts; at += kForkLoads * kThreads) {
    u32x4 data[kForkLoads];
#pragma unroll
    for (int i = 0; i < kForkLoads; ++i) {
      const int part = at + i * kThreads;
      if (part < parts) data[i] = load16(tail + origins[part / lanes] * tail_bytes + (part & (lanes - 1)) * 16);
    }
#pragma unroll
    for (int i = 0; i < kForkLoads; ++i)
      if (at + i * kThreads < parts) held[at + i * kThreads] = data[i];
  }
  __syncthreads();
  for (int part = threadIdx.x; part < parts; part += kThreads)
    store16(tail + targets[part / lanes] * tail_bytes + (part & (lanes - 1)) * 16, held[part]);
}

struct TakeBackArgs {
  const uint8_t* codes[2];  // keys, values
  const float* scales[2];
  void* tails[2];
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* ends;
  int64_t blocks, max_blocks;
  int heads, head_values;  // values of a head's block
};

// A sequence whose end falls into a complete block gets that block back into its
// tail: codes times their scale, exact in 16 bits wherever the type reaches.  Tails
// are laid out as the codes are, so a thread turns 16 codes in a row, and a workgroup a
// head's block of keys or values.  64 sequences of 16 heads of 64, few of which go back
// into a complete block, 3.7 us, 32 of 8 heads of 128, all of which do (12 MB), 5.3: a
// length, an entry and the codes one after the other.
template <typename T>
__global__ __launch_bounds__(kThreads) void cache_take_back_kernel(const TakeBackArgs a) {
  typedef typename Vec8<T>::type V8;
  const int64_t pair = blockIdx.x >> 1;
  const int which = blockIdx.x & 1;
  const int64_t b = pair / a.heads;
  const int h = (int)(pair - b * a.heads);
  const int64_t length = a.lengths[b], end = a.ends[b];
  if (end < 0 || end % kBlockTokens == 0 || end / kBlockTokens >= length / kBlockTokens) return;
  const int64_t block = end / kBlockTokens;
  const int64_t id = block < a.max_blocks ? (int64_t)a.table[b * a.max_blocks + block] : -1;
  const bool held = is_place(id, a.blocks);
  const float scale = held ? a.scales[which][id * a.heads + h] : NAN;
  const uint8_t* codes = held ? a.codes[which] + (id * a.heads + h) * (int64_t)a.head_values : nullptr;
  T* tail = static_cast<T*>(a.tails[which]) + pair * a.head_values;
  for (int at = threadIdx.x * 16; at < a.head_values; at += kThreads * 16) {
    const u32x4 raw = held ? load16(codes + at) : (u32x4){0u, 0u, 0u, 0u};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const V8 values = e4m3_operand<T>(raw[2 * half], raw[2 * half + 1], 1.0f);
      V8 out;
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = in_range<T>(to_f32(values[e]) * scale);
      *reinterpret_cast<V8*>(tail + at + 8 * half) = out;
    }
  }
}

int check_pool(const char* what, const Pool& p, int64_t batch, int64_t max_blocks) {
  if (batch < 0 || batch > INT32_MAX / kScanThreads || max_blocks < 0 || max_blocks > INT32_MAX / kBlockTokens ||
      p.blocks < 0 || p.blocks > INT32_MAX - kScanTile)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: bad batch or block count", what);
  if (batch * max_blocks > INT32_MAX)  // entries are counted in 32 bits
    return fail(SAH_ERR_UNSUPPORTED, "%s: the block table has 2^31 entries or more", what);
  if ((batch != 0 && max_blocks != 0 && p.table == nullptr) || (p.blocks != 0 && p.holders == nullptr))
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: null block table or holders", what);
  if (((reinterpret_cast<uintptr_t>(p.table) | reinterpret_cast<uintptr_t>(p.holders)) & 3u) != 0)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: block table and holders must be 4-byte aligned", what);
  return SAH_OK;
}

template <int N>
int check_words(const char* what, const void* const (&words)[N]) {
  for (const void* p : words) {
    if (p == nullptr) return fail(SAH_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", what);
    if ((reinterpret_cast<uintptr_t>(p) & 3u) != 0)
      return fail(SAH_ERR_INVALID_ARGUMENT, "%s: whole numbers and scales must be 4-byte aligned", what);
  }
  return SAH_OK;
}

int check_places(const char* what, int64_t kv_heads, int64_t head_dim, int64_t num_blocks) {
  if (head_dim != 64 && head_dim != 128)
    return fail(SAH_ERR_UNSUPPORTED, "%s: head_dim %lld is not 64 or 128", what, (long long)head_dim);
  if (kv_heads <= 0 || kv_heads > 65536 || num_blocks < 0 || num_blocks > INT32_MAX)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: bad head or block count", what);
  return SAH_OK;
}

int check_workspace(const char* what, const void* workspace, size_t bytes, size_t need) {
  if (workspace == nullptr || bytes < need)
    return fail(SAH_ERR_WORKSPACE, "%s: workspace of %zu bytes, needs %zu", what, workspace == nullptr ? 0 : bytes, need);
  if ((reinterpret_cast<uintptr_t>(workspace) & 3u) != 0)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: the workspace must be 4-byte aligned", what);
  return SAH_OK;
}

}  // namespace
}  // namespace sah

using namespace sah;

extern "C" size_t sah_block_pool_reserve_workspace_bytes(int64_t batch, int64_t max_blocks, int64_t num_blocks,
                                                         int64_t tokens) {
  if (batch <= 0 || max_blocks < 0 || num_blocks < 0 || tokens < 0) return 0;
  // places that the batch can ask for at once, and never more than there are
  const int64_t span = tokens / kBlockTokens + 1;
  const int64_t each = span < max_blocks ? span : max_blocks;
  const int64_t most = each == 0 ? 0 : num_blocks / each < batch ? num_blocks : batch * each;
  return (size_t)(batch + most) * sizeof(int32_t);
}

extern "C" int sah_block_pool_reserve(int32_t* block_table, int32_t* holders, const int32_t* starts,
                                      const int32_t* counts, int32_t* missing, int64_t batch, int64_t max_blocks,
                                      int64_t num_blocks, int64_t tokens, void* workspace, size_t workspace_bytes,
                                      sah_stream_t stream) {
  const char* what = "sah_block_pool_reserve";
  ReserveArgs a{};
  a.pool = {block_table, holders, num_blocks, (int)batch, (int)max_blocks};
  int status = check_pool(what, a.pool, batch, max_blocks);
  if (status != SAH_OK) return status;
  if (tokens < 0 || tokens > INT32_MAX)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: bad token count %lld", what, (long long)tokens);
  if (batch == 0) return SAH_OK;
  status = check_words(what, {starts, missing});
  if (status != SAH_OK) return status;
  if ((reinterpret_cast<uintptr_t>(counts) & 3u) != 0)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: counts must be 4-byte aligned", what);
  status = check_workspace(what, workspace, workspace_bytes,
                           sah_block_pool_reserve_workspace_bytes(batch, max_blocks, num_blocks, tokens));
  if (status != SAH_OK) return status;
  a.starts = starts;
  a.counts = counts;
  a.missing = missing;
  a.offsets = static_cast<int32_t*>(workspace);
  a.free = a.offsets + batch;
  a.tokens = tokens;
  a.lanes = 1;
  while (a.lanes < 64 && a.lanes < tokens / kBlockTokens + 1) a.lanes *= 2;
  hipLaunchKernelGGL(pool_reserve_kernel, dim3(1), dim3(kScanThreads), 0, reinterpret_cast<hipStream_t>(stream), a);
  return check_hip(hipGetLastError(), "block pool reserve launch");
}

extern "C" int sah_block_pool_release(int32_t* block_table, int32_t* holders, const int32_t* lengths, int64_t batch,
                                      int64_t max_blocks, int64_t num_blocks, sah_stream_t stream) {
  const char* what = "sah_block_pool_release";
  const Pool pool = {block_table, holders, num_blocks, (int)batch, (int)max_blocks};
  int status = check_pool(what, pool, batch, max_blocks);
  if (status != SAH_OK) return status;
  if (batch == 0 || max_blocks == 0) return SAH_OK;
  status = check_words(what, {lengths});
  if (status != SAH_OK) return status;
  const int64_t parts = ceil_div(max_blocks, kThreads);
  hipLaunchKernelGGL(pool_release_kernel, dim3((unsigned)(parts * batch)), dim3(kThreads), 0,
                     reinterpret_cast<hipStream_t>(stream), pool, lengths, (uint32_t)parts);
  return check_hip(hipGetLastError(), "block pool release launch");
}

extern "C" int sah_block_pool_fork(int32_t* block_table, int32_t* holders, const int32_t* sources,
                                   const int32_t* lengths, int64_t batch, int64_t max_blocks, int64_t num_blocks,
                                   sah_stream_t stream) {
  const char* what = "sah_block_pool_fork";
  const Pool pool = {block_table, holders, num_blocks, (int)batch, (int)max_blocks};
  int status = check_pool(what, pool, batch, max_blocks);
  if (status != SAH_OK) return status;
  if (batch > kMaxForked)
    return fail(SAH_ERR_UNSUPPORTED, "%s: batch %lld is above %d", what, (long long)batch, kMaxForked);
  if (batch == 0 || max_blocks == 0) return SAH_OK;
  status = check_words(what, {sources, lengths});
  if (status != SAH_OK) return status;
  hipLaunchKernelGGL(pool_fork_kernel, dim3((unsigned)ceil_div(max_blocks, kForkColumns)), dim3(kThreads),
                     (size_t)batch * kForkColumns * sizeof(int32_t), reinterpret_cast<hipStream_t>(stream), pool,
                     sources, lengths);
  return check_hip(hipGetLastError(), "block pool fork launch");
}

extern "C" size_t sah_block_pool_compact_workspace_bytes(int64_t num_blocks) {
  if (num_blocks < 0) return 0;
  return (size_t)(2 * (num_blocks / 2 + 1) + num_blocks + 1) * sizeof(int32_t);
}

extern "C" int sah_block_pool_compact(int32_t* block_table, int32_t* holders, int32_t* origins, int32_t* used,
                                      int64_t batch, int64_t max_blocks, int64_t num_blocks, void* workspace,
                                      size_t workspace_bytes, sah_stream_t stream) {
  const char* what = "sah_block_pool_compact";
  CompactArgs a{};
  a.pool = {block_table, holders, num_blocks, (int)batch, (int)max_blocks};
  int status = check_pool(what, a.pool, batch, max_blocks);
  if (status != SAH_OK) return status;
  status = check_words(what, {used});
  if (status != SAH_OK) return status;
  if (num_blocks != 0) {
    status = check_words(what, {origins});
    if (status != SAH_OK) return status;
  }
  status = check_workspace(what, workspace, workspace_bytes, sah_block_pool_compact_workspace_bytes(num_blocks));
  if (status != SAH_OK) return status;
  a.origins = origins;
  a.used = used;
  a.holes = static_cast<int32_t*>(workspace);
  a.movers = a.holes + num_blocks / 2 + 1;
  a.ranks = a.movers + num_blocks / 2 + 1;
  a.moves = a.ranks + num_blocks;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t entries = batch * max_blocks;
  if (entries <= kSmallPool && num_blocks <= kSmallPool) {
    hipLaunchKernelGGL(pool_compact_list_kernel<true>, dim3(1), dim3(kScanThreads), 0, s, a);
    return check_hip(hipGetLastError(), "block pool compact launch");
  }
  hipLaunchKernelGGL(pool_compact_list_kernel<false>, dim3(1), dim3(kScanThreads), 0, s, a);
  status = check_hip(hipGetLastError(), "block pool compact launch");
  if (status != SAH_OK) return status;
  const int64_t most = entries > num_blocks / 2 ? entries : num_blocks / 2;
  const int64_t grid = ceil_div(most, kThreads);
  hipLaunchKernelGGL(pool_compact_apply_kernel, dim3((unsigned)(grid < 2048 ? grid : 2048)), dim3(kThreads), 0, s, a);
  return check_hip(hipGetLastError(), "block pool compact launch");
}

extern "C" int sah_block_cache_copy(void* key_codes, void* value_codes, float* key_scales, float* value_scales,
                                    const int32_t* origins, int64_t kv_heads, int64_t head_dim, int64_t num_blocks,
                                    sah_stream_t stream) {
  const char* what = "sah_block_cache_copy";
  int status = check_places(what, kv_heads, head_dim, num_blocks);
  if (status != SAH_OK) return status;
  if (num_blocks == 0) return SAH_OK;
  status = check_words(what, {key_scales, value_scales, origins});
  if (status != SAH_OK) return status;
  if (key_codes == nullptr || value_codes == nullptr)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", what);
  if (!aligned16(key_codes) || !aligned16(value_codes))
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: codes must be 16-byte aligned", what);
  CopyArgs a{};
  a.codes[0] = static_cast<uint8_t*>(key_codes);
  a.codes[1] = static_cast<uint8_t*>(value_codes);
  a.scales[0] = key_scales;
  a.scales[1] = value_scales;
  a.origins = origins;
  a.blocks = num_blocks;
  a.place_bytes = kv_heads * kBlockTokens * head_dim;
  a.parts = (int)ceil_div(a.place_bytes, kCopyPart);
  a.units = num_blocks * 2 * a.parts;
  a.heads = (int)kv_heads;
  const unsigned grid = (unsigned)(a.units < 2048 ? a.units : 2048);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (2 * num_blocks * a.place_bytes > kPastBytes)
    hipLaunchKernelGGL(cache_copy_kernel<true>, dim3(grid), dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL(cache_copy_kernel<false>, dim3(grid), dim3(kThreads), 0, s, a);
  return check_hip(hipGetLastError(), "block cache copy launch");
}

extern "C" int sah_block_cache_fork(void* key_tail, void* value_tail, const int32_t* sources, int64_t batch,
                                    int64_t kv_heads, int64_t head_dim, sah_stream_t stream) {
  const char* what = "sah_block_cache_fork";
  int status = check_places(what, kv_heads, head_dim, 0);
  if (status != SAH_OK) return status;
  if (batch < 0) return fail(SAH_ERR_INVALID_ARGUMENT, "%s: bad batch %lld", what, (long long)batch);
  if (batch > kMaxForked)
    return fail(SAH_ERR_UNSUPPORTED, "%s: batch %lld is above %d", what, (long long)batch, kMaxForked);
  if (batch == 0) return SAH_OK;
  status = check_words(what, {sources});
  if (status != SAH_OK) return status;
  if (key_tail == nullptr || value_tail == nullptr)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", what);
  if (!aligned16(key_tail) || !aligned16(value_tail))
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: tails must be 16-byte aligned", what);
  // the widest slice whose part of every tail fits 48 KiB
  int slice = 512;
  while (slice * batch > 49152) slice /= 2;
  const int64_t tail_bytes = kv_heads * kBlockTokens * head_dim * 2;
  hipLaunchKernelGGL(cache_fork_kernel, dim3((unsigned)(2 * (tail_bytes / slice))), dim3(kThreads),
                     (size_t)(slice * batch), reinterpret_cast<hipStream_t>(stream), static_cast<char*>(key_tail),
                     static_cast<char*>(value_tail), sources, (int)batch, tail_bytes, slice);
  return check_hip(hipGetLastError(), "block cache fork launch");
}

extern "C" int sah_block_cache_take_back(const void* key_codes, const void* value_codes, const float* key_scales,
                                         const float* value_scales, void* key_tail, void* value_tail,
                                         const int32_t* block_table, const int32_t* lengths, const int32_t* ends,
                                         int64_t batch, int64_t kv_heads, int64_t head_dim, int64_t num_blocks,
                                         int64_t max_blocks, int dtype, sah_stream_t stream) {
  const char* what = "sah_block_cache_take_back";
  int status = check_places(what, kv_heads, head_dim, num_blocks);
  if (status != SAH_OK) return status;
  if (dtype != SAH_DTYPE_BF16 && dtype != SAH_DTYPE_F16)
    return fail(SAH_ERR_UNSUPPORTED, "%s: dtype %d is not bf16 or f16", what, dtype);
  if (batch < 0 || batch > INT32_MAX || max_blocks < 0 || max_blocks > INT32_MAX / kBlockTokens)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: bad batch or block count", what);
  if (batch == 0) return SAH_OK;
  status = check_words(what, {lengths, ends});
  if (status != SAH_OK) return status;
  if (key_tail == nullptr || value_tail == nullptr || (max_blocks != 0 && block_table == nullptr) ||
      (num_blocks != 0 &&
       (key_codes == nullptr || value_codes == nullptr || key_scales == nullptr || value_scales == nullptr)))
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: null cache pointer", what);
  if (!aligned16(key_tail) || !aligned16(value_tail) || !aligned16(key_codes) || !aligned16(value_codes))
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: codes and tails must be 16-byte aligned", what);
  if (((reinterpret_cast<uintptr_t>(key_scales) | reinterpret_cast<uintptr_t>(value_scales) |
        reinterpret_cast<uintptr_t>(block_table)) & 3u) != 0)
    return fail(SAH_ERR_INVALID_ARGUMENT, "%s: scales and block table must be 4-byte aligned", what);
  if (batch > (int64_t)(UINT32_MAX / kThreads) / (2 * kv_heads))
    return fail(SAH_ERR_UNSUPPORTED, "%s: too many heads for one launch", what);
  TakeBackArgs a{};
  a.codes[0] = static_cast<const uint8_t*>(key_codes);
  a.codes[1] = static_cast<const uint8_t*>(value_codes);
  a.scales[0] = key_scales;
  a.scales[1] = value_scales;
  a.tails[0] = key_tail;
  a.tails[1] = value_tail;
  a.table = block_table;
  a.lengths = lengths;
  a.ends = ends;
  a.blocks = num_blocks;
  a.max_blocks = max_blocks;
  a.heads = (int)kv_heads;
  a.head_values = (int)(kBlockTokens * head_dim);
  const dim3 grid((unsigned)(2 * batch * kv_heads));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == SAH_DTYPE_BF16)
    hipLaunchKernelGGL(cache_take_back_kernel<bf16>, grid, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL(cache_take_back_kernel<f16>, grid, dim3(kThreads), 0, s, a);
  return check_hip(hipGetLastError(), "block cache take back launch");
}
