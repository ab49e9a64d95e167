// Pages of a paged KV cache on the device: forked, copied, freed and compacted, gfx950.
//
// A block id is one page of every layer's key and value pools.  references[id] counts its holders beyond the first, so that
// blocks that were never shared need no entry and the reserving kernels (kv_cache.hip, kv_plan.hip) know nothing of it.
//   fork     a new row shares the full blocks of its source and gets a fresh block for a partly filled last one, whose page is
//            then copied: no row ever writes to a block that another holds.
//   release  a row's blocks lose a holder, and go back to the free list with the last one.
//   compact  the largest ids that the tables hold move to the lowest free ones as long as that is lower: then the pools' ends are
//            free.
// The free list stays ascending: release and compact mark the free blocks in a bitmap, 32 blocks a word, and write the list anew
// from it, a block's place being the bits below its own.  So the result does not depend on the order of the atomics that set the
// bits.  Where the books are small one workgroup does all of it in LDS, in one launch; else the bitmap lies in the workspace and a
// workgroup counts all words before its own (a few tens of KB out of L2) rather than wait for its neighbours.
//
// Books are small and latency bounds them; copies are bound by memory, each page read once and written once for each
// copy of it.
#include "qa_common.h"

#include <algorithm>

namespace qa {
namespace pages {

struct Books {
  int32_t* tables;
  int64_t table_stride, max_blocks;
  int32_t* lengths;
  int32_t* free_list;
  int32_t* free_state;  // head, count
  int32_t* references;
  int32_t* status;
  int64_t capacity, rows;
};

__device__ __forceinline__ int64_t index_of(const void* base, int is64, int64_t i) {
  return is64 ? reinterpret_cast<const int64_t*>(base)[i] : reinterpret_cast<const int32_t*>(base)[i];
}

__device__ __forceinline__ bool corrupt(const Books& k) {
  const int64_t head = k.free_state[0], count = k.free_state[1];
  return head < 0 || count < 0 || head + count > k.capacity;
}

// Inclusive sum over a workgroup of THREADS / 64 waves; total: of all.
template <int THREADS>
__device__ __forceinline__ int32_t block_scan(int32_t v, int32_t* s_wave, int32_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int32_t incl = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int32_t u = __shfl_up(incl, off, 64);
    if (lane >= off) incl += u;
  }
  __syncthreads();  // s_wave may still be read
  if (lane == 63) s_wave[wave] = incl;
  __syncthreads();
  int32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) before += s_wave[w];
    total += s_wave[w];
  }
  return before + incl;
}

// ---- fork -------------------------------------------------------------------

struct ForkParams {
  Books k;
  const void* source_rows;
  const void* target_rows;
  int n, rows_i64, bs;
  int32_t* sources;  // (n): the page to be copied, -1: none
  int32_t* targets;
};

constexpr int kForks = 1024;        // of a call: a thread each
constexpr int kMaxRows = 65533;
// Table entries up to which the forking workgroup writes them itself.
constexpr int64_t kInlineEntries = 8192;

// Entry e of fork i, and a holder more for a block that it shares.
__device__ __forceinline__ void fork_entry(const Books& k, int64_t source, int64_t target, int64_t e, int64_t entries, int32_t own) {
  int32_t id = k.tables[source * k.table_stride + e];
  if (own >= 0 && e == entries - 1)
    id = own;
  else if (id >= 0 && id < k.capacity)
    atomicAdd(&k.references[id], 1);
  k.tables[target * k.table_stride + e] = id;
}

__global__ __launch_bounds__(kForks) void fork_kernel(ForkParams p, int inline_entries) {
  __shared__ uint32_t s_targets[(kMaxRows + 31) / 32 + 1], s_sources[(kMaxRows + 31) / 32 + 1];
  __shared__ int32_t s_wave[kForks / 64];
  __shared__ int32_t s_row[kForks][2], s_own[kForks], s_entries[kForks];
  __shared__ int s_code;
  const Books& k = p.k;
  const int i = threadIdx.x;
  int64_t source = -1, target = -1;
  if (i < p.n) {
    source = index_of(p.source_rows, p.rows_i64, i);
    target = index_of(p.target_rows, p.rows_i64, i);
  }
  const bool live = source >= 0;  // -1: no fork
  const int64_t head = k.free_state[0], count = k.free_state[1];
  for (int w = i; w < (k.rows + 31) / 32; w += kForks) s_targets[w] = s_sources[w] = 0;
  if (i == 0) s_code = head < 0 || count < 0 || head + count > k.capacity ? 3 : 0;
  __syncthreads();
  const bool rows_ok = live && source < k.rows && target >= 0 && target < k.rows;
  int bad = live && !rows_ok ? 6 : 0;
  if (rows_ok) {
    const uint32_t bit = 1u << (target & 31);
    if (atomicOr(&s_targets[target >> 5], bit) & bit) bad = 6;  // named twice
    atomicOr(&s_sources[source >> 5], 1u << (source & 31));
  }
  int64_t length = 0;
  int32_t last = -1;
  if (rows_ok) {
    if (k.lengths[target] != 0) bad = 6;
    length = k.lengths[source];
    if (length < 0 || length > k.max_blocks * p.bs)
      bad = max(bad, 4);
    else if (length % p.bs != 0)
      last = k.tables[source * k.table_stride + length / p.bs];
  }
  __syncthreads();
  if (rows_ok && (s_sources[target >> 5] >> (target & 31) & 1)) bad = 6;
  if (bad != 0) atomicMax(&s_code, bad);
  const bool need = last >= 0 && last < k.capacity;
  int32_t total;
  const int32_t upto = block_scan<kForks>(need ? 1 : 0, s_wave, total);
  const int code = s_code != 0 ? s_code : total > count ? 1 : 0;  // the scan's barriers stand between the atomics and this
  const int32_t own = need && code == 0 ? k.free_list[head + upto - 1] : -1;
  if (i < p.n) {
    p.sources[i] = need && code == 0 ? last : -1;
    p.targets[i] = own;
    if (live && code == 0) k.lengths[target] = static_cast<int32_t>(length);
  }
  if (i == 0) {
    k.status[0] = code;
    if (code == 0) {
      k.free_state[0] = static_cast<int32_t>(head + total);
      k.free_state[1] = static_cast<int32_t>(count - total);
    }
  }
  if (!inline_entries || code != 0) return;
  s_row[i][0] = static_cast<int32_t>(source);
  s_row[i][1] = static_cast<int32_t>(target);
  s_own[i] = own;
  s_entries[i] = live ? static_cast<int32_t>((length + p.bs - 1) / p.bs) : 0;
  __syncthreads();
  for (int f = i / 64; f < p.n; f += kForks / 64)  // a wave a fork
    for (int e = i % 64; e < s_entries[f]; e += 64) fork_entry(k, s_row[f][0], s_row[f][1], e, s_entries[f], s_own[f]);
}

// Table entries of fork blockIdx.y, a holder more for each block that it shares.
__global__ __launch_bounds__(256) void fork_tables_kernel(ForkParams p) {
  const Books& k = p.k;
  const int i = blockIdx.y;
  const int64_t source = index_of(p.source_rows, p.rows_i64, i);
  if (source < 0 || k.status[0] != 0) return;
  const int64_t target = index_of(p.target_rows, p.rows_i64, i);
  const int64_t length = k.lengths[source];
  const int64_t entries = (length + p.bs - 1) / p.bs;
  const int32_t own = p.targets[i];
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < entries; e += static_cast<int64_t>(gridDim.x) * 256) fork_entry(k, source, target, e, entries, own);
}

// ---- the free list from a bitmap ----------------------------------------------

constexpr int kListThreads = 256;
constexpr int kListWords = 64;  // of a workgroup where the bitmap lies in the workspace, at most

// One workgroup does a release or a compaction where the pool has up to so many blocks, the rows so many table entries, and a
// compaction so many pairs.  us of a release and a compaction in one workgroup / in several: 8000 blocks 10 / 9 and 18 / 17, but a
// fill and a launch more each, 8 us of the host; 470 blocks, a compaction 6 / 13; 32000 blocks 27 / 9 and 50 / 22.
constexpr int kSmallThreads = 1024;  // each a word of the bitmap at most
constexpr int64_t kSmallBlocks = 8192;
constexpr int64_t kSmallEntries = 16384;
static_assert(kSmallBlocks <= 32 * kSmallThreads, "a word a thread");

__device__ __forceinline__ void set_bit(uint32_t* bits, int32_t id) { atomicOr(&bits[id >> 5], 1u << (id & 31)); }
__device__ __forceinline__ uint32_t below(int32_t id) { return (1u << (id & 31)) - 1u; }

// Marks the free list's blocks in the workspace's bitmap.  Neighbours in the list share words, so a wave gathers the bits of a word first; what is left after
// a few words goes by itself: a release in a pool of 322,000 blocks 105 -> 29 us.
__device__ __forceinline__ void mark_free(const Books& k, uint32_t* bits, int64_t first, int64_t step) {
  const int64_t head = k.free_state[0], count = k.free_state[1];
  const int lane = threadIdx.x & 63;
  for (int64_t i = first; i - lane < count; i += step) {
    const int32_t id = i < count ? k.free_list[head + i] : -1;
    bool left = id >= 0 && id < k.capacity;
    for (int turn = 0; turn < 4; ++turn) {
      const uint64_t some = __ballot(left);
      if (some == 0) break;
      const int leader = __ffsll(static_cast<unsigned long long>(some)) - 1;
      const int32_t word = __builtin_amdgcn_readlane(id >> 5, leader);
      const bool mine = left && id >> 5 == word;
      uint32_t all = mine ? 1u << (id & 31) : 0u;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) all |= __shfl_xor(all, off, 64);
      if (lane == leader) atomicOr(&bits[word], all);
      left = left && !mine;
    }
    if (left) set_bit(bits, id);
  }
}

__device__ __forceinline__ void mark_free_lds(const Books& k, uint32_t* bits, int tid) {
  const int64_t head = k.free_state[0], count = k.free_state[1];
  for (int64_t i = tid; i < count; i += kSmallThreads) {
    const int32_t id = k.free_list[head + i];
    if (id >= 0 && id < k.capacity) set_bit(bits, id);
  }
}

// Where the bitmap lies in the workspace: the bits below each of this workgroup's words go to s_before, `total` is all of them.
template <typename F>
__device__ __forceinline__ void count_words(int64_t words, int list_words, F word, int32_t* s_wave, int32_t* s_before, int32_t& total) {
  const int64_t base = static_cast<int64_t>(blockIdx.x) * list_words;
  int32_t before = 0, all = 0;
  for (int64_t w = threadIdx.x; w < words; w += kListThreads) {
    const int32_t c = __popc(word(w));
    if (w < base) before += c;
    all += c;
  }
  int32_t sum, own;
  block_scan<kListThreads>(before, s_wave, sum);
  block_scan<kListThreads>(all, s_wave, total);
  const int32_t mine = threadIdx.x < list_words && base + threadIdx.x < words ? __popc(word(base + threadIdx.x)) : 0;
  const int32_t incl = block_scan<kListThreads>(mine, s_wave, own);
  if (threadIdx.x < list_words) s_before[threadIdx.x] = sum + incl - mine;
  __syncthreads();
}

// Blocks id0, id0 + step .. below id1 of the list: a free block at the place that the bits below it give, -1 behind the end.
template <typename F>
__device__ __forceinline__ void write_list(const Books& k, int64_t id0, int64_t id1, int64_t step, F word, const int32_t* before, int64_t first_word, int32_t total) {
  for (int64_t i = id0; i < id1; i += step) {
    const int32_t id = static_cast<int32_t>(i);
    const uint32_t bits = word(id >> 5);
    if (bits >> (id & 31) & 1) k.free_list[before[(id >> 5) - first_word] + __popc(bits & below(id))] = id;
    if (i >= total) k.free_list[i] = -1;
  }
}

__device__ __forceinline__ void close_books(const Books& k, int32_t total) {
  k.free_state[0] = 0;
  k.free_state[1] = total;
  k.status[0] = 0;
}

// ---- release ------------------------------------------------------------------

struct ReleaseParams {
  Books k;
  const void* release_rows;
  int n, rows_i64;
  uint32_t* bits;    // (words + 1), zeros: free blocks; the last word is 1 where the free list's cursor is out of range
  int64_t words;
  int list_words;    // of a workgroup of the second launch
};

// The table entries first, first + step .. of a row lose their blocks, four at a time: each is a chain of a load and three atomics,
// one after the other 10.4 us for 16 rows of 256, so 8.8 to 9.0.
__device__ __forceinline__ void release_entries(const Books& k, int64_t row, int64_t first, int64_t step, uint32_t* bits) {
  constexpr int kAtOnce = 4;
  int32_t* entries = &k.tables[row * k.table_stride];
  for (int64_t e = first; e < k.max_blocks; e += kAtOnce * step) {
    int32_t id[kAtOnce], holders[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) id[j] = e + j * step < k.max_blocks ? entries[e + j * step] : -1;
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if (id[j] != -1) id[j] = atomicExch(&entries[e + j * step], -1);  // a row named twice is freed once
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      holders[j] = 1;
      if (static_cast<uint32_t>(id[j]) < static_cast<uint32_t>(k.capacity)) holders[j] = atomicSub(&k.references[id[j]], 1);
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) asm volatile("" : "+v"(holders[j]));  // all of them on their way before the first is looked at
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (holders[j] > 0) continue;
      atomicAdd(&k.references[id[j]], 1);
      set_bit(bits, id[j]);
    }
  }
}

// All of it in one workgroup.
__global__ __launch_bounds__(kSmallThreads) void release_small_kernel(ReleaseParams p) {
  __shared__ uint32_t s_bits[kSmallThreads];
  __shared__ int32_t s_before[kSmallThreads], s_wave[kSmallThreads / 64];
  const Books& k = p.k;
  const int tid = threadIdx.x;
  s_bits[tid] = 0;
  if (corrupt(k)) {
    if (tid == 0) k.status[0] = 3;
    return;
  }
  __syncthreads();
  mark_free_lds(k, s_bits, tid);
  for (int i = tid / 64; i < p.n; i += kSmallThreads / 64) {  // a wave a row
    const int64_t row = index_of(p.release_rows, p.rows_i64, i);
    if (row < 0 || row >= k.rows) continue;
    release_entries(k, row, tid % 64, 64, s_bits);
    if (tid % 64 == 0) k.lengths[row] = 0;
  }
  __syncthreads();
  int32_t total;
  const int32_t mine = __popc(s_bits[tid]);
  s_before[tid] = block_scan<kSmallThreads>(mine, s_wave, total) - mine;
  __syncthreads();
  write_list(k, tid, k.capacity, kSmallThreads, [&](int64_t w) { return s_bits[w]; }, s_before, 0, total);
  if (tid == 0) close_books(k, total);
}

// blockIdx.y < n: the blocks of a row; n: the free list.
__global__ __launch_bounds__(256) void release_kernel(ReleaseParams p) {
  const Books& k = p.k;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * 256;
  if (corrupt(k)) {
    if (first == 0) p.bits[p.words] = 1;
    return;
  }
  if (static_cast<int>(blockIdx.y) == p.n) {
    mark_free(k, p.bits, first, step);
    return;
  }
  const int64_t row = index_of(p.release_rows, p.rows_i64, blockIdx.y);
  if (row < 0 || row >= k.rows) return;
  release_entries(k, row, first, step, p.bits);
  if (first == 0) k.lengths[row] = 0;
}

__global__ __launch_bounds__(kListThreads) void release_list_kernel(ReleaseParams p) {
  __shared__ int32_t s_wave[kListThreads / 64], s_before[kListWords];
  const Books& k = p.k;
  if (p.bits[p.words] != 0) {
    if (blockIdx.x == 0 && threadIdx.x == 0) k.status[0] = 3;
    return;
  }
  auto word = [&](int64_t w) { return p.bits[w]; };
  int32_t total;
  count_words(p.words, p.list_words, word, s_wave, s_before, total);
  const int64_t w0 = static_cast<int64_t>(blockIdx.x) * p.list_words;
  write_list(k, 32 * w0 + threadIdx.x, min64(k.capacity, 32 * (w0 + p.list_words)), kListThreads, word, s_before, w0, total);
  if (blockIdx.x == 0 && threadIdx.x == 0) close_books(k, total);
}

// ---- compact --------------------------------------------------------------------

struct CompactParams {
  Books k;
  int64_t words, max_moves;
  uint32_t* free_bits;  // (words), zeros
  uint32_t* held;       // (words), zeros: blocks that the tables hold
  uint32_t* flip;       // (words), zeros: blocks that are taken or left
  uint32_t* refused;    // (1), zero
  int32_t* place;       // (capacity): where a block that is left has gone
  int32_t* sources;     // (max_moves)
  int32_t* targets;
  int list_words, list_groups;  // words of a workgroup that counts them, and workgroups
};

// Where a held block with `nth` held ones above it goes, -1: it stays.
__device__ __forceinline__ int32_t place_of(const CompactParams& p, int32_t nth, int32_t source) {
  if (nth >= min64(p.max_moves, p.k.free_state[1])) return -1;
  const int32_t target = p.k.free_list[p.k.free_state[0] + static_cast<int64_t>(nth)];
  return target < source ? target : -1;
}

__device__ __forceinline__ void move_block(const CompactParams& p, int32_t nth, int32_t source, int32_t target, uint32_t* flip) {
  p.sources[nth] = source;
  p.targets[nth] = target;
  p.k.references[target] = p.k.references[source];
  p.k.references[source] = 0;
  set_bit(flip, source);
  set_bit(flip, target);
}

// All of it in one workgroup.
__global__ __launch_bounds__(kSmallThreads) void compact_small_kernel(CompactParams p) {
  __shared__ uint32_t s_free[kSmallThreads], s_held[kSmallThreads], s_flip[kSmallThreads];
  __shared__ int32_t s_before[kSmallThreads], s_wave[kSmallThreads / 64];
  const Books& k = p.k;
  const int tid = threadIdx.x;
  s_free[tid] = s_held[tid] = s_flip[tid] = 0;
  for (int64_t i = tid; i < p.max_moves; i += kSmallThreads) p.sources[i] = p.targets[i] = -1;
  if (corrupt(k)) {
    if (tid == 0) k.status[0] = 3;
    return;
  }
  __syncthreads();
  mark_free_lds(k, s_free, tid);
  for (int64_t row = tid / 64; row < k.rows; row += kSmallThreads / 64)
    for (int64_t e = tid % 64; e < k.max_blocks; e += 64) {
      const int32_t id = k.tables[row * k.table_stride + e];
      if (id >= 0 && id < k.capacity) set_bit(s_held, id);
    }
  __syncthreads();
  s_held[tid] &= ~s_free[tid];
  int32_t total;
  const int32_t mine = __popc(s_held[tid]);
  s_before[tid] = block_scan<kSmallThreads>(mine, s_wave, total) - mine;
  __syncthreads();
  auto nth_of = [&](int32_t id) { return total - 1 - s_before[id >> 5] - __popc(s_held[id >> 5] & below(id)); };
  for (int64_t i = tid; i < k.capacity; i += kSmallThreads) {
    const int32_t id = static_cast<int32_t>(i);
    if (!(s_held[id >> 5] >> (id & 31) & 1)) continue;
    const int32_t nth = nth_of(id), target = place_of(p, nth, id);
    if (target >= 0) move_block(p, nth, id, target, s_flip);
  }
  __syncthreads();
  for (int64_t row = tid / 64; row < k.rows; row += kSmallThreads / 64)
    for (int64_t e = tid % 64; e < k.max_blocks; e += 64) {
      int32_t* entry = &k.tables[row * k.table_stride + e];
      const int32_t id = *entry;
      if (id >= 0 && id < k.capacity && (s_held[id >> 5] & s_flip[id >> 5]) >> (id & 31) & 1) *entry = place_of(p, nth_of(id), id);
    }
  __syncthreads();  // the old list has been read
  const uint32_t bits = s_free[tid] ^ s_flip[tid];
  const int32_t free_here = __popc(bits);
  const int32_t incl = block_scan<kSmallThreads>(free_here, s_wave, total);
  s_before[tid] = incl - free_here;
  s_free[tid] = bits;
  __syncthreads();
  write_list(k, tid, k.capacity, kSmallThreads, [&](int64_t w) { return s_free[w]; }, s_before, 0, total);
  if (tid == 0) close_books(k, total);
}

// blockIdx.y < rows: the blocks of a row; then the free list; then the pairs, set to none.
__global__ __launch_bounds__(256) void compact_mark_kernel(CompactParams p) {
  const Books& k = p.k;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * 256;
  const int64_t y = blockIdx.y;
  if (y == k.rows + 1) {
    for (int64_t i = first; i < p.max_moves; i += step) p.sources[i] = p.targets[i] = -1;
    return;
  }
  if (corrupt(k)) {
    if (first == 0) p.refused[0] = 1;
    return;
  }
  if (y == k.rows) {
    mark_free(k, p.free_bits, first, step);
    return;
  }
  for (int64_t e = first; e < k.max_blocks; e += step) {
    const int32_t id = k.tables[y * k.table_stride + e];
    if (id >= 0 && id < k.capacity) set_bit(p.held, id);
  }
}

__global__ __launch_bounds__(kListThreads) void compact_moves_kernel(CompactParams p) {
  __shared__ int32_t s_wave[kListThreads / 64], s_before[kListWords];
  const Books& k = p.k;
  if (p.refused[0] != 0) return;
  auto word = [&](int64_t w) { return p.held[w] & ~p.free_bits[w]; };
  int32_t total;
  count_words(p.words, p.list_words, word, s_wave, s_before, total);
  const int64_t w0 = static_cast<int64_t>(blockIdx.x) * p.list_words, end = min64(k.capacity, 32 * (w0 + p.list_words));
  for (int64_t i = 32 * w0 + threadIdx.x; i < end; i += kListThreads) {
    const int32_t id = static_cast<int32_t>(i);
    const uint32_t bits = word(id >> 5);
    if (!(bits >> (id & 31) & 1)) continue;
    const int32_t nth = total - 1 - s_before[(id >> 5) - w0] - __popc(bits & below(id)), target = place_of(p, nth, id);
    if (target < 0) continue;
    p.place[id] = target;
    move_block(p, nth, id, target, p.flip);
  }
}

// blockIdx.y 0: the free list; then the tables' rows.
__global__ __launch_bounds__(kListThreads) void compact_list_kernel(CompactParams p) {
  __shared__ int32_t s_wave[kListThreads / 64], s_before[kListWords];
  const Books& k = p.k;
  if (p.refused[0] != 0) {
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) k.status[0] = 3;
    return;
  }
  if (blockIdx.y == 0) {
    if (static_cast<int>(blockIdx.x) >= p.list_groups) return;
    auto word = [&](int64_t w) { return p.free_bits[w] ^ p.flip[w]; };
    int32_t total;
    count_words(p.words, p.list_words, word, s_wave, s_before, total);
    const int64_t w0 = static_cast<int64_t>(blockIdx.x) * p.list_words;
    write_list(k, 32 * w0 + threadIdx.x, min64(k.capacity, 32 * (w0 + p.list_words)), kListThreads, word, s_before, w0, total);
    if (blockIdx.x == 0 && threadIdx.x == 0) close_books(k, total);
    return;
  }
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * kListThreads + threadIdx.x; e < k.max_blocks; e += static_cast<int64_t>(gridDim.x) * kListThreads) {
    int32_t* entry = &k.tables[(blockIdx.y - 1) * k.table_stride + e];
    const int32_t id = *entry;
    if (id < 0 || id >= k.capacity) continue;
    if ((p.flip[id >> 5] & p.held[id >> 5] & ~p.free_bits[id >> 5]) >> (id & 31) & 1) *entry = p.place[id];
  }
}

// ---- copy -----------------------------------------------------------------------

constexpr int kPools = 32;  // of a launch

// Not uint4: an array of those went to LDS, by an address for which each workgroup read its launch's size from the host's memory,
// 12 us where the first workgroup of every CU did.
typedef uint32_t uintx4_v __attribute__((ext_vector_type(4)));

struct PoolOfPages {
  uint8_t* base;
  int64_t stride;  // bytes from page to page
  int64_t bytes;   // of a page
  int64_t count;   // pages
};

struct CopyParams {
  const void* sources;
  const void* targets;
  int64_t n;
  int ids_i64;
  uint32_t groups;  // gridDim.x
  PoolOfPages pools[kPools];
};

constexpr int kCopyThreads = 256;
constexpr int kInFlight = 4;  // units a thread has on their way
constexpr int64_t kCopyGroups = 4096;

// UNIT: 16 or 4 bytes.  Workgroups take pieces of kCopyThreads * kInFlight units of the pages of pool blockIdx.y in turn.
template <typename UNIT>
__global__ __launch_bounds__(kCopyThreads) void copy_kernel(CopyParams p) {
  const PoolOfPages pool = p.pools[blockIdx.y];
  const int64_t units = pool.bytes / static_cast<int64_t>(sizeof(UNIT));
  const uint32_t pieces = static_cast<uint32_t>((units + kCopyThreads * kInFlight - 1) / (kCopyThreads * kInFlight));  // memory ends long before 2^32
  if (pieces == 0) return;
  const uint32_t pairs_ahead = p.groups / pieces, pieces_ahead = p.groups - pairs_ahead * pieces;
  int64_t pair = blockIdx.x / pieces;
  uint32_t piece = blockIdx.x - static_cast<uint32_t>(pair) * pieces;
  while (pair < p.n) {
    const int64_t source = index_of(p.sources, p.ids_i64, pair), target = index_of(p.targets, p.ids_i64, pair);
    if (source >= 0 && target >= 0 && source < pool.count && target < pool.count) {
      const UNIT* from = reinterpret_cast<const UNIT*>(pool.base + source * pool.stride);
      UNIT* to = reinterpret_cast<UNIT*>(pool.base + target * pool.stride);
      const int64_t u0 = static_cast<int64_t>(piece) * (kCopyThreads * kInFlight) + threadIdx.x;
      UNIT u[kInFlight];
#pragma unroll
      for (int i = 0; i < kInFlight; ++i) u[i] = from[min64(u0 + i * kCopyThreads, units - 1)];
#pragma unroll
      for (int i = 0; i < kInFlight; ++i)
        if (u0 + i * kCopyThreads < units) to[u0 + i * kCopyThreads] = u[i];
    }
    pair += pairs_ahead;
    piece += pieces_ahead;
    if (piece >= pieces) {
      piece -= pieces;
      ++pair;
    }
  }
}

// ---- host -----------------------------------------------------------------------

static int64_t words_of(int64_t capacity) { return ceil_div(capacity, 32); }

// Whether one workgroup does a release or a compaction.
static bool small(int64_t capacity, int64_t entries, int64_t pairs) { return capacity <= kSmallBlocks && entries <= kSmallEntries && pairs <= kSmallBlocks; }

static int check_books(const char* what, const Books& k) {
  QA_REQUIRE(k.tables && k.free_list && k.free_state && k.references && k.status, "%s: pointers must be non-null", what);
  QA_REQUIRE(k.rows >= 1 && k.rows <= kMaxRows, "%s: the tables must have 1 to 65533 rows", what);
  QA_REQUIRE(k.max_blocks >= 1 && k.max_blocks <= 0x7fffffff, "%s: block table must have at least one entry", what);
  QA_REQUIRE(k.table_stride >= k.max_blocks || k.rows == 1, "table rows overlap: stride %lld < max_blocks %lld", static_cast<long long>(k.table_stride), static_cast<long long>(k.max_blocks));
  QA_REQUIRE(k.capacity >= 1 && k.capacity <= 0x7fffffff, "free list capacity must be in [1, 2^31)");
  return 0;
}

// Words of a workgroup that counts them: few, so that its threads have a block or two each, but no more workgroups than 256,
// since each reads all words.
static int list_words_of(int64_t words) { return static_cast<int>(std::min<int64_t>(kListWords, std::max<int64_t>(16, ceil_div(words, 256)))); }

// Workgroups along an axis of `n` entries: enough for a few entries a thread.
static unsigned groups_of(int64_t n) { return static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(ceil_div(n, 256), 1), 256)); }

}  // namespace pages
}  // namespace qa

extern "C" int qa_paged_kv_fork(int32_t* block_tables, int64_t table_stride, int64_t max_blocks, int32_t* lengths, int64_t rows, const void* source_rows,
                                const void* target_rows, int32_t rows_dtype, int64_t n, int32_t block_size, const int32_t* free_list, int64_t free_capacity,
                                int32_t* free_state, int32_t* references, int32_t* status, int32_t* sources, int32_t* targets, hipStream_t stream) {
  using namespace qa;
  using namespace qa::pages;
  ForkParams p{};
  p.k = {block_tables, table_stride, max_blocks, lengths, const_cast<int32_t*>(free_list), free_state, references, status, free_capacity, rows};
  if (int rc = check_books("paged_kv_fork", p.k)) return rc;
  QA_REQUIRE(is_index_dtype(rows_dtype), "paged_kv_fork: rows must be int32 or int64");
  QA_REQUIRE(n >= 0 && n <= kForks, "paged_kv_fork: at most %d forks a call", kForks);
  QA_REQUIRE(block_size > 0 && block_size <= 65536, "paged_kv_fork: block_size must be in [1, 65536]");
  QA_REQUIRE(lengths != nullptr && (n == 0 || (source_rows && target_rows && sources && targets)), "paged_kv_fork: pointers must be non-null");
  p.source_rows = source_rows;
  p.target_rows = target_rows;
  p.n = static_cast<int>(n);
  p.rows_i64 = rows_dtype == QA_I64;
  p.bs = block_size;
  p.sources = sources;
  p.targets = targets;
  {
    KernelTimer timer_("kv_fork", stream);
    hipLaunchKernelGGL(fork_kernel, dim3(1), dim3(kForks), 0, stream, p, n * max_blocks <= kInlineEntries ? 1 : 0);
  }
  if (int rc = check_launch("paged_kv_fork")) return rc;
  if (n * max_blocks <= kInlineEntries) return 0;
  {
    KernelTimer timer_("kv_fork_tables", stream);
    hipLaunchKernelGGL(fork_tables_kernel, dim3(groups_of(max_blocks), static_cast<unsigned>(n)), dim3(256), 0, stream, p);
  }
  return check_launch("paged_kv_fork");
}

extern "C" int64_t qa_paged_kv_release_workspace(int64_t free_capacity, int64_t n, int64_t max_blocks) {
  if (free_capacity <= 0 || n < 0 || max_blocks <= 0 || qa::pages::small(free_capacity, n * max_blocks, 0)) return 0;
  return 4 * (qa::pages::words_of(free_capacity) + 1);
}

extern "C" int qa_paged_kv_release(int32_t* block_tables, int64_t table_stride, int64_t max_blocks, int32_t* lengths, int64_t rows, const void* release_rows,
                                   int32_t rows_dtype, int64_t n, int32_t* free_list, int64_t free_capacity, int32_t* free_state, int32_t* references, int32_t* status,
                                   void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  using namespace qa;
  using namespace qa::pages;
  ReleaseParams p{};
  p.k = {block_tables, table_stride, max_blocks, lengths, free_list, free_state, references, status, free_capacity, rows};
  if (int rc = check_books("paged_kv_release", p.k)) return rc;
  QA_REQUIRE(is_index_dtype(rows_dtype), "paged_kv_release: rows must be int32 or int64");
  QA_REQUIRE(n >= 0 && n <= 65533, "paged_kv_release: at most 65533 rows a call");
  QA_REQUIRE(lengths != nullptr && (n == 0 || release_rows != nullptr), "paged_kv_release: pointers must be non-null");
  const int64_t need = qa_paged_kv_release_workspace(free_capacity, n, max_blocks);
  QA_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 3u) == 0),
             "paged_kv_release: workspace too small or not 4-byte aligned: need %lld bytes", static_cast<long long>(need));
  p.release_rows = release_rows;
  p.n = static_cast<int>(n);
  p.rows_i64 = rows_dtype == QA_I64;
  p.bits = reinterpret_cast<uint32_t*>(workspace);
  p.words = words_of(free_capacity);
  p.list_words = list_words_of(p.words);
  if (need == 0) {
    {
      KernelTimer timer_("kv_release", stream);
      hipLaunchKernelGGL(release_small_kernel, dim3(1), dim3(kSmallThreads), 0, stream, p);
    }
    return check_launch("paged_kv_release");
  }
  {
    KernelTimer timer_("kv_release", stream);
    hipLaunchKernelGGL(release_kernel, dim3(groups_of(std::max(max_blocks, free_capacity)), static_cast<unsigned>(n + 1)), dim3(256), 0, stream, p);
  }
  if (int rc = check_launch("paged_kv_release")) return rc;
  {
    KernelTimer timer_("kv_release_list", stream);
    hipLaunchKernelGGL(release_list_kernel, dim3(static_cast<unsigned>(ceil_div(p.words, p.list_words))), dim3(kListThreads), 0, stream, p);
  }
  return check_launch("paged_kv_release");
}

extern "C" int64_t qa_paged_kv_compact_workspace(int64_t free_capacity, int64_t rows, int64_t max_blocks, int64_t max_moves) {
  if (free_capacity <= 0 || rows <= 0 || max_blocks <= 0 || max_moves < 0 || qa::pages::small(free_capacity, rows * max_blocks, max_moves)) return 0;
  return 4 * (3 * qa::pages::words_of(free_capacity) + 1 + free_capacity);
}

extern "C" int qa_paged_kv_compact(int32_t* block_tables, int64_t table_stride, int64_t max_blocks, int64_t rows, int32_t* free_list, int64_t free_capacity,
                                   int32_t* free_state, int32_t* references, int32_t* status, int64_t max_moves, int32_t* sources, int32_t* targets, void* workspace,
                                   int64_t workspace_bytes, hipStream_t stream) {
  using namespace qa;
  using namespace qa::pages;
  CompactParams p{};
  p.k = {block_tables, table_stride, max_blocks, nullptr, free_list, free_state, references, status, free_capacity, rows};
  if (int rc = check_books("paged_kv_compact", p.k)) return rc;
  QA_REQUIRE(max_moves >= 0 && max_moves <= 0x7fffffff, "paged_kv_compact: max_moves out of range");
  QA_REQUIRE(max_moves == 0 || (sources && targets), "paged_kv_compact: pointers must be non-null");
  const int64_t need = qa_paged_kv_compact_workspace(free_capacity, rows, max_blocks, max_moves);
  QA_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 3u) == 0),
             "paged_kv_compact: workspace too small or not 4-byte aligned: need %lld bytes", static_cast<long long>(need));
  p.words = words_of(free_capacity);
  p.max_moves = max_moves;
  p.sources = sources;
  p.targets = targets;
  if (need == 0) {
    {
      KernelTimer timer_("kv_compact", stream);
      hipLaunchKernelGGL(compact_small_kernel, dim3(1), dim3(kSmallThreads), 0, stream, p);
    }
    return check_launch("paged_kv_compact");
  }
  p.free_bits = reinterpret_cast<uint32_t*>(workspace);
  p.held = p.free_bits + p.words;
  p.flip = p.held + p.words;
  p.refused = p.flip + p.words;
  p.place = reinterpret_cast<int32_t*>(p.refused + 1);
  p.list_words = list_words_of(p.words);
  const unsigned lists = static_cast<unsigned>(ceil_div(p.words, p.list_words));
  p.list_groups = static_cast<int>(lists);
  {
    KernelTimer timer_("kv_compact_mark", stream);
    hipLaunchKernelGGL(compact_mark_kernel, dim3(groups_of(std::max(max_blocks, free_capacity)), static_cast<unsigned>(rows + 2)), dim3(256), 0, stream, p);
  }
  if (int rc = check_launch("paged_kv_compact")) return rc;
  {
    KernelTimer timer_("kv_compact_moves", stream);
    hipLaunchKernelGGL(compact_moves_kernel, dim3(lists), dim3(kListThreads), 0, stream, p);
  }
  if (int rc = check_launch("paged_kv_compact")) return rc;
  {
    KernelTimer timer_("kv_compact_list", stream);
    hipLaunchKernelGGL(compact_list_kernel, dim3(std::max(lists, groups_of(max_blocks)), static_cast<unsigned>(rows + 1)), dim3(kListThreads), 0, stream, p);
  }
  return check_launch("paged_kv_compact");
}

extern "C" int qa_paged_kv_copy(void* const* pools, const int64_t* page_strides, const int64_t* page_bytes, const int64_t* page_counts, int64_t num_pools,
                                const void* sources, const void* targets, int32_t ids_dtype, int64_t n, hipStream_t stream) {
  using namespace qa;
  using namespace qa::pages;
  QA_REQUIRE(num_pools >= 0 && n >= 0 && n <= 0x7fffffff, "paged_kv_copy: counts out of range");
  QA_REQUIRE(is_index_dtype(ids_dtype), "paged_kv_copy: page ids must be int32 or int64");
  if (num_pools == 0 || n == 0) return 0;
  QA_REQUIRE(pools && page_strides && page_bytes && page_counts && sources && targets, "paged_kv_copy: pointers must be non-null");
  bool wide = true;
  for (int64_t i = 0; i < num_pools; ++i) {
    QA_REQUIRE(pools[i] != nullptr || page_counts[i] == 0, "paged_kv_copy: pool %lld is null", static_cast<long long>(i));
    QA_REQUIRE(page_counts[i] >= 0 && page_bytes[i] >= 0 && (page_strides[i] >= page_bytes[i] || page_counts[i] <= 1), "paged_kv_copy: pages of pool %lld overlap", static_cast<long long>(i));
    const uint64_t all = reinterpret_cast<uintptr_t>(pools[i]) | static_cast<uint64_t>(page_strides[i]) | static_cast<uint64_t>(page_bytes[i]);
    QA_REQUIRE((all & 3u) == 0, "paged_kv_copy: pages of pool %lld are not of 4-byte units", static_cast<long long>(i));
    if (all & 15u) wide = false;
  }
  for (int64_t i0 = 0; i0 < num_pools; i0 += kPools) {
    const int64_t here = std::min<int64_t>(kPools, num_pools - i0);
    CopyParams p{};
    int64_t units = 0;
    for (int64_t i = 0; i < here; ++i) {
      p.pools[i] = {reinterpret_cast<uint8_t*>(pools[i0 + i]), page_strides[i0 + i], page_bytes[i0 + i], page_counts[i0 + i]};
      units = std::max(units, p.pools[i].bytes / (wide ? 16 : 4));
    }
    if (units == 0) continue;
    p.sources = sources;
    p.targets = targets;
    p.n = n;
    p.ids_i64 = ids_dtype == QA_I64;
    p.groups = static_cast<uint32_t>(std::min<int64_t>(n * ceil_div(units, kCopyThreads * kInFlight), kCopyGroups));
    const dim3 grid(p.groups, static_cast<unsigned>(here));
    KernelTimer timer_("kv_copy", stream);
    if (wide)
      hipLaunchKernelGGL(copy_kernel<uintx4_v>, grid, dim3(kCopyThreads), 0, stream, p);
    else
      hipLaunchKernelGGL(copy_kernel<uint32_t>, grid, dim3(kCopyThreads), 0, stream, p);
  }
  return check_launch("paged_kv_copy");
}
