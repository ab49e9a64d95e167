// The split of a prefill over a paged cache in runs of 16 tokens, whatever a run holds: workgroups of COLS columns and tiles of
// 64 keys, the keys split over gridDim.z where the columns are few, and the launch that joins the parts.  One copy of it for
// each kernel that uses it.
#pragma once

#include "attention_paged.h"

#include <algorithm>
#include <cmath>

namespace qa {
namespace attn {
namespace {

struct PrefillParams {
  Params c;
  int64_t max_new;  // tokens of a row that are computed
  int splits;       // parts of the keys that the launch has workgroups for
  float per_tile;   // kPerTile / workgroups
  int64_t part_tokens;  // tokens that the partial results have room for
  int64_t per_row;      // 0: a token's are where its query is; else row b's begin at b per_row (a padded query)
  float* part_o;        // (splits, part_tokens, H, D)
  float* part_ml;       // (splits, part_tokens, H, 2)
};

constexpr int kTile = 64;      // keys
constexpr int kRuns = kTile / 16;
constexpr int kMaxSplits = 64;
// Batches up to this many rows start with the longest row, so that the launch ends on short ones: 60 rows of up to 300 new
// tokens behind up to 4000 439 -> 403 us, 12 of up to 1500 behind up to 8000 738 -> 677; 64 equal rows of 16 64.5 -> 65.8.
constexpr int kRankRows = 64;

// Keys that the columns up to the last, of a row with `prefix` cached tokens, see: not past the table.
template <typename P>
__device__ __forceinline__ int64_t keys_of(const P& p, int64_t prefix, int64_t last) {
  return max64(0, min64(prefix + over_group(p, static_cast<uint32_t>(last)) + 1, p.max_blocks << p.bs_shift));
}

// Where the partial results of row b begin, its first token being tok0.
template <typename P>
__device__ __forceinline__ int64_t part_base(const P& pp, int64_t b, int64_t tok0) { return pp.per_row != 0 ? b * pp.per_row : tok0; }

// Parts that `tiles` tiles are split into, the same in both launches: the tables may be much wider than the row.
template <typename P>
__device__ __forceinline__ int parts_of(const P& pp, int64_t tiles) {
  const float best = __builtin_sqrtf(pp.per_tile * static_cast<float>(tiles));
  return max(1, min(min(pp.splits, static_cast<int>(best)), static_cast<int>(min64(tiles, kMaxSplits))));
}

// The launch's parameters, read again: what only the start, the end or every sixteenth tile needs does not stay in scalar
// registers over the loop, which else spilled 46 of them to vector lanes and read them back each tile.
typedef const __attribute__((address_space(4))) PrefillParams* ParamsAgain;
__device__ __forceinline__ ParamsAgain params_again() {
  ParamsAgain p = (ParamsAgain)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

constexpr int kJoinAhead = 8;  // parts asked for at a time

// Joins the parts of one (token, head): a wave each, lane l dims l D/64 ..
template <int D, int COLS>
__global__ __launch_bounds__(256) void join_kernel(PrefillParams pp) {
  const Params& p = pp.c;
  constexpr int E = D / 64;
  typedef float vec_t __attribute__((ext_vector_type(E)));
  const int lane = threadIdx.x & 63;
  const int64_t x = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.y;
  const int64_t tok0 = read_index(p.cu, p.idx_i64, b);
  const int64_t n_new = min64(pp.max_new, min64(read_index(p.cu, p.idx_i64, b + 1), p.total) - tok0);
  if (tok0 < 0 || x >= n_new * p.H) return;
  const uint32_t n = static_cast<uint32_t>(x) / static_cast<uint32_t>(p.H), h = static_cast<uint32_t>(x) - n * static_cast<uint32_t>(p.H);
  // the workgroups that had this column
  const int64_t column = static_cast<int64_t>(n) * p.G + (h - over_group(p, h) * static_cast<uint32_t>(p.G));
  const int64_t last = min64(n_new * p.G, column / COLS * COLS + COLS) - 1;
  const int parts = parts_of(pp, (keys_of(p, read_index(p.prefix, p.idx_i64, b), last) + kTile - 1) / kTile);
  if (parts == 1) return;  // written by the workgroup itself
  const int64_t row = part_base(pp, b, tok0) * p.H + x;
  const int64_t stride = pp.part_tokens * p.H;
  const float2 ml = lane < parts ? *reinterpret_cast<const float2*>(pp.part_ml + (lane * stride + row) * 2) : make_float2(-INFINITY, 0.f);
  const float m = wave_max(ml.x);
  const float f = __builtin_amdgcn_exp2f(ml.x - (m == -INFINITY ? 0.f : m));
  const float l = wave_sum(f * ml.y);
  vec_t acc = vec_t(0.f);
  for (int s0 = 0; s0 < parts; s0 += kJoinAhead) {
    vec_t part[kJoinAhead];
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i)  // past the end: the last part again
      part[i] = *reinterpret_cast<const vec_t*>(pp.part_o + (min(s0 + i, parts - 1) * stride + row) * D + E * lane);
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i) {
      const float fs = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), min(s0 + i, parts - 1)));
      if (s0 + i < parts) acc += fs * part[i];
    }
  }
  typedef uint32_t packed_t __attribute__((ext_vector_type(E / 2)));
  packed_t gate = packed_t(0u), out;
  if (p.gate != nullptr) gate = *reinterpret_cast<const packed_t*>(p.gate + (tok0 + n) * p.gate_st + h * p.gate_sh + E * lane);
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    float lo = normalised(acc[e], l), hi = normalised(acc[e + 1], l);
    if (p.gate != nullptr) {
      lo *= sigmoid(__uint_as_float(gate[e / 2] << 16));
      hi *= sigmoid(__uint_as_float(gate[e / 2] & 0xffff0000u));
    }
    out[e / 2] = static_cast<uint32_t>(f32_to_bf16(lo)) | static_cast<uint32_t>(f32_to_bf16(hi)) << 16;
  }
  *reinterpret_cast<packed_t*>(p.out + (tok0 * p.H + x) * D + E * lane) = out;
}

// Parts the keys are split into where the workgroups leave CUs free.  A part saves a share of 1.5 us a tile and costs its
// piece of the partial results, in time like parts times workgroups, which puts the best number at a root; the 30 is from
// us with 1, 2, 4, 8, 16 parts, D = 256, one row: 16 tokens (2 workgroups) over 32 tiles 65.6 41.9 29.2 23.3 22.1, 128 tokens
// (16) over 17 tiles 42.3 31.9 27.7 30.8 35.4, 512 tokens (64) over 8 tiles 28.6 33.6 35.4 51.4 64.5, over 32 tiles 67.2
// 52.8 45.3 64.9 105.
// A workgroup of fewer columns has that much less of both, and more of them fit the chip.
static double per_tile_of(int cols) { return 30.0 * 128 / cols; }
static int slots_of(int cols) { return 256 * 128 / cols; }

static int64_t workgroups_of(int64_t batch, int kv_heads, int group, int64_t max_new, int cols) {
  return batch * kv_heads * ceil_div(max_new * group, cols);
}

// What the launch has room for, from the longest row that the tables hold; each row's own number is parts_of its tiles.
static int splits_of(int64_t batch, int kv_heads, int group, int64_t max_new, int64_t max_tokens, int cols) {
  const int64_t wgs = workgroups_of(batch, kv_heads, group, max_new, cols);
  const int64_t tiles = ceil_div(std::max<int64_t>(max_tokens, 1), kTile);
  if (wgs >= slots_of(cols)) return 1;
  const int64_t best = static_cast<int64_t>(std::sqrt(per_tile_of(cols) * static_cast<double>(tiles) / static_cast<double>(wgs)));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({kMaxSplits, slots_of(cols) / wgs, tiles, best})));
}

// Tokens that partial results are kept of: a query padded past its rows' bound is no reason for more.  With splits of at most
// 256 / workgroups of 128 columns they are below 35 MB at any padding and any width of the tables.
static int64_t part_tokens_of(int64_t total, int64_t batch, int64_t max_new) { return std::min(total, batch * max_new); }

static int64_t workspace_of(int splits, int64_t part_tokens, int heads, int head_dim) {
  return splits > 1 ? splits * part_tokens * heads * (static_cast<int64_t>(head_dim) + 2) * 4 : 0;
}

template <int D, int COLS>
static int join(const PrefillParams& p, const char* what, const char* label, hipStream_t stream) {
  if (p.splits > 1) {
    KernelTimer timer_(label, stream);
    const dim3 jgrid(static_cast<unsigned>(ceil_div(p.max_new * p.c.H, 4)), static_cast<unsigned>(p.c.B));
    hipLaunchKernelGGL((join_kernel<D, COLS>), jgrid, dim3(256), 0, stream, p);
  }
  return check_launch(what);
}

// The launch's parts and workspace; p.max_new stays 0 where there is nothing to compute.
static int share_out(PrefillParams& p, const Args& a, const void* cu_seqlens, const void* prefix_lens, int64_t max_new, void* workspace, int64_t workspace_bytes, int cols) {
  QA_REQUIRE(a.q_rows >= 0 && a.q_rows <= 0x7fffffff && max_new >= 0 && max_new <= 0x7fffffff, "%s: token counts out of range", a.what);
  if (a.batch == 0 || max_new == 0 || a.q_rows == 0) return 0;
  QA_REQUIRE(cu_seqlens && prefix_lens, "%s: pointers must be non-null", a.what);
  QA_REQUIRE(a.batch * a.kv->kv_heads <= 65535, "%s: batch * KV heads must fit 65535", a.what);
  max_new = std::min(max_new, a.q_rows);
  QA_REQUIRE(max_new * a.heads <= 0x7fffffff, "%s: max_new * a.heads out of range", a.what);
  p.c.cu = cu_seqlens;
  p.c.prefix = prefix_lens;
  p.c.total = a.q_rows;
  p.max_new = max_new;
  p.splits = splits_of(a.batch, a.kv->kv_heads, p.c.G, max_new, a.max_blocks * a.block_size, cols);
  p.per_tile = static_cast<float>(per_tile_of(cols) / static_cast<double>(workgroups_of(a.batch, a.kv->kv_heads, p.c.G, max_new, cols)));
  p.part_tokens = part_tokens_of(a.q_rows, a.batch, max_new);
  p.per_row = p.part_tokens < a.q_rows ? max_new : 0;
  const int64_t need = workspace_of(p.splits, p.part_tokens, a.heads, a.head_dim);
  QA_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0),
             "paged prefill workspace too small or not 16-byte aligned: need %lld bytes, have %lld", static_cast<long long>(need), static_cast<long long>(workspace_bytes));
  p.part_o = reinterpret_cast<float*>(workspace);
  p.part_ml = p.part_o + static_cast<int64_t>(p.splits) * p.part_tokens * a.heads * a.head_dim;
  return 0;
}

static int64_t workspace_bytes_of(int64_t total_new, int64_t batch, int64_t max_new, int heads, int kv_heads, int head_dim, int64_t max_tokens, int cols) {
  if (total_new <= 0 || batch <= 0 || max_new <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || head_dim <= 0 || max_tokens < 0) return 0;
  max_new = std::min(max_new, total_new);
  return workspace_of(splits_of(batch, kv_heads, heads / kv_heads, max_new, max_tokens, cols), part_tokens_of(total_new, batch, max_new), heads, head_dim);
}

}  // namespace
}  // namespace attn
}  // namespace qa
