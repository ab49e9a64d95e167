// The split of a decode over a paged cache in runs of 16 tokens, whatever a run holds: equal shares of all rows' units for the
// workgroups, and the merge of their partial results.  One copy of it for each kernel that uses it.
#pragma once

#include "attention_paged.h"

#include <algorithm>

namespace qa {
namespace attn {
namespace {

struct DecodeParams {
  Params c;
  int n_wgs;
  int short_rows;     // the tables hold no row that is split: no partials, no workspace
  float* part_o;      // (n_wgs + B Hkv, G, D)
  float* part_ml;     // (n_wgs + B Hkv, G, 2)
  int32_t* rg_wgs;    // (B Hkv, 2): first and last workgroup of a row group; -1: the result is written
};

constexpr int kWaves = 8;
constexpr int kUnit = 32;  // tokens
constexpr int kMaxWgs = 256;  // one per CU: eight waves of up to 256 registers fill it


// Tokens and units of row b (0 for rows of length <= 0); lengths past the table stop at it.
__device__ __forceinline__ int64_t row_tokens(const Params& p, int b) {
  const int64_t len = p.idx_i64 ? reinterpret_cast<const int64_t*>(p.lens)[b] : reinterpret_cast<const int32_t*>(p.lens)[b];
  return max64(0, min64(len, p.max_blocks << p.bs_shift));
}
__device__ __forceinline__ int units_of(int64_t tokens) { return static_cast<int>((tokens + kUnit - 1) / kUnit); }

// A row group: row b, KV head g, the units before it, its units.
struct Cursor {
  int b, g, cum, nu;
};

__device__ __forceinline__ void next_row_group(const Params& p, Cursor& c) {
  c.cum += c.nu;
  if (++c.g < p.Hkv) return;
  c.g = 0;
  do {
    ++c.b;
    c.nu = c.b < p.B ? __builtin_amdgcn_readfirstlane(units_of(row_tokens(p, c.b))) : 0;
  } while (c.nu == 0 && c.b < p.B);
}

// Inclusive sum over the lanes: shifts within rows of 16, then the rows' last sums passed on (DPP, no LDS).
__device__ __forceinline__ int lane_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);  // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);  // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);  // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// Merges the partials of one (row, head): slots first + rg .. last + rg.  A thread has four of a workgroup's CHUNK dims of
// every SHARE-th partial, kPartsInFlight of them on their way at once.
constexpr int kPartsInFlight = 8;
constexpr int kCombineThreads = kMaxWgs;  // a thread for each partial's m and l

template <int D, int CHUNK>
__global__ __launch_bounds__(kCombineThreads) void combine_kernel(DecodeParams dp) {
  const Params& p = dp.c;
  constexpr int ACROSS = CHUNK / 4;
  constexpr int SHARE = kCombineThreads / ACROSS;
  __shared__ float s_f[kMaxWgs];
  __shared__ float s_red[2][kCombineThreads / 64];
  __shared__ __align__(16) float s_o[SHARE][CHUNK];
  const int tid = threadIdx.x;
  const int64_t bh = blockIdx.x;
  const int b = static_cast<int>(static_cast<uint32_t>(bh) / static_cast<uint32_t>(p.H));
  const int h = static_cast<int>(bh) - b * p.H;
  const int g = static_cast<int>(over_group(p, h));
  const int hh = h - g * p.G;
  const int64_t rg = static_cast<int64_t>(b) * p.Hkv + g;
  const int first = dp.rg_wgs[2 * rg], last = dp.rg_wgs[2 * rg + 1];
  const int d0 = static_cast<int>(blockIdx.y) * CHUNK;
  bf16_t* out = p.out + bh * D + d0;
  if (row_tokens(p, b) == 0) {  // its record was never written
    if (tid < CHUNK) out[tid] = 0;
    return;
  }
  if (first < 0) return;
  const int n = last - first + 1;
  const int64_t row0 = (first + rg) * p.G + hh;
  const int share = tid / ACROSS, d = 4 * (tid % ACROSS);
  const float* po = dp.part_o + row0 * D + d0 + d;
  const int64_t so = static_cast<int64_t>(p.G) * D;
  floatx4_v part[kPartsInFlight];
  auto ask = [&](int s0) {
#pragma unroll
    for (int i = 0; i < kPartsInFlight; ++i) part[i] = *reinterpret_cast<const floatx4_v*>(po + min(s0 + i * SHARE, n - 1) * so);  // past the end: the last one again
  };
  ask(share);
  float2 ml = make_float2(-INFINITY, 0.f);
  if (tid < n) ml = *reinterpret_cast<const float2*>(dp.part_ml + (row0 + static_cast<int64_t>(tid) * p.G) * 2);
  float gate = 0.f;
  if (p.gate != nullptr && tid < CHUNK) gate = bf16_to_f32(p.gate[b * p.gate_st + h * p.gate_sh + d0 + tid]);
  const float wm = wave_max(ml.x);
  if ((tid & 63) == 0) s_red[0][tid >> 6] = wm;
  __syncthreads();
  float m = s_red[0][0];
#pragma unroll
  for (int w = 1; w < kCombineThreads / 64; ++w) m = fmaxf(m, s_red[0][w]);
  const float use = m == -INFINITY ? 0.f : m;
  const float f = tid < n ? __builtin_amdgcn_exp2f(ml.x - use) : 0.f;
  s_f[tid] = f;
  const float wl = wave_sum(tid < n ? f * ml.y : 0.f);
  if ((tid & 63) == 0) s_red[1][tid >> 6] = wl;
  __syncthreads();
  floatx4_v acc = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = share; s0 < n; s0 += kPartsInFlight * SHARE) {
    if (s0 != share) ask(s0);
#pragma unroll
    for (int i = 0; i < kPartsInFlight; ++i)
      if (s0 + i * SHARE < n) acc += s_f[s0 + i * SHARE] * part[i];
  }
  *reinterpret_cast<floatx4_v*>(&s_o[share][d]) = acc;
  __syncthreads();
  if (tid >= CHUNK) return;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < SHARE; ++i) sum += s_o[i][tid];
  float l = 0.f;
#pragma unroll
  for (int w = 0; w < kCombineThreads / 64; ++w) l += s_red[1][w];
  float r = normalised(sum, l);
  if (p.gate != nullptr) r *= sigmoid(gate);
  out[tid] = f32_to_bf16(r);
}

static int64_t decode_wgs(int64_t row_groups, int64_t max_tokens) {
  return std::min<int64_t>(kMaxWgs, std::max<int64_t>(1, ceil_div(row_groups * ceil_div(std::max<int64_t>(max_tokens, 1), kUnit), kWaves)));
}

// Rows of up to by_row_tokens are not split.
static int64_t workspace_bytes_of(int64_t batch, int heads, int kv_heads, int head_dim, int64_t max_tokens, int64_t by_row_tokens) {
  const int64_t groups = batch * kv_heads;
  if (max_tokens <= by_row_tokens) return 0;
  return (decode_wgs(groups, max_tokens) + groups) * (heads / kv_heads) * (head_dim + 2) * 4 + groups * 8;
}

template <int D>
static int merge(const DecodeParams& p, const char* what, const char* label, hipStream_t stream) {
  const unsigned rows = static_cast<unsigned>(static_cast<int64_t>(p.c.B) * p.c.H);
  // many partials a row group: more workgroups share its dims.  us of the whole call, not shared / shared: 1 row of 20000 16.9 /
  // 14.9, of 200000 30.8 / 28.0; 8 rows of 30000 31.4 / 32.0, 64 of up to 1024 25.5 / 34.3
  const bool many = p.n_wgs > 16 * static_cast<int64_t>(p.c.B) * p.c.Hkv;
  {
    KernelTimer timer_(label, stream);
    if (many)
      hipLaunchKernelGGL((combine_kernel<D, 32>), dim3(rows, D / 32), dim3(kCombineThreads), 0, stream, p);
    else
      hipLaunchKernelGGL((combine_kernel<D, D>), dim3(rows), dim3(kCombineThreads), 0, stream, p);
  }
  return check_launch(what);
}

// The launch's shares of the rows that `sequence_lengths` hold, and its workspace.
static int share_out(DecodeParams& p, const Args& a, const void* sequence_lengths, void* workspace, int64_t workspace_bytes, int64_t by_row_tokens) {
  QA_REQUIRE(sequence_lengths != nullptr, "sequence_lengths must be a device array");
  QA_REQUIRE(a.batch * a.heads <= 0x7fffffff, "%s: batch * heads out of range", a.what);
  p.c.lens = sequence_lengths;
  const int64_t groups = a.batch * a.kv->kv_heads;
  const int64_t max_tokens = a.max_blocks * a.block_size;
  QA_REQUIRE(groups * ceil_div(max_tokens, kUnit) <= 0x7fffffff, "%s: the tables cover too many tokens: %lld row groups of up to %lld", a.what, static_cast<long long>(groups),
             static_cast<long long>(max_tokens));
  const int64_t need = workspace_bytes_of(a.batch, a.heads, a.kv->kv_heads, a.head_dim, max_tokens, by_row_tokens);
  QA_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0),
             "paged decode workspace too small or not 16-byte aligned: need %lld bytes, have %lld", static_cast<long long>(need), static_cast<long long>(workspace_bytes));
  p.short_rows = max_tokens <= by_row_tokens;
  p.n_wgs = static_cast<int>(decode_wgs(groups, max_tokens));
  const int64_t rows = (p.n_wgs + groups) * p.c.G;
  p.part_o = reinterpret_cast<float*>(workspace);
  p.part_ml = p.part_o + rows * a.head_dim;
  p.rg_wgs = reinterpret_cast<int32_t*>(p.part_ml + rows * 2);
  return 0;
}

}  // namespace
}  // namespace attn
}  // namespace qa
