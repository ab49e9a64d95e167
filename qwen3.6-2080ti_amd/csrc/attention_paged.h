// What decode and prefill over a paged KV cache in runs of 16 tokens share, whatever a run holds (kv4.h, kv8.h): parameters,
// host checks, and what a wave does with scores and sums.
//
//   out[n][h] = softmax_t(scale q[n][h] . k[t][g]) v[t][g]  (* sigmoid(gate[n][h])),  g = h / (H / H_kv),
// over the cached tokens t that the query sees: t < length of its row (decode), t <= its own position (prefill).
// Tokens of blocks outside the pool are skipped; a query that sees nothing gives zeros.
#pragma once

#include "qa_common.h"

#include <atomic>

namespace qa {
namespace attn {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8_v;
typedef float floatx4_v __attribute__((ext_vector_type(4)));
typedef float floatx2_v __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
// The reference point of a row's exponentials moves only where a score is above it by more than this (log2 units), so
// the accumulators are rarely rescaled and probabilities stay below 2^8: the result is the same softmax, numerator and
// denominator share the point.
constexpr float kLazy = 8.f;

struct Params {
  const bf16_t* q;
  int64_t q_st, q_sh;
  const uint8_t* kpool;
  const uint8_t* vpool;
  int64_t num_blocks, sP, sG;
  const void* tables;
  int64_t table_stride, max_blocks;
  const void* lens;    // decode: (B)
  const void* cu;      // prefill: (B + 1)
  const void* prefix;  // prefill: (B)
  int64_t total;       // prefill: rows of query
  const bf16_t* gate;
  int64_t gate_st, gate_sh;
  bf16_t* out;
  int B, H, Hkv, G, bs_shift, table_i64, idx_i64;
  uint32_t g_mul, g_shift;  // x / G = x g_mul >> 32 >> g_shift for x below 2^31, where G > 1
  float scale;
};

// Entry i of an int32 or int64 array.  Without a branch, so that several are on their way at once.
__device__ __forceinline__ int64_t read_index(const void* base, int is64, int64_t i) {
  const int32_t* at = reinterpret_cast<const int32_t*>(base) + (i << is64);
  const int32_t lo = at[0], hi = at[is64];
  return is64 ? static_cast<int64_t>(hi) << 32 | static_cast<uint32_t>(lo) : lo;
}

__device__ __forceinline__ int64_t uniform64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(static_cast<uint64_t>(v) >> 32));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

// Physical block of a run of 16 tokens of row b, -1 where there is none.  Wave-uniform and without a branch (scalar
// loads under branches are waited for at each join): a run past the row reads a clamped entry, and an entry of either
// width is read as words.
template <typename P>  // Params, wherever they lie
__device__ __forceinline__ int32_t block_of_run(const P& p, int64_t b, int64_t run, int64_t runs) {
  typedef const __attribute__((address_space(4))) int32_t c32;
  const int64_t lb = run >> (p.bs_shift - 4);
  const int64_t at = (b * p.table_stride + max64(0, min64(lb, p.max_blocks - 1))) << p.table_i64;
  const int32_t lo = ((c32*)p.tables)[at];
  const int32_t hi = ((c32*)p.tables)[at + p.table_i64];  // the entry itself where it has one word
  const bool ok = (run < runs) & (lb < p.max_blocks) & (static_cast<uint32_t>(lo) < static_cast<uint32_t>(p.num_blocks)) & ((hi == 0) | (p.table_i64 == 0));
  return ok ? lo : -1;
}

// Cache policy of a load: kOnce (non-temporal) for tiles that one workgroup reads once (decode of 64 rows of 1k to 32k
// tokens 97 us, 110 without).
constexpr int kShared = 0, kOnce = 2;

// Max over the four quads of a column.
__device__ __forceinline__ float column_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float m = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float column_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float s = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(s), __float_as_uint(s), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// x / G, by a product with its reciprocal rounded up: with 2^s >= G the error of x ceil(2^(31 + s) / G) is below 2^(31 + s) / G.
template <typename P>  // Params, wherever they lie
__device__ __forceinline__ uint32_t over_group(const P& p, uint32_t x) { return p.G == 1 ? x : __umulhi(x, p.g_mul) >> p.g_shift; }

// o / l: zeros where a query saw nothing; a NaN stays one.
__device__ __forceinline__ float normalised(float o, float l) {
  const float r = o * (1.f / l);
  return l == 0.f ? 0.f : r;
}

// v_rcp_f32 is within an ulp and a division ten instructions: prefill of eight chunks of 512 went from 296 to 289 us.
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -kLog2e)); }

// ---- host ------------------------------------------------------------------
// Lets a kernel have `bytes` of dynamic LDS, once per device: the call costs the host about a microsecond.
template <auto KERNEL>
inline int reserve_lds(const char* what, int bytes) {
  static std::atomic<uint64_t> done{0};
  int device = 0;
  hipError_t err = hipGetDevice(&device);
  if (err != hipSuccess) return fail("%s: hipGetDevice failed: %s", what, hipGetErrorString(err));
  const uint64_t bit = uint64_t{1} << (device & 63);
  if (device < 64 && (done.load(std::memory_order_relaxed) & bit)) return 0;
  err = hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err != hipSuccess) return fail("%s: cannot reserve %d bytes of LDS: %s", what, bytes, hipGetErrorString(err));
  if (device < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return 0;
}

struct Args {
  const char* what;
  const void* query;
  int32_t q_dtype;
  int64_t q_st, q_sh;
  int64_t q_rows;
  int64_t batch;
  int32_t heads, head_dim;
  const qa_paged_kv* kv;
  const void* tables;
  int32_t table_dtype;
  int64_t table_stride, max_blocks;
  int32_t idx_dtype, block_size;
  float scale;
  const void* gate;
  int64_t gate_st, gate_sh;
  void* out;
};

// Checks the arguments and fills the parameters; the pool has been checked (check_pool of its format).
inline int fill_params(Params& p, const Args& a) {
  QA_REQUIRE(a.q_dtype == QA_BF16, "%s: query must be bfloat16", a.what);
  QA_REQUIRE(is_index_dtype(a.table_dtype) && is_index_dtype(a.idx_dtype), "%s: index arrays must be int32/int64", a.what);
  QA_REQUIRE(a.batch >= 0 && a.batch <= 0x7fffffff, "%s: batch out of range", a.what);
  QA_REQUIRE(a.heads > 0 && a.heads % a.kv->kv_heads == 0, "%s: query heads (%d) must be a multiple of KV heads (%d)", a.what, a.heads, a.kv->kv_heads);
  QA_REQUIRE(a.heads / a.kv->kv_heads <= 16, "%s: GQA group size %d is larger than 16", a.what, a.heads / a.kv->kv_heads);
  QA_REQUIRE(a.max_blocks > 0 && a.max_blocks <= 0x7fffffff && a.table_stride >= 0, "%s: block table must have at least one entry", a.what);
  if (a.batch > 0 && a.q_rows > 0) QA_REQUIRE(a.query && a.out && a.tables, "%s: pointers must be non-null", a.what);
  QA_REQUIRE(((reinterpret_cast<uintptr_t>(a.query) | reinterpret_cast<uintptr_t>(a.out)) & 15u) == 0 && a.q_st % 8 == 0 && a.q_sh % 8 == 0,
             "%s: query rows must be 16-byte aligned", a.what);
  QA_REQUIRE(a.gate == nullptr || ((reinterpret_cast<uintptr_t>(a.gate) & 7u) == 0 && a.gate_st % 4 == 0 && a.gate_sh % 4 == 0), "%s: gate rows must be 8-byte aligned", a.what);
  QA_REQUIRE(((a.q_st | a.q_sh | a.gate_st | a.gate_sh) & ~0xffffffffll) == 0, "%s: query and gate strides must be in [0, 2^32)", a.what);
  p.q = reinterpret_cast<const bf16_t*>(a.query);
  p.q_st = a.q_st;
  p.q_sh = a.q_sh;
  p.kpool = reinterpret_cast<const uint8_t*>(a.kv->key);
  p.vpool = reinterpret_cast<const uint8_t*>(a.kv->value);
  p.num_blocks = a.kv->num_blocks;
  p.sP = a.kv->stride_block;
  p.sG = a.kv->stride_head;
  p.tables = a.tables;
  p.table_stride = a.table_stride;
  p.max_blocks = a.max_blocks;
  p.gate = reinterpret_cast<const bf16_t*>(a.gate);
  p.gate_st = a.gate_st;
  p.gate_sh = a.gate_sh;
  p.out = reinterpret_cast<bf16_t*>(a.out);
  p.B = static_cast<int>(a.batch);
  p.H = a.heads;
  p.Hkv = a.kv->kv_heads;
  p.G = a.heads / a.kv->kv_heads;
  p.g_shift = 0;
  while ((2 << p.g_shift) < p.G) ++p.g_shift;  // ceil(log2 G) - 1
  p.g_mul = static_cast<uint32_t>(((1ull << (32 + p.g_shift)) + p.G - 1) / p.G);
  p.bs_shift = __builtin_ctz(static_cast<unsigned>(a.block_size));
  p.table_i64 = a.table_dtype == QA_I64;
  p.idx_i64 = a.idx_dtype == QA_I64;
  p.scale = a.scale > 0.f ? a.scale : 1.0f / sqrtf(static_cast<float>(a.head_dim));
  return 0;
}

}  // namespace attn
}  // namespace qa
