// What decode and prefill over the 4-bit paged KV cache (kv4.h) share: parameters, host checks, and the wave-level
// products of a run of 16 keys or of 32 values.
//
//   out[n][h] = softmax_t(scale q[n][h] . k[t][g]) v[t][g]  (* sigmoid(gate[n][h])),  g = h / (H / H_kv),
// over the cached tokens t that the query sees: t < length of its row (decode), t <= its own position (prefill).
// Tokens of blocks outside the pool are skipped; a query that sees nothing gives zeros.
//
// Scores.  v_mfma_scale_f32_16x16x128_f8f6f4 takes the keys' codes and scale bytes as they are (A: 16 tokens, 128 dims)
// and the query in fp8 (B: 16 columns).  A bf16 query has 8 significant bits and E4M3 4, so the query goes in as two
// pieces, hi = E4M3(x) and lo = E4M3(16 (x - hi)) with a scale 2^-4 below, and the products cost what two bf16 products of
// half the depth would, without unpacking a key.
// The instruction adds groups of eight dims in fixed point (measured): each product is cut, toward zero, 13 bits below
// the largest exponent of the eight, an exponent being the sum of the factors' own; the groups and the accumulator are
// then added in fp32.  So hi is first rounded to 2^-10 of the power of two at the largest element of its eight dims:
// its products are then whole units (a code's are halves, at most 6) and lose nothing, and what the cut takes of the
// lo products is below 2^-15 of that power times the key's scale.  hi + lo is x down to 2^-7 of the largest of the eight,
// and below within 2^-15 of it (or 2^-21 of the row's largest, where that is more).  Without the grid a score lost up to
// 2^-11 of its eight dims' largest product: 256 dims of normal numbers 7e-5 (root mean square) in place of 1e-5, with
// one element 300 times the others 1e-2 and 9e-4.
// Values.  v_cvt_scalef32_pk_bf16_fp4 turns a byte into two bf16 with the token's scale applied, exactly (their scales
// differ from token to token, so the reduction over tokens cannot take them as the product's block scales); v_perm pairs
// the tokens; the layout of kv4.h has a lane load the operand's own dims, so nothing goes through LDS.  The probabilities
// are rounded to bf16 for that product (2^-8 of each at most), as in the attention over bf16 pools: the bf16 instruction
// is the fastest that takes values of 4 bits and a scale a token exactly, and the rounding of many tokens averages out.
// The denominators sum the probabilities before it.  A result's error against 64 bits is then 2.0e-3 to 2.3e-3 of it (root
// mean square), 1.7e-3 being its own rounding to bf16.
#pragma once

#include "kv4.h"

#include <atomic>

namespace qa {
namespace attn4 {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8_v;
typedef int int8_v __attribute__((ext_vector_type(8)));
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

// A run of keys in registers: lane 16 q + t holds token t, dims 32 q .. 32 q + 31 of each slice of 128.
template <int D>
struct KeyRun {
  uint4 code[D / 128];
  uint32_t scale;  // byte i: slice i
};

// Cache policy of a load: kOnce (non-temporal) for tiles that one workgroup reads once (decode of 64 rows of 1k to 32k
// tokens 97 us, 110 without).
constexpr int kShared = 0, kOnce = 2;

template <int D, int POLICY>
__device__ __forceinline__ void load_keys(KeyRun<D>& k, __amdgpu_buffer_rsrc_t r, int lane) {
#pragma unroll
  for (int i = 0; i < D / 128; ++i) k.code[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, 16 * lane + 1024 * i, 0, POLICY));
  if constexpr (D == 256)
    k.scale = __builtin_amdgcn_raw_buffer_load_b16(r, kv4::Run<D>::kCodes + 2 * lane, 0, POLICY);
  else
    k.scale = __builtin_amdgcn_raw_buffer_load_b8(r, kv4::Run<D>::kCodes + lane, 0, POLICY);
}

// A run of values: lane 16 q + c holds tokens 4 q .. 4 q + 3, dims c D/16 ..
template <int D>
struct ValueRun {
  uint4 code[D / 128];
  uint32_t scale;  // byte r: token 4 q + r
};

template <int D, int POLICY>
__device__ __forceinline__ void load_values(ValueRun<D>& v, __amdgpu_buffer_rsrc_t r, int lane) {
#pragma unroll
  for (int i = 0; i < D / 128; ++i) v.code[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, 16 * lane + 1024 * i, 0, POLICY));
  const int group = (lane & 15) / (512 / D);
  v.scale = __builtin_amdgcn_raw_buffer_load_b32(r, kv4::Run<D>::kCodes + 16 * group + 4 * (lane >> 4), 0, POLICY);
}

// The query columns of a wave in fp8.  Byte order of the B operand: lane 16 q + n holds of column n and each slice of
// 128 dims 16 q .. 16 q + 15, then 64 + 16 q .. 64 + 16 q + 15; its scale byte belongs to dims 32 q .. 32 q + 31.  One
// scale serves the whole row.
template <int D>
struct QueryCols {
  int8_v code[D / 128];
  uint32_t scale;
};

// The scale byte of a row's hi piece: the row's largest element, of bits top, lands in [128, 256), the lo piece's scale is
// 2^-4 of it.  A row with an infinity or a NaN becomes NaN.
__device__ __forceinline__ uint32_t query_scale(uint32_t top) { return static_cast<uint32_t>(min(max(static_cast<int>(top >> 23) - 7, 5), 247)); }

// x + g - g is x on the grid of hi: top is the bits of the largest magnitude of the eight, times inv.  It may round up to the
// next power of two in E4M3, whose exponent then counts.
__device__ __forceinline__ float piece_grid(uint32_t top, float inv) {
  const uint32_t power = (__float_as_uint(__uint_as_float(top) * inv) + 0x80000u) >> 23;
  return __uint_as_float((power + 13u) << 23 | 0x400000u);  // 3 2^12 of it: its last place is 2^-10 of it
}

// Loads row qrow (null: zeros) of this lane's column and splits it.  LO: the second piece.  Both need the same row.
template <int D>
struct QueryRow {
  uint4 raw[D / 128][4];
  float x[D / 128][32];
  float grid[D / 128][4];  // of eight dims
  uint32_t byte;  // scale of hi

  __device__ __forceinline__ void ask(const bf16_t* qrow, int quad) {
#pragma unroll
    for (int i = 0; i < D / 128; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        raw[i][j] = make_uint4(0, 0, 0, 0);
        if (qrow != nullptr) raw[i][j] = *reinterpret_cast<const uint4*>(qrow + 128 * i + 64 * (j >> 1) + 16 * quad + 8 * (j & 1));
      }
  }

  __device__ __forceinline__ void widen() {
    uint32_t top = 0, near[D / 128][4];
#pragma unroll
    for (int i = 0; i < D / 128; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        near[i][j] = 0;
        const uint32_t w[4] = {raw[i][j].x, raw[i][j].y, raw[i][j].z, raw[i][j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[i][8 * j + 2 * e] = __uint_as_float(w[e] << 16);
          x[i][8 * j + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
          near[i][j] = max(near[i][j], max(w[e] << 16 & 0x7fffffffu, w[e] & 0x7fff0000u));
        }
        top = max(top, near[i][j]);
      }
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, 64)));
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, 64)));
    byte = query_scale(top);
    const float inv = __uint_as_float((254u - byte) << 23);
#pragma unroll
    for (int i = 0; i < D / 128; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) grid[i][j] = piece_grid(near[i][j], inv);
  }

  template <bool LO>
  __device__ __forceinline__ void split(QueryCols<D>& c) const {
    const float inv = __uint_as_float((254u - byte) << 23);
#pragma unroll
    for (int i = 0; i < D / 128; ++i)
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const float g = grid[i][w >> 1];
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = x[i][4 * w + e] * inv;
        uint32_t hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] + g - g, y[1] + g - g, 0, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] + g - g, y[3] + g - g, hi, true);
        if constexpr (LO) {
          const floatx2_v a = __builtin_amdgcn_cvt_pk_f32_fp8(hi, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(hi, true);
          hi = __builtin_amdgcn_cvt_pk_fp8_f32((y[0] - a[0]) * 16.f, (y[1] - a[1]) * 16.f, 0, false);
          hi = __builtin_amdgcn_cvt_pk_fp8_f32((y[2] - b[0]) * 16.f, (y[3] - b[1]) * 16.f, hi, true);
        }
        c.code[i][w] = static_cast<int>(hi);
      }
    c.scale = LO ? byte - 4u : byte;
  }
};

// S (16 tokens x 16 columns) += K Q: lane 16 q + n receives tokens 4 q + r of column n.
template <int D>
__device__ __forceinline__ floatx4_v score(const KeyRun<D>& k, const QueryCols<D>& q, floatx4_v acc) {
  auto operand = [](const uint4& u) { return int8_v{static_cast<int>(u.x), static_cast<int>(u.y), static_cast<int>(u.z), static_cast<int>(u.w), 0, 0, 0, 0}; };
  acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(k.code[0]), q.code[0], acc, 4, 0, 0, static_cast<int>(k.scale), 0, static_cast<int>(q.scale));
  if constexpr (D == 256)
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(k.code[1]), q.code[1], acc, 4, 0, 1, static_cast<int>(k.scale), 0, static_cast<int>(q.scale));
  return acc;
}

// The scale of token 4 q + r of a run of values as a float.
__device__ __forceinline__ float value_scale(uint32_t bytes, int r) {
  return __uint_as_float((r == 0 ? bytes << 23 : r == 1 ? bytes << 15 : r == 2 ? bytes << 7 : bytes >> 1) & 0x7f800000u);
}

// O^T += V^T P over 32 tokens (two runs): o[i] has row 4 q + r = dim (4 q + r) D/16 + i of column lane % 16.  p: the
// lane's probabilities, tokens 4 q + 0..3 of the first run, then of the second.
template <int D>
__device__ __forceinline__ void accumulate(const ValueRun<D> (&v)[2], bf16x8_v p, floatx4_v (&o)[D / 16]) {
  constexpr int W = D / 128;  // dwords of codes a token: 8 dims each
  float s[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) s[t] = value_scale(v[t >> 2].scale, t & 3);
  auto dword = [&](int t, int w) -> uint32_t {
    const ValueRun<D>& u = v[t >> 2];
    const int at = (t & 3) * W + w;  // dword of the lane's 4 W
    const uint4& c = u.code[at >> 2];
    return (at & 3) == 0 ? c.x : (at & 3) == 1 ? c.y : (at & 3) == 2 ? c.z : c.w;
  };
#pragma unroll
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      uint32_t pair[8];  // dims 8 w + 2 b and + 1 of each token
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const uint32_t c = dword(t, w);
        switch (b) {
          case 0: pair[t] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s[t], 0)); break;
          case 1: pair[t] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s[t], 1)); break;
          case 2: pair[t] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s[t], 2)); break;
          default: pair[t] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s[t], 3)); break;
        }
      }
      uint4 even, odd;
      even.x = __builtin_amdgcn_perm(pair[1], pair[0], 0x05040100u);
      even.y = __builtin_amdgcn_perm(pair[3], pair[2], 0x05040100u);
      even.z = __builtin_amdgcn_perm(pair[5], pair[4], 0x05040100u);
      even.w = __builtin_amdgcn_perm(pair[7], pair[6], 0x05040100u);
      odd.x = __builtin_amdgcn_perm(pair[1], pair[0], 0x07060302u);
      odd.y = __builtin_amdgcn_perm(pair[3], pair[2], 0x07060302u);
      odd.z = __builtin_amdgcn_perm(pair[5], pair[4], 0x07060302u);
      odd.w = __builtin_amdgcn_perm(pair[7], pair[6], 0x07060302u);
      const int i = 8 * w + 2 * b;
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_v, even), p, o[i], 0, 0, 0);
      o[i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_v, odd), p, o[i + 1], 0, 0, 0);
    }
}

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

inline int fill(Params& p, const Args& a) {
  if (int rc = kv4::check_pool(a.what, a.kv, a.head_dim, a.block_size)) return rc;
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

}  // namespace attn4
}  // namespace qa
