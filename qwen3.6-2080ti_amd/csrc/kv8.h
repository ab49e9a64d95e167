// The 8-bit paged KV cache: its layout and numbers.
//
// A run is 16 consecutive tokens of a block and one KV head, held as 16 D E4M3 codes and one scale 2^e (the byte e + 127).
// Of the finite values that a call writes to the run, e is the least integer with max|x| <= 448 2^e, 448 being the largest
// code; e is clamped to [-117, 120], so that a code times the scale is a normal bfloat16 or zero down to the least code, and
// 448 2^120 is above the largest float; at that scale 256, which would be 2^128, is held as 240.  A power of two costs no precision: a code has four significant bits wherever it lies
// between 2^-6 and 448, fifteen powers of two.  So reading the cache rounds nothing, and a run whose scale grows (a call that
// does not write its first token and brings larger values) keeps its codes' values but for those that become subnormal.
// An infinity or a NaN is held as a NaN, by itself: it has no part in the scale.
//
// A pool block of one head ("tile") is block_size / 16 runs of 16 D + 16 bytes: codes, then the scale byte and zeros.
//   keys    [slice of 64 dims][16 dims of it][token][16 bytes]: a wave reads 1 KB of consecutive bytes a slice, a lane 16 dims of
//           one token, which are two operands of a bf16 product once converted
//   values  [slice of 64 dims][token / 4][four dims c of it][dim % 4][token % 4]: a lane's 16 bytes are the four tokens of its
//           quad at four dims, as the A operand of V^T P wants them: no transpose
#pragma once

#include "qa_common.h"

namespace qa {
namespace kv8 {

constexpr int kRun = 16;  // tokens of a run
constexpr uint32_t kLeast = 10, kMost = 247;  // scale bytes

template <int D>
struct Run {
  static constexpr int kSlices = D / 64;
  static constexpr int kCodes = kRun * D;  // bytes
  static constexpr int kBytes = kCodes + 16;
  static_assert(D == 128 || D == 256, "head_dim 128 or 256");
};

// The scale byte for a largest magnitude (finite).  The exponent field of a float with 2^21 - 1 added below it is one more
// exactly where the mantissa is above 1.75, that is the magnitude above 448 2^(floor(log2) - 8).
__device__ __forceinline__ uint32_t scale_byte(uint32_t bits) {
  const int e = static_cast<int>((bits + 0x1fffffu) >> 23) - 8;  // biased by 127, as the byte
  return static_cast<uint32_t>(min(max(e, static_cast<int>(kLeast)), static_cast<int>(kMost)));
}

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float over_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }  // byte in [kLeast, kMost]

// Two codes times the scale, as bf16, exact.
template <bool HIGH>
__device__ __forceinline__ uint32_t widen(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH));
}

// Host: what every entry point asks of an 8-bit pool.
inline int check_pool(const char* what, const qa_paged_kv* kv, int32_t head_dim, int32_t block_size) {
  QA_REQUIRE(kv != nullptr && kv->key != nullptr && kv->value != nullptr && kv->row_key_ptrs == nullptr, "%s: needs one shared pool", what);
  QA_REQUIRE(kv->dtype == QA_KV8, "%s: the pool must be an 8-bit pool (float8_e4m3fn)", what);
  QA_REQUIRE(head_dim == 128 || head_dim == 256, "%s: head_dim must be 128 or 256 (got %d)", what, head_dim);
  QA_REQUIRE(block_size >= kRun && (block_size & (block_size - 1)) == 0 && block_size <= 1024, "%s: block_size must be a power of two from 16 to 1024 (got %d)", what, block_size);
  QA_REQUIRE(kv->kv_heads > 0 && kv->num_blocks >= 0 && kv->num_blocks <= 0x7fffffff, "%s: kv_heads must be positive and the blocks fit int32", what);
  const int64_t tile = static_cast<int64_t>(block_size) * (head_dim + 1);
  QA_REQUIRE(kv->stride_head >= tile && kv->stride_block >= tile, "%s: pool strides are smaller than a tile of %lld bytes", what, static_cast<long long>(tile));
  QA_REQUIRE(((reinterpret_cast<uintptr_t>(kv->key) | reinterpret_cast<uintptr_t>(kv->value)) & 15u) == 0 && kv->stride_head % 16 == 0 && kv->stride_block % 16 == 0,
             "%s: pool tiles must be 16-byte aligned", what);
  return 0;
}

}  // namespace kv8
}  // namespace qa
