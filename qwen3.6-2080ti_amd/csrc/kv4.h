// The 4-bit paged KV cache: its layout, and the device code that writes a group.
//
// A group is 32 consecutive dims of one token and KV head, held as a scale 2^e (the byte e + 127) and 32 E2M1 codes
// (sign; 0 0.5 1 1.5 2 3 4 6).  e is the least integer with max|x| <= 7 2^e: then no element is further from its code
// than half the spacing of E2M1 at it (7 is the far end of what rounds to 6), which floor(log2 max) would not hold for
// maxima above 7/4 of a power of two.  e is clamped to [-125, 125]: every value is then a normal bfloat16, and 6 2^125
// is finite.  Both the scale and a code times it are exact in bfloat16, so reading the cache rounds nothing.
// A group with an infinity or a NaN gets the byte 255 and reads as NaN.
//
// A pool block of one head ("tile") is block_size / 16 runs of 16 tokens, each 17 D / 2 bytes: codes, then scales.
//   keys    codes [group D/32][token][16 bytes], scales [group % 4][token][group / 4]: the order in which the lanes of
//           v_mfma_scale_f32_16x16x128_f8f6f4 hold an operand of 16 rows (lane 16 q + t: row t, dims 32 q .. 32 q + 31 of
//           a slice of 128), so a wave reads 1 KB of consecutive bytes per slice and multiplies them as they are
//   values  codes [pair][token / 4][lane chunk c][token within the pair][D/32 bytes], a pair being 512 / D of the four
//           tokens 4 q + r, a chunk the dims c D/16 .. (c + 1) D/16 - 1; scales [group][token].  Lane 16 q + c of a wave
//           then reads 16-byte pieces that hold the four tokens of its quad, as the A operand of V^T P wants them: no
//           transpose through LDS.
#pragma once

#include "qa_common.h"

namespace qa {
namespace kv4 {

constexpr int kRun = 16;  // tokens of a run

template <int D>
struct Run {
  static constexpr int kCodes = 8 * D;  // bytes
  static constexpr int kGroups = D / 32;
  static constexpr int kBytes = kCodes + kRun * kGroups;
  static constexpr int kPair = 512 / D;       // tokens of a 16-byte piece of values
  static constexpr int kChunk = D / 32;       // bytes of a value chunk of one token
  static_assert(D == 128 || D == 256, "head_dim 128 or 256");

  __device__ static constexpr int key_code(int t, int group) { return (group * kRun + t) * 16; }
  __device__ static constexpr int key_scale(int t, int group) { return kCodes + ((group & 3) * kRun + t) * (D / 128) + (group >> 2); }
  __device__ static constexpr int value_code(int t, int chunk) {
    return ((((t & 3) / kPair * 4 + (t >> 2)) * 16 + chunk) * kPair + (t & 3) % kPair) * kChunk;
  }
  __device__ static constexpr int value_scale(int t, int group) { return kCodes + group * kRun + t; }
};

// The scale byte of a group whose largest magnitude is amax (not negative).  The exponent field of a float with 2^21 - 1
// added below it is one more exactly where the mantissa is above 1.75, that is amax above 7 2^(floor(log2 amax) - 2).
__device__ __forceinline__ uint32_t scale_byte(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  if (bits >= 0x7f800000u) return 255u;
  const int e = static_cast<int>((bits + 0x1fffffu) >> 23) - 2;  // biased by 127, as the byte
  return static_cast<uint32_t>(min(max(e, 2), 252));
}

// Eight codes of x / 2^(byte - 127), the first in the low half of the lowest byte.  v_cvt_scalef32_pk_fp4_f32 rounds to
// nearest, ties to the even code, and saturates.  A group that is not finite has codes of 0.
__device__ __forceinline__ uint32_t pack_codes(const float (&x)[8], uint32_t byte) {
  const float s = __uint_as_float(byte << 23);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[0], x[1], s, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[2], x[3], s, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[4], x[5], s, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[6], x[7], s, 3);
  return byte == 255u ? 0u : r;
}

// Host: what every entry point asks of a 4-bit pool.
inline int check_pool(const char* what, const qa_paged_kv* kv, int32_t head_dim, int32_t block_size) {
  QA_REQUIRE(kv != nullptr && kv->key != nullptr && kv->value != nullptr && kv->row_key_ptrs == nullptr, "%s: needs one shared pool", what);
  QA_REQUIRE(kv->dtype == QA_KV4, "%s: the pool must be a 4-bit pool (uint8)", what);
  QA_REQUIRE(head_dim == 128 || head_dim == 256, "%s: head_dim must be 128 or 256 (got %d)", what, head_dim);
  QA_REQUIRE(block_size >= kRun && (block_size & (block_size - 1)) == 0 && block_size <= 1024, "%s: block_size must be a power of two from 16 to 1024 (got %d)", what, block_size);
  QA_REQUIRE(kv->kv_heads > 0 && kv->num_blocks >= 0 && kv->num_blocks <= 0x7fffffff, "%s: kv_heads must be positive and the blocks fit int32", what);
  const int64_t tile = static_cast<int64_t>(block_size) * 17 * head_dim / 32;
  QA_REQUIRE(kv->stride_head >= tile && kv->stride_block >= tile, "%s: pool strides are smaller than a tile of %lld bytes", what, static_cast<long long>(tile));
  QA_REQUIRE(((reinterpret_cast<uintptr_t>(kv->key) | reinterpret_cast<uintptr_t>(kv->value)) & 15u) == 0 && kv->stride_head % 16 == 0 && kv->stride_block % 16 == 0,
             "%s: pool tiles must be 16-byte aligned", what);
  return 0;
}

}  // namespace kv4
}  // namespace qa
