// What decode and prefill over the 8-bit paged KV cache (kv8.h) share beside attention_paged.h.
//
// Both multiply in bf16: a code times its run's scale is exact there, v_cvt_scalef32_pk_bf16_fp8 makes two of them an
// instruction, and a bf16 query goes in as it is, so that scores are as over a bf16 cache of the same values.  (The fp8
// product would take the codes as they are, but the query only in two pieces of four bits each: the same time on the matrix
// cores, and the instruction cuts small products beside large ones.)
#pragma once

#include "attention_paged.h"
#include "kv8.h"

namespace qa {
namespace attn8 {

using namespace attn;

// Eight codes times the scale: an operand of a bf16 product.
__device__ __forceinline__ bf16x8_v operand(uint32_t lo, uint32_t hi, float scale_lo, float scale_hi) {
  return __builtin_bit_cast(bf16x8_v, make_uint4(kv8::widen<false>(lo, scale_lo), kv8::widen<true>(lo, scale_lo), kv8::widen<false>(hi, scale_hi), kv8::widen<true>(hi, scale_hi)));
}

__device__ __forceinline__ uint32_t dword(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

// The bytes of tokens 0 .. n - 1 of the four in a dword of values.
__device__ __forceinline__ uint32_t tokens_mask(int64_t n) { return n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * static_cast<int>(n))) - 1u; }

inline int fill(Params& p, const Args& a) {
  if (int rc = kv8::check_pool(a.what, a.kv, a.head_dim, a.block_size)) return rc;
  return fill_params(p, a);
}

}  // namespace attn8
}  // namespace qa
