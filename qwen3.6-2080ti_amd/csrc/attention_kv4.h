// What decode and prefill over the 4-bit paged KV cache (kv4.h) share beside attention_paged.h: the wave-level
// products of a run of 16 keys or of 32 values.
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

#include "attention_paged.h"
#include "kv4.h"

namespace qa {
namespace attn4 {

using namespace attn;

typedef int int8_v __attribute__((ext_vector_type(8)));

// A run of keys in registers: lane 16 q + t holds token t, dims 32 q .. 32 q + 31 of each slice of 128.
template <int D>
struct KeyRun {
  uint4 code[D / 128];
  uint32_t scale;  // byte i: slice i
};

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

inline int fill(Params& p, const Args& a) {
  if (int rc = kv4::check_pool(a.what, a.kv, a.head_dim, a.block_size)) return rc;
  return fill_params(p, a);
}

}  // namespace attn4
}  // namespace qa
