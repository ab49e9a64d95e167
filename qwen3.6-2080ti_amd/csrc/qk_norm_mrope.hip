// q/k RMSNorm with the (1 + w) weight, rotary embedding of several position axes, and the K/V write through a slot map
// into a bf16 or a 4-bit paged pool, in one pass over the projection outputs, gfx950.
//
// Per token n and head:  y = x rsqrt(mean(x^2) + eps) (1 + w); for j < rd / 2, with a = axis(j) the position axis of
// frequency j and theta_j = positions[a][n] base^(-2 j / rd),
//   out_j = y_j cos - y_{j + rd/2} sin,   out_{j + rd/2} = y_{j + rd/2} cos + y_j sin,   the rest of the head is y.
// Text has the same position on every axis and the result of the usual embedding; a picture's tokens have a time, a row
// and a column.  All of it in fp32 with one rounding to bf16 at the end.  The angle is exact where it matters: the
// host gives base^(-2 j / rd) / (2 pi) as a 64-bit fraction of a turn, so position times it modulo 2^64 is the
// angle modulo a whole turn, at any position (an fp32 product is off by 6e-3 rad at position 1e5), and its top bits go
// to v_sin / v_cos, which take turns (measured error 1.3e-7).
// k goes to the pool rounded to bf16; a 4-bit pool holds the 4-bit form (kv4.h) of that bf16 value, so that both pools
// and paged_kv4_append agree bit for bit.
//
// Bound by memory, 2 D (H + 2 H_kv) bytes of bf16 read and written per token, with the arithmetic close behind.  Two
// kernels.  rows_kernel gives a lane eight dims, 16-byte accesses, and a head D / 8 lanes: a wave takes 2 or 4 heads at a
// time, the norm is a sum over one or two rows of lanes, the partner comes by DPP on packed values, and weight times
// cosine is formed once a token.  It needs rd / 2 a multiple of 8 and rows on 16 bytes.  heads_kernel gives a lane D / 64
// dims and a head the whole wave, and takes what is left (head_dim 64 among it).  5003 tokens of 16 + 2 x 4 heads of 128:
// 26.5 us there, 16.5 us here (3.7 TB/s; a copy runs at 4.8); 128 tokens of 16 + 2 x 2 heads of 256: 7.3 and 5.8 us; into
// a 4-bit pool 15.6 and 5.5 us here.  Heads of 64, half the bytes: 20.8 us there.
#include <algorithm>

#include "kv4.h"

namespace qa {
namespace mrope {

struct Params {
  const bf16_t* q;
  int64_t q_st, q_sh;
  const bf16_t* k;
  int64_t k_st, k_sh;
  const bf16_t* v;
  int64_t v_st, v_sh;
  const void* qw;
  const void* kw;
  const uint64_t* freq;   // (rd / 2): base^(-2 j / rd) / (2 pi) as a fraction of 2^64
  const uint8_t* axis;    // (rd / 2): position axis of each frequency
  const void* positions;  // (axes, tokens)
  int64_t pos_stride;     // elements between axes
  float eps;
  const void* slots;
  int64_t tokens;
  void* kpool;
  void* vpool;
  int64_t num_slots, sP, sG, sT;  // bf16 pool: element strides; 4-bit pool: bytes, sT unused
  int H, Hkv, rd, axes, bs;
  int w_f32, pos_i64, slots_i64;
  bf16_t* q_out;
};

constexpr int kTasksInFlight = 8;
constexpr int kMaxAxes = 4;

__device__ __forceinline__ int64_t read_index(const void* base, int is64, int64_t i) {
  return is64 ? reinterpret_cast<const int64_t*>(base)[i] : reinterpret_cast<const int32_t*>(base)[i];
}

template <int E>
struct Raw {
  uint32_t w[(E + 1) / 2];
};

template <int E>
__device__ __forceinline__ Raw<E> load_raw(const bf16_t* src) {
  Raw<E> r;
  if constexpr (E == 4) {
    const uint2 u = *reinterpret_cast<const uint2*>(src);
    r.w[0] = u.x, r.w[1] = u.y;
  } else if constexpr (E == 2) {
    r.w[0] = *reinterpret_cast<const uint32_t*>(src);
  } else {
    r.w[0] = *src;
  }
  return r;
}

template <int E>
__device__ __forceinline__ void store_raw(bf16_t* dst, const Raw<E>& r) {
  if constexpr (E == 4)
    *reinterpret_cast<uint2*>(dst) = make_uint2(r.w[0], r.w[1]);
  else if constexpr (E == 2)
    *reinterpret_cast<uint32_t*>(dst) = r.w[0];
  else
    *dst = static_cast<bf16_t>(r.w[0]);
}

template <int E>
__device__ __forceinline__ void widen(const Raw<E>& r, float (&x)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = __uint_as_float(e & 1 ? r.w[e / 2] & 0xffff0000u : r.w[e / 2] << 16);
}

template <int E>
__device__ __forceinline__ Raw<E> narrow(const float (&x)[E]) {
  Raw<E> r;
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    r.w[e / 2] = f32_to_bf16(x[e]);
    if (e + 1 < E) r.w[e / 2] |= static_cast<uint32_t>(f32_to_bf16(x[e + 1])) << 16;
  }
  return r;
}

// Max of non-negative floats' bits over the 32 / E lanes of a group of 32 dims.
template <int E>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  v = quad_max(v);
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x141, 0xF, 0xF, false)));  // row_half_mirror
  if constexpr (E == 2) v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x140, 0xF, 0xF, false)));  // row_mirror
  return v;
}

// A head of bf16 values into a run of a 4-bit pool: lane l holds dims E l ..
template <int E, bool KEY>
__device__ __forceinline__ void store_kv4(uint8_t* run, int t, int lane, const Raw<E>& r) {
  using R = kv4::Run<64 * E>;
  float x[E];
  widen<E>(r, x);
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
  const uint32_t byte = kv4::scale_byte(__uint_as_float(group_max<E>(m)));
  const float s = __uint_as_float(byte << 23);
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], s, 0);
  if constexpr (E == 4) c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], s, 1);
  if (byte == 255u) c = 0;
  const int group = lane / (32 / E);
  const int in_group = lane % (32 / E);
  constexpr int kLanes = (64 * E / 16) / E;  // lanes of a value chunk
  const int at = KEY ? R::key_code(t, group) + in_group * (E / 2) : R::value_code(t, lane / kLanes) + lane % kLanes * (E / 2);
  if constexpr (E == 4)
    *reinterpret_cast<uint16_t*>(run + at) = static_cast<uint16_t>(c);
  else
    run[at] = static_cast<uint8_t>(c);
  if (in_group == 0) run[KEY ? R::key_scale(t, group) : R::value_scale(t, group)] = static_cast<uint8_t>(byte);
}

template <int E, bool KV4>
__global__ __launch_bounds__(256) void heads_kernel(Params p) {
  constexpr int D = 64 * E;
  const int64_t n = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j0 = E * lane;
  const int half = p.rd / 2;
  const bool rot = j0 < p.rd;
  const int jh = rot ? (j0 < half ? j0 : j0 - half) : 0;  // E consecutive frequencies: half is a multiple of E

  const int64_t slot = read_index(p.slots, p.slots_i64, n);
  int64_t pos[kMaxAxes];
#pragma unroll
  for (int a = 0; a < kMaxAxes; ++a) pos[a] = read_index(p.positions, p.pos_i64, min(a, p.axes - 1) * p.pos_stride + n);
  float wq[E], wk[E], c[E], s[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    wq[e] = 1.f + (p.w_f32 ? reinterpret_cast<const float*>(p.qw)[j0 + e] : bf16_to_f32(reinterpret_cast<const bf16_t*>(p.qw)[j0 + e]));
    wk[e] = 1.f + (p.w_f32 ? reinterpret_cast<const float*>(p.kw)[j0 + e] : bf16_to_f32(reinterpret_cast<const bf16_t*>(p.kw)[j0 + e]));
    c[e] = 1.f;
    s[e] = 0.f;
    if (rot) {
      const int a = p.axis[jh + e];
      const int64_t at = a == 0 ? pos[0] : a == 1 ? pos[1] : a == 2 ? pos[2] : pos[3];
      // 24 bits of the turn: v_sin and v_cos see it without a rounding
      const uint64_t turn = static_cast<uint64_t>(at) * p.freq[jh + e];
      const float f = static_cast<float>(static_cast<uint32_t>(turn >> 40)) * 0x1p-24f;
      c[e] = __builtin_amdgcn_cosf(f);
      s[e] = __builtin_amdgcn_sinf(f);
    }
  }
  const int partner = j0 < half ? lane + half / E : lane - half / E;
  const float sign = j0 < half ? -1.f : 1.f;
  const bool live = slot >= 0 && slot < p.num_slots;
  const int64_t block = live ? slot / p.bs : 0;
  const int at = live ? static_cast<int>(slot - block * p.bs) : 0;

  const int ntask = p.H + 2 * p.Hkv;
  auto task_src = [&](int task) -> const bf16_t* {
    if (task < p.H) return p.q + n * p.q_st + static_cast<int64_t>(task) * p.q_sh;
    if (task < p.H + p.Hkv) return p.k + n * p.k_st + static_cast<int64_t>(task - p.H) * p.k_sh;
    return p.v + n * p.v_st + static_cast<int64_t>(task - p.H - p.Hkv) * p.v_sh;
  };
  for (int pass = wave; pass < ntask; pass += 4 * kTasksInFlight) {
    Raw<E> raw[kTasksInFlight];
#pragma unroll
    for (int i = 0; i < kTasksInFlight; ++i) raw[i] = load_raw<E>(task_src(min(pass + 4 * i, ntask - 1)) + j0);  // past the end: the last row again
#pragma unroll
    for (int i = 0; i < kTasksInFlight; ++i) {
      const int task = pass + 4 * i;
      if (task >= ntask) break;
      const bool isq = task < p.H;
      const bool isk = !isq && task < p.H + p.Hkv;
      Raw<E> out = raw[i];
      if (isq || isk) {
        float x[E], o[E];
        widen<E>(raw[i], x);
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss += x[e] * x[e];
        const float rs = rsqrtf(wave_sum_dpp(ss) * (1.f / D) + p.eps);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = x[e] * rs * (isq ? wq[e] : wk[e]);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float other = __shfl(x[e], partner, 64);
          o[e] = rot ? x[e] * c[e] + sign * other * s[e] : x[e];
        }
        out = narrow<E>(o);
      }
      if (isq) {
        store_raw<E>(p.q_out + (n * p.H + task) * D + j0, out);
      } else if (live) {
        const int h = task - p.H - (isk ? 0 : p.Hkv);
        if constexpr (KV4) {
          const int64_t run = block * p.sP + h * p.sG + static_cast<int64_t>(at >> 4) * kv4::Run<D>::kBytes;
          if (isk)
            store_kv4<E, true>(reinterpret_cast<uint8_t*>(p.kpool) + run, at & 15, lane, out);
          else
            store_kv4<E, false>(reinterpret_cast<uint8_t*>(p.vpool) + run, at & 15, lane, out);
        } else {
          const int64_t off = block * p.sP + h * p.sG + at * p.sT + j0;
          store_raw<E>(reinterpret_cast<bf16_t*>(isk ? p.kpool : p.vpool) + off, out);
        }
      }
    }
  }
}

// ---- a lane eight dims ---------------------------------------------------------
constexpr int kStepsInFlight = 2;  // steps whose loads a wave issues before it works on the first; 6 are 3 to 20 % slower at 5003 tokens
// Waves to aim at: with fewer tokens than this the heads of a token are shared among waves, at the price of the angles in
// each.  us at 1, 2, 4 and 10 waves a token, D = 256: 128 tokens 10.6 7.6 6.4 5.5, 512 tokens 11.3 8.7 7.9 7.8, 1024 tokens
// 11.9 9.8 9.5 12.0, 2000 tokens 15.8 14.3 16.0 19.7, 5003 tokens 22.8 25.8 29.3 40.9.
constexpr int kWaves = 4096;

// The dword that the lane `distance` lanes on (lanes of the first half of the rotated dims) or back holds.
__device__ __forceinline__ uint32_t partner_of(uint32_t x, int distance, bool first, int lane) {
  const int v = static_cast<int>(x);
  if (distance == 8) return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, v, 0x128, 0xF, 0xF, false));  // row_ror:8
  if (distance == 4) {
    const int up = __builtin_amdgcn_update_dpp(0, v, 0x104, 0xF, 0xF, false);    // row_shl:4
    const int down = __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);  // row_shr:4
    return static_cast<uint32_t>(first ? up : down);
  }
  return static_cast<uint32_t>(__shfl(v, first ? lane + distance : lane - distance, 64));
}

__device__ __forceinline__ void widen8(const uint4& u, float (&x)[8]) {
  const uint32_t d[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(e & 1 ? d[e / 2] & 0xffff0000u : d[e / 2] << 16);
}

__device__ __forceinline__ void load_weights(const void* base, int f32, int j, float (&w)[8]) {
  if (f32) {
    const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + j);
    const float4 b = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + j + 4);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
  } else {
    widen8(*reinterpret_cast<const uint4*>(reinterpret_cast<const bf16_t*>(base) + j), w);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] += 1.f;
}

template <int D, bool KV4>
__global__ __launch_bounds__(256) void rows_kernel(Params p, int waves_per_token) {
  constexpr int LANES = D / 8;       // of a head
  constexpr int SLOTS = 64 / LANES;  // heads of a step
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t all = static_cast<uint32_t>(blockIdx.x) * 4u + static_cast<uint32_t>(wave);
  const int64_t n = all / static_cast<uint32_t>(waves_per_token);
  const int part = static_cast<int>(all - static_cast<uint32_t>(n) * static_cast<uint32_t>(waves_per_token));
  if (n >= p.tokens) return;
  const int in_head = lane % LANES;
  const int sub = lane / LANES;
  const int j0 = 8 * in_head;
  const int half = p.rd / 2;
  const bool rot = j0 < p.rd;
  const bool first = j0 < half;
  const int jh = rot ? (first ? j0 : j0 - half) : 0;

  // steps of one kind each, so that no lane chooses between kinds: the queries' heads, then the keys', then the values'
  const int nq = (p.H + SLOTS - 1) / SLOTS, nk = (p.Hkv + SLOTS - 1) / SLOTS;
  const int steps = nq + 2 * nk;
  auto source = [&](int step) -> const bf16_t* {  // lanes past the last head read it again
    if (step < nq) return p.q + n * p.q_st + static_cast<int64_t>(min(step * SLOTS + sub, p.H - 1)) * p.q_sh;
    if (step < nq + nk) return p.k + n * p.k_st + static_cast<int64_t>(min((step - nq) * SLOTS + sub, p.Hkv - 1)) * p.k_sh;
    return p.v + n * p.v_st + static_cast<int64_t>(min((step - nq - nk) * SLOTS + sub, p.Hkv - 1)) * p.v_sh;
  };
  uint4 raw[kStepsInFlight];
  auto load_pass = [&](int from) {
#pragma unroll
    for (int i = 0; i < kStepsInFlight; ++i) {
      if (from + i * waves_per_token < steps) raw[i] = *reinterpret_cast<const uint4*>(source(from + i * waves_per_token) + j0);
    }
  };
  load_pass(part);
  const int64_t slot = read_index(p.slots, p.slots_i64, n);

  // a lane an angle or two, then every lane its eight through LDS: eight a lane cost 0.4 us a wave more
  __shared__ __align__(16) float s_cos[4][D / 2], s_sin[4][D / 2];
  for (int j = lane; j < half; j += 64) {
    const int64_t at = read_index(p.positions, p.pos_i64, min(static_cast<int>(p.axis[j]), p.axes - 1) * p.pos_stride + n);
    const uint64_t turn = static_cast<uint64_t>(at) * p.freq[j];
    const float f = static_cast<float>(static_cast<uint32_t>(turn >> 40)) * 0x1p-24f;  // as in heads_kernel
    s_cos[wave][j] = __builtin_amdgcn_cosf(f);
    s_sin[wave][j] = __builtin_amdgcn_sinf(f);
  }
  // out = rs (x A + x' B), x' the dim's partner: A = (1 + w) cos, B = (1 + w') (-+ sin)
  float qa[8], qb[8], ka[8], kb[8];
  load_weights(p.qw, p.w_f32, j0, qa);
  load_weights(p.kw, p.w_f32, j0, ka);
  const int jp = !rot ? j0 : first ? j0 + half : j0 - half;
  load_weights(p.qw, p.w_f32, jp, qb);
  load_weights(p.kw, p.w_f32, jp, kb);
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // the wave reads only what it wrote
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float c = rot ? s_cos[wave][jh + e] : 1.f;
    const float s = !rot ? 0.f : first ? -s_sin[wave][jh + e] : s_sin[wave][jh + e];
    qa[e] *= c;
    ka[e] *= c;
    qb[e] *= s;
    kb[e] *= s;
  }
  const uint32_t turns = rot ? ~0u : 0u;  // a lane that does not turn would get anyone's value, a NaN perhaps
  const bool live = slot >= 0 && slot < p.num_slots;
  // a 32-bit division where the pool allows it: a fifth of a 64-bit one
  const int64_t block = !live ? 0 : p.num_slots <= 0xffffffffll ? static_cast<uint32_t>(slot) / static_cast<uint32_t>(p.bs) : slot / p.bs;
  const int at = live ? static_cast<int>(slot - block * p.bs) : 0;

  auto normalised = [&](const uint4& u, const float (&A)[8], const float (&B)[8]) {
    float x[8], y[8];
    widen8(u, x);
    widen8(make_uint4(partner_of(u.x, half / 8, first, lane) & turns, partner_of(u.y, half / 8, first, lane) & turns, partner_of(u.z, half / 8, first, lane) & turns,
                      partner_of(u.w, half / 8, first, lane) & turns), y);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
    ss = row16_sum(ss);
    if constexpr (D == 256) {
      const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(ss), __float_as_uint(ss), false, false);
      ss = __uint_as_float(both[0]) + __uint_as_float(both[1]);
    }
    const float rs = rsqrtf(ss * (1.f / D) + p.eps);
    uint32_t out[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float lo = (x[2 * e] * A[2 * e] + y[2 * e] * B[2 * e]) * rs;
      const float hi = (x[2 * e + 1] * A[2 * e + 1] + y[2 * e + 1] * B[2 * e + 1]) * rs;
      out[e] = static_cast<uint32_t>(f32_to_bf16(lo)) | static_cast<uint32_t>(f32_to_bf16(hi)) << 16;
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
  };
  auto append = [&](const uint4& u, int h, bool value) {
    if (!live || h >= p.Hkv) return;
    if constexpr (KV4) {
      using R = kv4::Run<D>;
      uint8_t* run = reinterpret_cast<uint8_t*>(value ? p.vpool : p.kpool) + block * p.sP + h * p.sG + static_cast<int64_t>(at >> 4) * R::kBytes;
      float z[8];
      widen8(u, z);
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(z[e]) & 0x7fffffffu);
      const uint32_t byte = kv4::scale_byte(__uint_as_float(quad_max(top)));
      const uint32_t codes = kv4::pack_codes(z, byte);
      const int t = at & 15, group = in_head / 4;
      const int to = value ? R::value_code(t, j0 / (D / 16)) + j0 % (D / 16) / 2 : R::key_code(t, group) + 4 * (in_head & 3);
      *reinterpret_cast<uint32_t*>(run + to) = codes;
      if ((in_head & 3) == 0) run[value ? R::value_scale(t, group) : R::key_scale(t, group)] = static_cast<uint8_t>(byte);
    } else {
      *reinterpret_cast<uint4*>(reinterpret_cast<bf16_t*>(value ? p.vpool : p.kpool) + block * p.sP + h * p.sG + at * p.sT + j0) = u;
    }
  };

  for (int from = part; from < steps; from += kStepsInFlight * waves_per_token) {
    if (from != part) load_pass(from);
#pragma unroll
    for (int i = 0; i < kStepsInFlight; ++i) {
      const int step = from + i * waves_per_token;
      if (step >= steps) break;
      if (step < nq) {
        const uint4 out = normalised(raw[i], qa, qb);
        const int h = step * SLOTS + sub;
        if (h < p.H) *reinterpret_cast<uint4*>(p.q_out + (n * p.H + h) * D + j0) = out;
      } else if (step < nq + nk) {
        append(normalised(raw[i], ka, kb), (step - nq) * SLOTS + sub, false);
      } else {
        append(raw[i], (step - nq - nk) * SLOTS + sub, true);
      }
    }
  }
}

}  // namespace mrope
}  // namespace qa

extern "C" int qa_qk_norm_mrope_append(const void* q_proj, int64_t q_stride_t, int64_t q_stride_h, const void* k_proj, int64_t k_stride_t, int64_t k_stride_h,
                                       const void* v_proj, int64_t v_stride_t, int64_t v_stride_h, const void* q_norm_weight, const void* k_norm_weight,
                                       int32_t weight_dtype, float eps, const uint64_t* freq_turns, const uint8_t* freq_axis, int32_t rotary_dim,
                                       const void* positions, int32_t positions_dtype, int64_t positions_stride, int32_t axes, int64_t tokens, int32_t heads,
                                       int32_t head_dim, const qa_paged_kv* kv, const void* slots, int32_t slots_dtype, int32_t block_size, void* q_out,
                                       hipStream_t stream) {
  using namespace qa;
  using namespace qa::mrope;
  QA_REQUIRE(kv != nullptr && (kv->dtype == QA_BF16 || kv->dtype == QA_KV4), "qk_norm_mrope_append: the KV pool must be bfloat16 or 4-bit");
  QA_REQUIRE(kv->row_key_ptrs == nullptr && kv->key && kv->value, "qk_norm_mrope_append: needs one shared pool");
  const bool kv4_pool = kv->dtype == QA_KV4;
  if (kv4_pool) {
    if (int rc = kv4::check_pool("qk_norm_mrope_append", kv, head_dim, block_size)) return rc;
  }
  QA_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "qk_norm_mrope_append: head_dim must be 64, 128 or 256");
  QA_REQUIRE(weight_dtype == QA_BF16 || weight_dtype == QA_F32, "qk_norm_mrope_append: norm weights must be bfloat16 or float32");
  QA_REQUIRE(is_index_dtype(positions_dtype) && is_index_dtype(slots_dtype), "qk_norm_mrope_append: index arrays must be int32/int64");
  const int E = head_dim / 64;
  QA_REQUIRE(rotary_dim > 0 && rotary_dim <= head_dim && rotary_dim % (2 * E) == 0, "qk_norm_mrope_append: rotary_dim must be in (0, head_dim] and a multiple of %d", 2 * E);
  QA_REQUIRE(axes >= 1 && axes <= kMaxAxes, "qk_norm_mrope_append: 1 to %d position axes", kMaxAxes);
  QA_REQUIRE(kv->kv_heads > 0 && heads > 0 && heads % kv->kv_heads == 0, "qk_norm_mrope_append: query heads must be a multiple of KV heads");
  QA_REQUIRE(kv->num_blocks >= 0 && block_size > 0, "qk_norm_mrope_append: block_size must be positive");
  QA_REQUIRE(eps >= 0.f, "qk_norm_mrope_append: eps must be non-negative");
  QA_REQUIRE(tokens >= 0 && tokens <= 0x7fffffff, "qk_norm_mrope_append: tokens out of range");
  if (tokens == 0) return 0;
  QA_REQUIRE(q_proj && k_proj && v_proj && q_norm_weight && k_norm_weight && freq_turns && freq_axis && positions && slots && q_out,
             "qk_norm_mrope_append: pointers must be non-null");
  const int64_t al = E;  // E-element vector accesses
  const bool pool_rows = kv4_pool || (kv->stride_block % al == 0 && kv->stride_head % al == 0 && kv->stride_token % al == 0 &&
                                      ((reinterpret_cast<uintptr_t>(kv->key) | reinterpret_cast<uintptr_t>(kv->value)) & static_cast<uintptr_t>(2 * E - 1)) == 0);
  QA_REQUIRE(pool_rows && q_stride_t % al == 0 && q_stride_h % al == 0 && k_stride_t % al == 0 && k_stride_h % al == 0 && v_stride_t % al == 0 && v_stride_h % al == 0 &&
                 ((reinterpret_cast<uintptr_t>(q_proj) | reinterpret_cast<uintptr_t>(k_proj) | reinterpret_cast<uintptr_t>(v_proj) | reinterpret_cast<uintptr_t>(q_out)) &
                  static_cast<uintptr_t>(2 * E - 1)) == 0,
             "qk_norm_mrope_append: rows must be %d-byte aligned", 2 * E);
  Params p{};
  p.q = reinterpret_cast<const bf16_t*>(q_proj);
  p.q_st = q_stride_t;
  p.q_sh = q_stride_h;
  p.k = reinterpret_cast<const bf16_t*>(k_proj);
  p.k_st = k_stride_t;
  p.k_sh = k_stride_h;
  p.v = reinterpret_cast<const bf16_t*>(v_proj);
  p.v_st = v_stride_t;
  p.v_sh = v_stride_h;
  p.qw = q_norm_weight;
  p.kw = k_norm_weight;
  p.w_f32 = weight_dtype == QA_F32;
  p.freq = freq_turns;
  p.axis = freq_axis;
  p.positions = positions;
  p.pos_stride = positions_stride;
  p.pos_i64 = positions_dtype == QA_I64;
  p.axes = axes;
  p.eps = eps;
  p.slots = slots;
  p.slots_i64 = slots_dtype == QA_I64;
  p.tokens = tokens;
  p.kpool = kv->key;
  p.vpool = kv->value;
  p.num_slots = kv->num_blocks * block_size;
  p.sP = kv->stride_block;
  p.sG = kv->stride_head;
  p.sT = kv->stride_token;
  p.H = heads;
  p.Hkv = kv->kv_heads;
  p.rd = rotary_dim;
  p.bs = block_size;
  p.q_out = reinterpret_cast<bf16_t*>(q_out);
  auto rows16 = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; };
  const bool rows = E >= 2 && rotary_dim % 16 == 0 && rows16(q_proj) && rows16(k_proj) && rows16(v_proj) && rows16(q_out) && rows16(q_norm_weight) && rows16(k_norm_weight) &&
                    q_stride_t % 8 == 0 && q_stride_h % 8 == 0 && k_stride_t % 8 == 0 && k_stride_h % 8 == 0 && v_stride_t % 8 == 0 && v_stride_h % 8 == 0 &&
                    (kv4_pool || (rows16(kv->key) && rows16(kv->value) && kv->stride_block % 8 == 0 && kv->stride_head % 8 == 0 && kv->stride_token % 8 == 0));
  KernelTimer timer_("qk_norm_mrope", stream);
  if (rows) {
    const int at_once = E == 4 ? 2 : 4;
    const int64_t steps = ceil_div(p.H, at_once) + 2 * ceil_div(p.Hkv, at_once);
    const int waves = static_cast<int>(std::min(steps, std::max<int64_t>(1, kWaves / tokens)));
    const dim3 grid(static_cast<unsigned>(ceil_div(tokens * waves, 4)));
    if (E == 4) {
      if (kv4_pool)
        hipLaunchKernelGGL((rows_kernel<256, true>), grid, dim3(256), 0, stream, p, waves);
      else
        hipLaunchKernelGGL((rows_kernel<256, false>), grid, dim3(256), 0, stream, p, waves);
    } else {
      if (kv4_pool)
        hipLaunchKernelGGL((rows_kernel<128, true>), grid, dim3(256), 0, stream, p, waves);
      else
        hipLaunchKernelGGL((rows_kernel<128, false>), grid, dim3(256), 0, stream, p, waves);
    }
  } else {
    const dim3 grid(static_cast<unsigned>(tokens));
    if (kv4_pool) {
      if (E == 4)
        hipLaunchKernelGGL((heads_kernel<4, true>), grid, dim3(256), 0, stream, p);
      else
        hipLaunchKernelGGL((heads_kernel<2, true>), grid, dim3(256), 0, stream, p);
    } else {
      if (E == 4)
        hipLaunchKernelGGL((heads_kernel<4, false>), grid, dim3(256), 0, stream, p);
      else if (E == 2)
        hipLaunchKernelGGL((heads_kernel<2, false>), grid, dim3(256), 0, stream, p);
      else
        hipLaunchKernelGGL((heads_kernel<1, false>), grid, dim3(256), 0, stream, p);
    }
  }
  return check_launch("qk_norm_mrope_append");
}
