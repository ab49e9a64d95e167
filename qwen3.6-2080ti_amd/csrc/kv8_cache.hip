// Writes and dense reads of the 8-bit paged KV cache (layout and number format: kv8.h), gfx950.
//
// Both are bound by memory: per token and KV head the append reads 2 x 2 D bytes of bf16 and writes 2 x D, the gather the
// other way round.  A wave takes the keys, or the values, of one run: its scale needs the largest magnitude of all tokens of the
// run that the call brings, so one wave holds them all in registers and reads them once, and no two waves write to one run.
// Tokens of a run follow one another in the slot map, with none but skipped ones between them; the first of them leads, and the waves
// look for leaders among `window` tokens each.
// Four prompts of 6003 tokens, two heads of 256, 74 MB each way: append 18.0 to 18.6 us (16.5 where the caches still hold the rows),
// gather 14.0; a token for each of seven rows 5.7 to 6.0, and their dense view of 428 tokens 4.2.
#include "kv8.h"

namespace qa {
namespace kv8 {

struct AppendParams {
  const void* key;
  const void* value;
  int64_t k_st, k_sh, v_st, v_sh;  // element strides
  uint8_t* kpool;
  uint8_t* vpool;
  int64_t num_slots, sP, sG;  // blocks * block_size; byte strides
  const void* slots;
  int64_t tokens;
  int Hkv, bs_shift, window;
};

// N elements at off as floats.
template <bool F32, int N>
__device__ __forceinline__ void load(const void* base, int64_t off, float (&x)[N]) {
  if constexpr (F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + off + i);
      x[i] = a.x, x[i + 1] = a.y, x[i + 2] = a.z, x[i + 3] = a.w;
    }
  } else {
    uint32_t w[N / 2];
    if constexpr (N == 4) {
      const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const bf16_t*>(base) + off);
      w[0] = u.x, w[1] = u.y;
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; i += 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16_t*>(base) + off + 2 * i);
        w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
      }
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// The largest finite magnitude's bits; what is not finite becomes a NaN.
__device__ __forceinline__ uint32_t finite_bits(float& x) {
  const uint32_t bits = __float_as_uint(x) & 0x7fffffffu;
  if (bits < 0x7f800000u) return bits;
  x = __uint_as_float(0x7fc00000u);
  return 0u;
}

// Four codes; v_cvt_pk_fp8_f32 rounds to nearest, ties to the even code.
__device__ __forceinline__ uint32_t pack(float a, float b, float c, float d) {
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}

// Four codes rounded to a scale that is `down` (a power of two, or 0) times their own.
__device__ __forceinline__ uint32_t rescaled(uint32_t codes, float down) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
  return pack(lo[0] * down, lo[1] * down, hi[0] * down, hi[1] * down);
}

// Of a run: where its codes lie, and what the call brings.
struct Bring {
  uint8_t* at;
  int64_t n;       // the first of the call's tokens of the run
  int64_t head;    // of the source: h * head stride
  int nth;         // lane t < 16: 1 + how far behind that one token t stands, 0: none
  int first;       // the first token that the call brings
  int count;
  uint32_t old;    // scale byte before; 0 where the run starts anew
};

// The run's scale byte, and what its old codes are multiplied with: 1 where they stay.
__device__ __forceinline__ uint32_t settle(const Bring& r, uint32_t top, float& down) {
  const uint32_t fresh = scale_byte(wave_max_bits(top));
  const uint32_t byte = max(fresh, r.old);
  down = r.old == 0 || byte == r.old ? 1.f : __uint_as_float(static_cast<uint32_t>(max(0, 127 + static_cast<int>(r.old) - static_cast<int>(byte))) << 23);
  return byte;
}

// At the largest scale, in the codes that a lane has written (the bytes of `fresh`): 240 in place of 256.  Behind the writing, where it is
// hardly ever reached: beside the packing, each code's branch took prompts of 4 x 6003 tokens from 35.1 to 36.3 us.
template <int D>
__device__ __forceinline__ void below_256(uint32_t byte, uint4* codes, uint32_t fresh) {
  if (__builtin_amdgcn_readfirstlane(byte) != kMost || fresh == 0) return;
  auto lower = [&](uint32_t w) {
    const uint32_t size = w & 0x7f7f7f7fu;
    const uint32_t over = (size + 0x08080808u) & ~(size + 0x01010101u) & fresh & 0x80808080u;  // 0x78, no NaN; none is between them
    return w - (over >> 7);
  };
#pragma unroll 1
  for (int s = 0; s < Run<D>::kSlices; ++s) {
    const uint4 c = codes[64 * s];
    codes[64 * s] = make_uint4(lower(c.x), lower(c.y), lower(c.z), lower(c.w));
  }
}

template <int D, bool F32>
__device__ __forceinline__ void write_keys(const AppendParams& p, const Bring& r, int lane) {
  constexpr int S = Run<D>::kSlices;
  const int t = lane & 15, quad = lane >> 4;
  const int nth = __shfl(r.nth, t, 64);
  const int64_t off = (r.n + max(nth, 1) - 1) * p.k_st + r.head + 16 * quad;
  float x[S][16];
#pragma unroll
  for (int s = 0; s < S; ++s) load<F32>(p.key, off + 64 * s, x[s]);
  uint32_t top = 0;
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, finite_bits(x[s][i]));
  float down;
  const uint32_t byte = settle(r, nth > 0 ? top : 0u, down);
  const float inv = over_scale(byte);
  uint4* codes = reinterpret_cast<uint4*>(r.at) + lane;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (nth > 0) {
      uint4 c;
      c.x = pack(x[s][0] * inv, x[s][1] * inv, x[s][2] * inv, x[s][3] * inv);
      c.y = pack(x[s][4] * inv, x[s][5] * inv, x[s][6] * inv, x[s][7] * inv);
      c.z = pack(x[s][8] * inv, x[s][9] * inv, x[s][10] * inv, x[s][11] * inv);
      c.w = pack(x[s][12] * inv, x[s][13] * inv, x[s][14] * inv, x[s][15] * inv);
      codes[64 * s] = c;
    } else if (down != 1.f && t < r.first) {
      const uint4 c = codes[64 * s];
      codes[64 * s] = make_uint4(rescaled(c.x, down), rescaled(c.y, down), rescaled(c.z, down), rescaled(c.w, down));
    }
  }
  below_256<D>(byte, codes, nth > 0 ? ~0u : 0u);
  if (lane == 0) *reinterpret_cast<uint4*>(r.at + Run<D>::kCodes) = make_uint4(byte, 0, 0, 0);
}

template <int D, bool F32>
__device__ __forceinline__ void write_values(const AppendParams& p, const Bring& r, int lane) {
  constexpr int S = Run<D>::kSlices;
  const int c = lane & 15, quad = lane >> 4;
  uint4* codes = reinterpret_cast<uint4*>(r.at) + lane;
  int nth[4];
  uint32_t fresh = 0, before = 0;  // bytes of the tokens that the call brings, and of those before the first of them
  float x[S][4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    nth[i] = __shfl(r.nth, 4 * quad + i, 64);
    if (nth[i] > 0) fresh |= 255u << (8 * i);
    if (4 * quad + i < r.first) before |= 255u << (8 * i);
    const int64_t off = (r.n + max(nth[i], 1) - 1) * p.v_st + r.head + 4 * c;
#pragma unroll
    for (int s = 0; s < S; ++s) load<F32>(p.value, off + 64 * s, x[s][i]);
  }
  uint4 have[S];
  if (r.count < kRun) {
#pragma unroll
    for (int s = 0; s < S; ++s) have[s] = codes[64 * s];
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t of = 0;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int m = 0; m < 4; ++m) of = max(of, finite_bits(x[s][i][m]));
    if (nth[i] > 0) top = max(top, of);
  }
  float down;
  const uint32_t byte = settle(r, top, down);
  const float inv = over_scale(byte);
  if (fresh != 0 || (down != 1.f && before != 0)) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      uint32_t w[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) w[m] = pack(x[s][0][m] * inv, x[s][1][m] * inv, x[s][2][m] * inv, x[s][3][m] * inv);
      if (r.count < kRun) {
        const uint32_t was[4] = {have[s].x, have[s].y, have[s].z, have[s].w};
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          uint32_t keep = was[m];
          if (down != 1.f) keep = (rescaled(keep, down) & before) | (keep & ~before);
          w[m] = (w[m] & fresh) | (keep & ~fresh);
        }
      }
      codes[64 * s] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  below_256<D>(byte, codes, fresh);
  if (lane == 0) *reinterpret_cast<uint4*>(r.at + Run<D>::kCodes) = make_uint4(byte, 0, 0, 0);
}

template <int D, bool F32, bool S64>
__global__ __launch_bounds__(256) void append_kernel(AppendParams p) {
  const int lane = threadIdx.x & 63;
  const int h = blockIdx.y >> 1;
  const bool values = blockIdx.y & 1;
  const int64_t n0 = (static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * p.window;
  if (n0 >= p.tokens) return;
  int at;  // place of the token in its run
  auto run_of = [&](int64_t n) -> int64_t {  // -1: skipped
    const int64_t nn = max64(0, min64(n, p.tokens - 1));
    const int64_t slot = S64 ? reinterpret_cast<const int64_t*>(p.slots)[nn] : reinterpret_cast<const int32_t*>(p.slots)[nn];
    at = static_cast<int>(slot & 15);
    return n == nn && slot >= 0 && slot < p.num_slots ? slot >> 4 : -1;
  };
  auto of_lane = [&](int64_t v, int from) {
    return (static_cast<int64_t>(__shfl(static_cast<int>(v >> 32), from, 64)) << 32) | static_cast<uint32_t>(__shfl(static_cast<int>(v), from, 64));
  };
  // Of the groups of 64 tokens n + 64 j, j from 0 (step 64) or 0 down (step -64), the first one, by its first token, that are not all
  // skipped: a stretch of skipped tokens goes by 512 at a time (a call of 10 tokens with 8182 skipped ones behind them 39.5 -> 16.9 us; 1024 at a time 13.0, but 40
  // registers more, with which a long prompt took 33.5 and not 31.6).
  auto past_skipped = [&](int64_t n, int64_t step) {
    constexpr int kGroups = 8;
    while (n < p.tokens && n > -64) {
      uint32_t some = 0;
#pragma unroll
      for (int j = 0; j < kGroups; ++j) some |= (run_of(n + step * j + lane) >= 0 ? 1u : 0u) << j;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) some |= __shfl_xor(some, off, 64);
      if (some != 0) return n + step * (__ffs(static_cast<int>(some)) - 1);
      n += step * kGroups;
    }
    return n;
  };
  // Lane i has token n0 - 1 + i: the one before the window, the window, and those that may follow its last leader.  A token leads
  // its run where the last one before it that is not skipped belongs to another.
  const int64_t run = run_of(n0 - 1 + lane);
  const int place = at;
  const uint64_t there = __ballot(run >= 0);
  const uint64_t below = there & ((1ull << lane) - 1ull);
  int64_t before = of_lane(run, below != 0 ? 63 - __clzll(static_cast<long long>(below)) : 0);
  if ((there & 1) == 0 && (there >> 1 & ((1ull << p.window) - 1)) != 0) {
    int64_t last = -1;  // of the tokens before those: the last that is not skipped
    const int64_t n = past_skipped(n0 - 65, -64);
    const int64_t earlier = run_of(n + lane);
    const uint64_t some = __ballot(earlier >= 0);
    if (some != 0) last = of_lane(earlier, 63 - __clzll(static_cast<long long>(some)));
    if (below == 0) before = last;
  }
  uint64_t leaders = __ballot(run >= 0 && run != before && lane >= 1 && lane <= p.window);
  while (leaders != 0) {
    const int lead = __ffsll(static_cast<unsigned long long>(leaders)) - 1;
    leaders &= leaders - 1;
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(run), lead), hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(run >> 32), lead);
    const int64_t own = static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
    Bring r;
    r.n = n0 - 1 + lead;
    r.nth = 0;
    r.count = 0;
    int64_t mine = run;  // of this lane's token, lane `from` being the first that counts
    int its = place, from = lead;
    for (int64_t n = n0 - 1;;) {
      const uint64_t others = __ballot(mine >= 0 && mine != own) >> from;
      const int end = others != 0 ? from + __ffsll(static_cast<unsigned long long>(others)) - 1 : 64;
      const bool member = mine == own && lane >= from && lane < end;
      // each token of the run tells the lane of its place; the others talk past lane 31
      const int nth = __builtin_amdgcn_ds_permute(4 * (member ? its : 32 + (lane & 31)), static_cast<int>(n + lane - r.n) + 1);
      if (lane < kRun) r.nth = max(r.nth, nth);
      r.count = __popcll(__ballot(r.nth > 0));
      n += 64;
      if (end < 64 || r.count == kRun || n >= p.tokens) break;
      mine = run_of(n + lane);
      if (__ballot(mine >= 0) == 0) {
        n = past_skipped(n + 64, 64);
        if (n >= p.tokens) break;
        mine = run_of(n + lane);
      }
      its = at;
      from = 0;
    }
    r.first = __ffsll(static_cast<unsigned long long>(__ballot(r.nth > 0))) - 1;
    const int bs_runs = p.bs_shift - 4;
    const int64_t o = (own >> bs_runs) * p.sP + h * p.sG + (own & ((1 << bs_runs) - 1)) * Run<D>::kBytes;
    r.at = (values ? p.vpool : p.kpool) + o;
    r.head = h * (values ? p.v_sh : p.k_sh);
    r.old = 0;
    if (r.first > 0) r.old = min(max(static_cast<uint32_t>(r.at[Run<D>::kCodes]), kLeast), kMost);
    if (values)
      write_values<D, F32>(p, r, lane);
    else
      write_keys<D, F32>(p, r, lane);
  }
}

struct GatherParams {
  const uint8_t* kpool;
  const uint8_t* vpool;
  int64_t num_blocks, sP, sG;
  const void* tables;
  int64_t table_stride, max_blocks;
  int64_t valid;
  bf16_t* key_out;  // (B, Hkv, valid, D)
  bf16_t* value_out;
  int Hkv, bs_shift;
};

template <int D, bool T64>
__global__ __launch_bounds__(256) void gather_kernel(GatherParams p) {
  constexpr int S = Run<D>::kSlices;
  const int lane = threadIdx.x & 63;
  const int h = blockIdx.y >> 1;
  const bool values = blockIdx.y & 1;
  const int64_t b = blockIdx.z;
  const int64_t run = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (run * kRun >= p.valid) return;
  const int64_t logical = run >> (p.bs_shift - 4);
  int64_t phys = -1;
  if (logical < p.max_blocks) {
    const int64_t off = b * p.table_stride + logical;
    phys = T64 ? reinterpret_cast<const int64_t*>(p.tables)[off] : reinterpret_cast<const int32_t*>(p.tables)[off];
  }
  uint4 code[S];
  float scale = 1.f;
#pragma unroll
  for (int s = 0; s < S; ++s) code[s] = make_uint4(0, 0, 0, 0);
  if (phys >= 0 && phys < p.num_blocks) {
    const uint8_t* at = (values ? p.vpool : p.kpool) + phys * p.sP + h * p.sG + (run & ((1 << (p.bs_shift - 4)) - 1)) * Run<D>::kBytes;
#pragma unroll
    for (int s = 0; s < S; ++s) code[s] = reinterpret_cast<const uint4*>(at)[64 * s + lane];
    scale = scale_of(at[Run<D>::kCodes]);
  }
  const int64_t row0 = ((b * p.Hkv + h) * p.valid + run * kRun) * D;
  const int left = static_cast<int>(min64(kRun, p.valid - run * kRun));  // tokens
  if (!values) {
    const int t = lane & 15, quad = lane >> 4;
    if (t >= left) return;
    bf16_t* out = p.key_out + row0 + t * D + 16 * quad;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const uint4 c = code[s];
      *reinterpret_cast<uint4*>(out + 64 * s) = make_uint4(widen<false>(c.x, scale), widen<true>(c.x, scale), widen<false>(c.y, scale), widen<true>(c.y, scale));
      *reinterpret_cast<uint4*>(out + 64 * s + 8) = make_uint4(widen<false>(c.z, scale), widen<true>(c.z, scale), widen<false>(c.w, scale), widen<true>(c.w, scale));
    }
    return;
  }
  const int c0 = lane & 15, t = 4 * (lane >> 4);
  bf16_t* out = p.value_out + row0 + t * D + 4 * c0;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const uint32_t w[4] = {code[s].x, code[s].y, code[s].z, code[s].w};
    uint32_t even[4], odd[4];  // tokens 0 and 1, 2 and 3, of dim m
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      even[m] = widen<false>(w[m], scale);
      odd[m] = widen<true>(w[m], scale);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (t + i >= left) continue;
      const uint32_t* u = i < 2 ? even : odd;
      const uint32_t pick = i & 1 ? 0x07060302u : 0x05040100u;
      *reinterpret_cast<uint2*>(out + i * D + 64 * s) = make_uint2(__builtin_amdgcn_perm(u[1], u[0], pick), __builtin_amdgcn_perm(u[3], u[2], pick));
    }
  }
}

template <int D, bool F32>
static void launch_append(const AppendParams& p, bool s64, dim3 grid, hipStream_t stream) {
  if (s64)
    hipLaunchKernelGGL((append_kernel<D, F32, true>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((append_kernel<D, F32, false>), grid, dim3(256), 0, stream, p);
}

template <int D>
static void launch_gather(const GatherParams& p, bool t64, dim3 grid, hipStream_t stream) {
  if (t64)
    hipLaunchKernelGGL((gather_kernel<D, true>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((gather_kernel<D, false>), grid, dim3(256), 0, stream, p);
}

// Tokens among which a wave looks for leaders: one where there are few, so that every run has a wave at once; more where waves
// that lead nothing would be too many.  us with windows of 1, 4, 16, two heads of 256: 128 rows of a token 5.0 14.3 45.0, 512 rows 6.5
// 13.7 46.6, 2000 rows 16.7 19.8 48.0; prompts of 500 tokens 4.3 4.2 4.6, of 1000 4.6 4.3 4.7, 4000 14.0 5.9 5.1, 24000 66 20.6 16.5.
static int window_of(int64_t tokens) { return tokens <= 1024 ? 1 : tokens <= 4096 ? 4 : 16; }

static int shift_of(int32_t block_size) { return __builtin_ctz(static_cast<unsigned>(block_size)); }

}  // namespace kv8
}  // namespace qa

extern "C" int qa_paged_kv8_append(const void* key_new, const void* value_new, int32_t dtype, int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t,
                                   int64_t v_stride_h, int64_t tokens, int32_t head_dim, const qa_paged_kv* kv, const void* slots, int32_t slots_dtype,
                                   int32_t block_size, hipStream_t stream) {
  using namespace qa;
  using namespace qa::kv8;
  if (int rc = check_pool("paged_kv8_append", kv, head_dim, block_size)) return rc;
  QA_REQUIRE(is_float_dtype(dtype), "paged_kv8_append: key/value must be float32 or bfloat16");
  QA_REQUIRE(is_index_dtype(slots_dtype), "paged_kv8_append: slots must be int32 or int64");
  QA_REQUIRE(tokens >= 0 && tokens <= 0x7fffffff, "paged_kv8_append: tokens out of range");
  if (tokens == 0) return 0;
  QA_REQUIRE(key_new && value_new && slots, "paged_kv8_append: pointers must be non-null");
  const int64_t al = dtype == QA_F32 ? 4 : 8;
  QA_REQUIRE(k_stride_t % al == 0 && k_stride_h % al == 0 && v_stride_t % al == 0 && v_stride_h % al == 0 &&
                 ((reinterpret_cast<uintptr_t>(key_new) | reinterpret_cast<uintptr_t>(value_new)) & 15u) == 0,
             "paged_kv8_append: rows must be 16-byte aligned");
  QA_REQUIRE(kv->kv_heads <= 32767, "paged_kv8_append: too many KV heads");
  AppendParams p{};
  p.key = key_new;
  p.value = value_new;
  p.k_st = k_stride_t;
  p.k_sh = k_stride_h;
  p.v_st = v_stride_t;
  p.v_sh = v_stride_h;
  p.kpool = reinterpret_cast<uint8_t*>(kv->key);
  p.vpool = reinterpret_cast<uint8_t*>(kv->value);
  p.num_slots = kv->num_blocks * block_size;
  p.sP = kv->stride_block;
  p.sG = kv->stride_head;
  p.slots = slots;
  p.tokens = tokens;
  p.Hkv = kv->kv_heads;
  p.bs_shift = shift_of(block_size);
  p.window = window_of(tokens);
  const dim3 grid(static_cast<unsigned>(ceil_div(tokens, 4 * p.window)), 2u * kv->kv_heads);
  const bool s64 = slots_dtype == QA_I64;
  {
    KernelTimer timer_("kv8_append", stream);
    if (head_dim == 256)
      dtype == QA_F32 ? launch_append<256, true>(p, s64, grid, stream) : launch_append<256, false>(p, s64, grid, stream);
    else
      dtype == QA_F32 ? launch_append<128, true>(p, s64, grid, stream) : launch_append<128, false>(p, s64, grid, stream);
  }
  return check_launch("paged_kv8_append");
}

extern "C" int qa_paged_kv8_gather(const qa_paged_kv* kv, int32_t head_dim, int64_t batch, const void* block_tables, int32_t table_dtype, int64_t table_stride,
                                   int64_t max_blocks, int64_t valid, int32_t block_size, void* key_out, void* value_out, hipStream_t stream) {
  using namespace qa;
  using namespace qa::kv8;
  if (int rc = check_pool("paged_kv8_gather", kv, head_dim, block_size)) return rc;
  QA_REQUIRE((block_tables != nullptr || batch == 0) && is_index_dtype(table_dtype), "block table must be an int32/int64 device array");
  QA_REQUIRE(batch >= 0 && batch <= 65535, "paged_kv8_gather: batch must be in [0, 65535]");
  QA_REQUIRE(max_blocks > 0 && table_stride >= 0, "paged_kv8_gather: max_blocks must be positive");
  QA_REQUIRE(valid >= 0 && valid <= 0x7fffffff, "paged_kv8_gather: valid out of range");
  if (valid == 0 || batch == 0) return 0;
  QA_REQUIRE(key_out && value_out && ((reinterpret_cast<uintptr_t>(key_out) | reinterpret_cast<uintptr_t>(value_out)) & 15u) == 0,
             "paged_kv8_gather: outputs must be non-null and 16-byte aligned");
  QA_REQUIRE(kv->kv_heads <= 32767, "paged_kv8_gather: too many KV heads");
  GatherParams p{};
  p.kpool = reinterpret_cast<const uint8_t*>(kv->key);
  p.vpool = reinterpret_cast<const uint8_t*>(kv->value);
  p.num_blocks = kv->num_blocks;
  p.sP = kv->stride_block;
  p.sG = kv->stride_head;
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.max_blocks = max_blocks;
  p.valid = valid;
  p.key_out = reinterpret_cast<bf16_t*>(key_out);
  p.value_out = reinterpret_cast<bf16_t*>(value_out);
  p.Hkv = kv->kv_heads;
  p.bs_shift = shift_of(block_size);
  const dim3 grid(static_cast<unsigned>(ceil_div(valid, 4 * kRun)), 2u * kv->kv_heads, static_cast<unsigned>(batch));
  {
    KernelTimer timer_("kv8_gather", stream);
    head_dim == 256 ? launch_gather<256>(p, table_dtype == QA_I64, grid, stream) : launch_gather<128>(p, table_dtype == QA_I64, grid, stream);
  }
  return check_launch("paged_kv8_gather");
}
