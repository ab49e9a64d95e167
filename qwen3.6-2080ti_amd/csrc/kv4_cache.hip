// Writes and dense reads of the 4-bit paged KV cache (layout and number format: kv4.h), gfx950.
//
// Both are bound by memory: per token and KV head the append reads 2 x 2 D bytes of bf16 and writes 2 x 17 D / 32, the
// gather the other way round.  A wave takes groups (head, 32 dims) of 16 consecutive tokens, four lanes a token and eight
// dims a lane: loads are 64-byte pieces of rows, the group's maximum needs two quad swaps, and the 16 tokens of
// a run land in 256 consecutive bytes of keys.  Rows that are adjacent in the source but not in the pool stay right:
// every lane takes its own token's slot.  Three prompts of 4001 tokens, two heads of 256, 31 MB each way: append 7.3 us,
// gather 7.3 (a launch that does nothing takes 2.5 of it, a copy of as much 6.4), append of fp32 rows, 56 MB, 9.3; five rows
// of one and of 334: 2.9, 3.6 us.
#include "kv4.h"

namespace qa {
namespace kv4 {

// Groups of 32 dims a wave takes, its loads on their way together.  us at 1, 2 and 4 groups, heads of 256: append of 3 x 4001
// tokens 10.1 7.8 8.4, of 8 x 8000 42.2 32.8 32.1, of 5 2.5 2.8 3.1; the gathers of as many 8.9 8.1 7.5, 38.8 30.9 28.9.
constexpr int kAppendGroups = 2, kGatherGroups = 4;

struct AppendParams {
  const void* key;
  const void* value;
  int64_t k_st, k_sh, v_st, v_sh;  // element strides
  uint8_t* kpool;
  uint8_t* vpool;
  int64_t num_slots, sP, sG;  // blocks * block_size; byte strides
  const void* slots;
  int64_t tokens;
  int Hkv, bs_shift;
};

template <bool F32>
__device__ __forceinline__ void load8(const void* base, int64_t off, float (&x)[8]) {
  if constexpr (F32) {
    const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + off);
    const float4 b = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + off + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16_t*>(base) + off);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ uint32_t group_byte(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  return scale_byte(__uint_as_float(quad_max(m)));
}

template <int D, bool F32, bool S64>
__global__ __launch_bounds__(256) void append_kernel(AppendParams p) {
  using R = Run<D>;
  const int lane = threadIdx.x & 63;
  constexpr int kSteps = R::kGroups / kAppendGroups;
  const int group0 = blockIdx.y % kSteps * kAppendGroups;
  const int h = blockIdx.y / kSteps;
  const int64_t n = (static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)) * kRun + (lane >> 2);
  const int sub = lane & 3;
  const int64_t nn = min64(n, p.tokens - 1);  // no branch round the loads: a lane past the end reads the last token
  const int64_t slot = S64 ? reinterpret_cast<const int64_t*>(p.slots)[nn] : reinterpret_cast<const int32_t*>(p.slots)[nn];
  float k[kAppendGroups][8], v[kAppendGroups][8];
#pragma unroll
  for (int u = 0; u < kAppendGroups; ++u) {
    load8<F32>(p.key, nn * p.k_st + h * p.k_sh + (group0 + u) * 32 + 8 * sub, k[u]);
    load8<F32>(p.value, nn * p.v_st + h * p.v_sh + (group0 + u) * 32 + 8 * sub, v[u]);
  }
  const bool there = n < p.tokens && slot >= 0 && slot < p.num_slots;
  const int at = there ? static_cast<int>(slot & ((1 << p.bs_shift) - 1)) : 0;
  const int t = at & 15;
  const int64_t run = there ? (slot >> p.bs_shift) * p.sP + h * p.sG + static_cast<int64_t>(at >> 4) * R::kBytes : 0;
#pragma unroll
  for (int u = 0; u < kAppendGroups; ++u) {
    const uint32_t kb = group_byte(k[u]), vb = group_byte(v[u]);
    const uint32_t kc = pack_codes(k[u], kb), vc = pack_codes(v[u], vb);
    if (!there) continue;
    const int group = group0 + u;
    const int d0 = group * 32 + 8 * sub;
    *reinterpret_cast<uint32_t*>(p.kpool + run + R::key_code(t, group) + 4 * sub) = kc;
    // eight dims are half a chunk of values at D = 256 and a whole one at D = 128
    *reinterpret_cast<uint32_t*>(p.vpool + run + R::value_code(t, d0 / (D / 16)) + d0 % (D / 16) / 2) = vc;
    if (sub == 0) {
      p.kpool[run + R::key_scale(t, group)] = static_cast<uint8_t>(kb);
      p.vpool[run + R::value_scale(t, group)] = static_cast<uint8_t>(vb);
    }
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

__device__ __forceinline__ uint4 unpack_codes(uint32_t codes, uint32_t byte) {
  const float s = __uint_as_float(byte << 23);
  uint4 u;
  u.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 0));
  u.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 1));
  u.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 2));
  u.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 3));
  return u;
}

template <int D, bool T64>
__global__ __launch_bounds__(256) void gather_kernel(GatherParams p) {
  using R = Run<D>;
  const int lane = threadIdx.x & 63;
  constexpr int kSteps = R::kGroups / kGatherGroups;
  const int group0 = blockIdx.y % kSteps * kGatherGroups;
  const int h = blockIdx.y / kSteps;
  const int64_t b = blockIdx.z;
  const int64_t run16 = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);  // the wave's run of 16 tokens
  const int t = lane >> 2, sub = lane & 3;
  if (run16 * kRun >= p.valid) return;
  const int64_t logical = run16 >> (p.bs_shift - 4);
  int64_t phys = -1;
  if (logical < p.max_blocks) {
    const int64_t off = b * p.table_stride + logical;
    phys = T64 ? reinterpret_cast<const int64_t*>(p.tables)[off] : reinterpret_cast<const int32_t*>(p.tables)[off];
  }
  uint4 k[kGatherGroups], v[kGatherGroups];
#pragma unroll
  for (int u = 0; u < kGatherGroups; ++u) k[u] = v[u] = make_uint4(0, 0, 0, 0);
  if (phys >= 0 && phys < p.num_blocks) {
    const int64_t run = phys * p.sP + h * p.sG + (run16 & ((1 << (p.bs_shift - 4)) - 1)) * R::kBytes;
    uint32_t kc[kGatherGroups], vc[kGatherGroups], kb[kGatherGroups], vb[kGatherGroups];
#pragma unroll
    for (int u = 0; u < kGatherGroups; ++u) {
      const int group = group0 + u;
      const int d0 = group * 32 + 8 * sub;
      kc[u] = *reinterpret_cast<const uint32_t*>(p.kpool + run + R::key_code(t, group) + 4 * sub);
      vc[u] = *reinterpret_cast<const uint32_t*>(p.vpool + run + R::value_code(t, d0 / (D / 16)) + d0 % (D / 16) / 2);
      kb[u] = p.kpool[run + R::key_scale(t, group)];
      vb[u] = p.vpool[run + R::value_scale(t, group)];
    }
#pragma unroll
    for (int u = 0; u < kGatherGroups; ++u) {
      k[u] = unpack_codes(kc[u], kb[u]);
      v[u] = unpack_codes(vc[u], vb[u]);
    }
  }
  const int64_t n = run16 * kRun + t;
  if (n >= p.valid) return;
  const int64_t out = ((b * p.Hkv + h) * p.valid + n) * D + group0 * 32 + 8 * sub;
#pragma unroll
  for (int u = 0; u < kGatherGroups; ++u) {
    *reinterpret_cast<uint4*>(p.key_out + out + 32 * u) = k[u];
    *reinterpret_cast<uint4*>(p.value_out + out + 32 * u) = v[u];
  }
}

template <int D, bool F32>
static void launch_append(const AppendParams& p, bool s64, dim3 grid, hipStream_t stream) {
  if (s64)
    hipLaunchKernelGGL((append_kernel<D, F32, true>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((append_kernel<D, F32, false>), grid, dim3(256), 0, stream, p);
}

static int shift_of(int32_t block_size) { return __builtin_ctz(static_cast<unsigned>(block_size)); }

}  // namespace kv4
}  // namespace qa

extern "C" int qa_paged_kv4_append(const void* key_new, const void* value_new, int32_t dtype, int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t,
                                   int64_t v_stride_h, int64_t tokens, int32_t head_dim, const qa_paged_kv* kv, const void* slots, int32_t slots_dtype,
                                   int32_t block_size, hipStream_t stream) {
  using namespace qa;
  using namespace qa::kv4;
  if (int rc = check_pool("paged_kv4_append", kv, head_dim, block_size)) return rc;
  QA_REQUIRE(is_float_dtype(dtype), "paged_kv4_append: key/value must be float32 or bfloat16");
  QA_REQUIRE(is_index_dtype(slots_dtype), "paged_kv4_append: slots must be int32 or int64");
  QA_REQUIRE(tokens >= 0 && tokens <= 0x7fffffff, "paged_kv4_append: tokens out of range");
  if (tokens == 0) return 0;
  QA_REQUIRE(key_new && value_new && slots, "paged_kv4_append: pointers must be non-null");
  const int64_t al = dtype == QA_F32 ? 4 : 8;
  QA_REQUIRE(k_stride_t % al == 0 && k_stride_h % al == 0 && v_stride_t % al == 0 && v_stride_h % al == 0 &&
                 ((reinterpret_cast<uintptr_t>(key_new) | reinterpret_cast<uintptr_t>(value_new)) & 15u) == 0,
             "paged_kv4_append: rows must be 16-byte aligned");
  const int64_t gy = static_cast<int64_t>(kv->kv_heads) * (head_dim / 32 / kAppendGroups);
  QA_REQUIRE(gy <= 65535, "paged_kv4_append: too many KV heads");
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
  const dim3 grid(static_cast<unsigned>(ceil_div(tokens, 4 * kRun)), static_cast<unsigned>(gy));
  const bool s64 = slots_dtype == QA_I64;
  {
    KernelTimer timer_("kv4_append", stream);
    if (head_dim == 256)
      dtype == QA_F32 ? launch_append<256, true>(p, s64, grid, stream) : launch_append<256, false>(p, s64, grid, stream);
    else
      dtype == QA_F32 ? launch_append<128, true>(p, s64, grid, stream) : launch_append<128, false>(p, s64, grid, stream);
  }
  return check_launch("paged_kv4_append");
}

extern "C" int qa_paged_kv4_gather(const qa_paged_kv* kv, int32_t head_dim, int64_t batch, const void* block_tables, int32_t table_dtype, int64_t table_stride,
                                   int64_t max_blocks, int64_t valid, int32_t block_size, void* key_out, void* value_out, hipStream_t stream) {
  using namespace qa;
  using namespace qa::kv4;
  if (int rc = check_pool("paged_kv4_gather", kv, head_dim, block_size)) return rc;
  QA_REQUIRE((block_tables != nullptr || batch == 0) && is_index_dtype(table_dtype), "block table must be an int32/int64 device array");
  QA_REQUIRE(batch >= 0 && batch <= 65535, "paged_kv4_gather: batch must be in [0, 65535]");
  QA_REQUIRE(max_blocks > 0 && table_stride >= 0, "paged_kv4_gather: max_blocks must be positive");
  QA_REQUIRE(valid >= 0 && valid <= 0x7fffffff, "paged_kv4_gather: valid out of range");
  if (valid == 0 || batch == 0) return 0;
  QA_REQUIRE(key_out && value_out && ((reinterpret_cast<uintptr_t>(key_out) | reinterpret_cast<uintptr_t>(value_out)) & 15u) == 0,
             "paged_kv4_gather: outputs must be non-null and 16-byte aligned");
  const int64_t gy = static_cast<int64_t>(kv->kv_heads) * (head_dim / 32 / kGatherGroups);
  QA_REQUIRE(gy <= 65535, "paged_kv4_gather: too many KV heads");
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
  const dim3 grid(static_cast<unsigned>(ceil_div(valid, 4 * kRun)), static_cast<unsigned>(gy), static_cast<unsigned>(batch));
  const bool t64 = table_dtype == QA_I64;
  {
    KernelTimer timer_("kv4_gather", stream);
    if (head_dim == 256) {
      if (t64)
        hipLaunchKernelGGL((gather_kernel<256, true>), grid, dim3(256), 0, stream, p);
      else
        hipLaunchKernelGGL((gather_kernel<256, false>), grid, dim3(256), 0, stream, p);
    } else {
      if (t64)
        hipLaunchKernelGGL((gather_kernel<128, true>), grid, dim3(256), 0, stream, p);
      else
        hipLaunchKernelGGL((gather_kernel<128, false>), grid, dim3(256), 0, stream, p);
    }
  }
  return check_launch("paged_kv4_gather");
}
