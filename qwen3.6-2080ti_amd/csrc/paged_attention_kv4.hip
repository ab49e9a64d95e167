// Attention over the 4-bit paged KV cache (kv4.h), gfx950: one token per row, or packed new tokens of a step.
//
//   out[n][h] = softmax_t(scale q[n][h] . k[t][g]) v[t][g]  (* sigmoid(gate[n][h])),  g = h / (H / H_kv),
// over the cached tokens t that the query sees: t < length of its row (decode), t <= its own position (prefill).
// Tokens of blocks outside the pool are skipped; a query that sees nothing gives zeros.
//
// One wave per (token, head).  Lane t of a tile of 64 keys takes one key: its codes of a group are 16 consecutive
// bytes, and 16 lanes read 256 consecutive bytes.  The probabilities go through LDS, then lane l owns dims
// l D/64 .. of the output and walks the tile's tokens.
#include "kv4.h"

namespace qa {
namespace simple4 {

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
  int H, Hkv, bs_shift, table_i64, idx_i64;
  float scale;
};

__device__ __forceinline__ int64_t read_index(const void* base, int is64, int64_t i) {
  return is64 ? reinterpret_cast<const int64_t*>(base)[i] : reinterpret_cast<const int32_t*>(base)[i];
}

__device__ __forceinline__ float code_value(uint32_t c) {
  const uint32_t m = c & 7u;
  const float v = m < 2u ? 0.5f * static_cast<float>(m) : __uint_as_float(((m >> 1) + 126u) << 23 | (m & 1u) << 22);
  return c & 8u ? -v : v;
}

__device__ __forceinline__ float scale_value(uint32_t byte) { return byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23); }

template <int D>
__global__ __launch_bounds__(64) void simple_kernel(Params p) {
  using R = kv4::Run<D>;
  constexpr int E = D / 64;
  __shared__ float s_q[D];
  __shared__ float s_p[64];
  __shared__ int64_t s_run[64];
  const int lane = threadIdx.x;
  const int h = blockIdx.y % p.H;
  const int64_t b = blockIdx.y / p.H;
  int64_t n, len;
  if (p.cu != nullptr) {
    const int64_t lo = read_index(p.cu, p.idx_i64, b), hi = min64(read_index(p.cu, p.idx_i64, b + 1), p.total);
    n = lo + blockIdx.x;
    if (lo < 0 || n >= hi) return;
    len = read_index(p.prefix, p.idx_i64, b) + blockIdx.x + 1;
  } else {
    n = b;
    len = read_index(p.lens, p.idx_i64, b);
  }
  len = min64(len, p.max_blocks << p.bs_shift);
  const int g = h / (p.H / p.Hkv);
  for (int d = lane; d < D; d += 64) s_q[d] = bf16_to_f32(p.q[n * p.q_st + h * p.q_sh + d]) * p.scale;
  __syncthreads();
  float m_run = -INFINITY, l_run = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int64_t t0 = 0; t0 < len; t0 += 64) {
    const int64_t t = t0 + lane;
    int64_t run = -1;
    if (t < len) {
      const int64_t phys = read_index(p.tables, p.table_i64, b * p.table_stride + (t >> p.bs_shift));
      if (phys >= 0 && phys < p.num_blocks) run = phys * p.sP + g * p.sG + ((t & ((1 << p.bs_shift) - 1)) >> 4) * R::kBytes;
    }
    float sc = -INFINITY;
    if (run >= 0) {
      sc = 0.f;
      for (int gr = 0; gr < R::kGroups; ++gr) {
        const uint4 u = *reinterpret_cast<const uint4*>(p.kpool + run + R::key_code(t & 15, gr));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) part += code_value(w[i / 8] >> (4 * (i % 8)) & 15u) * s_q[gr * 32 + i];
        sc += part * scale_value(p.kpool[run + R::key_scale(t & 15, gr)]);
      }
    }
    const float m_new = fmaxf(m_run, wave_max(sc));
    const float use = m_new == -INFINITY ? 0.f : m_new;
    const float corr = __expf(m_run - use);
    const float pr = __expf(sc - use);
    m_run = m_new;
    l_run = l_run * corr + wave_sum(pr);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= corr;
    s_p[lane] = pr;
    s_run[lane] = run;
    __syncthreads();
    const int cnt = static_cast<int>(min64(64, len - t0));
    for (int i = 0; i < cnt; ++i) {
      if (s_run[i] < 0) continue;
      const uint8_t* v = p.vpool + s_run[i];
      const int tt = static_cast<int>((t0 + i) & 15);
      const float sv = scale_value(v[R::value_scale(tt, lane * E / 32)]) * s_p[i];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = lane * E + e;
        const uint32_t byte = v[R::value_code(tt, d / (D / 16)) + d % (D / 16) / 2];
        o[e] += sv * code_value(d & 1 ? byte >> 4 : byte & 15u);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float r = l_run > 0.f ? o[e] / l_run : l_run == 0.f ? 0.f : l_run;  // a NaN stays one
    const int d = lane * E + e;
    if (p.gate != nullptr) r *= 1.f / (1.f + __expf(-bf16_to_f32(p.gate[n * p.gate_st + h * p.gate_sh + d])));
    p.out[(n * p.H + h) * D + d] = f32_to_bf16(r);
  }
}

struct Args {
  const char* what;
  const void* query;
  int32_t q_dtype;
  int64_t q_st, q_sh;
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

static int fill(Params& p, const Args& a) {
  if (int rc = kv4::check_pool(a.what, a.kv, a.head_dim, a.block_size)) return rc;
  QA_REQUIRE(a.q_dtype == QA_BF16, "%s: query must be bfloat16", a.what);
  QA_REQUIRE(is_index_dtype(a.table_dtype) && is_index_dtype(a.idx_dtype), "%s: index arrays must be int32/int64", a.what);
  QA_REQUIRE(a.batch >= 0 && a.batch <= 0x7fffffff, "%s: batch out of range", a.what);
  QA_REQUIRE(a.heads > 0 && a.heads % a.kv->kv_heads == 0, "%s: query heads (%d) must be a multiple of KV heads (%d)", a.what, a.heads, a.kv->kv_heads);
  QA_REQUIRE(a.heads / a.kv->kv_heads <= 16, "%s: GQA group size %d is larger than 16", a.what, a.heads / a.kv->kv_heads);
  QA_REQUIRE(a.max_blocks > 0 && a.max_blocks <= 0x7fffffff && a.table_stride >= 0, "%s: block table must have at least one entry", a.what);
  if (a.batch > 0) QA_REQUIRE(a.query && a.out && a.tables, "%s: pointers must be non-null", a.what);
  QA_REQUIRE(((reinterpret_cast<uintptr_t>(a.query) | reinterpret_cast<uintptr_t>(a.out)) & 15u) == 0 && a.q_st % 8 == 0 && a.q_sh % 8 == 0,
             "%s: query rows must be 16-byte aligned", a.what);
  QA_REQUIRE(a.gate == nullptr || ((reinterpret_cast<uintptr_t>(a.gate) & 7u) == 0 && a.gate_st % 4 == 0 && a.gate_sh % 4 == 0), "%s: gate rows must be 8-byte aligned", a.what);
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
  p.H = a.heads;
  p.Hkv = a.kv->kv_heads;
  p.bs_shift = __builtin_ctz(static_cast<unsigned>(a.block_size));
  p.table_i64 = a.table_dtype == QA_I64;
  p.idx_i64 = a.idx_dtype == QA_I64;
  p.scale = a.scale > 0.f ? a.scale : 1.0f / sqrtf(static_cast<float>(a.head_dim));
  return 0;
}

static int launch(const Params& p, int D, int64_t x, int64_t y, const char* what, hipStream_t stream) {
  QA_REQUIRE(y <= 65535, "%s: batch * heads must fit 65535", what);
  const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>(y));
  if (D == 256)
    hipLaunchKernelGGL(simple_kernel<256>, grid, dim3(64), 0, stream, p);
  else
    hipLaunchKernelGGL(simple_kernel<128>, grid, dim3(64), 0, stream, p);
  return check_launch(what);
}

}  // namespace simple4
}  // namespace qa

extern "C" int qa_paged_attention_prefill_kv4(const void* query, int32_t q_dtype, int64_t q_stride_t, int64_t q_stride_h, int64_t total_new, const void* cu_seqlens,
                                              const void* prefix_lens, int32_t idx_dtype, int64_t batch, int64_t max_new, int32_t heads, int32_t head_dim,
                                              const qa_paged_kv* kv, const void* block_tables, int32_t table_dtype, int64_t table_stride, int64_t max_blocks,
                                              int32_t block_size, float scale, const void* gate, int64_t gate_stride_t, int64_t gate_stride_h, void* output,
                                              hipStream_t stream) {
  using namespace qa;
  using namespace qa::simple4;
  Params p{};
  const Args a{"paged_attention_prefill_kv4", query, q_dtype, q_stride_t, q_stride_h, batch, heads, head_dim, kv, block_tables, table_dtype, table_stride, max_blocks,
               idx_dtype, block_size, scale, gate, gate_stride_t, gate_stride_h, output};
  if (int rc = fill(p, a)) return rc;
  QA_REQUIRE(total_new >= 0 && total_new <= 0x7fffffff && max_new >= 0 && max_new <= 0x7fffffff, "%s: token counts out of range", a.what);
  if (batch == 0 || max_new == 0 || total_new == 0) return 0;
  QA_REQUIRE(cu_seqlens && prefix_lens, "%s: pointers must be non-null", a.what);
  p.cu = cu_seqlens;
  p.prefix = prefix_lens;
  p.total = total_new;
  return launch(p, head_dim, max_new, batch * heads, a.what, stream);
}
