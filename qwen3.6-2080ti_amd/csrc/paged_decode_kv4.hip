// Decode attention over the 4-bit paged KV cache (attention_kv4.h, kv4.h), gfx950: one token per row.
//
// Bound by memory: 17 D / 32 bytes a cached token, KV head and K or V, each read once for the G query heads that share
// it.  All (row, KV head, unit of 32 tokens) are laid end to end, T units, and workgroup w of W takes the range
// [T w / W, T (w + 1) / W): equal shares whatever the lengths.  Inside a row group the workgroup's eight waves take its
// units in turn, so that neighbouring waves read neighbouring tiles, each with an online softmax of its own and no
// barrier; where the range leaves the row group they merge in LDS and write one partial (m, l, o) of the G heads.  A
// workgroup that had the whole row group writes the result; the other groups' partials are merged by combine_kernel.
//
// A wave loads a unit's keys and values two units ahead into registers (buffer loads of zero records for what is
// skipped, so every step issues the same loads and the wait counts are fixed).  Columns of the scores' product: with up
// to eight heads the first eight are the heads' hi pieces and the last eight their lo pieces, one product a slice, and a
// row rotation adds the two; with more the pieces take two products.
#include "attention_kv4.h"

#include <algorithm>

namespace qa {
namespace attn4 {

struct DecodeParams {
  Params c;
  int n_wgs;
  float* part_o;      // (n_wgs + B Hkv, G, D)
  float* part_ml;     // (n_wgs + B Hkv, G, 2)
  int32_t* rg_wgs;    // (B Hkv, 2): first and last workgroup of a row group; -1: the result is written
};

constexpr int kWaves = 8;
constexpr int kUnit = 32;  // tokens
constexpr int kMaxWgs = 256;  // one per CU: eight waves of up to 256 registers fill it

// Units of row b (0 for rows of length <= 0); lengths past the table stop at it.
__device__ __forceinline__ int64_t row_tokens(const Params& p, int b) {
  const int64_t len = p.idx_i64 ? reinterpret_cast<const int64_t*>(p.lens)[b] : reinterpret_cast<const int32_t*>(p.lens)[b];
  return max64(0, min64(len, p.max_blocks << p.bs_shift));
}
__device__ __forceinline__ int64_t row_units(const Params& p, int b) { return (row_tokens(p, b) + kUnit - 1) / kUnit; }

struct Cursor {
  int b, g;
  int64_t cum, nu;  // units before the row group, units of it
};

// Units of all row groups.
__device__ int64_t total_units(const Params& p, int lane) {
  int64_t sum = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) sum += b0 + lane < p.B ? row_units(p, b0 + lane) : 0;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
  return sum * p.Hkv;
}

// The row group that holds unit t < T.
__device__ Cursor locate(const Params& p, int64_t t, int lane) {
  int64_t base = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int64_t nu = b0 + lane < p.B ? row_units(p, b0 + lane) : 0;
    int64_t incl = nu * p.Hkv;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t up = __shfl_up(incl, off, 64);
      if (lane >= off) incl += up;
    }
    const int64_t chunk = __shfl(incl, 63, 64);
    if (t < base + chunk) {
      const int first = __ffsll(static_cast<unsigned long long>(__ballot(base + incl > t))) - 1;
      const int64_t n = __shfl(nu, first, 64);
      const int64_t before = base + __shfl(incl, first, 64) - n * p.Hkv;
      Cursor c;
      c.b = b0 + first;
      c.g = static_cast<int>((t - before) / n);
      c.cum = before + c.g * n;
      c.nu = n;
      return c;
    }
    base += chunk;
  }
  return Cursor{p.B, 0, base, 0};
}

template <int D, bool WIDE>
struct Smem {
  static constexpr int kHeads = WIDE ? 16 : 8;
  static constexpr int kRow = D + 4;  // floats: neighbouring heads start four banks apart
  static constexpr int kO = kWaves * kHeads * kRow;
  static constexpr int kBytes = (kO + 2 * kWaves * 16) * 4;
};

// WIDE: more than eight heads a group.
template <int D, bool WIDE>
__global__ __launch_bounds__(64 * kWaves, 2) void decode_kernel(DecodeParams dp) {
  const Params& p = dp.c;
  using S = Smem<D, WIDE>;
  constexpr int MT = D / 16;
  extern __shared__ __align__(16) float smem[];
  float* s_m = smem + S::kO;              // (kWaves, 16)
  float* s_l = s_m + kWaves * 16;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15;
  const int quad = lane >> 4;
  const int head = WIDE ? col : col & 7;

  const int64_t T = uniform64(total_units(p, lane));
  // a workgroup has a unit for each wave before another one starts
  const int64_t W = min64(dp.n_wgs, (T + kWaves - 1) / kWaves);
  const int64_t wg = blockIdx.x;
  if (wg >= W) return;
  const int64_t lo = T * wg / W;
  const int64_t hi = T * (wg + 1) / W;
  Cursor cur = locate(p, lo, lane);
  cur.b = __builtin_amdgcn_readfirstlane(cur.b);
  cur.g = __builtin_amdgcn_readfirstlane(cur.g);
  cur.cum = uniform64(cur.cum);
  cur.nu = uniform64(cur.nu);
  const float qk_scale = p.scale * kLog2e;

  for (int64_t at = lo; at < hi;) {
    const int64_t seg_end = min64(hi, cur.cum + cur.nu);
    const int64_t len = uniform64(row_tokens(p, cur.b));
    const int64_t runs = (len + kv4::kRun - 1) / kv4::kRun;
    const uint8_t* kb = p.kpool + cur.g * p.sG;
    const uint8_t* vb = p.vpool + cur.g * p.sG;
    const int64_t u1 = seg_end - cur.cum;  // end of the segment in the row group's units
    int64_t u = at - cur.cum + wave;

    KeyRun<D> kr[2][2];
    ValueRun<D> vr[2][2];
    int32_t phys[2][2];    // of the units in kr / vr
    int32_t ahead[2];      // of the unit after those
    auto entries = [&](int64_t unit, int32_t (&e)[2]) {
#pragma unroll
      for (int j = 0; j < 2; ++j) e[j] = unit < u1 ? block_of_run(p, cur.b, 2 * unit + j, runs) : -1;
    };
    auto fetch_keys = [&](int s, int64_t unit) {
#pragma unroll
      for (int j = 0; j < 2; ++j) load_keys<D>(kr[s][j], run_rsrc<D>(p, kb, phys[s][j], 2 * unit + j), lane);
    };
    auto fetch_values = [&](int s, int64_t unit) {
#pragma unroll
      for (int j = 0; j < 2; ++j) load_values<D>(vr[s][j], run_rsrc<D>(p, vb, phys[s][j], 2 * unit + j), lane);
    };
#pragma unroll
    for (int s = 0; s < 2; ++s) entries(u + s * kWaves, phys[s]);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      fetch_keys(s, u + s * kWaves);
      fetch_values(s, u + s * kWaves);
    }
    entries(u + 2 * kWaves, ahead);

    QueryCols<D> qa_, qb_;
    {
      QueryRow<D> row;
      row.load(head < p.G ? p.q + static_cast<int64_t>(cur.b) * p.q_st + static_cast<int64_t>(cur.g * p.G + head) * p.q_sh : nullptr, quad);
      row.template split<false>(qa_);
      row.template split<true>(qb_);
      if constexpr (!WIDE) {
        if (col >= 8) qa_ = qb_;
      }
    }
    float m_run = -INFINITY, l_run = 0.f;
    floatx4_v o[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i] = floatx4_v{0.f, 0.f, 0.f, 0.f};

    auto step = [&](int s) {
      // ---- scores: this lane's are tokens 4 quad + r of both runs, of head `head`
      float sc[8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        floatx4_v a = score<D>(kr[s][j], qa_, floatx4_v{0.f, 0.f, 0.f, 0.f});
        if constexpr (WIDE) a = score<D>(kr[s][j], qb_, a);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = a[r];
          if constexpr (!WIDE) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xF, 0xF, false));  // row_ror:8
          sc[4 * j + r] = x * qk_scale;
        }
      }
      // ---- what is not there: the last unit of a row, and blocks outside the pool
      const int64_t t0 = u * kUnit;
      if (!(t0 + kUnit <= len && phys[s][0] >= 0 && phys[s][1] >= 0)) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int64_t left = phys[s][j] < 0 ? 0 : len - t0 - kv4::kRun * j - 4 * quad;  // this lane's tokens that are there
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r >= left) sc[4 * j + r] = -INFINITY;
          // their values may be anything, and 0 times a NaN is one
          vr[s][j].scale &= left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * static_cast<int>(left))) - 1u;
        }
      }
      const int64_t next = u + 2 * kWaves;
#pragma unroll
      for (int j = 0; j < 2; ++j) phys[s][j] = ahead[j];
      fetch_keys(s, next);
      entries(next + kWaves, ahead);

      // ---- online softmax
      float mx = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
      if (__ballot(mx > m_run + kLazy) != 0) {
        const float m_new = fmaxf(m_run, column_max(mx));
        const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_run *= corr;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[i] *= corr;
      }
      const float use = m_run == -INFINITY ? 0.f : m_run;
      bf16x8_v pb;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float pr = __builtin_amdgcn_exp2f(sc[i] - use);
        l_run += pr;
        pb[i] = static_cast<__bf16>(pr);
      }
      // ---- values
      accumulate<D>(vr[s], pb, o);
      fetch_values(s, next);
      u += kWaves;
    };
    while (u < u1) {
      step(0);
      if (u >= u1) break;
      step(1);
    }

    // ---- merge the waves
    l_run = column_sum(l_run);
    if (quad == 0) {
      s_m[wave * 16 + col] = m_run;
      s_l[wave * 16 + col] = l_run;
    }
    __syncthreads();
    float big = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) big = fmaxf(big, s_m[w * 16 + col]);
    const float use = big == -INFINITY ? 0.f : big;
    const float f = __builtin_amdgcn_exp2f(m_run - use);
    if (col < S::kHeads && col < p.G) {
      float* so = smem + (wave * S::kHeads + col) * S::kRow;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < MT; i += 4)
          *reinterpret_cast<floatx4_v*>(so + (4 * quad + r) * MT + i) = floatx4_v{o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]} * f;
    }
    __syncthreads();
    const int64_t rg = static_cast<int64_t>(cur.b) * p.Hkv + cur.g;
    const bool whole = at == cur.cum && seg_end == cur.cum + cur.nu;
    const int64_t slot = wg + rg;
    for (int e = tid; e < p.G * D; e += 64 * kWaves) {
      const int h = e / D, d = e % D;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) m = fmaxf(m, s_m[w * 16 + h]);
      const float mu = m == -INFINITY ? 0.f : m;
      float sum = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        sum += smem[(w * S::kHeads + h) * S::kRow + d];
        l += s_l[w * 16 + h] * __builtin_amdgcn_exp2f(s_m[w * 16 + h] - mu);
      }
      if (whole) {
        const int64_t hq = cur.g * p.G + h;
        float r = normalised(sum, l);
        if (p.gate != nullptr) r *= sigmoid(bf16_to_f32(p.gate[cur.b * p.gate_st + hq * p.gate_sh + d]));
        p.out[(static_cast<int64_t>(cur.b) * p.H + hq) * D + d] = f32_to_bf16(r);
      } else {
        dp.part_o[(slot * p.G + h) * D + d] = sum;
        if (d == 0) *reinterpret_cast<float2*>(dp.part_ml + (slot * p.G + h) * 2) = make_float2(m, l);
      }
    }
    if (tid == 0) {
      if (at == cur.cum) dp.rg_wgs[2 * rg] = whole ? -1 : static_cast<int32_t>(wg);
      if (seg_end == cur.cum + cur.nu) dp.rg_wgs[2 * rg + 1] = static_cast<int32_t>(wg);
    }
    at = seg_end;
    if (at < hi) {
      __syncthreads();  // smem is written again
      cur.cum += cur.nu;
      if (++cur.g == p.Hkv) {
        cur.g = 0;
        do {
          ++cur.b;
          cur.nu = cur.b < p.B ? uniform64(row_units(p, cur.b)) : 0;
        } while (cur.nu == 0 && cur.b < p.B);
      }
    }
  }
}

// Merges the partials of one (row, head): slots first + rg .. last + rg.  A workgroup of THREADS, each thread a dim of
// every (THREADS / D)-th partial with up to kRowsInFlight loads in flight.
constexpr int kRowsInFlight = 16;

template <int D, int THREADS>
__global__ __launch_bounds__(THREADS) void combine_kernel(DecodeParams dp) {
  const Params& p = dp.c;
  constexpr int SHARE = THREADS / D;
  __shared__ float s_f[kMaxWgs];
  __shared__ float s_red[2][THREADS / 64];
  __shared__ float s_o[SHARE][D];
  const int tid = threadIdx.x;
  const int64_t bh = blockIdx.x;
  const int b = static_cast<int>(bh / p.H);
  const int h = static_cast<int>(bh - static_cast<int64_t>(b) * p.H);
  const int g = h / p.G;
  const int hh = h - g * p.G;
  const int64_t rg = static_cast<int64_t>(b) * p.Hkv + g;
  const int first = dp.rg_wgs[2 * rg], last = dp.rg_wgs[2 * rg + 1];
  bf16_t* out = p.out + bh * D;
  if (row_tokens(p, b) == 0) {  // its record was never written
    if (tid < D) out[tid] = 0;
    return;
  }
  if (first < 0) return;
  const int n = last - first + 1;
  const int64_t row0 = (first + rg) * p.G + hh;
  const int d = tid % D, share = tid / D;
  const float* po = dp.part_o + row0 * D + d;
  const int64_t so = static_cast<int64_t>(p.G) * D;
  float pre[kRowsInFlight];
#pragma unroll
  for (int i = 0; i < kRowsInFlight; ++i) pre[i] = share + i * SHARE < n ? po[(share + i * SHARE) * so] : 0.f;
  float2 ml = make_float2(-INFINITY, 0.f);
  if (tid < n) ml = *reinterpret_cast<const float2*>(dp.part_ml + (row0 + static_cast<int64_t>(tid) * p.G) * 2);
  const float wm = wave_max(ml.x);
  if ((tid & 63) == 0) s_red[0][tid >> 6] = wm;
  __syncthreads();
  float m = s_red[0][0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) m = fmaxf(m, s_red[0][w]);
  const float use = m == -INFINITY ? 0.f : m;
  const float f = tid < n ? __builtin_amdgcn_exp2f(ml.x - use) : 0.f;
  if (tid < n) s_f[tid] = f;
  const float wl = wave_sum(tid < n ? f * ml.y : 0.f);
  if ((tid & 63) == 0) s_red[1][tid >> 6] = wl;
  __syncthreads();
  float acc = 0.f;
#pragma unroll
  for (int i = 0; i < kRowsInFlight; ++i)
    if (share + i * SHARE < n) acc += s_f[share + i * SHARE] * pre[i];
  for (int s0 = share + kRowsInFlight * SHARE; s0 < n; s0 += kRowsInFlight * SHARE) {
    float row[kRowsInFlight];
#pragma unroll
    for (int i = 0; i < kRowsInFlight; ++i) row[i] = s0 + i * SHARE < n ? po[(s0 + i * SHARE) * so] : 0.f;
#pragma unroll
    for (int i = 0; i < kRowsInFlight; ++i)
      if (s0 + i * SHARE < n) acc += s_f[s0 + i * SHARE] * row[i];
  }
  if constexpr (SHARE > 1) {
    s_o[share][d] = acc;
    __syncthreads();
    if (share != 0) return;
#pragma unroll
    for (int i = 1; i < SHARE; ++i) acc += s_o[i][d];
  }
  float l = 0.f;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) l += s_red[1][w];
  float r = normalised(acc, l);
  if (p.gate != nullptr) r *= sigmoid(bf16_to_f32(p.gate[b * p.gate_st + h * p.gate_sh + d]));
  out[d] = f32_to_bf16(r);
}

// Workgroups of a launch: as many as there could be units for, up to one a CU.
static int64_t decode_wgs(int64_t row_groups, int64_t max_tokens) {
  return std::min<int64_t>(kMaxWgs, std::max<int64_t>(1, ceil_div(row_groups * ceil_div(std::max<int64_t>(max_tokens, 1), kUnit), kWaves)));
}

static int64_t workspace_bytes_of(int64_t batch, int heads, int kv_heads, int head_dim, int64_t max_tokens) {
  const int64_t groups = batch * kv_heads;
  return (decode_wgs(groups, max_tokens) + groups) * (heads / kv_heads) * (head_dim + 2) * 4 + groups * 8;
}

template <int D, bool WIDE>
static int launch(const DecodeParams& p, hipStream_t stream) {
  using S = Smem<D, WIDE>;
  const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(&decode_kernel<D, WIDE>), hipFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
  if (err != hipSuccess) return fail("paged_attention_decode_kv4: cannot reserve %d bytes of LDS: %s", S::kBytes, hipGetErrorString(err));
  {
    KernelTimer timer_("decode_kv4", stream);
    hipLaunchKernelGGL((decode_kernel<D, WIDE>), dim3(p.n_wgs), dim3(64 * kWaves), S::kBytes, stream, p);
  }
  if (int rc = check_launch("paged_attention_decode_kv4")) return rc;
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(p.c.B) * p.c.H));
  // many partials a row group: 1024 threads share them, so that fewer rounds of loads follow one another
  const bool many = p.n_wgs > 16 * static_cast<int64_t>(p.c.B) * p.c.Hkv;
  {
    KernelTimer timer_("decode_kv4_combine", stream);
    if (many)
      hipLaunchKernelGGL((combine_kernel<D, 1024>), grid, dim3(1024), 0, stream, p);
    else
      hipLaunchKernelGGL((combine_kernel<D, 256>), grid, dim3(256), 0, stream, p);
  }
  return check_launch("paged_attention_decode_kv4");
}

}  // namespace attn4
}  // namespace qa

extern "C" int64_t qa_paged_attention_decode_kv4_workspace(int64_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim, int64_t max_tokens) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_tokens < 0) return 0;
  return qa::attn4::workspace_bytes_of(batch, heads, kv_heads, head_dim, max_tokens);
}

extern "C" int qa_paged_attention_decode_kv4(const void* query, int32_t q_dtype, int64_t q_stride_b, int64_t q_stride_h, int64_t batch, int32_t heads,
                                             int32_t head_dim, const qa_paged_kv* kv, const void* block_tables, int32_t table_dtype, int64_t table_stride,
                                             int64_t max_blocks, const void* sequence_lengths, int32_t lengths_dtype, int32_t block_size, float scale,
                                             const void* gate, int64_t gate_stride_b, int64_t gate_stride_h, void* output, void* workspace,
                                             int64_t workspace_bytes, hipStream_t stream) {
  using namespace qa;
  using namespace qa::attn4;
  DecodeParams p{};
  const Args a{"paged_attention_decode_kv4", query, q_dtype, q_stride_b, q_stride_h, batch, heads, head_dim, kv, block_tables, table_dtype, table_stride, max_blocks,
               lengths_dtype, block_size, scale, gate, gate_stride_b, gate_stride_h, output};
  if (int rc = fill(p.c, a)) return rc;
  if (batch == 0) return 0;
  QA_REQUIRE(sequence_lengths != nullptr, "sequence_lengths must be a device array");
  QA_REQUIRE(batch * heads <= 0x7fffffff, "%s: batch * heads out of range", a.what);
  p.c.lens = sequence_lengths;
  const int64_t groups = batch * kv->kv_heads;
  const int64_t max_tokens = max_blocks * block_size;
  const int64_t need = workspace_bytes_of(batch, heads, kv->kv_heads, head_dim, max_tokens);
  QA_REQUIRE(workspace != nullptr && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0,
             "paged decode workspace too small or not 16-byte aligned: need %lld bytes, have %lld", static_cast<long long>(need), static_cast<long long>(workspace_bytes));
  p.n_wgs = static_cast<int>(decode_wgs(groups, max_tokens));
  const int64_t rows = (p.n_wgs + groups) * p.c.G;
  p.part_o = reinterpret_cast<float*>(workspace);
  p.part_ml = p.part_o + rows * head_dim;
  p.rg_wgs = reinterpret_cast<int32_t*>(p.part_ml + rows * 2);
  if (head_dim == 256) return p.c.G > 8 ? launch<256, true>(p, stream) : launch<256, false>(p, stream);
  return p.c.G > 8 ? launch<128, true>(p, stream) : launch<128, false>(p, stream);
}
