// Decode attention over the 8-bit paged KV cache (attention_kv8.h, kv8.h), gfx950: one token per row.
//
// Bound by memory: D + 1 bytes a cached token, KV head and K or V, each read once for the G query heads that share it.  The
// shares are those of decode_split.h: all (row, KV head, unit of 32 tokens) laid end to end, an equal range of them for each
// workgroup, its eight waves taking units in turn, each with an online softmax of its own and no barrier; where the range
// leaves a row group they merge in LDS and write one partial (m, l, o) of the G heads, or the result where the workgroup had
// the whole row group.  Where all rows are short a workgroup takes a row group as it is.
//
// A wave asks for the next unit's keys when the scores have used this one's, and for its values when the products have: so
// three quarters of a unit of each of eight waves are on their way all the time, across row groups.  Buffer loads of zero
// records stand for what is skipped, so every step issues the same loads and the wait counts are fixed.  Lane j of a wave holds where unit j
// of its next 64 lies; one search and one vector load of the tables serve them all, and a step reads its lane.  The columns of the
// products are the heads, up to 16 of a group.
//
// 64 rows of 1k to 32k tokens, two KV heads of 256: 159 us for 994 MB, 6.2 TB/s (what a pure reader reaches), and 4.7 to merge; one
// row of 200k, a head of 128: 12.8 + 3.8; four of 300 to 700: 10.4, all latency.
#include "attention_kv8.h"
#include "decode_split.h"

namespace qa {
namespace attn8 {

// Where no row is longer than this, a workgroup takes a row group and nothing is merged; where the tables cannot hold a
// longer one, the second launch is left out.  us on the GPU split / by row, 2 KV heads of 256: 4 rows of 512 9.4 / 9.4, of 1024 13.1 /
// 16.0, of 2048 12.6 / 24.1; 64 rows of 500 11.5 / 11.5, of 1024 22.2 / 18.7, of 2048 32.0 / 31.5; 200 of 500 27.4 / 25.6.  The host
// takes 17 us for a split call and 12.5 for the other.
constexpr int kByRowTokens = 1024;
// Row groups up to which a call of long tables has the workgroups for that; each of them reads all the lengths first.  us
// split / by row, rows of 300 tokens, 2 KV heads: 100 rows 24.6 / 12.7, 200 37.5 / 24.3, 500 71.2 / 56.3, 1000 130.9 / 129.6, 2000
// 249.7 / 321.7.
constexpr int kByRowGroups = 2048;

template <int D>
struct Smem {
  static constexpr int kHeads = 16;
  static constexpr int kRow = D + 4;                      // floats: neighbouring heads start four banks apart
  static constexpr int kM = kWaves * kHeads * kRow * 4;   // after the waves' sums: (kWaves, 16) reference points,
  static constexpr int kL = kM + kWaves * 16 * 4;         // (kWaves, 16) denominators,
  static constexpr int kTotal = kL + kWaves * 16 * 4;     // the merged ones (2, 16)
  static constexpr int kBytes = kTotal + 2 * 16 * 4;
};

template <int D>
__global__ __launch_bounds__(64 * kWaves, 2) void decode_kernel(DecodeParams dp) {
  const Params& p = dp.c;
  using S = Smem<D>;
  constexpr int MT = D / 16;
  extern __shared__ __align__(16) unsigned char smem[];
  float* s_o = reinterpret_cast<float*>(smem);
  float* s_m = reinterpret_cast<float*>(smem + S::kM);
  float* s_l = reinterpret_cast<float*>(smem + S::kL);
  float* s_total = reinterpret_cast<float*>(smem + S::kTotal);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15;
  const int quad = lane >> 4;

  // ---- this workgroup's share: units lo .. hi - 1
  const int wg = blockIdx.x;
  Cursor cur{0, 0, 0, 0};
  int lo = 0, hi;
  int64_t len_first = 0;  // rows of up to 64 are loaded and summed once, for the total and for the search below
  int incl_first = 0, T = 0;
  bool by_row = dp.short_rows != 0;
  if (!by_row) {
    uint32_t longest = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      const int64_t len = b0 + lane < p.B ? row_tokens(p, b0 + lane) : 0;
      const int nu = units_of(len);
      const int incl = lane_scan(nu * p.Hkv);
      T += __builtin_amdgcn_readlane(incl, 63);
      longest = max(longest, wave_max_bits(nu));
      if (b0 == 0) {
        len_first = len;
        incl_first = incl;
      }
    }
    by_row = longest <= kByRowTokens / kUnit && static_cast<int64_t>(p.B) * p.Hkv <= kByRowGroups;
  }
  if (by_row) {
    cur.b = wg / p.Hkv;
    cur.g = wg - cur.b * p.Hkv;
    if (cur.b >= p.B) return;
    len_first = row_tokens(p, cur.b);
    cur.nu = __builtin_amdgcn_readfirstlane(units_of(len_first));
    hi = cur.nu;
    if (hi == 0) {
      for (int e = 4 * tid; e < p.G * D; e += 4 * 64 * kWaves) *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(cur.b) * p.H + cur.g * p.G) * D + e) = make_uint2(0, 0);
      return;
    }
  } else {
    // a workgroup has a unit for each wave before another one starts
    const int W = min(dp.n_wgs, (T + kWaves - 1) / kWaves);
    if (wg >= W) return;
    lo = static_cast<int>(static_cast<int64_t>(T) * wg / W);
    hi = static_cast<int>(static_cast<int64_t>(T) * (wg + 1) / W);
  }

  // ---- where the wave's units lie: lane j holds unit 64 c + j, that is unit lo + wave + kWaves (64 c + j) of all
  int64_t at0, at1;  // offsets of its two runs in the pools, -1: not there
  int left;          // its tokens
  auto locate = [&](int c, bool begin) {
    const int gu = lo + wave + kWaves * (64 * c + lane);
    int row = -1, g = 0, u = 0;
    int64_t tokens = 0;
    int base = 0;
    if (by_row) {
      row = cur.b;
      g = cur.g;
      u = gu;
      tokens = len_first;
    }
    for (int b0 = 0; b0 < p.B && !by_row; b0 += 64) {
      const int64_t len = b0 == 0 ? len_first : b0 + lane < p.B ? row_tokens(p, b0 + lane) : 0;
      const int nu = units_of(len);
      const int incl = b0 == 0 ? incl_first : lane_scan(nu * p.Hkv);
      const int chunk = __builtin_amdgcn_readlane(incl, 63);
      if (begin && lo >= base && lo < base + chunk) {
        const int first = __ffsll(static_cast<unsigned long long>(__ballot(base + incl > lo))) - 1;
        cur.b = b0 + first;
        cur.nu = __builtin_amdgcn_readlane(nu, first);
        const int before = base + __builtin_amdgcn_readlane(incl, first) - cur.nu * p.Hkv;
        cur.g = (lo - before) / cur.nu;
        cur.cum = before + cur.g * cur.nu;
      }
      int pos = 0;  // rows of the block that end at or before gu
      const int rows = min(63, p.B - b0);
      for (int r = 0; r < rows; ++r) pos += base + __builtin_amdgcn_readlane(incl, r) <= gu;
      const int n = __shfl(nu, pos, 64);
      const int before = base + __shfl(incl, pos, 64) - n * p.Hkv;
      const int64_t t = (static_cast<int64_t>(__shfl(static_cast<int>(len >> 32), pos, 64)) << 32) | static_cast<uint32_t>(__shfl(static_cast<int>(len), pos, 64));
      if (gu >= base && gu < base + chunk) {
        row = b0 + pos;
        g = (gu - before) / n;
        u = gu - before - g * n;
        tokens = t;
      }
      base += chunk;
      if (base >= hi) break;
    }
    at0 = at1 = -1;
    left = 0;
    if (gu < hi && row >= 0) {
      left = static_cast<int>(min64(kUnit, tokens - static_cast<int64_t>(u) * kUnit));
      const int sub_shift = p.bs_shift - 4;
      auto offset = [&](int64_t run) -> int64_t {
        const int64_t e = (static_cast<int64_t>(row) * p.table_stride + (run >> sub_shift)) << p.table_i64;
        const int32_t id = reinterpret_cast<const int32_t*>(p.tables)[e];
        const int32_t high = reinterpret_cast<const int32_t*>(p.tables)[e + p.table_i64];  // the entry itself where it has one word
        const bool ok = (static_cast<uint32_t>(id) < static_cast<uint32_t>(p.num_blocks)) & ((high == 0) | (p.table_i64 == 0));
        return ok ? static_cast<int64_t>(id) * p.sP + (run & ((1 << sub_shift) - 1)) * kv8::Run<D>::kBytes + g * p.sG : -1;
      };
      at0 = offset(2 * static_cast<int64_t>(u));
      if (left > kv8::kRun) at1 = offset(2 * static_cast<int64_t>(u) + 1);
    }
  };
  locate(0, true);

  constexpr int N = kv8::Run<D>::kSlices;
  uint4 kr[2][N], vr[2][N];   // codes of the unit's two runs
  uint32_t kscale[2], vscale[2];
  int64_t where[2];  // of the unit being asked for
  int have, next;    // tokens of the unit at hand and of the one asked for, and 256 / 512 where the first / second run is not there
  auto look = [&](int i) {
    const int j = i & 63;
    auto read = [&](int64_t v) {
      const uint32_t l = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), j), h = __builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), j);
      return static_cast<int64_t>(static_cast<uint64_t>(h) << 32 | l);
    };
    where[0] = read(at0);
    where[1] = read(at1);
    next = __builtin_amdgcn_readlane(left, j) | (where[0] < 0 ? 256 : 0) | (where[1] < 0 ? 512 : 0);
  };
  auto fetch = [&](const uint8_t* base, uint4 (&codes)[2][N], uint32_t (&scale)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t o = where[j];
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base + (o < 0 ? 0 : o)), 0, o < 0 ? 0 : kv8::Run<D>::kBytes, 0x00020000);
#pragma unroll
      for (int s = 0; s < N; ++s) codes[j][s] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, 16 * lane + 1024 * s, 0, kOnce));
      scale[j] = __builtin_amdgcn_raw_buffer_load_b8(r, kv8::Run<D>::kCodes, 0, kOnce);
    }
  };

  // ---- the query of a row group: lane 16 q + n has dims 64 s + 16 q .. + 15 of head n, as the keys' lanes have them
  bf16x8_v q[2 * N];
  auto fetch_query = [&](const Cursor& c) {
    const bool there = col < p.G && c.b < p.B;
    const uint4* row = reinterpret_cast<const uint4*>(p.q + (there ? static_cast<int64_t>(c.b) * p.q_st + static_cast<int64_t>(c.g * p.G + col) * p.q_sh + 16 * quad : 0));
#pragma unroll
    for (int s = 0; s < N; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (there) u = row[8 * s + e];
        q[2 * s + e] = __builtin_bit_cast(bf16x8_v, u);
      }
  };
  fetch_query(cur);  // before the tiles: loads are waited for in their order
  look(0);
  fetch(p.kpool, kr, kscale);
  fetch(p.vpool, vr, vscale);
  const float qk_scale = p.scale * kLog2e;

  int i = 0;                // the wave's next unit
  int gu = lo + wave;       // that unit among all
  for (int at = lo; at < hi;) {
    const int seg_end = min(hi, cur.cum + cur.nu);
    Cursor nxt = cur;
    if (seg_end < hi) next_row_group(p, nxt);

    float m_run = -INFINITY, l_run = 0.f;
    floatx4_v o[MT];
#pragma unroll
    for (int k = 0; k < MT; ++k) o[k] = floatx4_v{0.f, 0.f, 0.f, 0.f};

    for (; gu < seg_end; gu += kWaves) {
      have = next;
      ++i;
      if ((i & 63) == 0) locate(i >> 6, false);
      look(i);
      // ---- scores: this lane's are tokens 4 quad + r of both runs, of head col
      float sc[8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        floatx4_v a = {0.f, 0.f, 0.f, 0.f};
        const float scale = kv8::scale_of(kscale[j]);
#pragma unroll
        for (int s = 0; s < N; ++s) {
          a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(kr[j][s].x, kr[j][s].y, scale, scale), q[2 * s], a, 0, 0, 0);
          a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(kr[j][s].z, kr[j][s].w, scale, scale), q[2 * s + 1], a, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[4 * j + r] = a[r] * qk_scale;
      }
      fetch(p.kpool, kr, kscale);
      // ---- what is not there: the last unit of a row, and blocks outside the pool
      if (have != kUnit) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int mine = (have >> (8 + j) & 1) ? 0 : (have & 255) - kv8::kRun * j - 4 * quad;  // this lane's tokens that are there
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r >= mine) sc[4 * j + r] = -INFINITY;
          // their values may be anything, and 0 times a NaN is one
          const uint32_t mask = tokens_mask(mine);
#pragma unroll
          for (int s = 0; s < N; ++s) {
            vr[j][s].x &= mask;
            vr[j][s].y &= mask;
            vr[j][s].z &= mask;
            vr[j][s].w &= mask;
          }
        }
      }

      // ---- online softmax
      float mx = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
      if (__ballot(mx > m_run + kLazy) != 0) {
        const float m_new = fmaxf(m_run, column_max(mx));
        const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_run *= corr;
#pragma unroll
        for (int k = 0; k < MT; ++k) o[k] *= corr;
      }
      const float use = m_run == -INFINITY ? 0.f : m_run;
      bf16x8_v pb;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float pr = __builtin_amdgcn_exp2f(sc[k] - use);
        l_run += pr;
        pb[k] = static_cast<__bf16>(pr);  // for the bf16 product; l_run has it unrounded
      }
      // ---- values: o[4 s + m] has row 4 quad + r = dim 64 s + 16 quad + 4 r + m
      const float s0 = kv8::scale_of(vscale[0]), s1 = kv8::scale_of(vscale[1]);
#pragma unroll
      for (int s = 0; s < N; ++s)
#pragma unroll
        for (int m = 0; m < 4; ++m)
          o[4 * s + m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(dword(vr[0][s], m), dword(vr[1][s], m), s0, s1), pb, o[4 * s + m], 0, 0, 0);
      fetch(p.vpool, vr, vscale);
    }
    if (seg_end < hi) fetch_query(nxt);  // of the next row group

    // ---- merge the waves
    l_run = column_sum(l_run);
    if (quad == 0) {
      s_m[wave * 16 + col] = m_run;
      s_l[wave * 16 + col] = l_run;
    }
    __syncthreads();
    float big = -INFINITY;
    float wm[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      wm[w] = s_m[w * 16 + col];
      big = fmaxf(big, wm[w]);
    }
    const float use = big == -INFINITY ? 0.f : big;
    if (wave == 0 && quad == 0) {
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) l += s_l[w * 16 + col] * __builtin_amdgcn_exp2f(wm[w] - use);
      s_total[col] = big;
      s_total[16 + col] = l;
    }
    const float f = __builtin_amdgcn_exp2f(m_run - use);
    if (col < S::kHeads && col < p.G) {
      float* so = s_o + (wave * S::kHeads + col) * S::kRow;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int s = 0; s < N; ++s)
          *reinterpret_cast<floatx4_v*>(so + 64 * s + 16 * quad + 4 * r) = floatx4_v{o[4 * s][r], o[4 * s + 1][r], o[4 * s + 2][r], o[4 * s + 3][r]} * f;
    }
    __syncthreads();
    const int64_t rg = static_cast<int64_t>(cur.b) * p.Hkv + cur.g;
    const bool whole = at == cur.cum && seg_end == cur.cum + cur.nu;
    const int64_t slot = wg + rg;
    for (int e = 4 * tid; e < p.G * D; e += 4 * 64 * kWaves) {
      const int h = e / D, d = e % D;
      const float l = s_total[16 + h];
      const int64_t hq = cur.g * p.G + h;
      uint2 gate = make_uint2(0, 0);
      if (whole && p.gate != nullptr) gate = *reinterpret_cast<const uint2*>(p.gate + cur.b * p.gate_st + hq * p.gate_sh + d);
      floatx4_v sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) sum += *reinterpret_cast<const floatx4_v*>(s_o + (w * S::kHeads + h) * S::kRow + d);
      if (whole) {
        float r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          r[k] = normalised(sum[k], l);
          if (p.gate != nullptr) {
            const uint32_t w = k < 2 ? gate.x : gate.y;
            r[k] *= sigmoid(__uint_as_float(k & 1 ? w & 0xffff0000u : w << 16));
          }
        }
        uint2 packed;
        packed.x = static_cast<uint32_t>(f32_to_bf16(r[0])) | static_cast<uint32_t>(f32_to_bf16(r[1])) << 16;
        packed.y = static_cast<uint32_t>(f32_to_bf16(r[2])) | static_cast<uint32_t>(f32_to_bf16(r[3])) << 16;
        *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(cur.b) * p.H + hq) * D + d) = packed;
      } else {
        *reinterpret_cast<floatx4_v*>(dp.part_o + (slot * p.G + h) * D + d) = sum;
        if (d == 0) *reinterpret_cast<float2*>(dp.part_ml + (slot * p.G + h) * 2) = make_float2(s_total[h], l);
      }
    }
    if (tid == 0 && !dp.short_rows) {
      if (at == cur.cum) dp.rg_wgs[2 * rg] = whole ? -1 : wg;
      if (seg_end == cur.cum + cur.nu) dp.rg_wgs[2 * rg + 1] = wg;
    }
    at = seg_end;
    cur = nxt;
  }
}

template <int D>
static int launch(const DecodeParams& p, hipStream_t stream) {
  if (int rc = reserve_lds<&decode_kernel<D>>("paged_attention_decode_kv8", Smem<D>::kBytes)) return rc;
  {
    const int64_t groups = static_cast<int64_t>(p.c.B) * p.c.Hkv;
    const unsigned wgs = static_cast<unsigned>(p.short_rows ? groups : groups <= kByRowGroups ? std::max<int64_t>(p.n_wgs, groups) : p.n_wgs);
    KernelTimer timer_("decode_kv8", stream);
    hipLaunchKernelGGL(decode_kernel<D>, dim3(wgs), dim3(64 * kWaves), Smem<D>::kBytes, stream, p);
  }
  if (int rc = check_launch("paged_attention_decode_kv8")) return rc;
  if (p.short_rows) return 0;
  return merge<D>(p, "paged_attention_decode_kv8", "decode_kv8_combine", stream);
}

}  // namespace attn8
}  // namespace qa

extern "C" int64_t qa_paged_attention_decode_kv8_workspace(int64_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim, int64_t max_tokens) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_tokens < 0) return 0;
  return qa::attn8::workspace_bytes_of(batch, heads, kv_heads, head_dim, max_tokens, qa::attn8::kByRowTokens);
}

extern "C" int qa_paged_attention_decode_kv8(const void* query, int32_t q_dtype, int64_t q_stride_b, int64_t q_stride_h, int64_t batch, int32_t heads,
                                             int32_t head_dim, const qa_paged_kv* kv, const void* block_tables, int32_t table_dtype, int64_t table_stride,
                                             int64_t max_blocks, const void* sequence_lengths, int32_t lengths_dtype, int32_t block_size, float scale,
                                             const void* gate, int64_t gate_stride_b, int64_t gate_stride_h, void* output, void* workspace,
                                             int64_t workspace_bytes, hipStream_t stream) {
  using namespace qa;
  using namespace qa::attn8;
  DecodeParams p{};
  const Args a{"paged_attention_decode_kv8", query, q_dtype, q_stride_b, q_stride_h, batch, batch, heads, head_dim, kv, block_tables, table_dtype, table_stride, max_blocks,
               lengths_dtype, block_size, scale, gate, gate_stride_b, gate_stride_h, output};
  if (int rc = fill(p.c, a)) return rc;
  if (batch == 0) return 0;
  if (int rc = share_out(p, a, sequence_lengths, workspace, workspace_bytes, kByRowTokens)) return rc;
  return head_dim == 256 ? launch<256>(p, stream) : launch<128>(p, stream);
}
