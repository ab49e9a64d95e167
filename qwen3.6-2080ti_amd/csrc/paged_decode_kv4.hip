// Decode attention over the 4-bit paged KV cache (attention_kv4.h, kv4.h), gfx950: one token per row.
//
// Bound by memory: 17 D / 32 bytes a cached token, KV head and K or V, each read once for the G query heads that share
// it.  All (row, KV head, unit of 32 tokens) are laid end to end, T units, and workgroup w of W takes the range
// [T w / W, T (w + 1) / W): equal shares whatever the lengths.  The workgroup's eight waves take its units in turn, so
// that neighbouring waves read neighbouring tiles, each with an online softmax of its own and no barrier; where the
// range leaves a row group they merge in LDS and write one partial (m, l, o) of the G heads.  A workgroup that had the
// whole row group writes the result; the other groups' partials are merged by combine_kernel.  Where all rows are short a
// workgroup takes a row group as it is.  64 rows of 1k to 32k tokens, two KV heads of 256: 91.6 us for 529 MB, 5.8 TB/s (a
// pure reader reaches 6.2), and 4.7 to merge; one row of 200k, a head of 128: 12.1 + 4.0; four of 512: 9.0, all latency.
//
// A wave keeps two units of keys and values in flight in registers (buffer loads of zero records for what is skipped, so
// every step issues the same loads and the wait counts are fixed), across row groups: the merge of one and the query of
// the next run while the next one's tiles arrive.  Lane j of a wave holds where unit j of its next 64 lies; one search and
// one vector load of the tables serve them all, and a step reads its lane.  Columns of the scores' product: with up to
// eight heads the first eight are the heads' hi pieces and the last eight their lo pieces, one product a slice, and a
// row rotation adds the two; with more the pieces take two products.  The query is split once a workgroup, a head a wave,
// through LDS.
#include "attention_kv4.h"
#include "decode_split.h"

namespace qa {
namespace attn4 {

// Where no row is longer than this, a workgroup takes a row group and nothing is merged; where the tables cannot hold a
// longer one, the second launch is left out.  us split / by row, 2 KV heads of 256: 4 rows of 512 12.1 / 9.1, of 1024 12.4 /
// 13.3, of 2048 12.2 / 19.4; 64 rows of up to 1024 25.5 / 14.1, of up to 4096 34.5 / 36.3; 200 rows of 500 37.7 / 22.0.
constexpr int kByRowTokens = 1024;
// Row groups up to which a call of long tables has the workgroups for that; each of them reads all the lengths first.  us
// split / by row, rows of 300, 2 KV heads: 200 rows 36 / 23, 500 68 / 51, 1000 122 / 116, 2000 229 / 291.
constexpr int kByRowGroups = 2048;
template <int D, bool WIDE>
struct Smem {
  static constexpr int kHeads = WIDE ? 16 : 8;
  static constexpr int kRow = D + 4;                      // floats: neighbouring heads start four banks apart
  static constexpr int kM = kWaves * kHeads * kRow * 4;   // after the waves' sums: (kWaves, 16) reference points,
  static constexpr int kL = kM + kWaves * 16 * 4;         // (kWaves, 16) denominators,
  static constexpr int kTotal = kL + kWaves * 16 * 4;     // the merged ones (2, 16),
  static constexpr int kQ = kTotal + 2 * 16 * 4;          // the query's pieces, 32 rows of D bytes,
  static constexpr int kQRow = D + 16;
  static constexpr int kQScale = kQ + 32 * kQRow;         // and their scales
  static constexpr int kBytes = kQScale + 32 * 4;
};

// WIDE: more than eight heads a group.
template <int D, bool WIDE>
__global__ __launch_bounds__(64 * kWaves, 2) void decode_kernel(DecodeParams dp) {
  const Params& p = dp.c;
  using S = Smem<D, WIDE>;
  constexpr int MT = D / 16;
  extern __shared__ __align__(16) unsigned char smem[];
  float* s_o = reinterpret_cast<float*>(smem);
  float* s_m = reinterpret_cast<float*>(smem + S::kM);
  float* s_l = reinterpret_cast<float*>(smem + S::kL);
  float* s_total = reinterpret_cast<float*>(smem + S::kTotal);
  uint32_t* s_qscale = reinterpret_cast<uint32_t*>(smem + S::kQScale);
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
        return ok ? static_cast<int64_t>(id) * p.sP + (run & ((1 << sub_shift) - 1)) * kv4::Run<D>::kBytes + g * p.sG : -1;
      };
      at0 = offset(2 * static_cast<int64_t>(u));
      if (left > kv4::kRun) at1 = offset(2 * static_cast<int64_t>(u) + 1);
    }
  };
  locate(0, true);

  KeyRun<D> kr[2][2];
  ValueRun<D> vr[2][2];
  int64_t where[2];  // of the unit being asked for
  int have[2];       // tokens of the units in kr / vr, and 256 / 512 where the first / second run is not there
  auto look = [&](int i, int s) {
    const int j = i & 63;
    auto read = [&](int64_t v) {
      const uint32_t l = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), j), h = __builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), j);
      return static_cast<int64_t>(static_cast<uint64_t>(h) << 32 | l);
    };
    where[0] = read(at0);
    where[1] = read(at1);
    have[s] = __builtin_amdgcn_readlane(left, j) | (where[0] < 0 ? 256 : 0) | (where[1] < 0 ? 512 : 0);
  };
  auto rsrc = [&](const uint8_t* base, int64_t o) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base + (o < 0 ? 0 : o)), 0, o < 0 ? 0 : kv4::Run<D>::kBytes, 0x00020000);
  };
  auto fetch_keys = [&](int s) {
#pragma unroll
    for (int j = 0; j < 2; ++j) load_keys<D, kOnce>(kr[s][j], rsrc(p.kpool, where[j]), lane);
  };
  auto fetch_values = [&](int s) {
#pragma unroll
    for (int j = 0; j < 2; ++j) load_values<D, kOnce>(vr[s][j], rsrc(p.vpool, where[j]), lane);
  };

  // ---- the query of a row group: wave w takes heads w and w + 8, lane l dims E l ..
  constexpr int E = D / 64;
  uint32_t qraw[WIDE ? 2 : 1][E / 2];
  auto fetch_query = [&](const Cursor& c) {
#pragma unroll
    for (int k = 0; k < (WIDE ? 2 : 1); ++k) {
      const int h = wave + 8 * k;
#pragma unroll
      for (int e = 0; e < E / 2; ++e) qraw[k][e] = 0;
      if (h < p.G && c.b < p.B) {
        const bf16_t* row = p.q + static_cast<int64_t>(c.b) * p.q_st + static_cast<int64_t>(c.g * p.G + h) * p.q_sh + E * lane;
        if constexpr (E == 4) {
          const uint2 u = *reinterpret_cast<const uint2*>(row);
          qraw[k][0] = u.x, qraw[k][1] = u.y;
        } else {
          qraw[k][0] = *reinterpret_cast<const uint32_t*>(row);
        }
      }
    }
  };
  // rows of s_q: head h's hi piece at h, its lo piece at h + (WIDE ? 16 : 8)
  auto split_query = [&]() {
#pragma unroll
    for (int k = 0; k < (WIDE ? 2 : 1); ++k) {
      const int h = wave + 8 * k;
      uint32_t top = 0;
      float x[E];
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        const uint32_t w = qraw[k][e];
        x[2 * e] = __uint_as_float(w << 16);
        x[2 * e + 1] = __uint_as_float(w & 0xffff0000u);
        top = max(top, max(w << 16 & 0x7fffffffu, w & 0x7fff0000u));
      }
      const uint32_t byte = query_scale(wave_max_bits(top));
      const float inv = __uint_as_float((254u - byte) << 23);
      uint32_t near = max(top, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0xB1, 0xF, 0xF, false)));  // of the eight dims: quad_perm [1,0,3,2]
      if constexpr (E == 2) near = max(near, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(near), 0x4E, 0xF, 0xF, false)));  // quad_perm [2,3,0,1]
      const float grid = piece_grid(near, inv);
      uint32_t hi8 = 0, lo8 = 0;
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float y0 = x[e] * inv, y1 = x[e + 1] * inv;
        const uint32_t h2 = __builtin_amdgcn_cvt_pk_fp8_f32(y0 + grid - grid, y1 + grid - grid, 0, false);
        const floatx2_v a = __builtin_amdgcn_cvt_pk_f32_fp8(h2, false);
        const uint32_t l2 = __builtin_amdgcn_cvt_pk_fp8_f32((y0 - a[0]) * 16.f, (y1 - a[1]) * 16.f, 0, false);
        hi8 |= (h2 & 0xffffu) << (8 * e);
        lo8 |= (l2 & 0xffffu) << (8 * e);
      }
      unsigned char* hi_row = smem + S::kQ + h * S::kQRow + E * lane;
      unsigned char* lo_row = hi_row + S::kHeads * S::kQRow;
      if constexpr (E == 4) {
        *reinterpret_cast<uint32_t*>(hi_row) = hi8;
        *reinterpret_cast<uint32_t*>(lo_row) = lo8;
      } else {
        *reinterpret_cast<uint16_t*>(hi_row) = static_cast<uint16_t>(hi8);
        *reinterpret_cast<uint16_t*>(lo_row) = static_cast<uint16_t>(lo8);
      }
      if (lane == 0) {
        s_qscale[h] = byte;
        s_qscale[h + S::kHeads] = byte - 4u;
      }
    }
  };
  auto read_query = [&](QueryCols<D>& q, int row) {
    const unsigned char* at = smem + S::kQ + row * S::kQRow + 16 * quad;
#pragma unroll
    for (int i = 0; i < D / 128; ++i) {
      const uint4 a = *reinterpret_cast<const uint4*>(at + 128 * i), b = *reinterpret_cast<const uint4*>(at + 128 * i + 64);
      q.code[i] = int8_v{static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w),
                         static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w)};
    }
    q.scale = s_qscale[row];
  };
  fetch_query(cur);  // before the tiles: loads are waited for in their order
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    look(s, s);
    fetch_keys(s);
    fetch_values(s);
  }
  const float qk_scale = p.scale * kLog2e;

  int i = 0;                // the wave's next unit, in slot i & 1
  int gu = lo + wave;       // that unit among all
  for (int at = lo; at < hi;) {
    const int seg_end = min(hi, cur.cum + cur.nu);
    split_query();
    __syncthreads();  // the query is there; the waves are done with the last merge
    QueryCols<D> qa_, qb_;
    read_query(qa_, col);
    if constexpr (WIDE) read_query(qb_, 16 + col);
    Cursor nxt = cur;
    if (seg_end < hi) {
      next_row_group(p, nxt);
      fetch_query(nxt);
    }

    float m_run = -INFINITY, l_run = 0.f;
    floatx4_v o[MT];
#pragma unroll
    for (int k = 0; k < MT; ++k) o[k] = floatx4_v{0.f, 0.f, 0.f, 0.f};

    auto step = [&](int s) {
      // ---- scores: this lane's are tokens 4 quad + r of both runs, of head col & 7 (WIDE: col)
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
      if (have[s] != kUnit) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int mine = (have[s] >> (8 + j) & 1) ? 0 : (have[s] & 255) - kv4::kRun * j - 4 * quad;  // this lane's tokens that are there
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r >= mine) sc[4 * j + r] = -INFINITY;
          // their values may be anything, and 0 times a NaN is one
          vr[s][j].scale &= mine >= 4 ? 0xffffffffu : mine <= 0 ? 0u : (1u << (8 * mine)) - 1u;
        }
      }
      if (((i + 2) & 63) == 0) locate((i + 2) >> 6, false);
      look(i + 2, s);
      fetch_keys(s);

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
      // ---- values
      accumulate<D>(vr[s], pb, o);
      fetch_values(s);
      ++i;
      gu += kWaves;
    };
    while (gu < seg_end) {
      if ((i & 1) == 0) {
        step(0);
        if (gu >= seg_end) break;
      }
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
        for (int k = 0; k < MT; k += 4)
          *reinterpret_cast<floatx4_v*>(so + (4 * quad + r) * MT + k) = floatx4_v{o[k][r], o[k + 1][r], o[k + 2][r], o[k + 3][r]} * f;
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

template <int D, bool WIDE>
static int launch(const DecodeParams& p, hipStream_t stream) {
  using S = Smem<D, WIDE>;
  if (int rc = reserve_lds<&decode_kernel<D, WIDE>>("paged_attention_decode_kv4", S::kBytes)) return rc;
  {
    const int64_t groups = static_cast<int64_t>(p.c.B) * p.c.Hkv;
    const unsigned wgs = static_cast<unsigned>(p.short_rows ? groups : groups <= kByRowGroups ? std::max<int64_t>(p.n_wgs, groups) : p.n_wgs);
    KernelTimer timer_("decode_kv4", stream);
    hipLaunchKernelGGL((decode_kernel<D, WIDE>), dim3(wgs), dim3(64 * kWaves), S::kBytes, stream, p);
  }
  if (int rc = check_launch("paged_attention_decode_kv4")) return rc;
  if (p.short_rows) return 0;
  return merge<D>(p, "paged_attention_decode_kv4", "decode_kv4_combine", stream);
}

}  // namespace attn4
}  // namespace qa

extern "C" int64_t qa_paged_attention_decode_kv4_workspace(int64_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim, int64_t max_tokens) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_tokens < 0) return 0;
  return qa::attn4::workspace_bytes_of(batch, heads, kv_heads, head_dim, max_tokens, qa::attn4::kByRowTokens);
}

extern "C" int qa_paged_attention_decode_kv4(const void* query, int32_t q_dtype, int64_t q_stride_b, int64_t q_stride_h, int64_t batch, int32_t heads,
                                             int32_t head_dim, const qa_paged_kv* kv, const void* block_tables, int32_t table_dtype, int64_t table_stride,
                                             int64_t max_blocks, const void* sequence_lengths, int32_t lengths_dtype, int32_t block_size, float scale,
                                             const void* gate, int64_t gate_stride_b, int64_t gate_stride_h, void* output, void* workspace,
                                             int64_t workspace_bytes, hipStream_t stream) {
  using namespace qa;
  using namespace qa::attn4;
  DecodeParams p{};
  const Args a{"paged_attention_decode_kv4", query, q_dtype, q_stride_b, q_stride_h, batch, batch, heads, head_dim, kv, block_tables, table_dtype, table_stride, max_blocks,
               lengths_dtype, block_size, scale, gate, gate_stride_b, gate_stride_h, output};
  if (int rc = fill(p.c, a)) return rc;
  if (batch == 0) return 0;
  if (int rc = share_out(p, a, sequence_lengths, workspace, workspace_bytes, kByRowTokens)) return rc;
  if (head_dim == 256) return p.c.G > 8 ? launch<256, true>(p, stream) : launch<256, false>(p, stream);
  return p.c.G > 8 ? launch<128, true>(p, stream) : launch<128, false>(p, stream);
}
