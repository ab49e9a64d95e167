// Chunked causal prefill attention over the 4-bit paged KV cache (attention_kv4.h, kv4.h), gfx950.
//
// Columns of the products are (new position, query head of the KV head's group), position-major, so any group size
// fills them.  A workgroup owns kCols of one row and KV head, a wave 16 NCT of them, and walks the keys in tiles of 64.
// Keys go from memory straight into each wave's registers as the scores' A operand, one tile ahead (1/4 of a bf16
// tile's bytes, so the waves' repeated reads are cheap).  Values are unpacked once a workgroup: every wave turns its
// share of the next tile into bf16 operand fragments in LDS, [unit of 32 keys][dims][lane][16 bytes], which all waves
// read back without bank conflicts.  One barrier a tile.
//
// Iteration t: the scores of tile t + 1 (matrix unit) next to the softmax of tile t (vector unit), then the products of
// tile t's values next to the unpacking of tile t + 1's.
//
// With few columns the keys are split over gridDim.z and a second launch joins the parts.
#include "attention_kv4.h"

#include <algorithm>

namespace qa {
namespace prefill4 {

using namespace attn4;

struct PrefillParams {
  Params c;
  int splits;
  float* part_o;   // (splits, total, H, D)
  float* part_ml;  // (splits, total, H, 2)
};

constexpr int kTile = 64;      // keys
constexpr int kRuns = kTile / kv4::kRun;
constexpr int kWaves = 4;
constexpr int kColTiles = 2;   // 16-column tiles of a wave
constexpr int kCols = kWaves * kColTiles * 16;
constexpr int kRankRows = 64;  // batches up to this many rows start with the longest row

template <int D>
struct Smem {
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kBytes = 2 * kTileBytes + 16;  // two tiles of values; for each, the last tile that had a NaN group
};

template <int N>
__device__ __forceinline__ uint32_t load_bytes(__amdgpu_buffer_rsrc_t r, int off) {
  if constexpr (N == 4)
    return __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
  else
    return __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
}

template <int D>
__global__ __launch_bounds__(64 * kWaves, 1) void prefill_kernel(PrefillParams pp) {
  const Params& p = pp.c;
  constexpr int MT = D / 16;
  constexpr int HB = D / 64;        // bytes of a token's value chunk that a wave unpacks: half of the chunk
  constexpr int NCT = kColTiles;
  extern __shared__ __align__(16) unsigned char smem[];
  int* s_flag = reinterpret_cast<int*>(smem + 2 * Smem<D>::kTileBytes);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15;
  const int quad = lane >> 4;

  // rows from the longest down, the last columns of a row first: a short tail of the launch
  const int rr = blockIdx.y / p.Hkv;
  const int g = blockIdx.y - rr * p.Hkv;
  int b = rr;
  if (p.B <= kRankRows && p.B > 1) {
    int64_t* s_len = reinterpret_cast<int64_t*>(smem);
    int* s_order = reinterpret_cast<int*>(smem + 8 * kRankRows);
    if (tid < p.B) {
      const int64_t c0 = p.idx_i64 ? reinterpret_cast<const int64_t*>(p.cu)[tid] : reinterpret_cast<const int32_t*>(p.cu)[tid];
      const int64_t c1 = p.idx_i64 ? reinterpret_cast<const int64_t*>(p.cu)[tid + 1] : reinterpret_cast<const int32_t*>(p.cu)[tid + 1];
      s_len[tid] = c1 - c0 + (p.idx_i64 ? reinterpret_cast<const int64_t*>(p.prefix)[tid] : reinterpret_cast<const int32_t*>(p.prefix)[tid]);
    }
    __syncthreads();
    if (tid < p.B) {
      const int64_t mine = s_len[tid];
      int rank = 0;
      for (int u = 0; u < p.B; ++u) rank += s_len[u] > mine || (s_len[u] == mine && u < tid);
      s_order[rank] = tid;
    }
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(s_order[rr]);
    __syncthreads();
  }
  const int64_t tok0 = read_index(p.cu, p.idx_i64, b);
  const int64_t n_new = min64(read_index(p.cu, p.idx_i64, b + 1), p.total) - tok0;
  const int64_t ct0 = static_cast<int64_t>(gridDim.x) - 1 - blockIdx.x;
  const int64_t x0 = ct0 * kCols;  // first column of the workgroup
  if (tok0 < 0 || x0 >= n_new * p.G) return;
  const int64_t prefix = read_index(p.prefix, p.idx_i64, b);
  const int64_t last = min64(n_new * p.G, x0 + kCols) - 1;
  // keys that any column sees: not past the table
  const int64_t kv_end = max64(0, min64(prefix + last / p.G + 1, p.max_blocks << p.bs_shift));
  const int64_t first_pos = prefix + x0 / p.G;  // every column sees the keys up to here
  const int64_t runs = (kv_end + kv4::kRun - 1) / kv4::kRun;
  const int64_t all_tiles = (kv_end + kTile - 1) / kTile;
  const int64_t kt0 = all_tiles * blockIdx.z / pp.splits;
  const int64_t kt1 = all_tiles * (blockIdx.z + 1) / pp.splits;
  const uint8_t* kb = p.kpool + g * p.sG;
  const uint8_t* vb = p.vpool + g * p.sG;

  int64_t pos[NCT], tok[NCT];
  int head[NCT];
  bool live[NCT];
#pragma unroll
  for (int c = 0; c < NCT; ++c) {
    const int64_t x = x0 + (wave * NCT + c) * 16 + col;
    live[c] = x <= last;
    const int64_t n = (live[c] ? x : last) / p.G;
    head[c] = static_cast<int>((live[c] ? x : last) - n * p.G) + g * p.G;
    pos[c] = prefix + n;
    tok[c] = tok0 + n;
  }

  // ---- the tiles' loads
  KeyRun<D> kr[kRuns];
  uint32_t vcode[2][4], vscale[2];  // this wave's share: unit wave / 2, half (wave & 1) of each chunk
  const int vunit = wave >> 1, vhalf = wave & 1;
  int32_t phys[kRuns];
  auto entries = [&](int64_t kt) {
#pragma unroll
    for (int j = 0; j < kRuns; ++j) phys[j] = kt < kt1 ? block_of_run(p, b, kRuns * kt + j, runs) : -1;
  };
  auto there = [&]() { return (phys[0] >= 0 ? 1 : 0) | (phys[1] >= 0 ? 2 : 0) | (phys[2] >= 0 ? 4 : 0) | (phys[3] >= 0 ? 8 : 0); };
  auto fetch_keys = [&](int64_t kt) {
#pragma unroll
    for (int j = 0; j < kRuns; ++j) load_keys<D>(kr[j], run_rsrc<D>(p, kb, phys[j], kRuns * kt + j), lane);
  };
  auto fetch_values = [&](int64_t kt) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int32_t ph = vunit == 0 ? phys[j] : phys[2 + j];
      const __amdgpu_buffer_rsrc_t r = run_rsrc<D>(p, vb, ph, kRuns * kt + 2 * vunit + j);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int off = D == 256 ? 1024 * (t >> 1) + 16 * lane + 8 * (t & 1) + HB * vhalf : 16 * lane + 4 * t + HB * vhalf;
        vcode[j][t] = load_bytes<HB>(r, off);
      }
      vscale[j] = __builtin_amdgcn_raw_buffer_load_b32(r, kv4::Run<D>::kCodes + 16 * (col / (512 / D)) + 4 * quad, 0, 0);
    }
  };
  // unpacks the share of tile kt that is in vcode / vscale into buffer buf
  auto unpack = [&](int64_t kt, int buf) {
    if (kt * kTile + kTile > first_pos + 1) {  // some column does not see all of the tile
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // keys that no column sees may hold anything, and 0 times a NaN is one
        const int64_t left = kv_end - kt * kTile - kv4::kRun * (2 * vunit + j) - 4 * quad;
        vscale[j] &= left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * static_cast<int>(left))) - 1u;
        // a NaN group reaches only the columns that see its token: out of the product, and nan_groups adds it
        uint32_t drop = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if ((vscale[j] >> (8 * t) & 255u) == 255u) drop |= 255u << (8 * t);
        vscale[j] &= ~drop;
        if (drop != 0) s_flag[buf] = static_cast<int>(kt - kt0) + 1;
      }
    }
    float s[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) s[t] = value_scale(vscale[t >> 2], t & 3);
    uint4* dst = reinterpret_cast<uint4*>(smem + buf * Smem<D>::kTileBytes) + (vunit * MT + 2 * HB * vhalf) * 64 + lane;
#pragma unroll
    for (int e = 0; e < HB; ++e) {
      uint32_t pair[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const uint32_t c = vcode[t >> 2][t & 3];
        switch (e) {
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
      dst[(2 * e) * 64] = even;
      dst[(2 * e + 1) * 64] = odd;
    }
  };

  float m_run[NCT], l_run[NCT];
  floatx4_v o[NCT][MT];
#pragma unroll
  for (int c = 0; c < NCT; ++c) {
    m_run[c] = -INFINITY;
    l_run[c] = 0.f;
#pragma unroll
    for (int i = 0; i < MT; ++i) o[c][i] = floatx4_v{0.f, 0.f, 0.f, 0.f};
  }

  if (kt0 < kt1) {
    if (tid < 2) s_flag[tid] = 0;
    entries(kt0);
    int there_cur = there();
    fetch_keys(kt0);
    fetch_values(kt0);
    QueryCols<D> qh[NCT], ql[NCT];
#pragma unroll
    for (int c = 0; c < NCT; ++c) {
      QueryRow<D> row;
      row.load(live[c] ? p.q + tok[c] * p.q_st + static_cast<int64_t>(head[c]) * p.q_sh : nullptr, quad);
      row.template split<false>(qh[c]);
      row.template split<true>(ql[c]);
    }
    floatx4_v sc[NCT][kRuns];
    auto scores = [&]() {
#pragma unroll
      for (int c = 0; c < NCT; ++c)
#pragma unroll
        for (int j = 0; j < kRuns; ++j) sc[c][j] = floatx4_v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kRuns; ++j) {
#pragma unroll
        for (int c = 0; c < NCT; ++c) sc[c][j] = score<D>(kr[j], qh[c], sc[c][j]);
#pragma unroll
        for (int c = 0; c < NCT; ++c) sc[c][j] = score<D>(kr[j], ql[c], sc[c][j]);
      }
    };
    scores();
    __syncthreads();  // the flags
    unpack(kt0, 0);
    entries(kt0 + 1);
    int there_next = there();
    fetch_keys(kt0 + 1);
    fetch_values(kt0 + 1);
    __syncthreads();

    const float qk_scale = p.scale * kLog2e;
    for (int64_t kt = kt0; kt < kt1; ++kt) {
      const int buf = static_cast<int>((kt - kt0) & 1);
      const int64_t key0 = kt * kTile;
      // ---- mask
      if (!(key0 + kTile <= first_pos + 1 && there_cur == 15)) {
#pragma unroll
        for (int c = 0; c < NCT; ++c) {
          const int lim = static_cast<int>(max64(-1, min64(kTile - 1, min64(pos[c], kv_end - 1) - key0)));  // the last key the column sees
#pragma unroll
          for (int j = 0; j < kRuns; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (16 * j + 4 * quad + r > lim || !(there_cur >> j & 1)) sc[c][j][r] = -INFINITY;
        }
      }
      // ---- softmax of tile kt
      bf16x8_v pb[NCT][2];
#pragma unroll
      for (int c = 0; c < NCT; ++c) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < kRuns; ++j) mx = fmaxf(mx, fmaxf(fmaxf(sc[c][j][0], sc[c][j][1]), fmaxf(sc[c][j][2], sc[c][j][3])));
        mx *= qk_scale;
        if (__ballot(mx > m_run[c] + kLazy) != 0) {
          const float m_new = fmaxf(m_run[c], column_max(mx));
          const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run[c] - m_new);
          m_run[c] = m_new;
          l_run[c] *= corr;
#pragma unroll
          for (int i = 0; i < MT; ++i) o[c][i] *= corr;
        }
        const float use = m_run[c] == -INFINITY ? 0.f : m_run[c];
#pragma unroll
        for (int j = 0; j < kRuns; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[c][j][r], qk_scale, -use));
            l_run[c] += pr;
            pb[c][j >> 1][4 * (j & 1) + r] = static_cast<__bf16>(pr);
          }
      }
      // ---- scores of tile kt + 1, keys of kt + 2
      scores();
      entries(kt + 2);
      fetch_keys(kt + 2);
      // ---- values of tile kt
      const uint4* vt = reinterpret_cast<const uint4*>(smem + buf * Smem<D>::kTileBytes) + lane;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const bf16x8_v a = __builtin_bit_cast(bf16x8_v, vt[(u * MT + i) * 64]);
#pragma unroll
          for (int c = 0; c < NCT; ++c) o[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[c][u], o[c][i], 0, 0, 0);
        }
      // ---- NaN groups among keys that not every column sees
      if (s_flag[buf] == static_cast<int>(kt - kt0) + 1) {
        for (int t = 0; t < kTile; ++t) {
          const int64_t key = key0 + t;
          if (!(there_cur >> (t >> 4) & 1) || key >= kv_end) continue;
          const int32_t ph = block_of_run(p, b, key >> 4, runs);
          const uint8_t* run = vb + static_cast<int64_t>(ph) * p.sP + ((key >> 4) & ((1 << (p.bs_shift - 4)) - 1)) * kv4::Run<D>::kBytes;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool nan = run[kv4::Run<D>::value_scale(t & 15, (4 * quad + r) / (512 / D))] == 255;
#pragma unroll
            for (int c = 0; c < NCT; ++c)
              if (nan && key <= pos[c]) {
#pragma unroll
                for (int i = 0; i < MT; ++i) o[c][i][r] = __uint_as_float(0x7fc00000u);
              }
          }
        }
      }
      // ---- the next tile's values
      unpack(kt + 1, buf ^ 1);
      fetch_values(kt + 2);
      there_cur = there_next;
      there_next = there();
      lds_barrier();
    }
  }

  // ---- out
#pragma unroll
  for (int c = 0; c < NCT; ++c) {
    const float l = column_sum(l_run[c]);
    if (!live[c]) continue;
    const int64_t row = tok[c] * p.H + head[c];
    if (pp.splits > 1) {
      const int64_t at = blockIdx.z * p.total * p.H + row;
      if (quad == 0) *reinterpret_cast<float2*>(pp.part_ml + at * 2) = make_float2(m_run[c], l);
      if (kt0 < kt1) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < MT; i += 4)
            *reinterpret_cast<floatx4_v*>(pp.part_o + at * D + (4 * quad + r) * MT + i) = floatx4_v{o[c][i][r], o[c][i + 1][r], o[c][i + 2][r], o[c][i + 3][r]};
      }
      continue;
    }
    const bf16_t* gate = p.gate != nullptr ? p.gate + tok[c] * p.gate_st + static_cast<int64_t>(head[c]) * p.gate_sh : nullptr;
    uint2 graw[4][MT / 4];
    if (gate != nullptr) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < MT / 4; ++i) graw[r][i] = *reinterpret_cast<const uint2*>(gate + (4 * quad + r) * MT + 4 * i);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < MT; i += 4) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = normalised(o[c][i + e][r], l);
          if (gate != nullptr) {
            const uint32_t w = e < 2 ? graw[r][i / 4].x : graw[r][i / 4].y;
            v[e] *= sigmoid(__uint_as_float(e & 1 ? w & 0xffff0000u : w << 16));
          }
        }
        uint2 packed;
        packed.x = static_cast<uint32_t>(f32_to_bf16(v[0])) | static_cast<uint32_t>(f32_to_bf16(v[1])) << 16;
        packed.y = static_cast<uint32_t>(f32_to_bf16(v[2])) | static_cast<uint32_t>(f32_to_bf16(v[3])) << 16;
        *reinterpret_cast<uint2*>(p.out + row * D + (4 * quad + r) * MT + i) = packed;
      }
  }
}

// Joins the parts of one (token, head): a wave each, lane l dims l D/64 ..
template <int D>
__global__ __launch_bounds__(256) void join_kernel(PrefillParams pp, int64_t max_new) {
  const Params& p = pp.c;
  constexpr int E = D / 64;
  typedef float vec_t __attribute__((ext_vector_type(E)));
  const int lane = threadIdx.x & 63;
  const int64_t x = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.y;
  const int64_t tok0 = read_index(p.cu, p.idx_i64, b);
  const int64_t n_new = min64(max_new, min64(read_index(p.cu, p.idx_i64, b + 1), p.total) - tok0);
  if (tok0 < 0 || x >= n_new * p.H) return;
  const int64_t row = tok0 * p.H + x;
  const int64_t stride = p.total * p.H;
  const float2 ml = lane < pp.splits ? *reinterpret_cast<const float2*>(pp.part_ml + (lane * stride + row) * 2) : make_float2(-INFINITY, 0.f);
  const float m = wave_max(ml.x);
  const float f = __builtin_amdgcn_exp2f(ml.x - (m == -INFINITY ? 0.f : m));
  const float l = wave_sum(f * ml.y);
  vec_t acc = vec_t(0.f);
  for (int s = 0; s < pp.splits; ++s) {
    const float fs = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), s));
    const float ls = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ml.y), s));
    if (ls != 0.f) acc += fs * *reinterpret_cast<const vec_t*>(pp.part_o + (s * stride + row) * D + E * lane);  // a part that saw nothing wrote nothing
  }
  const int64_t n = x / p.H, h = x - n * p.H;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float r = normalised(acc[e], l);
    if (p.gate != nullptr) r *= sigmoid(bf16_to_f32(p.gate[(tok0 + n) * p.gate_st + h * p.gate_sh + E * lane + e]));
    p.out[row * D + E * lane + e] = f32_to_bf16(r);
  }
}

constexpr int kMaxSplits = 64;

// Parts the keys are split into: as many as fill the chip, of at least four tiles each where every row is as long as its table.
static int splits_of(int64_t batch, int kv_heads, int group, int64_t max_new, int64_t max_tokens) {
  const int64_t wgs = batch * kv_heads * ceil_div(max_new * group, kCols);
  const int64_t tiles = ceil_div(std::max<int64_t>(max_tokens, 1), kTile);
  if (wgs >= 256) return 1;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({kMaxSplits, 256 / wgs, tiles / 4})));
}

static int64_t workspace_of(int splits, int64_t total, int heads, int head_dim) {
  return splits > 1 ? splits * total * heads * (static_cast<int64_t>(head_dim) + 2) * 4 : 0;
}

template <int D>
static int launch(const PrefillParams& p, dim3 grid, int64_t max_new, hipStream_t stream) {
  const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(&prefill_kernel<D>), hipFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::kBytes);
  if (err != hipSuccess) return fail("paged_attention_prefill_kv4: cannot reserve %d bytes of LDS: %s", Smem<D>::kBytes, hipGetErrorString(err));
  {
    KernelTimer timer_("prefill_kv4", stream);
    hipLaunchKernelGGL(prefill_kernel<D>, grid, dim3(64 * kWaves), Smem<D>::kBytes, stream, p);
  }
  if (int rc = check_launch("paged_attention_prefill_kv4")) return rc;
  if (p.splits > 1) {
    KernelTimer timer_("prefill_kv4_join", stream);
    const dim3 jgrid(static_cast<unsigned>(ceil_div(max_new * p.c.H, 4)), static_cast<unsigned>(p.c.B));
    hipLaunchKernelGGL(join_kernel<D>, jgrid, dim3(256), 0, stream, p, max_new);
  }
  return check_launch("paged_attention_prefill_kv4");
}

}  // namespace prefill4
}  // namespace qa

extern "C" int64_t qa_paged_attention_prefill_kv4_workspace(int64_t total_new, int64_t batch, int64_t max_new, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                                            int64_t max_tokens) {
  if (total_new <= 0 || batch <= 0 || max_new <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || head_dim <= 0 || max_tokens < 0) return 0;
  return qa::prefill4::workspace_of(qa::prefill4::splits_of(batch, kv_heads, heads / kv_heads, std::min(max_new, total_new), max_tokens), total_new, heads, head_dim);
}

extern "C" int qa_paged_attention_prefill_kv4(const void* query, int32_t q_dtype, int64_t q_stride_t, int64_t q_stride_h, int64_t total_new, const void* cu_seqlens,
                                              const void* prefix_lens, int32_t idx_dtype, int64_t batch, int64_t max_new, int32_t heads, int32_t head_dim,
                                              const qa_paged_kv* kv, const void* block_tables, int32_t table_dtype, int64_t table_stride, int64_t max_blocks,
                                              int32_t block_size, float scale, const void* gate, int64_t gate_stride_t, int64_t gate_stride_h, void* output,
                                              void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  using namespace qa;
  using namespace qa::prefill4;
  PrefillParams p{};
  const Args a{"paged_attention_prefill_kv4", query, q_dtype, q_stride_t, q_stride_h, batch, heads, head_dim, kv, block_tables, table_dtype, table_stride, max_blocks,
               idx_dtype, block_size, scale, gate, gate_stride_t, gate_stride_h, output};
  if (int rc = fill(p.c, a)) return rc;
  QA_REQUIRE(total_new >= 0 && total_new <= 0x7fffffff && max_new >= 0 && max_new <= 0x7fffffff, "%s: token counts out of range", a.what);
  if (batch == 0 || max_new == 0 || total_new == 0) return 0;
  QA_REQUIRE(cu_seqlens && prefix_lens, "%s: pointers must be non-null", a.what);
  QA_REQUIRE(batch * kv->kv_heads <= 65535, "%s: batch * KV heads must fit 65535", a.what);
  max_new = std::min(max_new, total_new);
  QA_REQUIRE(max_new * heads <= 0x7fffffff, "%s: max_new * heads out of range", a.what);
  p.c.cu = cu_seqlens;
  p.c.prefix = prefix_lens;
  p.c.total = total_new;
  p.splits = splits_of(batch, kv->kv_heads, p.c.G, max_new, max_blocks * block_size);
  const int64_t need = workspace_of(p.splits, total_new, heads, head_dim);
  QA_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0),
             "paged prefill workspace too small or not 16-byte aligned: need %lld bytes, have %lld", static_cast<long long>(need), static_cast<long long>(workspace_bytes));
  p.part_o = reinterpret_cast<float*>(workspace);
  p.part_ml = p.part_o + static_cast<int64_t>(p.splits) * total_new * heads * head_dim;
  const dim3 grid(static_cast<unsigned>(ceil_div(max_new * p.c.G, kCols)), static_cast<unsigned>(batch * kv->kv_heads), static_cast<unsigned>(p.splits));
  return head_dim == 256 ? launch<256>(p, grid, max_new, stream) : launch<128>(p, grid, max_new, stream);
}
