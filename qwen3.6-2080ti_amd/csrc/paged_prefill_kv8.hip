// Chunked causal prefill attention over the 8-bit paged KV cache (attention_kv8.h, kv8.h), gfx950.
//
// Columns of the products are (new position, query head of the KV head's group), position-major, so any group size
// fills them.  A workgroup owns 128 or 64 of one row and KV head (columns_of) and walks the keys in tiles of 64.  Its waves are
// pairs of 32 columns: a wave takes the scores and the softmax of half of the tile's keys, then the products with the values of
// all of them for half of the dims, its partner's probabilities through LDS.  So a key read from LDS feeds 32 columns and is
// converted once a pair, and the accumulators of a wave stay at 64 registers, two waves to a SIMD.
//
// Codes go from memory to LDS as they are, a run a wave, and to bf16 next to the products: exact, where
// products of 8 bits would round the query and the probabilities to 4.  Keys converted into LDS, once a workgroup, cost more
// there than they save (1048 -> 1090 us at the longest size below).
//
// 128 columns, eight waves, one barrier an iteration: the probabilities of tile i, for which the pair shares its columns'
// reference points, between the products of tile i - 1's values, then the scores of tile i + 1.  64 columns, four waves, keys
// and values in one buffer each, so that two workgroups fill a CU and work while the other waits: a barrier after the
// products with values and one after the scores.
//
// With few columns the keys are split over gridDim.z and a second launch joins the parts.
//
// What bounds it: power, and issue.  A tile of 64 keys, D = 256, is 32 matrix instructions of 32 cycles a wave, two waves a SIMD,
// and beside them 128 conversions, 16 exponentials and their shares of loads, masks and sums.  It takes 4050 cycles, the
// matrix units busy for half of them, at 1.95 to 2.1 GHz of 2.4: with fewer cycles the clock falls.  A copy of the kernel without its
// tiles' writes to LDS had 11% fewer cycles and took 5% less time; zeros for data took 988 us at the longest size below.
// Measured, 16 heads, 2 of keys, D = 256: 2048 new behind 32 000 1046 us (1108 Gflop, 1060 Tflop/s; a library's 8192 x 8192
// x 8192 product 1268), 8 x 512 behind up to 8192 333 us (925 Tflop/s; 512 workgroups of up to 129 tiles, one a CU:
// the last ends after 157 tiles where the mean is 145, so 8% of it is the launch's tail); 20 heads, 4 of keys, D = 128, five prompts of up
// to 700 25.7 us.
// Values' products at a raised wave priority 1048 -> 1034, probabilities between them 1221 -> 1055.  Not kept, us at that size: the
// two halves of the workgroup half a tile apart 1040, two accumulators of scores 1049, three key buffers 1065, four waves of 64
// columns with 512 registers 1187, workgroups of 64 columns 1130; within 1% of the kernel, each against it on one card: four waves that
// share 64 columns' values (96 conversions for 128), counters in LDS for the barrier, runs copied straight to LDS two or three
// tiles ahead, a wave's own probabilities kept in registers and its first values asked for before the barrier.
#include "attention_kv8.h"
#include "prefill_split.h"

#include <type_traits>

namespace qa {
namespace prefill8 {

using namespace attn8;

typedef float floatx16_v __attribute__((ext_vector_type(16)));

template <int D, int COLS>
struct Smem {
  static constexpr int kWaves = COLS / 16;
  static constexpr int kKeyBufs = COLS == 128 ? 2 : 1;
  static constexpr int kValueBufs = COLS == 128 ? 4 : 1;
  static constexpr int kPBufs = COLS == 128 ? 2 : 1;
  static constexpr int kRunBytes = kv8::Run<D>::kCodes;
  static constexpr int kTileBytes = kRuns * kRunBytes;
  static constexpr int kValues = kKeyBufs * kTileBytes;               // after the keys: [buffer][run]
  static constexpr int kP = kValues + kValueBufs * kTileBytes;        // probabilities: [buffer][wave][run][lane][16 bytes]
  static constexpr int kMax = kP + kPBufs * kWaves * 2 * 1024;        // [buffer][wave][32] floats; at the end sums and reference points
  static constexpr int kScale = kMax + std::max(kPBufs * kWaves * 32, 3 * COLS) * 4;  // of keys [buffer][run], of values [buffer][run]
  static constexpr int kFlag = kScale + (kKeyBufs + kValueBufs) * kRuns * 4;  // whether a tile that not every column sees whole had a NaN
  static constexpr int kBytes = kFlag + 16;
};

template <int D, int COLS>
__global__ __launch_bounds__(4 * COLS, 2) void prefill_kernel(PrefillParams pp) {
  const Params& p = pp.c;
  constexpr int N = kv8::Run<D>::kSlices;
  constexpr int MT = D / 64;        // tiles of 32 dims of a wave
  constexpr bool kWide = COLS == 128;
  using S = Smem<D, COLS>;
  constexpr int kWaves = S::kWaves;
  extern __shared__ __align__(16) unsigned char smem[];
  float* s_max = reinterpret_cast<float*>(smem + S::kMax);
  float* s_kscale = reinterpret_cast<float*>(smem + S::kScale);
  float* s_vscale = s_kscale + S::kKeyBufs * kRuns;
  int* s_flag = reinterpret_cast<int*>(smem + S::kFlag);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int pair = wave >> 1;
  const int col = lane & 31;  // of the pair's
  const int hi = lane >> 5;

  // rows from the longest down, the last columns of a row first: a short tail of the launch
  const int rr = blockIdx.y / p.Hkv;
  const int g = blockIdx.y - rr * p.Hkv;
  int b = rr;
  int64_t tok0, tok1, prefix;
  if (p.B <= kRankRows && p.B > 1) {
    int64_t* s_len = reinterpret_cast<int64_t*>(smem);
    int64_t* s_row = s_len + kRankRows;  // of the row of each rank: itself, its first token, the next row's, its prefix
    int64_t c0 = 0, c1 = 0, before = 0;
    if (tid < p.B) {
      c0 = read_index(p.cu, p.idx_i64, tid);
      c1 = read_index(p.cu, p.idx_i64, tid + 1);
      before = read_index(p.prefix, p.idx_i64, tid);
      s_len[tid] = c1 - c0 + before;
    }
    __syncthreads();
    if (tid < p.B) {
      const int64_t mine = c1 - c0 + before;
      int rank = 0;
      for (int u = 0; u < p.B; ++u) rank += s_len[u] > mine || (s_len[u] == mine && u < tid);
      s_row[4 * rank] = tid;
      s_row[4 * rank + 1] = c0;
      s_row[4 * rank + 2] = c1;
      s_row[4 * rank + 3] = before;
    }
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(static_cast<int>(s_row[4 * rr]));
    tok0 = uniform64(s_row[4 * rr + 1]);
    tok1 = uniform64(s_row[4 * rr + 2]);
    prefix = uniform64(s_row[4 * rr + 3]);
    __syncthreads();
  } else {
    tok0 = read_index(p.cu, p.idx_i64, b);
    tok1 = read_index(p.cu, p.idx_i64, b + 1);
    prefix = read_index(p.prefix, p.idx_i64, b);
  }
  const int64_t n_new = min64(pp.max_new, min64(tok1, p.total) - tok0);
  const int64_t ct0 = static_cast<int64_t>(gridDim.x) - 1 - blockIdx.x;
  const int64_t x0 = ct0 * COLS;  // first column of the workgroup
  if (tok0 < 0 || x0 >= n_new * p.G) return;
  const int64_t last = min64(n_new * p.G, x0 + COLS) - 1;  // columns fit 31 bits
  const int64_t kv_end = keys_of(p, prefix, last);          // keys that any column sees
  const int64_t first_new = over_group(p, static_cast<uint32_t>(x0));
  const int64_t first_pos = prefix + first_new;  // every column sees the keys up to here
  const int64_t runs = (kv_end + kv8::kRun - 1) / kv8::kRun;
  const int64_t all_tiles = (kv_end + kTile - 1) / kTile;
  int64_t kt0 = 0, kt1 = all_tiles;
  int parts = 1;
  if (pp.splits > 1) {
    parts = parts_of(pp, all_tiles);
    if (static_cast<int>(blockIdx.z) >= parts) return;
    kt0 = all_tiles * blockIdx.z / parts;
    kt1 = all_tiles * (blockIdx.z + 1) / parts;
  }
  const uint8_t* kb = p.kpool + g * p.sG;
  const uint8_t* vb = p.vpool + g * p.sG;

  // columns and their positions past first_pos
  const int n_cols = static_cast<int>(last - x0) + 1;
  // A column as a token past the workgroup's first one and a head of the group, both small: offsets are 32 by 32 bits on
  // top of uniform addresses (64-bit products of every row's own were 3000 cycles of a workgroup).
  const int64_t first_tok = tok0 + first_new;
  const uint32_t x_head = static_cast<uint32_t>(x0 - (first_tok - tok0) * p.G);  // head of the workgroup's first column
  struct Place {
    uint32_t token, head;
  };
  auto place_of = [&](const auto& c, int x) {
    const uint32_t t = over_group(c, x_head + x);
    return Place{t, x_head + x - t * static_cast<uint32_t>(c.G)};
  };
  auto row_of = [](const bf16_t* base, const Place& at, int64_t st, int64_t sh) {  // strides below 2^32
    return base + (static_cast<uint64_t>(at.token) * static_cast<uint32_t>(st) + static_cast<uint64_t>(at.head) * static_cast<uint32_t>(sh));
  };
  // this lane's column as a position past first_pos
  const int ahead = static_cast<int>(place_of(p, min(pair * 32 + col, n_cols - 1)).token);

  // ---- the tiles' loads
  // Lane l of `cur` holds the offset in the head's pool of run 64 c + l (-1: not there), of `nxt` that of the next 64,
  // one vector load each 16 tiles (scalar loads of the table share their wait counter with LDS, and every tile stalled
  // about 1000 cycles for them); the masks say which runs are there.
  int64_t cur, nxt;
  uint64_t cur_mask, nxt_mask;
  auto chunk = [&](int64_t c) -> int64_t {
    const ParamsAgain q = params_again();
    const int64_t run = 64 * c + lane;
    const int64_t lb = run >> (q->c.bs_shift - 4);
    const int64_t at = (b * q->c.table_stride + min64(lb, q->c.max_blocks - 1)) << q->c.table_i64;
    const int32_t lo = reinterpret_cast<const int32_t*>(q->c.tables)[at];
    const int32_t hi = reinterpret_cast<const int32_t*>(q->c.tables)[at + q->c.table_i64];  // the entry itself where it has one word
    const bool ok = (run < runs) & (static_cast<uint32_t>(lo) < static_cast<uint32_t>(q->c.num_blocks)) & ((hi == 0) | (q->c.table_i64 == 0));
    const int64_t o = static_cast<int64_t>(ok ? lo : 0) * q->c.sP + (run & ((1 << (q->c.bs_shift - 4)) - 1)) * kv8::Run<D>::kBytes;
    return ok ? o : -1;
  };
  // A wave loads run wave % 4 of a tile: of eight, 0 to 3 its keys and 4 to 7 its values; of four, its keys and then its values.
  // One that is not there has no records and reads zeros.
  const bool of_values = kWide && wave >= 4;
  int64_t own;  // offset of that run of the tile last asked for, -1: not there
  int there;    // which runs of that tile are there
  auto offsets = [&](int64_t kt) {
    const int at = static_cast<int>(kt & 15) * kRuns;
    if (at == 0 && kt != kt0) {
      cur = nxt;
      cur_mask = nxt_mask;
      nxt = chunk((kt >> 4) + 1);
      nxt_mask = __ballot(nxt >= 0);
    }
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(cur), at + (wave & 3));
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(cur >> 32), at + (wave & 3));
    own = static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
    there = static_cast<int>(cur_mask >> at) & 15;
  };
  uint4 stage[N];
  uint32_t stage_scale;
  auto ask = [&](const uint8_t* pool, int64_t at) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(pool + (at < 0 ? 0 : at)), 0, at < 0 ? 0 : kv8::Run<D>::kBytes, 0x00020000);
#pragma unroll
    for (int s = 0; s < N; ++s) stage[s] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, 16 * lane + 1024 * s, 0, kShared));
    stage_scale = __builtin_amdgcn_raw_buffer_load_b8(r, kv8::Run<D>::kCodes, 0, kShared);
  };
  // What of the stage no column sees leaves the product.  A NaN among what not every column sees leaves it too: 0 times it is
  // one.  It is marked at the end for the columns that see it.
  const int64_t first_mixed = (first_pos + 1) / kTile;  // the first tile that not every column sees whole
  auto nans_of = [](uint32_t w) -> uint32_t { return ((w & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u; };  // 1 in each byte 0x7f or 0xff
  auto trim = [&](int64_t kt) {
    if (kt < first_mixed) return;
    const uint32_t mask = tokens_mask(kv_end - kt * kTile - kv8::kRun * (wave & 3) - 4 * (lane >> 4));  // past it the pool may hold anything
    uint32_t any = 0;
    auto clean = [&](uint32_t& w) {
      w &= mask;
      const uint32_t bad = nans_of(w);
      w &= ~(bad * 255u);
      any |= bad;
    };
#pragma unroll
    for (int s = 0; s < N; ++s) {
      clean(stage[s].x);
      clean(stage[s].y);
      clean(stage[s].z);
      clean(stage[s].w);
    }
    if (any != 0) *s_flag = 1;
  };
  auto put = [&](bool values, int i) {
    const int buf = values ? i & (S::kValueBufs - 1) : i & (S::kKeyBufs - 1);
    if (values) trim(kt0 + i);
    uint4* dst = reinterpret_cast<uint4*>(smem + (values ? S::kValues : 0) + (buf * kRuns + (wave & 3)) * S::kRunBytes) + lane;
#pragma unroll
    for (int s = 0; s < N; ++s) dst[64 * s] = stage[s];
    if (lane == 0) (values ? s_vscale : s_kscale)[buf * kRuns + (wave & 3)] = kv8::scale_of(stage_scale);
  };

  float m_run = -INFINITY, l_run = 0.f, corr = 1.f;  // of the lane's column; corr: what the sums are still to be multiplied with
  floatx16_v o[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) o[m] = floatx16_v(0.f);

  // The output leaves through LDS as whole rows, a lane eight dims: the first half of the columns, then the other
  constexpr int kLanes = D / 8;  // of a row
  constexpr int kRowsAtOnce = 64 * kWaves / kLanes;
  constexpr int kSweeps = COLS / 2 / kRowsAtOnce;
  const int in_row = tid % kLanes;
  auto column_of = [&](int pass, int i) {
    return COLS / 2 * pass + tid / kLanes + i * kRowsAtOnce;
  };
  uint4 gate[2][kSweeps];
  auto ask_gate = [&](ParamsAgain late) {
    if (late->c.gate == nullptr || parts > 1) return;
    const bf16_t* base = late->c.gate + first_tok * late->c.gate_st + static_cast<int64_t>(g) * late->c.G * late->c.gate_sh;
#pragma unroll
    for (int pass = 0; pass < 2; ++pass)
#pragma unroll
      for (int i = 0; i < kSweeps; ++i) {
        const Place at = place_of(late->c, min(column_of(pass, i), n_cols - 1));
        const uint2* src = reinterpret_cast<const uint2*>(row_of(base, at, late->c.gate_st, late->c.gate_sh) + 8 * in_row);
        const uint2 lo = src[0], hi = src[1];
        gate[pass][i] = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
  };
  if (kt0 < kt1) {
    if (tid == 0) *s_flag = 0;
    // the query: lane 32 h + n has dims 64 s + 16 (h + 2 e) .. + 15 of column n, as the keys' lanes have them
    bf16x8_v q[4 * N];
    {
      const int x = pair * 32 + col;
      const bf16_t* base = p.q + first_tok * p.q_st + static_cast<int64_t>(g) * p.G * p.q_sh;
      const uint4* row = reinterpret_cast<const uint4*>(row_of(base, place_of(p, min(x, n_cols - 1)), p.q_st, p.q_sh) + 16 * hi);
#pragma unroll
      for (int f = 0; f < 2 * N; ++f)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint4 u = row[4 * f + e];
          if (x >= n_cols) u = make_uint4(0, 0, 0, 0);
          q[2 * f + e] = __builtin_bit_cast(bf16x8_v, u);
        }
    }
    cur = chunk(kt0 >> 4);
    nxt = chunk((kt0 >> 4) + 1);
    cur_mask = __ballot(cur >= 0);
    nxt_mask = __ballot(nxt >= 0);
    const float qk_scale = p.scale * kLog2e;
    const int n = static_cast<int>(kt1 - kt0);
    offsets(kt0);
    const uint8_t* own_pool = of_values ? vb : kb;
    ask(own_pool, own);
    int64_t own_keys = own;    // of the tile asked for last, its keys'
    int64_t own_values = own;  // of the tile before it, its values'
    int there_next = there;
    lds_barrier();  // the flag
    put(of_values, 0);
    lds_barrier();  // the first tile
    float top = 0.f;  // the largest score of the lane's column in this wave's half of the tile whose probabilities come next
    const unsigned char* key_lane = smem + 2 * (wave & 1) * S::kRunBytes + (col >> 4) * S::kRunBytes + hi * 256 + (col & 15) * 16;
    // o[m] has row 8 (r >> 2) + 4 h + (r & 3) = chunk c of 16 slice + c, dim 64 slice + 4 c + m of the wave's half (D = 256: slices 2
    // and 3 are the second half; D = 128: m 2 and 3 are)
    constexpr int kHalf = D == 256 ? 2 * 1024 : 8;
    const unsigned char* value_lane = smem + S::kValues + (wave & 1) * kHalf + (col >> 4) * 1024 + hi * 256 + (col & 15) * 16;
    uint4* p_own = reinterpret_cast<uint4*>(smem + S::kP) + wave * 128 + lane;
    // masks the scores of tile i and tells the pair their largest
    auto largest = [&](int i, int have, floatx16_v& x) {
      const int64_t key0 = (kt0 + i) * kTile;
      if (!(key0 + kTile <= first_pos + 1 && have == 15)) {
        const int lim = static_cast<int>(max64(-1, min64(kTile - 1, min64(first_pos + ahead, kv_end - 1) - key0))) - 32 * (wave & 1);  // the last key the column sees
        const int runs2 = have >> (2 * (wave & 1));
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (8 * (r >> 2) + 4 * hi + (r & 3) > lim || !(runs2 >> (r >> 3) & 1)) x[r] = -INFINITY;
      }
      float mx = fmaxf(x[0], x[1]);
#pragma unroll
      for (int r = 2; r < 16; ++r) mx = fmaxf(mx, x[r]);
      const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
      top = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
      if (hi == 0) s_max[((i & (S::kPBufs - 1)) * kWaves + wave) * 32 + col] = top;
    };
    // Iteration i: the probabilities of tile i between the products of tile i - 1's values, then the scores of tile i + 1.
    constexpr int kValues = 4 * MT;  // products of a tile's values
    floatx16_v sc;
    auto iterate = [&](int i, auto has_scores, auto has_probs, auto has_values) {
      if constexpr (kWide && has_scores) {
        offsets(kt0 + i + 2);
        ask(own_pool, own);
      }
      const unsigned char* vat = value_lane + ((i - 1) & (S::kValueBufs - 1)) * S::kTileBytes;
      const float* vsc = s_vscale + ((i - 1) & (S::kValueBufs - 1)) * kRuns;
      const uint4* pat = p_own + ((i - 1) & (S::kPBufs - 1)) * kWaves * 128 - (wave & 1) * 128;  // runs 0 and 1 are the first wave's of the pair
      uint32_t vlo[2][MT], vup[2][MT];
      float vscale[2];
      bf16x8_v pv[2];
      auto ask_values = [&](int r) {
        vscale[r & 1] = vsc[r];
        pv[r & 1] = __builtin_bit_cast(bf16x8_v, pat[(r >> 1) * 128 + 64 * (r & 1)]);
        if constexpr (D == 256) {
          const uint4 a = *reinterpret_cast<const uint4*>(vat + r * S::kRunBytes), c = *reinterpret_cast<const uint4*>(vat + r * S::kRunBytes + 512);
          vlo[r & 1][0] = a.x, vlo[r & 1][1] = a.y, vlo[r & 1][2] = a.z, vlo[r & 1][3] = a.w;
          vup[r & 1][0] = c.x, vup[r & 1][1] = c.y, vup[r & 1][2] = c.z, vup[r & 1][3] = c.w;
        } else {
          const uint2 a = *reinterpret_cast<const uint2*>(vat + r * S::kRunBytes), c = *reinterpret_cast<const uint2*>(vat + r * S::kRunBytes + 512);
          vlo[r & 1][0] = a.x, vlo[r & 1][1] = a.y;
          vup[r & 1][0] = c.x, vup[r & 1][1] = c.y;
        }
      };
      if constexpr (has_values) {
        ask_values(0);
        if (__ballot(corr != 1.f) != 0) {  // columns whose reference point moved at the tile whose products come now
#pragma unroll
          for (int m = 0; m < MT; ++m) o[m] *= corr;
        }
      }
      // ---- the reference points of tile i: both waves of a pair move their columns' alike
      float use = 0.f;
      if constexpr (has_probs) {
        const float mx = fmaxf(top, s_max[((i & (S::kPBufs - 1)) * kWaves + (wave ^ 1)) * 32 + col]) * qk_scale;
        corr = 1.f;
        if (__ballot(mx > m_run + kLazy) != 0) {
          const float m_new = fmaxf(m_run, mx);
          corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
          m_run = m_new;
          l_run *= corr;
        }
        use = m_run == -INFINITY ? 0.f : m_run;
      }
      // a wave in its value products goes ahead of its neighbour on the SIMD that is at its scores: 1034 us against 1048 without
      // priorities and 1052 the other way round, 2048 tokens behind 32000
      __builtin_amdgcn_s_setprio(1);
      bf16x8_v pb[2];
#pragma unroll
      for (int f = 0; f < kValues; ++f) {
        if constexpr (has_values) {
          const int r = f / MT, m = f % MT;
          if (m == 0 && r + 1 < kRuns) ask_values(r + 1);
          o[m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand(vlo[r & 1][m], vup[r & 1][m], vscale[r & 1], vscale[r & 1]), pv[r & 1], o[m], 0, 0, 0);
        }
        if constexpr (has_probs) {
#pragma unroll
          for (int r = f * (16 / kValues); r < (f + 1) * (16 / kValues); ++r) {
            const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], qk_scale, -use));
            l_run += pr;
            pb[r >> 3][r & 7] = static_cast<__bf16>(pr);  // for the bf16 product; l_run has it unrounded
            if (kWide && (r & 7) == 7) p_own[(i & (S::kPBufs - 1)) * kWaves * 128 + 64 * (r >> 3)] = __builtin_bit_cast(uint4, pb[r >> 3]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (!kWide && has_probs) {
        if constexpr (has_scores) put(false, i + 1);
        ask(vb, own_values);
        lds_barrier();
#pragma unroll
        for (int r = 0; r < 2; ++r) p_own[64 * r] = __builtin_bit_cast(uint4, pb[r]);
      }
      if constexpr (has_scores) {
        const int kbuf = (i + 1) & (S::kKeyBufs - 1);
        const unsigned char* kat = key_lane + kbuf * S::kTileBytes;
        const float kscale = s_kscale[kbuf * kRuns + 2 * (wave & 1) + (col >> 4)];
        uint4 kc[3];
        kc[0] = *reinterpret_cast<const uint4*>(kat);
        kc[1] = *reinterpret_cast<const uint4*>(kat + 512);
        __builtin_amdgcn_s_setprio(0);
        sc = floatx16_v(0.f);
#pragma unroll
        for (int f = 0; f < 2 * N; ++f) {
          const uint4 u = kc[f % 3];
          if (f + 2 < 2 * N) kc[(f + 2) % 3] = *reinterpret_cast<const uint4*>(kat + 512 * (f + 2));
          sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand(u.x, u.y, kscale, kscale), q[2 * f], sc, 0, 0, 0);
          sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand(u.z, u.w, kscale, kscale), q[2 * f + 1], sc, 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if constexpr (!kWide && has_probs) {
        put(true, i);
      }
      if constexpr (has_scores) {
        largest(i + 1, there_next, sc);
        if constexpr (!kWide) {
          own_values = own_keys;
          offsets(kt0 + i + 2);
          own_keys = own;
          ask(kb, own);
        }
        there_next = there;
        if constexpr (kWide) {
          put(of_values, i + 2);
        }
      }
      if constexpr (has_probs || has_scores) lds_barrier();
    };
    using yes = std::integral_constant<bool, true>;
    using no = std::integral_constant<bool, false>;
    iterate(-1, yes{}, no{}, no{});  // the first scores
    if (n > 1) {
      iterate(0, yes{}, yes{}, no{});
      for (int i = 1; i + 1 < n; ++i) iterate(i, yes{}, yes{}, yes{});
      iterate(n - 1, no{}, yes{}, yes{});
    } else {
      iterate(0, no{}, yes{}, no{});
    }
    iterate(n, no{}, no{}, yes{});

    // ---- NaNs among keys that not every column sees: products of their places with what each column sees
    if (*s_flag != 0) {
      uint16_t* s_nans = reinterpret_cast<uint16_t*>(smem);  // [run][slice][lane]: a bit a code
      for (int64_t kt = max64(kt0, first_mixed); kt < kt1; ++kt) {
        __syncthreads();
        if (wave < kRuns) {
          const ParamsAgain again = params_again();
          const int64_t run = kt * kRuns + wave;
          const int32_t id = block_of_run(again->c, b, run, runs);
          const uint4* at = reinterpret_cast<const uint4*>(vb + static_cast<int64_t>(max(id, 0)) * again->c.sP + (run & ((1 << (again->c.bs_shift - 4)) - 1)) * kv8::Run<D>::kBytes) + lane;
          const uint32_t mask = id < 0 ? 0u : tokens_mask(kv_end - run * kv8::kRun - 4 * (lane >> 4));
#pragma unroll
          for (int s = 0; s < N; ++s) {
            const uint4 u = at[64 * s];
            uint32_t bits = 0;
#pragma unroll
            for (int m = 0; m < 4; ++m) bits |= ((nans_of(dword(u, m) & mask) * 0x10204080u) >> 28) << (4 * m);  // a dword's four side by side, token t at bit t
            s_nans[(wave * N + s) * 64 + lane] = static_cast<uint16_t>(bits);
          }
        }
        __syncthreads();
        const uint16_t* at = s_nans + ((D == 256 ? 2 * (wave & 1) : 0) + (col >> 4)) * 64 + hi * 16 + (col & 15);
        const int seen = static_cast<int>(max64(-1, min64(kTile, first_pos + ahead - kt * kTile)));  // the last key of the tile that the column sees
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int shift = 4 * m + (D == 256 ? 0 : 8 * (wave & 1));
          floatx16_v found = floatx16_v(0.f);
          for (int r = 0; r < kRuns; ++r) {
            const uint32_t lo = at[r * N * 64] >> shift, up = at[r * N * 64 + 32] >> shift;
            bf16x8_v there, sees;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              there[e] = static_cast<__bf16>(static_cast<float>((e < 4 ? lo : up) >> (e & 3) & 1));
              sees[e] = static_cast<__bf16>(16 * r + 8 * (e >> 2) + 4 * hi + (e & 3) <= seen ? 1.f : 0.f);
            }
            found = __builtin_amdgcn_mfma_f32_32x32x16_bf16(there, sees, found, 0, 0, 0);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (found[r] > 0.f) o[m][r] = __uint_as_float(0x7fc00000u);
        }
      }
    }
  }

  // ---- out, through LDS
  const ParamsAgain late = params_again();
  const int64_t row0 = first_tok * late->c.H + static_cast<int64_t>(g) * late->c.G;  // of the output
  ask_gate(late);
  __syncthreads();
  float* s_l = s_max;  // [half][column]; then the reference points
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
  if (hi == 0) {
    s_l[(wave & 1) * COLS + 32 * pair + col] = __uint_as_float(both[0]) + __uint_as_float(both[1]);
    s_l[2 * COLS + 32 * pair + col] = m_run;  // of either wave, the same
  }
  constexpr int kRowFloats = D + 4;
  static_assert(COLS / 2 * kRowFloats * 4 <= S::kMax, "half of the columns fit below the sums");
  float* s_o = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    if (pass == 1) lds_barrier();  // the first columns have been read
    if (pair / (COLS / 64) == pass) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float* row = s_o + (32 * (pair % (COLS / 64)) + col) * kRowFloats + 64 * (r >> 3) + 4 * (8 * (r >> 2 & 1) + 4 * hi + (r & 3));
        if constexpr (D == 256)
          *reinterpret_cast<floatx4_v*>(row + 128 * (wave & 1)) = floatx4_v{o[0][r], o[1][r], o[2][r], o[3][r]};
        else
          *reinterpret_cast<floatx2_v*>(row + 2 * (wave & 1)) = floatx2_v{o[0][r], o[1][r]};
      }
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < kSweeps; ++i) {
      const int x = column_of(pass, i);
      if (x >= n_cols) continue;
      const float* at = s_o + (tid / kLanes + i * kRowsAtOnce) * kRowFloats;
      const Place pl = place_of(late->c, x);
      const uint32_t row = pl.token * static_cast<uint32_t>(late->c.H) + pl.head;  // past row0
      const float l = s_l[x] + s_l[COLS + x];
      if (parts > 1) {
        const int64_t part = (blockIdx.z * late->part_tokens + part_base(*late, b, tok0) - tok0) * late->c.H + row0 + row;
        if (in_row == 0) *reinterpret_cast<float2*>(late->part_ml + part * 2) = make_float2(s_l[2 * COLS + x], l);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          *reinterpret_cast<floatx4_v*>(late->part_o + part * D + 4 * in_row + k * D / 2) = *reinterpret_cast<const floatx4_v*>(at + 4 * in_row + k * D / 2);
        continue;
      }
      const float over = l == 0.f ? 0.f : 1.f / l;  // a query that saw nothing has sums of 0
      const floatx4_v lo = *reinterpret_cast<const floatx4_v*>(at + 8 * in_row), hi = *reinterpret_cast<const floatx4_v*>(at + 8 * in_row + 4);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (e < 4 ? lo[e & 3] : hi[e & 3]) * over;
      if (late->c.gate != nullptr) {
        const uint32_t w[4] = {gate[pass][i].x, gate[pass][i].y, gate[pass][i].z, gate[pass][i].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= sigmoid(__uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16));
      }
      uint32_t out[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = static_cast<uint32_t>(f32_to_bf16(v[2 * e])) | static_cast<uint32_t>(f32_to_bf16(v[2 * e + 1])) << 16;
      *reinterpret_cast<uint4*>(late->c.out + row0 * D + (static_cast<uint64_t>(row) * D + 8 * in_row)) = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
}

template <int D, int COLS>
static int launch(const PrefillParams& p, hipStream_t stream) {
  using S = Smem<D, COLS>;
  if (int rc = reserve_lds<&prefill_kernel<D, COLS>>("paged_attention_prefill_kv8", S::kBytes)) return rc;
  {
    KernelTimer timer_("prefill_kv8", stream);
    const dim3 grid(static_cast<unsigned>(ceil_div(p.max_new * p.c.G, COLS)), static_cast<unsigned>(p.c.B * p.c.Hkv), static_cast<unsigned>(p.splits));
    hipLaunchKernelGGL((prefill_kernel<D, COLS>), grid, dim3(64 * S::kWaves), S::kBytes, stream, p);
  }
  if (int rc = check_launch("paged_attention_prefill_kv8")) return rc;
  return join<D, COLS>(p, "paged_attention_prefill_kv8", "prefill_kv8_join", stream);
}

// Columns of a workgroup.  64, two workgroups a CU, end sooner where the keys are few, and start sooner; 128 read each key half as
// often.  us with 64 / 128, D = 256, 16 heads, rows x new tokens behind cached ones: 1 x 64 behind none 12.4 / 17.0, 1 x 512 23.2 /
// 29.1, 8 x 512 46.5 / 52.3, 2 x 256 behind 500 33.7 / 36.6, 64 x 8 behind 1000 35.8 / 43.3, 1 x 512 behind 2000 49.3 / 48.0 and behind
// 8000 96.2 / 91.6, 16 x 128 behind 500 38.6 / 37.7 and behind 4000 158 / 147, 1 x 4096 behind 4096 433 / 405.  D = 128, 20 heads, 4 of
// keys: 1 x 512 17.2 / 20.6, 16 x 128 behind 4000 175 / 181, 1 x 4096 behind 4096 393 / 393, 1 x 512 behind 8000 80.3 / 77.3.
static int columns_of(int64_t batch, int kv_heads, int group, int64_t max_new, int head_dim, int64_t max_tokens) {
  return head_dim == 128 || max_tokens <= 1024 || workgroups_of(batch, kv_heads, group, max_new, 128) <= 64 ? 64 : 128;
}

}  // namespace prefill8
}  // namespace qa

extern "C" int64_t qa_paged_attention_prefill_kv8_workspace(int64_t total_new, int64_t batch, int64_t max_new, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                                            int64_t max_tokens) {
  // of either number of columns, so that tables narrower than these need no more
  return std::max(qa::attn::workspace_bytes_of(total_new, batch, max_new, heads, kv_heads, head_dim, max_tokens, 64),
                  qa::attn::workspace_bytes_of(total_new, batch, max_new, heads, kv_heads, head_dim, max_tokens, 128));
}

extern "C" int qa_paged_attention_prefill_kv8(const void* query, int32_t q_dtype, int64_t q_stride_t, int64_t q_stride_h, int64_t total_new, const void* cu_seqlens,
                                              const void* prefix_lens, int32_t idx_dtype, int64_t batch, int64_t max_new, int32_t heads, int32_t head_dim,
                                              const qa_paged_kv* kv, const void* block_tables, int32_t table_dtype, int64_t table_stride, int64_t max_blocks,
                                              int32_t block_size, float scale, const void* gate, int64_t gate_stride_t, int64_t gate_stride_h, void* output,
                                              void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  using namespace qa;
  using namespace qa::prefill8;
  PrefillParams p{};
  const Args a{"paged_attention_prefill_kv8", query, q_dtype, q_stride_t, q_stride_h, total_new, batch, heads, head_dim, kv, block_tables, table_dtype, table_stride, max_blocks,
               idx_dtype, block_size, scale, gate, gate_stride_t, gate_stride_h, output};
  if (int rc = fill(p.c, a)) return rc;
  const int cols = columns_of(batch, p.c.Hkv, p.c.G, std::min(max_new, total_new), head_dim, max_blocks * block_size);
  if (int rc = share_out(p, a, cu_seqlens, prefix_lens, max_new, workspace, workspace_bytes, cols)) return rc;
  if (p.max_new == 0) return 0;
  if (head_dim == 128) return launch<128, 64>(p, stream);
  return cols == 64 ? launch<256, 64>(p, stream) : launch<256, 128>(p, stream);
}
