// Chunked causal prefill attention over the 4-bit paged KV cache (attention_kv4.h, kv4.h), gfx950.
//
// Columns of the products are (new position, query head of the KV head's group), position-major, so any group size
// fills them.  A workgroup owns 128 of one row and KV head and walks the keys in tiles of 64.  Its eight waves are four
// pairs of 32 columns.  A wave takes the scores and the softmax of 16 of them, then the products with the values of all
// 32 for half of the dims, with its partner's probabilities through LDS: so that each operand of values read from LDS
// feeds two products (with 16 columns and all dims a wave, LDS would be as busy as the matrix units), and the
// accumulators of a wave stay at 64 registers, two waves to a SIMD (with 32 columns and all dims in one wave a SIMD,
// accumulators and query took 512 registers, 300 moves a tile between the two halves of the file: 1571 us where this
// form took 895, 2048 tokens behind 32000).
//
// Keys go from memory into LDS as they are, two tiles ahead, 1 KB a wave through its registers (with each wave loading
// all of them the vector memory path was busy longer than the matrix units: 1328 us; copies straight to LDS each held
// their wave for about 450 cycles).  Values are unpacked once a workgroup: waves 0 to 3, one a
// SIMD, turn a run of the next tile each into bf16 operand fragments in LDS, [unit of 32 keys][dim tile][run][lane][8
// bytes], read back without bank conflicts.
//
// Iteration t, one barrier: scores and softmax of tile t + 1, products of tile t's values, unpacking of tile t + 1's.
//
// With few columns the keys are split over gridDim.z and a second launch joins the parts.
//
// Bound by the matrix and vector units together.  16 heads of 256 over 2: 2048 tokens behind 32000 856 us, 1300 TFLOP/s of
// the two products (a large bf16 library product runs at 1210), eight chunks of 512 behind up to 8k 283 us, 1090; five
// prompts of up to 700, 20 heads of 128 over 4, 29 us: a workgroup's start and end are 10 of them and its longest row 13.
#include "attention_kv4.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace qa {
namespace prefill4 {

using namespace attn4;

struct PrefillParams {
  Params c;
  int64_t max_new;  // tokens of a row that are computed
  int splits;       // parts of the keys that the launch has workgroups for
  float per_tile;   // kPerTile / workgroups
  int64_t part_tokens;  // tokens that the partial results have room for
  int64_t per_row;      // 0: a token's are where its query is; else row b's begin at b per_row (a padded query)
  float* part_o;        // (splits, part_tokens, H, D)
  float* part_ml;       // (splits, part_tokens, H, 2)
};

constexpr int kTile = 64;      // keys
constexpr int kRuns = kTile / kv4::kRun;
constexpr int kWaves = 8;
constexpr int kCols = kWaves * 16;
constexpr int kMaxSplits = 64;
// Batches up to this many rows start with the longest row, so that the launch ends on short ones: 60 rows of up to 300 new
// tokens behind up to 4000 439 -> 403 us, 12 of up to 1500 behind up to 8000 738 -> 677; 64 equal rows of 16 64.5 -> 65.8.
constexpr int kRankRows = 64;

// Keys that the columns up to the last, of a row with `prefix` cached tokens, see: not past the table.
template <typename P>
__device__ __forceinline__ int64_t keys_of(const P& p, int64_t prefix, int64_t last) {
  return max64(0, min64(prefix + over_group(p, static_cast<uint32_t>(last)) + 1, p.max_blocks << p.bs_shift));
}

// Where the partial results of row b begin, its first token being tok0.
template <typename P>
__device__ __forceinline__ int64_t part_base(const P& pp, int64_t b, int64_t tok0) { return pp.per_row != 0 ? b * pp.per_row : tok0; }

// Parts that `tiles` tiles are split into, the same in both launches: the tables may be much wider than the row.
template <typename P>
__device__ __forceinline__ int parts_of(const P& pp, int64_t tiles) {
  const float best = __builtin_sqrtf(pp.per_tile * static_cast<float>(tiles));
  return max(1, min(min(pp.splits, static_cast<int>(best)), static_cast<int>(min64(tiles, kMaxSplits))));
}

template <int D>
struct Smem {
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kP = 2 * kTileBytes;                    // probabilities: [buffer][wave][unit][lane][16 bytes]
  static constexpr int kCorr = kP + 2 * kWaves * 2 * 1024;     // [buffer][wave][16] floats
  static constexpr int kFlag = kCorr + 2 * kWaves * 16 * 4;    // [buffer]: the last tile that had a NaN group
  static constexpr int kKeys = kFlag + 16;                     // [buffer][run]: codes; then [buffer][run]: scales
  static constexpr int kRunCodes = kv4::Run<D>::kCodes;
  static constexpr int kRunScales = kv4::Run<D>::kBytes - kRunCodes;
  static constexpr int kScales = kKeys + 2 * kRuns * kRunCodes;
  static constexpr int kBytes = kScales + 2 * kRuns * kRunScales;
};

// The products stay where they are written: the compiler would move them to where their sums are used.
__device__ __forceinline__ void keep(floatx4_v (&s)[kRuns]) { asm volatile("" : "+v"(s[0]), "+v"(s[1]), "+v"(s[2]), "+v"(s[3])); }

// The launch's parameters, read again: what only the start, the end or every sixteenth tile needs does not stay in scalar
// registers over the loop, which else spilled 46 of them to vector lanes and read them back each tile.
typedef const __attribute__((address_space(4))) PrefillParams* ParamsAgain;
__device__ __forceinline__ ParamsAgain params_again() {
  ParamsAgain p = (ParamsAgain)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

template <int D>
__global__ __launch_bounds__(64 * kWaves, 2) void prefill_kernel(PrefillParams pp) {
  const Params& p = pp.c;
  constexpr int MT = D / 16;
  constexpr int MH = MT / 2;        // dim tiles of a wave
  using S = Smem<D>;
  extern __shared__ __align__(16) unsigned char smem[];
  float* s_corr = reinterpret_cast<float*>(smem + S::kCorr);
  int* s_flag = reinterpret_cast<int*>(smem + S::kFlag);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = wave & 1;
  const int col = lane & 15;
  const int quad = lane >> 4;

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
  const int64_t x0 = ct0 * kCols;  // first column of the workgroup
  if (tok0 < 0 || x0 >= n_new * p.G) return;
  const int64_t last = min64(n_new * p.G, x0 + kCols) - 1;  // columns fit 31 bits
  const int64_t kv_end = keys_of(p, prefix, last);          // keys that any column sees
  const int64_t first_new = over_group(p, static_cast<uint32_t>(x0));
  const int64_t first_pos = prefix + first_new;  // every column sees the keys up to here
  const int64_t runs = (kv_end + kv4::kRun - 1) / kv4::kRun;
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

  // columns: [0] the wave's own 16, [1] its partner's; their position past first_pos
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
  int ahead[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) ahead[c] = static_cast<int>(place_of(p, min((wave ^ c) * 16 + col, n_cols - 1)).token);

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
    const int64_t o = static_cast<int64_t>(ok ? lo : 0) * q->c.sP + (run & ((1 << (q->c.bs_shift - 4)) - 1)) * kv4::Run<D>::kBytes;
    return ok ? o : -1;
  };
  // A wave loads only run `wave % 4` of a tile: waves 0 to 3 its values and half of its keys' codes, waves 4 to 7 the
  // rest of its keys.
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
  // That run as a buffer; one that is not there has no records and reads zeros.
  auto rsrc = [&](const uint8_t* base) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base + (own < 0 ? 0 : own)), 0, own < 0 ? 0 : kv4::Run<D>::kBytes, 0x00020000);
  };
  // The wave's part of a tile's keys on its way to LDS: 1 KB of codes (at D = 128 only waves 4 to 7), the waves that do
  // not unpack a run's scales too.
  constexpr int PER = D / 128;  // KB of codes of a run
  uint4 kcode = make_uint4(0, 0, 0, 0);
  uint32_t kscale = 0;
  auto fetch_keys = [&]() {
    const __amdgpu_buffer_rsrc_t r = rsrc(kb);
    const int part = PER == 2 ? wave >> 2 : 0;
    if (PER == 2 || wave >= 4) kcode = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, 1024 * part + 16 * lane, 0, 0));
    if (wave >= 4) kscale = __builtin_amdgcn_raw_buffer_load_b32(r, S::kRunCodes + 4 * (lane % (S::kRunScales / 4)), 0, 0);
  };
  auto store_keys = [&](int buf) {
    const int part = PER == 2 ? wave >> 2 : 0;
    if (PER == 2 || wave >= 4) *reinterpret_cast<uint4*>(smem + S::kKeys + (buf * kRuns + (wave & 3)) * S::kRunCodes + 1024 * part + 16 * lane) = kcode;
    if (wave >= 4 && lane < S::kRunScales / 4) *reinterpret_cast<uint32_t*>(smem + S::kScales + (buf * kRuns + (wave & 3)) * S::kRunScales + 4 * lane) = kscale;
  };
  const bool unpacks = wave < 4;
  ValueRun<D> vr;
  auto fetch_values = [&]() { load_values<D, kShared>(vr, rsrc(vb), lane); };
  // what of vr no column sees, or not every column where it is NaN, leaves the product
  auto trim = [&](int64_t kt, int buf) {
    if (kt * kTile + kTile <= first_pos + 1) return;  // every column sees all of the tile
    // keys that no column sees may hold anything, and 0 times a NaN is one
    const int64_t left = kv_end - kt * kTile - kv4::kRun * wave - 4 * quad;
    vr.scale &= left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * static_cast<int>(left))) - 1u;
    // a NaN group reaches only the columns that see its token: marked for them below
    uint32_t drop = 0;
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if ((vr.scale >> (8 * t) & 255u) == 255u) drop |= 255u << (8 * t);
    vr.scale &= ~drop;
    if (drop != 0) s_flag[buf] = static_cast<int>(kt - kt0) + 1;
  };
  // Byte e of the lane's chunk of vr's four tokens: dims 2 e and 2 e + 1, converted and written to buffer buf.  A
  // fragment is two planes of 512 bytes, one a run, so that neither the writes nor the reads conflict on banks.
  float vs[4];
  auto unpack_byte = [&](int e, int buf) {
    uint32_t pair[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (e == 0) vs[t] = value_scale(vr.scale, t);
      const int at = t * (D / 128) + (e >> 2);  // dword of the lane's chunk of token t
      const uint4& c = vr.code[at >> 2];
      const uint32_t w = (at & 3) == 0 ? c.x : (at & 3) == 1 ? c.y : (at & 3) == 2 ? c.z : c.w;
      switch (e & 3) {
        case 0: pair[t] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, vs[t], 0)); break;
        case 1: pair[t] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, vs[t], 1)); break;
        case 2: pair[t] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, vs[t], 2)); break;
        default: pair[t] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, vs[t], 3)); break;
      }
    }
    uint2* dst = reinterpret_cast<uint2*>(smem + buf * S::kTileBytes) + ((wave >> 1) * MT + 2 * e) * 128 + 64 * (wave & 1) + lane;
    dst[0] = make_uint2(__builtin_amdgcn_perm(pair[1], pair[0], 0x05040100u), __builtin_amdgcn_perm(pair[3], pair[2], 0x05040100u));
    dst[128] = make_uint2(__builtin_amdgcn_perm(pair[1], pair[0], 0x07060302u), __builtin_amdgcn_perm(pair[3], pair[2], 0x07060302u));
  };
  constexpr int kBytesOfChunk = D / 32;

  float m_run = -INFINITY, l_run = 0.f;  // of the own column
  floatx4_v o[2][MH];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int i = 0; i < MH; ++i) o[c][i] = floatx4_v{0.f, 0.f, 0.f, 0.f};
  uint32_t nan_rows = 0;  // bit 4 c + r: column c saw a NaN group at the dims of accumulator row r

  // The output leaves through LDS as whole rows (31 us against 33 for five prompts of up to 700: as pieces of 8 bytes its
  // stores kept the address unit busy), a lane eight dims: rows of column tiles 0 2 4 6 first, then of 1 3 5 7
  constexpr int kLanes = D / 8;  // of a row
  constexpr int kRowsAtOnce = 64 * kWaves / kLanes;
  constexpr int kSweeps = kCols / 2 / kRowsAtOnce;
  const int in_row = tid % kLanes;
  auto column_of = [&](int pass, int i) {
    const int at = tid / kLanes + i * kRowsAtOnce;
    return (2 * (at >> 4) + pass) * 16 + (at & 15);
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
    if (tid < 2) s_flag[tid] = 0;
    // what the first tiles need is asked for before any of it is waited for: the query, the table, then two tiles' keys
    QueryRow<D> row;
    {
      const int x = wave * 16 + col;
      const bf16_t* base = p.q + first_tok * p.q_st + static_cast<int64_t>(g) * p.G * p.q_sh;
      row.ask(x < n_cols ? row_of(base, place_of(p, x), p.q_st, p.q_sh) : nullptr, quad);
    }
    cur = chunk(kt0 >> 4);
    nxt = chunk((kt0 >> 4) + 1);
    cur_mask = __ballot(cur >= 0);
    nxt_mask = __ballot(nxt >= 0);
    offsets(kt0);
    int there_cur = there;
    fetch_keys();
    const uint4 kcode0 = kcode;
    const uint32_t kscale0 = kscale;
    if (unpacks) fetch_values();
    offsets(kt0 + 1);
    int there_next = there;
    fetch_keys();
    const uint4 kcode1 = kcode;
    const uint32_t kscale1 = kscale;
    kcode = kcode0;
    kscale = kscale0;
    QueryCols<D> qh, ql;
    row.widen();
    row.template split<false>(qh);
    row.template split<true>(ql);
    const float qk_scale = p.scale * kLog2e;
    floatx4_v sc[kRuns];
    float use = 0.f;
    bf16x8_v pb[2];  // the own probabilities of the two units
    // The scores: operand f of a tile is slice f / kRuns of run f % kRuns and feeds the products of both pieces; two
    // operands go together, so that products of one accumulator do not follow each other.
    constexpr int kOperands = kRuns * (D / 128);
    auto kread = [&](int f, int buf) {
      const int j = f % kRuns, i = f / kRuns;
      const uint4 u = *reinterpret_cast<const uint4*>(smem + S::kKeys + (buf * kRuns + j) * S::kRunCodes + 1024 * i + 16 * lane);
      return int8_v{static_cast<int>(u.x), static_cast<int>(u.y), static_cast<int>(u.z), static_cast<int>(u.w), 0, 0, 0, 0};
    };
    auto sread = [&](int j, int buf) {
      const unsigned char* at = smem + S::kScales + (buf * kRuns + j) * S::kRunScales + lane * (D / 128);
      return D == 256 ? static_cast<int>(*reinterpret_cast<const uint16_t*>(at)) : static_cast<int>(*at);
    };
    auto product = [&](int f, const int8_v& a, int scale, bool lo) {
      const int j = f % kRuns, i = f / kRuns;
      const floatx4_v acc = i == 0 && !lo ? floatx4_v{0.f, 0.f, 0.f, 0.f} : sc[j];
      const int8_v& code = lo ? ql.code[i] : qh.code[i];
      const int qs = static_cast<int>(lo ? ql.scale : qh.scale);
      if (i == 0)
        sc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, code, acc, 4, 0, 0, scale, 0, qs);
      else
        sc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, code, acc, 4, 0, 1, scale, 0, qs);
    };
    static_assert(kOperands == kBytesOfChunk, "a byte of the chunk goes with each operand");
    constexpr int kAheadK = 4;
    auto scores = [&](int buf, auto slice) {
      int scale[kRuns];
#pragma unroll
      for (int j = 0; j < kRuns; ++j) scale[j] = sread(j, buf);
      int8_v ka[kAheadK];
#pragma unroll
      for (int f = 0; f < kAheadK; ++f) ka[f] = kread(f, buf);
#pragma unroll
      for (int f = 0; f < kOperands; f += 2) {
        const int8_v a0 = ka[f % kAheadK], a1 = ka[(f + 1) % kAheadK];
        product(f, a0, scale[f % kRuns], false);
        slice(f);
        __builtin_amdgcn_sched_barrier(0);
        product(f + 1, a1, scale[(f + 1) % kRuns], false);
        product(f, a0, scale[f % kRuns], true);
        if (f + kAheadK < kOperands) ka[f % kAheadK] = kread(f + kAheadK, buf);
        slice(f + 1);
        __builtin_amdgcn_sched_barrier(0);
        product(f + 1, a1, scale[(f + 1) % kRuns], true);
        if (f + 1 + kAheadK < kOperands) ka[(f + 1) % kAheadK] = kread(f + 1 + kAheadK, buf);
        __builtin_amdgcn_sched_barrier(0);
      }
      keep(sc);
    };
    // masks the scores of tile kt and moves the own column's reference point where they ask for it
    auto reference = [&](int64_t kt, int have, int buf) {
      const int64_t key0 = kt * kTile;
      if (!(key0 + kTile <= first_pos + 1 && have == 15)) {
        const int lim = static_cast<int>(max64(-1, min64(kTile - 1, min64(first_pos + ahead[0], kv_end - 1) - key0)));  // the last key the column sees
#pragma unroll
        for (int j = 0; j < kRuns; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * j + 4 * quad + r > lim || !(have >> j & 1)) sc[j][r] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < kRuns; ++j) mx = fmaxf(mx, fmaxf(fmaxf(sc[j][0], sc[j][1]), fmaxf(sc[j][2], sc[j][3])));
      mx *= qk_scale;
      float corr = 1.f;
      if (__ballot(mx > m_run + kLazy) != 0) {
        const float m_new = fmaxf(m_run, column_max(mx));
        corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_run *= corr;
        use = m_run == -INFINITY ? 0.f : m_run;
      }
      if (quad == 0) s_corr[(buf * kWaves + wave) * 16 + col] = corr;
    };
    // the probability of score k of the lane's 16
    auto prob = [&](int k) {
      const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[k >> 2][k & 3], qk_scale, -use));
      l_run += pr;
      pb[k >> 3][k & 7] = static_cast<__bf16>(pr);  // for the bf16 product; l_run has it unrounded
    };
    auto publish = [&](int buf) {
      uint4* dst = reinterpret_cast<uint4*>(smem + S::kP) + (buf * kWaves + wave) * 128 + lane;
      dst[0] = __builtin_bit_cast(uint4, pb[0]);
      dst[64] = __builtin_bit_cast(uint4, pb[1]);
    };
    store_keys(0);
    __syncthreads();  // the flags and the first tile's keys
    scores(0, [](int) {});
    reference(kt0, there_cur, 0);
#pragma unroll
    for (int k = 0; k < 16; ++k) prob(k);
    publish(0);
    if (unpacks) {
      trim(kt0, 0);
#pragma unroll
      for (int e = 0; e < kBytesOfChunk; ++e) unpack_byte(e, 0);
    }
    if (unpacks) fetch_values();
    kcode = kcode1;
    kscale = kscale1;
    store_keys(1);
    __syncthreads();

    // Iteration kt.  The products are laid between slices of the vector work that does not depend on them, with fences
    // that keep the order: the scores of tile kt + 1 with its unpacking, the values of tile kt with the exponentials.
    // (Waves 4 to 7 with the values first, half an iteration apart from the waves they share SIMDs with: no faster, 901
    // us against 895, 2048 tokens behind 32000.)
    auto iterate = [&](int64_t kt, auto more) {
      const int buf = static_cast<int>((kt - kt0) & 1);
      // a wave in its value products goes ahead of its neighbour on the SIMD that is still unpacking: 867 us against 901
      // without priorities, 878 the other way round
      __builtin_amdgcn_s_setprio(0);
      const int flag = s_flag[buf];
      const float c0 = s_corr[(buf * kWaves + wave) * 16 + col], c1 = s_corr[(buf * kWaves + (wave ^ 1)) * 16 + col];
      if constexpr (more) {
        offsets(kt + 2);
        fetch_keys();
      }
      if constexpr (more) {
        if (unpacks) {
          trim(kt + 1, buf ^ 1);
          scores(buf ^ 1, [&](int f) { unpack_byte(f, buf ^ 1); });
          fetch_values();
        } else {
          scores(buf ^ 1, [](int) {});
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      bf16x8_v pv[2][2];
      pv[0][0] = pb[0];
      pv[0][1] = pb[1];
      const uint4* src = reinterpret_cast<const uint4*>(smem + S::kP) + (buf * kWaves + (wave ^ 1)) * 128 + lane;
      pv[1][0] = __builtin_bit_cast(bf16x8_v, src[0]);
      pv[1][1] = __builtin_bit_cast(bf16x8_v, src[64]);
      if (__ballot(c0 != 1.f || c1 != 1.f) != 0) {  // columns whose reference point moved at this tile
#pragma unroll
        for (int i = 0; i < MH; ++i) {
          o[0][i] *= c0;
          o[1][i] *= c1;
        }
      }
      if constexpr (more) reference(kt + 1, there_next, buf ^ 1);
      __builtin_amdgcn_s_setprio(1);
      const uint2* vt = reinterpret_cast<const uint2*>(smem + buf * S::kTileBytes) + half * MH * 128 + lane;
      constexpr int kAhead = 4;
      auto vread = [&](int f) {
        const uint2 a = vt[(f / MH * MT + f % MH) * 128], c = vt[(f / MH * MT + f % MH) * 128 + 64];
        return __builtin_bit_cast(bf16x8_v, make_uint4(a.x, a.y, c.x, c.y));
      };
      bf16x8_v va[kAhead];
#pragma unroll
      for (int f = 0; f < kAhead; ++f) va[f] = vread(f);
#pragma unroll
      for (int f = 0; f < 2 * MH; ++f) {
        const bf16x8_v a = va[f % kAhead];
        const int u = f / MH, i = f % MH;
        o[0][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pv[0][u], o[0][i], 0, 0, 0);
        if constexpr (more) prob(f * (16 / (2 * MH)));
        o[1][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pv[1][u], o[1][i], 0, 0, 0);
        if constexpr (more && MH == 4) prob(f * 2 + 1);
        if (f + kAhead < 2 * MH) va[f % kAhead] = vread(f + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (more) publish(buf ^ 1);
      // ---- NaN groups among keys that not every column sees
      if (flag == static_cast<int>(kt - kt0) + 1) {
        const ParamsAgain q = params_again();
        for (int t = 0; t < kTile; ++t) {
          const int64_t key = kt * kTile + t;
          if (!(there_cur >> (t >> 4) & 1) || key >= kv_end) continue;
          const int32_t ph = block_of_run(q->c, b, key >> 4, runs);
          const uint8_t* run = q->c.vpool + g * q->c.sG + static_cast<int64_t>(ph) * q->c.sP + ((key >> 4) & ((1 << (q->c.bs_shift - 4)) - 1)) * kv4::Run<D>::kBytes;
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (run[kv4::Run<D>::value_scale(t & 15, (4 * quad + r) / (512 / D))] == 255)
              nan_rows |= (key <= first_pos + ahead[0] ? 1u : 0u) << r | (key <= first_pos + ahead[1] ? 16u : 0u) << r;
        }
      }
      there_cur = there_next;
      there_next = there;
      if constexpr (more) store_keys(buf);
      lds_barrier();
    };
    using yes = std::integral_constant<bool, true>;
    using no = std::integral_constant<bool, false>;
    // The loop begins four bytes past a multiple of 64, whatever code lies before it: where its instructions lie in the
    // lines that they are fetched by is worth 2 %.  2048 tokens behind 32000, 0, 4, 8, 16 and 32 bytes past: 886 871 872
    // 875 885 us.
    asm volatile(".p2align 6\n\ts_nop 0");
    for (int64_t kt = kt0; kt + 1 < kt1; ++kt) {
      iterate(kt, yes{});
    }
    iterate(kt1 - 1, no{});
  }

  // ---- out, through LDS
  const ParamsAgain late = params_again();
  const int64_t row0 = first_tok * late->c.H + static_cast<int64_t>(g) * late->c.G;  // of the output
  ask_gate(late);
  __syncthreads();
  float* s_l = s_corr;  // [column]; then the reference points
  const float l_own = column_sum(l_run);
  if (quad == 0) {
    s_l[wave * 16 + col] = l_own;
    s_l[(kWaves + wave) * 16 + col] = m_run;
  }
  constexpr int kRowFloats = D + 4;
  static_assert(kCols / 2 * kRowFloats * 4 <= S::kCorr, "half of the columns fit below the sums");
  float* s_o = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (nan_rows >> (4 * c + r) & 1) {
#pragma unroll
        for (int i = 0; i < MH; ++i) o[c][i][r] = __uint_as_float(0x7fc00000u);
      }
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    if (pass == 1) lds_barrier();  // the first tiles have been read
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < MH; i += 4) {
        floatx4_v v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = half == pass ? o[0][i + e][r] : o[1][i + e][r];
        *reinterpret_cast<floatx4_v*>(s_o + (16 * (wave >> 1) + col) * kRowFloats + (4 * quad + r) * MT + half * MH + i) = v;
      }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < kSweeps; ++i) {
      const int x = column_of(pass, i);
      if (x >= n_cols) continue;
      const float* at = s_o + (tid / kLanes + i * kRowsAtOnce) * kRowFloats;
      const Place pl = place_of(late->c, x);
      const uint32_t row = pl.token * static_cast<uint32_t>(late->c.H) + pl.head;  // past row0
      const float l = s_l[x];
      if (parts > 1) {
        const int64_t part = (blockIdx.z * late->part_tokens + part_base(*late, b, tok0) - tok0) * late->c.H + row0 + row;
        if (in_row == 0) *reinterpret_cast<float2*>(late->part_ml + part * 2) = make_float2(s_l[kWaves * 16 + x], l);
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

constexpr int kJoinAhead = 8;  // parts asked for at a time

// Joins the parts of one (token, head): a wave each, lane l dims l D/64 ..
template <int D>
__global__ __launch_bounds__(256) void join_kernel(PrefillParams pp) {
  const Params& p = pp.c;
  constexpr int E = D / 64;
  typedef float vec_t __attribute__((ext_vector_type(E)));
  const int lane = threadIdx.x & 63;
  const int64_t x = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.y;
  const int64_t tok0 = read_index(p.cu, p.idx_i64, b);
  const int64_t n_new = min64(pp.max_new, min64(read_index(p.cu, p.idx_i64, b + 1), p.total) - tok0);
  if (tok0 < 0 || x >= n_new * p.H) return;
  const uint32_t n = static_cast<uint32_t>(x) / static_cast<uint32_t>(p.H), h = static_cast<uint32_t>(x) - n * static_cast<uint32_t>(p.H);
  // the workgroups that had this column
  const int64_t column = static_cast<int64_t>(n) * p.G + (h - over_group(p, h) * static_cast<uint32_t>(p.G));
  const int64_t last = min64(n_new * p.G, column / kCols * kCols + kCols) - 1;
  const int parts = parts_of(pp, (keys_of(p, read_index(p.prefix, p.idx_i64, b), last) + kTile - 1) / kTile);
  if (parts == 1) return;  // written by the workgroup itself
  const int64_t row = part_base(pp, b, tok0) * p.H + x;
  const int64_t stride = pp.part_tokens * p.H;
  const float2 ml = lane < parts ? *reinterpret_cast<const float2*>(pp.part_ml + (lane * stride + row) * 2) : make_float2(-INFINITY, 0.f);
  const float m = wave_max(ml.x);
  const float f = __builtin_amdgcn_exp2f(ml.x - (m == -INFINITY ? 0.f : m));
  const float l = wave_sum(f * ml.y);
  vec_t acc = vec_t(0.f);
  for (int s0 = 0; s0 < parts; s0 += kJoinAhead) {
    vec_t part[kJoinAhead];
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i)  // past the end: the last part again
      part[i] = *reinterpret_cast<const vec_t*>(pp.part_o + (min(s0 + i, parts - 1) * stride + row) * D + E * lane);
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i) {
      const float fs = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), min(s0 + i, parts - 1)));
      if (s0 + i < parts) acc += fs * part[i];
    }
  }
  typedef uint32_t packed_t __attribute__((ext_vector_type(E / 2)));
  packed_t gate = packed_t(0u), out;
  if (p.gate != nullptr) gate = *reinterpret_cast<const packed_t*>(p.gate + (tok0 + n) * p.gate_st + h * p.gate_sh + E * lane);
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    float lo = normalised(acc[e], l), hi = normalised(acc[e + 1], l);
    if (p.gate != nullptr) {
      lo *= sigmoid(__uint_as_float(gate[e / 2] << 16));
      hi *= sigmoid(__uint_as_float(gate[e / 2] & 0xffff0000u));
    }
    out[e / 2] = static_cast<uint32_t>(f32_to_bf16(lo)) | static_cast<uint32_t>(f32_to_bf16(hi)) << 16;
  }
  *reinterpret_cast<packed_t*>(p.out + (tok0 * p.H + x) * D + E * lane) = out;
}

// Parts the keys are split into where the workgroups leave CUs free.  A part saves a share of 1.5 us a tile and costs its
// piece of the partial results, in time like parts times workgroups, which puts the best number at a root; the 30 is from
// us with 1, 2, 4, 8, 16 parts, D = 256, one row: 16 tokens (2 workgroups) over 32 tiles 65.6 41.9 29.2 23.3 22.1, 128 tokens
// (16) over 17 tiles 42.3 31.9 27.7 30.8 35.4, 512 tokens (64) over 8 tiles 28.6 33.6 35.4 51.4 64.5, over 32 tiles 67.2
// 52.8 45.3 64.9 105.
constexpr double kPerTile = 30.0;

static int64_t workgroups_of(int64_t batch, int kv_heads, int group, int64_t max_new) { return batch * kv_heads * ceil_div(max_new * group, kCols); }

// What the launch has room for, from the longest row that the tables hold; each row's own number is parts_of its tiles.
static int splits_of(int64_t batch, int kv_heads, int group, int64_t max_new, int64_t max_tokens) {
  const int64_t wgs = workgroups_of(batch, kv_heads, group, max_new);
  const int64_t tiles = ceil_div(std::max<int64_t>(max_tokens, 1), kTile);
  if (wgs >= 256) return 1;
  const int64_t best = static_cast<int64_t>(std::sqrt(kPerTile * static_cast<double>(tiles) / static_cast<double>(wgs)));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({kMaxSplits, 256 / wgs, tiles, best})));
}

// Tokens that partial results are kept of: a query padded past its rows' bound is no reason for more.  With splits of at most
// 256 / workgroups and a workgroup per 128 columns they are below 35 MB at any padding and any width of the tables.
static int64_t part_tokens_of(int64_t total, int64_t batch, int64_t max_new) { return std::min(total, batch * max_new); }

static int64_t workspace_of(int splits, int64_t part_tokens, int heads, int head_dim) {
  return splits > 1 ? splits * part_tokens * heads * (static_cast<int64_t>(head_dim) + 2) * 4 : 0;
}

template <int D>
static int launch(const PrefillParams& p, dim3 grid, hipStream_t stream) {
  if (int rc = reserve_lds<&prefill_kernel<D>>("paged_attention_prefill_kv4", Smem<D>::kBytes)) return rc;
  {
    KernelTimer timer_("prefill_kv4", stream);
    hipLaunchKernelGGL(prefill_kernel<D>, grid, dim3(64 * kWaves), Smem<D>::kBytes, stream, p);
  }
  if (int rc = check_launch("paged_attention_prefill_kv4")) return rc;
  if (p.splits > 1) {
    KernelTimer timer_("prefill_kv4_join", stream);
    const dim3 jgrid(static_cast<unsigned>(ceil_div(p.max_new * p.c.H, 4)), static_cast<unsigned>(p.c.B));
    hipLaunchKernelGGL(join_kernel<D>, jgrid, dim3(256), 0, stream, p);
  }
  return check_launch("paged_attention_prefill_kv4");
}

}  // namespace prefill4
}  // namespace qa

extern "C" int64_t qa_paged_attention_prefill_kv4_workspace(int64_t total_new, int64_t batch, int64_t max_new, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                                            int64_t max_tokens) {
  if (total_new <= 0 || batch <= 0 || max_new <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || head_dim <= 0 || max_tokens < 0) return 0;
  max_new = std::min(max_new, total_new);
  return qa::prefill4::workspace_of(qa::prefill4::splits_of(batch, kv_heads, heads / kv_heads, max_new, max_tokens),
                                    qa::prefill4::part_tokens_of(total_new, batch, max_new), heads, head_dim);
}

extern "C" int qa_paged_attention_prefill_kv4(const void* query, int32_t q_dtype, int64_t q_stride_t, int64_t q_stride_h, int64_t total_new, const void* cu_seqlens,
                                              const void* prefix_lens, int32_t idx_dtype, int64_t batch, int64_t max_new, int32_t heads, int32_t head_dim,
                                              const qa_paged_kv* kv, const void* block_tables, int32_t table_dtype, int64_t table_stride, int64_t max_blocks,
                                              int32_t block_size, float scale, const void* gate, int64_t gate_stride_t, int64_t gate_stride_h, void* output,
                                              void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  using namespace qa;
  using namespace qa::prefill4;
  PrefillParams p{};
  const Args a{"paged_attention_prefill_kv4", query, q_dtype, q_stride_t, q_stride_h, total_new, batch, heads, head_dim, kv, block_tables, table_dtype, table_stride, max_blocks,
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
  p.max_new = max_new;
  p.splits = splits_of(batch, kv->kv_heads, p.c.G, max_new, max_blocks * block_size);
  p.per_tile = static_cast<float>(kPerTile / static_cast<double>(workgroups_of(batch, kv->kv_heads, p.c.G, max_new)));
  p.part_tokens = part_tokens_of(total_new, batch, max_new);
  p.per_row = p.part_tokens < total_new ? max_new : 0;
  const int64_t need = workspace_of(p.splits, p.part_tokens, heads, head_dim);
  QA_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0),
             "paged prefill workspace too small or not 16-byte aligned: need %lld bytes, have %lld", static_cast<long long>(need), static_cast<long long>(workspace_bytes));
  p.part_o = reinterpret_cast<float*>(workspace);
  p.part_ml = p.part_o + static_cast<int64_t>(p.splits) * p.part_tokens * heads * head_dim;
  const dim3 grid(static_cast<unsigned>(ceil_div(max_new * p.c.G, kCols)), static_cast<unsigned>(batch * kv->kv_heads), static_cast<unsigned>(p.splits));
  return head_dim == 256 ? launch<256>(p, grid, stream) : launch<128>(p, grid, stream);
}
