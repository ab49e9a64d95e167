// The plan of a batched step on the device: block tables grown from the free list, and the slot map of the step's
// packed tokens, from the requests' lengths and new-token counts.
//
// Row b grows from L_b to L_b + n_b tokens.  With need_b = ceil((L_b + n_b) / bs) - ceil(L_b / bs), the exclusive sums
// over the rows c_b of n and f_b of need give everything: packed token i of row b (i - c_b = x) sits at position
// L_b + x; its logical block lb is the row's old one while lb < ceil(L_b / bs), else free_list[head + f_b + lb -
// ceil(L_b / bs)]; its slot is id * bs + position % bs.  A fresh block always holds a new token at its first position,
// so the token there writes the table entry: no pass of its own over the tables.  Where every row has per_row entries of
// the token arrays instead, the row of an entry is a division and the rest the same.
//
// A few KB move, so latency bounds it: a launch of one workgroup reads lengths, counts and state at once (with a thread a
// row the scan that plans is also the sum that is checked), looks the tokens' rows up in LDS and writes them.  128 rows of
// one token: 5.5 us.  From kInlineTokens on a second launch of one workgroup per kSpanTokens tokens writes them, because
// one CU stores only a few tens of GB/s; 61 rows of up to 8192 tokens: 4.4 + 5.0 us.
#include "qa_common.h"

namespace qa {
namespace kvplan {

struct Params {
  int32_t* tables;
  int64_t table_stride, max_blocks;
  int32_t* lengths;
  const void* counts;  // null: count_scalar
  int64_t count_scalar;
  const int32_t* free_list;
  int32_t* free_state;
  int32_t* status;
  int32_t* cu;         // (B + 1)
  int32_t* starts;     // (B)
  int32_t* first;      // (B): where each row's fresh blocks begin in the free list
  int32_t* positions;  // (max_tokens)
  int64_t* slots;      // (max_tokens)
  int64_t max_tokens, capacity;
  uint32_t per_row;    // 0: the tokens are packed; else row b's are entries b per_row ..
  int B, bs, counts_i64;
  int inline_tokens;   // the planning workgroup writes the tokens too
};

constexpr int kThreads = 1024;
constexpr int kSpanTokens = 256;    // tokens of a workgroup of the second launch; with 1024, four dependent chains one after the other, 7.9 us in place of 5.5 for 61 rows of 8192
// Tokens that the planning workgroup writes itself.  us there, and with a second launch (whose gap comes on top): 128 tokens
// 5.5 and 4.2 + 2.3, 1024 tokens 5.8 and 4.4 + 3.4, 4096 tokens 8.8 and 4.3 + 3.8, 8192 tokens 12.6 and 4.3 + 3.6.
constexpr int kInlineTokens = 4096;
constexpr int kRowsInLds = 4096;    // rows whose sums a workgroup looks up in LDS: what 48 KB hold of the three arrays

__device__ __forceinline__ int64_t count_of(const Params& p, int b) {
  if (p.counts == nullptr) return p.count_scalar;
  return p.counts_i64 ? reinterpret_cast<const int64_t*>(p.counts)[b] : reinterpret_cast<const int32_t*>(p.counts)[b];
}

// Blocks of n tokens.  In 32 bits: a row that is planned has n + bs below 2^31.
__device__ __forceinline__ uint32_t blocks_of(const Params& p, int64_t n) { return (static_cast<uint32_t>(n) + p.bs - 1) / p.bs; }

// What the writing of tokens reads of the rows: in LDS, or in memory where they are too many.
struct Rows {
  const int32_t* cu;
  const int32_t* starts;
  const int32_t* first;
};

// Writes positions, slots and fresh table entries of tokens lo .. hi - 1.
__device__ void write_tokens(const Params& p, const Rows& rows, int64_t lo, int64_t hi) {
  const int32_t total = rows.cu[p.B];
  for (int64_t i = lo + threadIdx.x; i < hi; i += blockDim.x) {
    int32_t position = -1;
    int64_t slot = -1;
    int a = 0;
    int32_t nth = 0;
    bool token = i < total;
    if (p.per_row != 0) {
      a = static_cast<int>(static_cast<uint32_t>(i) / p.per_row);
      nth = static_cast<int32_t>(i - static_cast<int64_t>(a) * p.per_row);
      token = nth < rows.cu[a + 1] - rows.cu[a];
    } else if (token) {
      int z = p.B;  // cu[a] <= i < cu[z]
      while (z - a > 1) {
        const int m = (a + z) >> 1;
        if (rows.cu[m] <= i)
          a = m;
        else
          z = m;
      }
      nth = static_cast<int32_t>(i - rows.cu[a]);
    }
    if (token) {
      const int32_t start = rows.starts[a];
      position = start + nth;
      const uint32_t lb = static_cast<uint32_t>(position) / p.bs;
      const uint32_t have = blocks_of(p, start);
      const uint32_t at = position - lb * p.bs;
      int32_t id;
      if (lb < have) {
        id = p.tables[a * p.table_stride + lb];
      } else {
        id = p.free_list[rows.first[a] + static_cast<int64_t>(lb - have)];
        if (at == 0) p.tables[a * p.table_stride + lb] = id;
      }
      if (id >= 0) slot = static_cast<int64_t>(id) * p.bs + at;
    }
    p.positions[i] = position;
    p.slots[i] = slot;
  }
}

__global__ __launch_bounds__(kThreads) void plan_kernel(Params p) {
  __shared__ int64_t s_need[kThreads / 64], s_count[kThreads / 64];
  __shared__ int s_bad[kThreads / 64];
  __shared__ int32_t s_cu[kRowsInLds + 1], s_starts[kRowsInLds], s_first[kRowsInLds];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int64_t head = p.free_state[0];
  const int64_t avail = p.free_state[1];

  // a row's length, tokens and blocks; what it asks for if that can be counted at all
  int64_t len, n, need;
  int bad = 0;
  auto row = [&](int b) {
    len = n = need = 0;
    if (b >= p.B) return;
    len = p.lengths[b];
    n = count_of(p, b);
    if (len < 0 || n < 0 || n > 0x7fffffff || len + n > 0x7fffffff - p.bs) {
      bad |= 4;
      n = 0;
      return;
    }
    const uint32_t want = blocks_of(p, len + n);
    if (want > p.max_blocks) bad |= 2;
    if (p.per_row != 0 && n > p.per_row) bad |= 8;
    need = want - blocks_of(p, len);
  };
  // sums over the workgroup: of all rows, or up to and with a thread's own
  int64_t total_need = 0, total_count = 0;
  auto totals = [&](int64_t of_need, int64_t of_count) {  // of_*: a wave's sums, in its last lane
    for (int off = 32; off > 0; off >>= 1) bad |= __shfl_xor(bad, off, 64);
    if (lane == 63) {
      s_need[wave] = of_need;
      s_count[wave] = of_count;
      s_bad[wave] = bad;
    }
    __syncthreads();
    total_need = total_count = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
      total_need += s_need[w];
      total_count += s_count[w];
      bad |= s_bad[w];
    }
  };
  int64_t need_incl, n_incl;
  auto scan_wave = [&]() {
    need_incl = need;
    n_incl = n;
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t nu = __shfl_up(n_incl, off, 64), ku = __shfl_up(need_incl, off, 64);
      if (lane >= off) {
        n_incl += nu;
        need_incl += ku;
      }
    }
  };

  // the checks; with a thread for every row the sums they need are the ones the plan needs
  const bool one = p.B <= kThreads;
  if (one) {
    row(tid);
    scan_wave();
    totals(need_incl, n_incl);
  } else {
    int64_t my_need = 0, my_count = 0;
    for (int b = tid; b < p.B; b += kThreads) {
      row(b);
      my_need += need;
      my_count += n;
    }
    for (int off = 32; off > 0; off >>= 1) {
      my_need += __shfl_xor(my_need, off, 64);
      my_count += __shfl_xor(my_count, off, 64);
    }
    totals(my_need, my_count);
  }
  int code = 0;
  if (head < 0 || avail < 0 || head + avail > p.capacity) code = 3;
  else if (bad & 4) code = 4;
  else if (bad & 2) code = 2;
  else if (total_need > avail) code = 1;
  else if (total_count > p.max_tokens || (bad & 8)) code = 5;
  const int64_t taken = total_need;

  // the row sums; a step that is refused plans no token and takes nothing
  int64_t need_before = head, count_before = 0;
  for (int r0 = 0; r0 < p.B; r0 += kThreads) {
    const int b = r0 + tid;
    if (!one) {
      __syncthreads();  // s_need and s_count are used again
      row(b);
      scan_wave();
      totals(need_incl, n_incl);
    }
    int64_t need_at = need_before, n_at = count_before;
    for (int w = 0; w < wave; ++w) {
      need_at += s_need[w];
      n_at += s_count[w];
    }
    if (b < p.B) {
      const int32_t c = code ? 0 : static_cast<int32_t>(n_at + n_incl - n);
      const int32_t f = code ? 0 : static_cast<int32_t>(need_at + need_incl - need);
      p.cu[b] = c;
      p.starts[b] = static_cast<int32_t>(len);
      if (b < kRowsInLds) {
        s_cu[b] = c;
        s_starts[b] = static_cast<int32_t>(len);
        s_first[b] = f;
      }
      if (!p.inline_tokens) p.first[b] = f;
      if (code == 0) p.lengths[b] = static_cast<int32_t>(len + n);
    }
    need_before += total_need;
    count_before += total_count;
  }
  if (tid == 0) {
    const int32_t total = code ? 0 : static_cast<int32_t>(count_before);
    p.cu[p.B] = total;
    if (p.B <= kRowsInLds) s_cu[p.B] = total;
    if (code == 0) {
      p.free_state[0] = static_cast<int32_t>(head + taken);
      p.free_state[1] = static_cast<int32_t>(avail - taken);
    }
    p.status[0] = code;
  }
  if (!p.inline_tokens) return;
  lds_barrier();
  write_tokens(p, {s_cu, s_starts, s_first}, 0, p.max_tokens);
}

__global__ __launch_bounds__(256) void plan_tokens_kernel(Params p) {
  __shared__ int32_t s_cu[kRowsInLds + 1];
  const int64_t lo = static_cast<int64_t>(blockIdx.x) * kSpanTokens;
  const int64_t hi = min64(p.max_tokens, lo + kSpanTokens);
  if (p.B <= kRowsInLds) {
    for (int b = threadIdx.x; b <= p.B; b += blockDim.x) s_cu[b] = p.cu[b];
    __syncthreads();
  }
  write_tokens(p, {p.B <= kRowsInLds ? s_cu : p.cu, p.starts, p.first}, lo, hi);
}

}  // namespace kvplan
}  // namespace qa

extern "C" int qa_paged_kv_plan(int32_t* block_tables, int64_t table_stride, int64_t max_blocks, int32_t* lengths, const void* counts, int32_t counts_dtype,
                                int64_t count_scalar, int64_t batch, int32_t block_size, const int32_t* free_list, int64_t free_capacity, int32_t* free_state,
                                int32_t* status, int64_t max_tokens, int64_t per_row, int32_t* cu_seqlens, int32_t* starts, int32_t* positions, int64_t* slots, int32_t* workspace,
                                int64_t workspace_bytes, hipStream_t stream) {
  using namespace qa;
  using namespace qa::kvplan;
  QA_REQUIRE(batch >= 1 && batch <= 0xffffff, "paged_kv_plan: batch must be in [1, 2^24)");
  QA_REQUIRE(block_tables && lengths && free_list && free_state && status && cu_seqlens && starts && workspace, "paged_kv_plan: pointers must be non-null");
  QA_REQUIRE(counts == nullptr || is_index_dtype(counts_dtype), "paged_kv_plan: counts must be int32/int64");
  QA_REQUIRE(counts != nullptr || (count_scalar >= 0 && count_scalar <= 0x7fffffff), "paged_kv_plan: count must be non-negative");
  QA_REQUIRE(block_size > 0 && block_size <= 65536 && max_blocks > 0, "paged_kv_plan: block_size must be in [1, 65536] and max_blocks positive");
  QA_REQUIRE(table_stride >= max_blocks || batch <= 1, "table rows overlap: stride %lld < max_blocks %lld", static_cast<long long>(table_stride),
             static_cast<long long>(max_blocks));
  QA_REQUIRE(free_capacity > 0 && free_capacity <= 0x7fffffff, "free list capacity must be in [1, 2^31)");
  QA_REQUIRE(max_tokens >= 0 && max_tokens <= 0x3fffffff, "paged_kv_plan: max_tokens must be in [0, 2^30)");
  QA_REQUIRE(per_row >= 0 && per_row <= 0x3fffffff && (per_row == 0 || per_row * batch == max_tokens), "paged_kv_plan: with %lld entries a row max_tokens must be %lld", static_cast<long long>(per_row),
             static_cast<long long>(per_row * batch));
  QA_REQUIRE(max_tokens == 0 || (positions && slots), "paged_kv_plan: pointers must be non-null");
  QA_REQUIRE(workspace_bytes >= batch * 4, "paged_kv_plan: workspace too small: need %lld bytes", static_cast<long long>(batch * 4));
  Params p{};
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.max_blocks = max_blocks;
  p.lengths = lengths;
  p.counts = counts;
  p.count_scalar = count_scalar;
  p.free_list = free_list;
  p.free_state = free_state;
  p.status = status;
  p.cu = cu_seqlens;
  p.starts = starts;
  p.first = workspace;
  p.positions = positions;
  p.slots = slots;
  p.max_tokens = max_tokens;
  p.per_row = static_cast<uint32_t>(per_row);
  p.capacity = free_capacity;
  p.B = static_cast<int>(batch);
  p.bs = block_size;
  p.counts_i64 = counts_dtype == QA_I64;
  p.inline_tokens = max_tokens <= kInlineTokens && batch <= kRowsInLds;
  {
    KernelTimer timer_("kv_plan", stream);
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kThreads), 0, stream, p);
  }
  if (int rc = check_launch("paged_kv_plan")) return rc;
  if (!p.inline_tokens && max_tokens > 0) {
    KernelTimer timer_("kv_plan_tokens", stream);
    hipLaunchKernelGGL(plan_tokens_kernel, dim3(static_cast<unsigned>(ceil_div(max_tokens, kSpanTokens))), dim3(256), 0, stream, p);
  }
  return check_launch("paged_kv_plan");
}
