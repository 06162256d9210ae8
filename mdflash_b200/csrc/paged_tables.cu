// One step of the paged K/V cache's tables, from the requests' lengths before and after it.
//
// With page size s, request r has had_r = ceil(old_r / s) pages and needs need_r = ceil(new_r /
// s).  It gives back max(had - need, 0) of them (its last ones) or takes max(need - had, 0), and
// has max(new - old, 0) new tokens.  The exclusive prefixes B, M and T of the three over the
// requests place everything:
//   push   free[count + B_r + j] = table[r, need_r + j]                    j < had_r - need_r
//   pop    table[r, had_r + j] = stack[count + B_R - 1 - (M_r + j)]        j < need_r - had_r
//   token  T_r + i: position old_r + i, slot table[r, position / s] * s + position % s
// where stack is free[0, count) with the pushed pages on top.  A popped or new page is looked up
// by that formula wherever it is needed (stack_at), so nothing in the launch reads what another
// part of it wrote, and the parts need no order between them.
//
// Every CTA scans the lengths of all requests itself (at most 2048 of them, two per thread)
// and then covers its share of the pages and tokens; the grid's last CTA (a ticket, no waiting)
// writes the outputs that may alias inputs.  Bound by latency: a step of 64 decoding requests
// is one CTA and a few dependent reads, 5.3 us in a recorded graph; 1000 requests with 49k new
// tokens (1 MB in and out) take 9.2 us (109 on one CTA).
#include "common.cuh"

namespace ddt {
namespace paged {

constexpr int kThreads = 1024;
constexpr int kPer = DDT_MAX_PAGED_REQUESTS / kThreads;

struct TableArgs {
  const int32_t* old_lens;
  const int32_t* new_lens;
  int n_requests;
  int32_t* block_table;
  long long table_stride, max_pages;
  int page_shift;
  int32_t* free_pages;
  long long free_capacity;
  const int32_t* free_count;
  int32_t* kv_lens;
  int32_t* cu_new;
  int64_t* slot_map;
  int64_t* positions;
  long long max_tokens;
  int32_t* free_count_out;
  unsigned int* ticket;
  int32_t* status;
};

// Exclusive block scans of kScans values per (thread, kPer consecutive requests), in one pass;
// the totals go to `total`.
constexpr int kScans = 3;
__device__ __forceinline__ void block_scan(long long (&v)[kScans][kPer],
                                           long long (&s_warp)[kScans][kThreads / 32],
                                           long long (&total)[kScans]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long sum[kScans], incl[kScans];
#pragma unroll
  for (int q = 0; q < kScans; ++q) {
    sum[q] = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const long long x = v[q][k];
      v[q][k] = sum[q];
      sum[q] += x;
    }
    incl[q] = sum[q];
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int q = 0; q < kScans; ++q) {
      const long long y = __shfl_up_sync(DDT_FULL_MASK, incl[q], o);
      if (lane >= o) incl[q] += y;
    }
  if (lane == 31)
#pragma unroll
    for (int q = 0; q < kScans; ++q) s_warp[q][warp] = incl[q];
  __syncthreads();
  // every warp scans the warps' sums
  static_assert(kThreads / 32 == 32, "one warp sum per lane");
#pragma unroll
  for (int q = 0; q < kScans; ++q) {
    const long long own = s_warp[q][lane];
    long long w = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(DDT_FULL_MASK, w, o);
      if (lane >= o) w += y;
    }
    total[q] = __shfl_sync(DDT_FULL_MASK, w, 31);
    const long long before = __shfl_sync(DDT_FULL_MASK, w - own, warp) + incl[q] - sum[q];
#pragma unroll
    for (int k = 0; k < kPer; ++k) v[q][k] += before;
  }
}

// The request whose range of the exclusive prefix `first` [n + 1] holds x < first[n].
__device__ __forceinline__ int owner(const int32_t* first, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads, 1) page_tables_kernel(const TableArgs a) {
  __shared__ long long s_warp[kScans][kThreads / 32];
  __shared__ int32_t s_back[DDT_MAX_PAGED_REQUESTS + 1], s_more[DDT_MAX_PAGED_REQUESTS + 1],
      s_tok[DDT_MAX_PAGED_REQUESTS + 1];
  const int tid = threadIdx.x, n = a.n_requests;
  const long long page = 1ll << a.page_shift;
  after_stream();
  let_next_begin();
  int32_t old_len[kPer], new_len[kPer];
  long long v[kScans][kPer], total[kScans];
  auto &back = v[0], &more = v[1], &tok = v[2];
  bool fine = true;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int r = tid * kPer + k;
    old_len[k] = r < n ? a.old_lens[r] : 0;
    new_len[k] = r < n ? a.new_lens[r] : 0;
    const long long had = (old_len[k] + page - 1) >> a.page_shift;
    const long long need = (new_len[k] + page - 1) >> a.page_shift;
    if (old_len[k] < 0 || new_len[k] < 0 || had > a.max_pages || need > a.max_pages) fine = false;
    back[k] = had > need ? had - need : 0;
    more[k] = need > had ? need - had : 0;
    tok[k] = new_len[k] > old_len[k] ? static_cast<long long>(new_len[k]) - old_len[k] : 0;
  }
  const long long count = *a.free_count;
  block_scan(v, s_warp, total);
  const long long n_back = total[0], n_more = total[1], n_tok = total[2];
  // every sum fits 32 bits where the step is accepted
  fine = fine && count >= 0 && count + n_back <= a.free_capacity && count + n_back >= n_more &&
         n_tok <= a.max_tokens;
  const bool ok = __syncthreads_and(fine);
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int r = tid * kPer + k;
    if (r < n) {
      s_back[r] = static_cast<int32_t>(back[k]);
      s_more[r] = static_cast<int32_t>(more[k]);
      s_tok[r] = static_cast<int32_t>(tok[k]);
    }
  }
  if (tid == 0) {
    s_back[n] = static_cast<int32_t>(n_back);
    s_more[n] = static_cast<int32_t>(n_more);
    s_tok[n] = static_cast<int32_t>(n_tok);
  }
  __syncthreads();

  const long long stride = static_cast<long long>(gridDim.x) * kThreads;
  const long long first = static_cast<long long>(blockIdx.x) * kThreads + tid;
  auto pages_of = [&](int32_t len) { return (len + page - 1) >> a.page_shift; };
  if (ok) {
    // the page that request r gave back as its j-th
    auto given = [&](int f) {
      const int r = owner(s_back, n, f);
      return a.block_table[r * a.table_stride + pages_of(a.new_lens[r]) + f - s_back[r]];
    };
    // the t-th page taken from the stack
    auto taken = [&](int t) {
      const long long at = count + n_back - 1 - t;
      return at >= count ? given(static_cast<int>(at - count)) : a.free_pages[at];
    };
    for (long long f = first; f < n_back; f += stride)
      a.free_pages[count + f] = given(static_cast<int>(f));
    for (long long t = first; t < n_more; t += stride) {
      const int r = owner(s_more, n, static_cast<int>(t));
      a.block_table[r * a.table_stride + pages_of(a.old_lens[r]) + t - s_more[r]] =
          taken(static_cast<int>(t));
    }
    for (long long t = first; t < a.max_tokens; t += stride) {
      int64_t slot = -1, pos = 0;
      if (t < n_tok) {
        const int r = owner(s_tok, n, static_cast<int>(t));
        const int32_t old = a.old_lens[r];
        pos = old + (t - s_tok[r]);
        const long long j = pos >> a.page_shift, had = pages_of(old);
        const int32_t pg = j < had ? a.block_table[r * a.table_stride + j]
                                   : taken(static_cast<int>(s_more[r] + j - had));
        slot = (static_cast<int64_t>(pg) << a.page_shift) + (pos & (page - 1));
      }
      a.slot_map[t] = slot;
      a.positions[t] = pos;
    }
  } else {
    for (long long t = first; t < a.max_tokens; t += stride) {
      a.slot_map[t] = -1;
      a.positions[t] = 0;
    }
  }
  if (blockIdx.x == 0)
    for (int r = tid; r <= n; r += kThreads) a.cu_new[r] = ok ? s_tok[r] : 0;

  // the last CTA writes what may alias an input: every CTA has read its inputs by then
  __shared__ bool s_last;
  __syncthreads();
  if (gridDim.x > 1) {
    if (tid == 0) {
      __threadfence();
      s_last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!s_last) return;
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int r = tid * kPer + k;
    if (r < n) a.kv_lens[r] = ok ? new_len[k] : old_len[k];
  }
  if (tid == 0) {
    *a.free_count_out = static_cast<int32_t>(ok ? count + n_back - n_more : count);
    if (!ok && a.status) atomicOr(a.status, DDT_STATUS_PAGES);
    if (gridDim.x > 1) *a.ticket = 0u;
  }
}

}  // namespace paged
}  // namespace ddt

using namespace ddt;

extern "C" size_t ddt_page_tables_workspace_bytes(int64_t n_requests) {
  (void)n_requests;
  return sizeof(unsigned int);
}

extern "C" int ddt_page_tables(const int32_t* old_lens, const int32_t* new_lens,
                               int64_t n_requests, int32_t* block_table, int64_t table_stride,
                               int64_t max_pages, int64_t page_size, int32_t* free_pages,
                               int64_t free_capacity, const int32_t* free_count, int32_t* kv_lens,
                               int32_t* cu_new, int64_t* slot_map, int64_t* positions,
                               int64_t max_tokens, int32_t* free_count_out, void* workspace,
                               size_t workspace_bytes, int32_t* status, void* stream) {
  if (!old_lens || !new_lens || !block_table || (free_capacity > 0 && !free_pages) ||
      !free_count || !kv_lens || !cu_new || !free_count_out ||
      (max_tokens > 0 && (!slot_map || !positions)))
    return DDT_ERR_INVALID;
  if (n_requests <= 0 || max_pages <= 0 || table_stride < max_pages || max_tokens < 0 ||
      free_capacity < 0)
    return DDT_ERR_INVALID;
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return DDT_ERR_CAPACITY;
  if (n_requests > DDT_MAX_PAGED_REQUESTS || max_tokens > 0x7fffffff || free_capacity > 0x7fffffff ||
      max_pages > (int64_t(1) << 30) / page_size)
    return DDT_ERR_CAPACITY;
  if (!workspace || workspace_bytes < sizeof(unsigned int)) return DDT_ERR_WORKSPACE;
  if (!aligned(workspace, 4)) return DDT_ERR_ALIGN;
  paged::TableArgs a;
  a.old_lens = old_lens;
  a.new_lens = new_lens;
  a.n_requests = static_cast<int>(n_requests);
  a.block_table = block_table;
  a.table_stride = table_stride;
  a.max_pages = max_pages;
  a.page_shift = __builtin_ctzll(static_cast<unsigned long long>(page_size));
  a.free_pages = free_pages;
  a.free_capacity = free_capacity;
  a.free_count = free_count;
  a.kv_lens = kv_lens;
  a.cu_new = cu_new;
  a.slot_map = slot_map;
  a.positions = positions;
  a.max_tokens = max_tokens;
  a.free_count_out = free_count_out;
  a.ticket = static_cast<unsigned int*>(workspace);
  a.status = status;
  // a CTA per 1024 tokens or 128 requests (whose pages move), up to one per SM
  const int64_t by_tokens = (max_tokens + paged::kThreads - 1) / paged::kThreads;
  const int64_t by_requests = (n_requests + 127) / 128;
  int64_t blocks = by_tokens > by_requests ? by_tokens : by_requests;
  if (blocks > 148) blocks = 148;
  return launch_early(paged::page_tables_kernel, dim3(static_cast<unsigned>(blocks)),
                      dim3(paged::kThreads), 0, static_cast<cudaStream_t>(stream), 0, a);
}
