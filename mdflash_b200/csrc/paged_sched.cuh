// Work distribution of the paged attention kernels, computed by every CTA from the device-side
// lengths (no plan is built on the host or kept between calls, so one recorded launch serves
// every length).
//
// A unit is (KV head, request, up to so many consecutive new tokens of it); it attends to the
// keys [0, past + its last token + 1) in tiles of kTile keys.  Its cost is its tiles plus kItem
// (loading Q, filling the pipeline, the masked tiles, the epilogue).  Fitted over the CTAs of four
// chunks of up to 2048 tokens it is 2.7 tiles of 128 keys.  Recorded, in turn, with 2, 3 and 4: four
// chunks 387.6, 385.0 and 386.6 us, 16 blocks of 16 tokens, whose tiles go two at a time, 48.2, 50.6
// and 50.1 (means of three runs, which agree within 0.3%).  The units of all heads, head by head,
// form one line of W cost positions that is cut into equal pieces, one per CTA; a CTA runs the tiles
// that lie in its piece.  A unit that crosses a cut is finished in parts: the part that holds the
// unit's first tile goes to slot 2 c + 1 of its CTA c, every later one to slot 2 c of its CTA; they
// are consecutive CTAs, and a CTA has at most one of each kind.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>

#include "common.cuh"
#include "tc.cuh"

namespace ddt {
namespace paged_attn {

constexpr int kHeadDim = 128;
constexpr int kMaxGroup = 64;
constexpr int kItem = 2;
constexpr int kSms = 148;
constexpr int kStatusTimeout = 1;
constexpr uint64_t kTimeoutNs = 2000000000ull;

struct Params {
  const int32_t* block_table;
  long long table_stride, max_keys, n_pages;
  int page_shift;
  const int32_t* cu_new;
  const int32_t* kv_lens;
  int n_requests, n_tokens, max_new, group, kv_heads;
  int from_new, to_new;  // the launch takes the requests with so many new tokens
  int beside;            // launched beside the few-rows kernel, which waited for what is read here
  float scale_log2;
  __nv_bfloat16* out;
  long long o_token_stride, o_head_stride;
  float* o_part;   // partial O of each slot
  float* ml_part;  // [slot][rows per unit][2]: m (log2 units) and l
  int4* parts;     // [CTAs]: a unit that starts in this CTA and is finished by others
  unsigned int* arrived;  // [CTAs]: parts written of the unit that starts in this CTA
  int32_t* status;
  unsigned long long timeout_ns;
  unsigned int withhold_from;  // check of the waits: CTAs from this one on issue no load
};

// First query row, new tokens and key count of request r; no tokens where another launch takes
// the request, or (and the status bit, from one CTA) where they are out of range.
struct Request {
  int first, n, len;
};
__device__ __forceinline__ Request request(const Params& p, int r) {
  Request q;
  q.first = p.cu_new[r];
  const int end = p.cu_new[r + 1];
  q.len = p.kv_lens[r];
  const bool fine = q.first >= 0 && end >= q.first && end <= p.n_tokens &&
                    end - q.first <= p.max_new && q.len >= 0 && q.len <= p.max_keys;
  const int n = end - q.first;
  q.n = fine && n >= p.from_new && n <= p.to_new ? n : 0;
  if (!fine && p.status && blockIdx.x == 0) atomicOr(p.status, DDT_STATUS_PAGED_RANGE);
  return q;
}

// The page of request r that holds key `key`, or n_pages, from where the tensor maps read zeros (and
// the status bit), where the table names no page of the pool.
__device__ __forceinline__ int page_of(const Params& p, int r, long long key) {
  const int page = p.block_table[r * p.table_stride + (key >> p.page_shift)];
  if (page >= 0 && page < p.n_pages) return page;
  if (p.status) atomicOr(p.status, DDT_STATUS_PAGED_RANGE);
  return static_cast<int>(p.n_pages);
}

struct Item {
  int h, r;
  int tok0, n_tok;  // query rows of the unit: [tok0, tok0 + n_tok), all heads of the group
  int past;         // keys before the unit's first token
  int len;          // keys of the request
  int t0, nt;       // key tiles of this piece
  int slot;         // -1: the unit's only piece
  long long x_first, x_last;  // positions of the unit's first and last tile
};

// The piece of the line that this CTA runs, and a warp's place in it.  Both live in shared
// memory: the walk is a few dozen instructions of one lane per item, and its state in registers
// made the kernel's warps spill.
struct Piece {
  long long per_head, total, ctas, x0, x1;
};
struct Place {
  int h, r, j;
  long long u0;
  Request q;
  Item it;
  int more;
};

template <int kTile>
__device__ __forceinline__ int tiles_of(const Request& q, int tok_end) {
  const int end = q.len - q.n + tok_end;
  return end > 0 ? (end - 1) / kTile + 1 : 0;
}

// The CTA whose piece holds position x of an item's unit, searched for from this CTA on: piece c
// holds it when c * total < (x + 1) * ctas <= (c + 1) * total.
__device__ __forceinline__ int cta_of(const Piece& c, long long x) {
  int at = blockIdx.x;
  while (at * c.total >= (x + 1) * c.ctas) --at;
  while ((at + 1) * c.total < (x + 1) * c.ctas) ++at;
  return at;
}

// a * b / c for factors whose product fits 32 bits or not (a 64-bit division is a few hundred
// cycles on the way to a CTA's first load)
__device__ __forceinline__ long long mul_div(long long a, long long b, long long c) {
  const long long n = a * b;
  if ((n | c) >> 32) return n / c;
  return static_cast<uint32_t>(n) / static_cast<uint32_t>(c);
}

// Costs of the requests for one KV head into s_first [n_requests + 1] (exclusive prefix), this
// CTA's piece of at most `most` ones, and the place of its first unit; all threads of the block
// call it.
template <int kTile>
__device__ void walk_begin(const Params& p, int tokens, long long most, long long* s_first,
                           long long* s_warp, Piece& piece, Place* places, int n_places) {
  const int nthr = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.n_requests + nthr - 1) / nthr;
  const int r0 = min(tid * per, p.n_requests), r1 = min(r0 + per, p.n_requests);
  long long sum = 0;
  for (int r = r0; r < r1; ++r) {
    const Request q = request(p, r);
    s_first[r] = sum;
    for (int t = 0; t < q.n; t += tokens) sum += kItem + tiles_of<kTile>(q, min(t + tokens, q.n));
  }
  long long incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(DDT_FULL_MASK, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  long long before = incl - sum;
  for (int w = 0; w < warp; ++w) before += s_warp[w];
  for (int r = r0; r < r1; ++r) s_first[r] += before;
  if (tid == nthr - 1) s_first[p.n_requests] = before + sum;
  __syncthreads();
  if (tid < n_places) {
    Piece c;
    c.per_head = s_first[p.n_requests];
    c.total = c.per_head * p.kv_heads;
    c.ctas = min(min(static_cast<long long>(gridDim.x), most), c.total);
    c.x0 = c.x1 = 0;
    Place w;
    w.h = p.kv_heads;
    w.r = w.j = w.more = 0;
    w.u0 = 0;
    w.it.slot = -1;
    if (blockIdx.x < c.ctas) {
      c.x0 = mul_div(blockIdx.x, c.total, c.ctas);
      c.x1 = mul_div(blockIdx.x + 1, c.total, c.ctas);
      w.h = static_cast<int>(mul_div(c.x0, 1, c.per_head));
      const long long at = c.x0 - w.h * c.per_head;
      int lo = 0, hi = p.n_requests - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_first[mid] <= at) lo = mid;
        else hi = mid - 1;
      }
      w.r = lo;
      w.q = request(p, lo);
      long long u = s_first[lo];
      for (;;) {
        const int cost = kItem + tiles_of<kTile>(w.q, min((w.j + 1) * tokens, w.q.n));
        if (u + cost > at) break;
        u += cost;
        ++w.j;
      }
      w.u0 = w.h * c.per_head + u;
    }
    places[tid] = w;
    if (tid == 0) piece = c;
  }
}

// The next item of this warp's walk into w.it (whole warp); false after the last one.
template <int kTile>
__device__ __forceinline__ bool walk_next(const Params& p, int tokens, const long long* s_first,
                                          const Piece& c, Place& w) {
  __syncwarp();  // the previous item is no longer read
  if ((threadIdx.x & 31) == 0) {
    w.more = 0;
    while (w.h < p.kv_heads && w.u0 < c.x1) {
      const int tok = w.j * tokens, n_tok = min(tokens, w.q.n - tok);
      const int tiles = tiles_of<kTile>(w.q, tok + n_tok);
      const long long b = c.x0 - w.u0 - kItem, e = c.x1 - w.u0 - kItem;
      const int lo = b <= 0 ? 0 : static_cast<int>(b < tiles ? b : tiles);
      const int hi = e <= 0 ? 0 : static_cast<int>(e < tiles ? e : tiles);
      const bool here = hi > lo || (tiles == 0 && w.u0 >= c.x0);
      if (here) {
        w.it.h = w.h;
        w.it.r = w.r;
        w.it.tok0 = w.q.first + tok;
        w.it.n_tok = n_tok;
        w.it.past = w.q.len - w.q.n + tok;
        w.it.len = w.q.len;
        w.it.t0 = lo;
        w.it.nt = hi - lo;
        w.it.slot = hi - lo == tiles ? -1 : 2 * static_cast<int>(blockIdx.x) + (lo == 0 ? 1 : 0);
        w.it.x_first = w.u0 + kItem;
        w.it.x_last = w.u0 + kItem + tiles - 1;
      }
      ++w.j;
      w.u0 += kItem + tiles;
      if (w.j * tokens >= w.q.n) {
        w.j = 0;
        do {
          if (++w.r == p.n_requests) {
            w.r = 0;
            ++w.h;
          }
        } while (s_first[w.r] == s_first[w.r + 1]);
        if (w.h < p.kv_heads && w.u0 < c.x1) w.q = request(p, w.r);
      }
      if (here) {
        w.more = 1;
        break;
      }
    }
  }
  __syncwarp();
  return w.more != 0;
}

// 4-D tiled load into this CTA's shared memory, completion counted on `bar`.
__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(tc::smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(tc::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2),
      "r"(c3)
      : "memory");
}

// ---- host: tensor maps ----
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  }
  return fn;
}

// bf16 tensor map of `rank` dimensions (the first contiguous; strides in elements of the
// others), 128-byte swizzle, zero fill out of bounds.
inline int make_map(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims,
                    const int64_t* strides, const cuuint32_t* box) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return DDT_ERR_CUDA;
  cuuint64_t bytes[4];
  for (int i = 0; i + 1 < rank; ++i) bytes[i] = static_cast<cuuint64_t>(strides[i]) * 2;
  const cuuint32_t es[5] = {1, 1, 1, 1, 1};
  const CUresult r =
      fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, bytes, box, es,
         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? DDT_OK : DDT_ERR_ALIGN;
}

// The launch of the kernel for requests of few new tokens (paged_decode.cu): all rows of a
// request and KV head, max_new * group <= kShortRows, in one unit.
constexpr int kShortRows = 32;
constexpr int kShortCtas = 2 * kSms;
size_t short_workspace_bytes();
int launch_short(Params& p, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                 int64_t q_heads, const CUtensorMap& tm_k, const CUtensorMap& tm_v, void* workspace,
                 cudaStream_t st);

}  // namespace paged_attn
}  // namespace ddt
