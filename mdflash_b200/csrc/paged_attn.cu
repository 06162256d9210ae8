// Causal attention of every request's new tokens over its pages of the K/V cache.
//
// Row i of request r (new token i, one query head) sees the keys j <= len_r - n_r + i:
//   o_i = sum_j 2^(s_ij - m_i) v_j / sum_j 2^(s_ij - m_i),   s_ij = q_i . k_j * scale * log2 e
// with the running maximum m and sum l of a one-pass softmax: a new maximum m' rescales what
// was summed by 2^(m - m').  A row that sees no key gives 0.
//
// One CTA per (token, KV head), one warp per key at a time; the heads of the group share the
// key.
#include <cuda_bf16.h>

#include "common.cuh"
#include "tc.cuh"

namespace ddt {
namespace paged_attn {

constexpr int kHeadDim = 128;
constexpr int kMaxGroup = 64;
constexpr int kWarps = 8;

struct Params {
  const __nv_bfloat16* q;
  long long q_token_stride, q_head_stride;
  const __nv_bfloat16* k_pages;
  const __nv_bfloat16* v_pages;
  long long page_stride, head_stride, row_stride, n_pages;
  int page_shift;
  const int32_t* block_table;
  long long table_stride, max_keys;
  const int32_t* cu_new;
  const int32_t* kv_lens;
  int n_requests, n_tokens, max_new, group;
  float scale_log2;
  __nv_bfloat16* out;
  long long o_token_stride, o_head_stride;
  int32_t* status;
};

// Lengths of request r, or false (and the status bit) where they are out of range.
__device__ __forceinline__ bool request(const Params& p, int r, int& first, int& n, int& len) {
  first = p.cu_new[r];
  const int end = p.cu_new[r + 1];
  len = p.kv_lens[r];
  if (first < 0 || end < first || end > p.n_tokens || end - first > p.max_new || len < 0 ||
      len > p.max_keys) {
    if (p.status) atomicOr(p.status, DDT_STATUS_PAGED_RANGE);
    n = 0;
    return false;
  }
  n = end - first;
  return true;
}

constexpr int kHeads = 4;  // heads of the group per pass over the keys

__global__ void __launch_bounds__(kWarps * 32) paged_attn_simple_kernel(const Params p) {
  const int tok = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // the request that owns this token
  int lo = 0, hi = p.n_requests - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.cu_new[mid] <= tok) lo = mid;
    else hi = mid - 1;
  }
  int first, n, len;
  if (!request(p, lo, first, n, len) || tok < first || tok >= first + n) return;
  const int keys = max(len - n + (tok - first) + 1, 0);
  __shared__ float s_m[kWarps][kHeads], s_l[kWarps][kHeads];
  __shared__ float s_o[kWarps][kHeads][kHeadDim];
  for (int g0 = 0; g0 < p.group; g0 += kHeads) {
    float q[kHeads][4], o[kHeads][4], m[kHeads], l[kHeads];
#pragma unroll
    for (int g = 0; g < kHeads; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.f;
      uint2 raw = make_uint2(0, 0);
      if (g0 + g < p.group)
        raw = *reinterpret_cast<const uint2*>(p.q + tok * p.q_token_stride +
                                              (h * p.group + g0 + g) * p.q_head_stride + lane * 4);
      q[g][0] = __uint_as_float(raw.x << 16);
      q[g][1] = __uint_as_float(raw.x & 0xffff0000u);
      q[g][2] = __uint_as_float(raw.y << 16);
      q[g][3] = __uint_as_float(raw.y & 0xffff0000u);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[g][e] = 0.f;
    }
    for (int j = warp; j < keys; j += kWarps) {
      const long long pg = p.block_table[lo * p.table_stride + (j >> p.page_shift)];
      if (pg < 0 || pg >= p.n_pages) continue;
      const long long at = pg * p.page_stride + h * p.head_stride +
                           (j & ((1 << p.page_shift) - 1)) * p.row_stride + lane * 4;
      const uint2 kr = *reinterpret_cast<const uint2*>(p.k_pages + at);
      const uint2 vr = *reinterpret_cast<const uint2*>(p.v_pages + at);
      const float kf[4] = {__uint_as_float(kr.x << 16), __uint_as_float(kr.x & 0xffff0000u),
                           __uint_as_float(kr.y << 16), __uint_as_float(kr.y & 0xffff0000u)};
      const float vf[4] = {__uint_as_float(vr.x << 16), __uint_as_float(vr.x & 0xffff0000u),
                           __uint_as_float(vr.y << 16), __uint_as_float(vr.y & 0xffff0000u)};
#pragma unroll
      for (int g = 0; g < kHeads; ++g) {
        float s = q[g][0] * kf[0] + q[g][1] * kf[1] + q[g][2] * kf[2] + q[g][3] * kf[3];
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(DDT_FULL_MASK, s, w);
        s *= p.scale_log2;
        const float mn = fmaxf(m[g], s);
        const float alpha = mn == -INFINITY ? 1.f : exp2f(m[g] - mn);
        const float w = mn == -INFINITY ? 0.f : exp2f(s - mn);
        m[g] = mn;
        l[g] = l[g] * alpha + w;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[g][e] = o[g][e] * alpha + w * vf[e];
      }
    }
#pragma unroll
    for (int g = 0; g < kHeads; ++g) {
      if (lane == 0) {
        s_m[warp][g] = m[g];
        s_l[warp][g] = l[g];
      }
      *reinterpret_cast<float4*>(&s_o[warp][g][lane * 4]) =
          make_float4(o[g][0], o[g][1], o[g][2], o[g][3]);
    }
    __syncthreads();
    for (int x = threadIdx.x; x < kHeads * kHeadDim; x += kWarps * 32) {
      const int g = x / kHeadDim, d = x % kHeadDim;
      if (g0 + g < p.group) {
        float M = -INFINITY, L = 0.f, acc = 0.f;
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w][g]);
        for (int w = 0; w < kWarps; ++w) {
          const float f = s_m[w][g] == -INFINITY ? 0.f : exp2f(s_m[w][g] - M);
          L += f * s_l[w][g];
          acc += f * s_o[w][g][d];
        }
        p.out[tok * p.o_token_stride + (h * p.group + g0 + g) * p.o_head_stride + d] =
            __float2bfloat16_rn(L > 0.f ? acc / L : 0.f);
      }
    }
    __syncthreads();
  }
}

}  // namespace paged_attn
}  // namespace ddt

using namespace ddt;

extern "C" size_t ddt_paged_attn_workspace_bytes(int64_t n_tokens, int64_t max_new,
                                                 int64_t q_heads, int64_t kv_heads) {
  (void)n_tokens;
  (void)max_new;
  (void)q_heads;
  (void)kv_heads;
  return 0;
}

extern "C" int ddt_paged_attn(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                              const void* k_pages, const void* v_pages, int64_t n_pages,
                              int64_t page_size, int64_t page_stride, int64_t head_stride,
                              int64_t row_stride, const int32_t* block_table, int64_t table_stride,
                              int64_t max_pages, const int32_t* cu_new, const int32_t* kv_lens,
                              int64_t n_requests, int64_t n_tokens, int64_t max_new,
                              int64_t q_heads, int64_t kv_heads, int64_t head_dim, float scale,
                              void* out, int64_t o_token_stride, int64_t o_head_stride,
                              void* workspace, size_t workspace_bytes, int32_t* status,
                              void* stream) {
  using namespace paged_attn;
  (void)workspace;
  (void)workspace_bytes;
  if (n_requests <= 0 || n_tokens < 0 || max_new < 0 || q_heads <= 0 || kv_heads <= 0 ||
      q_heads % kv_heads || n_pages <= 0 || max_pages <= 0 || table_stride < max_pages)
    return DDT_ERR_INVALID;
  if (head_dim != kHeadDim || q_heads / kv_heads > kMaxGroup) return DDT_ERR_CAPACITY;
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return DDT_ERR_CAPACITY;
  if (n_requests > DDT_MAX_PAGED_REQUESTS || n_tokens > 0x7fffffff || n_pages > 0x7fffffff ||
      max_pages * page_size > 0x7fffffff || kv_heads > 65535)
    return DDT_ERR_CAPACITY;
  if (n_tokens == 0 || max_new == 0) return DDT_OK;
  if (!q || !k_pages || !v_pages || !block_table || !cu_new || !kv_lens || !out)
    return DDT_ERR_INVALID;
  if (!aligned(q, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(out, 16) ||
      q_token_stride % 8 || q_head_stride % 8 || page_stride % 8 || head_stride % 8 ||
      row_stride % 8 || o_token_stride % 8 || o_head_stride % 8)
    return DDT_ERR_ALIGN;
  Params p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_token_stride = q_token_stride;
  p.q_head_stride = q_head_stride;
  p.k_pages = static_cast<const __nv_bfloat16*>(k_pages);
  p.v_pages = static_cast<const __nv_bfloat16*>(v_pages);
  p.page_stride = page_stride;
  p.head_stride = head_stride;
  p.row_stride = row_stride;
  p.n_pages = n_pages;
  p.page_shift = __builtin_ctzll(static_cast<unsigned long long>(page_size));
  p.block_table = block_table;
  p.table_stride = table_stride;
  p.max_keys = max_pages * page_size;
  p.cu_new = cu_new;
  p.kv_lens = kv_lens;
  p.n_requests = static_cast<int>(n_requests);
  p.n_tokens = static_cast<int>(n_tokens);
  p.max_new = static_cast<int>(max_new < n_tokens ? max_new : n_tokens);
  p.group = static_cast<int>(q_heads / kv_heads);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.o_token_stride = o_token_stride;
  p.o_head_stride = o_head_stride;
  p.status = status;
  paged_attn_simple_kernel<<<dim3(static_cast<unsigned>(n_tokens), static_cast<unsigned>(kv_heads)),
                             kWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return launch_status();
}
