// q / k RMS norm and rotary embedding of the fused projection, with the K / V rows written to
// their slots of the paged cache.
//
// For head vector x (128 values), weight w and rotary angles a_i (i < 64):
//   y = w * x / sqrt(mean(x^2) + eps)
//   out_i = y_i cos a_i - y_{i+64} sin a_i,  out_{i+64} = y_{i+64} cos a_i + y_i sin a_i
// in fp32, rounded to bf16 once at the end.  (ddt_qk_norm_rope_cache rounds after the norm, the
// weight and each product, as the transformers modules do; one rounding halves the error.)
//
// One warp per (token, head): lane l holds elements [4 l, 4 l + 4), the rotary partner of an
// element lies in lane l ^ 16.
#include <cuda_bf16.h>

#include "common.cuh"

namespace ddt {
namespace paged {

constexpr int kHeadDim = 128;

struct WriteArgs {
  const __nv_bfloat16* qkv;
  long long qkv_stride;
  long long n_tokens;
  int q_heads, kv_heads;
  const __nv_bfloat16* qw;
  const __nv_bfloat16* kw;
  float eps;
  const uint32_t* rope;  // [n_tokens, 64]: bf16 cos | bf16 sin << 16
  const int64_t* slots;
  __nv_bfloat16* q_out;
  __nv_bfloat16* k_pages;
  __nv_bfloat16* v_pages;
  long long n_slots;
  int page_shift;
  long long page_stride, head_stride, row_stride;
};

__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__global__ void __launch_bounds__(256) paged_write_kernel(const WriteArgs a) {
  const int lane = threadIdx.x & 31;
  const long long gw = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int heads = a.q_heads + 2 * a.kv_heads;
  if (gw >= a.n_tokens * heads) return;
  const long long tok = gw / heads;
  const int hh = static_cast<int>(gw - tok * heads);
  const uint2 raw =
      *reinterpret_cast<const uint2*>(a.qkv + tok * a.qkv_stride + hh * kHeadDim + lane * 4);
  const bool is_q = hh < a.q_heads, is_v = hh >= a.q_heads + a.kv_heads;
  uint2 outv = raw;
  if (!is_v) {
    const uint2 wraw = *reinterpret_cast<const uint2*>((is_q ? a.qw : a.kw) + lane * 4);
    const uint4 cs = *reinterpret_cast<const uint4*>(a.rope + tok * (kHeadDim / 2) + (lane & 15) * 4);
    float x[4] = {lo_f(raw.x), hi_f(raw.x), lo_f(raw.y), hi_f(raw.y)};
    const float w[4] = {lo_f(wraw.x), hi_f(wraw.x), lo_f(wraw.y), hi_f(wraw.y)};
    const uint32_t c[4] = {cs.x, cs.y, cs.z, cs.w};
    float ss = x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(DDT_FULL_MASK, ss, o);
    const float inv = rsqrtf(ss * (1.f / kHeadDim) + a.eps);
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= inv * w[e];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float partner = __shfl_xor_sync(DDT_FULL_MASK, x[e], 16);
      y[e] = x[e] * lo_f(c[e]) + (lane < 16 ? -partner : partner) * hi_f(c[e]);
    }
    __nv_bfloat16* oe = reinterpret_cast<__nv_bfloat16*>(&outv);
#pragma unroll
    for (int e = 0; e < 4; ++e) oe[e] = __float2bfloat16_rn(y[e]);
  }
  if (is_q) {
    *reinterpret_cast<uint2*>(a.q_out + (tok * a.q_heads + hh) * kHeadDim + lane * 4) = outv;
    return;
  }
  const long long slot = a.slots[tok];
  if (slot < 0 || slot >= a.n_slots) return;
  const int h = hh - a.q_heads - (is_v ? a.kv_heads : 0);
  __nv_bfloat16* dst = (is_v ? a.v_pages : a.k_pages) + (slot >> a.page_shift) * a.page_stride +
                       h * a.head_stride +
                       (slot & ((1ll << a.page_shift) - 1)) * a.row_stride + lane * 4;
  *reinterpret_cast<uint2*>(dst) = outv;
}

}  // namespace paged
}  // namespace ddt

using namespace ddt;

extern "C" int ddt_paged_qk_norm_rope(const void* qkv, int64_t qkv_stride, int64_t n_tokens,
                                      int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                      const void* q_norm_w, const void* k_norm_w, float eps,
                                      const void* rope_table, const int64_t* slot_map, void* q_out,
                                      void* k_pages, void* v_pages, int64_t n_pages,
                                      int64_t page_size, int64_t page_stride, int64_t head_stride,
                                      int64_t row_stride, void* stream) {
  if (n_tokens < 0 || q_heads <= 0 || kv_heads <= 0 || n_pages <= 0) return DDT_ERR_INVALID;
  if (head_dim != paged::kHeadDim) return DDT_ERR_CAPACITY;
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return DDT_ERR_CAPACITY;
  if (qkv_stride < (q_heads + 2 * kv_heads) * head_dim) return DDT_ERR_INVALID;
  const int64_t warps = n_tokens * (q_heads + 2 * kv_heads);
  if (n_tokens > 0x7fffffff || (warps + 7) / 8 > 0x7fffffff) return DDT_ERR_CAPACITY;
  if (n_tokens == 0) return DDT_OK;
  if (!qkv || !q_norm_w || !k_norm_w || !rope_table || !slot_map || !q_out || !k_pages || !v_pages)
    return DDT_ERR_INVALID;
  if (!aligned(qkv, 16) || !aligned(q_norm_w, 16) || !aligned(k_norm_w, 16) ||
      !aligned(rope_table, 16) || !aligned(slot_map, 8) || !aligned(q_out, 16) ||
      !aligned(k_pages, 16) || !aligned(v_pages, 16) || qkv_stride % 8 || page_stride % 8 ||
      head_stride % 8 || row_stride % 8)
    return DDT_ERR_ALIGN;
  paged::WriteArgs a;
  a.qkv = static_cast<const __nv_bfloat16*>(qkv);
  a.qkv_stride = qkv_stride;
  a.n_tokens = n_tokens;
  a.q_heads = static_cast<int>(q_heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.qw = static_cast<const __nv_bfloat16*>(q_norm_w);
  a.kw = static_cast<const __nv_bfloat16*>(k_norm_w);
  a.eps = eps;
  a.rope = static_cast<const uint32_t*>(rope_table);
  a.slots = slot_map;
  a.q_out = static_cast<__nv_bfloat16*>(q_out);
  a.k_pages = static_cast<__nv_bfloat16*>(k_pages);
  a.v_pages = static_cast<__nv_bfloat16*>(v_pages);
  a.n_slots = n_pages * page_size;
  a.page_shift = __builtin_ctzll(static_cast<unsigned long long>(page_size));
  a.page_stride = page_stride;
  a.head_stride = head_stride;
  a.row_stride = row_stride;
  paged::paged_write_kernel<<<static_cast<unsigned>((warps + 7) / 8), 256, 0,
                              static_cast<cudaStream_t>(stream)>>>(a);
  return launch_status();
}
