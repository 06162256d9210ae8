// q / k RMS norm and rotary embedding of the fused projection, with the K / V rows written to
// their slots of the paged cache.
//
// For head vector x (128 values), weight w and rotary angles a_i (i < 64):
//   y = w * x / sqrt(mean(x^2) + eps)
//   out_i = y_i cos a_i - y_{i+64} sin a_i,  out_{i+64} = y_{i+64} cos a_i + y_i sin a_i
// in fp32, rounded to bf16 once at the end.  (ddt_qk_norm_rope_cache rounds after the norm, the
// weight and each product, as the transformers modules do; one rounding halves the error.)
//
// HBM-bound (12.3 KB read and written per token at 32 + 8 heads).  A warp takes some heads of one
// token, two at a time: 16 lanes per head, lane c the elements [4 c, 4 c + 4) and their rotary
// partners 64 on; the token's angles and the norm weights stay in registers, eight loads are in
// flight.  8191 tokens take 40 us, 5.0 TB/s or 0.77 of the copy rate.  (One head per warp: 70 us;
// 16-byte loads with the partner fetched by a shuffle: 46 us; two pairs in flight: 45 us.)
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
__device__ __forceinline__ void spread4(const uint2& r, float* x) {
  x[0] = lo_f(r.x);
  x[1] = hi_f(r.x);
  x[2] = lo_f(r.y);
  x[3] = hi_f(r.y);
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

constexpr int kWriteThreads = 256;
constexpr int kBatch = 4;  // pairs of heads in flight

__global__ void __launch_bounds__(kWriteThreads)
paged_write_kernel(const WriteArgs a, const int heads_per_warp, const int chunks) {
  const int lane = threadIdx.x & 31;
  let_next_begin();  // the attention's
  const long long gw =
      static_cast<long long>(blockIdx.x) * (kWriteThreads / 32) + (threadIdx.x >> 5);
  const long long tok = gw / chunks;
  if (tok >= a.n_tokens) return;
  const int h0 = static_cast<int>(gw - tok * chunks) * heads_per_warp;
  const int heads = a.q_heads + 2 * a.kv_heads;
  const int h1 = min(h0 + heads_per_warp, heads);
  const int sub = lane >> 4, c = lane & 15;  // head of the pair, elements 4 c .. and 64 + 4 c ..
  const __nv_bfloat16* src = a.qkv + tok * a.qkv_stride + c * 4;
  const long long slot = a.slots[tok];
  const bool writes = slot >= 0 && slot < a.n_slots;
  const long long at = (slot >> a.page_shift) * a.page_stride +
                       (slot & ((1ll << a.page_shift) - 1)) * a.row_stride + c * 4;
  const uint4 angles = *reinterpret_cast<const uint4*>(a.rope + tok * (kHeadDim / 2) + c * 4);
  const uint32_t ang[4] = {angles.x, angles.y, angles.z, angles.w};
  uint2 qw[2], kw[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    qw[p] = *reinterpret_cast<const uint2*>(a.qw + p * 64 + c * 4);
    kw[p] = *reinterpret_cast<const uint2*>(a.kw + p * 64 + c * 4);
  }
  for (int hb = h0; hb < h1; hb += 2 * kBatch) {
    uint2 raw[kBatch][2];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = hb + 2 * i + sub;
#pragma unroll
      for (int p = 0; p < 2; ++p)
        raw[i][p] = h < h1 ? *reinterpret_cast<const uint2*>(src + h * kHeadDim + p * 64)
                           : make_uint2(0, 0);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (hb + 2 * i >= h1) break;  // warp-uniform
      const int h = hb + 2 * i + sub;
      const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.kv_heads;
      float x[8], w[8], ss = 0.f;
      spread4(raw[i][0], x);
      spread4(raw[i][1], x + 4);
      spread4(is_q ? qw[0] : kw[0], w);
      spread4(is_q ? qw[1] : kw[1], w + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(DDT_FULL_MASK, ss, o);
      const float inv = rsqrtf(ss * (1.f / kHeadDim) + a.eps);
      uint2 out[2] = {raw[i][0], raw[i][1]};
      if (!is_v) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float u = x[e] * (inv * w[e]), v = x[e + 4] * (inv * w[e + 4]);
          const float cs = lo_f(ang[e]), sn = hi_f(ang[e]);
          y[e] = u * cs - v * sn;
          y[e + 4] = v * cs + u * sn;
        }
        out[0] = make_uint2(pack2(y[0], y[1]), pack2(y[2], y[3]));
        out[1] = make_uint2(pack2(y[4], y[5]), pack2(y[6], y[7]));
      }
      if (h >= h1 || !(is_q || writes)) continue;
      __nv_bfloat16* dst =
          is_q ? a.q_out + (tok * a.q_heads + h) * kHeadDim + c * 4
               : (is_v ? a.v_pages : a.k_pages) + at +
                     (h - a.q_heads - (is_v ? a.kv_heads : 0)) * a.head_stride;
      *reinterpret_cast<uint2*>(dst) = out[0];
      *reinterpret_cast<uint2*>(dst + 64) = out[1];
    }
  }
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
  if (n_tokens > 0x7fffffff || q_heads + 2 * kv_heads > 0xffff) return DDT_ERR_CAPACITY;
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
  // few tokens: 2 heads per warp, so that they still cover the SMs; many: 24, which read the
  // token's angles once (64 tokens of 48 heads: 2.9 us in a recorded graph)
  const int64_t heads = q_heads + 2 * kv_heads;
  const int per_warp = n_tokens * heads <= 148 * 64 * 2 ? 2 : n_tokens * heads <= 148 * 64 * 8 ? 8 : 24;
  const int64_t chunks = (heads + per_warp - 1) / per_warp;
  const int64_t blocks = (n_tokens * chunks + paged::kWriteThreads / 32 - 1) / (paged::kWriteThreads / 32);
  if (blocks > 0x7fffffff) return DDT_ERR_CAPACITY;
  // (not launch_early: behind a kernel of 3 us it costs the host 1.2 us more, and gains 0.2)
  paged::paged_write_kernel<<<static_cast<unsigned>(blocks), paged::kWriteThreads, 0,
                              static_cast<cudaStream_t>(stream)>>>(a, per_warp,
                                                                   static_cast<int>(chunks));
  return launch_status();
}
