// Sampling with temperature, top-k, top-p and min-p from given uniforms, one token per row.
//
// Weights are whole numbers, w_i = floor(exp((x_i - max) / T) * 2^40), so every sum of them is
// exact and the token does not depend on the order in which a launch adds.  The kept tokens are
// a prefix of the order (logit descending, index ascending), so they are described by a key
// (the order-preserving image of a logit) and an index: a token is kept when its key is above
// the key, or equal and its index at most the index.
//
// One CTA per row.  The key of the k-th token, and of the token at which the running weight
// reaches top_p of the total, are found by a search over the 32 bits of the key, one pass over
// the row per bit.
#include <cuda_bf16.h>

#include "common.cuh"

namespace ddt {
namespace sample {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr float kUnit = 1099511627776.f;  // 2^40
constexpr double kLogUnit = 27.725887222397812;  // 40 ln 2

struct Args {
  const void* logits;
  int vocab;
  long long row_stride;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* tokens;
  float* logprobs;
};

template <bool kBF16>
__device__ __forceinline__ float load_logit(const void* row, int i) {
  float x;
  if constexpr (kBF16)
    x = bf16_bits_to_f32(static_cast<const uint16_t*>(row)[i]);
  else
    x = static_cast<const float*>(row)[i];
  return isnan(x) ? -INFINITY : x;
}

// (exp of the scaled distance to the maximum, a plain division and CUDA's expf: the weight is
// defined by them)
__device__ __forceinline__ float scaled(float x, float top, float temp) {
  return x == top ? 0.f : (x - top) / temp;
}
__device__ __forceinline__ long long weight_of(float e) { return static_cast<long long>(e * kUnit); }

__device__ __forceinline__ long long block_sum(long long v, long long* s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(DDT_FULL_MASK, v, o);
  __syncthreads();
  if (lane == 0) s[warp] = v;
  __syncthreads();
  long long t = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) t += s[w];
  return t;
}

template <bool kBF16>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Args a) {
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int V = a.vocab;
  const void* x = static_cast<const char*>(a.logits) + row * a.row_stride * (kBF16 ? 2 : 4);
  __shared__ long long s_sum[kWarps];
  __shared__ uint32_t s_key[kWarps];
  __shared__ int s_pick;
  auto logit = [&](int i) { return load_logit<kBF16>(x, i); };

  uint32_t top_key = 0;
  for (int i = tid; i < V; i += kThreads) top_key = max(top_key, f32_key(logit(i)));
  top_key = __reduce_max_sync(DDT_FULL_MASK, top_key);
  if (lane == 0) s_key[warp] = top_key;
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) top_key = max(top_key, s_key[w]);
  const float top = key_f32(top_key);
  if (top == -INFINITY) {
    if (tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  const float temp_in = a.temperature[row];
  const bool greedy = !(temp_in >= 1e-5f);
  const float temp = greedy ? 1.f : temp_in;
  const int k_in = a.top_k ? a.top_k[row] : 0;
  const int k = greedy ? 1 : (k_in > 0 && k_in < V ? k_in : V);
  const double p = a.top_p && !greedy ? static_cast<double>(a.top_p[row]) : 1.0;
  const float min_p = a.min_p && !greedy ? fminf(a.min_p[row], 1.f) : 0.f;
  auto weight = [&](float v) { return weight_of(expf(scaled(v, top, temp))); };

  // The kept set: keys above `key`, and the first `ties` (by index) of the keys equal to it.
  uint32_t key = 0;
  long long ties = V;
  if (k < V) {
    // the largest key with at least k keys at or above it
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t cand = key | (1u << bit);
      long long c = 0;
      for (int i = tid; i < V; i += kThreads) c += f32_key(logit(i)) >= cand;
      if (block_sum(c, s_sum) >= k) key = cand;
    }
    long long c = 0;
    for (int i = tid; i < V; i += kThreads) c += f32_key(logit(i)) > key;
    ties = k - block_sum(c, s_sum);
  }
  if (p < 1.0) {
    // of the kept ones: the weight strictly above a key, with the ties of the boundary key
    const uint32_t k_key = key;
    const long long k_ties = ties;
    const bool bounded = k < V;
    auto above = [&](uint32_t c) {  // weight of the kept tokens with keys above c
      long long s = 0, t = 0;
      for (int i = tid; i < V; i += kThreads) {
        const float v = logit(i);
        const uint32_t kk = f32_key(v);
        if (kk > c && (!bounded || kk > k_key)) s += weight(v);
      }
      if (bounded && c < k_key) t = k_ties * weight(key_f32(k_key));
      return block_sum(s, s_sum) + t;
    };
    const double reach = p * static_cast<double>(above(0));
    // the smallest key whose strictly greater kept weight is below the reach
    uint32_t lo = 0, hi = top_key;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (static_cast<double>(above(mid)) < reach) hi = mid;
      else lo = mid + 1;
    }
    if (lo > k_key || !bounded) {
      key = lo;
      ties = V;
    }
    // of the tokens with this key the first ones whose weight before them is below the reach
    const long long before = above(key), each = weight(key_f32(key));
    if (each > 0) {
      long long a0 = 0, a1 = ties;  // number of ties kept, by bisection on the exact test
      while (a0 < a1) {
        const long long mid = a0 + (a1 - a0) / 2;
        if (static_cast<double>(before + mid * each) < reach) a0 = mid + 1;
        else a1 = mid;
      }
      ties = a0;
    }
    if (key == top_key && ties < 1) ties = 1;
  }

  // Total weight, then the token, walking the row in blocks of kThreads indices.
  auto kept = [&](int i, float v, int& tie_base) {  // collective; ties counted in index order
    const uint32_t kk = i < V ? f32_key(v) : 0;
    const bool tie = i < V && kk == key;
    const unsigned int b = __ballot_sync(DDT_FULL_MASK, tie);
    __syncthreads();
    if (lane == 0) s_key[warp] = __popc(b);
    __syncthreads();
    int mine = tie_base + __popc(b & ((1u << lane) - 1u)), all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) mine += s_key[w];
      all += s_key[w];
    }
    tie_base += all;
    return i < V && (kk > key || (tie && mine < ties)) && expf(scaled(v, top, temp)) >= min_p;
  };
  long long sum = 0;
  int tie_base = 0;
  for (int i0 = 0; i0 < V; i0 += kThreads) {
    const int i = i0 + tid;
    const float v = i < V ? logit(i) : -INFINITY;
    if (kept(i, v, tie_base)) sum += weight(v);
  }
  const long long total = block_sum(sum, s_sum);
  long long target = static_cast<long long>(floor(static_cast<double>(a.u[row]) * static_cast<double>(total)));
  target = max(min(target, total - 1), 0ll);
  long long run = 0;
  tie_base = 0;
  if (tid == 0) s_pick = V;
  for (int i0 = 0; i0 < V; i0 += kThreads) {
    const int i = i0 + tid;
    const float v = i < V ? logit(i) : -INFINITY;
    const long long w = kept(i, v, tie_base) ? weight(v) : 0;
    const long long block = block_sum(w, s_sum);
    if (run + block > target) {
      long long incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(DDT_FULL_MASK, incl, o);
        if (lane >= o) incl += y;
      }
      __syncthreads();
      if (lane == 31) s_sum[warp] = incl;
      __syncthreads();
      for (int q = 0; q < warp; ++q) incl += s_sum[q];
      if (run + incl > target && w > 0) atomicMin(&s_pick, i);
      break;
    }
    run += block;
  }
  __syncthreads();
  if (tid == 0) {
    a.tokens[row] = s_pick;
    if (a.logprobs)
      a.logprobs[row] = static_cast<float>(static_cast<double>(scaled(logit(s_pick), top, temp)) -
                                           (log(static_cast<double>(total)) - kLogUnit));
  }
}

}  // namespace sample
}  // namespace ddt

using namespace ddt;

extern "C" size_t ddt_sample_workspace_bytes(int64_t rows, int64_t vocab) {
  (void)rows;
  (void)vocab;
  return 0;
}

extern "C" int ddt_sample(const void* logits, int dtype, int64_t rows, int64_t vocab,
                          int64_t row_stride, const float* u, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p,
                          int64_t* tokens, float* logprobs, void* workspace,
                          size_t workspace_bytes, void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  if (dtype != DDT_F32 && dtype != DDT_BF16) return DDT_ERR_DTYPE;
  if (rows < 0 || vocab <= 0 || row_stride < vocab) return DDT_ERR_INVALID;
  if (vocab >= (int64_t(1) << 22) || rows > 0x7fffffff) return DDT_ERR_CAPACITY;
  if (rows == 0) return DDT_OK;
  if (!logits || !u || !temperature || !tokens) return DDT_ERR_INVALID;
  if (!aligned(logits, dtype == DDT_F32 ? 4 : 2)) return DDT_ERR_ALIGN;
  sample::Args a{logits, static_cast<int>(vocab), row_stride, u, temperature, top_k, top_p, min_p,
                 tokens, logprobs};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == DDT_BF16)
    sample::sample_kernel<true><<<static_cast<unsigned>(rows), sample::kThreads, 0, st>>>(a);
  else
    sample::sample_kernel<false><<<static_cast<unsigned>(rows), sample::kThreads, 0, st>>>(a);
  return launch_status();
}
