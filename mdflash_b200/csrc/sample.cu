// Sampling with temperature, top-k, top-p and min-p from given uniforms, one token per row.
//
// Weights are whole numbers, w_i = floor(exp((x_i - max) / T) * 2^40), so every sum of them is
// exact and the token does not depend on the order in which a launch adds.  The kept tokens are
// a prefix of the order (logit descending, index ascending), so they are described by a key
// (the order-preserving image of a logit) and an index: a token is kept when its key is above
// the key, or equal and its index at most the index.
//
// A row is shared by a cluster of 1 to 8 CTAs; every warp owns a contiguous range of indices and
// reads it with 16-byte loads in every pass (the first from HBM, the others from L2):
//   1. the maximum
//   2. (top-k, top-p) the boundary key, by three radix steps of 11, 11 and 10 bits: counts and
//      weights of the tokens that share the digits found so far, per value of the next digit;
//      the histograms of the cluster's CTAs are added by each of them through distributed
//      shared memory
//   3. (a cut inside a run of equal logits) the index of the last one kept
//   4. the weight of the kept tokens; the warp that holds the target then walks its range
// Passes exchange one value per CTA through distributed shared memory and one cluster barrier.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "common.cuh"

namespace ddt {
namespace sample {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = 2048;
constexpr int kOwn = kBins / kThreads;  // bins per thread
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
  int vectors;  // rows start at 16-byte boundaries
};

// exp of the scaled distance to the maximum: a plain division and CUDA's expf, by which the
// weight is defined
__device__ __forceinline__ float scaled(float x, float top, float temp) {
  return x == top ? 0.f : (x - top) / temp;
}
// floor(e * 2^40) = hi * 2^20 + lo for e in [0, 1], hi <= 2^20, lo < 2^20: adding 8 with
// rounding toward zero leaves multiples of 2^-20 in the low mantissa bits (a conversion to 64
// bits runs at an eighth of the rate)
__device__ __forceinline__ void limbs(float e, uint32_t& hi, uint32_t& lo) {
  const float t = __fadd_rz(e, 8.f);
  hi = __float_as_uint(t) - 0x41000000u;
  lo = __float_as_uint(__fmaf_rz(e - (t - 8.f), 1048576.f, 8.f)) - 0x41000000u;
}
__device__ __forceinline__ unsigned long long whole(float e) {
  uint32_t hi, lo;
  limbs(e, hi, lo);
  return (static_cast<unsigned long long>(hi) << 20) + lo;
}

// What a CTA shows to the others of its cluster; one field per exchange, so that each needs
// one cluster barrier only.
struct Shared {
  alignas(16) uint32_t count[kBins], lo[kBins], hi[kBins];  // weight of a bin: hi * 2^32 + lo
  unsigned long long warp_sum[2][kWarps];
  unsigned long long sum;    // kept weight of the CTA
  uint32_t top_key;
  int ties, tie_index;
  // found by one thread of the CTA for all of its threads
  int bin;
  unsigned long long before_c, before_w, bin_c;
};

// Exclusive block scan of (c, w) in thread order; returns the totals too.
__device__ __forceinline__ void scan2(unsigned long long c, unsigned long long w, Shared& s,
                                      unsigned long long& c_before, unsigned long long& w_before,
                                      unsigned long long& c_all, unsigned long long& w_all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long ci = c, wi = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long yc = __shfl_up_sync(DDT_FULL_MASK, ci, o);
    const unsigned long long yw = __shfl_up_sync(DDT_FULL_MASK, wi, o);
    if (lane >= o) {
      ci += yc;
      wi += yw;
    }
  }
  __syncthreads();
  if (lane == 31) {
    s.warp_sum[0][warp] = ci;
    s.warp_sum[1][warp] = wi;
  }
  __syncthreads();
  c_before = ci - c;
  w_before = wi - w;
  c_all = w_all = 0;
#pragma unroll 8
  for (int k = 0; k < kWarps; ++k) {
    const unsigned long long a = s.warp_sum[0][k], b = s.warp_sum[1][k];
    if (k < warp) {
      c_before += a;
      w_before += b;
    }
    c_all += a;
    w_all += b;
  }
}

template <bool kBF16>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Args a) {
  constexpr int kVec = kBF16 ? 8 : 4;  // elements per 16-byte load
  constexpr int kStep = 32 * kVec;
  __shared__ Shared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int V = a.vocab;
  const char* x = static_cast<const char*>(a.logits) + row * a.row_stride * (kBF16 ? 2 : 4);

  // this warp's range of indices
  const int per_warp =
      ((V + ranks * kWarps - 1) / (ranks * kWarps) + kStep - 1) / kStep * kStep;
  const int seg0 = min(static_cast<long long>(rank * kWarps + warp) * per_warp,
                       static_cast<long long>(V));
  const int seg1 = min(seg0 + per_warp, V);

  // the kVec elements from index i on (-inf past the end; NaN as -inf)
  auto load = [&](int i, float (&v)[kVec]) {
    if (a.vectors && i + kVec <= seg1) {
      const uint4 r = *reinterpret_cast<const uint4*>(x + static_cast<long long>(i) * (kBF16 ? 2 : 4));
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        if constexpr (kBF16)
          v[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
        else
          v[e] = __uint_as_float(w[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        v[e] = -INFINITY;
        if (i + e < seg1) {
          if constexpr (kBF16)
            v[e] = bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(x)[i + e]);
          else
            v[e] = reinterpret_cast<const float*>(x)[i + e];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) v[e] = isnan(v[e]) ? -INFINITY : v[e];
  };

  // ---- 1. maximum ----------------------------------------------------------------------
  float mx = -INFINITY;
#pragma unroll 4
  for (int i = seg0 + lane * kVec; i < seg1; i += kStep) {
    float v[kVec];
    load(i, v);
#pragma unroll
    for (int e = 0; e < kVec; ++e) mx = fmaxf(mx, v[e]);
  }
  uint32_t top_key = __reduce_max_sync(DDT_FULL_MASK, f32_key(mx));
  if (tid == 0) s.top_key = 0;
  __syncthreads();
  if (lane == 0) atomicMax(&s.top_key, top_key);
  cluster.sync();
  top_key = __reduce_max_sync(DDT_FULL_MASK,
                              lane < ranks ? cluster.map_shared_rank(&s, lane)->top_key : 0u);
  const float top = key_f32(top_key);
  if (top == -INFINITY) {
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    cluster.sync();
    return;
  }

  const float temp_in = a.temperature[row];
  const bool greedy = !(temp_in >= 1e-5f);
  const float temp = greedy ? 1.f : temp_in;
  const int k_in = a.top_k ? a.top_k[row] : 0;
  const int k = greedy ? 1 : (k_in > 0 && k_in < V ? k_in : V);
  const double p = a.top_p && !greedy ? static_cast<double>(a.top_p[row]) : 1.0;
  const float min_p = a.min_p && !greedy ? fminf(a.min_p[row], 1.f) : 0.f;
  // logits this far below the maximum have weight 0: exp(-28) * 2^40 < 1
  const float floor_x = -28.f * temp;
  auto weight = [&](float v) {
    return v - top < floor_x ? 0ull : whole(expf(scaled(v, top, temp)));
  };

  // ---- 2. boundary key: kept are the keys above `key` and the first `ties` equal to it ----
  uint32_t key = 0;
  unsigned long long ties = ~0ull;   // of the `n_ties` tokens with this key
  unsigned long long n_ties = 0;
  // One search: the key of token number `want` (counts), or of the last token whose weight
  // before it is below `reach` (weights).  Of the keys equal to k_key only k_ties count.
  // Leaves the count / weight of the tokens above the key.
  auto search = [&](bool by_weight, bool weigh, unsigned long long want, double reach, double frac,
                    bool bounded, uint32_t k_key, unsigned long long k_ties,
                    unsigned long long& above_w) {
    uint32_t prefix = 0;
    unsigned long long above_c = 0;
    above_w = 0;
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
      const int known = level == 0 ? 32 : level == 1 ? 21 : 10;  // key >> known == prefix
      const uint32_t mask = level == 2 ? 1023u : 2047u;
      for (int b = tid; b < kBins; b += kThreads) s.count[b] = s.lo[b] = s.hi[b] = 0;
      __syncthreads();
#pragma unroll 2
      for (int i = seg0 + lane * kVec; i < seg1; i += kStep) {
        float v[kVec];
        load(i, v);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const uint32_t kk = f32_key(v[e]);
          if (i + e < seg1 && (level == 0 || (kk >> known) == prefix) &&
              (!bounded || kk > k_key)) {
            const uint32_t b = (kk >> shift) & mask;
            if (weigh) {
              const unsigned long long w = weight(v[e]);
              if (w) {
                const uint32_t wl = static_cast<uint32_t>(w), old = atomicAdd(&s.lo[b], wl);
                const uint32_t wh = static_cast<uint32_t>(w >> 32) + (old + wl < old ? 1u : 0u);
                if (wh) atomicAdd(&s.hi[b], wh);
              }
            }
            if (!by_weight || level == 2) atomicAdd(&s.count[b], 1u);
          }
        }
      }
      cluster.sync();
      // bins in descending order, kOwn per thread
      unsigned long long c[kOwn] = {}, w[kOwn] = {}, c_sum = 0, w_sum = 0;
      const int b0 = kBins - (tid + 1) * kOwn;  // its lowest bin
      for (int r = 0; r < ranks; ++r) {
        const Shared* o = cluster.map_shared_rank(&s, r);
        const uint4 oc = *reinterpret_cast<const uint4*>(&o->count[b0]);
        c[0] += oc.w, c[1] += oc.z, c[2] += oc.y, c[3] += oc.x;
        if (weigh) {
          const uint4 ol = *reinterpret_cast<const uint4*>(&o->lo[b0]),
                      oh = *reinterpret_cast<const uint4*>(&o->hi[b0]);
          w[0] += (static_cast<unsigned long long>(oh.w) << 32) + ol.w;
          w[1] += (static_cast<unsigned long long>(oh.z) << 32) + ol.z;
          w[2] += (static_cast<unsigned long long>(oh.y) << 32) + ol.y;
          w[3] += (static_cast<unsigned long long>(oh.x) << 32) + ol.x;
        }
      }
#pragma unroll
      for (int h = 0; h < kOwn; ++h) {
        if (bounded && (level == 0 || (k_key >> known) == prefix) &&
            ((k_key >> shift) & mask) == b0 + kOwn - 1 - h) {
          c[h] += k_ties;
          w[h] += k_ties * weight(key_f32(k_key));
        }
        c_sum += c[h];
        w_sum += w[h];
      }
      unsigned long long cb, wb, call, wall;
      scan2(c_sum, w_sum, s, cb, wb, call, wall);
      if (level == 0 && by_weight) reach = frac * static_cast<double>(wall);
      if (tid == 0) s.bin = -1;
      __syncthreads();
      unsigned long long c0 = above_c + cb, w0 = above_w + wb;
#pragma unroll
      for (int h = 0; h < kOwn; ++h) {
        // the bin that holds the boundary: it starts before it and ends at or past it
        const bool here = by_weight
                              ? static_cast<double>(w0) < reach && !(static_cast<double>(w0 + w[h]) < reach)
                              : c0 < want && want <= c0 + c[h];
        if (here) {
          s.bin = b0 + kOwn - 1 - h;
          s.before_c = c0;
          s.before_w = w0;
          s.bin_c = c[h];
        }
        c0 += c[h];
        w0 += w[h];
      }
      __syncthreads();
      // no bin: reach is 0 or less, and the first token alone is kept
      const uint32_t digit = s.bin < 0 ? (top_key >> shift) & mask : static_cast<uint32_t>(s.bin);
      if (s.bin >= 0) {
        above_c = s.before_c;
        above_w = s.before_w;
        n_ties = s.bin_c;
      }
      prefix = level == 0 ? digit : (prefix << (level == 1 ? 11 : 10)) | digit;
      cluster.sync();  // the histograms are read
    }
    key = prefix;
    ties = by_weight ? 0 : want - above_c;
    if (by_weight) {
      // of the tokens with this key the first ones whose weight before them is below the reach
      const unsigned long long each = weight(key_f32(key));
      unsigned long long a0 = 0, a1 = each ? n_ties : 0;
      while (a0 < a1) {
        const unsigned long long mid = a0 + (a1 - a0) / 2;
        if (static_cast<double>(above_w + mid * each) < reach) a0 = mid + 1;
        else a1 = mid;
      }
      ties = a0;
      if (reach <= 0.0) {
        key = top_key;
        ties = 1;
        n_ties = V;
      }
    }
  };
  if (k == 1) {
    key = top_key;
    ties = 1;
    n_ties = V;
  } else if (k < V || p < 1.0) {
    unsigned long long above_w = 0;
    if (k < V) search(false, false, k, 0.0, 0.0, false, 0, 0, above_w);
    if (p < 1.0) {
      const uint32_t k_key = key;
      const unsigned long long k_ties = ties, k_all = n_ties;
      search(true, true, 0, 0.0, p, k < V, k_key, k_ties, above_w);
      // the run of equal logits at the top-k boundary is longer than what top-k keeps of it
      if (k < V && key == k_key) n_ties = k_all;
    }
  }

  // ---- 3. index of the last kept token of the boundary key ---------------------------------
  int last = V;
  const float edge = key_f32(key);
  const bool bounded = ties != ~0ull;
  if (bounded && ties < n_ties) {
    int mine = 0;
    for (int i = seg0 + lane * kVec; i < seg1; i += kStep) {
      float v[kVec];
      load(i, v);
#pragma unroll
      for (int e = 0; e < kVec; ++e) mine += i + e < seg1 && v[e] == edge;
    }
    mine = __reduce_add_sync(DDT_FULL_MASK, mine);
    __syncthreads();
    if (lane == 0) s.warp_sum[0][warp] = mine;
    if (tid == 0) s.tie_index = V;
    __syncthreads();
    long long before = 0, all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s.warp_sum[0][w];
      all += s.warp_sum[0][w];
    }
    if (tid == 0) s.ties = static_cast<int>(all);
    cluster.sync();
    before += __reduce_add_sync(DDT_FULL_MASK,
                                lane < rank ? cluster.map_shared_rank(&s, lane)->ties : 0);
    const long long want = static_cast<long long>(ties) - before;  // of this warp's ties
    if (want >= 1 && want <= mine) {
      long long left = want;
      for (int i0 = seg0; i0 < seg1; i0 += kStep) {
        const int i = i0 + lane * kVec;
        float v[kVec];
        load(i, v);
        int n = 0;
#pragma unroll
        for (int e = 0; e < kVec; ++e) n += i + e < seg1 && v[e] == edge;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(DDT_FULL_MASK, incl, o);
          if (lane >= o) incl += y;
        }
        const int all_n = __shfl_sync(DDT_FULL_MASK, incl, 31);
        if (left <= all_n) {
          int at = incl - n;
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            if (i + e < seg1 && v[e] == edge && ++at == left) s.tie_index = i + e;
          break;
        }
        left -= all_n;
      }
    }
    cluster.sync();
    last = __reduce_min_sync(DDT_FULL_MASK,
                             lane < ranks ? cluster.map_shared_rank(&s, lane)->tie_index : V);
  }

  // ---- 4. kept weight, target, token -------------------------------------------------------
  auto kept = [&](float v, int i) { return !bounded || v > edge || (v == edge && i <= last); };
  auto kept_weight = [&](float v, int i) -> unsigned long long {
    if (v - top < floor_x || !kept(v, i)) return 0ull;
    const float e = expf(scaled(v, top, temp));
    return e >= min_p ? whole(e) : 0ull;
  };
  unsigned long long mine = 0;
#pragma unroll 2
  for (int i = seg0 + lane * kVec; i < seg1; i += kStep) {
    float v[kVec];
    load(i, v);
    // (past the end v is -inf, of weight 0)
#pragma unroll
    for (int e = 0; e < kVec; ++e) mine += kept_weight(v[e], i + e);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(DDT_FULL_MASK, mine, o);
  __syncthreads();
  if (lane == 0) s.warp_sum[0][warp] = mine;
  __syncthreads();
  unsigned long long before = 0, all = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += s.warp_sum[0][w];
    all += s.warp_sum[0][w];
  }
  if (tid == 0) s.sum = all;
  cluster.sync();
  unsigned long long total = lane < ranks ? cluster.map_shared_rank(&s, lane)->sum : 0ull;
  unsigned long long earlier = lane < rank ? total : 0ull;
#pragma unroll
  for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
    total += __shfl_xor_sync(DDT_FULL_MASK, total, o);
    earlier += __shfl_xor_sync(DDT_FULL_MASK, earlier, o);
  }
  total = __shfl_sync(DDT_FULL_MASK, total, 0);
  before += __shfl_sync(DDT_FULL_MASK, earlier, 0);
  long long t = static_cast<long long>(floor(static_cast<double>(a.u[row]) * static_cast<double>(total)));
  t = max(min(t, static_cast<long long>(total) - 1), 0ll);
  unsigned long long target = static_cast<unsigned long long>(t);
  if (before <= target && target < before + mine) {
    target -= before;
    for (int i0 = seg0; i0 < seg1; i0 += kStep) {
      const int i = i0 + lane * kVec;
      float v[kVec];
      load(i, v);
      unsigned long long w[kVec], n = 0;
#pragma unroll
      for (int e = 0; e < kVec; ++e) n += w[e] = kept_weight(v[e], i + e);
      unsigned long long incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(DDT_FULL_MASK, incl, o);
        if (lane >= o) incl += y;
      }
      const unsigned long long step = __shfl_sync(DDT_FULL_MASK, incl, 31);
      if (target < step) {
        unsigned long long at = incl - n;
        if (at <= target && target < incl) {
          int pick = 0;
          float value = 0.f;
#pragma unroll
          for (int e = 0; e < kVec; ++e) {
            if (at <= target && target < at + w[e]) {
              pick = i + e;
              value = v[e];
            }
            at += w[e];
          }
          a.tokens[row] = pick;
          if (a.logprobs)
            a.logprobs[row] =
                static_cast<float>(static_cast<double>(scaled(value, top, temp)) -
                                   (log(static_cast<double>(total)) - kLogUnit));
        }
        break;
      }
      target -= step;
    }
  }
  cluster.sync();  // no CTA leaves while another may read its shared memory
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
  if (vocab >= (int64_t(1) << 22) || rows > 0x7fffffff / sample::kMaxCluster) return DDT_ERR_CAPACITY;
  if (rows == 0) return DDT_OK;
  if (!logits || !u || !temperature || !tokens) return DDT_ERR_INVALID;
  const int64_t size = dtype == DDT_F32 ? 4 : 2;
  if (!aligned(logits, size)) return DDT_ERR_ALIGN;
  sample::Args a{logits, static_cast<int>(vocab), row_stride, u, temperature, top_k, top_p, min_p,
                 tokens, logprobs, aligned(logits, 16) && (row_stride * size) % 16 == 0};
  // as many CTAs per row as keep the rows in one wave (two CTAs per SM), and no
  // more than leave each warp one load
  int ranks = 1;
  while (ranks < sample::kMaxCluster && rows * ranks * 2 <= 2 * 148 &&
         vocab > ranks * sample::kThreads * (16 / size))
    ranks *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * ranks));
  cfg.blockDim = dim3(sample::kThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = dtype == DDT_BF16 ? cudaLaunchKernelEx(&cfg, sample::sample_kernel<true>, a)
                                          : cudaLaunchKernelEx(&cfg, sample::sample_kernel<false>, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return DDT_ERR_CUDA;
  }
  return DDT_OK;
}
