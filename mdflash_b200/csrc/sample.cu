// Sampling with temperature, top-k, top-p and min-p from given uniforms, one token per row.
//
// Weights are whole numbers, w_i = floor(exp((x_i - max) / T) * 2^40), so every sum of them is
// exact and the token does not depend on the order in which a launch adds.  The kept tokens are
// a prefix of the order (logit descending, index ascending), described by its last token: kept
// are the logits above `edge`, and the equal ones up to index `last`.
//
// A row is shared by a cluster of 1 to 8 CTAs; every warp owns a contiguous range of indices and
// reads it with 16-byte loads in every pass (the first from HBM, the others from L2):
//   1. the maximum (and, where the row is truncated, the minimum)
//   2. top-k and top-p: counts of the row over 2048 equal intervals of the logits, added over
//      the cluster through distributed shared memory (for top-p alone also the row's weight)
//      - top-k: the interval that holds token number k; all tokens down to it are listed (some
//        tens or hundreds of 152k) and sorted, and the rest happens on the list
//      - top-p alone: the interval where the running weight should reach top_p, judged by the
//        intervals' counts and middles; the tokens of it and its neighbours are listed and
//        sorted, the ones above weighed, and the boundary taken from the exact sums
//      - where a list is too long (a large k, long runs of equal logits) or the boundary lies
//        outside it: exact weights per interval, and a search by the bits of the key
//   3. the weight of the kept tokens; the warps of the CTA that holds the target share the
//      range of the warp that holds it, until that is one load per lane
// CTAs exchange values through distributed shared memory, with one cluster barrier each time.
//
// Measured over 151936 logits: one fp32 row with top-k 50 and top-p 0.95 18 us, with top-p alone
// 30 us, untruncated 12 us (all latency: passes of 3 to 8 us, barriers and remote reads between
// them); 64 bf16 rows of mixed rules 55 us (the slowest row); 257 fp32 rows untruncated 82 us,
// 1.9 TB/s: the exponential, its quotient and the split into whole numbers are 25 instructions
// per logit, and rows in step read HBM and compute in turn.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "common.cuh"

namespace ddt {
namespace sample {

namespace cg = cooperative_groups;

// (the row's passes are lambdas over its elements; out of line their captures would live in
// local memory)
#define DDT_INLINE __attribute__((always_inline))

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = 2048;
constexpr int kOwn = kBins / kThreads;  // bins per thread
constexpr int kList = 2048;
constexpr int kPer = kList / kThreads;  // listed tokens per thread
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

// a / b, correctly rounded, for the many a of one b: with y the correctly rounded reciprocal
// and q within one unit in the last place, q + (a - q b) y rounds to the quotient (P. Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor", IBM J. Res.
// Dev. 34, 1990); the first step brings a y that close.  (Five instructions without a branch
// between the elements of a load; equal to the division for 2^35 random pairs and 2^33 with a
// significand of b of all ones or close to it.)
struct Divisor {
  float b, y;
  __device__ explicit Divisor(float d) : b(d), y(1.f / d) {}
  __device__ __forceinline__ float operator()(float a) const {
    float q = a * y;
    q = __fmaf_rn(__fmaf_rn(-q, b, a), y, q);
    return __fmaf_rn(__fmaf_rn(-q, b, a), y, q);
  }
};

// floor(e * 2^40) = hi * 2^20 + lo for e in [0, 1], hi <= 2^20, lo < 2^20: adding 8 with
// rounding toward zero leaves multiples of 2^-20 in the low mantissa bits (a conversion to 64
// bits runs at a fraction of the rate)
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

// What a CTA shows to the others of its cluster, and its own scratch.
struct Shared {
  alignas(16) uint32_t count[kBins], lo[kBins], hi[kBins];  // weight of a bin: hi * 2^32 + lo
  unsigned long long list[kList];  // this CTA's part of a list (ordered())
  unsigned long long all[kList];   // the cluster's list
  unsigned long long warp_sum[2][kWarps];
  unsigned long long sum, above;  // weights of the CTA
  uint32_t top_key, low_key;
  int n_list, ties, tie_index;
  // found by one thread of the CTA for all of its threads
  int bin, window, kept, range0, range1;
  unsigned long long before_c, before_w, bin_c;
};

// A token as a whole number: larger for a larger logit, then for a smaller index.
__device__ __forceinline__ unsigned long long ordered(float v, int i) {
  return (static_cast<unsigned long long>(f32_key(v)) << 32) | static_cast<uint32_t>(~i);
}
__device__ __forceinline__ float value_of(unsigned long long t) {
  return key_f32(static_cast<uint32_t>(t >> 32));
}
__device__ __forceinline__ int index_of(unsigned long long t) {
  return static_cast<int>(~static_cast<uint32_t>(t));
}

// Exclusive block scan of (c, w) in thread order; returns the totals too.
__device__ __forceinline__ void scan2(unsigned long long c, unsigned long long w, Shared& s,
                                      unsigned long long& c_before, unsigned long long& w_before,
                                      unsigned long long& w_all) {
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
  w_all = 0;
#pragma unroll 4
  for (int k = 0; k < kWarps; ++k) {
    const unsigned long long a = s.warp_sum[0][k], b = s.warp_sum[1][k];
    if (k < warp) {
      c_before += a;
      w_before += b;
    }
    w_all += b;
  }
}

// Sort of n <= kList numbers `a` in descending order by the whole block; zeros are dropped, and
// the number of the others is returned.  `bin` maps a number to an interval in [0, kBins), no
// larger number to a higher one.  Up to kRanked numbers by counting the larger ones of each (140
// numbers in 0.4 us).  More by the intervals: a count, the prefix of the counts, every number to
// its interval's part of `scratch` [kList], and counting within the part (1400 numbers in about
// 3 us; a bitonic sort's 66 barriers took 25).
constexpr int kRanked = 256;
static_assert(kRanked <= kThreads, "one number per thread");
template <typename Bin>
__device__ __forceinline__ int sort_descending(unsigned long long* a, int n,
                                               unsigned long long* scratch, Shared& s, Bin bin) {
  const int tid = threadIdx.x;
  if (n <= kRanked) {
    const unsigned long long x = tid < n ? a[tid] : 0ull;
    int rank = 0;
    if (x) {
#pragma unroll 8
      for (int o = 0; o < n; ++o) rank += a[o] > x;
    }
    const int m = __syncthreads_count(x != 0);
    if (x) a[rank] = x;
    __syncthreads();
    return m;
  }
  for (int b = tid; b < kBins; b += kThreads) s.count[b] = 0;
  __syncthreads();
  unsigned long long x[kPer], before, w0, w_all;
  int b[kPer], at[kPer];
#pragma unroll
  for (int h = 0; h < kPer; ++h) {
    const int j = tid + h * kThreads;
    x[h] = j < n ? a[j] : 0ull;
    if (x[h]) {
      b[h] = bin(x[h]);
      at[h] = atomicAdd(&s.count[b[h]], 1u);
    }
  }
  __syncthreads();
  const uint4 c = *reinterpret_cast<const uint4*>(&s.count[tid * kOwn]);
  static_assert(kOwn == 4, "one load per thread");
  scan2(static_cast<unsigned long long>(c.x) + c.y + c.z + c.w, c.x + c.y + c.z + c.w, s, before, w0,
        w_all);
  const uint32_t f = static_cast<uint32_t>(before);
  *reinterpret_cast<uint4*>(&s.lo[tid * kOwn]) =
      make_uint4(f, f + c.x, f + c.x + c.y, f + c.x + c.y + c.z);
  __syncthreads();
#pragma unroll
  for (int h = 0; h < kPer; ++h)
    if (x[h]) scratch[s.lo[b[h]] + at[h]] = x[h];
  __syncthreads();
#pragma unroll
  for (int h = 0; h < kPer; ++h) {
    if (!x[h]) continue;
    const uint32_t from = s.lo[b[h]], to = from + s.count[b[h]];
    uint32_t rank = from;
    for (uint32_t o = from; o < to; ++o) rank += scratch[o] > x[h];
    a[rank] = x[h];
  }
  __syncthreads();
  return static_cast<int>(w_all);
}

template <bool kBF16>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const Args a) {
  constexpr int kVec = kBF16 ? 8 : 4;  // elements per 16-byte load
  constexpr int kStep = 32 * kVec;
  extern __shared__ unsigned char smem_raw[];
  Shared& s = *reinterpret_cast<Shared*>(smem_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int V = a.vocab;
  const char* x = static_cast<const char*>(a.logits) + row * a.row_stride * (kBF16 ? 2 : 4);
  auto peer = [&](int r) { return cluster.map_shared_rank(&s, r); };

  after_stream();
  let_next_begin();

  // ---- the row's rules --------------------------------------------------------------------
  const float temp_in = a.temperature[row];
  const bool greedy = !(temp_in >= 1e-5f);
  const float temp = greedy ? 1.f : fminf(temp_in, 1e30f);  // (its reciprocal is normal)
  const float p_in = a.top_p && !greedy ? a.top_p[row] : 1.f;
  const int k_in = a.top_k ? a.top_k[row] : 0;
  const int k = greedy || p_in <= 0.f ? 1 : (k_in > 0 && k_in < V ? k_in : V);
  const double p = k > 1 ? static_cast<double>(p_in) : 1.0;
  const float min_p = a.min_p && !greedy ? fminf(a.min_p[row], 1.f) : 0.f;
  const Divisor by_temp(temp);

  // ---- reading ------------------------------------------------------------------------------
  // this warp's range of indices
  const int per_warp =
      ((V + ranks * kWarps - 1) / (ranks * kWarps) + kStep - 1) / kStep * kStep;
  const int seg0 = min(static_cast<long long>(rank * kWarps + warp) * per_warp,
                       static_cast<long long>(V));
  const int seg1 = min(seg0 + per_warp, V);
  bool inf_top = false;  // +inf takes all of the weight: the row is then read as 0 and -inf
  // kVec elements of a 16-byte load
  auto spread = [&](const uint4& r, float (&v)[kVec]) DDT_INLINE {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      if constexpr (kBF16)
        v[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
      else
        v[e] = __uint_as_float(w[e]);
    }
    if (inf_top) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = v[e] == INFINITY ? 0.f : -INFINITY;
    }
  };
  auto vec_at = [&](int i) DDT_INLINE {
    return __ldg(reinterpret_cast<const uint4*>(x + static_cast<long long>(i) * (kBF16 ? 2 : 4)));
  };
  // the kVec elements from index i on; NaN at and past `end`: like every NaN they are below
  // all, equal to none and of weight 0
  auto load = [&](int i, int end, float (&v)[kVec]) DDT_INLINE {
    if (a.vectors && i + kVec <= end) {
      spread(vec_at(i), v);
      return;
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      v[e] = __uint_as_float(0x7fffffffu);
      if (i + e < end) {
        if constexpr (kBF16)
          v[e] = bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(x)[i + e]);
        else
          v[e] = reinterpret_cast<const float*>(x)[i + e];
        if (inf_top) v[e] = v[e] == INFINITY ? 0.f : -INFINITY;
      }
    }
  };
  // f(first index, kVec values) over [begin, end) of this warp, every `every`-th step of it:
  // kBatch loads are in flight before the first is used
  auto vectors = [&](int begin, int end, int every, auto f) DDT_INLINE {
    constexpr int kBatch = 4;
    const int step = kStep * every;
    int i = begin + lane * kVec;
    if (a.vectors)
      for (; i - lane * kVec + (kBatch - 1) * step + kStep <= end; i += kBatch * step) {
        uint4 r[kBatch];
#pragma unroll
        for (int h = 0; h < kBatch; ++h) r[h] = vec_at(i + h * step);
#pragma unroll
        for (int h = 0; h < kBatch; ++h) {
          float v[kVec];
          spread(r[h], v);
          f(i + h * step, v);
        }
      }
    for (; i < end; i += step) {
      float v[kVec];
      load(i, end, v);
      f(i, v);
    }
  };
  // f(index, value) over this warp's range
  auto each = [&](auto f) DDT_INLINE {
    vectors(seg0, seg1, 1, [&](int i, float (&v)[kVec]) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) f(i + e, v[e]);
    });
  };

  // ---- 1. maximum and minimum ------------------------------------------------------------
  float mx = -INFINITY, mn = INFINITY;
  if (k < V || p < 1.0) {
    each([&](int, float v) {
      mx = fmaxf(mx, v);
      mn = fminf(mn, v);
    });
  } else {
    each([&](int, float v) { mx = fmaxf(mx, v); });
  }
  uint32_t top_key = __reduce_max_sync(DDT_FULL_MASK, f32_key(mx));
  uint32_t low_key = __reduce_min_sync(DDT_FULL_MASK, f32_key(mn));
  if (tid == 0) {
    s.top_key = 0;
    s.low_key = ~0u;
    s.tie_index = V;
  }
  __syncthreads();
  if (lane == 0) {
    atomicMax(&s.top_key, top_key);
    atomicMin(&s.low_key, low_key);
  }
  cluster.sync();
  top_key = __reduce_max_sync(DDT_FULL_MASK, lane < ranks ? peer(lane)->top_key : 0u);
  low_key = __reduce_min_sync(DDT_FULL_MASK, lane < ranks ? peer(lane)->low_key : ~0u);
  float top = key_f32(top_key);
  if (top == -INFINITY) {
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    cluster.sync();
    return;
  }
  if (top == INFINITY) {
    inf_top = true;
    top = 0.f;
    low_key = f32_key(-INFINITY);
  }

  // ---- weights ------------------------------------------------------------------------------
  // exp of the scaled distance to the maximum, by CUDA's expf; -200 stands for all that is
  // far below a weight of 1 and for the NaN of -inf and NaN logits
  auto scaled = [&](float v) { return fmaxf(by_temp(v - top), -200.f); };
  auto weight = [&](float v) { return whole(expf(scaled(v))); };
  // what is kept: the logits above `edge`, and the equal ones up to index `last`
  float edge = -INFINITY;
  int last = V;
  bool all_kept = true;  // of the tokens that have weight
  auto kept = [&](int i, float v) { return all_kept || v > edge || (v == edge && i <= last); };
  auto warp_total = [&](unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(DDT_FULL_MASK, v, o);
    return v;
  };
  // sum of `part` over the CTA's warps before this one, and over all of them
  auto before_warp = [&](unsigned long long part, unsigned long long& all) {
    __syncthreads();
    if (lane == 0) s.warp_sum[0][warp] = part;
    __syncthreads();
    unsigned long long before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const unsigned long long o = s.warp_sum[0][w];
      if (w < warp) before += o;
      all += o;
    }
    return before;
  };
  // sum over the cluster's CTAs of a value that they published, and over those before this one
  auto cluster_total = [&](unsigned long long mine_at_lane, unsigned long long& earlier) {
    unsigned long long total = lane < ranks ? mine_at_lane : 0ull;
    earlier = lane < rank ? total : 0ull;
#pragma unroll
    for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
      total += __shfl_xor_sync(DDT_FULL_MASK, total, o);
      earlier += __shfl_xor_sync(DDT_FULL_MASK, earlier, o);
    }
    earlier = __shfl_sync(DDT_FULL_MASK, earlier, 0);
    return __shfl_sync(DDT_FULL_MASK, total, 0);
  };

  // ---- the draw -------------------------------------------------------------------------------
  // floor(u * total), at most total - 1
  auto target_of = [&](unsigned long long total) {
    const long long t =
        static_cast<long long>(floor(static_cast<double>(a.u[row]) * static_cast<double>(total)));
    return static_cast<unsigned long long>(max(min(t, static_cast<long long>(total) - 1), 0ll));
  };
  auto write = [&](float v, int i, unsigned long long total) {
    a.tokens[row] = i;
    if (a.logprobs)
      a.logprobs[row] = static_cast<float>(static_cast<double>(scaled(v)) -
                                           (log(static_cast<double>(total)) - kLogUnit));
  };

  // ---- 2. what top-k and top-p keep -----------------------------------------------------------
  // interval of a logit: equal intervals from the maximum down to the minimum, or to where
  // weights end (the last interval takes the rest)
  const float span = fminf(top - key_f32(low_key), 28.f * temp);
  const float per_unit = span > 0.f ? (kBins - 1) / span : 0.f;
  auto place_of = [&](float v) { return __fmul_rn(__fsub_rn(top, v), per_unit); };
  // (adding 2^23 with rounding toward zero leaves the whole part in the low bits, at four times
  // the rate of a conversion; of NaN it makes the last interval)
  auto bin_of = [&](float v) {
    return static_cast<int>(__float_as_uint(__fadd_rz(fminf(place_of(v), kBins - 1.f), 8388608.f)) -
                            0x4b000000u);
  };
  // Where a search only has to come close (its result is checked), a quarter of the row is
  // counted: the counters' updates, several to one bank, are what a counting pass waits for.
  const int every = per_warp >= 8 * kStep ? 4 : 1;
  // interval of a listed token among kBins that share the intervals [b0, b1] of the row
  auto list_bin = [&](int b0, int b1) {
    const float scale = (kBins - 1.f) / (b1 + 1 - b0);
    return [&, b0, scale](unsigned long long t) {
      const float at = (place_of(value_of(t)) - b0) * scale;
      return __float2int_rz(fminf(fmaxf(at, 0.f), kBins - 1.f));
    };
  };
  auto clear = [&] {
    for (int b = tid; b < kBins; b += kThreads) s.count[b] = s.lo[b] = s.hi[b] = 0;
    if (tid == 0) {
      s.bin = -1;
      s.n_list = s.window = 0;
    }
    __syncthreads();
  };
  // this thread's kOwn bins b0 .. of every CTA of the cluster, all loads in flight together (one
  // after the other eight of them took 5 us)
  auto bins_of_all = [&](const uint32_t* own, int b0, auto add) {
    uint4 o[kMaxCluster];
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r)
      o[r] = r < ranks ? *reinterpret_cast<const uint4*>(cluster.map_shared_rank(own, r) + b0)
                       : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      add(0, o[r].x);
      add(1, o[r].y);
      add(2, o[r].z);
      add(3, o[r].w);
    }
  };
  auto bin_counts = [&](int b0, unsigned long long (&c)[kOwn]) {
    bins_of_all(s.count, b0, [&](int h, uint32_t x) { c[h] += x; });
  };
  // Histogram of the kept tokens by `bin` (those with a bin >= 0), added over the cluster; then
  // the bin that holds the boundary: by weight the last one whose weight before it is below
  // `reach`, else the one that holds token number `want`.  s.bin, s.before_c, s.before_w, s.bin_c.
  double reach = 0.0;
  auto boundary = [&](bool by_weight, bool count, bool ascending, unsigned long long want,
                      unsigned long long above_c, unsigned long long above_w, bool set_reach,
                      auto bin) DDT_INLINE {
    clear();
    each([&](int i, float v) {
      const int b = v == v && kept(i, v) ? bin(v) : -1;
      if (b >= 0) {
        if (by_weight) {
          const unsigned long long w = weight(v);
          if (w) {
            const uint32_t wl = static_cast<uint32_t>(w), old = atomicAdd(&s.lo[b], wl);
            const uint32_t wh = static_cast<uint32_t>(w >> 32) + (old + wl < old ? 1u : 0u);
            if (wh) atomicAdd(&s.hi[b], wh);
          }
        }
        if (count) atomicAdd(&s.count[b], 1u);
      }
    });
    cluster.sync();
    // thread t owns kOwn bins, in the order of the tokens
    unsigned long long c[kOwn] = {}, w[kOwn] = {}, c_sum = 0, w_sum = 0;
    const int b0 = (ascending ? tid : kThreads - 1 - tid) * kOwn;
    if (count) bin_counts(b0, c);
    if (by_weight) {
      bins_of_all(s.lo, b0, [&](int h, uint32_t x) { w[h] += x; });
      bins_of_all(s.hi, b0, [&](int h, uint32_t x) { w[h] += static_cast<unsigned long long>(x) << 32; });
    }
#pragma unroll
    for (int h = 0; h < kOwn; ++h) {
      c_sum += c[h];
      w_sum += w[h];
    }
    unsigned long long c0, w0, w_all;
    scan2(c_sum, w_sum, s, c0, w0, w_all);
    if (set_reach) reach = p * static_cast<double>(w_all);
    c0 += above_c;
    w0 += above_w;
#pragma unroll
    for (int g = 0; g < kOwn; ++g) {
      const int h = ascending ? g : kOwn - 1 - g;
      const bool here = by_weight ? static_cast<double>(w0) < reach &&
                                        !(static_cast<double>(w0 + w[h]) < reach)
                                  : c0 < want && want <= c0 + c[h];
      if (here) {
        s.bin = b0 + h;
        s.before_c = c0;
        s.before_w = w0;
        s.bin_c = c[h];
      }
      c0 += c[h];
      w0 += w[h];
    }
    __syncthreads();
  };
  // this CTA's part of a list, as far as it fits
  auto append = [&](int i, float v) {
    const int at = atomicAdd(&s.n_list, 1);
    if (at < kList) s.list[at] = ordered(v, i);
  };
  // The cluster's list into s.all, in any order; its length (nothing is copied above kList).
  auto gather = [&] {
    const int mine = lane < ranks ? peer(lane)->n_list : 0;
    const int n = __reduce_add_sync(DDT_FULL_MASK, mine);
    if (n > kList) return n;
    int length[kMaxCluster];
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) length[r] = __shfl_sync(DDT_FULL_MASK, mine, r);
    unsigned long long t[kPer];  // loaded from all CTAs at once
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      int j = tid + h * kThreads, from = 0;
      if (j >= n) continue;
#pragma unroll
      for (int r = 0; r < kMaxCluster - 1; ++r)
        if (from == r && j >= length[r]) {
          j -= length[r];
          ++from;
        }
      t[h] = peer(from)->list[j];
    }
#pragma unroll
    for (int h = 0; h < kPer; ++h)
      if (tid + h * kThreads < n) s.all[tid + h * kThreads] = t[h];
    __syncthreads();
    return n;
  };
  // weights before this thread's kPer tokens of the sorted s.all, and of all n
  auto running = [&](int n, unsigned long long (&w)[kPer], unsigned long long& all) {
    unsigned long long sum = 0, c0, before;
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      const int j = tid * kPer + h;
      w[h] = sum;
      if (j < n) sum += weight(value_of(s.all[j]));
    }
    scan2(0ull, sum, s, c0, before, all);
#pragma unroll
    for (int h = 0; h < kPer; ++h) w[h] += before;
  };
  // Moves (edge, last) to the last token of the sorted s.all that keep(number in the list, weight
  // before it) holds for: a prefix of it, and at least the first.  Returns how many.
  auto settle = [&](int n, const unsigned long long (&w)[kPer], auto keep) {
    int held = 0;
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      const int j = tid * kPer + h;
      held += j < n && keep(j, w[h]);
    }
    held = __reduce_add_sync(DDT_FULL_MASK, held);
    if (tid == 0) s.kept = 0;
    __syncthreads();
    if (lane == 0) atomicAdd(&s.kept, held);
    __syncthreads();
    const int m = s.kept;
    edge = value_of(s.all[m - 1]);
    last = index_of(s.all[m - 1]);
    all_kept = false;
    return m;
  };

  // top-k on a list of all candidates, by the first CTA: false, and nothing done, where the
  // list would be too long, or turns out too long or too short.
  auto by_list = [&]() -> bool {
    clear();
    vectors(seg0, seg1, every, [&](int, float (&v)[kVec]) {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (v[e] == v[e]) atomicAdd(&s.count[bin_of(v[e])], 1u);
    });
    cluster.sync();
    unsigned long long c[kOwn] = {}, c_sum = 0, c0, w0, w_all;
    bin_counts(tid * kOwn, c);
#pragma unroll
    for (int h = 0; h < kOwn; ++h) c_sum += c[h];
    scan2(c_sum, 0ull, s, c0, w0, w_all);
    // half as many again as k, and some: a count of a quarter is off by a few square roots
    const unsigned long long want = (k + k / 2 + 64) / every;
#pragma unroll
    for (int h = 0; h < kOwn; ++h) {
      if (c0 < want && want <= c0 + c[h]) {
        s.bin = tid * kOwn + h;
        s.window = static_cast<int>(min(c0 + c[h], 1ull << 20)) * every;
      }
      c0 += c[h];
    }
    __syncthreads();
    const int bin = s.bin < 0 ? kBins - 1 : s.bin;  // (none: the row has not that many)
    const bool fits = s.bin < 0 ? V <= kList : s.window <= kList;
    cluster.sync();  // the histograms are read
    if (!fits) return false;
    const float past = bin + 1.f;
    vectors(seg0, seg1, 1, [&](int i, float (&v)[kVec]) {
      float top_of = v[0];
#pragma unroll
      for (int e = 1; e < kVec; ++e) top_of = fmaxf(top_of, v[e]);
      if (!(place_of(top_of) < past)) return;
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (place_of(v[e]) < past) append(i + e, v[e]);
    });
    cluster.sync();
    const int listed = __reduce_add_sync(DDT_FULL_MASK, lane < ranks ? peer(lane)->n_list : 0);
    const bool good = listed >= k && listed <= kList;
    if (good && rank == 0) gather();
    cluster.sync();  // the lists are read
    if (!good || rank != 0) return good;
    sort_descending(s.all, listed, s.list, s, list_bin(0, bin));
    const int n = min(listed, k);
    unsigned long long w[kPer], all;
    running(n, w, all);
    const double limit = p * static_cast<double>(all);
    // the kept ones, as (~index | key), to be drawn from in the order of the indices
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      const int j = tid * kPer + h;
      if (j >= n) continue;
      const unsigned long long t = s.all[j];
      const bool in = (j == 0 || !(p < 1.0) || static_cast<double>(w[h]) < limit) &&
                      expf(scaled(value_of(t))) >= min_p;
      s.list[j] = in ? (t << 32) | (t >> 32) : 0ull;
    }
    __syncthreads();
    // (intervals of equal runs of indices)
    const int run = max(32 - __clz(V - 1) - 11, 0);
    const int m = sort_descending(s.list, n, s.all, s, [&](unsigned long long t) {
      return static_cast<int>(~static_cast<uint32_t>(t >> 32) >> run);
    });
    unsigned long long own[kPer], sum = 0, before, total;
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      const int j = tid * kPer + h;
      own[h] = j < m ? weight(key_f32(static_cast<uint32_t>(s.list[j]))) : 0ull;
      sum += own[h];
    }
    scan2(0ull, sum, s, c0, before, total);
    const unsigned long long target = target_of(total);
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      if (before <= target && target < before + own[h]) {
        const unsigned long long t = s.list[tid * kPer + h];
        write(key_f32(static_cast<uint32_t>(t)), static_cast<int>(~static_cast<uint32_t>(t >> 32)),
              total);
      }
      before += own[h];
    }
    return true;
  };

  // top-p alone: (edge, last), and the weight that this warp's range keeps.  False, and nothing
  // done, where the intervals' middles mislead or a list would be too long.
  auto nucleus = [&](unsigned long long& mine) -> bool {
    clear();
    unsigned long long sum = 0, all, earlier;
    vectors(seg0, seg1, 1, [&](int, float (&v)[kVec]) {
      uint32_t hi = 0, lo = 0;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        if (v[e] == v[e]) atomicAdd(&s.count[bin_of(v[e])], 1u);
        uint32_t h, l;
        limbs(expf(scaled(v[e])), h, l);
        hi += h;
        lo += l;
      }
      sum += (static_cast<unsigned long long>(hi) << 20) + lo;
    });
    before_warp(warp_total(sum), all);
    if (tid == 0) s.sum = all;
    cluster.sync();
    const unsigned long long whole_row =
        cluster_total(lane < ranks ? peer(lane)->sum : 0ull, earlier);
    reach = p * static_cast<double>(whole_row);
    unsigned long long c[kOwn] = {}, w[kOwn], c_sum = 0, w_sum = 0, c0, w0, w_all;
    const int b0 = tid * kOwn;
    bin_counts(b0, c);
    const float width = per_unit > 0.f ? 1.f / per_unit : 0.f;
#pragma unroll
    for (int h = 0; h < kOwn; ++h) {
      w[h] = c[h] * whole(expf(scaled(top - (b0 + h + 0.5f) * width)));
      c_sum += c[h];
      w_sum += w[h];
    }
    if (tid == 0) {
      s.range0 = kBins;
      s.range1 = -1;
    }
    scan2(c_sum, w_sum, s, c0, w0, w_all);
    // judged from the row's end: what follows the boundary is many light tokens, whose
    // distances from their intervals' middles cancel; a heavy token's would not
    double from = static_cast<double>(whole_row) - static_cast<double>(w_all - w0);
    unsigned long long at = c0;
#pragma unroll
    for (int h = 0; h < kOwn; ++h) {
      const double to = from + static_cast<double>(w[h]);
      if (from < reach && !(to < reach)) {
        s.bin = b0 + h;
        s.before_c = at;
      }
      from = to;
      at += c[h];
    }
    __syncthreads();
    // and its neighbours: one interval on either side, and more where they hold few tokens (the
    // list is sorted)
    const long long near = static_cast<long long>(s.before_c), room = 128;
    at = c0;
#pragma unroll
    for (int h = 0; h < kOwn; ++h) {
      const int b = b0 + h;
      if (b <= s.bin && (b >= s.bin - 1 || static_cast<long long>(at) >= near - room))
        atomicMin(&s.range0, b);
      at += c[h];
      if (s.bin >= 0 && b >= s.bin && (b <= s.bin + 1 || static_cast<long long>(at) <= near + room))
        atomicMax(&s.range1, b);
      if (b >= s.bin - 1 && b <= s.bin + 1) atomicAdd(&s.window, static_cast<int>(c[h]));
    }
    __syncthreads();
    const int lo_bin = s.range0, hi_bin = s.range1;
    const bool fits = s.bin >= 0 && s.window <= kList - 2 * room;
    cluster.sync();  // the histograms are read
    if (!fits) return false;
    const float from_here = static_cast<float>(lo_bin), past = hi_bin + 1.f;
    unsigned long long above = 0, counted = 0;  // weights above the window, and of min_p or more
    vectors(seg0, seg1, 1, [&](int i, float (&v)[kVec]) {
      float top_of = v[0];
#pragma unroll
      for (int e = 1; e < kVec; ++e) top_of = fmaxf(top_of, v[e]);
      if (!(place_of(top_of) < past)) return;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float at = place_of(v[e]);
        if (at < from_here) {
          const float x = expf(scaled(v[e]));
          const unsigned long long w = whole(x);
          above += w;
          if (x >= min_p) counted += w;
        } else if (at < past) {
          append(i + e, v[e]);
        }
      }
    });
    before_warp(warp_total(above), all);
    if (tid == 0) s.above = all;
    cluster.sync();
    const unsigned long long over =
        cluster_total(lane < ranks ? peer(lane)->above : 0ull, earlier);
    const int n = gather();
    cluster.sync();  // the lists are read
    if (n > kList) return false;
    sort_descending(s.all, n, s.list, s, list_bin(lo_bin, hi_bin));
    unsigned long long lw[kPer], l_all;
    running(n, lw, l_all);
    if (!(static_cast<double>(over) < reach) || static_cast<double>(over + l_all) < reach) return false;
    const int m = settle(n, lw, [&](int, unsigned long long before) {
      return static_cast<double>(over + before) < reach;
    });
    for (int j = lane; j < m; j += 32) {
      const int i = index_of(s.all[j]);
      if (i < seg0 || i >= seg1) continue;
      const float x = expf(scaled(value_of(s.all[j])));
      if (x >= min_p) counted += whole(x);
    }
    mine = warp_total(counted);
    return true;
  };

  // Moves (edge, last) to token number `want` of the kept ones, or to the last of them whose
  // weight before it is below p times the weight of all: for every row, with exact sums.
  auto cut = [&](bool by_weight, unsigned long long want) {
    boundary(by_weight, !by_weight, true, want, 0, 0, by_weight, bin_of);
    const int bin = s.bin;
    if (bin < 0) {  // fewer tokens than `want` (NaN is none): all stay, in every CTA alike
      cluster.sync();  // the histograms are read
      return;
    }
    const unsigned long long above_c = s.before_c, above_w = s.before_w;
    each([&](int i, float v) {
      if (v == v && kept(i, v) && bin_of(v) == bin) append(i, v);
    });
    cluster.sync();
    const int n = gather();
    cluster.sync();  // the lists are read
    if (n <= kList) {
      sort_descending(s.all, n, s.list, s, list_bin(bin, bin));
      unsigned long long w[kPer] = {}, all;
      if (by_weight) running(n, w, all);
      settle(n, w, [&](int j, unsigned long long before) {
        return by_weight ? static_cast<double>(above_w + before) < reach : above_c + j < want;
      });
      return;
    }
    // a long list: three steps over the bits of the key, from the top
    uint32_t prefix = 0;
    unsigned long long c_above = 0, w_above = 0, n_ties = 0;
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
      const int known = level == 0 ? 32 : level == 1 ? 21 : 10;  // key >> known == prefix
      const uint32_t mask = level == 2 ? 1023u : 2047u;
      boundary(by_weight, !by_weight || level == 2, false, want, c_above, w_above, false,
               [&](float v) {
                 const uint32_t key = f32_key(v);
                 return level == 0 || (key >> known) == prefix ? static_cast<int>((key >> shift) & mask)
                                                               : -1;
               });
      c_above = s.before_c;
      w_above = s.before_w;
      n_ties = s.bin_c;
      prefix = level == 0 ? s.bin : (prefix << (level == 1 ? 11 : 10)) | s.bin;
      cluster.sync();  // the histograms are read
    }
    const float value = key_f32(prefix);
    // how many of the tokens with this logit stay
    unsigned long long ties = want - c_above;
    if (by_weight) {
      const unsigned long long one = weight(value);
      unsigned long long a0 = 0, a1 = n_ties;
      while (a0 < a1) {
        const unsigned long long mid = a0 + (a1 - a0) / 2;
        if (static_cast<double>(w_above + mid * one) < reach) a0 = mid + 1;
        else a1 = mid;
      }
      ties = a0;
    }
    // and the index of the last of them
    int mine = 0;
    each([&](int i, float v) { mine += v == value && kept(i, v); });
    mine = __reduce_add_sync(DDT_FULL_MASK, mine);
    unsigned long long all, earlier;
    unsigned long long before = before_warp(mine, all);
    if (tid == 0) {
      s.ties = static_cast<int>(all);
      s.tie_index = V;
    }
    cluster.sync();
    cluster_total(lane < ranks ? peer(lane)->ties : 0, earlier);
    long long left = static_cast<long long>(ties - before - earlier);  // of this warp's
    if (left >= 1 && left <= mine) {
      for (int i0 = seg0; i0 < seg1; i0 += kStep) {
        const int i = i0 + lane * kVec;
        float v[kVec];
        load(i, seg1, v);
        int m = 0;
#pragma unroll
        for (int e = 0; e < kVec; ++e) m += v[e] == value && kept(i + e, v[e]);
        int incl = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(DDT_FULL_MASK, incl, o);
          if (lane >= o) incl += y;
        }
        const int step = __shfl_sync(DDT_FULL_MASK, incl, 31);
        if (left <= step) {
          int at = incl - m;
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            if (v[e] == value && kept(i + e, v[e]) && ++at == left) s.tie_index = i + e;
          break;
        }
        left -= step;
      }
    }
    cluster.sync();
    last = __reduce_min_sync(DDT_FULL_MASK, lane < ranks ? peer(lane)->tie_index : V);
    edge = value;
    all_kept = false;
    cluster.sync();  // before the next search writes again
  };

  unsigned long long mine = 0;  // kept weight of this warp's range
  bool weighed = false;
  if (k == 1) {
    // the first of the largest
    int first = V;
    each([&](int i, float v) { first = v == top ? min(first, i) : first; });
    first = __reduce_min_sync(DDT_FULL_MASK, first);
    if (lane == 0) atomicMin(&s.tie_index, first);
    cluster.sync();
    first = __reduce_min_sync(DDT_FULL_MASK, lane < ranks ? peer(lane)->tie_index : V);
    if (rank == 0 && tid == 0) write(top, first, whole(1.f));
    cluster.sync();
    return;
  }
  if (k < V) {
    if (by_list()) return;
    cut(false, k);
    if (p < 1.0) cut(true, 0);
  } else if (p < 1.0) {
    weighed = nucleus(mine);
    if (!weighed) cut(true, 0);
  }

  // ---- 3. kept weight, target, token ---------------------------------------------------------
  auto kept_limbs = [&](int i, float v, uint32_t& hi, uint32_t& lo) {
    const float e = expf(scaled(v));
    const bool in = e >= min_p && kept(i, v);
    limbs(e, hi, lo);
    hi = in ? hi : 0;
    lo = in ? lo : 0;
  };
  // kept weight of the warp's [begin, end)
  auto weigh = [&](int begin, int end) {
    unsigned long long sum = 0;
    if (all_kept) {
      vectors(begin, end, 1, [&](int, float (&v)[kVec]) {
        uint32_t hi = 0, lo = 0;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float x = expf(scaled(v[e]));
          uint32_t h, l;
          limbs(x, h, l);
          if (x >= min_p) {
            hi += h;
            lo += l;
          }
        }
        sum += (static_cast<unsigned long long>(hi) << 20) + lo;
      });
    } else {
      vectors(begin, end, 1, [&](int i, float (&v)[kVec]) {
        float top_of = v[0];
#pragma unroll
        for (int e = 1; e < kVec; ++e) top_of = fmaxf(top_of, v[e]);
        if (!(top_of >= edge)) return;
        uint32_t hi = 0, lo = 0;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          uint32_t h, l;
          kept_limbs(i + e, v[e], h, l);
          hi += h;
          lo += l;
        }
        sum += (static_cast<unsigned long long>(hi) << 20) + lo;
      });
    }
    return warp_total(sum);
  };
  unsigned long long all, earlier;
  if (!weighed) mine = weigh(seg0, seg1);
  unsigned long long before = before_warp(mine, all);
  if (tid == 0) s.sum = all;
  cluster.sync();
  const unsigned long long total =
      cluster_total(lane < ranks ? peer(lane)->sum : 0ull, earlier);
  // the last look at another CTA's shared memory: those without the token leave once all have
  // had theirs
  cluster.barrier_arrive();
  unsigned long long target = target_of(total);
  if (earlier <= target && target < earlier + all) {  // this CTA holds the token
    // its warps share the range of the warp that holds it, until a warp's part is one step
    target -= earlier;
    int begin = seg0, end = seg1;
    while (true) {
      if (before <= target && target < before + mine && lane == 0) {
        s.range0 = begin;
        s.range1 = end;
        s.before_w = before;
      }
      __syncthreads();
      target -= s.before_w;
      const int r0 = s.range0, r1 = s.range1;
      if (r1 - r0 <= kStep) break;
      const int part = ((r1 - r0 + kWarps - 1) / kWarps + kStep - 1) / kStep * kStep;
      begin = min(r0 + warp * part, r1);
      end = min(begin + part, r1);
      mine = weigh(begin, end);
      before = before_warp(mine, all);
    }
    if (warp == 0) {
      const int i = s.range0 + lane * kVec;
      float v[kVec];
      load(i, s.range1, v);
      unsigned long long w[kVec], n = 0;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        uint32_t h, l;
        kept_limbs(i + e, v[e], h, l);
        n += w[e] = (static_cast<unsigned long long>(h) << 20) + l;
      }
      unsigned long long at = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(DDT_FULL_MASK, at, o);
        if (lane >= o) at += y;
      }
      at -= n;
      if (at <= target && target < at + n) {
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
        write(value, pick, total);
      }
    }
  }
  cluster.barrier_wait();
}

}  // namespace sample
}  // namespace ddt

using namespace ddt;

extern "C" int ddt_sample(const void* logits, int dtype, int64_t rows, int64_t vocab,
                          int64_t row_stride, const float* u, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p,
                          int64_t* tokens, float* logprobs, void* stream) {
  if (dtype != DDT_F32 && dtype != DDT_BF16) return DDT_ERR_DTYPE;
  if (rows < 0 || vocab <= 0 || (row_stride < vocab && row_stride != 0)) return DDT_ERR_INVALID;
  if (vocab >= (int64_t(1) << 22) || rows > 0x7fffffff / sample::kMaxCluster) return DDT_ERR_CAPACITY;
  if (rows == 0) return DDT_OK;
  if (!logits || !u || !temperature || !tokens) return DDT_ERR_INVALID;
  const int64_t size = dtype == DDT_F32 ? 4 : 2;
  if (!aligned(logits, size)) return DDT_ERR_ALIGN;
  sample::Args a{logits, static_cast<int>(vocab), row_stride, u, temperature, top_k, top_p, min_p,
                 tokens, logprobs, aligned(logits, 16) && (row_stride * size) % 16 == 0};
  // as many CTAs per row as keep the rows in one wave (two CTAs per SM; of the clusters of eight,
  // whose SMs are neighbours, no more than 13: 24 fp32 rows with top-k and top-p take 18.9 us with
  // 4 CTAs each, 24.9 with 8, and 32 rows 20.3 and 32.8; 13 rows with top-p alone 38.2 with 4, 31.0
  // with 8), or the rows in flight in L2 (they are read again; 257 rows of 608 KB: 82 us with 2
  // CTAs each, 95 with 4), and no more than leave each thread one load
  int ranks = 1;
  while (ranks < sample::kMaxCluster && vocab > ranks * sample::kThreads * (16 / size) &&
         (rows * ranks * 2 <= (ranks < 4 ? 2 * 148 : 104) ||
          2 * 148 / ranks * vocab * size > (int64_t(100) << 20)))
    ranks *= 2;
  auto kernel = dtype == DDT_BF16 ? sample::sample_kernel<true> : sample::sample_kernel<false>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           sizeof(sample::Shared)) != cudaSuccess)
    return DDT_ERR_CUDA;
  return launch_early(kernel, dim3(static_cast<unsigned>(rows * ranks)), dim3(sample::kThreads),
                      sizeof(sample::Shared), static_cast<cudaStream_t>(stream),
                      static_cast<unsigned>(ranks), a);
}
