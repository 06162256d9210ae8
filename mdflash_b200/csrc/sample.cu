// Sampling with temperature, top-k, top-p and min-p from given uniforms, one token per row.
//
// Weights are whole numbers, w_i = floor(exp((x_i - max) / T) * 2^40), so every sum of them is
// exact and the token does not depend on the order in which a launch adds.  The kept tokens are
// a prefix of the order (logit descending, index ascending), described by its last token: kept
// are the logits above `edge`, and the equal ones up to index `last`.
//
// A row is shared by a cluster of 1 to 8 CTAs; every warp owns a contiguous range of indices and
// reads it with 16-byte loads in every pass (the first from HBM, the others from L2):
//   1. maximum and minimum
//   2. for top-k (by counts), then for top-p (by weights, of what top-k keeps): a histogram of
//      the row over 2048 equal intervals of the logits, added over the cluster through
//      distributed shared memory; the interval that holds the boundary; a pass that lists its
//      tokens (a few hundred of 152k where the row looks like a model's); and every listed token
//      compared with every other, which gives each its exact count and weight before it.  Lists of
//      more than 1024 tokens (long runs of equal logits) are searched by the bits of the key.
//   3. the weight of the kept tokens; the warps of the CTA that holds the target share the
//      range of the warp that holds it, until that is one load per lane
// CTAs exchange values through distributed shared memory, with one cluster barrier each time.
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
constexpr int kList = 1024;
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
// Dev. 34, 1990), unless b's significand is all ones; the first step brings a y that close.
// Those b, and ones whose reciprocal is not a normal number, take the plain division.
struct Divisor {
  float b, y;
  bool plain;
  __device__ explicit Divisor(float d) : b(d), y(1.f / d) {
    plain = (__float_as_uint(d) & 0x7fffffu) == 0x7fffffu || d > 1e30f;
  }
  __device__ __forceinline__ float operator()(float a) const {
    if (plain) return a / b;
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
  float list_x[kList];                                      // this CTA's part of a list
  int list_i[kList];
  float all_x[kList];  // the cluster's list
  int all_i[kList];
  unsigned long long all_w[kList];
  unsigned long long warp_sum[2][kWarps];
  unsigned long long sum;  // kept weight of the CTA
  uint32_t top_key, low_key;
  int n_list, ties, tie_index;
  // found by one thread of the CTA for all of its threads
  int bin;
  unsigned long long before_c, before_w, bin_c;
  float edge;
  int last, range0, range1;
};

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

template <bool kBF16>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const Args a) {
  constexpr int kVec = kBF16 ? 8 : 4;  // elements per 16-byte load
  constexpr int kStep = 32 * kVec;
  constexpr int kBatch = 4;
  extern __shared__ unsigned char smem_raw[];
  Shared& s = *reinterpret_cast<Shared*>(smem_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int V = a.vocab;
  const char* x = static_cast<const char*>(a.logits) + row * a.row_stride * (kBF16 ? 2 : 4);
  auto peer = [&](int r) { return cluster.map_shared_rank(&s, r); };

  // this warp's range of indices
  const int per_warp =
      ((V + ranks * kWarps - 1) / (ranks * kWarps) + kStep - 1) / kStep * kStep;
  const int seg0 = min(static_cast<long long>(rank * kWarps + warp) * per_warp,
                       static_cast<long long>(V));
  const int seg1 = min(seg0 + per_warp, V);

  bool inf_top = false;  // +inf takes all of the weight: the row is then read as 0 and -inf
  // kVec elements of a 16-byte load
  auto spread = [&](const uint4& r, float (&v)[kVec]) {
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
  auto vec_at = [&](int i) {
    return __ldg(reinterpret_cast<const uint4*>(x + static_cast<long long>(i) * (kBF16 ? 2 : 4)));
  };
  // the kVec elements from index i on; NaN at and past `end`: like every NaN they are below
  // all, equal to none and of weight 0
  auto load = [&](int i, int end, float (&v)[kVec]) {
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
  // f(first index, kVec values) over [begin, end) of this warp: kBatch loads are in flight
  // before the first is used
  auto vectors = [&](int begin, int end, auto f) {
    int i = begin + lane * kVec;
    if (a.vectors)
      for (; i - lane * kVec + kBatch * kStep <= end; i += kBatch * kStep) {
        uint4 r[kBatch];
#pragma unroll
        for (int h = 0; h < kBatch; ++h) r[h] = vec_at(i + h * kStep);
#pragma unroll
        for (int h = 0; h < kBatch; ++h) {
          float v[kVec];
          spread(r[h], v);
          f(i + h * kStep, v);
        }
      }
    for (; i < end; i += kStep) {
      float v[kVec];
      load(i, end, v);
      f(i, v);
    }
  };
  // f(index, value) over this warp's range
  auto each = [&](auto f) {
    vectors(seg0, seg1, [&](int i, float (&v)[kVec]) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) f(i + e, v[e]);
    });
  };

  // ---- 1. maximum and minimum ------------------------------------------------------------
  float mx = -INFINITY, mn = INFINITY;
  each([&](int, float v) {
    mx = fmaxf(mx, v);
    mn = fminf(mn, v);
  });
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

  const float temp_in = a.temperature[row];
  const bool greedy = !(temp_in >= 1e-5f);
  const float temp = greedy ? 1.f : temp_in;
  const float p_in = a.top_p && !greedy ? a.top_p[row] : 1.f;
  const int k_in = a.top_k ? a.top_k[row] : 0;
  const int k = greedy || p_in <= 0.f ? 1 : (k_in > 0 && k_in < V ? k_in : V);
  const double p = k > 1 ? static_cast<double>(p_in) : 1.0;
  const float min_p = a.min_p && !greedy ? fminf(a.min_p[row], 1.f) : 0.f;
  const Divisor by_temp(temp);
  // exp of the scaled distance to the maximum, by CUDA's expf; -200 stands for all that is
  // far below a weight of 1 and for the NaN of -inf and NaN logits
  auto scaled = [&](float v) { return fmaxf(by_temp(v - top), -200.f); };
  auto weight = [&](float v) { return whole(expf(scaled(v))); };

  // ---- 2. what top-k and top-p keep -----------------------------------------------------------
  float edge = -INFINITY;
  int last = V;
  bool all_kept = true;  // of the tokens that have weight
  auto kept = [&](int i, float v) { return all_kept || v > edge || (v == edge && i <= last); };
  // interval of a logit: equal intervals from the maximum down to the minimum, or to where
  // weights end (the last interval takes the rest)
  const float span = fminf(top - key_f32(low_key), 28.f * temp);
  const float per_unit = span > 0.f ? (kBins - 1) / span : 0.f;
  auto bin_of = [&](float v) {
    return min(__float2int_rz(__fmul_rn(__fsub_rn(top, v), per_unit)), kBins - 1);
  };
  // Histogram of the kept tokens by `bin` (those with a bin >= 0), added over the cluster; then
  // the bin that holds the boundary: by weight the last one whose weight before it is below
  // `reach`, else the one that holds token number `want`.  s.bin, s.before_c, s.before_w, s.bin_c.
  double reach = 0.0;
  auto boundary = [&](bool by_weight, bool count, bool ascending, unsigned long long want,
                      unsigned long long above_c, unsigned long long above_w, bool set_reach,
                      auto bin) {
    for (int b = tid; b < kBins; b += kThreads) s.count[b] = s.lo[b] = s.hi[b] = 0;
    __syncthreads();
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
    if (tid == 0) s.bin = -1;
    cluster.sync();
    // thread t owns kOwn bins, in the order of the tokens
    unsigned long long c[kOwn] = {}, w[kOwn] = {}, c_sum = 0, w_sum = 0;
    const int b0 = (ascending ? tid : kThreads - 1 - tid) * kOwn;
    for (int r = 0; r < ranks; ++r) {
      const Shared* o = peer(r);
      if (count) {
        const uint4 oc = *reinterpret_cast<const uint4*>(&o->count[b0]);
        c[0] += oc.x, c[1] += oc.y, c[2] += oc.z, c[3] += oc.w;
      }
      if (by_weight) {
        const uint4 ol = *reinterpret_cast<const uint4*>(&o->lo[b0]),
                    oh = *reinterpret_cast<const uint4*>(&o->hi[b0]);
        w[0] += (static_cast<unsigned long long>(oh.x) << 32) + ol.x;
        w[1] += (static_cast<unsigned long long>(oh.y) << 32) + ol.y;
        w[2] += (static_cast<unsigned long long>(oh.z) << 32) + ol.z;
        w[3] += (static_cast<unsigned long long>(oh.w) << 32) + ol.w;
      }
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
  // Moves (edge, last) to token number `want` of the kept ones, or to the last of them whose
  // weight before it is below p times the weight of all.
  auto cut = [&](bool by_weight, unsigned long long want) {
    if (tid == 0) s.n_list = 0;
    boundary(by_weight, !by_weight, true, want, 0, 0, by_weight, bin_of);
    const int bin = s.bin;
    if (bin < 0) {  // fewer tokens than `want` (NaN is none): all stay, in every CTA alike
      cluster.sync();  // the histograms are read
      return;
    }
    const unsigned long long above_c = s.before_c, above_w = s.before_w;
    each([&](int i, float v) {
      if (v == v && kept(i, v) && bin_of(v) == bin) {
        const int at = atomicAdd(&s.n_list, 1);
        if (at < kList) {
          s.list_x[at] = v;
          s.list_i[at] = i;
        }
      }
    });
    cluster.sync();
    int first = lane < ranks ? peer(lane)->n_list : 0;
    const int n = __reduce_add_sync(DDT_FULL_MASK, first);
    if (n <= kList) {
      // every CTA takes the whole list and finds the boundary by itself
      for (int r = 0, at = 0; r < ranks; ++r) {
        const Shared* o = peer(r);
        const int m = __shfl_sync(DDT_FULL_MASK, first, r);
        for (int j = tid; j < m; j += kThreads) {
          const float v = o->list_x[j];
          s.all_x[at + j] = v;
          s.all_i[at + j] = o->list_i[j];
          s.all_w[at + j] = by_weight ? weight(v) : 0ull;
        }
        at += m;
      }
      __syncthreads();
      int kept_here = 0, order[kList / kThreads] = {};
#pragma unroll
      for (int h = 0; h < kList / kThreads; ++h) {
        const int j = tid + h * kThreads;
        order[h] = -1;
        if (j < n) {
          const float v = s.all_x[j];
          const int i = s.all_i[j];
          unsigned long long c = 0, w = 0;
          for (int o = 0; o < n; ++o) {
            const float vo = s.all_x[o];
            if (vo > v || (vo == v && s.all_i[o] < i)) {
              ++c;
              w += s.all_w[o];
            }
          }
          if (by_weight ? static_cast<double>(above_w + w) < reach : above_c + c < want) {
            ++kept_here;
            order[h] = static_cast<int>(c);
          }
        }
      }
      kept_here = __reduce_add_sync(DDT_FULL_MASK, kept_here);
      if (lane == 0) s.warp_sum[0][warp] = kept_here;
      __syncthreads();
      int m = 0;
      for (int w = 0; w < kWarps; ++w) m += static_cast<int>(s.warp_sum[0][w]);
#pragma unroll
      for (int h = 0; h < kList / kThreads; ++h)
        if (order[h] == m - 1) {
          s.edge = s.all_x[tid + h * kThreads];
          s.last = s.all_i[tid + h * kThreads];
        }
      cluster.sync();  // the lists are read; (edge, last) is there
      edge = s.edge;
      last = s.last;
      all_kept = false;
      return;
    }
    // a long list: three steps over the bits of the key, from the top
    cluster.sync();
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
    before += __reduce_add_sync(DDT_FULL_MASK, lane < rank ? peer(lane)->ties : 0);
    long long left = static_cast<long long>(ties) - before;  // of this warp's
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
  if (k == 1) {
    // the first of the largest
    int first = V;
    each([&](int i, float v) { first = v == top ? min(first, i) : first; });
    first = __reduce_min_sync(DDT_FULL_MASK, first);
    if (lane == 0) atomicMin(&s.tie_index, first);
    cluster.sync();
    edge = top;
    all_kept = false;
    last = __reduce_min_sync(DDT_FULL_MASK, lane < ranks ? peer(lane)->tie_index : V);
  } else {
    if (k < V) cut(false, k);
    if (p < 1.0) cut(true, 0);
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
    vectors(begin, end, [&](int i, float (&v)[kVec]) {
      uint32_t hi = 0, lo = 0;
      bool any = all_kept;
      if (!any) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) any |= v[e] >= edge;
      }
      if (any) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          uint32_t h, l;
          kept_limbs(i + e, v[e], h, l);
          hi += h;
          lo += l;
        }
      }
      sum += (static_cast<unsigned long long>(hi) << 20) + lo;
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(DDT_FULL_MASK, sum, o);
    return sum;
  };
  // weight before this warp's part, of the parts of the CTA's warps in order
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
  unsigned long long mine = weigh(seg0, seg1), all;
  unsigned long long before = before_warp(mine, all);
  if (tid == 0) s.sum = all;
  cluster.sync();
  unsigned long long total = lane < ranks ? peer(lane)->sum : 0ull;
  unsigned long long earlier = lane < rank ? total : 0ull;
#pragma unroll
  for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
    total += __shfl_xor_sync(DDT_FULL_MASK, total, o);
    earlier += __shfl_xor_sync(DDT_FULL_MASK, earlier, o);
  }
  total = __shfl_sync(DDT_FULL_MASK, total, 0);
  earlier = __shfl_sync(DDT_FULL_MASK, earlier, 0);
  long long t = static_cast<long long>(floor(static_cast<double>(a.u[row]) * static_cast<double>(total)));
  t = max(min(t, static_cast<long long>(total) - 1), 0ll);
  unsigned long long target = static_cast<unsigned long long>(t);
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
        a.tokens[row] = pick;
        if (a.logprobs)
          a.logprobs[row] = static_cast<float>(static_cast<double>(scaled(value)) -
                                               (log(static_cast<double>(total)) - kLogUnit));
      }
    }
  }
  cluster.sync();  // no CTA leaves while another may read its shared memory
}

}  // namespace sample
}  // namespace ddt

using namespace ddt;

extern "C" int ddt_sample(const void* logits, int dtype, int64_t rows, int64_t vocab,
                          int64_t row_stride, const float* u, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p,
                          int64_t* tokens, float* logprobs, void* stream) {
  if (dtype != DDT_F32 && dtype != DDT_BF16) return DDT_ERR_DTYPE;
  if (rows < 0 || vocab <= 0 || row_stride < vocab) return DDT_ERR_INVALID;
  if (vocab >= (int64_t(1) << 22) || rows > 0x7fffffff / sample::kMaxCluster) return DDT_ERR_CAPACITY;
  if (rows == 0) return DDT_OK;
  if (!logits || !u || !temperature || !tokens) return DDT_ERR_INVALID;
  const int64_t size = dtype == DDT_F32 ? 4 : 2;
  if (!aligned(logits, size)) return DDT_ERR_ALIGN;
  sample::Args a{logits, static_cast<int>(vocab), row_stride, u, temperature, top_k, top_p, min_p,
                 tokens, logprobs, aligned(logits, 16) && (row_stride * size) % 16 == 0};
  // as many CTAs per row as keep the rows in one wave (two CTAs per SM), or the rows in flight
  // in half of L2 (they are read again), and no more than leave each thread one load
  int ranks = 1;
  while (ranks < sample::kMaxCluster && vocab > ranks * sample::kThreads * (16 / size) &&
         (rows * ranks * 2 <= 2 * 148 || 2 * 148 / ranks * vocab * size > (int64_t(64) << 20)))
    ranks *= 2;
  auto kernel = dtype == DDT_BF16 ? sample::sample_kernel<true> : sample::sample_kernel<false>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           sizeof(sample::Shared)) != cudaSuccess)
    return DDT_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * ranks));
  cfg.blockDim = dim3(sample::kThreads);
  cfg.dynamicSmemBytes = sizeof(sample::Shared);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) {
    cudaGetLastError();
    return DDT_ERR_CUDA;
  }
  return DDT_OK;
}
