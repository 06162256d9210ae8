// Paged attention of requests with few new tokens: single tokens, drafted blocks.
//
// With at most 32 query rows per (request, KV head) a tile of 128 rows for tcgen05.mma would be
// mostly padding, and its chain (S, TMEM read, softmax, TMEM write, P V) per key tile is longer
// than the tile takes to arrive: one decoded token for each of 64 requests ran at 3.2 TB/s on
// it.  Here the bound is the read of K and V, and the products are small enough for
// mma.sync.m16n8k16 (16 query rows a time) beside it.
//
// One unit: a request and KV head, its rows = (token, head of the group) in one or two tiles
// of 16.  A CTA is one producer warp and four consumer warps, two CTAs per SM.  The producer
// streams K and V tiles of 64 keys (16 KB each, page by page, by TMA) through a ring of as many
// 16 KB buffers as fit.  For each tile the consumers
//   1. take 16 keys each: S = Q K^T, masked, and the row maxima over their keys
//   2. exchange the maxima: each row's reference m moves only when the maximum grew by more
//      than 2^8 (rescaling O and l), the same decision in every warp
//   3. write P = 2^(S - m) as bf16 to shared memory; l adds the unrounded values
//   4. take 32 dims each: O += P V over all 64 keys
// The matrix instruction takes P as bf16, good to 2^-9.  Units of at most 8 rows (a token of a group
// of 8 heads) leave half of its 16 rows free: there the other rows hold what the rounding left,
// P - bf16(P), and the two products are added at the end, so P is good to 2^-17 and the error is
// that of the output's own rounding (relative 2-norm 1.7e-3; 2.2e-3 with P rounded).  Units of more
// rows would need instructions of their own for that: 64 x 8 tokens of 9000 keys, 32 rows, 434 to
// 530 us; there P stays rounded.
// so K and V leave shared memory once, whether there are 16 rows or 32.  V rows past the request's
// length may hold anything; their fragments are replaced by zeros in registers.
// Measured, one token for each of 64 requests of 1k to 32k keys, 32 query heads over 8 (2.38 GB
// of K and V): 362 us, 6.57 TB/s, the measured copy rate, with 1.003 times the bytes read from
// HBM.  One request of 1000 keys takes 9.1 to 9.7 us, two thirds of it dependent reads (lengths, page
// ids, K, the parts).
// Units are cut over the CTAs as in paged_sched.cuh; the CTA that brings a cut unit's last part
// merges all of them, in the order of the CTAs, so the result does not depend on which it is, and
// sets the unit's counter back to zero.
#include "paged_sched.cuh"

namespace ddt {
namespace paged_attn {

namespace {

constexpr int kKeys = 64;          // keys per tile
constexpr int kConsumers = 4;      // warps
constexpr int kShortThreads = (kConsumers + 1) * 32;
constexpr uint32_t kBufHalf = kKeys * 128;       // 64 dims of 64 keys
constexpr uint32_t kBufBytes = 2 * kBufHalf;     // 16 KB: one K or V tile
constexpr int kMaxBufs = 8;
constexpr int kMaxParts = 32;      // CTAs per unit on average, for 16 rows (merging is latency)
constexpr float kRescale = 8.0f;
constexpr size_t kShortPartO = size_t(2) * kShortCtas * kShortRows * kHeadDim * sizeof(float);
constexpr size_t kShortPartMl = size_t(2) * kShortCtas * kShortRows * 2 * sizeof(float);

struct ShortBars {
  uint64_t q_full[2], q_empty[2], full[kMaxBufs], empty[kMaxBufs];
  int abort;
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// d += a b: 16 x 8 x 16, bf16 in, fp32 sums
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// address of 16-byte chunk `c` (0..15) of row `row` in a tile of two halves of 64 dims, 128-byte
// swizzled rows (as TMA writes them)
__device__ __forceinline__ uint32_t chunk_at(uint32_t base, uint32_t half_bytes, int row, int c) {
  return base + (c >> 3) * half_bytes + row * 128 + (((c & 7) ^ (row & 7)) << 4);
}

// The parts of a unit, CTAs c0 to c1 in order, merged by the four warps:
//   o = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i,  M the largest m_i.
// A warp takes kR rows at a time, 32 / kR lanes and so kR loads of 16 bytes per row and part;
// 16 / kR parts are in flight.  The reads are latency, not bytes: rows one after the other took
// 23 us for 32 rows of 18 parts.
template <int kR>
__device__ __forceinline__ void merge_rows(const Params& p, const Item& it, int c0, int c1,
                                           int rows) {
  constexpr int kLanes = 32 / kR, kParts = 16 / kR;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / kLanes, at = lane % kLanes;
  for (int r = warp * kR + sub; r < rows; r += kConsumers * kR) {
    float M = -INFINITY, sum = 0.f;
    float4 acc[kR];
#pragma unroll
    for (int f = 0; f < kR; ++f) acc[f] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int b = c0; b <= c1; b += kParts) {
      float2 ml[kParts];
      float4 v[kParts][kR];
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        const int c = min(b + i, c1);
        const long long row = static_cast<long long>(2 * c + (c == c0)) * kShortRows + r;
        ml[i] = __ldcg(reinterpret_cast<const float2*>(p.ml_part + row * 2));
        if (b + i > c1) ml[i] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int f = 0; f < kR; ++f)
          v[i][f] = __ldcg(reinterpret_cast<const float4*>(p.o_part + row * kHeadDim) +
                           f * kLanes + at);
      }
      float mn = M;
#pragma unroll
      for (int i = 0; i < kParts; ++i) mn = fmaxf(mn, ml[i].x);
      if (mn == -INFINITY) continue;
      const float x = M == -INFINITY ? 0.f : tc::ex2_approx(M - mn);
      M = mn;
      sum *= x;
#pragma unroll
      for (int f = 0; f < kR; ++f)
        acc[f] = make_float4(acc[f].x * x, acc[f].y * x, acc[f].z * x, acc[f].w * x);
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        const float y = ml[i].x == -INFINITY ? 0.f : tc::ex2_approx(ml[i].x - M);
        sum += ml[i].y * y;
#pragma unroll
        for (int f = 0; f < kR; ++f) {
          acc[f].x += v[i][f].x * y;
          acc[f].y += v[i][f].y * y;
          acc[f].z += v[i][f].z * y;
          acc[f].w += v[i][f].w * y;
        }
      }
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    const int tok = r / p.group;
    __nv_bfloat16* dst = p.out + (it.tok0 + tok) * p.o_token_stride +
                         (it.h * p.group + r - tok * p.group) * p.o_head_stride;
#pragma unroll
    for (int f = 0; f < kR; ++f)
      *reinterpret_cast<uint2*>(dst + (f * kLanes + at) * 4) =
          make_uint2(tc::pack_bf16x2(acc[f].x * inv, acc[f].y * inv),
                     tc::pack_bf16x2(acc[f].z * inv, acc[f].w * inv));
  }
}

// kM: tiles of 16 query rows.  Shared memory: Q (two buffers), P, the ring, maxima / sums, the
// cost prefix.
constexpr int unit_rows(int m, bool two_parts) { return two_parts ? 8 : 16 * m; }
template <int kM>
struct Layout {
  static constexpr int kRows = 16 * kM;
  static constexpr uint32_t kQHalf = kRows * 128;
  static constexpr uint32_t kQ = 0;                         // 2 x [2 halves][kRows][64]
  static constexpr uint32_t kP = kQ + 2 * 2 * kQHalf;       // [kRows][64 keys]
  static constexpr uint32_t kRing = (kP + kRows * 128 + 1023) / 1024 * 1024;
  static uint32_t bytes(int bufs, int64_t n_requests) {
    return kRing + bufs * kBufBytes + kRows * 4 * sizeof(float) +
           static_cast<uint32_t>((n_requests + 1) * sizeof(long long)) + 1024;
  }
};

// kTwoParts: the unit has at most 8 rows; rows 8 to 15 of its tile hold the second part of P.
template <int kM, bool kTwoParts>
__global__ void __launch_bounds__(kShortThreads, 2)
paged_decode_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Params p,
                    const int bufs) {
  using L = Layout<kM>;
  static_assert(!kTwoParts || kM == 1, "one tile");
  constexpr int kH = kTwoParts ? 1 : 2;  // rows of a lane in a tile: g, and 8 on
  constexpr int kUnit = unit_rows(kM, kTwoParts);
  extern __shared__ unsigned char smem_raw[];
  __shared__ ShortBars bars;
  __shared__ long long s_warp[kConsumers + 1];
  __shared__ Piece piece;
  __shared__ Place places[kConsumers + 1];
  __shared__ int s_last_arrival, s_c0, s_c1;
  const uint32_t raw = tc::smem_u32(smem_raw);
  unsigned char* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const uint32_t base = tc::smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float* s_max = reinterpret_cast<float*>(smem + L::kRing + bufs * kBufBytes);  // [row][warp]
  long long* s_first = reinterpret_cast<long long*>(s_max + L::kRows * 4);
  const int unit_tok = kUnit / p.group;  // tokens a unit has room for

  if (tid == kConsumers * 32) {
    tc::tma_prefetch_desc(&tm_q);
    tc::tma_prefetch_desc(&tm_k);
    tc::tma_prefetch_desc(&tm_v);
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bars.q_full[i], 1);
      tc::mbar_init(&bars.q_empty[i], kConsumers);
    }
    for (int i = 0; i < bufs; ++i) {
      tc::mbar_init(&bars.full[i], 1);
      tc::mbar_init(&bars.empty[i], kConsumers);
    }
    bars.abort = 0;
    tc::fence_mbar_init();
  }
  after_stream();
  walk_begin<kKeys>(p, unit_tok, static_cast<long long>(kMaxParts / kM) * p.kv_heads * p.n_requests,
                    s_first, s_warp, piece, places, kConsumers + 1);
  __syncthreads();
  // the other kernel of a mixed batch may take the SMs that this one leaves; it reads what was
  // written before this one, which is over by now
  let_next_begin();
  volatile int* abort_flag = &bars.abort;
  const Item& it = places[warp].it;
  auto next = [&] { return walk_next<kKeys>(p, unit_tok, s_first, piece, places[warp]); };

  if (warp == kConsumers) {
    // ---------------------------- TMA producer ---------------------------------------
    const int box_rows = p.page_shift < 6 ? 1 << p.page_shift : kKeys;
    const bool issues = lane < 2 * (kKeys / box_rows);
    const int half = lane & 1, box_row = (lane >> 1) * box_rows;
    const uint32_t box_at = half * kBufHalf + box_row * 128;
    const uint32_t q_bytes = 2u * static_cast<uint32_t>(unit_tok * p.group) * 128u;
    int n_item = 0, buf = 0;
    uint32_t used = 0;  // buffers filled so far, and the ring's turn
    uint32_t turn = 0;
    bool ok = true;
    // page of this lane's box in key tile t, or n_pages (zeros) past the request's pages
    auto page_id = [&](int t) -> int {
      const int key = t * kKeys + box_row;
      return issues && key < it.len ? page_of(p, it.r, key) : static_cast<int>(p.n_pages);
    };
    auto fill = [&](const CUtensorMap* map, int row, int pg) {
      if (used >= static_cast<uint32_t>(bufs) &&
          !(ok = tc::mbar_wait_warp(&bars.empty[buf], (turn - 1) & 1, abort_flag, p.timeout_ns)))
        return;
      if (lane == 0) tc::mbar_expect_tx(&bars.full[buf], kBufBytes);
      __syncwarp();
      if (issues)
        tma_load_4d(smem + L::kRing + buf * kBufBytes + box_at, map, &bars.full[buf], half * 64, row,
                    it.h, pg);
      ++used;
      if (++buf == bufs) {
        buf = 0;
        ++turn;
      }
    };
    while (ok && blockIdx.x < p.withhold_from && next()) {
      const int t0 = it.t0, nt = it.nt;
      if (nt == 0) continue;
      const int qb = n_item & 1;
      if (n_item >= 2 && !(ok = tc::mbar_wait_warp(&bars.q_empty[qb], ((n_item >> 1) - 1) & 1,
                                                   abort_flag, p.timeout_ns)))
        break;
      if (lane == 0) tc::mbar_expect_tx(&bars.q_full[qb], q_bytes);
      __syncwarp();
      if (lane < 2)
        tc::tma_load_3d(smem + L::kQ + qb * 2 * L::kQHalf + lane * L::kQHalf, &tm_q,
                        &bars.q_full[qb], lane * 64, it.h * p.group, it.tok0);
      ++n_item;
      int pg_next = page_id(t0);
      for (int j = 0; ok && j < nt; ++j) {
        const int pg = pg_next;
        if (j + 1 < nt) pg_next = page_id(t0 + j + 1);
        const int row = ((t0 + j) * kKeys + box_row) & ((1 << p.page_shift) - 1);
        fill(&tm_k, row, pg);
        if (ok) fill(&tm_v, row, pg);
      }
    }
    if (!ok) {
      if (lane == 0) {
        *abort_flag = 1;
        if (p.status) atomicOr(p.status, kStatusTimeout);
      }
    }
    __syncwarp();
    if (*abort_flag) {
      // let the loads already in flight land before the CTA releases its shared memory
      for (int i = n_item > 2 ? n_item - 2 : 0; i < n_item; ++i)
        tc::mbar_wait_drain(&bars.q_full[i & 1], (i >> 1) & 1, kTimeoutNs);
      for (uint32_t i = used > static_cast<uint32_t>(bufs) ? used - bufs : 0; i < used; ++i)
        tc::mbar_wait_drain(&bars.full[i % bufs], (i / bufs) & 1, kTimeoutNs);
    }
    return;
  }

  // ---------------------------- consumers ----------------------------------------------
  const int g = lane >> 2, t4 = lane & 3;          // accumulator row and column pair
  const int mi = lane >> 3, lr = lane & 7;         // ldmatrix: matrix and row of this lane
  const uint32_t sP = base + L::kP;
  const float sl2 = p.scale_log2;
  int n_item = 0, buf = 0;
  uint32_t turn = 0;
  bool ok = true;
  auto release = [&] {
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&bars.empty[buf]);
    if (++buf == bufs) {
      buf = 0;
      ++turn;
    }
  };
  // (after a failed wait the walk goes on without work: this CTA's parts are still counted, so
  // that the counters of cut units end at zero)
  while (next()) {
    const bool works = ok;  // the same in all four warps
    const int t0 = it.t0, nt = it.nt, len = it.len;
    const int rows = it.n_tok * p.group;
    float o[kM][4][4], m[kM][kH], l[kM][kH];
    int lim[kM][kH];  // keys that the row sees
#pragma unroll
    for (int a = 0; a < kM; ++a) {
#pragma unroll
      for (int h = 0; h < kH; ++h) {
        const int r = a * 16 + h * 8 + g;
        lim[a][h] = r < rows ? it.past + r / p.group + 1 : 0x7fffffff;
        m[a][h] = -INFINITY;
        l[a][h] = 0.f;
      }
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[a][n][e] = 0.f;
    }
    const uint32_t sQ = base + L::kQ + (n_item & 1) * 2 * L::kQHalf;
    if (works && nt > 0)
      ok = tc::mbar_wait_warp(&bars.q_full[n_item & 1], (n_item >> 1) & 1, abort_flag, p.timeout_ns);
    for (int j = 0; works && j < nt; ++j) {
      const int key0 = (t0 + j) * kKeys;
      // 1. S of this warp's 16 keys
      ok = ok && tc::mbar_wait_warp(&bars.full[buf], turn & 1, abort_flag, p.timeout_ns);
      float s[kM][2][4];
#pragma unroll
      for (int a = 0; a < kM; ++a)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[a][n][e] = 0.f;
      const uint32_t sK = base + L::kRing + buf * kBufBytes;
#pragma unroll
      for (int k = 0; k < kHeadDim / 16; ++k) {
        uint32_t b[4];
        ldsm4(b, chunk_at(sK, kBufHalf, warp * 16 + (mi >> 1) * 8 + lr, k * 2 + (mi & 1)));
#pragma unroll
        for (int a = 0; a < kM; ++a) {
          uint32_t q[4];
          ldsm4(q, chunk_at(sQ, L::kQHalf, a * 16 + (mi & 1) * 8 + lr, k * 2 + (mi >> 1)));
          mma16816(s[a][0], q, b[0], b[1]);
          mma16816(s[a][1], q, b[2], b[3]);
        }
      }
      release();
      if (j + 1 == nt) {  // the item's Q is read
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&bars.q_empty[n_item & 1]);
      }
      const int kw = key0 + warp * 16 + t4 * 2;  // key of s[.][0][0]
#pragma unroll
      for (int a = 0; a < kM; ++a)
#pragma unroll
        for (int h = 0; h < kH; ++h) {
          const int left = lim[a][h] - kw;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (n * 8 + e >= left) s[a][n][h * 2 + e] = -INFINITY;
          float mx = fmaxf(fmaxf(s[a][0][h * 2], s[a][0][h * 2 + 1]),
                           fmaxf(s[a][1][h * 2], s[a][1][h * 2 + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(DDT_FULL_MASK, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(DDT_FULL_MASK, mx, 2));
          if (t4 == 0) s_max[(a * 16 + h * 8 + g) * 4 + warp] = mx;
        }
      // 2. the tile's row maxima
      if (!tc::named_sync_and(1, kConsumers * 32, ok)) {
        ok = false;
        break;
      }
#pragma unroll
      for (int a = 0; a < kM; ++a)
#pragma unroll
        for (int h = 0; h < kH; ++h) {
          const float4 w = *reinterpret_cast<const float4*>(&s_max[(a * 16 + h * 8 + g) * 4]);
          const float ms = fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)) * sl2;
          if (ms > m[a][h] + kRescale || (m[a][h] == -INFINITY && ms > -INFINITY)) {
            const float alpha = tc::ex2_approx(m[a][h] - ms);
            m[a][h] = ms;
            l[a][h] *= alpha;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              o[a][n][h * 2] *= alpha;
              o[a][n][h * 2 + 1] *= alpha;
              if (kTwoParts) {
                o[a][n][2] *= alpha;
                o[a][n][3] *= alpha;
              }
            }
          }
          // 3. P
          const float nm = m[a][h] == -INFINITY ? 0.f : -m[a][h];
          const int r = a * 16 + h * 8 + g;
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float x = tc::ex2_approx(fmaf(s[a][n][h * 2], sl2, nm));
            const float y = tc::ex2_approx(fmaf(s[a][n][h * 2 + 1], sl2, nm));
            l[a][h] += x + y;
            const uint32_t at = sP + r * 128 + (((warp * 2 + n) ^ (r & 7)) << 4) + t4 * 4;
            const uint32_t xy = tc::pack_bf16x2(x, y);
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(xy) : "memory");
            if (kTwoParts) {
              const uint32_t rest = tc::pack_bf16x2(x - __uint_as_float(xy << 16),
                                                    y - __uint_as_float(xy & 0xffff0000u));
              asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + 8 * 128), "r"(rest) : "memory");
            }
          }
        }
      tc::named_sync(1, kConsumers * 32);
      // 4. O += P V, this warp's 32 dims
      ok = tc::mbar_wait_warp(&bars.full[buf], turn & 1, abort_flag, p.timeout_ns);
      const uint32_t sV = base + L::kRing + buf * kBufBytes;
      const bool tail = len - key0 < kKeys;
#pragma unroll
      for (int k = 0; k < kKeys / 16; ++k) {
        uint32_t v[2][4];
#pragma unroll
        for (int n2 = 0; n2 < 2; ++n2) {
          ldsm4_t(v[n2], chunk_at(sV, kBufHalf, k * 16 + (mi & 1) * 8 + lr,
                                  warp * 4 + n2 * 2 + (mi >> 1)));
          if (tail) {
            // registers 0, 2: keys k * 16 + 2 t4 + {0, 1}; 1, 3: eight keys on
            const int left = len - key0 - k * 16 - t4 * 2;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int n_ok = left - (e & 1) * 8;
              v[n2][e] = n_ok <= 0 ? 0u : n_ok == 1 ? v[n2][e] & 0xffffu : v[n2][e];
            }
          }
        }
#pragma unroll
        for (int a = 0; a < kM; ++a) {
          uint32_t pa[4];
          const int r = a * 16 + (mi & 1) * 8 + lr;
          ldsm4(pa, sP + r * 128 + (((k * 2 + (mi >> 1)) ^ (r & 7)) << 4));
#pragma unroll
          for (int n = 0; n < 4; ++n)
            mma16816(o[a][n], pa, v[n >> 1][(n & 1) * 2], v[n >> 1][(n & 1) * 2 + 1]);
        }
      }
      release();
    }
    if (kTwoParts) {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        o[0][n][0] += o[0][n][2];
        o[0][n][1] += o[0][n][3];
      }
    }
    // the rows' sums over the warps' keys
#pragma unroll
    for (int a = 0; a < kM; ++a)
#pragma unroll
      for (int h = 0; h < kH; ++h) {
        l[a][h] += __shfl_xor_sync(DDT_FULL_MASK, l[a][h], 1);
        l[a][h] += __shfl_xor_sync(DDT_FULL_MASK, l[a][h], 2);
        if (ok && t4 == 0) s_max[(a * 16 + h * 8 + g) * 4 + warp] = l[a][h];
      }
    ok = tc::named_sync_and(1, kConsumers * 32, ok);
    if (!ok && lane == 0) *abort_flag = 1;  // the producer's waits end too
    if (nt > 0) ++n_item;
#pragma unroll
    for (int a = 0; a < kM; ++a)
#pragma unroll
      for (int h = 0; h < kH; ++h) {
        const int r = a * 16 + h * 8 + g;
        const float4 w = *reinterpret_cast<const float4*>(&s_max[r * 4]);
        const float sum = (w.x + w.y) + (w.z + w.w);
        if (r >= rows) continue;
        if (!ok) {  // a part without weight
          if (it.slot >= 0 && warp == 0 && t4 == 0)
            *reinterpret_cast<float2*>(p.ml_part +
                                       (static_cast<long long>(it.slot) * kShortRows + r) * 2) =
                make_float2(-INFINITY, 0.f);
        } else if (it.slot < 0) {
          const float inv = sum > 0.f ? 1.f / sum : 0.f;
          const int tok = r / p.group;
          __nv_bfloat16* dst = p.out + (it.tok0 + tok) * p.o_token_stride +
                               (it.h * p.group + r - tok * p.group) * p.o_head_stride + warp * 32 +
                               t4 * 2;
#pragma unroll
          for (int n = 0; n < 4; ++n)
            *reinterpret_cast<uint32_t*>(dst + n * 8) =
                tc::pack_bf16x2(o[a][n][h * 2] * inv, o[a][n][h * 2 + 1] * inv);
        } else {
          const long long row = static_cast<long long>(it.slot) * kShortRows + r;
          float* dst = p.o_part + row * kHeadDim + warp * 32 + t4 * 2;
#pragma unroll
          for (int n = 0; n < 4; ++n)
            *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[a][n][h * 2], o[a][n][h * 2 + 1]);
          if (warp == 0 && t4 == 0)
            *reinterpret_cast<float2*>(p.ml_part + row * 2) = make_float2(m[a][h], sum);
        }
      }
    if (it.slot >= 0) {
      // the CTA that brings the last part merges all of them
      __threadfence();
      tc::named_sync(1, kConsumers * 32);
      if (tid == 0) {
        s_c0 = cta_of(piece, it.x_first);
        s_c1 = cta_of(piece, it.x_last);
        s_last_arrival = atomicAdd(&p.arrived[s_c0], 1u) == static_cast<unsigned int>(s_c1 - s_c0);
        if (s_last_arrival) p.arrived[s_c0] = 0u;
      }
      tc::named_sync(1, kConsumers * 32);
      if (s_last_arrival) {
        __threadfence();
        if (rows <= kConsumers) merge_rows<1>(p, it, s_c0, s_c1, rows);
        else if (rows <= 2 * kConsumers) merge_rows<2>(p, it, s_c0, s_c1, rows);
        else merge_rows<4>(p, it, s_c0, s_c1, rows);
      }
    }
    tc::named_sync(1, kConsumers * 32);  // s_max and s_last_arrival are read
  }
  if (!ok && lane == 0) {
    *abort_flag = 1;
    if (p.status) atomicOr(p.status, kStatusTimeout);
  }
}

template <int kM, bool kTwoParts>
int launch_m(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
             const Params& p, cudaStream_t st) {
  using L = Layout<kM>;
  // two CTAs per SM: 227 KB less 1 KB each for the system and the static part
  constexpr uint32_t kRoom = (227 * 1024) / 2 - 1024 - 1536;
  int bufs = kMaxBufs;
  while (bufs > 2 && L::bytes(bufs, p.n_requests) > kRoom) --bufs;
  const uint32_t smem = L::bytes(bufs, p.n_requests);
  if (cudaFuncSetAttribute(paged_decode_kernel<kM, kTwoParts>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(smem)) != cudaSuccess)
    return DDT_ERR_CUDA;
  return launch_early(paged_decode_kernel<kM, kTwoParts>, dim3(kShortCtas), dim3(kShortThreads), smem,
                      st, 0, tm_q, tm_k, tm_v, p, bufs);
}

}  // namespace

size_t short_workspace_bytes() {
  return kShortPartO + kShortPartMl + kShortCtas * sizeof(unsigned int);
}

int launch_short(Params& p, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                 int64_t q_heads, const CUtensorMap& tm_k, const CUtensorMap& tm_v, void* workspace,
                 cudaStream_t st) {
  p.o_part = static_cast<float*>(workspace);
  p.ml_part = p.o_part + kShortPartO / sizeof(float);
  p.arrived = reinterpret_cast<unsigned int*>(p.ml_part + kShortPartMl / sizeof(float));
  p.parts = nullptr;
  const int rows = p.to_new * p.group, m = rows <= 16 ? 1 : 2;
  const bool two_parts = rows <= unit_rows(1, true);
  CUtensorMap tm_q;
  const cuuint64_t dims[3] = {kHeadDim, static_cast<cuuint64_t>(q_heads),
                              static_cast<cuuint64_t>(p.n_tokens)};
  const int64_t strides[2] = {q_head_stride, q_token_stride};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(p.group),
                             static_cast<cuuint32_t>(unit_rows(m, two_parts) / p.group)};
  const int rc = make_map(&tm_q, q, 3, dims, strides, box);
  if (rc) return rc;
  return two_parts ? launch_m<1, true>(tm_q, tm_k, tm_v, p, st)
         : m == 1  ? launch_m<1, false>(tm_q, tm_k, tm_v, p, st)
                   : launch_m<2, false>(tm_q, tm_k, tm_v, p, st);
}

}  // namespace paged_attn
}  // namespace ddt
