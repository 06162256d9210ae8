// Causal attention of every request's new tokens over its pages of the K/V cache.
//
// Row i of request r (new token i, one query head) sees the keys j <= len_r - n_r + i:
//   o_i = sum_j 2^(s_ij - m_i) v_j / sum_j 2^(s_ij - m_i),   s_ij = q_i . k_j * scale * log2 e
// with the running maximum m and sum l of a one-pass softmax: a new maximum m' rescales what
// was summed by 2^(m - m').  A row that sees no key gives 0.
//
// Work unit: one KV head and two tiles of 128 query rows, row = (token, query head of the
// group), token-major, so that the whole group shares every K / V tile of 128 keys.  A group
// that does not divide 128 leaves the last 128 mod group rows of each tile unused.  Units are
// distributed by paged_sched.cuh.  Warp roles (12 warps):
//   warp 0      producer: Q tiles and, page by page, K and V tiles by TMA (128-byte swizzle,
//               two stages each; the lanes issue a tile's page boxes side by side, the next
//               tile's page ids are read one tile ahead).  Pages past the request's last one
//               are read from beyond the pool, where the tensor map fills zeros.
//   warps 1, 3  MMA issuers of query tile 0 and 1: S = Q K^T into TMEM, O += P V with P read
//               from TMEM.  They take turns, so the two softmax warpgroups stay half a period
//               apart.
//   warp 2      zeroes the V rows of a request's last page that lie past its length: they may
//               hold anything, and 0 * NaN would reach every row of the tile (K needs no care:
//               its scores are replaced by the mask).
//   warps 4-11  softmax, one query row per thread: the S row in one TMEM read, masked maximum,
//               P = exp2 back to TMEM as bf16 in two halves.  P is rounded to bf16 because the
//               matrix instruction takes it so; the row sum l is of the unrounded values (adding
//               the rounded ones instead makes a lone heavy key exact but costs 4.7%: four chunks
//               of 2048 tokens, 7k keys each on average, 457 against 437 us).  O is rescaled in
//               TMEM only when the maximum grew by more than 2^8.
// TMEM columns: S0/P0 [0,128) O0 [128,256) S1/P1 [256,384) O1 [384,512).
// Every wait is bounded; a timeout sets *status and unwinds the CTA.
//
// Measured, four chunks of up to 2048 tokens over 3k to 9.5k keys, 32 query heads over 8
// (452 GFLOP): 380 us or 1190 TFLOP/s, 0.72 of the measured bf16 burst; 448 us in a loop of
// seconds, where the power limit lowers the clock.  The tensor pipe is active in 65% of the
// cycles; the bound is one query tile's chain per key tile (TMEM read, maximum, exponentials,
// TMEM write, P V, the next S), which two query tiles do not quite hide.  Two threads per row
// (16 softmax warps, half a row each) made it slower (420 us).
#include <cuda.h>
#include <cuda_bf16.h>

#include "common.cuh"
#include "paged_sched.cuh"
#include "tc.cuh"

namespace ddt {
namespace paged_attn {

constexpr int kBlockM = 128;
constexpr int kBlockN = 128;
constexpr int kStages = 2;
constexpr int kThreads = 384;
// Register split (setmaxnreg): 384 threads are launched with 168 registers each; warpgroup 0
// goes down to 64, the softmax warpgroups up to 216: 128 * 64 + 256 * 216 <= 384 * 168.
constexpr int kRegsLaunch = 168;
constexpr int kRegsControl = 64;
constexpr int kRegsSoftmax = 216;
static_assert(128 * kRegsControl + 256 * kRegsSoftmax <= kThreads * kRegsLaunch,
              "register split exceeds the launch's registers");
constexpr int kUnitRows = 2 * kBlockM;
constexpr uint32_t kTmemCols = 512;
constexpr float kRescaleLog2 = 8.0f;
constexpr uint32_t kHalfBytes = kBlockM * 64 * 2;  // one 64-dim half of a 128-row tile
constexpr uint32_t kTileBytes = 2 * kHalfBytes;    // 32 KB
constexpr uint32_t kSmemQ = 0;                     // Q0, Q1
constexpr uint32_t kSmemK = kSmemQ + 2 * kTileBytes;
constexpr uint32_t kSmemV = kSmemK + kStages * kTileBytes;
constexpr uint32_t kSmemFirst = kSmemV + kStages * kTileBytes;  // cost prefix of the requests
inline uint32_t smem_alloc(int64_t n_requests) {
  return kSmemFirst + static_cast<uint32_t>((n_requests + 1) * sizeof(long long)) + 1024;
}
static_assert(kSmemFirst + (DDT_MAX_PAGED_REQUESTS + 1) * 8 + 1024 + 1024 <= 232448,
              "shared memory");
constexpr uint32_t kIdescS = tc::idesc_bf16_f32(kBlockM, kBlockN, false, false);
constexpr uint32_t kIdescPV = tc::idesc_bf16_f32(kBlockM, kHeadDim, false, true);
// of every 16 pairs of exponentials, the ones computed by the FMA-pipe polynomial beside MUFU
constexpr uint32_t kPolyPairs = 0x1249u;

__device__ __forceinline__ uint32_t col_s(int q) { return q ? 256u : 0u; }
__device__ __forceinline__ uint32_t col_o(int q) { return q ? 384u : 128u; }

struct Bars {
  uint64_t q_full, q_empty, k_full[kStages], v_full[kStages], k_empty[kStages],
      v_empty[kStages], v_clean[kStages], s_full[2], p_half[2], p_full[2], o_ready[2], mma_done[2];
  uint32_t issued[2];
  uint32_t tmem_base;
  int abort;
};

__device__ __forceinline__ void raise_abort(Bars& b, int32_t* status) {
  *reinterpret_cast<volatile int*>(&b.abort) = 1;
  if (status) atomicOr(status, kStatusTimeout);
}

// A unit of at most one query tile gives both tiles the same rows: tile 0 takes the even key
// tiles of the item and tile 1 the odd ones, so that two chains of S, softmax and P V run side by
// side; the epilogue joins them.
__device__ __forceinline__ bool paired(const Item& it, int tile_tok) { return it.n_tok <= tile_tok; }

// whether the item's last tile holds rows past the request's length
__device__ __forceinline__ bool ragged(const Item& it) {
  return it.nt > 0 && it.len - (it.t0 + it.nt - 1) * kBlockN < kBlockN;
}

__global__ void __launch_bounds__(kThreads, 1)
paged_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Params p) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ Bars bars;
  __shared__ long long s_warp[kThreads / 32];
  __shared__ Piece piece;
  __shared__ Place places[kThreads / 32];
  __shared__ float2 s_ml[2][kBlockM];  // (m, l) of a paired unit's two halves
  const uint32_t raw = tc::smem_u32(smem_raw);
  unsigned char* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tile_tok = kBlockM / p.group;  // tokens per query tile
  long long* s_first = reinterpret_cast<long long*>(smem + kSmemFirst);

  if (tid == 0) {
    tc::mbar_init(&bars.q_full, 1);
    tc::mbar_init(&bars.q_empty, 2);  // one commit per MMA issuer
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(&bars.k_full[s], 1);
      tc::mbar_init(&bars.v_full[s], 1);
      tc::mbar_init(&bars.k_empty[s], 2);
      tc::mbar_init(&bars.v_empty[s], 3);  // and warp 2
      tc::mbar_init(&bars.v_clean[s], 1);
    }
    for (int q = 0; q < 2; ++q) {
      tc::mbar_init(&bars.s_full[q], 1);
      tc::mbar_init(&bars.p_half[q], 4);  // one arrive per softmax warp
      tc::mbar_init(&bars.p_full[q], 4);
      bars.issued[q] = 0;
      tc::mbar_init(&bars.o_ready[q], 1);
      tc::mbar_init(&bars.mma_done[q], 1);
    }
    bars.abort = 0;
    tc::fence_mbar_init();
  }
  // before the allocation: a kernel that is still running may have yet to take its TMEM
  if (!p.beside) after_stream();
  if (warp == 1) {
    tc::tmem_alloc(&bars.tmem_base, kTmemCols);
    tc::tmem_relinquish();
  }
  walk_begin<kBlockN>(p, 2 * tile_tok, gridDim.x, s_first, s_warp, piece, places, kThreads / 32);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = bars.tmem_base;
  // the merge kernel may be scheduled from here on (it waits for this grid's end)
  let_next_begin();
  volatile int* abort_flag = &bars.abort;
  const Item& it = places[warp].it;  // the warp's current item
  auto next = [&] { return walk_next<kBlockN>(p, 2 * tile_tok, s_first, piece, places[warp]); };

  unsigned char* sQ = smem + kSmemQ;
  unsigned char* sK = smem + kSmemK;
  unsigned char* sV = smem + kSmemV;

  if (warp < 4) {
    tc::reg_dealloc<kRegsControl>();
    if (warp == 0) {
      // ---------------------------- TMA producer -------------------------------------
      if (lane == 0) {
        tc::tma_prefetch_desc(&tm_q);
        tc::tma_prefetch_desc(&tm_k);
        tc::tma_prefetch_desc(&tm_v);
      }
      // lane l issues box l / 2 of a tile, its dims [64 (l & 1), 64 (l & 1) + 64)
      const int box_rows = p.page_shift < 7 ? 1 << p.page_shift : kBlockN;
      const int boxes = kBlockN / box_rows;
      const bool issues = lane < 2 * boxes;
      const int half = lane & 1, box_row = (lane >> 1) * box_rows;
      const uint32_t q_bytes = 2u * static_cast<uint32_t>(tile_tok * p.group) * 128u * 2u;
      int q_loads = 0, issued_k = 0, issued_v = 0, J = 0, n_item = 0;
      bool ok = true;
      auto load_q = [&]() {
        if (lane == 0) tc::mbar_expect_tx(&bars.q_full, q_bytes);
        __syncwarp();
        // a query tile past the last row reads zeros
        if (lane < 4)
          tc::tma_load_3d(sQ + (lane >> 1) * kTileBytes + half * kHalfBytes, &tm_q, &bars.q_full,
                          half * 64, it.h * p.group,
                          it.tok0 + (paired(it, tile_tok) ? 0 : (lane >> 1) * tile_tok));
        ++q_loads;
      };
      // page of this lane's box in key tile t, or n_pages (zeros) past the request's pages
      auto page_id = [&](int t) -> int {
        const long long key = static_cast<long long>(t) * kBlockN + box_row;
        return issues && key < it.len ? page_of(p, it.r, key) : static_cast<int>(p.n_pages);
      };
      while (ok && blockIdx.x < p.withhold_from && next()) {
        const int t0 = it.t0, nt = it.nt;
        if (nt == 0) continue;
        int pg_next = page_id(t0);
        if (n_item == 0) load_q();
        for (int j = 0; j < nt; ++j) {
          const int jg = J + j;
          const int st = jg % kStages;
          const uint32_t ph = ((jg / kStages) - 1) & 1;  // release phase of tile jg - kStages
          const int pg = pg_next;
          if (j + 1 < nt) pg_next = page_id(t0 + j + 1);
          const int row = static_cast<int>(
              (static_cast<long long>(t0 + j) * kBlockN + box_row) & ((1 << p.page_shift) - 1));
          if (jg >= kStages &&
              !(ok = tc::mbar_wait_warp(&bars.k_empty[st], ph, abort_flag, p.timeout_ns)))
            break;
          if (lane == 0) tc::mbar_expect_tx(&bars.k_full[st], kTileBytes);
          __syncwarp();
          if (issues)
            tma_load_4d(sK + st * kTileBytes + half * kHalfBytes + box_row * 128, &tm_k,
                        &bars.k_full[st], half * 64, row, it.h, pg);
          issued_k = jg + 1;
          if (jg >= kStages &&
              !(ok = tc::mbar_wait_warp(&bars.v_empty[st], ph, abort_flag, p.timeout_ns)))
            break;
          if (lane == 0) tc::mbar_expect_tx(&bars.v_full[st], kTileBytes);
          __syncwarp();
          if (issues)
            tma_load_4d(sV + st * kTileBytes + half * kHalfBytes + box_row * 128, &tm_v,
                        &bars.v_full[st], half * 64, row, it.h, pg);
          issued_v = jg + 1;
          if (j == 0 && n_item > 0) {
            // the item's Q replaces the previous item's once both its S MMAs are done; the
            // first K / V tile of the item is already on its way
            if (!(ok = tc::mbar_wait_warp(&bars.q_empty, (n_item - 1) & 1, abort_flag,
                                          p.timeout_ns)))
              break;
            load_q();
          }
        }
        J += nt;
        ++n_item;
      }
      if (!ok && lane == 0) raise_abort(bars, p.status);
      __syncwarp();
      if (*abort_flag) {
        // let the loads already in flight land before the CTA releases its shared memory
        if (q_loads > 0) tc::mbar_wait_drain(&bars.q_full, (q_loads - 1) & 1, kTimeoutNs);
        for (int j = issued_k > kStages ? issued_k - kStages : 0; j < issued_k; ++j)
          tc::mbar_wait_drain(&bars.k_full[j % kStages], (j / kStages) & 1, kTimeoutNs);
        for (int j = issued_v > kStages ? issued_v - kStages : 0; j < issued_v; ++j)
          tc::mbar_wait_drain(&bars.v_full[j % kStages], (j / kStages) & 1, kTimeoutNs);
      }
    } else if (warp == 2) {
      // ---------------------------- V rows past the length -----------------------------
      int J = 0;
      bool ok = true;
      while (ok && next()) {
        // every tile is waited for and released, so that this warp keeps step with the stages'
        // phases
        const int nt = it.nt;
        const bool tail = ragged(it);
        for (int j = 0; j < nt; ++j) {
          const int jg = J + j, st = jg % kStages;
          if (!(ok = tc::mbar_wait_warp(&bars.v_full[st], (jg / kStages) & 1, abort_flag,
                                        p.timeout_ns)))
            break;
          if (tail && j + 1 == nt) {
            const int row0 = it.len - (it.t0 + j) * kBlockN;
            unsigned char* vd = sV + st * kTileBytes;
            // whole rows of 128 bytes in either half, so the swizzle does not matter
            for (int b = row0 * 8 + lane; b < kBlockN * 8; b += 32) {
              *reinterpret_cast<uint4*>(vd + b * 16) = make_uint4(0, 0, 0, 0);
              *reinterpret_cast<uint4*>(vd + kHalfBytes + b * 16) = make_uint4(0, 0, 0, 0);
            }
            tc::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&bars.v_clean[st]);
          }
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&bars.v_empty[st]);
        }
        J += it.nt;
      }
      if (!ok && lane == 0) raise_abort(bars, p.status);
    } else {
      // ---------------------------- MMA issuers, one per query tile ------------------
      // The whole warp runs the loop and its waits; an elected lane issues.
      const int q = warp == 1 ? 0 : 1;
      // descriptor low words of the Q, K and V tiles; every MMA adds a constant to them
      constexpr uint32_t kDescHi = tc::desc_sw128_hi(1024);
      const uint32_t a_q = tc::desc_sw128_lo(tc::smem_u32(sQ), 16) + q * (kTileBytes >> 4);
      const uint32_t k_lo = tc::desc_sw128_lo(tc::smem_u32(sK), 16);
      const uint32_t v_lo = tc::desc_sw128_lo(tc::smem_u32(sV), kHalfBytes);
      const uint32_t d_s = tmem + col_s(q), d_o = tmem + col_o(q);
      volatile uint32_t* my_turns = &bars.issued[q];
      const volatile uint32_t* other_turns = &bars.issued[q ^ 1];
      auto issue_s = [&](int jg, uint32_t turn) {
        const uint32_t b = k_lo + (jg % kStages) * (kTileBytes >> 4);
        tc::mma_bf16_ss_w<0>(d_s, a_q, b, kDescHi, kIdescS);
#pragma unroll
        for (int kk = 1; kk < kHeadDim / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * kHalfBytes + (kk & 3) * 32) >> 4;
          tc::mma_bf16_ss_w<1>(d_s, a_q + off, b + off, kDescHi, kIdescS);
          if (kk == kHeadDim / 16 - 1) *my_turns = turn;
        }
        tc::mma_commit(&bars.s_full[q]);
      };
      auto issue_pv = [&](int jg, int j, int half) {
        const uint32_t b = v_lo + (jg % kStages) * (kTileBytes >> 4);
#pragma unroll
        for (int k4 = 0; k4 < kBlockN / 32; ++k4) {
          const int kk = half * (kBlockN / 32) + k4;
          tc::mma_bf16_ts_w(d_o, d_s + kk * 8, b + ((kk * 2048) >> 4), kDescHi, kIdescPV,
                            (j > 0 || kk > 0) ? 1u : 0u);
        }
        if (half) tc::mma_commit(&bars.o_ready[q]);
      };
      // plain (volatile) turn counters: they order only the issue of the two tiles' MMAs
      auto wait_turn = [&](uint32_t target) {
        uint64_t t0 = 0;
        for (uint32_t n = 0;; ++n) {
          if (__all_sync(DDT_FULL_MASK, *other_turns >= target)) return true;
          if ((n & 255u) == 255u) {
            const uint64_t now = global_timer_ns();
            if (t0 == 0) t0 = now;
            if (__any_sync(DDT_FULL_MASK, *abort_flag != 0 || now - t0 > p.timeout_ns))
              return false;
          }
        }
      };
      bool ok = true;
      uint32_t base = 0;
      int J = 0, Js = 0, n_item = 0;  // Js: tiles of this query tile
      uint32_t cleaned = 0;           // phases of v_clean, a bit per stage
      auto wait = [&](uint64_t* bar, int phase) {
        return tc::mbar_wait_warp(bar, phase & 1, abort_flag, p.timeout_ns);
      };
      auto kbar = [&](int jg) { return wait(&bars.k_full[jg % kStages], jg / kStages); };
      // V of the tile landed and, where the tile is ragged, was cleaned.  A stage is released
      // after this, so neither barrier can get two phases ahead of a waiter.
      auto vbar = [&](int jg, bool dirty) {
        const int st = jg % kStages;
        if (!wait(&bars.v_full[st], jg / kStages)) return false;
        if (!dirty) return true;
        const int phase = cleaned >> st;
        cleaned ^= 1u << st;
        return wait(&bars.v_clean[st], phase);
      };
      while (ok && next()) {
        const int nt = it.nt;
        if (nt == 0) continue;
        const bool tail = ragged(it);
        if (!(ok = wait(&bars.q_full, n_item))) break;
        if (paired(it, tile_tok)) {
          // the other query tile's key tiles are waited for and released too, so that this
          // warp keeps step with the stages' phases
          for (int j = 0; ok && j < nt; ++j) {
            const int jg = J + j, st = jg % kStages;
            if ((j & 1) != q) {
              if (j > 0) continue;  // released with the tile before it
              if (!(ok = kbar(jg) && vbar(jg, tail && nt == 1))) break;
              if (lane == 0) {
                tc::mbar_arrive(&bars.k_empty[st]);
                tc::mbar_arrive(&bars.v_empty[st]);
              }
              __syncwarp();
              continue;
            }
            if (!(ok = kbar(jg))) break;
            tc::tc_fence_after();
            if (tc::elect_one()) {
              issue_s(jg, base);
              tc::mma_commit(&bars.k_empty[st]);
            }
            __syncwarp();
            const bool other = j + 1 < nt;
            if (other) {
              if (!(ok = kbar(jg + 1))) break;
              if (lane == 0) tc::mbar_arrive(&bars.k_empty[(jg + 1) % kStages]);
              __syncwarp();
            }
            if (!(ok = vbar(jg, tail && !other))) break;
            if (!(ok = wait(&bars.p_half[q], Js))) break;
            tc::tc_fence_after();
            if (tc::elect_one()) issue_pv(jg, j - q, 0);
            __syncwarp();
            if (!(ok = wait(&bars.p_full[q], Js))) break;
            tc::tc_fence_after();
            if (tc::elect_one()) {
              issue_pv(jg, j - q, 1);
              tc::mma_commit(&bars.v_empty[st]);
            }
            __syncwarp();
            ++Js;
            if (other) {
              if (!(ok = vbar(jg + 1, tail && j + 2 == nt))) break;
              if (lane == 0) tc::mbar_arrive(&bars.v_empty[(jg + 1) % kStages]);
              __syncwarp();
            }
          }
          if (ok && lane == 0) *my_turns = base + nt + 1;
          __syncwarp();
        } else {
          if (!(ok = kbar(J))) break;
          if (!(ok = wait_turn(q == 0 ? base : base + 1))) break;
          tc::tc_fence_after();
          if (tc::elect_one()) {
            issue_s(J, base + 1);
            tc::mma_commit(&bars.k_empty[J % kStages]);
          }
          __syncwarp();
          for (int j = 0; j < nt; ++j) {
            const int jg = J + j;
            const bool more = j + 1 < nt;
            // K / V of the tile landed long before P_q(j): waited first, while the softmax runs
            if (!(ok = vbar(jg, tail && !more))) break;
            if (more && !(ok = kbar(jg + 1))) break;
            if (!(ok = wait(&bars.p_half[q], Js))) break;
            if (!(ok = wait_turn(q == 0 ? base + j + 1 : base + j + 2))) break;
            tc::tc_fence_after();
            if (tc::elect_one()) issue_pv(jg, j, 0);
            __syncwarp();
            if (!(ok = wait(&bars.p_full[q], Js))) break;
            tc::tc_fence_after();
            if (tc::elect_one()) {
              issue_pv(jg, j, 1);
              tc::mma_commit(&bars.v_empty[jg % kStages]);
              if (more) {
                issue_s(jg + 1, base + j + 2);  // reuses S_q / P_q: runs after the P V above
                tc::mma_commit(&bars.k_empty[(jg + 1) % kStages]);
              } else {
                *my_turns = base + j + 2;
              }
            }
            __syncwarp();
            ++Js;
          }
        }
        // the item's S MMAs are all issued: Q may be replaced once they are done
        if (ok && tc::elect_one()) tc::mma_commit(&bars.q_empty);
        __syncwarp();
        base += nt + 1;
        J += nt;
        ++n_item;
      }
      if (!ok && lane == 0) raise_abort(bars, p.status);
      // every MMA and commit of this warp is done before the CTA's barriers and TMEM go
      if (n_item > 0 || !ok) {
        if (tc::elect_one()) tc::mma_commit(&bars.mma_done[q]);
        __syncwarp();
        tc::mbar_wait_drain(&bars.mma_done[q], 0, kTimeoutNs);
      }
    }
  } else {
    tc::reg_alloc<kRegsSoftmax>();
    // ---------------------------- softmax warpgroups -------------------------------
    const int q = (warp - 4) >> 2;  // query tile of this warpgroup (warps 4-7 / 8-11)
    const int wq = warp & 3;        // TMEM lane quarter a warp may access: warp id % 4
    const int r = wq * 32 + lane;
    const uint32_t tl = tmem + (static_cast<uint32_t>(wq * 32) << 16);
    const uint32_t tS = tl + col_s(q);
    const uint32_t tO = tl + col_o(q);
    const float sl2 = p.scale_log2;
    const tc::Exp2Poly exp2_poly;
    const int row_tok = r / p.group;               // token of this row within its tile
    const int row_head = r - row_tok * p.group;
    const bool row_used = row_tok < tile_tok;
    bool ok = true;
    int J = 0;  // S tiles of this query tile so far
    // (after a failed wait the walk goes on without work, so that both warpgroups meet at every
    // barrier of the paired units)
    while (next()) {
      const bool pair = paired(it, tile_tok);
      const int tok = (pair ? 0 : q * tile_tok) + row_tok;  // token of this row within the unit
      const bool valid = row_used && tok < it.n_tok;
      // keys this row sees: [0, lim); rows that are not stored see them all
      const int lim = valid ? it.past + tok + 1 : 0x7fffffff;
      const int t0 = it.t0 + (pair ? q : 0), step = pair ? 2 : 1;
      const int nt = pair ? (it.nt + 1 - q) >> 1 : it.nt;  // this query tile's key tiles
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; ok && j < nt; ++j) {
        const int jg = J + j;
        if (!tc::mbar_wait_warp(&bars.s_full[q], jg & 1, abort_flag, p.timeout_ns)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        const int left = lim - (t0 + j * step) * kBlockN;  // columns [0, left) are visible
        const bool masked = __any_sync(DDT_FULL_MASK, left < kBlockN);
        // the whole S row (128 fp32) comes out of TMEM in one round trip
        uint32_t sv[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tc::tmem_ld32(tS + c * 32, sv[c]);
        tc::tmem_wait_ld();
        if (masked) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c * 32 + e >= left) sv[c][e] = __float_as_uint(-INFINITY);
        }
        // row max of the raw scores: three-input maxima in 8 independent chains
        float mx8[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) mx8[k] = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            mx8[(e >> 1) & 7] = tc::fmax3(mx8[(e >> 1) & 7], __uint_as_float(sv[c][e]),
                                          __uint_as_float(sv[c][e + 1]));
        const float mx = tc::fmax3(tc::fmax3(mx8[0], mx8[1], mx8[2]),
                                   tc::fmax3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7]));
        bool rescale = false;
        float alpha = 1.f;
        if (mx > -INFINITY) {
          const float ms = mx * sl2;
          if (m_used == -INFINITY) {
            m_used = ms;
            l = 0.f;  // what the polynomial lanes made of masked keys
          } else if (ms > m_used + kRescaleLog2) {
            alpha = tc::ex2_approx(m_used - ms);
            m_used = ms;
            rescale = true;
          }
        }
        if (__any_sync(DDT_FULL_MASK, rescale)) {
          // O_q is stable once the previous P V MMA of this item completed
          if (j > 0 &&
              !tc::mbar_wait_warp(&bars.o_ready[q], (jg - 1) & 1, abort_flag, p.timeout_ns)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            tc::tmem_ld32(tO + c * 32, o);
            tc::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tc::tmem_st32(tO + c * 32, o);
          }
          l *= alpha;
        }
        const float nm = (m_used == -INFINITY) ? 0.f : -m_used;
        // P = exp2(S * scale - m), packed bf16 into columns [0, 64) of S_q (masked keys hold
        // -inf and give 0, or 2^-126 on the polynomial lanes)
        const uint64_t sl2x2 = tc::f2_pack(sl2, sl2), nmx2 = tc::f2_pack(nm, nm);
        uint64_t ls2[4] = {0ull, 0ull, 0ull, 0ull};
        // keys [0, 64) first: their P columns are stored and signalled (p_half) while the
        // second half is computed, so the first four P V MMAs overlap it
        uint32_t pk[2][32];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const uint64_t x = tc::f2_fma(tc::f2_pack(__uint_as_float(sv[hf * 2 + c][e]),
                                                        __uint_as_float(sv[hf * 2 + c][e + 1])),
                                            sl2x2, nmx2);
              float a, b;
              if ((kPolyPairs >> (e >> 1)) & 1u) {
                exp2_poly(x, a, b);
              } else {
                float y0, y1;
                tc::f2_unpack(x, y0, y1);
                a = tc::ex2_approx(y0);
                b = tc::ex2_approx(y1);
              }
              ls2[(e >> 1) & 3] = tc::f2_add(ls2[(e >> 1) & 3], tc::f2_pack(a, b));
              pk[hf][c * 16 + e / 2] = tc::pack_bf16x2(a, b);
            }
          }
          if (hf == 0) tc::tmem_st32(tS, pk[0]);
        }
        tc::tmem_wait_st();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&bars.p_half[q]);
        tc::tmem_st32(tS + 32, pk[1]);
        float l0, l1, l2, l3;
        tc::f2_unpack(tc::f2_add(ls2[0], ls2[1]), l0, l1);
        tc::f2_unpack(tc::f2_add(ls2[2], ls2[3]), l2, l3);
        l += (l0 + l1) + (l2 + l3);
        tc::tmem_wait_st();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&bars.p_full[q]);
      }
      if (ok && nt > 0 &&
          !tc::mbar_wait_warp(&bars.o_ready[q], (J + nt - 1) & 1, abort_flag, p.timeout_ns))
        ok = false;
      if (!ok && lane == 0) raise_abort(bars, p.status);
      // warp-uniform: O holds this query tile's sums of the item
      bool have = ok && nt > 0;
      if (have) tc::tc_fence_after();
      float m2 = -INFINITY, l2 = 0.f;  // of the other half of a paired unit
      if (pair) {
        const bool seen = have && m_used > -INFINITY;
        s_ml[q][r] = make_float2(seen ? m_used : -INFINITY, seen ? l : 0.f);
        tc::tc_fence_before();
        ok = tc::named_sync_and(1, 2 * kBlockM, ok);
        tc::tc_fence_after();
        const float2 o = s_ml[q ^ 1][r];
        m2 = o.x;
        l2 = o.y;
        have = ok && it.nt > 0;
      }
      if (!(m_used > -INFINITY) || !ok) l = 0.f;
      // O = w O_q + w2 O_(q ^ 1), l alike; weights of 0 where a half saw no key
      const float M = fmaxf(m_used, m2);
      const float w = pair ? (m_used == -INFINITY ? 0.f : tc::ex2_approx(m_used - M)) : 1.f;
      const float w2 = m2 == -INFINITY ? 0.f : tc::ex2_approx(m2 - M);
      l = l * w + l2 * w2;
      const bool seen = have && M > -INFINITY;  // per row: some key was visible
      // columns of O that this thread stores: all 128, or its warpgroup's half of a paired unit
      const int c0 = pair ? q * 2 : 0, c1 = pair ? q * 2 + 2 : 4;
      const int ur = (pair ? 0 : q * kBlockM) + r;
      float* op = p.o_part + (it.slot >= 0 ? static_cast<long long>(it.slot) * kUnitRows * kHeadDim : 0ll) +
                  ur * 4;
      __nv_bfloat16* orow = p.out + (it.tok0 + tok) * p.o_token_stride +
                            (it.h * p.group + row_head) * p.o_head_stride;
      const float inv = seen && l > 0.f ? 1.f / l : 0.f;
      for (int c = c0; c < c1; ++c) {
        uint32_t o[32];
        if (have) {
          tc::tmem_ld32(tO + c * 32, o);
          tc::tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (pair && have) {  // a half without key tiles has nothing in TMEM: select, not multiply
          uint32_t o2[32];
          tc::tmem_ld32(tl + col_o(q ^ 1) + c * 32, o2);
          tc::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float x = w > 0.f ? __uint_as_float(o[e]) * w : 0.f;
            const float y = w2 > 0.f ? __uint_as_float(o2[e]) * w2 : 0.f;
            o[e] = __float_as_uint(x + y);
          }
        }
        if (!valid) continue;
        if (it.slot >= 0) {
          // a part: unnormalised O in fp32, [dim / 4][row][4] so that a warp's rows
          // (consecutive) store 512 contiguous bytes at a time
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<uint4*>(op + ((c * 32 + e) / 4) * kUnitRows * 4) =
                make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint4 v;
            v.x = tc::pack_bf16x2(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
            v.y = tc::pack_bf16x2(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
            v.z = tc::pack_bf16x2(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
            v.w = tc::pack_bf16x2(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
            *reinterpret_cast<uint4*>(orow + c * 32 + e) = v;
          }
        }
      }
      if (it.slot >= 0 && valid && (!pair || q == 0))
        *reinterpret_cast<float2*>(p.ml_part +
                                   (static_cast<long long>(it.slot) * kUnitRows + ur) * 2) =
            make_float2(seen ? M : -INFINITY, seen ? l : 0.f);
      // the O columns are read: the next item's first P V MMA may overwrite them (it waits
      // for p_half of that item, which comes after this point, from either warpgroup)
      tc::tc_fence_before();
      if (pair) tc::named_sync(1, 2 * kBlockM);
      J += nt;
    }
  }
  // what the merge kernel needs of a unit that starts in this CTA and ends in another: its
  // first row, tokens, head and last CTA (at most one such unit: the CTA's last item)
  if (tid == kThreads - 1)
    p.parts[blockIdx.x] = (it.slot >= 0 && (it.slot & 1) )
                              ? make_int4(it.tok0, it.n_tok, it.h, cta_of(piece, it.x_last))
                              : make_int4(0, 0, 0, -1);
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
  // a short kernel launched before this one is over before this one is: what follows in the
  // stream waits for this one only
  after_stream();
}

// ---- merge of the parts ----------------------------------------------------------------
// o = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i over the parts of a unit in CTA order, M the
// largest m_i.  One warp per (unit, 32 rows, 16 dims): lane = row, so that every load is 512
// contiguous bytes.
constexpr int kMergeDims = 16;
constexpr int kMergeWarps = 8;

__global__ void __launch_bounds__(kMergeWarps * 32) paged_merge_kernel(const Params p) {
  const int c0 = blockIdx.x;
  // launched while the attention kernel still runs: its writes are there after this wait
  after_stream();
  const int4 part = p.parts[c0];
  if (part.w < 0) return;
  const int w = blockIdx.y * kMergeWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rows32 = w / (kHeadDim / kMergeDims), d0 = (w % (kHeadDim / kMergeDims)) * kMergeDims;
  const int ur = rows32 * 32 + lane;
  const int tile_tok = kBlockM / p.group, r = ur % kBlockM;
  const int row_tok = r / p.group, tok = (ur / kBlockM) * tile_tok + row_tok;
  if (row_tok >= tile_tok || tok >= part.y) return;
  float M = -INFINITY, L = 0.f, acc[kMergeDims];
#pragma unroll
  for (int e = 0; e < kMergeDims; ++e) acc[e] = 0.f;
  for (int c = c0; c <= part.w; ++c) {
    const long long slot = 2 * c + (c == c0 ? 1 : 0);
    const float2 ml = *reinterpret_cast<const float2*>(p.ml_part + (slot * kUnitRows + ur) * 2);
    if (ml.x == -INFINITY) continue;
    const float* op = p.o_part + slot * kUnitRows * kHeadDim + ur * 4;
    float4 o[kMergeDims / 4];
#pragma unroll
    for (int e = 0; e < kMergeDims / 4; ++e)
      o[e] = *reinterpret_cast<const float4*>(op + (d0 / 4 + e) * kUnitRows * 4);
    const float Mn = fmaxf(M, ml.x), a = M == -INFINITY ? 0.f : exp2f(M - Mn),
                b = exp2f(ml.x - Mn);
    M = Mn;
    L = L * a + ml.y * b;
#pragma unroll
    for (int e = 0; e < kMergeDims / 4; ++e) {
      acc[4 * e] = acc[4 * e] * a + o[e].x * b;
      acc[4 * e + 1] = acc[4 * e + 1] * a + o[e].y * b;
      acc[4 * e + 2] = acc[4 * e + 2] * a + o[e].z * b;
      acc[4 * e + 3] = acc[4 * e + 3] * a + o[e].w * b;
    }
  }
  const float inv = L > 0.f ? 1.f / L : 0.f;
  __nv_bfloat16* orow = p.out + (part.x + tok) * p.o_token_stride +
                        (part.z * p.group + (r - row_tok * p.group)) * p.o_head_stride + d0;
#pragma unroll
  for (int e = 0; e < kMergeDims; e += 8) {
    uint4 v;
    v.x = tc::pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
    v.y = tc::pack_bf16x2(acc[e + 2] * inv, acc[e + 3] * inv);
    v.z = tc::pack_bf16x2(acc[e + 4] * inv, acc[e + 5] * inv);
    v.w = tc::pack_bf16x2(acc[e + 6] * inv, acc[e + 7] * inv);
    *reinterpret_cast<uint4*>(orow + e) = v;
  }
}

// Workspace: partial O, partial (m, l), and the record of the unit that starts in each CTA.
constexpr size_t kPartO = size_t(2) * kSms * kUnitRows * kHeadDim * sizeof(float);
constexpr size_t kPartMl = size_t(2) * kSms * kUnitRows * 2 * sizeof(float);
constexpr size_t kWorkspace = kPartO + kPartMl + kSms * sizeof(int4);
// The long kernel's area comes after the short one's, whose counters have to stay zero.
inline size_t workspace_bytes() { return (short_workspace_bytes() + 255) / 256 * 256 + kWorkspace; }

// A call of either entry point: timeout_ns bounds every wait, CTAs from withhold_from on issue no
// load (the check of the waits).
int call(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k_pages,
         const void* v_pages, int64_t n_pages, int64_t page_size, int64_t page_stride,
         int64_t head_stride, int64_t row_stride, const int32_t* block_table, int64_t table_stride,
         int64_t max_pages, const int32_t* cu_new, const int32_t* kv_lens, int64_t n_requests,
         int64_t n_tokens, int64_t max_new, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
         float scale, void* out, int64_t o_token_stride, int64_t o_head_stride, void* workspace,
         size_t ws_bytes, int32_t* status, void* stream, uint64_t timeout_ns, unsigned withhold_from) {
  if (n_requests <= 0 || n_tokens < 0 || max_new < 0 || q_heads <= 0 || kv_heads <= 0 ||
      q_heads % kv_heads || n_pages <= 0 || max_pages <= 0 || table_stride < max_pages ||
      !(scale >= 0.f))
    return DDT_ERR_INVALID;
  if (head_dim != kHeadDim || q_heads / kv_heads > kMaxGroup) return DDT_ERR_CAPACITY;
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return DDT_ERR_CAPACITY;
  if (n_requests > DDT_MAX_PAGED_REQUESTS || n_tokens > 0x7fffffff || n_pages >= 0x7fffffff ||
      max_pages > (int64_t(1) << 30) / page_size || kv_heads > 65535)
    return DDT_ERR_CAPACITY;
  if (n_tokens == 0 || max_new == 0) return DDT_OK;
  if (!q || !k_pages || !v_pages || !block_table || !cu_new || !kv_lens || !out)
    return DDT_ERR_INVALID;
  if (!aligned(q, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(out, 16) ||
      q_token_stride % 8 || q_head_stride % 8 || page_stride % 8 || head_stride % 8 ||
      row_stride % 8 || o_token_stride % 8 || o_head_stride % 8)
    return DDT_ERR_ALIGN;
  if (!workspace || ws_bytes < workspace_bytes()) return DDT_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return DDT_ERR_ALIGN;
  const int64_t group = q_heads / kv_heads;
  Params p;
  p.block_table = block_table;
  p.table_stride = table_stride;
  p.max_keys = max_pages * page_size;
  p.n_pages = n_pages;
  p.page_shift = __builtin_ctzll(static_cast<unsigned long long>(page_size));
  p.cu_new = cu_new;
  p.kv_lens = kv_lens;
  p.n_requests = static_cast<int>(n_requests);
  p.n_tokens = static_cast<int>(n_tokens);
  p.max_new = static_cast<int>(max_new < n_tokens ? max_new : n_tokens);
  p.group = static_cast<int>(group);
  p.kv_heads = static_cast<int>(kv_heads);
  // a scale of 0 (all keys alike) is taken as one too small to tell them apart: a masked score
  // of -inf keeps its sign
  p.scale_log2 = fmaxf(scale * 1.4426950408889634f, 1e-30f);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.o_token_stride = o_token_stride;
  p.o_head_stride = o_head_stride;
  p.status = status;
  p.timeout_ns = timeout_ns;
  p.withhold_from = withhold_from;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Which kernel takes which request: few rows go to the short one, the rest to this one, and
  // a batch of long chunks with single tokens between them to both.  The host knows only the
  // longest request, so the others are judged by their mean: where they are not 16 rows or
  // fewer, or too few to fill the SMs, this kernel takes all.  (Recorded graph, a 1000-token
  // chunk among 32 decoded tokens of 1k to 7k keys: 118 us on this kernel alone, 105 on both;
  // among 3, where it takes all, 49.)  Groups of more than 16 heads have no room in that kernel's
  // tile of 16 rows.
  const bool few = p.max_new * group <= kShortRows;
  const int64_t others = n_requests - 1, one_tile = 16 / group;
  const bool both = !few && one_tile > 0 && others * kv_heads >= kSms &&
                    n_tokens - p.max_new <= one_tile * others;
  CUtensorMap tm_q, tm_k, tm_v;
  const cuuint64_t kdims[4] = {kHeadDim, static_cast<cuuint64_t>(page_size),
                               static_cast<cuuint64_t>(kv_heads), static_cast<cuuint64_t>(n_pages)};
  const int64_t kstrides[3] = {row_stride, head_stride, page_stride};
  auto kv_maps = [&](int64_t tile) {
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(page_size < tile ? page_size : tile), 1, 1};
    const int e = make_map(&tm_k, k_pages, 4, kdims, kstrides, box);
    return e ? e : make_map(&tm_v, v_pages, 4, kdims, kstrides, box);
  };
  int rc;
  p.from_new = 1;
  p.to_new = p.max_new;
  if (few || both) {
    if (both) p.to_new = static_cast<int>(one_tile);
    if ((rc = kv_maps(64)) ||
        (rc = launch_short(p, q, q_token_stride, q_head_stride, q_heads, tm_k, tm_v, workspace, st)) ||
        few)
      return rc;
    p.from_new = p.to_new + 1;
    p.to_new = p.max_new;
  }
  if ((rc = kv_maps(kBlockN))) return rc;
  const cuuint64_t dims[3] = {kHeadDim, static_cast<cuuint64_t>(q_heads),
                              static_cast<cuuint64_t>(n_tokens)};
  const int64_t strides[2] = {q_head_stride, q_token_stride};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(group),
                             static_cast<cuuint32_t>(kBlockM / group)};
  if ((rc = make_map(&tm_q, q, 3, dims, strides, box))) return rc;
  p.o_part = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                      (short_workspace_bytes() + 255) / 256 * 256);
  p.ml_part = p.o_part + kPartO / sizeof(float);
  p.parts = reinterpret_cast<int4*>(p.ml_part + kPartMl / sizeof(float));
  p.arrived = nullptr;
  const uint32_t smem = smem_alloc(n_requests);
  if (cudaFuncSetAttribute(paged_attn_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(smem)) != cudaSuccess)
    return DDT_ERR_CUDA;
  // beside the few-rows kernel's last CTAs: the two share no output
  p.beside = both;
  rc = launch_early(paged_attn_kernel, dim3(kSms), dim3(kThreads), smem, st, 0, tm_q, tm_k, tm_v, p);
  if (rc) return rc;
  // the merge's CTAs take the SMs as the attention's leave them and wait there for its end,
  // instead of being launched after it
  return launch_early(paged_merge_kernel,
                      dim3(kSms, kUnitRows / 32 * (kHeadDim / kMergeDims) / kMergeWarps),
                      dim3(kMergeWarps * 32), 0, st, 0, p);
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
  // how units are cut depends on device-side lengths: one size for all calls
  return paged_attn::workspace_bytes();
}

extern "C" int ddt_paged_attn(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                              const void* k_pages, const void* v_pages, int64_t n_pages,
                              int64_t page_size, int64_t page_stride, int64_t head_stride,
                              int64_t row_stride, const int32_t* block_table, int64_t table_stride,
                              int64_t max_pages, const int32_t* cu_new, const int32_t* kv_lens,
                              int64_t n_requests, int64_t n_tokens, int64_t max_new,
                              int64_t q_heads, int64_t kv_heads, int64_t head_dim, float scale,
                              void* out, int64_t o_token_stride, int64_t o_head_stride,
                              void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  return paged_attn::call(q, q_token_stride, q_head_stride, k_pages, v_pages, n_pages, page_size,
                          page_stride, head_stride, row_stride, block_table, table_stride,
                          max_pages, cu_new, kv_lens, n_requests, n_tokens, max_new, q_heads,
                          kv_heads, head_dim, scale, out, o_token_stride, o_head_stride, workspace,
                          workspace_bytes, status, stream, paged_attn::kTimeoutNs, ~0u);
}

extern "C" int ddt_paged_attn_wait_check(const void* q, int64_t q_token_stride,
                                         int64_t q_head_stride, const void* k_pages,
                                         const void* v_pages, int64_t n_pages, int64_t page_size,
                                         int64_t page_stride, int64_t head_stride,
                                         int64_t row_stride, const int32_t* block_table,
                                         int64_t table_stride, int64_t max_pages,
                                         const int32_t* cu_new, const int32_t* kv_lens,
                                         int64_t n_requests, int64_t n_tokens, int64_t max_new,
                                         int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                         float scale, void* out, int64_t o_token_stride,
                                         int64_t o_head_stride, void* workspace,
                                         size_t workspace_bytes, int32_t* status, int64_t first_cta,
                                         uint64_t timeout_ns, void* stream) {
  if (!status || first_cta < 0 || timeout_ns < 100000ull || timeout_ns > paged_attn::kTimeoutNs)
    return DDT_ERR_INVALID;
  const unsigned first = first_cta < 0x7fffffff ? static_cast<unsigned>(first_cta) : 0x7fffffffu;
  return paged_attn::call(q, q_token_stride, q_head_stride, k_pages, v_pages, n_pages, page_size,
                          page_stride, head_stride, row_stride, block_table, table_stride,
                          max_pages, cu_new, kv_lens, n_requests, n_tokens, max_new, q_heads,
                          kv_heads, head_dim, scale, out, o_token_stride, o_head_stride, workspace,
                          workspace_bytes, status, stream, timeout_ns, first);
}
