// Log probabilities of given tokens straight from the rows that enter the output head: logits = x . w^T (capped), their running
// maximum, sum of exponentials and sum of d exp(d) (row_stats.cuh) in the product's epilogue.  The logits are never stored: for
// 2,048 rows over 256,000 columns they would be 2 GB, written once and read once.
//
// Shape.  Tokens are the MMA's M (a thread of the epilogue owns one token's lane of tensor memory and reduces along its columns in
// registers, without shuffles), vocabulary rows its N = 256.  Up to 128 tokens one block works alone (cta_group::1; the weights'
// bytes bound it), above that CTA pairs on 256 x 256 tiles (cta_group::2; the tensor cores bound it).  Persistent blocks walk
// (vocabulary tile, token tile), token tiles fastest, so that the blocks side by side read the same weights, which come from
// memory once, and all of x, which stays in L2.  Warp 0 issues the TMA loads, warp 1 the MMAs, warps 2 to 9 drain.
//
// The tensor cores' 32-bit accumulators round towards zero at every step of 16 products, always shrinking the sum: with all of K = 2304 in one
// sum the log probabilities are off by 1.0e-6 of their size (2-norm), by 3e-6 where all products are positive.  So a tile's K is cut into runs
// (RUN): two accumulators in tensor memory take turns, and a run's sum is drained into 32-bit registers, rounded to nearest there, while the
// next run is multiplied.
//
// Every block keeps one set of statistics per token and column half, in registers while it stays on a token tile and in a
// workspace between; a second kernel joins them.  The order of all sums is fixed by the sizes, so results repeat bit by bit.
// Waits are bounded (tc_common.cuh); a block that gives up records its code and leaves NaN as its statistics.
#include "row_stats.cuh"
#include "tc_common.cuh"

namespace {

using namespace kf_tc;
using kf_row::Stats;
using kf_row::u64;

constexpr int BN = 256;                                         // vocabulary rows of a tile
// Most blocks of 64 of a run of K, and of a K that is not cut.  Shorter runs are more exact and more to drain.  K = 2304 over 32,000 columns, cap
// 30: runs of 512 are off by 2.3e-7 and runs of 768 by 3.3e-7 (2-norm of the log probabilities; torch's 32-bit product and softmax by 3.4e-7 to
// 5.1e-7).  Single blocks, which memory bounds, take 512 for nothing (40 rows over 256,000 columns 208 us either way); for pairs 768 is the
// choice, since draining 512 at a time delays the tensor cores (2,048 rows 1,524 to 1,550 us against 1,657, 512 rows 412 to 426 against 445).
template <bool PAIR> constexpr int RUN = PAIR ? 12 : 8;
constexpr int RUN_ALONE = 8;
constexpr int EPI_WARPS = 8, HEAD_THREADS = 64 + 32 * EPI_WARPS;
constexpr int COLS = BN / 2;                                    // columns of a thread: two warps share 32 lanes
constexpr int ERR_BASE = 64;
// Caps above it take the form that is exact relative to the logit (2,048 x 256,000 x 2304 1,850 to 1,910 us against 1,520 with a cap of 30).
constexpr float WIDE_CAP = 64.f;
// Blocks of 64 of K that arrive, are multiplied and are given back at a time.  Two for pairs, which the tensor cores bound (2,048 x 256,000 x
// 2304 1,754 -> 1,570 us, 512 rows 437 -> 406); one for single blocks, which memory bounds (40 rows 210 us, two blocks 212).
template <bool PAIR> constexpr int STAGE_BLOCKS = PAIR ? 2 : 1;

// A test can make the producers leave out the loads of every stage from this one on (-1: never); see kf_test_head_give_up.
static __device__ int g_test_drop_from_stage = -1;

struct HeadArgs {
  const int* tokens;                                            // [R]
  float* given;                                                 // [R]: the token's logit, written by whoever meets it
  float4* stats;                                                // [parts][rows_padded]: m, s, u
  int* error_flag;
  int R, V, K, rows_padded, x_rows, stages;                     // x_rows: rows of the box a block loads of x
  float cap;
};

__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
// 32 columns of this thread's lane, on their way; after `tmem_arrived`, `after_wait16` keeps their uses behind the wait
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]),
        "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]),
        "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]),
        "=f"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_arrived() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void after_wait16(float* v) {
  asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]),
               "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])::"memory");
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 1 / d for d in [1, 2^41], two at a time on the FMA units (the hardware's reciprocal shares its unit with the exponential, which bounds
// the epilogue): a first guess from the exponent's and fraction's bits (a constant less these; its largest error is 5.05 %, and neighbouring
// constants differ in the fifth digit), and three Newton-Raphson steps r (2 - d r), each of which squares the error.
__device__ __forceinline__ u64 reciprocal2(u64 d) {
  const float2 f = kf_row::unpack2(d);
  u64 r = kf_row::pack2(__int_as_float(0x7ef31200 - __float_as_int(f.x)), __int_as_float(0x7ef31200 - __float_as_int(f.y)));
  const u64 minus = kf_row::pack2(-f.x, -f.y), two = kf_row::pack2(2.f, 2.f);
#pragma unroll
  for (int i = 0; i < 3; ++i) r = kf_row::mul2(r, kf_row::fma2(minus, r, two));
  return r;
}
// cap tanh(v / cap) of two logits where the quotient form's error, which counts with the cap, is more than they can bear: up to the cap itself
// v P((v / cap)^2), P of degree 6 fitted to tanh(t) / t on Chebyshev nodes of [0, 1] (relative error 1.8e-7); beyond it the quotient form.
__device__ __forceinline__ float2 capped_by_size(float a, float b, float2 quotient_form, float cap, float inverse) {
  const u64 v = kf_row::pack2(a, b), t = kf_row::mul2(v, kf_row::pack2(inverse, inverse)), z = kf_row::mul2(t, t);
  auto both = [](float c) { return kf_row::pack2(c, c); };
  u64 p = kf_row::fma2(z, both(1.045553596e-03f), both(-6.217069924e-03f));
  p = kf_row::fma2(p, z, both(2.030551992e-02f));
  p = kf_row::fma2(p, z, both(-5.346517637e-02f));
  p = kf_row::fma2(p, z, both(1.332539767e-01f));
  p = kf_row::fma2(p, z, both(-3.333285749e-01f));
  const float2 r = kf_row::unpack2(kf_row::mul2(kf_row::fma2(p, z, both(9.999999404e-01f)), v));
  return make_float2(fabsf(a) <= cap ? r.x : quotient_form.x, fabsf(b) <= cap ? r.y : quotient_form.y);
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <bool PAIR>
__global__ void __launch_bounds__(HEAD_THREADS, 1)
head_logprobs_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ HeadArgs p) {
  // KS blocks of 64 of K a stage, each a pair of operand tiles
  constexpr int A_BYTES = BM * BK * 2, B_ROWS = PAIR ? BN / 2 : BN, B_BYTES = B_ROWS * BK * 2, KS = STAGE_BLOCKS<PAIR>, STAGE = KS * (A_BYTES + B_BYTES);
  constexpr int TMEM_COLS = 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = (uint64_t*)(smem + (size_t)p.stages * STAGE);
  uint64_t* empty = full + p.stages;
  uint64_t* acc_full = empty + p.stages;                          // [2]
  uint64_t* acc_empty = acc_full + 2;                             // [2] (the leader's)
  uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);
  volatile int* s_abort = (volatile int*)(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank = 0;
  if (PAIR) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int worker = PAIR ? blockIdx.x >> 1 : blockIdx.x, n_workers = PAIR ? gridDim.x >> 1 : gridDim.x;
  constexpr int TILE_ROWS = PAIR ? 2 * BM : BM;
  const int n_tt = (p.R + TILE_ROWS - 1) / TILE_ROWS, n_vt = (p.V + BN - 1) / BN;
  const long n_tiles = (long)n_vt * n_tt;
  const int nkb = (p.K + KS * BK - 1) / (KS * BK);               // stages a tile: a last one that K does not fill multiplies zeros
  const int runs = nkb * KS <= RUN_ALONE ? 1 : nkb * KS <= 2 * RUN<PAIR> ? 2 : (nkb * KS + RUN<PAIR> - 1) / RUN<PAIR>;
  const int per_run = (nkb + runs - 1) / runs;                    // runs of nearly equal length; (runs - 1) * per_run < nkb
  const int drop = g_test_drop_from_stage;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], (PAIR ? 2 : 1) * EPI_WARPS); }
    *s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (PAIR) cluster_sync();                                       // the peer's barriers exist before anyone signals them
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  kf_pdl_trigger();                                               // after the allocation (tc_common.cuh)
  kf_pdl_wait();
  auto give_up = [&](int code) { record_error(p.error_flag, ERR_BASE + code); *s_abort = 1; __threadfence_block(); };

  if (warp == 0) {
    // ---- TMA producer: the block's own tokens, its share of the vocabulary rows; a pair's bytes are counted in the leader --------
    if (lane == 0) {
      const int bytes = KS * (p.x_rows * BK * 2 + B_BYTES);
      const uint32_t full0 = PAIR ? in_leader(smem_u32(&full[0])) : 0u;
      int s = 0, issued = 0;
      uint32_t ph = 1;
      bool ok = true;
      for (long tile = worker; tile < n_tiles && ok; tile += n_workers) {
        const int vt = (int)(tile / n_tt), tt = (int)(tile - (long)vt * n_tt);
        const int t0 = tt * TILE_ROWS + (int)rank * BM, v0 = vt * BN + (int)rank * B_ROWS;
        for (int kb = 0; kb < nkb; ++kb) {
          if (!mbar_wait(&empty[s], ph)) { give_up(ERR_WAIT_EMPTY); ok = false; break; }
          if (drop >= 0 && issued >= drop) { ok = false; break; }
          uint8_t* st = smem + (size_t)s * STAGE;
          if (rank == 0) mbar_expect_tx(&full[s], PAIR ? 2 * bytes : bytes);
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            const int k = (kb * KS + i) * BK;
            if (PAIR) {
              tma_load_pair(st + i * A_BYTES, &tm_x, full0 + 8u * (uint32_t)s, k, t0);
              tma_load_pair(st + KS * A_BYTES + i * B_BYTES, &tm_w, full0 + 8u * (uint32_t)s, k, v0);
            } else {
              tma_load_2d(st + i * A_BYTES, &tm_x, &full[s], k, t0);
              tma_load_2d(st + KS * A_BYTES + i * B_BYTES, &tm_w, &full[s], k, v0);
            }
          }
          ++issued;
          if (++s == p.stages) { s = 0; ph ^= 1; }
        }
      }
      // every load asked for has landed before this block's shared memory becomes another's
      if (rank == 0)
        for (int i = max(0, issued - p.stages); i < issued; ++i) mbar_wait(&full[i % p.stages], (uint32_t)(i / p.stages) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---- MMA issuer (a pair's leader) --------------------------------------------------------------------------------------
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(TILE_ROWS >> 4) << 24);
      const uint64_t da0 = umma_desc(smem), db0 = umma_desc(smem + KS * A_BYTES);
      int s = 0;
      uint32_t ph = 0;
      long unit = 0;                                              // runs so far
      bool ok = true;
      for (long tile = worker; tile < n_tiles && ok; tile += n_workers) {
        for (int r = 0; r < runs && ok; ++r, ++unit) {
          const int buf = (int)(unit & 1);
          if (unit >= 2 && !mbar_wait(&acc_empty[buf], (uint32_t)((unit >> 1) - 1) & 1)) { give_up(ERR_WAIT_EMPTY); ok = false; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t acc = tmem + buf * BN;
          const int kb0 = r * per_run, kb1 = min(nkb, kb0 + per_run);
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait(&full[s], ph)) { give_up(ERR_WAIT_FULL); ok = false; break; }
            const uint64_t so = (uint64_t)((uint32_t)s * (uint32_t)(STAGE >> 4));
#pragma unroll
            for (int k = 0; k < KS * (BK / UMMA_K); ++k) {
              const uint32_t accumulate = (kb > kb0 || k > 0) ? 1u : 0u;
              const int block = k / (BK / UMMA_K), in_block = 2 * (k % (BK / UMMA_K));
              const uint64_t da = da0 + so + block * (A_BYTES >> 4) + in_block, db = db0 + so + block * (B_BYTES >> 4) + in_block;
              if (PAIR)
                asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                             ::"r"(acc), "l"(da), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
              else
                umma(acc, da, db, idesc, accumulate);
            }
            if (PAIR)
              asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                           ::"r"(smem_u32(&empty[s])), "h"((uint16_t)3) : "memory");
            else
              umma_commit(&empty[s]);
            if (++s == p.stages) { s = 0; ph ^= 1; }
          }
          if (!ok) break;                                         // nobody is told of half a sum: the epilogues' waits run out too
          if (PAIR)
            asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                         ::"r"(smem_u32(&acc_full[buf])), "h"((uint16_t)3) : "memory");
          else
            umma_commit(&acc_full[buf]);
        }
      }
    }
    __syncwarp();
  } else {
    // ---- epilogue: a thread's token, its half of the tile's columns ------------------------------------------------------------
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16) + half * COLS;
    const int in_tile = (int)rank * BM + quarter * 32 + lane;
    float4* mine = p.stats + (size_t)(worker * 2 + half) * p.rows_padded + in_tile;
    for (int tt = 0; tt < n_tt; ++tt) mine[(size_t)tt * TILE_ROWS] = make_float4(-INFINITY, 0.f, 0.f, 0.f);
    Stats st = {-INFINITY, 0.f, 0.f};
    int tt_now = -1, token = -1;
    long unit = 0;
    bool ok = true;
    for (long tile = worker; tile < n_tiles && ok; tile += n_workers) {
      const int vt = (int)(tile / n_tt), tt = (int)(tile - (long)vt * n_tt);
      if (tt != tt_now) {
        if (tt_now >= 0) mine[(size_t)tt_now * TILE_ROWS] = make_float4(st.m, st.s, st.u, 0.f);
        const float4 was = mine[(size_t)tt * TILE_ROWS];
        st = {was.x, was.y, was.z};
        tt_now = tt;
        const int row = tt * TILE_ROWS + in_tile;
        token = row < p.R ? p.tokens[row] : -1;
      }
      const bool idle = tt * TILE_ROWS + in_tile - lane >= p.R;   // none of the warp's rows exists
      const int col0 = vt * BN + half * COLS;
      float acc[COLS];
#pragma unroll 1
      for (int r = 0; r < runs; ++r, ++unit) {
        const int buf = (int)(unit & 1);
        ok = mbar_wait(&acc_full[buf], (uint32_t)(unit >> 1) & 1, 2) && !*s_abort;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          if (lane == 0) give_up(ERR_WAIT_ACC);
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        auto release = [&]() {                                    // one arrival a warp: 16 of a pair's, not 512, meet at the leader's barrier
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            if (PAIR)
              asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_leader(smem_u32(&acc_empty[buf]))) : "memory");
            else
              mbar_arrive(&acc_empty[buf]);
          }
        };
        if (idle) {
          release();
          continue;
        }
        const uint32_t from = lane_addr + buf * BN;
        if (r == 0) {                                             // straight into the sums' registers, with one wait
#pragma unroll
          for (int q = 0; q < COLS; q += 32) tmem_ld32_async(from + q, acc + q);
          tmem_arrived();
#pragma unroll
          for (int q = 0; q < COLS; q += 16) after_wait16(acc + q);
        } else {
#pragma unroll
          for (int q = 0; q < COLS; q += 32) {
            float v[32];
            tmem_ld32_async(from + q, v);
            tmem_arrived();
            after_wait16(v);
            after_wait16(v + 16);
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float2 sum = kf_row::unpack2(kf_row::add2(kf_row::pack2(acc[q + j], acc[q + j + 1]), kf_row::pack2(v[j], v[j + 1])));
              acc[q + j] = sum.x;
              acc[q + j + 1] = sum.y;
            }
          }
        }
        release();
      }
      if (!ok || idle) continue;
      if (p.cap > 0.f) {
        // cap tanh(v / cap) = cap - 2 cap / (exp(2 v / cap) + 1): within 2e-7 of the cap.  From 2^40 on the quotient is nothing.  Up to
        // WIDE_CAP that is 1.3e-5 of a logit at most; a larger cap would take the digits of small logits.
        const u64 in = kf_row::pack2(2.f * kf_row::LOG2E / p.cap, 2.f * kf_row::LOG2E / p.cap), one = kf_row::pack2(1.f, 1.f);
        const u64 twice = kf_row::pack2(-2.f * p.cap, -2.f * p.cap), cap2 = kf_row::pack2(p.cap, p.cap);
        auto quotient_form = [&](float a, float b) {
          float2 e = kf_row::unpack2(kf_row::mul2(kf_row::pack2(a, b), in));
          const u64 d = kf_row::add2(kf_row::pack2(kf_row::exp2_fast(min_nan(e.x, 40.f)), kf_row::exp2_fast(min_nan(e.y, 40.f))), one);
          return kf_row::unpack2(kf_row::fma2(reciprocal2(d), twice, cap2));
        };
        if (p.cap <= WIDE_CAP) {
#pragma unroll
          for (int j = 0; j < COLS; j += 2) {
            const float2 e = quotient_form(acc[j], acc[j + 1]);
            acc[j] = e.x;
            acc[j + 1] = e.y;
          }
        } else {
          const float inverse = 1.f / p.cap;
#pragma unroll
          for (int j = 0; j < COLS; j += 2) {
            const float2 e = capped_by_size(acc[j], acc[j + 1], quotient_form(acc[j], acc[j + 1]), p.cap, inverse);
            acc[j] = e.x;
            acc[j + 1] = e.y;
          }
        }
      }
      if (col0 + COLS > p.V) {                                    // columns beyond the vocabulary
#pragma unroll
        for (int j = 0; j < COLS; ++j)
          if (col0 + j >= p.V) acc[j] = -INFINITY;
      }
      const int at = token - col0;
      if (token < p.V && at >= 0 && at < COLS) {
        float g = 0.f;
#pragma unroll
        for (int j = 0; j < COLS; ++j) g = j == at ? acc[j] : g;
        p.given[tt * TILE_ROWS + in_tile] = g;
      }
      float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
      for (int j = 0; j < COLS; j += 2) {
        m0 = fmaxf(m0, acc[j]);
        m1 = fmaxf(m1, acc[j + 1]);
      }
      kf_row::move_to(st, fmaxf(st.m, fmaxf(m0, m1)));
      kf_row::add_exponentials<COLS>(st, [&](int j) { return acc[j]; });
    }
    const float nan = __int_as_float(0x7fffffff);
    if (!ok)
      for (int tt = 0; tt < n_tt; ++tt) mine[(size_t)tt * TILE_ROWS] = make_float4(-INFINITY, nan, nan, 0.f);
    else if (tt_now >= 0)
      mine[(size_t)tt_now * TILE_ROWS] = make_float4(st.m, st.s, st.u, 0.f);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*s_abort) {                                                 // a peer's loads that this block cannot wait for land within microseconds: a millisecond
    const unsigned long long t0 = global_ns();
    for (int i = 0; i < 1000000 && global_ns() - t0 < 1000000ull; ++i) __nanosleep(1000);
  }
  if (PAIR) cluster_sync();                                       // no MMA of the pair is in flight, nobody signals a block that left
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
}

// Joins the parts of 8 rows: neighbouring lanes take neighbouring rows, and 32 groups of threads every 32nd part.
constexpr int JOIN_ROWS = 8, JOIN_THREADS = 256, JOIN_GROUPS = JOIN_THREADS / JOIN_ROWS;
__global__ void __launch_bounds__(JOIN_THREADS) head_join_kernel(const float4* stats, int parts, int rows_padded, const float* given,
                                                                 const int* tokens, int R, int V, float* logprob, float* entropy) {
  kf_pdl_trigger();
  kf_pdl_wait();
  __shared__ Stats part[JOIN_THREADS / 32][JOIN_ROWS];
  const int tid = threadIdx.x, row = blockIdx.x * JOIN_ROWS + tid % JOIN_ROWS;
  Stats st = {-INFINITY, 0.f, 0.f};
#pragma unroll 8
  for (int i = tid / JOIN_ROWS; i < parts; i += JOIN_GROUPS) {
    const float4 f = stats[(size_t)i * rows_padded + row];
    kf_row::join(st, {f.x, f.y, f.z});
  }
#pragma unroll
  for (int o = JOIN_ROWS; o < 32; o *= 2)
    kf_row::join(st, {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.u, o)});
  if (tid % 32 < JOIN_ROWS) part[tid / 32][tid % 32] = st;
  __syncthreads();
  if (tid >= JOIN_ROWS || row >= R) return;
#pragma unroll
  for (int i = 1; i < JOIN_THREADS / 32; ++i) kf_row::join(st, part[i][tid]);
  const int token = tokens[row];
  if (token < 0) return;
  logprob[row] = kf_row::row_logprob(st, token < V ? given[row] : __int_as_float(0x7fffffff));
  if (entropy) entropy[row] = kf_row::row_entropy(st);
}

int padded(int R) { return (R + 255) / 256 * 256; }
// blocks (of a launch of single blocks) or pairs
int workers(int R, int V) {
  const long tiles = (long)kf_ceil_div(V, BN) * (R > BM ? kf_ceil_div(R, 2 * BM) : 1);
  const int most = R > BM ? kf_sm_count() / 2 : kf_sm_count();
  return tiles < most ? (int)tiles : most;
}

template <bool PAIR>
int launch(const CUtensorMap& tx, const CUtensorMap& tw, HeadArgs p, int n_workers, cudaStream_t stream) {
  constexpr int STAGE = STAGE_BLOCKS<PAIR> * (BM + (PAIR ? BN / 2 : BN)) * BK * 2;
  p.stages = PAIR ? 3 : 4;                                        // 192 KB
  const size_t smem = (size_t)p.stages * STAGE + 1024 + 256;
  static bool configured[64] = {};                                // by device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(head_logprobs_kernel<PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
      kf_record_cuda_error(cudaGetLastError());
      return KF_ERR_SETUP;
    }
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((PAIR ? 2 : 1) * n_workers);
  cfg.blockDim = dim3(HEAD_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (kf_pdl_enabled()) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (PAIR) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = 2;
    attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
    ++na;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  cudaLaunchKernelEx(&cfg, head_logprobs_kernel<PAIR>, tx, tw, p);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

}  // namespace

// Whether this kernel takes the operands: bfloat16 rows that are multiples of 16 bytes, on 16-byte addresses.
KF_API int kf_head_logprobs_supported(const void* x, const void* w, int K) {
  return K > 0 && K % 8 == 0 && (((uintptr_t)x | (uintptr_t)w) & 15) == 0 && tensor_maps_available();
}
// Floats of workspace for R rows over V columns.
KF_API long kf_head_logprobs_workspace(int R, int V) { return (long)padded(R) * (1 + 4l * 2 * workers(R, V)); }

// x [R, K], w [V, K] bfloat16; tokens [R] (negative: the row's results stay as they are; >= V: NaN); logprob [R], entropy [R] or null.
KF_API int kf_head_logprobs(const void* x, const void* w, const int* tokens, int R, int V, int K, float cap, float* logprob,
                            float* entropy, float* workspace, int* error_flag, cudaStream_t stream) {
  if (R <= 0) return KF_OK;
  if (V <= 0 || V > 0x7ffffe00 || R > 0x7fffff00 || !tokens || !logprob || !workspace) return KF_ERR_SIZE;
  if (!kf_head_logprobs_supported(x, w, K) || ((uintptr_t)workspace & 15)) return KF_ERR_ALIGN;
  const bool pair = R > BM;
  int box = 16;
  while (box < BM && box < R) box *= 2;
  HeadArgs p{};
  p.tokens = tokens;
  p.rows_padded = padded(R);
  p.stats = reinterpret_cast<float4*>(workspace);
  const int n_workers = workers(R, V);
  p.given = workspace + 4l * 2 * n_workers * p.rows_padded;
  p.error_flag = error_flag;
  p.R = R, p.V = V, p.K = K, p.x_rows = box, p.cap = cap;
  CUtensorMap tx, tw;
  if (!tensor_map(x, R, K, box, &tx) || !tensor_map(w, V, K, pair ? BN / 2 : BN, &tw)) return KF_ERR_SETUP;
  const int rc = pair ? launch<true>(tx, tw, p, n_workers, stream) : launch<false>(tx, tw, p, n_workers, stream);
  if (rc != KF_OK) return rc;
  kf_launch(head_join_kernel, dim3(kf_ceil_div(R, JOIN_ROWS)), dim3(JOIN_THREADS), 0, stream, (const float4*)p.stats, 2 * n_workers, p.rows_padded,
            (const float*)p.given, tokens, R, V, logprob, entropy);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

// For tests: as kf_test_gemm_give_up (gemm_tc.cu), for this kernel.
KF_API int kf_test_head_give_up(unsigned long long limit_ns, int drop_from_stage) {
  const unsigned long long lim = limit_ns ? limit_ns : WAIT_LIMIT_NS;
  if (cudaMemcpyToSymbol(g_wait_limit_ns, &lim, sizeof(lim)) != cudaSuccess ||
      cudaMemcpyToSymbol(g_test_drop_from_stage, &drop_from_stage, sizeof(int)) != cudaSuccess) {
    kf_record_cuda_error(cudaGetLastError());
    return KF_ERR_SETUP;
  }
  return KF_OK;
}
