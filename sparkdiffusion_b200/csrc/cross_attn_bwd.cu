// Backward of the attention to another sequence's states (cross_attn.cu), on
// tcgen05, without atomics.  From the forward's base-2 log-sum-exp:
//
//   delta[i] = sum_d dO[i, d] O[i, d]   (by the way, in the dq kernel, which has dO;
//              O is the rounded output.  Over 64 keys or fewer, where dP and delta
//              nearly cancel and that rounding would be the largest error of dQ and dK
//              (2 keys: 0.0037 of their norm, without it 0.0024), it is sum_j P dP,
//              the same number)
//   P  = exp2(q.k D^-1/2 log2(e) - lse[i])             (recomputed, fp32; 0 past len[b])
//   dP = dO V^T,  dS = P (dP - delta[i])
//   dQ = D^-1/2 dS K                    query-stationary   (cross_bwd_dq_tcgen05)
//   dV = P^T dO,  dK = D^-1/2 dS^T Q    key-stationary     (cross_bwd_dkdv_tcgen05)
//
// P and dS are rounded to bf16 where they feed a product; sums are fp32 in
// tensor memory.  dK and dV of a key head sum over its G query heads: the key
// tile stays and the steps walk the rows of all of them.  An encoder's states
// are few key tiles and many query rows, so a tile's rows are dealt to several
// CTAs, whose fp32 partials are added in a fixed order.
// Keys past len[b] contribute nothing whatever they hold: their scores are
// dropped by selection, their K rows cleared before dS K.
#include "common.cuh"
#include "kernels.h"

namespace rola {

// rows [valid, 64) of a [64 x 128] half tile := 0
__device__ __forceinline__ void clear_half_rows(uint8_t* half, int valid, int lane) {
  for (int i = valid * 8 + lane; i < 64 * 8; i += 32) {
    *reinterpret_cast<uint4*>(half + i * 16) = make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4*>(half + bwd::BOX + i * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// ---------------------------------------------------------------------------
// dq: persistent CTAs walk items (128 query rows of a head) in steps of 64 keys.
// A step is a chain, (S, dP) -> dS -> dQ, three in flight across the items' ends
// (S and dP of a step take 128 columns of tensor memory, dQ 128), as the units of
// cross_attn_tcgen05; one CTA per item spent more time on its ends than on the 8
// steps of 512 keys (1.06 ms at 32760 x 512, 40 heads; now 0.53: 965 TFLOP/s, 0.58 of
// the matrix peak).  The three chains bound it, 4150 clocks each: 3 x 256 of products,
// about 2000 of the softmax warpgroup, the hand-offs between them.  Tried and slower:
// S ahead of the dQ of the step before in its columns (0.64), dQ read by warpgroup 4
// (0.57), rings of 3 K and 3 V tiles (0.6).
//   warp 0   TMA producer of Q and dO (2 x 64 KB); it also stores an item's dQ,
//            left in the item's Q tile, before that is loaded again
//   warp 3   TMA producer of K (4 x 16 KB) and V (2 x 16 KB)
//   warp 1   issues S and dP; owner of the tensor memory
//   warp 2   issues dQ; clears the K rows past len[b] first
//   warpgroups 1-3: dS of the steps u with u % 3 == warpgroup - 1 (thread = row);
//            the step that ends an item leaves its dQ in bf16
//   warpgroup 4  delta of the items ahead, for this kernel and the next: dO from
//            shared memory, O from global memory (a kernel of its own read dO once more
//            and took 0.13 ms)
// ---------------------------------------------------------------------------
namespace xdq {
constexpr int THREADS = 640, LAUNCH_REGS = 96;  // 65536 / 640, in steps of 8
constexpr int REGS_LOAD = 56, REGS_SOFTMAX = 112, REGS_DELTA = 88;
static_assert(128 * (REGS_LOAD + 3 * REGS_SOFTMAX + REGS_DELTA) <= THREADS * LAUNCH_REGS, "register split");
constexpr int NT = 2, NK = 4, NV = 2, NS = 3;
constexpr int OFF_T = 0;                                // NT x (Q, dO)
constexpr int OFF_K = OFF_T + NT * 2 * bwd::TILE, OFF_V = OFF_K + NK * bwd::HALF;
constexpr int OFF_DELTA = OFF_V + NV * bwd::HALF;       // [NT][128]
constexpr int OFF_BAR = OFF_DELTA + NT * 512;
constexpr int SMEM = OFF_BAR + 384;
constexpr int ACC = 128 * NS;                           // TMEM: S of step u at 128 (u % 3), dP 64 behind, dQ at ACC
enum : int {
  TF = 0, TE = TF + NT,  // TE: the item's dQ is in its Q tile, 4 warp arrivals
  DR = TE + NT,          // delta of the item's rows in shared memory, 4 arrivals
  KF = DR + NT, KE = KF + NK, VF = KE + NK, VE = VF + NV,
  SF = VE + NV,          // S and dP of a step in TMEM
  DS = SF + NS,          // dS of a step in TMEM, 4 arrivals
  DQ = DS + NS,          // dQ of a step done
  OE = DQ + NS,          // dQ of an item read, 4 arrivals
  DRAIN_S = OE + 1, DRAIN_Q, COUNT
};
static_assert(8 * COUNT + 16 <= 384 && SMEM <= 227 * 1024, "shared memory");
}  // namespace xdq

// The items of a CTA, w = blockIdx.x, + gridDim.x, ...: query tile fastest, then
// head and batch; digits advanced by the step's own with carries
struct QueryItems {
  uint32_t w;
  int m, h, b, dm, dh, db;
  int len, cnt;  // valid keys, steps of 64
  __device__ __forceinline__ void range(const CrossBwdParams& p) {
    if (!live(p)) return;
    len = kv_len(p.kv_lens, b, p.Lk);
    cnt = (len + 63) >> 6;
  }
  __device__ __forceinline__ explicit QueryItems(const CrossBwdParams& p) : w(blockIdx.x) {
    auto digits = [&](uint32_t x, int& m_, int& h_, int& b_) {
      const uint32_t r = x / (uint32_t)p.NQT;
      m_ = (int)(x - r * (uint32_t)p.NQT);
      b_ = (int)(r / (uint32_t)p.H);
      h_ = (int)(r - (uint32_t)b_ * (uint32_t)p.H);
    };
    digits(w, m, h, b);
    digits(gridDim.x, dm, dh, db);
    range(p);
  }
  __device__ __forceinline__ bool live(const CrossBwdParams& p) const { return w < (uint32_t)(p.NQT * p.H * p.B); }
  __device__ __forceinline__ void next(const CrossBwdParams& p) {
    w += gridDim.x;
    m += dm;
    int c = m >= p.NQT;
    m -= c ? p.NQT : 0;
    h += dh + c;
    c = h >= p.H;
    h -= c ? p.H : 0;
    b += db + c;
    range(p);
  }
};

__global__ void __launch_bounds__(xdq::THREADS, 1)
    cross_bwd_dq_tcgen05(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                         const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tdo,
                         const __grid_constant__ CUtensorMap tdq, const CrossBwdParams p) {
  using namespace xdq;
  constexpr int TILE = bwd::TILE, HALF = bwd::HALF, BOX = bwd::BOX, BOX128 = bwd::BOX128;
  extern __shared__ __align__(1024) uint8_t smem1k[];
  const uint32_t base = smem_u32(smem1k);
  auto bar = [&](int i) { return base + OFF_BAR + 8u * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem1k + OFF_BAR + 8 * COUNT);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem1k + OFF_BAR + 8 * COUNT + 8);
  // broadcast values are warp-uniform to the compiler too (uniform registers for the MMAs)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < COUNT; ++i)
      mbar_init(bar(i), (i >= TE && i < KF) || (i >= DS && i < DQ) || i == OE ? 4 : 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tq);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
    prefetch_tmap(&tdo);
    prefetch_tmap(&tdq);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  bool ok = true;
  auto wait = [&](int i, uint32_t parity, int code) {
    if (ok) ok = __all_sync(0xffffffffu, mbar_spin(bar(i), parity, abort_flag, code));
    tc_fence_after();
    return ok;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_LOAD));
    constexpr uint32_t hi = sdesc_hi(1024);
    if (warp == 0) {
      if (lane == 0) {
        // ------------------------------------------ TMA: Q, dO; dQ of the items
        int q = 0;
        int om[NT] = {}, oh[NT] = {}, ob[NT] = {};
        auto store_out = [&](int e, int n) {
          if (!mbar_spin(bar(TE + e), n & 1, abort_flag, kDevTimeoutSoftmax, 2 * (uint32_t)(p.Lk >> 6))) return false;
          const uint32_t src = base + OFF_T + e * 2 * TILE;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (om[e] * 128 + 64 * (c & 1) < p.Lq)  // 64-row boxes: the second may lie past the last row
              tma_store_4d(&tdq, src + (c >> 1) * BOX128 + (c & 1) * BOX, 64 * (c >> 1), om[e] * 128 + 64 * (c & 1), oh[e],
                           ob[e]);
          tma_store_commit();
          tma_store_wait_read();
          return true;
        };
        for (QueryItems it(p); it.live(p) && ok; it.next(p)) {
          if (it.cnt == 0) continue;
          const int e = q % NT;
          if (q >= NT && !(ok = store_out(e, q / NT - 1))) break;
          mbar_expect_tx(bar(TF + e), 2 * TILE);
          load_tile(base + OFF_T + e * 2 * TILE, &tq, bar(TF + e), 128 * it.m, it.h, it.b);
          load_tile(base + OFF_T + e * 2 * TILE + TILE, &tdo, bar(TF + e), 128 * it.m, it.h, it.b);
          om[e] = it.m;
          oh[e] = it.h;
          ob[e] = it.b;
          ++q;
        }
        for (int n = max(0, q - NT); n < q && ok; ++n) ok = store_out(n % NT, n / NT);
        // no copy may still target shared memory when the CTA exits; the waits
        // ignore the abort flag and share one limit
        const uint64_t deadline = globaltimer_ns() + kWaitLimitNs;
        bool drained = true;
        for (int n = max(0, q - NT); n < q && drained; ++n)
          drained = mbar_wait_until(bar(TF + n % NT), (n / NT) & 1, deadline);
      }
    } else if (warp == 3) {
      if (lane == 0) {
        // ------------------------------------------------------ TMA: K and V
        int k = 0;
        for (QueryItems it(p); it.live(p) && ok; it.next(p)) {
          const int hk = it.h / p.G;
          for (int i = 0; i < it.cnt; ++i, ++k) {
            const int ek = k % NK, ev = k % NV;
            if (!(ok = mbar_spin(bar(KE + ek), ((k / NK) & 1) ^ 1, abort_flag, kDevTimeoutMma))) break;
            mbar_expect_tx(bar(KF + ek), HALF);
            load_half(base + OFF_K + ek * HALF, &tk, bar(KF + ek), 64 * i, hk, it.b);
            if (!(ok = mbar_spin(bar(VE + ev), ((k / NV) & 1) ^ 1, abort_flag, kDevTimeoutMma))) {
              ++k;  // this K is on its way, its V is not
              break;
            }
            mbar_expect_tx(bar(VF + ev), HALF);
            load_half(base + OFF_V + ev * HALF, &tv, bar(VF + ev), 64 * i, hk, it.b);
          }
        }
        const uint64_t deadline = globaltimer_ns() + kWaitLimitNs;
        bool drained = true;
        for (int n = max(0, k - NK); n < k && drained; ++n)
          drained = mbar_wait_until(bar(KF + n % NK), (n / NK) & 1, deadline);
        const int v = ok ? k : k - 1;
        for (int n = max(0, v - NV); n < v && drained; ++n)
          drained = mbar_wait_until(bar(VF + n % NV), (n / NV) & 1, deadline);
      }
    } else if (warp == 1) {
      // ------------------------------------- MMA: S = Q K^T, dP = dO V^T
      constexpr uint32_t id_s = idesc_bf16_f32(128, 64, false, false);
      int et = 0, ek = 0, ev = 0, g = 0;
      uint32_t t_ph = 0, k_ph = 0, v_ph = 0, g_ph = 1;
      for (QueryItems it(p); it.live(p) && ok; it.next(p)) {
        const int cnt = __shfl_sync(0xffffffffu, it.cnt, 0);
        if (cnt == 0) continue;
        if (!wait(TF + et, t_ph, kDevTimeoutLoad)) break;
        const uint32_t dq = sdesc_lo(base + OFF_T + et * 2 * TILE, 16), ddo = sdesc_lo(base + OFF_T + et * 2 * TILE + TILE, 16);
        for (int i = 0; i < cnt; ++i) {
          if (!wait(KF + ek, k_ph, kDevTimeoutLoad) || !wait(VF + ev, v_ph, kDevTimeoutLoad) ||
              !wait(DQ + g, g_ph, kDevTimeoutMma))
            break;
          if (elect_one()) {
            const uint32_t dk = sdesc_lo(base + OFF_K + ek * HALF, 16), dv = sdesc_lo(base + OFF_V + ev * HALF, 16);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
              const uint32_t ka = ((kk >> 2) * BOX128 + (kk & 3) * 32) >> 4, kb = ((kk >> 2) * BOX + (kk & 3) * 32) >> 4;
              mma_bf16_ss_lo(tmem + 128 * g, dq + ka, hi, dk + kb, hi, id_s, kk > 0 ? 1u : 0u);
            }
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
              const uint32_t ka = ((kk >> 2) * BOX128 + (kk & 3) * 32) >> 4, kb = ((kk >> 2) * BOX + (kk & 3) * 32) >> 4;
              mma_bf16_ss_lo(tmem + 128 * g + 64, ddo + ka, hi, dv + kb, hi, id_s, kk > 0 ? 1u : 0u);
            }
            mma_commit(bar(SF + g));
            mma_commit(bar(VE + ev));
          }
          __syncwarp();
          if (++ek == NK) ek = 0, k_ph ^= 1u;
          if (++ev == NV) ev = 0, v_ph ^= 1u;
          if (++g == NS) g = 0, g_ph ^= 1u;
        }
        if (++et == NT) et = 0, t_ph ^= 1u;
      }
      // every MMA issued has completed before TMEM is freed, also on the abort path
      if (elect_one()) {
        mma_commit(bar(DRAIN_S));
        mbar_wait_until(bar(DRAIN_S), 0, globaltimer_ns() + kWaitLimitNs);
      }
      __syncwarp();
    } else {
      // ------------------------------------------------- MMA: dQ += dS K
      constexpr uint32_t id_q = idesc_bf16_f32(128, 128, false, true);
      int ek = 0, g = 0;
      uint32_t g_ph = 0, o_ph = 1;
      for (QueryItems it(p); it.live(p) && ok; it.next(p)) {
        const int cnt = __shfl_sync(0xffffffffu, it.cnt, 0);
        if (cnt == 0) continue;
        const int valid = it.len - 64 * (it.cnt - 1);  // keys of the last step
        const int tail = __shfl_sync(0xffffffffu, it.len < p.Lk ? valid : 64, 0);
        for (int i = 0; i < cnt; ++i) {
          // dS is in place, hence S has been computed from this K (which may be cleared now)
          if (!wait(DS + g, g_ph, kDevTimeoutSoftmax)) break;
          if (i == 0 && !wait(OE, o_ph, kDevTimeoutSoftmax)) break;  // dQ of the previous item has been read
          if (tail < 64 && i + 1 == cnt) clear_half_rows(smem1k + OFF_K + ek * HALF, tail, lane);
          if (elect_one()) {
            const uint32_t dk = sdesc_lo(base + OFF_K + ek * HALF, BOX);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_bf16_ts_lo(tmem + ACC, tmem + 128 * g + 8 * kk, dk + ((kk * 2048) >> 4), hi, id_q,
                             (i > 0 || kk > 0) ? 1u : 0u);
            mma_commit(bar(DQ + g));
            mma_commit(bar(KE + ek));
          }
          __syncwarp();
          if (++ek == NK) ek = 0;
          if (++g == NS) g = 0, g_ph ^= 1u;
        }
        o_ph ^= 1u;
      }
      if (elect_one()) {
        mma_commit(bar(DRAIN_Q));
        mbar_wait_until(bar(DRAIN_Q), 0, globaltimer_ns() + kWaitLimitNs);
      }
      __syncwarp();
    }
  } else if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_DELTA));
    // ------------------------------------------------------------------ delta
    const int row = (warp & 3) * 32 + lane;
    int j = 0;
    for (QueryItems it(p); it.live(p) && ok; it.next(p)) {
      if (it.cnt == 0) continue;
      const int e = j % NT, tok = 128 * it.m + row;
      const uint8_t* dos = smem1k + OFF_T + e * 2 * TILE + TILE + row * 128;
      const uint4* o = reinterpret_cast<const uint4*>(p.o + it.b * p.o_sB + it.h * p.o_sH + (int64_t)min(tok, p.Lq - 1) * p.o_sT);
      // (loaded once the item before the previous one has left its tile: an item's time)
      ok = __all_sync(0xffffffffu, mbar_spin(bar(TF + e), (j / NT) & 1, abort_flag, kDevTimeoutLoad, 2 * (uint32_t)(p.Lk >> 6)));
      if (!ok) break;
      if (it.cnt > 1) {
        float acc = 0.f;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const uint4 ov = __ldg(o + c);
          const uint4 dv = *reinterpret_cast<const uint4*>(dos + (c >> 3) * BOX128 + (((c & 7) ^ (row & 7)) << 4));
          const uint32_t oa[4] = {ov.x, ov.y, ov.z, ov.w}, da[4] = {dv.x, dv.y, dv.z, dv.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float o0, o1, d0, d1;
            unpack_bf2(oa[k], o0, o1);
            unpack_bf2(da[k], d0, d1);
            acc = fmaf(o0, d0, acc);
            acc = fmaf(o1, d1, acc);
          }
        }
        if (tok >= p.Lq) acc = 0.f;  // a padding row (its P is 0, its delta has to be a number)
        reinterpret_cast<float*>(smem1k + OFF_DELTA)[e * 128 + row] = acc;
        p.delta[((int64_t)it.b * p.H + it.h) * p.Lpad + tok] = acc;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(DR + e));
      ++j;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    // -------------------------------------------------- dS, and dQ of an item
    const int g = (warp >> 2) - 1, q = warp & 3, row = q * 32 + lane;
    const uint32_t lane_off = (uint32_t)(q * 32) << 16;
    const uint32_t tS = tmem + 128 * g + lane_off, tdP = tS + 64, tQ = tmem + ACC + lane_off;
    const uint64_t sc2 = f2_pack(p.qk_scale, p.qk_scale);
    int u = 0, j = 0, items = 0;  // steps, items with keys, items
    uint32_t ph = 0;              // of this warpgroup's steps
    // the row's log-sum-exp, one item ahead
    auto stat = [&](const QueryItems& it) {
      return it.live(p) ? __ldg(p.lse + ((int64_t)it.b * p.H + it.h) * p.Lpad + 128 * it.m + row) : 0.f;
    };
    QueryItems it(p);
    float lse_next = stat(it);
    while (it.live(p) && ok) {
      const int m = it.m, h = it.h, b = it.b, len = it.len, cnt = it.cnt;
      const float lse = lse_next;
      it.next(p);
      lse_next = stat(it);
      if (cnt == 0) {
        // no keys: zeros (one warpgroup in turn; no step, nothing to wait for)
        const int tok = 128 * m + row;
        if (items % 3 == g && tok < p.Lq) {
          uint4* dst = reinterpret_cast<uint4*>(p.dq + b * p.dq_sB + h * p.dq_sH + tok * p.dq_sT);
#pragma unroll
          for (int c = 0; c < 16; ++c) dst[c] = make_uint4(0u, 0u, 0u, 0u);
        }
        __syncwarp();
        ++items;
        continue;
      }
      const uint64_t nl2 = f2_pack(-lse, -lse);
      uint64_t nd2 = 0ull;
      bool have_delta = false;
      for (int i = 0; i < cnt; ++i, ++u) {
        if (u % NS != g) continue;
        if (!wait(SF + g, ph, kDevTimeoutMma)) break;
        if (!have_delta) {
          // Only with a step of the item at hand: a warpgroup without one may find the
          // barrier two phases on, which parity cannot tell from not yet.  Items of one step
          // wait too, although they make delta themselves: the item's TE, and with it the
          // reload of its tiles, comes behind this wait, which keeps the delta warps within
          // NT items (nothing else does; they too know phases by parity)
          if (!wait(DR + j % NT, (j / NT) & 1, kDevTimeoutSoftmax)) break;
          float dlt = 0.f;
          if (cnt == 1) {
            // every key of the row is here: delta as sum_j P dP, from fp32 alone
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t sv[32], dv[32];
              tmem_ld32(tS + 32 * c, sv);
              tmem_ld32(tdP + 32 * c, dv);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (32 * c + e < len)
                  dlt = fmaf(ex2_approx(fmaf(__uint_as_float(sv[e]), p.qk_scale, -lse)), __uint_as_float(dv[e]), dlt);
            }
            p.delta[((int64_t)b * p.H + h) * p.Lpad + 128 * m + row] = dlt;
          } else {
            dlt = reinterpret_cast<const float*>(smem1k + OFF_DELTA)[(j % NT) * 128 + row];
          }
          nd2 = f2_pack(-dlt, -dlt);
          have_delta = true;
        }
        const int valid = len - 64 * i;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t sv[32], dv[32];
          tmem_ld32(tS + 32 * c, sv);
          tmem_ld32(tdP + 32 * c, dv);
          tmem_ld_wait();
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x0, x1, d0, d1;
            f2_unpack(fma_f32x2(f2_pack(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), sc2, nl2), x0, x1);
            const uint64_t pd = mul_f32x2(
                f2_pack(ex2_approx(x0), ex2_approx(x1)),
                add_f32x2(f2_pack(__uint_as_float(dv[2 * e]), __uint_as_float(dv[2 * e + 1])), nd2));
            f2_unpack(pd, d0, d1);
            w[e] = pack_bf2(d0, d1);
          }
          if (valid < 64) {  // by selection: past len[b] the products may be anything
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int col = 32 * c + 2 * e;
              w[e] = col + 1 < valid ? w[e] : col < valid ? w[e] & 0xffffu : 0u;
            }
          }
          tmem_st16(tS + 16 * c, w);  // packed dS over the first 32 S columns of the step
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(DS + g));
        if (i + 1 == cnt) {
          if (!wait(DQ + g, ph, kDevTimeoutMma)) break;
          // the row of the item's Q tile, whose last product is done: 16-byte chunk c of a
          // box at c ^ (row & 7), the maps' swizzle
          uint8_t* stage = smem1k + OFF_T + (j % NT) * 2 * TILE + row * 128;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t v[64];
            tmem_ld32(tQ + 64 * c, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
            tmem_ld32(tQ + 64 * c + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
            tmem_ld_wait();
            if (c == 1) {
              // dQ is in registers: the next item may start its own
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(OE));
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              uint32_t w4[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                w4[k] = pack_bf2(__uint_as_float(v[8 * e + 2 * k]) * bwd::kSmScale,
                                 __uint_as_float(v[8 * e + 2 * k + 1]) * bwd::kSmScale);
              *reinterpret_cast<uint4*>(stage + c * BOX128 + ((e ^ (row & 7)) << 4)) =
                  make_uint4(w4[0], w4[1], w4[2], w4[3]);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(TE + j % NT));
        }
        ph ^= 1u;
      }
      ++j;
      ++items;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// dk, dv: the steps (64 query rows against a 128-row key tile) of all key tiles
// that hold a valid key, one tile after the other, are dealt to the CTAs in equal
// runs.  A CTA's run is a few segments, each within one tile; a tile within one
// run is stored as it is, the others' segments leave fp32 partials that
// cross_bwd_join_kernel adds in order.  (An encoder's states are few tiles: 160 at
// 512 states and 40 heads.  12 slices of each as CTAs of their own took 0.64 ms with
// the join, of it 0.1 in their ends and last round.)  Measured there: 0.56 ms and
// 0.013 for the join, 1220 TFLOP/s, 0.73 of the matrix peak; two steps in flight,
// which is all that tensor memory holds beside dV and dK, bound it.
//   warp 0   TMA producer: K and V of the tile, the ring of (Q, dO, lse, delta)
//   warp 1   issues S^T = K Q^T and dP^T = V dO^T of a step, then dV += P^T dO and
//            dK += dS^T Q of the step before: in one warp's order the columns of a step
//            are overwritten without a wait (a second issuing warp, which has to wait
//            for that, measured 10 % slower: there are two steps in flight, not three);
//            owner of the tensor memory
//   warps 4-11  P^T and dS^T: both warpgroups on every step, 32 columns each
// ---------------------------------------------------------------------------
namespace xkv {
constexpr int THREADS = 384;
constexpr int NR = 4;                                        // ring entries
constexpr int ENTRY = 2 * bwd::HALF + 1024;                  // + 64 lse + 64 delta
constexpr int OFF_K = 0, OFF_V = bwd::TILE, OFF_RING = 2 * bwd::TILE;
constexpr int OFF_BAR = OFF_RING + NR * ENTRY;
constexpr int SMEM = OFF_BAR + 256;
enum : int {
  TF = 0,            // K and V of a segment loaded
  RF, RE = RF + NR,  // ring
  SF = RE + NR,      // S^T and dP^T of a step in TMEM
  DS = SF + 2,       // P^T and dS^T of a step in TMEM, 8 warp arrivals
  AF = DS + 2,       // dV and dK of a segment final
  AE,                // dV and dK of a segment read, 8 arrivals
  DRAIN, COUNT
};
static_assert(8 * COUNT + 16 <= 256 && SMEM <= 227 * 1024, "shared memory");
}  // namespace xkv

// Key tiles (b, key head, J), J * 128 < len[b], in that order
struct KvTiles {
  int b = 0;
  int64_t base = 0;  // tiles before batch b
  int len = 0, n = 0;  // of batch b
  __device__ __forceinline__ explicit KvTiles(const CrossBwdParams& p) { at(p); }
  __device__ __forceinline__ void at(const CrossBwdParams& p) {
    len = kv_len(p.kv_lens, b, p.Lk);
    n = (len + 127) >> 7;
  }
  // tile t (not before an earlier call's).  Equal lengths are divided out: the walk takes
  // 50 ns a sequence (65536 of them 3.3 ms), over a million as long as the other roles'
  // waits for this one may last.  Lengths of their own are walked; the 65536 sequences
  // that the entry point takes are 6 ms
  __device__ __forceinline__ void find(const CrossBwdParams& p, int64_t t, int& hk, int& J) {
    if (p.kv_lens == nullptr) {
      b = (int)(t / ((int64_t)n * p.Hkv));
      base = (int64_t)b * n * p.Hkv;
    }
    while (t >= base + (int64_t)n * p.Hkv && b + 1 < p.B) {
      base += (int64_t)n * p.Hkv;
      ++b;
      at(p);
    }
    const int r = (int)(t - base);
    hk = r / max(n, 1);
    J = r - hk * n;
  }
};
// valid key tiles of batches [0, end), by all threads of the CTA (s: a shared word)
__device__ __forceinline__ int64_t kv_tiles_before(const CrossBwdParams& p, int end, unsigned long long* s) {
  if (p.kv_lens == nullptr) return (int64_t)end * p.Hkv * p.NKT;
  __syncthreads();
  if (threadIdx.x == 0) *s = 0ull;
  __syncthreads();
  unsigned long long v = 0;
  for (int b = threadIdx.x; b < end; b += blockDim.x) v += (unsigned)((kv_len(p.kv_lens, b, p.Lk) + 127) >> 7);
  if (v) atomicAdd(s, v);  // whole numbers: the order does not matter
  __syncthreads();
  return (int64_t)*s * p.Hkv;
}

__global__ void __launch_bounds__(xkv::THREADS, 1)
    cross_bwd_dkdv_tcgen05(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                           const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tdo,
                           const CrossBwdParams p) {
  using namespace xkv;
  constexpr int TILE = bwd::TILE, HALF = bwd::HALF, BOX = bwd::BOX, BOX128 = bwd::BOX128;
  extern __shared__ __align__(1024) uint8_t smem1k[];
  const uint32_t base = smem_u32(smem1k);
  auto bar = [&](int i) { return base + OFF_BAR + 8u * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem1k + OFF_BAR + 8 * COUNT);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem1k + OFF_BAR + 8 * COUNT + 8);
  // broadcast values are warp-uniform to the compiler too (uniform registers for the MMAs)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  const int64_t tiles = kv_tiles_before(p, p.B, reinterpret_cast<unsigned long long*>(smem1k));
  const int NH = (p.Lq + 63) / 64, T = p.G * NH;  // steps per query head, per tile
  const int64_t x0 = tiles * T * blockIdx.x / gridDim.x, x1 = tiles * T * (blockIdx.x + 1) / gridDim.x;
  __syncthreads();

  if (threadIdx.x == 0) {
    for (int i = 0; i < COUNT; ++i) mbar_init(bar(i), (i >= DS && i < AF) || i == AE ? 8 : 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tq);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
    prefetch_tmap(&tdo);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  constexpr uint32_t hi = sdesc_hi(1024);
  bool ok = true;
  auto wait = [&](int i, uint32_t parity, int code) {
    if (ok) ok = __all_sync(0xffffffffu, mbar_spin(bar(i), parity, abort_flag, code));
    tc_fence_after();
    return ok;
  };
  auto steps_of = [&](int64_t x) {  // steps of the segment that starts at x
    const int64_t s0 = x % T;
    return (int)min((int64_t)T - s0, x1 - x);
  };

  if (warp == 0) {
    if (lane == 0) {
      // -------------------------------------------------------------- TMA
      KvTiles kt(p);
      int seg = 0, r = 0;
      for (int64_t x = x0; x < x1 && ok; ++seg) {
        const int n = steps_of(x), first = (int)(x % T);
        int hk, J;
        kt.find(p, x / T, hk, J);
        // the previous segment's products have read its K and V
        if (seg > 0 && !(ok = mbar_spin(bar(AF), (seg - 1) & 1, abort_flag, kDevTimeoutMma))) break;
        mbar_expect_tx(bar(TF), 2 * TILE);
        load_tile(base + OFF_K, &tk, bar(TF), 128 * J, hk, kt.b);
        load_tile(base + OFF_V, &tv, bar(TF), 128 * J, hk, kt.b);
        int g = first / NH, h64 = first - g * NH;
        for (int i = 0; i < n; ++i, ++r) {
          const int e = r % NR;
          if (!(ok = mbar_spin(bar(RE + e), ((r / NR) & 1) ^ 1, abort_flag, kDevTimeoutMma))) break;
          const uint32_t dst = base + OFF_RING + e * ENTRY;
          const int h = hk * p.G + g, r0 = 64 * h64;
          const int64_t row = ((int64_t)kt.b * p.H + h) * p.Lpad + r0;
          mbar_expect_tx(bar(RF + e), 2 * HALF + 512);
          load_half(dst, &tq, bar(RF + e), r0, h, kt.b);
          load_half(dst + HALF, &tdo, bar(RF + e), r0, h, kt.b);
          bulk_load(dst + 2 * HALF, p.lse + row, 256, bar(RF + e));
          bulk_load(dst + 2 * HALF + 256, p.delta + row, 256, bar(RF + e));
          if (++h64 == NH) h64 = 0, ++g;
        }
        x += n;
      }
      // no copy may still target shared memory when the CTA exits; the waits
      // ignore the abort flag and share one limit
      const uint64_t deadline = globaltimer_ns() + kWaitLimitNs;
      bool drained = true;
      if (seg > 0) drained = mbar_wait_until(bar(TF), (seg - 1) & 1, deadline);
      for (int n = max(0, r - NR); n < r && drained; ++n)
        drained = mbar_wait_until(bar(RF + n % NR), (n / NR) & 1, deadline);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA
    if (elect_one()) {
      constexpr uint32_t id_s = idesc_bf16_f32(128, 64, false, false), id_a = idesc_bf16_f32(128, 128, false, true);
      const uint32_t dk = sdesc_lo(base + OFF_K, 16), dv = sdesc_lo(base + OFF_V, 16);
      int r = 0, seg = 0;
      // dV and dK of step `at` (the i-th of its segment)
      auto issue_acc = [&](int at, bool first, bool last) {
        const int e = at % NR, g = at & 1;
        if (!(ok = mbar_spin(bar(DS + g), (at >> 1) & 1, abort_flag, kDevTimeoutSoftmax))) return;
        tc_fence_after();
        const uint32_t dq = sdesc_lo(base + OFF_RING + e * ENTRY, BOX), ddo = sdesc_lo(base + OFF_RING + e * ENTRY + HALF, BOX);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {  // queries 16 kk .. of warpgroup kk / 2
          const uint32_t a = 32 * (kk >> 1) + 8 * (kk & 1);
          mma_bf16_ts_lo(tmem + 256, tmem + 128 * g + a, ddo + ((kk * 2048) >> 4), hi, id_a, (!first || kk > 0) ? 1u : 0u);
          mma_bf16_ts_lo(tmem + 384, tmem + 128 * g + 64 + a, dq + ((kk * 2048) >> 4), hi, id_a,
                         (!first || kk > 0) ? 1u : 0u);
        }
        mma_commit(bar(RE + e));
        if (last) mma_commit(bar(AF));
      };
      for (int64_t x = x0; x < x1 && ok; ++seg) {
        const int n = steps_of(x);
        if (!(ok = mbar_spin(bar(TF), seg & 1, abort_flag, kDevTimeoutLoad))) break;
        for (int i = 0; i < n && ok; ++i, ++r) {
          const int e = r % NR, g = r & 1;
          if (!(ok = mbar_spin(bar(RF + e), (r / NR) & 1, abort_flag, kDevTimeoutLoad))) break;
          tc_fence_after();
          const uint32_t dq = sdesc_lo(base + OFF_RING + e * ENTRY, 16), ddo = sdesc_lo(base + OFF_RING + e * ENTRY + HALF, 16);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint32_t ka = ((kk >> 2) * BOX128 + (kk & 3) * 32) >> 4, kb = ((kk >> 2) * BOX + (kk & 3) * 32) >> 4;
            mma_bf16_ss_lo(tmem + 128 * g, dk + ka, hi, dq + kb, hi, id_s, kk > 0 ? 1u : 0u);
          }
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint32_t ka = ((kk >> 2) * BOX128 + (kk & 3) * 32) >> 4, kb = ((kk >> 2) * BOX + (kk & 3) * 32) >> 4;
            mma_bf16_ss_lo(tmem + 128 * g + 64, dv + ka, hi, ddo + kb, hi, id_s, kk > 0 ? 1u : 0u);
          }
          mma_commit(bar(SF + g));
          if (i == 0) {
            // the previous segment's dV and dK have been read
            if (!(ok = mbar_spin(bar(AE), (seg & 1) ^ 1, abort_flag, kDevTimeoutSoftmax))) break;
          } else {
            issue_acc(r - 1, i == 1, false);
          }
        }
        if (ok) issue_acc(r - 1, n == 1, true);
        x += n;
      }
      // every MMA issued has completed before TMEM is freed, also on the abort path
      mma_commit(bar(DRAIN));
      mbar_wait_until(bar(DRAIN), 0, globaltimer_ns() + kWaitLimitNs);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ---------- P^T, dS^T of query columns [32 wg, 32 wg + 32) of every step, then dV and dK of the segment
    const int wg = (warp - 4) >> 2, q = warp & 3;
    const int row = q * 32 + lane;  // key row of the tile = TMEM lane
    const uint32_t lane_off = (uint32_t)(q * 32) << 16;
    const uint64_t sc2 = f2_pack(p.qk_scale, p.qk_scale);
    KvTiles kt(p);
    int r = 0, seg = 0;
    for (int64_t x = x0; x < x1 && ok; ++seg) {
      const int n = steps_of(x);
      const bool begins = x % T == 0, ends = (x + n) % T == 0;
      int hk, J;
      kt.find(p, x / T, hk, J);
      const int tok = 128 * J + row, b = kt.b;
      const bool sel = tok < kt.len;
      for (int i = 0; i < n; ++i, ++r) {
        const int e = r % NR, g = r & 1;
        const uint32_t tS = tmem + lane_off + 128 * g + 32 * wg, tdP = tS + 64;
        // the step's lse and delta (bulk copies) are visible once its load barrier completed
        if (!wait(RF + e, (r / NR) & 1, kDevTimeoutLoad) || !wait(SF + g, (r >> 1) & 1, kDevTimeoutMma)) break;
        const float* lse_s = reinterpret_cast<const float*>(smem1k + OFF_RING + e * ENTRY + 2 * HALF) + 32 * wg;
        const float* dlt_s = lse_s + 64;
        uint32_t sv[32], dv[32];
        tmem_ld32(tS, sv);
        tmem_ld32(tdP, dv);
        tmem_ld_wait();
        uint32_t wp[16], wd[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float2 l2 = *reinterpret_cast<const float2*>(lse_s + 2 * k);
          const float2 d2 = *reinterpret_cast<const float2*>(dlt_s + 2 * k);
          float y0, y1, p0, p1, d0, d1;
          f2_unpack(fma_f32x2(f2_pack(__uint_as_float(sv[2 * k]), __uint_as_float(sv[2 * k + 1])), sc2,
                              f2_pack(-l2.x, -l2.y)),
                    y0, y1);
          p0 = ex2_approx(y0), p1 = ex2_approx(y1);
          f2_unpack(mul_f32x2(f2_pack(p0, p1), add_f32x2(f2_pack(__uint_as_float(dv[2 * k]), __uint_as_float(dv[2 * k + 1])),
                                                         f2_pack(-d2.x, -d2.y))),
                    d0, d1);
          const uint32_t pp = pack_bf2(p0, p1), pd = pack_bf2(d0, d1);
          // by selection: a key row past len[b] may hold anything
          wp[k] = sel ? pp : 0u;
          wd[k] = sel ? pd : 0u;
        }
        tmem_st16(tS, wp);   // packed P^T over the first 16 of this warpgroup's S^T columns
        tmem_st16(tdP, wd);  // packed dS^T over the first 16 of its dP^T columns
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(DS + g));
      }
      if (!wait(AF, seg & 1, kDevTimeoutMma)) break;
      // dV, then dK (scaled by D^-1/2): columns [64 wg, 64 wg + 64)
      const bool whole = begins && ends;
      float* part = p.part + ((int64_t)(2 * blockIdx.x + (begins ? 1 : 0)) * 2 * 128 + row) * 128 + 64 * wg;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int which = c >> 1, col = 32 * (c & 1);
        uint32_t v[32];
        __syncwarp();  // the stores below diverge, the load is warp-collective
        tmem_ld32(tmem + 256 + 128 * which + lane_off + 64 * wg + col, v);
        tmem_ld_wait();
        if (c == 3) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(AE));
        }
        if (!whole) {
          float4* dst = reinterpret_cast<float4*>(part + which * 128 * 128 + col);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            dst[k] = make_float4(__uint_as_float(v[4 * k]), __uint_as_float(v[4 * k + 1]), __uint_as_float(v[4 * k + 2]),
                                 __uint_as_float(v[4 * k + 3]));
        } else if (tok < p.Lk) {
          const float sc = which ? bwd::kSmScale : 1.0f;
          uint4* dst = reinterpret_cast<uint4*>((which ? p.dk : p.dv) + b * p.dkv_sB + hk * p.dkv_sH + tok * p.dkv_sT +
                                                64 * wg + col);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t w4[4];
#pragma unroll
            for (int m = 0; m < 4; ++m)
              w4[m] = pack_bf2(__uint_as_float(v[8 * k + 2 * m]) * sc, __uint_as_float(v[8 * k + 2 * m + 1]) * sc);
            dst[k] = make_uint4(w4[0], w4[1], w4[2], w4[3]);
          }
        }
      }
      x += n;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// One CTA per 16 rows of a key tile: the sum of its segments' partials in order (a
// tile within one run has been stored already), zeros where no key of the tile is valid
__global__ void __launch_bounds__(256) cross_bwd_join_kernel(const CrossBwdParams p, int runs) {
  __shared__ unsigned long long s_sum;
  const int rows16 = (int)(blockIdx.x & 7), tile = (int)(blockIdx.x >> 3);
  const int J = tile % p.NKT, bk = tile / p.NKT, b = bk / p.Hkv, hk = bk - b * p.Hkv;
  const int len = kv_len(p.kv_lens, b, p.Lk);
  const int64_t before = kv_tiles_before(p, b, &s_sum);
  const int64_t tiles = kv_tiles_before(p, p.B, &s_sum);
  const bool any = 128 * J < len;
  const int T = p.G * ((p.Lq + 63) / 64);
  // run c covers the steps [S c / runs, S (c + 1) / runs)
  const int64_t S = tiles * T, t0 = (before + (int64_t)hk * ((len + 127) >> 7) + J) * T, t1 = t0 + T;
  auto run_start = [&](int64_t c) { return S * c / runs; };
  int64_t c0 = 0, c1 = 0;
  if (any) {
    c0 = t0 * runs / S;  // within one of the run of t0
    while (c0 > 0 && run_start(c0) > t0) --c0;
    while (run_start(c0 + 1) <= t0) ++c0;
    c1 = c0;
    while (run_start(c1 + 1) < t1) ++c1;
    if (c0 == c1) return;  // one run: stored
  }
  // 32 threads a row, 4 columns each; dV and dK of two rows a thread, whose loads of a
  // segment go out together (one after the other they took 26 us at 32760 x 512, 40 heads)
  const int row0 = 16 * rows16 + (threadIdx.x >> 5), col = 4 * (threadIdx.x & 31);
  float4 a[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) a[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (any) {
    for (int64_t c = c0; c <= c1; ++c) {
      const int64_t start = run_start(c);
      if (start == run_start(c + 1)) continue;  // an empty run
      const float* part = p.part + ((2 * c + (start <= t0 ? 1 : 0)) * 2 * 128 + row0) * 128 + col;
      float4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const float4*>(part + (128 * (k >> 1) + 8 * (k & 1)) * 128);
#pragma unroll
      for (int k = 0; k < 4; ++k) a[k].x += v[k].x, a[k].y += v[k].y, a[k].z += v[k].z, a[k].w += v[k].w;
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int which = k >> 1, tok = 128 * J + row0 + 8 * (k & 1);
    if (tok >= p.Lk) continue;
    const float sc = which ? bwd::kSmScale : 1.0f;
    *reinterpret_cast<uint2*>((which ? p.dk : p.dv) + b * p.dkv_sB + hk * p.dkv_sH + tok * p.dkv_sT + col) =
        make_uint2(pack_bf2(a[k].x * sc, a[k].y * sc), pack_bf2(a[k].z * sc, a[k].w * sc));
  }
}

// CTAs of the dk/dv kernel: one per SM, with 8 steps or more each (fewer do not
// pay for a segment's ends)
int cross_bwd_runs(int B, int H, int Hkv, int Lq, int Lk) {
  const int64_t steps = (int64_t)B * Hkv * ((Lk + 127) / 128) * (H / Hkv) * ((Lq + 63) / 64);
  const int64_t runs = (steps + 7) / 8;
  const int sms = device_sms();
  return (int)(runs < sms ? runs : sms);
}

int launch_cross_attn_bwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdo,
                          const CUtensorMap& tdq, const CrossBwdParams& p, cudaStream_t s) {
  static KernelReady ready_dq, ready_dkdv;
  int rc = kernel_ready(ready_dq, cross_bwd_dq_tcgen05, xdq::SMEM, xdq::LAUNCH_REGS);
  if (rc == 0) rc = kernel_ready(ready_dkdv, cross_bwd_dkdv_tcgen05, xkv::SMEM);
  if (rc != 0) return rc;
  cudaError_t e;
  const int64_t items = (int64_t)p.NQT * p.B * p.H;
  const int sms = device_sms();
  cross_bwd_dq_tcgen05<<<(unsigned)(items < sms ? items : sms), xdq::THREADS, xdq::SMEM, s>>>(tq, tk, tv, tdo, tdq, p);
  if ((e = cudaGetLastError()) != cudaSuccess) return (int)e;
  cross_bwd_dkdv_tcgen05<<<p.runs, xkv::THREADS, xkv::SMEM, s>>>(tq, tk, tv, tdo, p);
  if ((e = cudaGetLastError()) != cudaSuccess) return (int)e;
  cross_bwd_join_kernel<<<(unsigned)((int64_t)p.NKT * p.B * p.Hkv * 8), 256, 0, s>>>(p, p.runs);
  return (int)cudaGetLastError();
}

}  // namespace rola
