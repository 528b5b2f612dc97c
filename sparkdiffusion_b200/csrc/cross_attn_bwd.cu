// Backward of the attention to another sequence's states (cross_attn.cu), on
// tcgen05, without atomics.  From the forward's base-2 log-sum-exp:
//
//   delta[i] = sum_d dO[i, d] O[i, d]   (by the way, in the dq kernel, which has dO)
//   P  = exp2(q.k D^-1/2 log2(e) - lse[i])             (recomputed, fp32; 0 past len[b])
//   dP = dO V^T,  dS = P (dP - delta[i])
//   dQ = D^-1/2 dS K                    query-stationary   (cross_bwd_dq_tcgen05)
//   dV = P^T dO,  dK = D^-1/2 dS^T Q    key-stationary     (cross_bwd_dkdv_tcgen05)
//
// P and dS are rounded to bf16 where they feed a product; sums are fp32 in
// tensor memory.  dK and dV of a key head sum over its G query heads: the key
// tile stays and the steps walk the rows of all of them.  An encoder's states
// are few key tiles and many query rows, so the rows of one key tile are cut
// into slices (one CTA each) that leave fp32 partials, added in slice order.
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
// steps of 512 keys (1.06 ms at 32760 x 512, 40 heads).
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
        int om[NT], oh[NT], ob[NT];
        auto store_out = [&](int e, int n) {
          if (!mbar_spin(bar(TE + e), n & 1, abort_flag, kDevTimeoutSoftmax)) return false;
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
      if (!wait(TF + e, (j / NT) & 1, kDevTimeoutLoad)) break;
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
      if (!wait(DR + j % NT, (j / NT) & 1, kDevTimeoutSoftmax)) break;
      const float dlt = reinterpret_cast<const float*>(smem1k + OFF_DELTA)[(j % NT) * 128 + row];
      const uint64_t nl2 = f2_pack(-lse, -lse), nd2 = f2_pack(-dlt, -dlt);
      for (int i = 0; i < cnt; ++i, ++u) {
        if (u % NS != g) continue;
        if (!wait(SF + g, ph, kDevTimeoutMma)) break;
        const int valid = len - 64 * i;
#pragma unroll
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
// dk, dv: one CTA per (128-row key tile, b, key head, slice of the query rows);
// steps of 64 query rows, both softmax warpgroups on every step (32 columns each)
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(bwd::THREADS, 1)
    cross_bwd_dkdv_tcgen05(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                           const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tdo,
                           const CrossBwdParams p) {
  using namespace bwd;
  extern __shared__ __align__(1024) uint8_t smem1k[];
  const uint32_t base = smem_u32(smem1k);
  const uint32_t bars = base + KV_OFF_BAR;
  auto bar = [&](int i) { return bars + 8u * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem1k + KV_OFF_BAR + 8 * G_COUNT);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem1k + KV_OFF_BAR + 8 * G_COUNT + 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // slices of one key tile are neighbours
  const int split = (int)(blockIdx.x % p.nsplit);
  const int64_t rest = blockIdx.x / p.nsplit;
  const int J = (int)(rest % p.NKT), bk = (int)(rest / p.NKT), b = bk / p.Hkv, hk = bk % p.Hkv;
  const int len = kv_len(p.kv_lens, b, p.Lk);
  if (128 * J >= len) {  // no valid key (uniform over the CTA)
    if (p.nsplit == 1 && threadIdx.x < 256) {
      const int tok = 128 * J + (threadIdx.x >> 1);
      if (tok < p.Lk) {
        const int64_t off = b * p.dkv_sB + hk * p.dkv_sH + tok * p.dkv_sT + 64 * (threadIdx.x & 1);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          reinterpret_cast<uint4*>(p.dk + off)[c] = make_uint4(0u, 0u, 0u, 0u);
          reinterpret_cast<uint4*>(p.dv + off)[c] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
    }
    return;
  }
  const int NH = (p.Lq + 63) / 64;  // steps per query head
  const int64_t T = (int64_t)p.G * NH;
  const int first = (int)(T * split / p.nsplit), n = (int)(T * (split + 1) / p.nsplit) - first;

  if (threadIdx.x == 0) {
    mbar_init(bar(G_TILE), 1);
    for (int s = 0; s < KV_STAGES; ++s) {
      mbar_init(bar(G_FULL0 + s), 1);
      mbar_init(bar(G_EMPTY0 + s), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar(G_SF0 + t), 1);
      mbar_init(bar(G_DS0 + t), 8);
    }
    mbar_init(bar(G_ACC), 1);
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
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------------ TMA
      mbar_expect_tx(bar(G_TILE), 2 * TILE);
      load_tile(base + KV_OFF_K, &tk, bar(G_TILE), 128 * J, hk, b);
      load_tile(base + KV_OFF_V, &tv, bar(G_TILE), 128 * J, hk, b);
      for (int i = 0; i < n; ++i) {
        const int s = i % KV_STAGES;
        if (!mbar_wait(bar(G_EMPTY0 + s), ((i / KV_STAGES) & 1) ^ 1, abort_flag, kDevTimeoutMma)) break;
        const uint32_t dst = base + KV_OFF_RING + s * KV_ENTRY;
        mbar_expect_tx(bar(G_FULL0 + s), 2 * HALF + 512);
        const int h = hk * p.G + (first + i) / NH, r0 = 64 * ((first + i) % NH);
        const int64_t row = ((int64_t)b * p.H + h) * p.Lpad + r0;
        load_half(dst, &tq, bar(G_FULL0 + s), r0, h, b);
        load_half(dst + HALF, &tdo, bar(G_FULL0 + s), r0, h, b);
        bulk_load(dst + 2 * HALF, p.lse + row, 256, bar(G_FULL0 + s));
        bulk_load(dst + 2 * HALF + 256, p.delta + row, 256, bar(G_FULL0 + s));
      }
      const uint64_t deadline = globaltimer_ns() + kWaitLimitNs;
      bool drained = mbar_wait_until(bar(G_TILE), 0, deadline);
      for (int i = max(0, n - KV_STAGES); i < n && drained; ++i)
        drained = mbar_wait_until(bar(G_FULL0 + i % KV_STAGES), (i / KV_STAGES) & 1, deadline);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA
    if (elect_one()) {
      const uint32_t id_s = idesc_bf16_f32(128, 64, false, false);
      const uint32_t id_a = idesc_bf16_f32(128, 128, false, true);
      bool ok = mbar_wait(bar(G_TILE), 0, abort_flag, kDevTimeoutLoad);
      auto issue_acc = [&](int i) {
        if (!mbar_wait(bar(G_DS0 + (i & 1)), (i >> 1) & 1, abort_flag, kDevTimeoutSoftmax)) {
          ok = false;
          return;
        }
        tc_fence_after();
        const uint32_t sq = base + KV_OFF_RING + (i % KV_STAGES) * KV_ENTRY, sdo = sq + HALF;
        const uint32_t tb = tmem + 128 * (i & 1);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {  // dV += P^T dO, dK += dS^T Q; queries 16 kk.. of warpgroup kk / 2
          const uint32_t a = 32 * (kk >> 1) + 8 * (kk & 1);
          mma_bf16_ts(tmem + 256, tb + a, sdesc_sw128(sdo + kk * 2048, BOX, 1024), id_a, (i > 0 || kk > 0) ? 1u : 0u);
          mma_bf16_ts(tmem + 384, tb + 64 + a, sdesc_sw128(sq + kk * 2048, BOX, 1024), id_a,
                      (i > 0 || kk > 0) ? 1u : 0u);
        }
        mma_commit(bar(G_EMPTY0 + i % KV_STAGES));
      };
      for (int i = 0; i < n && ok; ++i) {
        const int s = i % KV_STAGES;
        if (!mbar_wait(bar(G_FULL0 + s), (i / KV_STAGES) & 1, abort_flag, kDevTimeoutLoad)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t sq = base + KV_OFF_RING + s * KV_ENTRY, sdo = sq + HALF;
        const uint32_t tb = tmem + 128 * (i & 1);
        mma_step_ss(tb, base + KV_OFF_K, sq, id_s);        // S^T  = K Q^T
        mma_step_ss(tb + 64, base + KV_OFF_V, sdo, id_s);  // dP^T = V dO^T
        mma_commit(bar(G_SF0 + (i & 1)));
        if (i > 0) issue_acc(i - 1);
      }
      if (ok && n > 0) issue_acc(n - 1);
      mma_commit(bar(G_ACC));
      // every MMA issued has completed before TMEM is freed, also on the abort path
      mbar_wait_until(bar(G_ACC), 0, globaltimer_ns() + kWaitLimitNs);
    }
  } else if (warp >= 4) {
    // ---------- P^T, dS^T of query columns [32 wg, 32 wg + 32) of every step, then the dK/dV epilogue
    const int wg = (warp - 4) >> 2;
    const int q = warp & 3;
    const int r = q * 32 + lane;  // key row of the tile = TMEM lane
    const int tok = 128 * J + r;
    const bool sel = tok < len;
    const uint32_t lane_off = (uint32_t)(q * 32) << 16;
    const uint64_t sc2 = f2_pack(p.qk_scale, p.qk_scale);
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int s = i % KV_STAGES;
      const uint32_t tS = tmem + lane_off + 128 * (i & 1) + 32 * wg, tdP = tS + 64;
      bool got = mbar_wait(bar(G_SF0 + (i & 1)), (i >> 1) & 1, abort_flag, kDevTimeoutMma);
      // the step's lse / delta (bulk copies) are visible once its load barrier completed
      got = got && mbar_wait(bar(G_FULL0 + s), (i / KV_STAGES) & 1, abort_flag, kDevTimeoutLoad);
      if (!__all_sync(0xffffffffu, got)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const float* lse_s = reinterpret_cast<const float*>(smem1k + KV_OFF_RING + s * KV_ENTRY + 2 * HALF) + 32 * wg;
      const float* dlt_s = lse_s + 64;
      uint32_t sv[32], dv[32];
      tmem_ld32(tS, sv);
      tmem_ld32(tdP, dv);
      tmem_ld_wait();
      uint32_t wp[16], wd[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float2 l2 = *reinterpret_cast<const float2*>(lse_s + 2 * e);
        const float2 d2 = *reinterpret_cast<const float2*>(dlt_s + 2 * e);
        float x0, x1;
        f2_unpack(fma_f32x2(f2_pack(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), sc2,
                            f2_pack(-l2.x, -l2.y)),
                  x0, x1);
        const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
        const uint32_t pp = pack_bf2(p0, p1);
        const uint32_t pd = pack_bf2(p0 * (__uint_as_float(dv[2 * e]) - d2.x), p1 * (__uint_as_float(dv[2 * e + 1]) - d2.y));
        wp[e] = sel ? pp : 0u;
        wd[e] = sel ? pd : 0u;
      }
      tmem_st16(tS, wp);   // packed P^T over the first 16 of this warpgroup's S^T columns
      tmem_st16(tdP, wd);  // packed dS^T over the first 16 of its dP^T columns
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(G_DS0 + (i & 1)));
    }
    if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait(bar(G_ACC), 0, abort_flag, kDevTimeoutMma));
    tc_fence_after();
    if (ok) {
#pragma unroll
      for (int which = 0; which < 2; ++which) {  // dV, then dK (scaled by D^-1/2)
        const float sc = which ? kSmScale : 1.0f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t v[32];
          __syncwarp();  // the stores below diverge, the load is warp-collective
          if (n > 0) {
            tmem_ld32(tmem + 256 + 128 * which + lane_off + 64 * wg + 32 * c, v);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0u;
          }
          if (p.nsplit > 1) {
            const int64_t row = (((int64_t)which * p.nsplit + split) * p.B * p.Hkv + bk) * (128ll * p.NKT) + tok;
            float4* dst = reinterpret_cast<float4*>(p.part + row * 128 + 64 * wg + 32 * c);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              dst[e] = make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]),
                                   __uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3]));
          } else if (tok < p.Lk) {
            uint4* dst = reinterpret_cast<uint4*>((which ? p.dk : p.dv) + b * p.dkv_sB + hk * p.dkv_sH + tok * p.dkv_sT +
                                                  64 * wg + 32 * c);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t w4[4];
#pragma unroll
              for (int j = 0; j < 4; ++j)
                w4[j] = pack_bf2(__uint_as_float(v[8 * e + 2 * j]) * sc, __uint_as_float(v[8 * e + 2 * j + 1]) * sc);
              dst[e] = make_uint4(w4[0], w4[1], w4[2], w4[3]);
            }
          }
        }
      }
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

// dk, dv = sum over the slices in order (0 past len[b]); one thread per 4 columns of a key
__global__ void __launch_bounds__(256) cross_bwd_join_kernel(const CrossBwdParams p) {
  const int64_t g = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int c = (int)(g & 31);
  int64_t r = g >> 5;
  const int tok = (int)(r % p.Lk);
  r /= p.Lk;
  const int64_t BHk = (int64_t)p.B * p.Hkv;
  const int64_t bk = r % BHk;
  const int which = (int)(r / BHk);
  if (which >= 2) return;
  const int b = (int)(bk / p.Hkv), hk = (int)(bk % p.Hkv);
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (tok < kv_len(p.kv_lens, b, p.Lk)) {
    const int64_t step = BHk * 128ll * p.NKT * 128;
    const float* src = p.part + ((which * p.nsplit * BHk + bk) * (128ll * p.NKT) + tok) * 128 + 4 * c;
    for (int s = 0; s < p.nsplit; ++s) {
      const float4 v = *reinterpret_cast<const float4*>(src + s * step);
      a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
    }
  }
  const float sc = which ? bwd::kSmScale : 1.0f;
  *reinterpret_cast<uint2*>((which ? p.dk : p.dv) + b * p.dkv_sB + hk * p.dkv_sH + tok * p.dkv_sT + 4 * c) =
      make_uint2(pack_bf2(a.x * sc, a.y * sc), pack_bf2(a.z * sc, a.w * sc));
}

// Slices of the query rows per key tile: the count (at most 12) whose waves of
// CTAs waste least, with 16 steps of 64 rows or more in each
int cross_bwd_splits(int B, int H, int Hkv, int Lq, int Lk) {
  const int64_t tiles = (int64_t)B * Hkv * ((Lk + 127) / 128);
  const int64_t steps = (int64_t)(H / Hkv) * ((Lq + 63) / 64);
  const int sms = device_sms();
  int best = 1;
  double cost = 1e30;
  for (int s = 1; s <= 12 && (s == 1 || steps / s >= 16); ++s) {
    const double waves = (double)((tiles * s + sms - 1) / sms) / s;
    if (waves < cost * 0.97) {
      cost = waves;
      best = s;
    }
  }
  return best;
}

int launch_cross_attn_bwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdo,
                          const CUtensorMap& tdq, const CrossBwdParams& p, cudaStream_t s) {
  using namespace bwd;
  static KernelReady ready_dq, ready_dkdv;
  int rc = kernel_ready(ready_dq, cross_bwd_dq_tcgen05, xdq::SMEM, xdq::LAUNCH_REGS);
  if (rc == 0) rc = kernel_ready(ready_dkdv, cross_bwd_dkdv_tcgen05, KV_SMEM);
  if (rc != 0) return rc;
  cudaError_t e;
  const int64_t items = (int64_t)p.NQT * p.B * p.H;
  const int sms = device_sms();
  cross_bwd_dq_tcgen05<<<(unsigned)(items < sms ? items : sms), xdq::THREADS, xdq::SMEM, s>>>(tq, tk, tv, tdo, tdq, p);
  if ((e = cudaGetLastError()) != cudaSuccess) return (int)e;
  cross_bwd_dkdv_tcgen05<<<(unsigned)((int64_t)p.NKT * p.B * p.Hkv * p.nsplit), THREADS, KV_SMEM, s>>>(tq, tk, tv, tdo,
                                                                                                  p);
  if ((e = cudaGetLastError()) != cudaSuccess) return (int)e;
  if (p.nsplit > 1) {
    const int64_t threads = 2ll * p.B * p.Hkv * p.Lk * 32;
    cross_bwd_join_kernel<<<(unsigned)((threads + 255) / 256), 256, 0, s>>>(p);
  }
  return (int)cudaGetLastError();
}

}  // namespace rola
