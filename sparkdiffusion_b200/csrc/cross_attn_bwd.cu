// Backward of the attention to another sequence's states (cross_attn.cu), on
// tcgen05, without atomics.  From the forward's base-2 log-sum-exp:
//
//   delta[i] = sum_d dO[i, d] O[i, d]                  (attn_bwd_delta_kernel)
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
// dq: one CTA per (128-row query tile, b, h); steps of 64 keys
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(bwd::DQ_THREADS, 1)
    cross_bwd_dq_tcgen05(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                         const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tdo,
                         const CrossBwdParams p) {
  using namespace bwd;
  extern __shared__ __align__(1024) uint8_t smem1k[];
  const uint32_t base = smem_u32(smem1k);
  const uint32_t bars = base + DQ_OFF_BAR;
  auto bar = [&](int i) { return bars + 8u * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem1k + DQ_OFF_BAR + 8 * G_COUNT);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem1k + DQ_OFF_BAR + 8 * G_COUNT + 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m = (int)(blockIdx.x % p.NQT), bh = (int)(blockIdx.x / p.NQT), b = bh / p.H, h = bh % p.H;
  const int len = kv_len(p.kv_lens, b, p.Lk);
  const int n = (len + 63) / 64;

  if (threadIdx.x == 0) {
    mbar_init(bar(G_TILE), 1);
    for (int s = 0; s < DQ_STAGES; ++s) {
      mbar_init(bar(G_FULL0 + s), 1);
      mbar_init(bar(G_EMPTY0 + s), 1);
    }
    for (int t = 0; t < DQ_NBUF; ++t) {
      mbar_init(bar(G_SF0 + t), 1);
      mbar_init(bar(G_DS0 + t), 4);
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
    if (lane == 0 && n > 0) {
      // ------------------------------------------------------------ TMA
      mbar_expect_tx(bar(G_TILE), 2 * TILE);
      load_tile(base + DQ_OFF_Q, &tq, bar(G_TILE), 128 * m, h, b);
      load_tile(base + DQ_OFF_DO, &tdo, bar(G_TILE), 128 * m, h, b);
      for (int i = 0; i < n; ++i) {
        const int s = i % DQ_STAGES;
        if (!mbar_wait(bar(G_EMPTY0 + s), ((i / DQ_STAGES) & 1) ^ 1, abort_flag, kDevTimeoutMma)) break;
        const uint32_t dst = base + DQ_OFF_RING + s * DQ_ENTRY;
        mbar_expect_tx(bar(G_FULL0 + s), 2 * HALF);
        load_half(dst, &tk, bar(G_FULL0 + s), 64 * i, h / p.G, b);
        load_half(dst + HALF, &tv, bar(G_FULL0 + s), 64 * i, h / p.G, b);
      }
      // no TMA may still target shared memory when the CTA exits
      const uint64_t deadline = globaltimer_ns() + kWaitLimitNs;
      bool drained = mbar_wait_until(bar(G_TILE), 0, deadline);
      for (int i = max(0, n - DQ_STAGES); i < n && drained; ++i)
        drained = mbar_wait_until(bar(G_FULL0 + i % DQ_STAGES), (i / DQ_STAGES) & 1, deadline);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA
    // S_i, dP_i, then dQ += dS_{i-2} K_{i-2}: the tensor core computes step i
    // while steps i-2 and i-1 are in the softmax.  The whole warp follows (it
    // clears K rows together), lane 0 issues.
    const uint32_t id_s = idesc_bf16_f32(128, 64, false, false);
    const uint32_t id_q = idesc_bf16_f32(128, 128, false, true);
    bool ok = true;
    auto wait = [&](int i, uint32_t parity, int code) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(i), parity, abort_flag, code));
      tc_fence_after();
      return ok;
    };
    if (n > 0) wait(G_TILE, 0, kDevTimeoutLoad);
    auto issue_dq = [&](int i) {
      if (!wait(G_DS0 + i % DQ_NBUF, (i / DQ_NBUF) & 1, kDevTimeoutSoftmax)) return;
      const int off = DQ_OFF_RING + (i % DQ_STAGES) * DQ_ENTRY;
      if (len - 64 * i < 64 && len < p.Lk) clear_half_rows(smem1k + off, len - 64 * i, lane);
      if (lane == 0) {
        mma_step_ts(tmem + DQ_ACC, tmem + 128 * (i % DQ_NBUF), base + off, id_q, i > 0);  // dQ += dS K
        mma_commit(bar(G_EMPTY0 + i % DQ_STAGES));
      }
      __syncwarp();
    };
    for (int i = 0; i < n && ok; ++i) {
      const int s = i % DQ_STAGES;
      if (!wait(G_FULL0 + s, (i / DQ_STAGES) & 1, kDevTimeoutLoad)) break;
      if (lane == 0) {
        const uint32_t sk = base + DQ_OFF_RING + s * DQ_ENTRY, sv = sk + HALF;
        const uint32_t tb = tmem + 128 * (i % DQ_NBUF);
        mma_step_ss(tb, base + DQ_OFF_Q, sk, id_s);        // S  = Q K^T
        mma_step_ss(tb + 64, base + DQ_OFF_DO, sv, id_s);  // dP = dO V^T
        mma_commit(bar(G_SF0 + i % DQ_NBUF));
      }
      __syncwarp();
      if (i >= DQ_NBUF - 1) issue_dq(i - (DQ_NBUF - 1));
    }
    for (int i = max(0, n - (DQ_NBUF - 1)); i < n && ok; ++i) issue_dq(i);
    if (lane == 0) {
      mma_commit(bar(G_ACC));
      // every MMA issued has completed before TMEM is freed, also on the abort path
      mbar_wait_until(bar(G_ACC), 0, globaltimer_ns() + kWaitLimitNs);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // -------------------------------------- dS of every third step, then the dQ epilogue
    const int wg = (warp - 4) >> 2;
    const int q = warp & 3;
    const int r = q * 32 + lane;  // query row of the tile = TMEM lane
    const uint32_t lane_off = (uint32_t)(q * 32) << 16;
    const uint32_t tS = tmem + lane_off + 128 * wg, tdP = tS + 64;
    const int tok = 128 * m + r;
    const float lse = p.lse[(int64_t)bh * p.Lpad + tok];
    const float dlt = p.delta[(int64_t)bh * p.Lpad + tok];
    const uint64_t sc2 = f2_pack(p.qk_scale, p.qk_scale), nl2 = f2_pack(-lse, -lse);
    bool ok = true;
    for (int i = wg; i < n; i += DQ_NBUF) {
      if (!__all_sync(0xffffffffu, mbar_wait(bar(G_SF0 + wg), (i / DQ_NBUF) & 1, abort_flag, kDevTimeoutMma))) {
        ok = false;
        break;
      }
      tc_fence_after();
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
          const int col = 32 * c + 2 * e;
          float x0, x1;
          f2_unpack(fma_f32x2(f2_pack(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), sc2, nl2), x0, x1);
          const float d0 = ex2_approx(x0) * (__uint_as_float(dv[2 * e]) - dlt);
          const float d1 = ex2_approx(x1) * (__uint_as_float(dv[2 * e + 1]) - dlt);
          w[e] = pack_bf2(col < valid ? d0 : 0.f, col + 1 < valid ? d1 : 0.f);
        }
        tmem_st16(tS + 16 * c, w);  // packed dS over the first 32 S columns of the buffer
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(G_DS0 + wg));
    }
    if (wg == 2) ok = false;  // the third warpgroup has no epilogue columns
    if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait(bar(G_ACC), 0, abort_flag, kDevTimeoutMma));
    tc_fence_after();
    if (ok) {
      const uint32_t tQ = tmem + DQ_ACC + lane_off + 64 * wg;
      uint32_t v[64];
      if (n > 0) {
        tmem_ld32(tQ, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
        tmem_ld32(tQ + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int e = 0; e < 64; ++e) v[e] = 0u;  // no keys
      }
      if (tok < p.Lq) {
        uint4* dst = reinterpret_cast<uint4*>(p.dq + b * p.dq_sB + h * p.dq_sH + tok * p.dq_sT + 64 * wg);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t w4[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w4[e] = pack_bf2(__uint_as_float(v[8 * c + 2 * e]) * kSmScale, __uint_as_float(v[8 * c + 2 * e + 1]) * kSmScale);
          dst[c] = make_uint4(w4[0], w4[1], w4[2], w4[3]);
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
                          const CrossBwdParams& p, cudaStream_t s) {
  using namespace bwd;
  static KernelReady ready_dq, ready_dkdv;
  int rc = kernel_ready(ready_dq, cross_bwd_dq_tcgen05, DQ_SMEM);
  if (rc == 0) rc = kernel_ready(ready_dkdv, cross_bwd_dkdv_tcgen05, KV_SMEM);
  if (rc != 0) return rc;
  cudaError_t e;
  cross_bwd_dq_tcgen05<<<(unsigned)((int64_t)p.NQT * p.B * p.H), DQ_THREADS, DQ_SMEM, s>>>(tq, tk, tv, tdo, p);
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
