// Attention to the states of another sequence (tcgen05): query rows i of head h
// attend to the keys j < len[b] of key head h / G,
//
//   o_i = sum_j softmax_j(q_i . k_j D^-1/2) v_j,      D = 128,
//
// a row without keys is 0.  Online softmax in base 2: running maximum m and sum
// l in fp32, P = exp2(s - m) rounded to bf16 for the second product, O in fp32.
// O is rescaled only when a row's maximum has grown by more than 2^8: until
// then P and l share the older maximum (the quotient is the same, P is at most
// 2^8 and rounds with the same relative error).
//
// Work items are (pair of 128-row query tiles, batch and head, slice of the
// keys); persistent CTAs, one per SM, walk them.  An encoder's states are few
// keys (512: four tiles), so an item is short and its ends must overlap its
// neighbours: the tiles' S products of the next item are issued right behind the
// last P V of this one, its Q tiles are loaded ahead through a ring of three,
// and the correction warps store an item's output while the next item's softmax
// runs.  Both query tiles of an item use each K and V tile once it is in shared
// memory (half the L2 reads of one tile per K/V load).  Roles (512 threads,
// registers split by setmaxnreg):
//   warp 0          TMA producer: Q ring (3 x 32 KB), K/V ring (4 x 32 KB)
//   warp 1          MMA issuer and TMEM owner: S = Q K^T (shared memory), O += P V
//                   (P in TMEM over the S columns, in chunks of 32 keys).  It also
//                   clears the V rows past len[b] (their P is 0, but 0 * NaN is not)
//   warps 4-7, 8-11 softmax of tile 0 / 1, thread = row = TMEM lane
//   warps 12-15     rescale O, then scale by 1/l and store
// Few rows: the keys of an item are cut into slices, each leaves O/l in fp32 and
// its log-sum-exp, and combine_kernel joins them.  When the G query heads of a
// key head have 128 rows or fewer together, they form one tile (one read of K/V
// for all of them).
#include "common.cuh"
#include "kernels.h"

namespace rola {

namespace xattn {
constexpr int THREADS = 512;
constexpr int LAUNCH_REGS = 128;  // 65536 / 512
constexpr int REGS_LOAD = 56, REGS_CORR = 96, REGS_SOFTMAX = 176;
static_assert(128 * (REGS_LOAD + REGS_CORR + 2 * REGS_SOFTMAX) <= THREADS * LAUNCH_REGS, "register split");
constexpr int BOX = 16384;        // [128 rows x 64 bf16], 128-byte swizzle
constexpr int TILE = 2 * BOX;     // 128 rows x 128 columns
constexpr int NQ = 3, NKV = 4;
constexpr int OFF_Q = 0;
constexpr int OFF_KV = NQ * TILE;
constexpr int OFF_ALPHA = OFF_KV + NKV * TILE;  // [2][128] rescale factors
constexpr int OFF_L = OFF_ALPHA + 1024;         // [2][128] row sums
constexpr int OFF_BAR = OFF_L + 1024;
constexpr int SMEM = OFF_BAR + 512;
constexpr float RESCALE = 8.0f;   // log2 growth of the maximum that triggers a rescale of O
enum : int {
  QF = 0, QE = QF + NQ, KF = QE + NQ, KE = KF + NKV,
  SF = KE + NKV,   // S of tile t in TMEM
  PF = SF + 2,     // P chunk c of tile t in TMEM: PF + 4 t + c, 4 warp arrivals
  OF = PF + 8,     // O of tile t final
  AR = OF + 2,     // rescale factors of tile t published (each step), 4 arrivals
  LF = AR + 2,     // row sums of tile t published (end of item), 4 arrivals
  OC = LF + 2,     // O of tile t may be accumulated into, 4 arrivals
  DRAIN = OC + 2,
  COUNT
};
static_assert(8 * COUNT + 16 <= 512, "barrier region");
static_assert(SMEM <= 227 * 1024, "shared memory");
}  // namespace xattn

// valid keys of batch b
__device__ __forceinline__ int kv_len(const int32_t* lens, int b, int Lk) {
  return lens ? min(max(lens[b], 0), Lk) : Lk;
}

struct CrossItem {
  int b, h, m0, nt, i0, cnt, split;  // h: head of the grid (key head when packed); key tiles [i0, i0 + cnt)
  int len;
};
__device__ __forceinline__ CrossItem cross_item(const CrossAttnParams& p, int64_t w) {
  CrossItem it;
  const int qp = (int)(w % p.nqp);
  int64_t r = w / p.nqp;
  it.split = (int)(r % p.nsplit);
  r /= p.nsplit;
  it.h = (int)(r % p.Hgrid);
  it.b = (int)(r / p.Hgrid);
  it.m0 = 2 * qp;
  it.nt = min(2, p.nqt - it.m0);
  it.len = kv_len(p.kv_lens, it.b, p.Lk);
  const int n = (it.len + 127) / 128;
  it.i0 = (int)((int64_t)n * it.split / p.nsplit);
  it.cnt = (int)((int64_t)n * (it.split + 1) / p.nsplit) - it.i0;
  return it;
}
// row r of tile m -> head and token; false past the last row
__device__ __forceinline__ bool cross_row(const CrossAttnParams& p, const CrossItem& it, int m, int r, int& h, int& t) {
  if (p.pack) {
    const int g = r / p.Lq;
    h = it.h * p.G + g;
    t = r - g * p.Lq;
    return g < p.G;
  }
  h = it.h;
  t = m * 128 + r;
  return t < p.Lq;
}

// shared memory row r >= valid of a [128 x 128] V tile := 0 (whole 128-byte rows, so the swizzle does not matter)
__device__ __forceinline__ void clear_rows(uint8_t* tile, int valid, int lane) {
  for (int i = valid * 8 + lane; i < 128 * 8; i += 32) {
    *reinterpret_cast<uint4*>(tile + i * 16) = make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4*>(tile + xattn::BOX + i * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

__global__ void __launch_bounds__(xattn::THREADS, 1)
    cross_attn_tcgen05(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                       const __grid_constant__ CUtensorMap tv, const CrossAttnParams p) {
  using namespace xattn;
  extern __shared__ __align__(1024) uint8_t smem1k[];
  const uint32_t base = smem_u32(smem1k);
  auto bar = [&](int i) { return base + OFF_BAR + 8u * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem1k + OFF_BAR + 8 * COUNT);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem1k + OFF_BAR + 8 * COUNT + 8);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < COUNT; ++i) mbar_init(bar(i), (i >= PF && i < OF) || (i >= AR && i < DRAIN) ? 4 : 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tq);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t id_qk = idesc_bf16_f32(128, 128, false, false);
  const uint32_t id_pv = idesc_bf16_f32(128, 128, false, true);

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_LOAD));
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------------ TMA
      int rq = 0, r = 0;
      bool ok = true;
      auto load_q = [&](const CrossItem& it, int t) {
        const int e = rq % NQ;
        if (!ok || !(ok = mbar_wait(bar(QE + e), ((rq / NQ) & 1) ^ 1, abort_flag, kDevTimeoutMma))) return;
        const uint32_t dst = base + OFF_Q + e * TILE;
        const int h = p.pack ? it.h * p.G : it.h;
        mbar_expect_tx(bar(QF + e), p.q_bytes);
        tma_load_4d(dst, &tq, bar(QF + e), 0, (it.m0 + t) * 128, h, it.b);
        tma_load_4d(dst + BOX, &tq, bar(QF + e), 64, (it.m0 + t) * 128, h, it.b);
        ++rq;
      };
      auto load_kv = [&](const CUtensorMap* m, const CrossItem& it, int i) {
        const int e = r % NKV;
        if (!ok || !(ok = mbar_wait(bar(KE + e), ((r / NKV) & 1) ^ 1, abort_flag, kDevTimeoutMma))) return;
        const uint32_t dst = base + OFF_KV + e * TILE;
        const int h = p.pack ? it.h : it.h / p.G;
        mbar_expect_tx(bar(KF + e), TILE);
        tma_load_4d(dst, m, bar(KF + e), 0, i * 128, h, it.b);
        tma_load_4d(dst + BOX, m, bar(KF + e), 64, i * 128, h, it.b);
        ++r;
      };
      for (int64_t w = blockIdx.x; w < p.items && ok; w += gridDim.x) {
        const CrossItem it = cross_item(p, w);
        if (it.cnt == 0) continue;
        load_q(it, 0);
        load_kv(&tk, it, it.i0);
        if (it.nt == 2) load_q(it, 1);
        for (int i = 0; i < it.cnt && ok; ++i) {
          load_kv(&tv, it, it.i0 + i);
          if (i + 1 < it.cnt) load_kv(&tk, it, it.i0 + i + 1);
        }
      }
      // no copy may still target shared memory when the CTA exits; the waits
      // ignore the abort flag and share one limit
      const uint64_t deadline = globaltimer_ns() + kWaitLimitNs;
      bool drained = true;
      for (int n = max(0, rq - NQ); n < rq && drained; ++n)
        drained = mbar_wait_until(bar(QF + n % NQ), (n / NQ) & 1, deadline);
      for (int n = max(0, r - NKV); n < r && drained; ++n)
        drained = mbar_wait_until(bar(KF + n % NKV), (n / NKV) & 1, deadline);
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMA
      // the whole warp follows the sequence (it clears V rows together); lane 0 issues
      int rq = 0, r = 0;
      int steps[2] = {0, 0};
      bool ok = true;
      auto wait = [&](int i, uint32_t parity, int code) {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(i), parity, abort_flag, code));
        tc_fence_after();
        return ok;
      };
      auto next_item = [&](int64_t& w, CrossItem& it) {
        for (; w < p.items; w += gridDim.x) {
          it = cross_item(p, w);
          if (it.cnt > 0) {
            w += gridDim.x;
            return true;
          }
        }
        return false;
      };
      // S_t = Q_t K^T with Q ring entry eq and K ring entry ek
      auto issue_s = [&](int t, int eq, int ek, bool last_of_q, bool last_of_k) {
        if (lane == 0) {
          const uint32_t sq = base + OFF_Q + eq * TILE, sk = base + OFF_KV + ek * TILE;
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint32_t off = (kk >> 2) * BOX + (kk & 3) * 32;
            mma_bf16_ss(tmem + 128 * t, sdesc_sw128(sq + off, 16, 1024), sdesc_sw128(sk + off, 16, 1024), id_qk,
                        kk > 0 ? 1u : 0u);
          }
          mma_commit(bar(SF + t));
          if (last_of_q) mma_commit(bar(QE + eq));
          if (last_of_k) mma_commit(bar(KE + ek));
        }
        __syncwarp();
      };
      int64_t w = blockIdx.x;
      CrossItem cur, nxt;
      bool have = next_item(w, cur);
      int eq[2] = {0, 0}, eq_next[2] = {0, 0}, ek = 0;
      auto open_item = [&](const CrossItem& it, int t) {  // S_t(0) of an item: its Q tile, and its first K tile once
        if (t == 0) {
          ek = r % NKV;
          if (!wait(KF + ek, (r / NKV) & 1, kDevTimeoutLoad)) return;
          ++r;
        }
        eq_next[t] = rq % NQ;
        if (!wait(QF + eq_next[t], (rq / NQ) & 1, kDevTimeoutLoad)) return;
        ++rq;
        issue_s(t, eq_next[t], ek, it.cnt == 1, t == it.nt - 1);
      };
      if (have)
        for (int t = 0; t < cur.nt && ok; ++t) open_item(cur, t);
      while (have && ok) {
        eq[0] = eq_next[0], eq[1] = eq_next[1];
        const bool more = next_item(w, nxt);
        for (int i = 0; i < cur.cnt && ok; ++i) {
          const bool last = i + 1 == cur.cnt;
          const int ev = r % NKV;
          if (!wait(KF + ev, (r / NKV) & 1, kDevTimeoutLoad)) break;
          ++r;
          const int valid = cur.len - (cur.i0 + i) * 128;
          if (valid < 128 && cur.len < p.Lk) clear_rows(smem1k + OFF_KV + ev * TILE, valid, lane);
          const uint32_t sv = base + OFF_KV + ev * TILE;
          for (int t = 0; t < cur.nt && ok; ++t) {
            const uint32_t ph = steps[t] & 1;
            if (!wait(OC + t, ph, kDevTimeoutSoftmax)) break;
            for (int c = 0; c < 4 && ok; ++c) {
              if (!wait(PF + 4 * t + c, ph, kDevTimeoutSoftmax)) break;
              if (lane == 0) {
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2) {
                  const int kk = 2 * c + k2;
                  mma_bf16_ts(tmem + 256 + 128 * t, tmem + 128 * t + kk * 8, sdesc_sw128(sv + kk * 2048, BOX, 1024),
                              id_pv, (i > 0 || kk > 0) ? 1u : 0u);
                }
              }
              __syncwarp();
            }
            if (!ok) break;
            ++steps[t];
            if (lane == 0) {
              if (t == cur.nt - 1) mma_commit(bar(KE + ev));
              if (last) mma_commit(bar(OF + t));
            }
            __syncwarp();
            if (!last) {
              if (t == 0) {
                ek = r % NKV;
                if (!wait(KF + ek, (r / NKV) & 1, kDevTimeoutLoad)) break;
                ++r;
              }
              issue_s(t, eq[t], ek, i + 2 == cur.cnt, t == cur.nt - 1);
            } else if (more && t < nxt.nt) {
              open_item(nxt, t);
            }
          }
        }
        if (ok && more && nxt.nt > cur.nt) open_item(nxt, 1);
        have = more;
        cur = nxt;
      }
      // every MMA issued has completed before TMEM is freed, also on the abort path
      if (lane == 0) {
        mma_commit(bar(DRAIN));
        mbar_wait_until(bar(DRAIN), 0, globaltimer_ns() + kWaitLimitNs);
      }
      __syncwarp();
    }
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CORR));
    // --------------------------------------------------- correction and output
    const int q = warp & 3, row = q * 32 + lane;
    const uint32_t lane_off = (uint32_t)(q * 32) << 16;
    const float* s_alpha = reinterpret_cast<const float*>(smem1k + OFF_ALPHA);
    const float* s_l = reinterpret_cast<const float*>(smem1k + OFF_L);
    int pub[2] = {0, 0}, fin[2] = {0, 0};  // phases of AR, and of LF and OF, passed
    bool ok = true;
    // output of a row of item `it`: v = O / l (zeros for an item without keys)
    auto out_row = [&](const CrossItem& it, int t, float inv_l, bool zero) {
      int h, tok;
      const bool live = cross_row(p, it, it.m0 + t, row, h, tok);
      const uint32_t tO = tmem + 256 + 128 * t + lane_off;
      const int64_t prow = p.nsplit > 1 ? (((int64_t)it.split * p.B + it.b) * p.H + h) * p.Lq + tok : 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t v[32];
        if (!zero) {
          __syncwarp();  // the stores below diverge, the load is warp-collective
          tmem_ld32(tO + 32 * c, v);
          tmem_ld_wait();
        }
        float f[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = zero ? 0.f : __uint_as_float(v[e]) * inv_l;
        if (live && p.nsplit > 1) {
          if (!zero) {
            float4* dst = reinterpret_cast<float4*>(p.part_o + prow * 128 + 32 * c);
#pragma unroll
            for (int e = 0; e < 8; ++e) dst[e] = make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
          }
        } else if (live) {
          uint4* dst = reinterpret_cast<uint4*>(p.out + it.b * p.o_sB + h * p.o_sH + tok * p.o_sT + 32 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            dst[e] = make_uint4(pack_bf2(f[8 * e], f[8 * e + 1]), pack_bf2(f[8 * e + 2], f[8 * e + 3]),
                                pack_bf2(f[8 * e + 4], f[8 * e + 5]), pack_bf2(f[8 * e + 6], f[8 * e + 7]));
        }
      }
    };
    auto wait = [&](int i, uint32_t parity, int code) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(i), parity, abort_flag, code));
      return ok;
    };
    CrossItem prev;
    prev.nt = 0;
    auto finish = [&](int t) {  // the previous item's tile t
      if (t >= prev.nt || !ok) return;
      if (!wait(LF + t, fin[t] & 1, kDevTimeoutSoftmax)) return;
      const float inv_l = 1.0f / s_l[t * 128 + row];
      if (!wait(OF + t, fin[t] & 1, kDevTimeoutMma)) return;
      ++fin[t];
      tc_fence_after();
      out_row(prev, t, inv_l, false);
    };
    for (int64_t w = blockIdx.x; w < p.items && ok; w += gridDim.x) {
      const CrossItem it = cross_item(p, w);
      if (it.cnt == 0) {
        for (int t = 0; t < it.nt; ++t) {
          out_row(it, t, 0.f, true);
          int h, tok;
          const bool live = cross_row(p, it, it.m0 + t, row, h, tok);
          if (p.nsplit > 1) {
            if (live) p.part_lse[(((int64_t)it.split * p.B + it.b) * p.H + h) * p.Lq + tok] = -INFINITY;
          } else if (p.lse && (live || !p.pack)) {
            p.lse[((int64_t)it.b * p.H + h) * p.lse_ld + tok] = INFINITY;
          }
        }
        continue;
      }
      for (int i = 0; i < it.cnt && ok; ++i) {
        for (int t = 0; t < 2 && ok; ++t) {
          if (i == 0) finish(t);
          if (t >= it.nt || !wait(AR + t, pub[t] & 1, kDevTimeoutSoftmax)) continue;
          ++pub[t];
          const float alpha = s_alpha[t * 128 + row];
          if (i > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
            tc_fence_after();
            const uint32_t tO = tmem + 256 + 128 * t + lane_off;
            const uint64_t a2 = f2_pack(alpha, alpha);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t ov[32];
              tmem_ld32(tO + 32 * c, ov);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                float o0, o1;
                f2_unpack(mul_f32x2(f2_pack(__uint_as_float(ov[2 * e]), __uint_as_float(ov[2 * e + 1])), a2), o0, o1);
                ov[2 * e] = __float_as_uint(o0);
                ov[2 * e + 1] = __float_as_uint(o1);
              }
              tmem_st32(tO + 32 * c, ov);
            }
            tmem_st_wait();
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(OC + t));
        }
      }
      prev = it;
    }
    for (int t = 0; t < 2; ++t) finish(t);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    // -------------------------------------------------------------- softmax
    const int t = (warp - 4) >> 2, q = warp & 3, row = q * 32 + lane;
    const uint32_t tS = tmem + 128 * t + ((uint32_t)(q * 32) << 16);
    float* s_alpha = reinterpret_cast<float*>(smem1k + OFF_ALPHA) + t * 128 + row;
    float* s_l = reinterpret_cast<float*>(smem1k + OFF_L) + t * 128 + row;
    const float scale = p.qk_scale;
    int steps = 0;
    bool ok = true;
    for (int64_t w = blockIdx.x; w < p.items && ok; w += gridDim.x) {
      const CrossItem it = cross_item(p, w);
      if (it.cnt == 0 || t >= it.nt) continue;
      float m_run = 0.f, l_run = 0.f;
      for (int i = 0; i < it.cnt; ++i, ++steps) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar(SF + t), steps & 1, abort_flag, kDevTimeoutMma));
        if (!ok) break;
        tc_fence_after();
        uint32_t v[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&v[c * 32]));
        tmem_ld_wait();
        const int valid = it.len - (it.i0 + i) * 128;
        if (valid < 128) {
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c >= valid) v[c] = __float_as_uint(-INFINITY);
        }
        float mx8[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          mx8[k] = __uint_as_float(v[k]);
#pragma unroll
          for (int j = 0; j < 7; ++j)
            mx8[k] = max3f(mx8[k], __uint_as_float(v[k + 8 + 16 * j]), __uint_as_float(v[k + 16 + 16 * j]));
          mx8[k] = fmaxf(mx8[k], __uint_as_float(v[k + 120]));
        }
        const float mx = max3f(fmaxf(mx8[0], mx8[1]), max3f(mx8[2], mx8[3], mx8[4]), max3f(mx8[5], mx8[6], mx8[7]));
        const float m_new = mx * scale;
        float alpha = 1.f;
        if (i == 0) {
          m_run = fmaxf(m_new, -FLT_MAX);  // finite, should every score of the tile be -inf
        } else if (m_new - m_run > RESCALE) {
          alpha = ex2_approx(m_run - m_new);
          m_run = m_new;
        }
        *s_alpha = alpha;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(AR + t));
        const uint64_t sc2 = f2_pack(scale, scale), nm2 = f2_pack(-m_run, -m_run);
        uint64_t rs2[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
        auto publish_p = [&](int c) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(PF + 4 * t + c));
        };
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pw[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x0, x1;
            f2_unpack(fma_f32x2(f2_pack(__uint_as_float(v[32 * c + 2 * e]), __uint_as_float(v[32 * c + 2 * e + 1])),
                                sc2, nm2),
                      x0, x1);
            const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
            rs2[e & 1] = add_f32x2(rs2[e & 1], f2_pack(p0, p1));
            pw[e] = pack_bf2(p0, p1);
          }
          if (c > 0) publish_p(c - 1);
          tmem_st16(tS + c * 16, pw);
        }
        publish_p(3);
        float ra, rb, rc, rd;
        f2_unpack(rs2[0], ra, rb);
        f2_unpack(rs2[1], rc, rd);
        l_run = l_run * alpha + ((ra + rc) + (rb + rd));
      }
      // the correction warps have taken this item's last factors, hence the previous
      // item's row sums too: a one-step item could otherwise overtake them
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(OC + t), (steps - 1) & 1, abort_flag, kDevTimeoutSoftmax));
      if (!ok) break;
      *s_l = l_run;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(LF + t));
      int h, tok;
      const bool live = cross_row(p, it, it.m0 + t, row, h, tok);
      const float lse = m_run + log2f(l_run);
      if (p.nsplit > 1) {
        if (live) p.part_lse[(((int64_t)it.split * p.B + it.b) * p.H + h) * p.Lq + tok] = lse;
      } else if (p.lse && (live || !p.pack)) {
        p.lse[((int64_t)it.b * p.H + h) * p.lse_ld + tok] = live ? lse : INFINITY;
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

// o = sum_s 2^(lse_s - lse) o_s over the slices, one warp per row; also the row's lse
__global__ void __launch_bounds__(128) cross_combine_kernel(const CrossAttnParams p) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)p.B * p.H * p.Lq;
  if (row >= rows) return;
  const int t = (int)(row % p.Lq);
  const int64_t bh = row / p.Lq;
  float top = -INFINITY;
  for (int s = 0; s < p.nsplit; ++s) top = fmaxf(top, p.part_lse[s * rows + row]);
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  bool bad = false;
  for (int s = 0; s < p.nsplit; ++s) {
    const float l = p.part_lse[s * rows + row];
    if (l == -INFINITY) continue;  // a slice without keys wrote no output
    bad |= l != l;
    const float w = exp2f(l - top);
    const float4 o = *reinterpret_cast<const float4*>(p.part_o + (s * rows + row) * 128 + 4 * lane);
    a.x = fmaf(w, o.x, a.x), a.y = fmaf(w, o.y, a.y), a.z = fmaf(w, o.z, a.z), a.w = fmaf(w, o.w, a.w);
    sum += w;
  }
  const bool empty = top == -INFINITY && !bad;
  const float inv = empty ? 0.f : 1.0f / sum;
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  *reinterpret_cast<uint2*>(p.out + b * p.o_sB + h * p.o_sH + t * p.o_sT + 4 * lane) =
      make_uint2(pack_bf2(a.x * inv, a.y * inv), pack_bf2(a.z * inv, a.w * inv));
  if (p.lse && lane == 0) p.lse[bh * p.lse_ld + t] = empty ? INFINITY : top + log2f(sum);
}

// lse of the padding rows [Lq, lse_ld) := +inf (rows that no tile of the forward reached)
__global__ void cross_lse_pad_kernel(float* lse, int64_t rows, int Lq, int ld) {
  const int64_t g = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int pad = ld - Lq;
  if (g < rows * pad) lse[(g / pad) * ld + Lq + g % pad] = INFINITY;
}

// How the keys are cut: with at least one item per SM they are not (every slice
// costs an fp32 partial); with fewer, into slices of two key tiles or more.
CrossAttnPlan cross_attn_plan(int B, int H, int Hkv, int Lq, int Lk) {
  CrossAttnPlan pl{};
  const int G = H / Hkv;
  pl.pack = G > 1 && (int64_t)G * Lq <= 128;
  pl.nqt = pl.pack ? 1 : (Lq + 127) / 128;
  pl.nqp = (pl.nqt + 1) / 2;
  const int64_t items = (int64_t)pl.nqp * B * (pl.pack ? Hkv : H);
  const int ntk = (Lk + 127) / 128, sms = device_sms();
  pl.nsplit = 1;
  if (items < sms && ntk >= 4) {
    const int64_t want = (sms + items - 1) / items;
    pl.nsplit = (int)(want < ntk / 2 ? want : ntk / 2);
  }
  return pl;
}

int launch_cross_attn(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CrossAttnParams& p,
                      cudaStream_t s) {
  using namespace xattn;
  static KernelReady ready;
  const int rc = kernel_ready(ready, cross_attn_tcgen05, SMEM, LAUNCH_REGS);
  if (rc != 0) return rc;
  cudaError_t e;
  const int sms = device_sms();
  cross_attn_tcgen05<<<(unsigned)(p.items < sms ? p.items : sms), THREADS, SMEM, s>>>(tq, tk, tv, p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return (int)e;
  const int64_t rows = (int64_t)p.B * p.H * p.Lq;
  if (p.nsplit > 1) {
    cross_combine_kernel<<<(unsigned)((rows + 3) / 4), 128, 0, s>>>(p);
    if ((e = cudaGetLastError()) != cudaSuccess) return (int)e;
  }
  if (p.lse && (p.nsplit > 1 || p.pack) && p.lse_ld > p.Lq) {
    const int64_t n = (int64_t)p.B * p.H * (p.lse_ld - p.Lq);
    cross_lse_pad_kernel<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(p.lse, (int64_t)p.B * p.H, p.Lq, p.lse_ld);
  }
  return (int)cudaGetLastError();
}

}  // namespace rola
