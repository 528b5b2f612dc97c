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
// The work is a stream of units, one 128 x 128 tile of scores each: the key tiles
// of an item (128 query rows of a head, or a slice of their keys), item after
// item, on persistent CTAs, one per SM.  A unit is a chain, S = Q K^T -> softmax
// -> O += P V, whose softmax takes longer than its products; what keeps the
// tensor core busy is the number of units in flight.  Tensor memory holds three
// S tiles beside one O, so there are three, each with a softmax warpgroup of its
// own, and they run across the items' ends: an encoder's states are few keys (512:
// four units), and the S products of the next item are issued while this one
// finishes.  m and l pass from unit to unit through shared memory, in order.
//   warp 0        TMA producer of Q (2 x 32 KB) and K tiles (2 x 32 KB)
//   warp 3        TMA producer of V tiles (3 x 32 KB)
//                 Both also store the outputs that wait in their tiles (out_in_q;
//                 rows stored by the lanes themselves held their warps 2500 clocks)
//   warp 1        issues S; owner of the tensor memory
//   warp 2        issues P V.  It also clears the V rows past len[b] (their P is 0,
//                 but 0 * NaN is not).  One warp for both products was the limit:
//                 2150 clocks a unit to issue what takes the tensor core 1024
//   warpgroup g = 1, 2, 3: the units u with u % 3 == g - 1; thread = row = TMEM lane.
//                 The unit that ends an item scales its O by 1/l and leaves it in bf16.
// Measured alone: 32760 rows x 512 keys, 40 heads 322 us (1068 TFLOP/s, 0.64 of the
// matrix peak), 32760 x 8192, 4 heads 413 us (1330, 0.79); in a long run the power
// limit takes 10 to 15 % of the clock.  With many keys a unit takes 1600 clocks, of
// which its products need 1041 and its exponentials 1024: neither is full, the three
// chains are what bounds it; an item's end costs some 1400 clocks more.  Tried and
// slower: two S and two P tiles apart (the next S starts once its tile is read, but
// only two wait), half units for four warpgroups, a warpgroup of its own for the outputs.
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
constexpr int REGS_LOAD = 56, REGS_SOFTMAX = 152;
static_assert(128 * (REGS_LOAD + 3 * REGS_SOFTMAX) <= THREADS * LAUNCH_REGS, "register split");
constexpr int BOX = 16384;        // [128 rows x 64 bf16], 128-byte swizzle
constexpr int TILE = 2 * BOX;     // 128 rows x 128 columns
constexpr int NQ = 2, NK = 2, NV = 3, NS = 3;
constexpr int OFF_Q = 0;
constexpr int OFF_K = NQ * TILE, OFF_V = OFF_K + NK * TILE;
constexpr int OFF_M = OFF_V + NV * TILE;  // [2][128] running maxima after even / odd units
constexpr int OFF_L = OFF_M + 1024;         // [2][128] running sums
constexpr int OFF_BAR = OFF_L + 1024;
constexpr int SMEM = OFF_BAR + 512;
constexpr int O_COL = 128 * NS;   // S of unit u at column 128 (u % 3), its P in the upper 64 of those; O behind them
constexpr float RESCALE = 8.0f;   // log2 growth of the maximum that triggers a rescale of O
enum : int {
  QF = 0, QE = QF + NQ,
  KF = QE + NQ, KE = KF + NK, VF = KE + NK, VE = VF + NV,
  SF = VE + NV,      // S of a unit in TMEM: SF + u % 3, as those below
  PB = SF + NS,      // P of keys [64, 128) in TMEM, 4 warp arrivals
  PA = PB + NS,      // P of keys [0, 64)
  OV = PA + NS,      // output of an item in the V tile of its last unit, 4 arrivals: OV + u % 3
  OQ = OV + NV,      // output of an item in its Q tile, 4 arrivals
  PV = OQ + NQ,      // P V of a unit done (its S columns are free, O holds it)
  MR = PV + NS,      // m after unit u published, 4 arrivals (a single barrier would not do: the unit that waits
                     // may find it two phases behind, which parity cannot tell from done)
  LR = MR + NS,      // l after unit u published, 4 arrivals
  OE = LR + NS,      // O read by the item's epilogue (phase: item), 4 arrivals
  DRAIN_S = OE + 1,
  DRAIN_P,
  COUNT
};
static_assert(8 * COUNT + 16 <= 512, "barrier region");
static_assert(SMEM <= 227 * 1024, "shared memory");
}  // namespace xattn

// Where an item's output waits for its TMA store.  A Q tile that holds one is loaded
// late, which an item of one or two units cannot hide from the S products three units
// on; a V tile is held up by the store, which costs the others 3 % (32760 x 128 / 256 /
// 512, 40 heads, us: in Q tiles 182 / 217 / 327, in V tiles 154 / 207 / 341).
__device__ __forceinline__ bool out_in_q(int units) { return units >= 3; }

// valid keys of batch b
__device__ __forceinline__ int kv_len(const int32_t* lens, int b, int Lk) {
  return lens ? min(max(lens[b], 0), Lk) : Lk;
}

// Walks the items of a CTA, w = blockIdx.x, + gridDim.x, ...: query tile m
// fastest, then the slice, the head of the grid (key head when packed), the
// batch.  The digits are advanced by the step's own digits with carries; a
// division per item cost each role about 2500 clocks.  Without slices (kSplit
// false) their digit is left out, and the stores of partials: with it a short item
// took a tenth longer (32760 x 128 / 256, 40 heads, 150 / 203 us instead of 131 / 181).
template <bool kSplit>
struct CrossItems {
  uint32_t w;
  int m, split = 0, h, b;
  int dm, ds = 0, dh, db;
  int len, i0 = 0, cnt;  // valid keys; key tiles [i0, i0 + cnt) of the item

  __device__ __forceinline__ static void digits(const CrossAttnParams& p, uint32_t w, int& m, int& s, int& h, int& b) {
    const uint32_t r = w / (uint32_t)p.nqt;
    m = (int)(w - r * (uint32_t)p.nqt);
    const uint32_t t = kSplit ? r / (uint32_t)p.nsplit : r;
    s = kSplit ? (int)(r - t * (uint32_t)p.nsplit) : 0;
    b = (int)(t / (uint32_t)p.Hgrid);
    h = (int)(t - (uint32_t)b * (uint32_t)p.Hgrid);
  }
  __device__ __forceinline__ void range(const CrossAttnParams& p) {
    if (w >= (uint32_t)p.items) return;
    len = kv_len(p.kv_lens, b, p.Lk);
    const int n = (len + 127) >> 7;
    cnt = n;
    if (kSplit) {
      i0 = (int)((uint32_t)n * (uint32_t)split / (uint32_t)p.nsplit);
      cnt = (int)((uint32_t)n * (uint32_t)(split + 1) / (uint32_t)p.nsplit) - i0;
    }
  }
  __device__ __forceinline__ explicit CrossItems(const CrossAttnParams& p) : w(blockIdx.x) {
    digits(p, w, m, split, h, b);
    digits(p, gridDim.x, dm, ds, dh, db);
    range(p);
  }
  __device__ __forceinline__ bool live(const CrossAttnParams& p) const { return w < (uint32_t)p.items; }
  __device__ __forceinline__ void next(const CrossAttnParams& p) {
    w += gridDim.x;
    m += dm;
    int c = m >= p.nqt;
    m -= c ? p.nqt : 0;
    if (kSplit) {
      split += ds + c;
      c = split >= p.nsplit;
      split -= c ? p.nsplit : 0;
    }
    h += dh + c;
    c = h >= p.Hgrid;
    h -= c ? p.Hgrid : 0;
    b += db + c;
    range(p);
  }
  // row r of the tile -> head and token; false past the last row
  __device__ __forceinline__ bool row(const CrossAttnParams& p, int r, int& head, int& t) const {
    if (p.pack) {
      const int g = r / p.Lq;
      head = h * p.G + g;
      t = r - g * p.Lq;
      return g < p.G;
    }
    head = h;
    t = m * 128 + r;
    return t < p.Lq;
  }
};

// shared memory row r >= valid of a [128 x 128] V tile := 0 (whole 128-byte rows, so the swizzle does not matter)
__device__ __forceinline__ void clear_rows(uint8_t* tile, int valid, int lane) {
  for (int i = valid * 8 + lane; i < 128 * 8; i += 32) {
    *reinterpret_cast<uint4*>(tile + i * 16) = make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4*>(tile + xattn::BOX + i * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

template <bool kSplit>
__global__ void __launch_bounds__(xattn::THREADS, 1)
    cross_attn_tcgen05(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                       const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap to,
                       const CrossAttnParams p) {
  using namespace xattn;
  using Items = CrossItems<kSplit>;
  extern __shared__ __align__(1024) uint8_t smem1k[];
  const uint32_t base = smem_u32(smem1k);
  auto bar = [&](int i) { return base + OFF_BAR + 8u * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem1k + OFF_BAR + 8 * COUNT);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem1k + OFF_BAR + 8 * COUNT + 8);
  // broadcast values are warp-uniform to the compiler too: the MMA warp's addresses and
  // descriptors stay in uniform registers, which its instructions need
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < COUNT; ++i) mbar_init(bar(i), (i >= PB && i < PV) || (i >= MR && i < DRAIN_S) ? 4 : 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tq);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
    if (!kSplit) prefetch_tmap(&to);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_LOAD));
    constexpr uint32_t hi = sdesc_hi(1024);
    bool ok = true;
    // warp-wide wait of the issuing warps
    auto wait = [&](int i, uint32_t parity, int code) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_spin(bar(i), parity, abort_flag, code));
      tc_fence_after();
      return ok;
    };
    // An item's output waits in one of its tiles until that is loaded again: the tiles
    // of one ring that hold one
    struct Outputs {
      uint32_t held = 0, phase = 0;  // bits: tile f holds the output of an item; phase of its barrier
      int m[NV] = {}, h[NV] = {}, b[NV] = {};
      __device__ __forceinline__ void expect(int f, const Items& it, const CrossAttnParams& p) {
        held |= 1u << f;
        m[f] = it.m * 128, h[f] = p.pack ? it.h * p.G : it.h, b[f] = it.b;
      }
    };
    auto store_out = [&](Outputs& o, int f, uint32_t tile, int staged) {
      if (!((o.held >> f) & 1)) return true;
      if (!mbar_spin(bar(staged), (o.phase >> f) & 1, abort_flag, kDevTimeoutSoftmax)) return false;
      o.held ^= 1u << f;
      o.phase ^= 1u << f;
      tma_store_4d(&to, tile, 0, o.m[f], o.h[f], o.b[f]);
      tma_store_4d(&to, tile + BOX, 64, o.m[f], o.h[f], o.b[f]);
      tma_store_commit();
      tma_store_wait_read();
      return true;
    };
    if (warp == 0) {
      if (lane == 0) {
        // -------------------------------------------- TMA: Q and K; outputs in Q tiles
        int q = 0, k = 0;  // tiles loaded
        Outputs outs;
        for (Items it(p); it.live(p) && ok; it.next(p)) {
          if (it.cnt == 0) continue;
          const int e = q % NQ;
          if (!(ok = mbar_spin(bar(QE + e), ((q / NQ) & 1) ^ 1, abort_flag, kDevTimeoutMma))) break;
          if (!(ok = store_out(outs, e, base + OFF_Q + e * TILE, OQ + e))) break;
          if (!kSplit && out_in_q(it.cnt)) outs.expect(e, it, p);
          mbar_expect_tx(bar(QF + e), p.q_bytes);
          const int hq = p.pack ? it.h * p.G : it.h, hk = p.pack ? it.h : it.h / p.G;
          tma_load_4d(base + OFF_Q + e * TILE, &tq, bar(QF + e), 0, it.m * 128, hq, it.b);
          tma_load_4d(base + OFF_Q + e * TILE + BOX, &tq, bar(QF + e), 64, it.m * 128, hq, it.b);
          ++q;
          for (int i = it.i0; i < it.i0 + it.cnt; ++i, ++k) {
            const int f = k % NK;
            if (!(ok = mbar_spin(bar(KE + f), ((k / NK) & 1) ^ 1, abort_flag, kDevTimeoutMma))) break;
            mbar_expect_tx(bar(KF + f), TILE);
            tma_load_4d(base + OFF_K + f * TILE, &tk, bar(KF + f), 0, i * 128, hk, it.b);
            tma_load_4d(base + OFF_K + f * TILE + BOX, &tk, bar(KF + f), 64, i * 128, hk, it.b);
          }
        }
        for (int n = max(0, q - NQ); n < q && ok; ++n)
          ok = store_out(outs, n % NQ, base + OFF_Q + n % NQ * TILE, OQ + n % NQ);
        // no copy may still target shared memory when the CTA exits; the waits
        // ignore the abort flag and share one limit
        const uint64_t deadline = globaltimer_ns() + kWaitLimitNs;
        bool drained = true;
        for (int n = max(0, q - NQ); n < q && drained; ++n)
          drained = mbar_wait_until(bar(QF + n % NQ), (n / NQ) & 1, deadline);
        for (int n = max(0, k - NK); n < k && drained; ++n)
          drained = mbar_wait_until(bar(KF + n % NK), (n / NK) & 1, deadline);
      }
    } else if (warp == 3) {
      if (lane == 0) {
        // ------------------------------------------------ TMA: V; outputs in V tiles
        int k = 0;
        Outputs outs;
        for (Items it(p); it.live(p) && ok; it.next(p)) {
          const int hk = p.pack ? it.h : it.h / p.G;
          for (int i = it.i0; i < it.i0 + it.cnt; ++i, ++k) {
            const int f = k % NV;
            if (!(ok = mbar_spin(bar(VE + f), ((k / NV) & 1) ^ 1, abort_flag, kDevTimeoutMma))) break;
            if (!(ok = store_out(outs, f, base + OFF_V + f * TILE, OV + f))) break;
            mbar_expect_tx(bar(VF + f), TILE);
            tma_load_4d(base + OFF_V + f * TILE, &tv, bar(VF + f), 0, i * 128, hk, it.b);
            tma_load_4d(base + OFF_V + f * TILE + BOX, &tv, bar(VF + f), 64, i * 128, hk, it.b);
            if (!kSplit && i + 1 == it.i0 + it.cnt && !out_in_q(it.cnt)) outs.expect(f, it, p);
          }
        }
        for (int n = max(0, k - NV); n < k && ok; ++n)
          ok = store_out(outs, n % NV, base + OFF_V + n % NV * TILE, OV + n % NV);
        const uint64_t deadline = globaltimer_ns() + kWaitLimitNs;
        bool drained = true;
        for (int n = max(0, k - NV); n < k && drained; ++n)
          drained = mbar_wait_until(bar(VF + n % NV), (n / NV) & 1, deadline);
      }
    } else if (warp == 1) {
      // ------------------------------------------------------- MMA: S = Q K^T
      constexpr uint32_t id_qk = idesc_bf16_f32(128, 128, false, false);
      int eq = 0, ek = 0, g = 0;
      uint32_t q_ph = 0, k_ph = 0, g_ph = 1;  // g_ph: the buffer's previous unit is done (passes at first)
      for (Items it(p); it.live(p) && ok; it.next(p)) {
        const int cnt = __shfl_sync(0xffffffffu, it.cnt, 0);
        if (cnt == 0) continue;
        if (!wait(QF + eq, q_ph, kDevTimeoutLoad)) break;
        const uint32_t dq = sdesc_lo(base + OFF_Q + eq * TILE, 16);
        for (int i = 0; i < cnt; ++i) {
          if (!wait(KF + ek, k_ph, kDevTimeoutLoad) || !wait(PV + g, g_ph, kDevTimeoutMma)) break;
          if (elect_one()) {
            const uint32_t dk = sdesc_lo(base + OFF_K + ek * TILE, 16);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
              const uint32_t off = ((kk >> 2) * BOX + (kk & 3) * 32) >> 4;
              mma_bf16_ss_lo(tmem + 128 * g, dq + off, hi, dk + off, hi, id_qk, kk > 0 ? 1u : 0u);
            }
            mma_commit(bar(SF + g));
            mma_commit(bar(KE + ek));
            if (i + 1 == cnt) mma_commit(bar(QE + eq));
          }
          __syncwarp();
          if (++ek == NK) {
            ek = 0;
            k_ph ^= 1u;
          }
          if (++g == NS) {
            g = 0;
            g_ph ^= 1u;
          }
        }
        if (++eq == NQ) {
          eq = 0;
          q_ph ^= 1u;
        }
      }
      // every MMA issued has completed before TMEM is freed, also on the abort path
      if (elect_one()) {
        mma_commit(bar(DRAIN_S));
        mbar_wait_until(bar(DRAIN_S), 0, globaltimer_ns() + kWaitLimitNs);
      }
      __syncwarp();
    } else {
      // ------------------------------------------------------- MMA: O += P V
      constexpr uint32_t id_pv = idesc_bf16_f32(128, 128, false, true);
      int ev = 0, g = 0;
      uint32_t v_ph = 0, g_ph = 0, o_ph = 1;
      for (Items it(p); it.live(p) && ok; it.next(p)) {
        const int cnt = __shfl_sync(0xffffffffu, it.cnt, 0);
        if (cnt == 0) continue;
        // valid keys of the item's last tile, where rows past them may hold anything
        const int valid = it.len - (it.i0 + it.cnt - 1) * 128;
        const int tail = __shfl_sync(0xffffffffu, it.len < p.Lk ? valid : 128, 0);
        for (int i = 0; i < cnt && ok; ++i) {
          if (!wait(VF + ev, v_ph, kDevTimeoutLoad)) break;
          if (tail < 128 && i + 1 == cnt) clear_rows(smem1k + OFF_V + ev * TILE, tail, lane);
          // O of the previous item has been read
          if (i == 0 && !wait(OE, o_ph, kDevTimeoutSoftmax)) break;
          const uint32_t dv = sdesc_lo(base + OFF_V + ev * TILE, BOX), tp = tmem + 128 * g + 64;
#pragma unroll
          for (int half = 1; half >= 0; --half) {  // keys [64, 128) first, as the softmax hands them over
            if (!wait((half ? PB : PA) + g, g_ph, kDevTimeoutSoftmax)) break;
            if (elect_one()) {
#pragma unroll
              for (int k4 = 0; k4 < 4; ++k4) {
                const int kk = 4 * half + k4;
                mma_bf16_ts_lo(tmem + O_COL, tp + 8 * kk, dv + ((kk * 2048) >> 4), hi, id_pv,
                               (i > 0 || half == 0 || k4 > 0) ? 1u : 0u);
              }
              if (half == 0) {
                mma_commit(bar(VE + ev));
                mma_commit(bar(PV + g));
              }
            }
            __syncwarp();
          }
          if (++ev == NV) {
            ev = 0;
            v_ph ^= 1u;
          }
          if (++g == NS) {
            g = 0;
            g_ph ^= 1u;
          }
        }
        o_ph ^= 1u;
      }
      if (elect_one()) {
        mma_commit(bar(DRAIN_P));
        mbar_wait_until(bar(DRAIN_P), 0, globaltimer_ns() + kWaitLimitNs);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    // ------------------------------------------------------- softmax and output
    const int g = (warp >> 2) - 1, q = warp & 3, row = q * 32 + lane;
    const uint32_t lane_off = (uint32_t)(q * 32) << 16;
    const uint32_t tS = tmem + 128 * g + lane_off, tP = tS + 64, tO = tmem + O_COL + lane_off;
    float* s_m = reinterpret_cast<float*>(smem1k + OFF_M) + row;
    float* s_l = reinterpret_cast<float*>(smem1k + OFF_L) + row;
    const float scale = p.qk_scale;
    bool ok = true;
    auto wait = [&](int i, uint32_t parity, int code) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_spin(bar(i), parity, abort_flag, code));
      return ok;
    };
    int u = 0, j = 0, items = 0;  // units, items with keys, items
    for (Items it(p); it.live(p) && ok; it.next(p)) {
      if (it.cnt == 0) {
        // no keys: zeros (one warpgroup in turn; no unit, nothing to wait for)
        if (items % 3 == g) {
          int h, tok;
          const bool live = it.row(p, row, h, tok);
          if (kSplit) {
            if (live) p.part_lse[(((int64_t)it.split * p.B + it.b) * p.H + h) * p.Lq + tok] = -INFINITY;
          } else {
            if (live) {
              uint4* dst = reinterpret_cast<uint4*>(p.out + it.b * p.o_sB + h * p.o_sH + tok * p.o_sT);
#pragma unroll
              for (int c = 0; c < 16; ++c) dst[c] = make_uint4(0u, 0u, 0u, 0u);
            }
            if (p.lse && (live || !p.pack)) p.lse[((int64_t)it.b * p.H + h) * p.lse_ld + tok] = INFINITY;
          }
        }
        ++items;
        continue;
      }
      for (int i = 0; i < it.cnt && ok; ++i, ++u) {
        if (u % NS != g) continue;
        const uint32_t ph = (u / NS) & 1;
        if (!wait(SF + g, ph, kDevTimeoutMma)) break;
        tc_fence_after();
        // maximum of the row, 32 columns at a time; the last two chunks stay in registers,
        // the first two are read again for the exponentials.  The loops over chunks stay
        // loops: unrolled, three warpgroups' places in the code overran the instruction
        // cache (28 % of their time)
        const int valid = it.len - (it.i0 + i) * 128;
        uint32_t v[2][32];
        if (valid < 128) {  // scores past the last key: -inf, in tensor memory
#pragma unroll 1
          for (int c = valid; c < 128;) {
            if (c & 15) {
              tmem_st1(tS + c++, 0xff800000u);
            } else {
              uint32_t w[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) w[e] = 0xff800000u;
              tmem_st16(tS + c, w);
              c += 16;
            }
          }
          tmem_st_wait();
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        auto fold = [&](const uint32_t(&x)[32]) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              m4[k] = max3f(m4[k], __uint_as_float(x[k + 8 * e]), __uint_as_float(x[k + 4 + 8 * e]));
        };
#pragma unroll 1
        for (int c = 0; c < 4; c += 2) {
          tmem_ld32(tS + 32 * c, v[0]);
          tmem_ld32(tS + 32 * c + 32, v[1]);
          tmem_ld_wait();
          fold(v[0]);
          fold(v[1]);
        }
        const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        // m after this unit, from the unit before (published in unit order)
        float m = fmaxf(mx * scale, -FLT_MAX), alpha = 1.f;  // finite, should every score be -inf
        if (u > 0 && !wait(MR + (u - 1) % NS, ((u - 1) / NS) & 1, kDevTimeoutSoftmax)) break;
        if (i > 0) {
          const float m_prev = s_m[128 * ((u & 1) ^ 1)];
          if (m - m_prev > RESCALE) {
            alpha = ex2_approx(m_prev - m);
          } else {
            m = m_prev;
          }
        }
        s_m[128 * (u & 1)] = m;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(MR + g));
        if (__any_sync(0xffffffffu, alpha != 1.f)) {
          // O of the units before, once the last of them is in
          if (!wait(PV + (u - 1) % NS, ((u - 1) / NS) & 1, kDevTimeoutMma)) break;
          tc_fence_after();
          const uint64_t a2 = f2_pack(alpha, alpha);
#pragma unroll 1
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
        const uint64_t sc2 = f2_pack(scale, scale), nm2 = f2_pack(-m, -m);
        uint64_t rs2[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
        // P of 32 keys, packed bf16
        auto exp32 = [&](const uint32_t(&x)[32], int c) {
          uint32_t pw[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x0, x1;
            f2_unpack(fma_f32x2(f2_pack(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), sc2, nm2), x0, x1);
            const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
            rs2[e & 1] = add_f32x2(rs2[e & 1], f2_pack(p0, p1));
            pw[e] = pack_bf2(p0, p1);
          }
          tmem_st16(tP + 16 * c, pw);
        };
        auto publish = [&](int b) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(b + g));
        };
#pragma unroll 1
        for (int c = 2; c >= 0; c -= 2) {
          exp32(v[1], c + 1);
          if (c == 2) tmem_ld32(tS + 32, v[1]);
          exp32(v[0], c);
          if (c == 2) tmem_ld32(tS, v[0]);
          publish(c == 2 ? PB : PA);
          if (c == 2) tmem_ld_wait();
        }
        float ra, rb, rc, rd;
        f2_unpack(rs2[0], ra, rb);
        f2_unpack(rs2[1], rc, rd);
        float l = (ra + rc) + (rb + rd);
        if (u > 0 && !wait(LR + (u - 1) % NS, ((u - 1) / NS) & 1, kDevTimeoutSoftmax)) break;
        if (i > 0) l = fmaf(s_l[128 * ((u & 1) ^ 1)], alpha, l);
        s_l[128 * (u & 1)] = l;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(LR + g));
        if (i + 1 < it.cnt) continue;

        // ------------------------------------------------- the item's output
        int h, tok;
        const bool live = it.row(p, row, h, tok);
        const float inv_l = 1.0f / l, lse = m + log2f(l);
        if (!wait(PV + g, ph, kDevTimeoutMma)) break;
        tc_fence_after();
        const int64_t prow = (((int64_t)it.split * p.B + it.b) * p.H + h) * p.Lq + tok;
        // the row of the item's Q tile or the unit's V tile, whose products are done: 16-byte
        // chunk c of a box at c ^ (row & 7), the maps' swizzle
        const bool in_q = out_in_q(it.cnt);
        uint8_t* stage = smem1k + (in_q ? OFF_Q + (j % NQ) * TILE : OFF_V + (u % NV) * TILE) + row * 128;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t v[64];
          __syncwarp();  // the stores of a slice's partial diverge, the load is warp-collective
          tmem_ld32(tO + 64 * c, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
          tmem_ld32(tO + 64 * c + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
          tmem_ld_wait();
          if (c == 1) {
            // O is in registers: the next item may start its own
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(OE));
          }
          if (!kSplit) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                w[k] = pack_bf2(__uint_as_float(v[8 * e + 2 * k]) * inv_l, __uint_as_float(v[8 * e + 2 * k + 1]) * inv_l);
              *reinterpret_cast<uint4*>(stage + c * BOX + ((e ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else if (live) {
            float4* d4 = reinterpret_cast<float4*>(p.part_o + prow * 128 + 64 * c);
#pragma unroll
            for (int e = 0; e < 16; ++e)
              d4[e] = make_float4(__uint_as_float(v[4 * e]) * inv_l, __uint_as_float(v[4 * e + 1]) * inv_l,
                                  __uint_as_float(v[4 * e + 2]) * inv_l, __uint_as_float(v[4 * e + 3]) * inv_l);
          }
        }
        if (!kSplit) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(in_q ? OQ + j % NQ : OV + u % NV));
        }
        if (kSplit) {
          if (live) p.part_lse[prow] = lse;
        } else if (p.lse && (live || !p.pack)) {
          p.lse[((int64_t)it.b * p.H + h) * p.lse_ld + tok] = live ? lse : INFINITY;
        }
      }
      ++items;
      ++j;
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

// How the keys are cut: into as many slices as give every SM one item at most
// (a second, partly filled round costs more than it balances: 32 items of 64 key
// tiles in us, slices 1 | 4 | 5 | 8: 57 | 29 | 40 | 32), of 8 key tiles or more (a
// slice costs its ends and an fp32 partial: 12 items of 64 tiles, 8 | 12 slices:
// 17.8 | 19.2; 12 items of 4 tiles, 1 | 2: 9.5 | 11.9).
CrossAttnPlan cross_attn_plan(int B, int H, int Hkv, int Lq, int Lk) {
  CrossAttnPlan pl{};
  const int G = H / Hkv;
  pl.pack = G > 1 && (int64_t)G * Lq <= 128;
  pl.nqt = pl.pack ? 1 : (Lq + 127) / 128;
  const int64_t items = (int64_t)pl.nqt * B * (pl.pack ? Hkv : H);
  const int ntk = (Lk + 127) / 128, sms = device_sms();
  pl.nsplit = 1;
  const int64_t most = sms / items;
  if (most > 1 && ntk >= 16) pl.nsplit = (int)(most < ntk / 8 ? most : ntk / 8);
  return pl;
}

int launch_cross_attn(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to,
                      const CrossAttnParams& p, cudaStream_t s) {
  using namespace xattn;
  static KernelReady ready, ready_split;
  const int rc = p.nsplit > 1 ? kernel_ready(ready_split, cross_attn_tcgen05<true>, SMEM, LAUNCH_REGS)
                              : kernel_ready(ready, cross_attn_tcgen05<false>, SMEM, LAUNCH_REGS);
  if (rc != 0) return rc;
  cudaError_t e;
  const int sms = device_sms();
  const unsigned grid = (unsigned)(p.items < sms ? p.items : sms);
  if (p.nsplit > 1) cross_attn_tcgen05<true><<<grid, THREADS, SMEM, s>>>(tq, tk, tv, to, p);
  else cross_attn_tcgen05<false><<<grid, THREADS, SMEM, s>>>(tq, tk, tv, to, p);
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
