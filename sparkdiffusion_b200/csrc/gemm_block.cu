// Product of e4m3 operands with one fp32 scale per block of 128 (tcgen05):
//
//   out[m, n] = sum_kb xs[m, kb] ws[n / 128, kb] (sum_{k in block kb} xq[m, k] wq[n, k]) + bias[n]
//
// xq [M, K] has a scale per row and 128 columns, wq [N, K] one per 128 x 128
// block.  The scales are fp32 and change along K, so the products of one block
// of 128 are summed by the tensor core into a fresh TMEM accumulator (4 MMAs of
// K = 32), and the running sum is kept in fp32 registers: the epilogue warps
// read every block's accumulator and add it times xs * ws.  Both sums are fp32;
// the result is rounded once, to bf16.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace rola {

// acc += v * s for 2 n columns, two at a time
template <int n>
__device__ __forceinline__ void scaled_add(uint64_t (&acc)[n], const uint32_t (&v)[2 * n], uint64_t s2) {
#pragma unroll
  for (int i = 0; i < n; ++i)
    acc[i] = fma_f32x2(f2_pack(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), s2, acc[i]);
}

// 2 n finished columns of one row: bias, rounding, 16-byte stores of 8 columns
template <int n>
__device__ __forceinline__ void store_row(const uint64_t (&acc)[n], const __nv_bfloat16* bias, __nv_bfloat16* row,
                                          int col, int N) {
#pragma unroll
  for (int i = 0; i < n / 4; ++i) {
    const int c = col + 8 * i;
    if (c < N) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) f2_unpack(acc[4 * i + e], f[2 * e], f[2 * e + 1]);
      if (bias) {
        const uint4 b = __ldg(reinterpret_cast<const uint4*>(bias + c));
        const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float b0, b1;
          unpack_bf2(w[e], b0, b1);
          f[2 * e] += b0;
          f[2 * e + 1] += b1;
        }
      }
      *reinterpret_cast<uint4*>(row + c) =
          make_uint4(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]), pack_bf2(f[4], f[5]), pack_bf2(f[6], f[7]));
    }
  }
}

// ---------------------------------------------------------------------------
// 128 x BN tiles (BN 256 or 128), persistent CTAs, one per SM.  Every K block is
// a hand-off from the MMA issuer to the epilogue and back, and what is in flight
// is bounded by the 512 columns of tensor memory, so the accumulators are small
// units with a hand-off each: 128 columns, four of them.  BN = 256 has two
// streams (column halves) of two, and a warpgroup of the epilogue each (128 sums
// a thread; the registers of the producer's warpgroup go to them by setmaxnreg);
// BN = 128 one stream of four that both warpgroups share, 64 columns each.
// Measured at 32760 x 15360 x 5120 (TFLOP/s): BN = 256 1939 alone (2657 us; 0.58 of
// twice the bf16 peak), 1650 in a long run under the power limit; with neither
// hand-off nor epilogue 2860 (operands from L2), hand-offs alone 2270, which is what
// bounds it: every 128 columns x 128 k of products, 64 x 4 clocks of the tensor core,
// pass through a barrier each way.  SM pairs (256 x 256 tiles, whose hand-offs cross
// SMs) 1340 with the hand-offs alone.
// Few tiles (kSplit): the CTAs of a cluster share a 128 x 128 tile, each takes a run
// of its K blocks; the sums meet in shared memory and are added in the CTAs' order.
// A warp of its own copies the scales of the next kScales blocks into shared
// memory (4-byte cp.async, so any strides): loaded by the epilogue itself, even
// four blocks ahead, they held it to one L2 access per block (1260 TFLOP/s).
// ---------------------------------------------------------------------------
namespace gemmb {
constexpr int BM = 128, BK = 128;             // one 128-byte row of e4m3 per K block
constexpr int GROUP_M = 16;                   // M tiles per raster group (operands in flight share L2)
constexpr int EPI_WARPS = 8, THREADS = 128 + 32 * EPI_WARPS;
constexpr int LAUNCH_REGS = 168, REGS_LOAD = 56, REGS_EPI = 224;  // 65536 / 384, in steps of 8
static_assert(128 * REGS_LOAD + 32 * EPI_WARPS * REGS_EPI <= THREADS * LAUNCH_REGS, "register split");
constexpr int kScales = 8;                    // blocks whose scales are on their way
constexpr int SUM_LD = 132;                   // kSplit: floats of a row of sums (+ 4: rows shift by four banks)
template <int BN>
struct Cfg {
  static constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = BN == 256 ? 4 : 6;
  static constexpr int STREAMS = BN / 128, NBUF = 4 / STREAMS;
  static constexpr int CW = BN / 2;           // columns of one epilogue warp
  static constexpr int SC_FLOATS = 132;       // 128 row scales, W scales of the streams
  static constexpr int OFF_SC = STAGES * STAGE;
  static constexpr int OFF_BAR = (OFF_SC + kScales * SC_FLOATS * 4 + 15) / 16 * 16;
  static constexpr int SMEM = OFF_BAR + 512 + 1024;
};
}  // namespace gemmb

// 4-byte asynchronous copy to shared memory; the arrival on `bar` once every earlier copy of this thread landed
__device__ __forceinline__ void cp_async4(uint32_t dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void ld_cluster(uint32_t a, float4& v) {
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
}

template <int BN, bool kSplit>
__global__ void __launch_bounds__(gemmb::THREADS, 1)
    gemm_block_tcgen05(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                            const GemmBlockParams p) {
  using namespace gemmb;
  using C = Cfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t bar0 = base + C::OFF_BAR;
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (C::STAGES + s); };
  auto acc_full = [&](int h, int a) { return bar0 + 8u * (2 * C::STAGES + C::NBUF * h + a); };
  auto acc_empty = [&](int h, int a) { return bar0 + 8u * (2 * C::STAGES + 4 + C::NBUF * h + a); };
  auto sc_full = [&](int s) { return bar0 + 8u * (2 * C::STAGES + 8 + s); };
  auto sc_empty = [&](int s) { return bar0 + 8u * (2 * C::STAGES + 8 + kScales + s); };
  const uint32_t drain = bar0 + 8u * (2 * C::STAGES + 8 + 2 * kScales);
  static_assert(8 * (2 * C::STAGES + 9 + 2 * kScales) <= 320, "barrier region");
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + C::OFF_BAR + 320);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + C::OFF_BAR + 328);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_tiles = p.tiles;
  const int all_k = (p.K + BK - 1) / BK;
  // this CTA's K blocks [kb0, kb0 + nk) and tiles
  const int rank = kSplit ? (int)cluster_ctarank() : 0, ks = kSplit ? p.ks : 1;
  const int kb0 = kSplit ? all_k * rank / ks : 0;
  const int nk = kSplit ? all_k * (rank + 1) / ks - kb0 : all_k;
  const int my_tiles = kSplit ? 1 : blockIdx.x < num_tiles ? (num_tiles - 1 - blockIdx.x) / gridDim.x + 1 : 0;
  auto tile_coords = [&](int lt, int& m0, int& n0) {
    int tile = kSplit ? blockIdx.x / ks : blockIdx.x + lt * gridDim.x, half = 0, width = BN;
    if (BN == 128 && p.tile0 >= 0) {  // the halves of the wide tiles from tile0 on
      half = tile & 1, width = 256;
      tile = p.tile0 + (tile >> 1);
    }
    const int num_m = (p.M + BM - 1) / BM, num_n = (p.N + width - 1) / width;
    const int per_group = GROUP_M * num_n;
    const int g = tile / per_group, r = tile % per_group;
    const int gm = min(GROUP_M, num_m - g * GROUP_M);
    m0 = (g * GROUP_M + r % gm) * BM;
    n0 = (r / gm) * width + 128 * half;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int h = 0; h < C::STREAMS; ++h)
      for (int a = 0; a < C::NBUF; ++a) {
        mbar_init(acc_full(h, a), 1);
        mbar_init(acc_empty(h, a), EPI_WARPS / C::STREAMS);
      }
    for (int c = 0; c < kScales; ++c) {
      mbar_init(sc_full(c), 32);
      mbar_init(sc_empty(c), EPI_WARPS);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&ta);
    prefetch_tmap(&tb);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // stream h, buffer a: columns [128 (NBUF h + a), + 128)

  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_LOAD));
  if (warp == 0) {
    if (elect_one()) {
      int it = 0;
      bool ok = true;
      for (int lt = 0; lt < my_tiles && ok; ++lt) {
        int m0, n0;
        tile_coords(lt, m0, n0);
        for (int kb = 0; kb < nk; ++kb, ++it) {
          const int s = it % C::STAGES;
          if (!mbar_spin(empty(s), ((it / C::STAGES) & 1) ^ 1, abort_flag, kDevTimeoutMma)) {
            ok = false;
            break;
          }
          const uint32_t sa = base + s * C::STAGE;
          mbar_expect_tx(full(s), C::STAGE);
          tma_load_2d(sa, &ta, full(s), (kb0 + kb) * BK, m0);
#pragma unroll
          for (int h = 0; h < C::STREAMS; ++h)
            tma_load_2d(sa + C::A_BYTES + h * 128 * BK, &tb, full(s), (kb0 + kb) * BK, n0 + 128 * h);
        }
      }
      // no load is still writing shared memory when the CTA exits
      const uint64_t deadline = globaltimer_ns() + kWaitLimitNs;
      bool drained = true;
      for (int k = max(0, it - C::STAGES); k < it && drained; ++k)
        drained = mbar_wait_until(full(k % C::STAGES), (k / C::STAGES) & 1, deadline);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = idesc_e4m3_f32(BM, 128);
      const int total = my_tiles * nk;
      bool ok = true;
      for (int it = 0; it < total && ok; ++it) {
        const int a = it % C::NBUF, s = it % C::STAGES;
        ok = mbar_spin(full(s), (it / C::STAGES) & 1, abort_flag, kDevTimeoutLoad);
        const uint32_t sa = base + s * C::STAGE, sb = sa + C::A_BYTES;
#pragma unroll
        for (int h = 0; h < C::STREAMS; ++h) {
          // the epilogue has read this accumulator (block it - NBUF)
          ok = ok && mbar_spin(acc_empty(h, a), ((it / C::NBUF) & 1) ^ 1, abort_flag, kDevTimeoutSoftmax);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f8_ss(tmem + 128 * (C::NBUF * h + a), sdesc_sw128(sa + kk * 32, 16, 1024),
                      sdesc_sw128(sb + h * 128 * BK + kk * 32, 16, 1024), idesc, kk > 0 ? 1u : 0u);
          mma_commit(acc_full(h, a));
        }
        if (ok) mma_commit(empty(s));
      }
      // every MMA issued has completed before TMEM is freed, also on the abort path
      mma_commit(drain);
      mbar_wait_until(drain, 0, globaltimer_ns() + kWaitLimitNs);
    }
  } else if (warp == 2) {
    // scales: slot c holds xs of the tile's 128 rows, then ws of its streams
    int it = 0;
    bool ok = true;
    for (int lt = 0; lt < my_tiles && ok; ++lt) {
      int m0, n0;
      tile_coords(lt, m0, n0);
      const float* ws = p.ws + (int64_t)min((n0 >> 7) + lane % C::STREAMS, (p.N - 1) >> 7) * p.ws_ld + kb0;
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int c = it % kScales;
        ok = __all_sync(0xffffffffu, mbar_spin(sc_empty(c), ((it / kScales) & 1) ^ 1, abort_flag, kDevTimeoutSoftmax));
        if (!ok) break;
        const uint32_t dst = base + C::OFF_SC + c * C::SC_FLOATS * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t m = min(m0 + 32 * i + lane, p.M - 1);
          cp_async4(dst + 4 * (32 * i + lane), p.xs + m * p.xs_sM + (kb0 + kb) * p.xs_sK);
        }
        if (lane < C::STREAMS) cp_async4(dst + 4 * (128 + lane), ws + kb);
        cp_async_arrive(sc_full(c));
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");  // no copy outlives the CTA
  } else if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_EPI));
    // warps 4-7: columns [0, CW) of the tile, warps 8-11: [CW, BN); TMEM lane quadrant = warp % 4
    const int q = warp & 3, group = (warp - 4) >> 2, h = C::STREAMS == 2 ? group : 0;
    const int row = q * 32 + lane;
    int it = 0;
    bool ok = true, ready = false;
    for (int lt = 0; lt < my_tiles && ok; ++lt) {
      int m0, n0;
      tile_coords(lt, m0, n0);
      const int64_t m = m0 + row;
      const int col = n0 + C::CW * group;
      uint64_t acc[C::CW / 32][16];
#pragma unroll
      for (int c = 0; c < C::CW / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[c][i] = 0ull;
      for (int kb = 0; kb < nk; ++kb, ++it) {
        // the block's scales and accumulator (`ready`: found complete while the block
        // before was still being added, so that the answer costs no time of its own)
        const int a = it % C::NBUF, c = it % kScales;
        if (!__all_sync(0xffffffffu, ready)) {
          const bool got = mbar_spin(sc_full(c), (it / kScales) & 1, abort_flag, kDevTimeoutLoad) &&
                           mbar_spin(acc_full(h, a), (it / C::NBUF) & 1, abort_flag, kDevTimeoutMma);
          ok = __all_sync(0xffffffffu, got);
          if (!ok) break;
        }
        tc_fence_after();
        const uint32_t t = tmem + 128 * (C::NBUF * h + a) + (C::CW * group) % 128 + ((uint32_t)(q * 32) << 16);
        uint32_t v[2][32];
        tmem_ld32(t, v[0]);
        const float* sc = reinterpret_cast<const float*>(gbase + C::OFF_SC) + c * C::SC_FLOATS;
        const float s = sc[row] * sc[128 + h];
        const uint64_t s2 = f2_pack(s, s);
#pragma unroll
        for (int i = 0; i < C::CW / 32; ++i) {
          tmem_ld_wait();
          if (i + 1 < C::CW / 32) {
            tmem_ld32(t + 32 * (i + 1), v[(i + 1) & 1]);
          } else {
            // the warp's part is in registers: the block NBUF further may overwrite it
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(acc_empty(h, a));
              mbar_arrive(sc_empty(c));
            }
            const int n = it + 1;
            ready = mbar_test(sc_full(n % kScales), (n / kScales) & 1) & mbar_test(acc_full(h, n % C::NBUF), (n / C::NBUF) & 1);
          }
          scaled_add(acc[i], v[i & 1], s2);
        }
      }
      if (kSplit) {
        // every load has landed and every product is done (the last block's was), so the
        // stages hold nothing any more: this CTA's sums take their place
        float4* dst = reinterpret_cast<float4*>(gbase + row * SUM_LD * 4 + C::CW * 4 * group);
#pragma unroll
        for (int c = 0; c < C::CW / 32; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float4 f;
            f2_unpack(acc[c][2 * i], f.x, f.y);
            f2_unpack(acc[c][2 * i + 1], f.z, f.w);
            if (ok) dst[8 * c + i] = f;
          }
      } else if (ok && m < p.M) {
        __nv_bfloat16* out = p.out + m * p.N;
#pragma unroll
        for (int c = 0; c < C::CW / 32; ++c) store_row(acc[c], p.bias, out, col + 32 * c, p.N);
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
  if (kSplit) {
    cluster_sync_all();  // every CTA's sums are in its shared memory
    int m0, n0;
    tile_coords(0, m0, n0);
    // rows [128 rank / ks, 128 (rank + 1) / ks): 16 threads a row, 8 columns each
    const int col = 8 * (threadIdx.x & 15);
    for (int row = 128 * rank / ks + (threadIdx.x >> 4); row < 128 * (rank + 1) / ks; row += THREADS / 16) {
      if (m0 + row >= p.M) break;
      float f[8] = {};
      for (int r = 0; r < ks; ++r) {
        const uint32_t src = mapa_shared(base + (row * SUM_LD + col) * 4, r);
        float4 a, b;
        ld_cluster(src, a);
        ld_cluster(src + 16, b);
        f[0] += a.x, f[1] += a.y, f[2] += a.z, f[3] += a.w;
        f[4] += b.x, f[5] += b.y, f[6] += b.z, f[7] += b.w;
      }
      const uint64_t acc[4] = {f2_pack(f[0], f[1]), f2_pack(f[2], f[3]), f2_pack(f[4], f[5]), f2_pack(f[6], f[7])};
      store_row(acc, p.bias, p.out + (int64_t)(m0 + row) * p.N, n0 + col, p.N);
    }
    __syncwarp();
    cluster_sync_all();  // no CTA leaves while another reads its sums
  }
}

// p.tiles tiles of 128 x BN
template <int BN>
static int launch_gemm_block_bn(const CUtensorMap& ta, const CUtensorMap& tb, const GemmBlockParams& p, int sms,
                                cudaStream_t s) {
  using C = gemmb::Cfg<BN>;
  static KernelReady ready;
  const int rc = kernel_ready(ready, gemm_block_tcgen05<BN, false>, C::SMEM, gemmb::LAUNCH_REGS);
  if (rc != 0) return rc;
  gemm_block_tcgen05<BN, false><<<p.tiles < sms ? p.tiles : sms, gemmb::THREADS, C::SMEM, s>>>(ta, tb, p);
  return (int)cudaGetLastError();
}

// p.tiles tiles of 128 x 128, p.ks CTAs each
static int launch_gemm_block_split(const CUtensorMap& ta, const CUtensorMap& tb, const GemmBlockParams& p,
                                   cudaStream_t s) {
  using C = gemmb::Cfg<128>;
  static_assert(128 * gemmb::SUM_LD * 4 <= C::OFF_SC, "the sums take the stages' place");
  static KernelReady ready;
  const int rc = kernel_ready(ready, gemm_block_tcgen05<128, true>, C::SMEM, gemmb::LAUNCH_REGS);
  if (rc != 0) return rc;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = (unsigned)p.ks;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.tiles * p.ks));
  cfg.blockDim = dim3(gemmb::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = s;
  cfg.attrs = &cluster;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, gemm_block_tcgen05<128, true>, ta, tb, p);
}

// p.tiles tiles of 128 x 128.  Few: their K blocks are cut over the CTAs of a cluster
// while most SMs can take one (clusters do not fill every group of SMs) and 8 blocks
// are left to each (us, whole | cut: 128 x 5120 x 5120 17.3 | 13.2 by 3, 128 x 1536 x
// 8960 25.4 | 14.0 by 4; 4 blocks each, 128 x 1536 x 1536 9.0 | 9.6)
static int gemm_block_cut(int64_t tiles, int K, int64_t sms) {
  const int64_t most = std::min<int64_t>(4, std::min(sms * 7 / 8 / tiles, (int64_t)((K + 127) / 128 / 8)));
  return most > 1 ? (int)most : 1;
}
static int launch_gemm_block_narrow(const CUtensorMap& ta, const CUtensorMap& tb, GemmBlockParams p, int sms,
                                    cudaStream_t s) {
  p.ks = gemm_block_cut(p.tiles, p.K, sms);
  return p.ks > 1 ? launch_gemm_block_split(ta, tb, p, s) : launch_gemm_block_bn<128>(ta, tb, p, sms, s);
}

// ---------------------------------------------------------------------------
// Few rows (M <= 8 NT): the weight is read once and little else matters, so the
// work is cut along N and K for bytes in flight: a CTA per 16 rows of wq, its 8
// warps take the K blocks in turn, and the partial sums meet in shared memory
// in warp order.  m16n8k32 MMAs with W as the row operand: a lane loads 16
// consecutive bytes of its W rows and of its token and uses them as the operand
// words of two MMAs; the order of k within a block is the same for both, which
// is all a sum over the block needs.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void mma_m16n8k32_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                  uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NT>
__global__ void __launch_bounds__(256) gemm_block_few_rows_kernel(const GemmBlockParams p) {
  __shared__ float s_part[8][16][8 * NT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16;
  const int nk = (p.K + 127) / 128;
  const uint8_t* w_lo = p.wq + (int64_t)(n0 + g) * p.K;
  const bool lo = n0 + g < p.N, hi = n0 + g + 8 < p.N;
  const float* ws = p.ws + (int64_t)(n0 / 128) * p.ws_ld;
  float acc[NT][4] = {};
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll(NT == 1 ? 2 : 1)
  for (int kb = warp; kb < nk; kb += 8) {
    uint4 wl[2], wh[2], xv[NT][2];
    float sx[NT][2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int k = kb * 128 + 64 * c + 16 * t;
      const bool in = k < p.K;
      wl[c] = in && lo ? __ldcs(reinterpret_cast<const uint4*>(w_lo + k)) : zero;
      wh[c] = in && hi ? __ldcs(reinterpret_cast<const uint4*>(w_lo + 8ll * p.K + k)) : zero;
#pragma unroll
      for (int j = 0; j < NT; ++j)
        xv[j][c] = in && 8 * j + g < p.M ? __ldg(reinterpret_cast<const uint4*>(p.xq + (int64_t)(8 * j + g) * p.K + k)) : zero;
    }
    const float sw = __ldg(ws + kb);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        sx[j][e] = __ldg(p.xs + (int64_t)min(8 * j + 2 * t + e, p.M - 1) * p.xs_sM + kb * p.xs_sK) * sw;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        mma_m16n8k32_e4m3(d, wl[c].x, wh[c].x, wl[c].y, wh[c].y, xv[j][c].x, xv[j][c].y);
        mma_m16n8k32_e4m3(d, wl[c].z, wh[c].z, wl[c].w, wh[c].w, xv[j][c].z, xv[j][c].w);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = fmaf(d[e], sx[j][e & 1], acc[j][e]);
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) s_part[warp][g + 8 * (e >> 1)][8 * j + 2 * t + (e & 1)] = acc[j][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * p.M; i += 256) {
    const int r = i & 15, m = i >> 4;
    if (n0 + r < p.N) {
      float v = 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) v += s_part[u][r][m];
      if (p.bias) v += bf2f(p.bias[n0 + r]);
      p.out[(int64_t)m * p.N + n0 + r] = f2bf(v);
    }
  }
}

template <int NT>
static int launch_gemm_block_few_rows(const GemmBlockParams& p, cudaStream_t s) {
  gemm_block_few_rows_kernel<NT><<<(p.N + 15) / 16, 256, 0, s>>>(p);
  return (int)cudaGetLastError();
}

int launch_gemm_block(const CUtensorMap& ta, const CUtensorMap& tb, GemmBlockParams p, cudaStream_t s) {
  // Up to 8 rows the weight's bytes decide (M = 8, us, few rows | tiles: N x K =
  // 15360 x 5120 18.9 | 19.5, 5120 x 5120 9.1 | 13.2, 1536 x 1536 3.7 | 7.8); from 9
  // to 16 the second token tile costs, and only small weights gain (M = 16: 29 |
  // 19.5, 15.5 | 13.2, 4.0 | 7.8).
  if (p.M <= 8) return launch_gemm_block_few_rows<1>(p, s);
  if (p.M <= 16 && (int64_t)p.N * p.K <= (16 << 20)) return launch_gemm_block_few_rows<2>(p, s);
  // Rounds of tiles over the SMs, in hundredths of a wide tile's time (a narrow one takes
  // about 0.6 of it, cut ones their part and 0.2; a second launch 0.1): wide tiles, narrow
  // ones, or whole rounds of wide tiles and the rest as narrow ones (M x N x K, us, the
  // three: 512 x 5120 x 5120 28.2 | 32.8 | -, 1001 x 5120 x 5120 50.0 | 46.0 | 39.8, 2048 x
  // 5120 x 5120 72.5 | - | 64.4, 4096 x 5120 x 5120 120 | 130 | 118, 32760 x 15360 x 5120
  // 2650 | 3040 | -)
  const int64_t sms = device_sms(), num_m = (p.M + 127) / 128;
  const int64_t wide = num_m * ((p.N + 255) / 256), narrow = num_m * ((p.N + 127) / 128);
  const int64_t full = wide / sms * sms, rest = wide - full;
  auto narrow_cost = [&](int64_t tiles) {
    const int ks = gemm_block_cut(tiles, p.K, sms);
    return ks > 1 ? 60 / ks + 20 : 60 * ((tiles + sms - 1) / sms);
  };
  const int64_t cost_wide = 100 * ((wide + sms - 1) / sms), cost_narrow = narrow_cost(narrow);
  const int64_t cost_both = full > 0 && rest > 0 ? 100 * (full / sms) + 10 + narrow_cost(2 * rest) : cost_wide;
  p.tile0 = -1;
  if (cost_narrow < cost_wide && cost_narrow <= cost_both) {
    p.tiles = (int)narrow;
    return launch_gemm_block_narrow(ta, tb, p, (int)sms, s);
  }
  p.tiles = (int)(cost_both < cost_wide ? full : wide);
  const int rc = launch_gemm_block_bn<256>(ta, tb, p, (int)sms, s);
  if (rc != 0 || p.tiles == wide) return rc;
  p.tile0 = (int)full, p.tiles = (int)(2 * rest);
  return launch_gemm_block_narrow(ta, tb, p, (int)sms, s);
}

}  // namespace rola
