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
#include "common.cuh"
#include "kernels.h"

namespace rola {

namespace gemmb {
constexpr int BM = 128, BK = 128;   // one 128-byte row of e4m3 per K block
constexpr int GROUP_M = 16;         // M tiles per raster group (A and W tiles in flight share L2)
template <int BN>
struct Cfg {
  static constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = BN >= 128 ? 6 : 8;
  static constexpr int NBUF = 4;                   // block accumulators in TMEM
  static constexpr int COLS = NBUF * BN;
  static constexpr int OFF_BAR = STAGES * STAGE;
  static constexpr int SMEM = OFF_BAR + 512 + 1024;
};
}  // namespace gemmb

// acc[0 .. 31] += v * s for 32 columns, two at a time
__device__ __forceinline__ void scaled_add32(uint64_t (&acc)[16], const uint32_t (&v)[32], uint64_t s2) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    acc[i] = fma_f32x2(f2_pack(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), s2, acc[i]);
}

// 32 finished columns of one row: bias, rounding, 16-byte stores of 8 columns
__device__ __forceinline__ void store_row32(const uint64_t (&acc)[16], const __nv_bfloat16* bias, __nv_bfloat16* row,
                                            int col, int N) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
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

template <int BN>
__global__ void __launch_bounds__(192, 1)
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
  auto acc_full = [&](int a) { return bar0 + 8u * (2 * C::STAGES + a); };
  auto acc_empty = [&](int a) { return bar0 + 8u * (2 * C::STAGES + C::NBUF + a); };
  const uint32_t drain = bar0 + 8u * (2 * C::STAGES + 2 * C::NBUF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + C::OFF_BAR + 256);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + C::OFF_BAR + 264);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_m = (p.M + BM - 1) / BM, num_n = (p.N + BN - 1) / BN;
  const int num_tiles = num_m * num_n;
  const int nk = (p.K + BK - 1) / BK;
  const int my_tiles = blockIdx.x < num_tiles ? (num_tiles - 1 - blockIdx.x) / gridDim.x + 1 : 0;
  auto tile_coords = [&](int lt, int& m0, int& n0) {
    const int tile = blockIdx.x + lt * gridDim.x;
    const int per_group = GROUP_M * num_n;
    const int g = tile / per_group, r = tile % per_group;
    const int gm = min(GROUP_M, num_m - g * GROUP_M);
    m0 = (g * GROUP_M + r % gm) * BM;
    n0 = (r / gm) * BN;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int a = 0; a < C::NBUF; ++a) {
      mbar_init(acc_full(a), 1);
      mbar_init(acc_empty(a), 4);  // one arrival per epilogue warp
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&ta);
    prefetch_tmap(&tb);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), C::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      int it = 0;
      bool ok = true;
      for (int lt = 0; lt < my_tiles && ok; ++lt) {
        int m0, n0;
        tile_coords(lt, m0, n0);
        for (int kb = 0; kb < nk; ++kb, ++it) {
          const int s = it % C::STAGES;
          if (!mbar_wait(empty(s), ((it / C::STAGES) & 1) ^ 1, abort_flag, kDevTimeoutMma)) {
            ok = false;
            break;
          }
          const uint32_t sa = base + s * C::STAGE;
          mbar_expect_tx(full(s), C::STAGE);
          tma_load_2d(sa, &ta, full(s), kb * BK, m0);
          tma_load_2d(sa + C::A_BYTES, &tb, full(s), kb * BK, n0);
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
      constexpr uint32_t idesc = idesc_e4m3_f32(BM, BN);
      const int total = my_tiles * nk;
      for (int it = 0; it < total; ++it) {
        const int a = it % C::NBUF, s = it % C::STAGES;
        // the epilogue has read this accumulator (block it - NBUF)
        if (!mbar_wait(acc_empty(a), ((it / C::NBUF) & 1) ^ 1, abort_flag, kDevTimeoutSoftmax)) break;
        if (!mbar_wait(full(s), (it / C::STAGES) & 1, abort_flag, kDevTimeoutLoad)) break;
        tc_fence_after();
        const uint32_t sa = base + s * C::STAGE, sb = sa + C::A_BYTES;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_f8_ss(tmem + a * BN, sdesc_sw128(sa + kk * 32, 16, 1024), sdesc_sw128(sb + kk * 32, 16, 1024), idesc,
                    kk > 0 ? 1u : 0u);
        mma_commit(empty(s));
        mma_commit(acc_full(a));
      }
      // every MMA issued has completed before TMEM is freed, also on the abort path
      mma_commit(drain);
      mbar_wait_until(drain, 0, globaltimer_ns() + kWaitLimitNs);
    }
  } else {
    // epilogue warps 2..5: TMEM lane quadrant = warp % 4, thread = row of the tile
    const int q = warp & 3;
    const int row = q * 32 + lane;
    int it = 0;
    bool ok = true;
    for (int lt = 0; lt < my_tiles && ok; ++lt) {
      int m0, n0;
      tile_coords(lt, m0, n0);
      const int64_t m = m0 + row;
      const float* xs = p.xs + (m < p.M ? m : 0) * p.xs_sM;
      const float* ws = p.ws + (int64_t)(n0 / 128) * p.ws_ld;
      uint64_t acc[BN / 32][16];
#pragma unroll
      for (int c = 0; c < BN / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[c][i] = 0ull;
      float s_next = __ldg(xs) * __ldg(ws);
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int a = it % C::NBUF;
        const float s = s_next;
        if (kb + 1 < nk) s_next = __ldg(xs + (kb + 1) * p.xs_sK) * __ldg(ws + kb + 1);
        ok = __all_sync(0xffffffffu, mbar_wait(acc_full(a), (it / C::NBUF) & 1, abort_flag, kDevTimeoutMma));
        if (!ok) break;
        tc_fence_after();
        const uint32_t t = tmem + a * BN + ((uint32_t)(q * 32) << 16);
        const uint64_t s2 = f2_pack(s, s);
        uint32_t v[2][32];
        tmem_ld32(t, v[0]);
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) {
          tmem_ld_wait();
          if (c + 1 < BN / 32) {
            tmem_ld32(t + 32 * (c + 1), v[(c + 1) & 1]);
          } else {
            // the whole accumulator is in registers: the next block may overwrite it
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty(a));
          }
          scaled_add32(acc[c], v[c & 1], s2);
        }
      }
      if (ok && m < p.M) {
        __nv_bfloat16* out = p.out + m * p.N;
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) store_row32(acc[c], p.bias, out, n0 + 32 * c, p.N);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::COLS);
  }
}

template <int BN>
static int launch_gemm_block_1sm(const CUtensorMap& ta, const CUtensorMap& tb, const GemmBlockParams& p, int sms,
                                 cudaStream_t s) {
  using C = gemmb::Cfg<BN>;
  cudaError_t e = cudaFuncSetAttribute(gemm_block_tcgen05<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return (int)e;
  const int64_t tiles = (int64_t)((p.M + 127) / 128) * ((p.N + BN - 1) / BN);
  gemm_block_tcgen05<BN><<<(unsigned)(tiles < sms ? tiles : sms), 192, C::SMEM, s>>>(ta, tb, p);
  return (int)cudaGetLastError();
}

int gemm_block_w_rows(int, int, int) { return 128; }

int launch_gemm_block(const CUtensorMap& ta, const CUtensorMap& tb, const GemmBlockParams& p, cudaStream_t s) {
  return launch_gemm_block_1sm<128>(ta, tb, p, device_sms(), s);
}

}  // namespace rola
