// Root-mean-square norm of rows with the residual's addition, in one pass, and
// its backward; e4m3 quantisation of rows and of weights with one scale per
// block of 128.
//
//   h = round(x + res)                      (res's type; h = x without a residual)
//   r = (mean_k h^2 + eps)^-1/2             (fp32)
//   y = h r w                               rounded once: to bf16, or to e4m3 of
//   yq = e4m3(y / s),  s = amax |y| / 448 + 1e-12
// over each 128 columns of a row or over the whole row (the recipe of
// quantize_rows_e4m3_kernel, from the unrounded y).
//
// h is rounded before it is normalised: it is what the next sublayer reads, so
// y is the norm of the stored stream and the backward can start from h alone.
//
// The pass reads x and res and writes h and y, and does a few operations per
// element: memory bound.  A row stays in registers between its statistics and
// its output (8 columns a vector, NV vectors a thread); rows up to 1024 columns
// take a warp each (no barrier), longer ones a CTA, whose next rows are fetched by
// bulk copies meanwhile (loads by the threads themselves left the memory idle
// between a row's load and its barriers: 255 us instead of 206 in the first line).
// Measured: 32760 x 5120, x and res bf16, to e4m3: 206 us, 5.7 TB/s (0.88 of a copy's
// rate); 16381 x 1536, x and res bf16, to bf16: 37 us, 5.4 TB/s; forward and backward
// of 32760 x 5120, x bf16, res fp32, with the weight's gradient 771 us at 28 bytes an
// element, 6.1 TB/s (0.94); 4 rows 3.2 us, a launch.
#include <atomic>

#include "common.cuh"
#include "kernels.h"

namespace rola {

namespace norm {
constexpr int kQBlock = 128;     // columns that share a scale
constexpr float kE4M3Max = 448.f;
constexpr int kRing = 3, kRingBwd = 2;  // rows on their way per CTA, where shared memory holds them
constexpr size_t kRingBytes = 220 * 1024;
}  // namespace norm

// 8 consecutive columns as fp32
__device__ __forceinline__ void load8(const void* base, bool fp32, int64_t off, float (&v)[8]) {
  if (fp32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + off);
    const float4 a = p[0], b = p[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(base) + off);
    unpack_bf2(u.x, v[0], v[1]);
    unpack_bf2(u.y, v[2], v[3]);
    unpack_bf2(u.z, v[4], v[5]);
    unpack_bf2(u.w, v[6], v[7]);
  }
}
__device__ __forceinline__ void store8(void* base, bool fp32, int64_t off, const float (&v)[8]) {
  if (fp32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + off);
    __stcs(p, make_float4(v[0], v[1], v[2], v[3]));
    __stcs(p + 1, make_float4(v[4], v[5], v[6], v[7]));
  } else {
    __stcs(reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(base) + off),
           make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7])));
  }
}
// maximum that keeps a NaN of either side
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float e4m3_scale(float amax) {
  return __fadd_rn(__fdiv_rn(amax, norm::kE4M3Max), 1e-12f);
}
__device__ __forceinline__ uint2 pack8_e4m3(const float (&y)[8], float inv) {
  const uint32_t lo = (uint32_t)cvt_e4m3x2(y[0] * inv, y[1] * inv) | ((uint32_t)cvt_e4m3x2(y[2] * inv, y[3] * inv) << 16);
  const uint32_t hi = (uint32_t)cvt_e4m3x2(y[4] * inv, y[5] * inv) | ((uint32_t)cvt_e4m3x2(y[6] * inv, y[7] * inv) << 16);
  return make_uint2(lo, hi);
}

template <int WIDTH, typename Op>
__device__ __forceinline__ float lanes_reduce(float v, Op op) {
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
struct AddOp {
  __device__ float operator()(float a, float b) const { return a + b; }
};
struct MaxOp {
  __device__ float operator()(float a, float b) const { return max_nan(a, b); }
};

// Reduction over the threads that share a row: the warp (kWarpRow) or the CTA.
// `slot`: a shared array of 32 floats that no thread still reads (the callers
// take another one for each reduction between two barriers of the CTA).
template <bool kWarpRow, typename Op>
__device__ __forceinline__ float row_reduce(float v, float* slot, Op op, float zero) {
  v = lanes_reduce<32>(v, op);
  if (kWarpRow) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  if (lane == 0) slot[warp] = v;
  __syncthreads();
  return lanes_reduce<32>(lane < nw ? slot[lane] : zero, op);
}

enum : int { kOutBf16 = 0, kOutE4M3Block = 1, kOutE4M3Row = 2 };

// Everything after a row's loads: v holds x (and r the residual's values) of
// NV vectors, 0 past the row.  `slots`: two arrays for this row's reductions;
// `rows_read` runs once every thread of the row has its values in registers.
template <int NV, bool kWarpRow, int kOut, typename Read>
__device__ __forceinline__ void norm_row(const AddRmsNormParams& p, int64_t m, float (&v)[NV][8], float (*slots)[32],
                                         Read rows_read) {
  const int lane_in_row = kWarpRow ? (threadIdx.x & 31) : threadIdx.x;
  const int row_threads = kWarpRow ? 32 : blockDim.x;
  const int nvec = p.K >> 3;
  if (p.norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(v[i][e], v[i][e], ss);
    ss = row_reduce<kWarpRow>(ss, slots[0], AddOp(), 0.f);
    rows_read();
    const float r = rsqrtf(ss * (1.0f / (float)p.K) + p.eps);
    if (p.rstd && lane_in_row == 0) p.rstd[m] = r;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane_in_row + i * row_threads;
      if (c < nvec) {
        float w[8];
        load8(p.w, p.w_fp32, 8 * c, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * r * w[e];
      }
    }
  } else {
    if (!kWarpRow) __syncthreads();
    rows_read();
  }
  if (kOut == kOutBf16) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane_in_row + i * row_threads;
      if (c < nvec) store8(p.y, false, m * p.K + 8 * c, v[i]);
    }
  } else {
    float amax[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      amax[i] = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) amax[i] = max_nan(amax[i], fabsf(v[i][e]));
    }
    if (kOut == kOutE4M3Row) {
      float a = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) a = max_nan(a, amax[i]);
      a = row_reduce<kWarpRow>(a, slots[1], MaxOp(), 0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) amax[i] = a;
    } else {
      // 16 neighbouring threads hold the 128 columns of a scale
#pragma unroll
      for (int i = 0; i < NV; ++i) amax[i] = lanes_reduce<16>(amax[i], MaxOp());
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane_in_row + i * row_threads;
      if (c < nvec) {
        const float s = e4m3_scale(amax[i]);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.yq) + m * p.K + 8 * c) = pack8_e4m3(v[i], 1.0f / s);
        if (kOut == kOutE4M3Row) {
          if (c == 0) p.scale[m] = s;
        } else if ((c & 15) == 0) {
          p.scale[m * p.scale_sM + (c >> 4) * p.scale_sK] = s;
        }
      }
    }
  }
}

// v (x) += residual in the stream's type, stored as h
__device__ __forceinline__ void add_residual(const AddRmsNormParams& p, int64_t m, int c, const void* res, int64_t off,
                                             float (&v)[8]) {
  float r[8];
  load8(res, p.res_fp32, off, r);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] += r[e];
  if (!p.res_fp32) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) rbf2(v[e], v[e + 1]);
  }
  store8(p.h, p.res_fp32, m * p.K + 8 * c, v);
}

// rows of up to 1024 columns: one warp each
template <int NV, int kOut>
__global__ void __launch_bounds__(128) add_rms_norm_warp_kernel(const AddRmsNormParams p) {
  const int lane = threadIdx.x & 31, nvec = p.K >> 3;
  const int64_t step = (int64_t)gridDim.x * 4;
  for (int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5); m < p.M; m += step) {
    float v[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane + i * 32;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
      if (c < nvec) {
        load8(p.x, p.x_fp32, m * p.x_ld + 8 * c, v[i]);
        if (p.res) add_residual(p, m, c, p.res, m * p.res_ld + 8 * c, v[i]);
      }
    }
    norm_row<NV, true, kOut>(p, m, v, nullptr, [] {});
  }
}

// End of a ring's CTA of `rows` rows, whose thread 0 has seen the first `seen` arrive.
// Fewer than all only after a wait that ran out (which has set the device error; what
// was computed from there on is undefined): the copies on their way land before shared
// memory goes.
__device__ __forceinline__ void ring_drain(const uint64_t* bars, int ring, int rows, int seen) {
  if (threadIdx.x != 0 || seen == rows) return;
  const uint64_t deadline = globaltimer_ns() + kWaitLimitNs;
  const int fetched = min(rows, seen + ring);
  for (int n = seen; n < fetched; ++n)
    if (!mbar_wait_until(smem_u32(&bars[n % ring]), (n / ring) & 1, deadline)) return;
}

// Longer rows: a CTA each, the next rows on their way.  Thread 0 fetches whole
// rows of x and res by bulk copies into a ring of kRing shared-memory stages (fewer where rows are too long);
// the barrier of the row's reduction also says that its stage is free.
template <int NV, int kOut>
__global__ void __launch_bounds__(512) add_rms_norm_ring_kernel(const AddRmsNormParams p) {
  extern __shared__ __align__(128) uint8_t smem_ring[];
  __shared__ float s_red[2][2][32];
  __shared__ uint64_t s_bar[norm::kRing];
  const int nvec = p.K >> 3;
  const uint32_t xb = (uint32_t)p.K * (p.x_fp32 ? 4 : 2), rb = p.res ? (uint32_t)p.K * (p.res_fp32 ? 4 : 2) : 0u;
  const uint32_t stage = xb + rb;
  auto fetch = [&](int64_t m, int s) {
    const uint32_t dst = smem_u32(smem_ring) + s * stage, bar = smem_u32(&s_bar[s]);
    mbar_expect_tx(bar, stage);
    bulk_load(dst, static_cast<const uint8_t*>(p.x) + m * p.x_ld * (p.x_fp32 ? 4 : 2), xb, bar);
    if (rb) bulk_load(dst + xb, static_cast<const uint8_t*>(p.res) + m * p.res_ld * (p.res_fp32 ? 4 : 2), rb, bar);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.ring; ++s) mbar_init(smem_u32(&s_bar[s]), 1);
    fence_barrier_init();
    for (int s = 0; s < p.ring; ++s)
      if (blockIdx.x + (int64_t)s * gridDim.x < p.M) fetch(blockIdx.x + (int64_t)s * gridDim.x, s);
  }
  __syncthreads();
  int n = 0, seen = 0;  // rows; of them arrived (fewer once a wait has run out)
  for (int64_t m = blockIdx.x; m < p.M; m += gridDim.x, ++n) {
    const int s = n % p.ring;
    if (seen == n) seen += mbar_wait_until(smem_u32(&s_bar[s]), (n / p.ring) & 1, globaltimer_ns() + kWaitLimitNs);
    const uint8_t* xs = smem_ring + s * stage;
    float v[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
      if (c < nvec) {
        load8(xs, p.x_fp32, 8 * c, v[i]);
        if (rb) add_residual(p, m, c, xs + xb, 8 * c, v[i]);
      }
    }
    norm_row<NV, false, kOut>(p, m, v, s_red[n & 1], [&] {
      const int64_t next = m + (int64_t)p.ring * gridDim.x;
      if (threadIdx.x == 0 && seen > n && next < p.M) fetch(next, s);
    });
  }
  ring_drain(s_bar, p.ring, n, seen);
}

// Backward.  With u = h r (the unit rows), g = dy w:
//   dh = dh_in + r (g - u mean(g u));   dx = dres = dh, each in its own type
//   dw = sum_m dy u: every CTA sums its own rows in registers (fixed order) and
//   leaves one fp32 row of partials; dw_reduce_kernel adds them in order, so the
//   result does not depend on timing.
template <int NV, bool kWarpRow, typename Read>
__device__ __forceinline__ void norm_bwd_row(const AddRmsNormBwdParams& p, int64_t m, const void* h, int64_t h_off,
                                             const void* dy, int64_t dy_off, const void* dh, int64_t dh_off,
                                             float (&dw)[NV][8], float* slot, Read rows_read) {
  const int lane_in_row = kWarpRow ? (threadIdx.x & 31) : threadIdx.x;
  const int row_threads = kWarpRow ? 32 : blockDim.x;
  const int nvec = p.K >> 3;
  const float r = p.rstd[m];
  float u[NV][8], g[NV][8], d[NV][8];
  float gu = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = lane_in_row + i * row_threads;
    if (c < nvec) {
      float w[8];
      load8(h, p.h_fp32, h_off + 8 * c, u[i]);
      load8(dy, false, dy_off + 8 * c, g[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) d[i][e] = 0.f;
      if (dh) load8(dh, p.dh_fp32, dh_off + 8 * c, d[i]);
      load8(p.w, p.w_fp32, 8 * c, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u[i][e] *= r;
        dw[i][e] = fmaf(g[i][e], u[i][e], dw[i][e]);
        g[i][e] *= w[e];
        gu = fmaf(g[i][e], u[i][e], gu);
      }
    }
  }
  gu = row_reduce<kWarpRow>(gu, slot, AddOp(), 0.f) * (1.0f / (float)p.K);
  rows_read();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = lane_in_row + i * row_threads;
    if (c < nvec) {
#pragma unroll
      for (int e = 0; e < 8; ++e) d[i][e] = fmaf(r, g[i][e] - u[i][e] * gu, d[i][e]);
      store8(p.dx, p.dx_fp32, m * p.K + 8 * c, d[i]);
      if (p.dres) store8(p.dres, p.dres_fp32, m * p.K + 8 * c, d[i]);
    }
  }
}

template <int NV>
__device__ __forceinline__ void store_dw_part(const AddRmsNormBwdParams& p, int64_t prow, int lane_in_row,
                                              int row_threads, const float (&dw)[NV][8]) {
  if (p.dw_part == nullptr) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = lane_in_row + i * row_threads;
    if (c < (p.K >> 3)) store8(p.dw_part, true, prow * p.K + 8 * c, dw[i]);
  }
}

template <int NV>
__global__ void __launch_bounds__(128) add_rms_norm_bwd_warp_kernel(const AddRmsNormBwdParams p) {
  const int64_t first = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), step = (int64_t)gridDim.x * 4;
  float dw[NV][8] = {};
  for (int64_t m = first; m < p.M; m += step)
    norm_bwd_row<NV, true>(p, m, p.h, m * p.h_ld, p.dy, m * p.dy_ld, p.dh, m * p.dh_ld, dw, nullptr, [] {});
  store_dw_part<NV>(p, first, threadIdx.x & 31, 32, dw);  // one row of partials per warp
}

// rows h, dy and dh through a ring, as add_rms_norm_ring_kernel
template <int NV>
__global__ void __launch_bounds__(512) add_rms_norm_bwd_ring_kernel(const AddRmsNormBwdParams p) {
  extern __shared__ __align__(128) uint8_t smem_ring[];
  __shared__ float s_red[2][32];
  __shared__ uint64_t s_bar[norm::kRingBwd];
  const uint32_t hb = (uint32_t)p.K * (p.h_fp32 ? 4 : 2), yb = (uint32_t)p.K * 2;
  const uint32_t db = p.dh ? (uint32_t)p.K * (p.dh_fp32 ? 4 : 2) : 0u, stage = hb + yb + db;
  auto fetch = [&](int64_t m, int s) {
    const uint32_t dst = smem_u32(smem_ring) + s * stage, bar = smem_u32(&s_bar[s]);
    mbar_expect_tx(bar, stage);
    bulk_load(dst, static_cast<const uint8_t*>(p.h) + m * p.h_ld * (p.h_fp32 ? 4 : 2), hb, bar);
    bulk_load(dst + hb, static_cast<const uint8_t*>(p.dy) + m * p.dy_ld * 2, yb, bar);
    if (db) bulk_load(dst + hb + yb, static_cast<const uint8_t*>(p.dh) + m * p.dh_ld * (p.dh_fp32 ? 4 : 2), db, bar);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.ring; ++s) mbar_init(smem_u32(&s_bar[s]), 1);
    fence_barrier_init();
    for (int s = 0; s < p.ring; ++s)
      if (blockIdx.x + (int64_t)s * gridDim.x < p.M) fetch(blockIdx.x + (int64_t)s * gridDim.x, s);
  }
  __syncthreads();
  float dw[NV][8] = {};
  int n = 0, seen = 0;  // rows; of them arrived (fewer once a wait has run out)
  for (int64_t m = blockIdx.x; m < p.M; m += gridDim.x, ++n) {
    const int s = n % p.ring;
    if (seen == n) seen += mbar_wait_until(smem_u32(&s_bar[s]), (n / p.ring) & 1, globaltimer_ns() + kWaitLimitNs);
    const uint8_t* hs = smem_ring + s * stage;
    norm_bwd_row<NV, false>(p, m, hs, 0, hs + hb, 0, db ? hs + hb + yb : nullptr, 0, dw, s_red[n & 1], [&] {
      const int64_t next = m + (int64_t)p.ring * gridDim.x;
      if (threadIdx.x == 0 && seen > n && next < p.M) fetch(next, s);
    });
  }
  ring_drain(s_bar, p.ring, n, seen);
  store_dw_part<NV>(p, blockIdx.x, threadIdx.x, blockDim.x, dw);
}

// dw[k] = sum_g part[g, k] in order of g: 8 warps take every 8th row of 32 columns, then add up
__global__ void __launch_bounds__(256) dw_reduce_kernel(const float* __restrict__ part, int G, int K, void* dw,
                                                        int dw_fp32) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int k = blockIdx.x * 32 + lane;
  float a = 0.f;
  if (k < K)
    for (int g = warp; g < G; g += 8) a += part[(int64_t)g * K + k];
  s[warp][lane] = a;
  __syncthreads();
  if (warp == 0 && k < K) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += s[i][lane];
    if (dw_fp32) {
      static_cast<float*>(dw)[k] = t;
    } else {
      static_cast<__nv_bfloat16*>(dw)[k] = f2bf(t);
    }
  }
}

// Weight [N, K] (bf16 or fp32, row stride ld) -> e4m3 with one scale per 128 x 128
// block.  One CTA per block: 256 threads hold 64 values each (16 threads a row).
__global__ void __launch_bounds__(256) quantize_tiles_e4m3_kernel(const void* __restrict__ w, int w_fp32, int64_t ld,
                                                                  int N, int K, uint8_t* __restrict__ wq,
                                                                  float* __restrict__ scale, int64_t scale_ld) {
  __shared__ float s_max[8];
  const int n0 = blockIdx.y * 128, c = blockIdx.x * 16 + (threadIdx.x & 15);
  float v[8][8];
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = n0 + (threadIdx.x >> 4) + 16 * i;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
    if (n < N && c < (K >> 3)) load8(w, w_fp32 != 0, n * ld + 8 * c, v[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) a = max_nan(a, fabsf(v[i][e]));
  }
  a = lanes_reduce<32>(a, MaxOp());
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = a;
  __syncthreads();
  a = s_max[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) a = max_nan(a, s_max[i]);
  const float s = e4m3_scale(a), inv = 1.0f / s;
  if (threadIdx.x == 0) scale[blockIdx.y * scale_ld + blockIdx.x] = s;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = n0 + (threadIdx.x >> 4) + 16 * i;
    if (n < N && c < (K >> 3)) *reinterpret_cast<uint2*>(wq + (int64_t)n * K + 8 * c) = pack8_e4m3(v[i], inv);
  }
}

// Vectors per thread and threads of a launch for rows of K columns
struct NormShape {
  int nv, threads;
  bool warp_row;
};
static NormShape norm_shape(int K) {
  const int nvec = K / 8;
  if (nvec <= 128) return {nvec <= 32 ? 1 : nvec <= 64 ? 2 : 4, 128, true};
  const int nv = nvec <= 1024 ? 2 : 4;
  return {nv, ((nvec + nv - 1) / nv + 31) / 32 * 32, false};
}

static int device_sms() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
    return 148;
  return sms;
}

// What a kernel's launches need once per device: its dynamic shared memory
// allowed and, where it splits its registers by setmaxnreg, as many of them as
// the split assumes (an increase beyond the launch's would wait).  One static
// KernelReady per kernel; a race of two first calls sets the same twice.
struct KernelReady {
  std::atomic<bool> done[64];
};
template <typename Kernel>
static int kernel_ready(KernelReady& r, Kernel* k, int smem, int min_regs = 0) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 0 && dev < 64 && r.done[dev].load(std::memory_order_acquire)) return 0;
  if (min_regs > 0) {
    cudaFuncAttributes fa;
    if ((e = cudaFuncGetAttributes(&fa, k)) != cudaSuccess) return (int)e;
    if (fa.numRegs < min_regs) return -1;
  }
  if ((e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return (int)e;
  if (dev >= 0 && dev < 64) r.done[dev].store(true, std::memory_order_release);
  return 0;
}

// CTAs that walk M rows: all at once when they are few, else as many as the
// SMs hold at `bytes` of shared memory a CTA
static int64_t norm_ctas(int64_t M, const NormShape& s, size_t bytes, int most) {
  const int64_t need = s.warp_row ? (M + 3) / 4 : M;
  int per_sm = most;
  if (!s.warp_row) {
    per_sm = (int)(norm::kRingBytes / bytes);
    if (per_sm > most) per_sm = most;
    if (per_sm < 1) per_sm = 1;
  }
  const int64_t cap = (int64_t)device_sms() * per_sm;
  return need < cap ? need : cap;
}

static int ring_depth(size_t stage, int most) {
  const int fit = (int)(norm::kRingBytes / stage);
  return fit < most ? (fit < 1 ? 1 : fit) : most;
}

template <int NV, int kOut>
static int launch_norm_ring(const AddRmsNormParams& p, const NormShape& s, unsigned grid, size_t smem,
                            cudaStream_t st) {
  static KernelReady ready;
  const int rc = kernel_ready(ready, add_rms_norm_ring_kernel<NV, kOut>, 224 * 1024);
  if (rc == 0) add_rms_norm_ring_kernel<NV, kOut><<<grid, s.threads, smem, st>>>(p);
  return rc;
}

template <int kOut>
static int launch_norm_out(AddRmsNormParams p, cudaStream_t st) {
  const NormShape s = norm_shape(p.K);
  const size_t stage = (size_t)p.K * ((p.x_fp32 ? 4 : 2) + (p.res ? (p.res_fp32 ? 4 : 2) : 0));
  p.ring = ring_depth(stage, norm::kRing);
  const size_t smem = p.ring * stage;
  const unsigned grid = (unsigned)norm_ctas(p.M, s, smem + 1024, s.warp_row ? 16 : 2048 / s.threads);
  if (!s.warp_row)
    return s.nv == 2 ? launch_norm_ring<2, kOut>(p, s, grid, smem, st) : launch_norm_ring<4, kOut>(p, s, grid, smem, st);
  if (s.nv == 1) add_rms_norm_warp_kernel<1, kOut><<<grid, s.threads, 0, st>>>(p);
  else if (s.nv == 2) add_rms_norm_warp_kernel<2, kOut><<<grid, s.threads, 0, st>>>(p);
  else add_rms_norm_warp_kernel<4, kOut><<<grid, s.threads, 0, st>>>(p);
  return 0;
}

int launch_add_rms_norm(const AddRmsNormParams& p, cudaStream_t s) {
  const int rc = p.y ? launch_norm_out<kOutBf16>(p, s)
                     : p.scale_row ? launch_norm_out<kOutE4M3Row>(p, s) : launch_norm_out<kOutE4M3Block>(p, s);
  return rc != 0 ? rc : (int)cudaGetLastError();
}

// the grid, and with it the order of dw's sums, follows from M, K and the
// widest row (fp32 h and dh), not from the types at hand
static int64_t norm_bwd_ctas(int64_t M, int K) {
  const NormShape s = norm_shape(K);
  return norm_ctas(M, s, (size_t)ring_depth((size_t)K * 10, norm::kRingBwd) * K * 10 + 1024, s.warp_row ? 4 : 2);
}

int add_rms_norm_bwd_parts(int64_t M, int K) {
  return (int)(norm_bwd_ctas(M, K) * (norm_shape(K).warp_row ? 4 : 1));
}

template <int NV>
static int launch_norm_bwd_ring(AddRmsNormBwdParams p, int threads, unsigned grid, cudaStream_t st) {
  static KernelReady ready;
  const int rc = kernel_ready(ready, add_rms_norm_bwd_ring_kernel<NV>, 224 * 1024);
  const size_t stage = (size_t)p.K * ((p.h_fp32 ? 4 : 2) + 2 + (p.dh ? (p.dh_fp32 ? 4 : 2) : 0));
  p.ring = ring_depth((size_t)p.K * 10, norm::kRingBwd);
  const size_t smem = p.ring * stage;
  if (rc == 0) add_rms_norm_bwd_ring_kernel<NV><<<grid, threads, smem, st>>>(p);
  return rc;
}

int launch_add_rms_norm_bwd(const AddRmsNormBwdParams& p, cudaStream_t st) {
  const NormShape s = norm_shape(p.K);
  const unsigned grid = (unsigned)norm_bwd_ctas(p.M, p.K);
  int rc = 0;
  if (!s.warp_row) {
    rc = s.nv == 2 ? launch_norm_bwd_ring<2>(p, s.threads, grid, st) : launch_norm_bwd_ring<4>(p, s.threads, grid, st);
  } else if (s.nv == 1) {
    add_rms_norm_bwd_warp_kernel<1><<<grid, s.threads, 0, st>>>(p);
  } else if (s.nv == 2) {
    add_rms_norm_bwd_warp_kernel<2><<<grid, s.threads, 0, st>>>(p);
  } else {
    add_rms_norm_bwd_warp_kernel<4><<<grid, s.threads, 0, st>>>(p);
  }
  if (rc == 0) rc = (int)cudaGetLastError();
  if (rc != 0) return rc;
  if (p.dw) {
    const int parts = add_rms_norm_bwd_parts(p.M, p.K);
    dw_reduce_kernel<<<(p.K + 31) / 32, 256, 0, st>>>(p.dw_part, parts, p.K, p.dw, p.w_fp32);
  }
  return (int)cudaGetLastError();
}

int launch_quantize_tiles_e4m3(const void* w, bool w_fp32, int64_t ld, int N, int K, uint8_t* wq, float* scale,
                               int64_t scale_ld, cudaStream_t s) {
  quantize_tiles_e4m3_kernel<<<dim3((K + 127) / 128, (N + 127) / 128), 256, 0, s>>>(w, w_fp32, ld, N, K, wq, scale,
                                                                                 scale_ld);
  return (int)cudaGetLastError();
}

}  // namespace rola
