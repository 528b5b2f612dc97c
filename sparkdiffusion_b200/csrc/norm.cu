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
// take a warp each (no barrier), longer ones a CTA.
#include "common.cuh"
#include "kernels.h"

namespace rola {

namespace norm {
constexpr int kQBlock = 128;     // columns that share a scale
constexpr float kE4M3Max = 448.f;
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
    p[0] = make_float4(v[0], v[1], v[2], v[3]);
    p[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(base) + off) =
        make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7]));
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

template <int NV, bool kWarpRow, int kOut>
__global__ void __launch_bounds__(kWarpRow ? 128 : 512) add_rms_norm_kernel(const AddRmsNormParams p) {
  __shared__ float s_red[2][2][32];
  const int lane_in_row = kWarpRow ? (threadIdx.x & 31) : threadIdx.x;
  const int row_threads = kWarpRow ? 32 : blockDim.x;
  const int rows_per_cta = kWarpRow ? (blockDim.x >> 5) : 1;
  const int64_t first = (int64_t)blockIdx.x * rows_per_cta + (kWarpRow ? (threadIdx.x >> 5) : 0);
  const int64_t step = (int64_t)gridDim.x * rows_per_cta;
  const int nvec = p.K >> 3;
  const float inv_k = 1.0f / (float)p.K;
  int parity = 0;
  for (int64_t m = first; m < p.M; m += step, parity ^= 1) {
    float v[NV][8];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane_in_row + i * row_threads;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
      if (c < nvec) {
        load8(p.x, p.x_fp32, m * p.x_ld + 8 * c, v[i]);
        if (p.res) {
          float r[8];
          load8(p.res, p.res_fp32, m * p.res_ld + 8 * c, r);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] += r[e];
          if (!p.res_fp32) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) rbf2(v[i][e], v[i][e + 1]);
          }
          store8(p.h, p.res_fp32, m * p.K + 8 * c, v[i]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(v[i][e], v[i][e], ss);
      }
    }
    if (p.norm) {
      ss = row_reduce<kWarpRow>(ss, s_red[parity][0], AddOp(), 0.f);
      const float r = rsqrtf(ss * inv_k + p.eps);
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
        a = row_reduce<kWarpRow>(a, s_red[parity][1], MaxOp(), 0.f);
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
}

// Backward.  With u = h r (the unit rows), g = dy w:
//   dh = dh_in + r (g - u mean(g u));   dx = dres = dh, each in its own type
//   dw = sum_m dy u: every CTA sums its own rows in registers (fixed order) and
//   leaves one fp32 row of partials; dw_reduce_kernel adds them in order, so the
//   result does not depend on timing.
template <int NV, bool kWarpRow>
__global__ void __launch_bounds__(kWarpRow ? 128 : 512) add_rms_norm_bwd_kernel(const AddRmsNormBwdParams p) {
  __shared__ float s_red[2][32];
  const int lane_in_row = kWarpRow ? (threadIdx.x & 31) : threadIdx.x;
  const int row_threads = kWarpRow ? 32 : blockDim.x;
  const int rows_per_cta = kWarpRow ? (blockDim.x >> 5) : 1;
  const int64_t first = (int64_t)blockIdx.x * rows_per_cta + (kWarpRow ? (threadIdx.x >> 5) : 0);
  const int64_t step = (int64_t)gridDim.x * rows_per_cta;
  const int nvec = p.K >> 3;
  const float inv_k = 1.0f / (float)p.K;
  float dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = 0.f;
  int parity = 0;
  for (int64_t m = first; m < p.M; m += step, parity ^= 1) {
    const float r = p.rstd[m];
    float u[NV][8], g[NV][8];
    float gu = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane_in_row + i * row_threads;
      if (c < nvec) {
        float w[8];
        load8(p.h, p.h_fp32, m * p.h_ld + 8 * c, u[i]);
        load8(p.dy, false, m * p.dy_ld + 8 * c, g[i]);
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
    gu = row_reduce<kWarpRow>(gu, s_red[parity], AddOp(), 0.f) * inv_k;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane_in_row + i * row_threads;
      if (c < nvec) {
        float d[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = r * (g[i][e] - u[i][e] * gu);
        if (p.dh) {
          float in[8];
          load8(p.dh, p.dh_fp32, m * p.dh_ld + 8 * c, in);
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] += in[e];
        }
        store8(p.dx, p.dx_fp32, m * p.K + 8 * c, d);
        if (p.dres) store8(p.dres, p.dres_fp32, m * p.K + 8 * c, d);
      }
    }
  }
  if (p.dw_part) {
    const int64_t prow = kWarpRow ? first : (int64_t)blockIdx.x;  // one row of partials per warp or CTA
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane_in_row + i * row_threads;
      if (c < nvec) store8(p.dw_part, true, prow * p.K + 8 * c, dw[i]);
    }
  }
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
  const int nv = nvec <= 512 ? 2 : 4;
  return {nv, ((nvec + nv - 1) / nv + 31) / 32 * 32, false};
}

static int device_sms() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
    return 148;
  return sms;
}

// CTAs that walk M rows: all at once when they are few, else a whole number per SM
static int64_t norm_ctas(int64_t M, const NormShape& s, int per_sm) {
  const int64_t need = s.warp_row ? (M + 3) / 4 : M;
  const int64_t cap = (int64_t)device_sms() * per_sm;
  return need < cap ? need : cap;
}

template <int kOut>
static void launch_norm_out(const AddRmsNormParams& p, const NormShape& s, unsigned grid, cudaStream_t st) {
  if (s.warp_row) {
    if (s.nv == 1) add_rms_norm_kernel<1, true, kOut><<<grid, s.threads, 0, st>>>(p);
    else if (s.nv == 2) add_rms_norm_kernel<2, true, kOut><<<grid, s.threads, 0, st>>>(p);
    else add_rms_norm_kernel<4, true, kOut><<<grid, s.threads, 0, st>>>(p);
  } else {
    if (s.nv == 2) add_rms_norm_kernel<2, false, kOut><<<grid, s.threads, 0, st>>>(p);
    else add_rms_norm_kernel<4, false, kOut><<<grid, s.threads, 0, st>>>(p);
  }
}

int launch_add_rms_norm(const AddRmsNormParams& p, cudaStream_t s) {
  const NormShape sh = norm_shape(p.K);
  const unsigned grid = (unsigned)norm_ctas(p.M, sh, 16);
  if (p.y) launch_norm_out<kOutBf16>(p, sh, grid, s);
  else if (p.scale_row) launch_norm_out<kOutE4M3Row>(p, sh, grid, s);
  else launch_norm_out<kOutE4M3Block>(p, sh, grid, s);
  return (int)cudaGetLastError();
}

int add_rms_norm_bwd_parts(int64_t M, int K) {
  const NormShape s = norm_shape(K);
  return (int)(norm_ctas(M, s, 2) * (s.warp_row ? 4 : 1));
}

int launch_add_rms_norm_bwd(const AddRmsNormBwdParams& p, cudaStream_t st) {
  const NormShape s = norm_shape(p.K);
  const unsigned grid = (unsigned)norm_ctas(p.M, s, 2);
  if (s.warp_row) {
    if (s.nv == 1) add_rms_norm_bwd_kernel<1, true><<<grid, s.threads, 0, st>>>(p);
    else if (s.nv == 2) add_rms_norm_bwd_kernel<2, true><<<grid, s.threads, 0, st>>>(p);
    else add_rms_norm_bwd_kernel<4, true><<<grid, s.threads, 0, st>>>(p);
  } else {
    if (s.nv == 2) add_rms_norm_bwd_kernel<2, false><<<grid, s.threads, 0, st>>>(p);
    else add_rms_norm_bwd_kernel<4, false><<<grid, s.threads, 0, st>>>(p);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return (int)e;
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
