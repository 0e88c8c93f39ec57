// The residual's addition with its root-mean-square norm, 8-bit output and gradients.
//
//   t = dt(x + gate y)                            the residual stream, rounded to its type; the norm reads it so
//   r = rsqrt(mean t^2 + eps),  h = t r w (1 + scale) + shift          in 32 bits, rounded once where h is written
//   z = h H per block of 256 (the rotation of the W4A8 linears),  step = max|z| / 127,  code = rint(z / step)
//   gradients, from dt_out (of t) and dh (of h):  u = dh (1 + scale) w,  d = dt_out + r (u - t r mean(u t r)),
//     dx = d,  dy = gate d,  dw = sum over the rows of dh (1 + scale) t r
// gate, scale and shift are rows of the token's segment; a row outside every segment keeps t = x, h = t r w (dy = 0).  Without a
// gate t = x + y everywhere.
#pragma once
#include <type_traits>

#include "h3b_common.cuh"
#include "launch.h"

namespace h3b {

template <int DT>
__device__ __forceinline__ float rn_load(const void* p, int64_t i) {
  if constexpr (DT == H3B_FP32) return static_cast<const float*>(p)[i];
  else if constexpr (DT == H3B_FP16) return __half2float(static_cast<const __half*>(p)[i]);
  else return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ float rn_load(const void* p, int64_t i, int dt) {
  return dt == H3B_FP32 ? rn_load<H3B_FP32>(p, i) : dt == H3B_FP16 ? rn_load<H3B_FP16>(p, i) : rn_load<H3B_BF16>(p, i);
}
template <int DT>
__device__ __forceinline__ void rn_store(void* p, int64_t i, float v) {
  if constexpr (DT == H3B_FP16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}
template <int DT>
__device__ __forceinline__ float rn_round(float v) {
  if constexpr (DT == H3B_FP16) return __half2float(__float2half_rn(v));
  else return __bfloat162float(__float2bfloat16_rn(v));
}
__device__ __forceinline__ float rn_block_sum(float v, float* part) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) v += part[i];
  return v;
}
__device__ __forceinline__ int rn_mod_row(const ResNormArgs& a, int64_t r) {
  int m = -1;
  if (a.token_rows) {
    m = a.token_rows[r];
    return m < a.n_rows ? m : -1;
  }
  for (int s = 0; s < a.segs.n; ++s)
    if (r >= a.segs.first[s] && r < a.segs.end[s]) m = a.segs.row[s];
  return m;
}

template <int DT>
__global__ void __launch_bounds__(256) resnorm_kernel(const ResNormArgs a) {
  extern __shared__ float z[];
  __shared__ float part[8];
  const int64_t r = blockIdx.x;
  const int mrow = rn_mod_row(a, r);
  const int K = a.K;
  float ss = 0.f;
  for (int c = threadIdx.x; c < K; c += 256) {
    float v = rn_load<DT>(a.x, r * a.ldx + c);
    if (!a.gate) v = __fadd_rn(v, rn_load<DT>(a.y, r * a.ldy + c));
    else if (mrow >= 0) v = __fadd_rn(v, __fmul_rn(rn_load<DT>(a.y, r * a.ldy + c), rn_load(a.gate, mrow * a.ldm + c, a.m_dtype)));
    v = rn_round<DT>(v);
    rn_store<DT>(a.t, r * a.ldt + c, v);
    z[c] = v;
    ss += v * v;
  }
  ss = rn_block_sum(ss, part);
  const float rs = rsqrtf(ss / K + a.eps);
  if (a.rstd && threadIdx.x == 0) a.rstd[r] = rs;
  for (int c = threadIdx.x; c < K; c += 256) {
    float v = z[c] * rs * rn_load(a.w, c, a.w_dtype);
    if (a.scale && mrow >= 0)
      v = v * (1.f + rn_load(a.scale, mrow * a.ldm + c, a.m_dtype)) + rn_load(a.shift, mrow * a.ldm + c, a.m_dtype);
    z[c] = v;
    if (a.h) rn_store<DT>(a.h, r * a.ldh + c, v);
  }
  if (!a.codes) return;
  for (int step = 1; step < 256; step *= 4) {
    __syncthreads();
    for (int i = threadIdx.x; i < K / 4; i += 256) {
      const int at = i / step * 4 * step + i % step;
      const float v0 = z[at], v1 = z[at + step], v2 = z[at + 2 * step], v3 = z[at + 3 * step], s = (v0 + v1) + (v2 + v3);
      z[at] = 0.5f * s - v3, z[at + step] = 0.5f * s - v2, z[at + 2 * step] = 0.5f * s - v1, z[at + 3 * step] = 0.5f * s - v0;
    }
  }
  __syncthreads();
  unsigned top = 0;
  for (int c = threadIdx.x; c < K; c += 256) top = max(top, __float_as_uint(z[c]) & 0x7FFFFFFFu);
  top = __reduce_max_sync(0xffffffffu, top);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = __uint_as_float(top);
  __syncthreads();
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(part[i]));
  const float amax = __uint_as_float(top), inv = amax > 0.f && amax < INFINITY ? 127.f / amax : 0.f;
  if (threadIdx.x == 0) a.scales[r] = amax / 127.f;
  for (int c = threadIdx.x; c < K; c += 256) a.codes[r * a.ldc + c] = inv > 0.f ? static_cast<int8_t>(rintf(z[c] * inv)) : 0;
}

template <int DT>
__global__ void __launch_bounds__(256) resnorm_grad_kernel(const ResNormArgs a) {
  __shared__ float part[8];
  const int64_t r = blockIdx.x;
  const int mrow = rn_mod_row(a, r);
  const float rs = a.rstd[r];
  float dot = 0.f;
  for (int c = threadIdx.x; c < a.K; c += 256) {
    float u = rn_load<DT>(a.dh, r * a.lddh + c) * rn_load(a.w, c, a.w_dtype);
    if (a.scale && mrow >= 0) u *= 1.f + rn_load(a.scale, mrow * a.ldm + c, a.m_dtype);
    dot += u * (rn_load<DT>(a.t, r * a.ldt + c) * rs);
  }
  dot = rn_block_sum(dot, part) / a.K;
  for (int c = threadIdx.x; c < a.K; c += 256) {
    float u = rn_load<DT>(a.dh, r * a.lddh + c) * rn_load(a.w, c, a.w_dtype);
    if (a.scale && mrow >= 0) u *= 1.f + rn_load(a.scale, mrow * a.ldm + c, a.m_dtype);
    const float d = (a.dt ? rn_load<DT>(a.dt, r * a.lddt + c) : 0.f) + rs * (u - rn_load<DT>(a.t, r * a.ldt + c) * rs * dot);
    rn_store<DT>(a.dx, r * a.lddx + c, d);
    if (a.dy) rn_store<DT>(a.dy, r * a.lddy + c, mrow >= 0 ? d * rn_load(a.gate, mrow * a.ldm + c, a.m_dtype) : 0.f);
  }
}
template <int DT>
__global__ void __launch_bounds__(256) resnorm_dw_kernel(const ResNormArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.K) return;
  float sum = 0.f;
  for (int64_t r = 0; r < a.M; ++r) {
    const int mrow = rn_mod_row(a, r);
    float g = rn_load<DT>(a.dh, r * a.lddh + c);
    if (a.scale && mrow >= 0) g *= 1.f + rn_load(a.scale, mrow * a.ldm + c, a.m_dtype);
    sum += g * (rn_load<DT>(a.t, r * a.ldt + c) * a.rstd[r]);
  }
  if (a.w_dtype == H3B_FP32) static_cast<float*>(a.dw)[c] = sum;
  else if (a.w_dtype == H3B_FP16) rn_store<H3B_FP16>(a.dw, c, sum);
  else rn_store<H3B_BF16>(a.dw, c, sum);
}

size_t resnorm_workspace(int64_t M, int K, bool backward) { return 0; }

template <int DT>
static int resnorm_t(const ResNormArgs& a, bool backward, cudaStream_t st) {
  if (!backward) {
    const int smem = a.K * 4;
    const cudaError_t e = cudaFuncSetAttribute(resnorm_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(resnorm)");
    resnorm_kernel<DT><<<static_cast<int>(a.M), 256, smem, st>>>(a);
    return check_launch("resnorm_kernel");
  }
  if (a.M > 0) resnorm_grad_kernel<DT><<<static_cast<int>(a.M), 256, 0, st>>>(a);
  if (int rc = check_launch("resnorm_grad_kernel")) return rc;
  if (!a.dw) return H3B_OK;
  resnorm_dw_kernel<DT><<<(a.K + 255) / 256, 256, 0, st>>>(a);
  return check_launch("resnorm_dw_kernel");
}
int resnorm_launch(const ResNormArgs& a, bool backward, cudaStream_t st) {
  return a.dtype == H3B_FP16 ? resnorm_t<H3B_FP16>(a, backward, st) : resnorm_t<H3B_BF16>(a, backward, st);
}

}  // namespace h3b
