// The residual's addition with its root-mean-square norm, 8-bit output and gradients.
//
//   t = dt(x + gate y)                            the residual stream, rounded to its type; the norm reads it so
//   r = rsqrt(mean t^2 + eps),  h = t r w (1 + scale) + shift          in 32 bits, rounded once where h is written
//   z = h H per block of 256 (the rotation of the W4A8 linears),  step = max|z| / 127,  code = rint(z / step)
//   gradients, from dt_out (of t) and dh (of h):  u = dh (1 + scale) w,  d = dt_out + r (u - t r mean(u t r)),
//     dx = d,  dy = gate d,  dw = sum over the rows of dh (1 + scale) t r
// gate, scale and shift are rows of the token's segment; a row outside every segment keeps t = x, h = t r w (dy = 0).  Without a
// gate t = x + y everywhere.
//
// HBM-bound: x and y are read and t and the codes written once, 7 bytes a channel (9 with h; the gradients 8 or 10).  A thread has 16
// channels of a row, so that a row stays in registers from its first load to its codes: the rotation's four butterfly digits are two in
// registers and two over the 16 threads of a block (through shared memory, as in rotq.cuh).  Two rows go through the butterflies at
// once, as the halves of packed fp32 instructions.  CTAs are persistent, and the next rows are on their way while these are worked on.
// w, gate, scale and shift come from L1 every time: 4 bytes a channel and pair of rows.
#pragma once
#include "rotq.cuh"

namespace h3b {

constexpr int RN_AHEAD = 512;  // up to so many threads to a row the next rows' numbers fit in registers

template <int DT>
__device__ __forceinline__ void rn_unpack(const uint32_t (&w)[8], float (&f)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 v = unpack2<DT>(w[i]);
    f[2 * i] = v.x, f[2 * i + 1] = v.y;
  }
}
// 16 numbers of 16 bits from p on, `left` of them there (a multiple of 8, also negative); wide: p on a 32-byte boundary
__device__ __forceinline__ void rn_load(const void* p, int left, bool wide, uint32_t (&v)[8]) {
  if (wide && left >= 16) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "l"(p)
                 : "memory");
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (left > 8 * i) u = reinterpret_cast<const uint4*>(p)[i];
    v[4 * i] = u.x, v[4 * i + 1] = u.y, v[4 * i + 2] = u.z, v[4 * i + 3] = u.w;
  }
}
__device__ __forceinline__ void rn_store(void* p, int left, bool wide, const uint32_t (&v)[8]) {
  if (wide && left >= 16) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (left > 8 * i) reinterpret_cast<uint4*>(p)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}
// 16 numbers of the weight or of a modulation row, of the stream's type (FAST) or of any
template <int DT, bool FAST>
__device__ __forceinline__ void rn_param(const void* p, int64_t at, int dt, int left, float (&f)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (left > 8 * i) {
      if constexpr (FAST) load8(p, at + 8 * i, DT == DT_BF16 ? H3B_BF16 : H3B_FP16, v);
      else load8(p, at + 8 * i, dt, v);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) f[8 * i + k] = v[k];
  }
}
__device__ __forceinline__ int rn_mod_row(const ResNormArgs& a, int64_t r) {
  int m = -1;
  if (r >= a.M) return m;
  if (a.token_rows) {
    m = a.token_rows[r];
    return m < a.n_rows ? m : -1;
  }
  for (int s = 0; s < a.segs.n; ++s)
    if (r >= a.segs.first[s] && r < a.segs.end[s]) m = a.segs.row[s];
  return m;
}
__device__ __forceinline__ char* rn_at(const void* p, int64_t row, int64_t ld, int col) {
  return static_cast<char*>(const_cast<void*>(p)) + 2 * (row * ld + col);
}
// A row's sum: every 16 threads leave theirs in `part`, everyone adds up the row's T / 16.  The barrier is the CTA's.
__device__ __forceinline__ float2 rn_sum(float2 v, float2* part, int mine, int first, int n) {
#pragma unroll
  for (int o = 8; o; o >>= 1) v.x += __shfl_xor_sync(0xffffffffu, v.x, o), v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  if ((threadIdx.x & 15) == 0) part[mine] = v;
  __syncthreads();
  float2 s = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int i = 0; i < n; ++i) s.x += part[first + i].x, s.y += part[first + i].y;
  return s;
}

// blockDim = G groups of T = K / 16 threads, rounded up to whole warps; a group has two rows at a time.
template <int DT, bool CODES, bool FAST, bool AHEAD>
__global__ void __launch_bounds__(AHEAD ? RN_AHEAD : 1024) resnorm_kernel(const ResNormArgs a, int T, int G, bool wide) {
  extern __shared__ __align__(16) unsigned char rn_smem[];
  const int tid = threadIdx.x, unit = tid / T, tr = tid - unit * T, col = 16 * tr, left = unit < G ? a.K - col : 0;
  const int half = tid >> 4, halves = blockDim.x >> 4, t16 = tid & 15, first = unit < G ? unit * (T >> 4) : 0, parts = unit < G ? T >> 4 : 0;
  float2* const part = reinterpret_cast<float2*>(rn_smem);
  uint2* const tops = reinterpret_cast<uint2*>(part + halves);
  float2* const gbuf = reinterpret_cast<float2*>(rn_smem + ((16 * halves + 15) & ~15)) + half * xgrp(16);
  const int64_t pairs = (a.M + 1) / 2, step = static_cast<int64_t>(gridDim.x) * G;
  int64_t r0 = 2 * (static_cast<int64_t>(blockIdx.x) * G + unit);
  if (unit >= G) r0 = a.M;  // threads behind the last group: no rows, but every barrier
  const float over_k = 1.f / static_cast<float>(a.K);
  uint32_t xs[2][8], ys[2][8];
  auto load = [&](int64_t r) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = r + h < a.M ? left : 0;
      rn_load(rn_at(a.x, r + h, a.ldx, col), n, wide, xs[h]);
      rn_load(rn_at(a.y, r + h, a.ldy, col), n, wide, ys[h]);
    }
  };
  if (AHEAD) load(r0);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * G; base < pairs; base += step, r0 += 2 * step) {
    if (!AHEAD) load(r0);
    const int n[2] = {r0 < a.M ? left : 0, r0 + 1 < a.M ? left : 0};
    const int mrow[2] = {rn_mod_row(a, r0), rn_mod_row(a, r0 + 1)};
    const bool same = mrow[0] == mrow[1];
    // ---- the stream
    float2 v[16], ss = make_float2(0.f, 0.f);
    float p[16];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[16], y[16];
      rn_unpack<DT>(xs[h], f);
      rn_unpack<DT>(ys[h], y);
      if (a.gate) {
        if (mrow[h] >= 0) {
          if (h == 0 || !same) rn_param<DT, FAST>(a.gate, mrow[h] * a.ldm + col, a.m_dtype, left, p);
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] = __fadd_rn(f[i], __fmul_rn(y[i], p[i]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = __fadd_rn(f[i], y[i]);
      }
      uint32_t t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = pack2<DT>(make_float2(f[2 * i], f[2 * i + 1]));
      rn_store(rn_at(a.t, r0 + h, a.ldt, col), n[h], wide, t);
      rn_unpack<DT>(t, f);
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s = fmaf(f[i], f[i], s);
        if (h == 0) v[i].x = f[i];
        else v[i].y = f[i];
      }
      if (h == 0) ss.x = s;
      else ss.y = s;
    }
    if (AHEAD && base + step < pairs) load(r0 + 2 * step);
    ss = rn_sum(ss, part, half, first, parts);
    const float2 rs = make_float2(rsqrtf(fmaf(ss.x, over_k, a.eps)), rsqrtf(fmaf(ss.y, over_k, a.eps)));
    if (a.rstd && tr == 0) {
      if (r0 < a.M) a.rstd[r0] = rs.x;
      if (r0 + 1 < a.M) a.rstd[r0 + 1] = rs.y;
    }
    // ---- the norm and its modulation
    rn_param<DT, FAST>(a.w, col, a.w_dtype, left, p);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __fmul2_rn(__fmul2_rn(v[i], rs), make_float2(p[i], p[i]));
    if (a.scale) {
      float q[16];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (mrow[h] < 0) continue;
        if (h == 0 || !same) {
          rn_param<DT, FAST>(a.scale, mrow[h] * a.ldm + col, a.m_dtype, left, p);
          rn_param<DT, FAST>(a.shift, mrow[h] * a.ldm + col, a.m_dtype, left, q);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (h == 0) v[i].x = fmaf(v[i].x, 1.f + p[i], q[i]);
          else v[i].y = fmaf(v[i].y, 1.f + p[i], q[i]);
        }
      }
    }
    if (a.h) {
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = pack2<DT>(make_float2(v[2 * i].x, v[2 * i + 1].x));
      rn_store(rn_at(a.h, r0, a.ldh, col), n[0], wide, o);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = pack2<DT>(make_float2(v[2 * i].y, v[2 * i + 1].y));
      rn_store(rn_at(a.h, r0 + 1, a.ldh, col), n[1], wide, o);
    }
    if constexpr (CODES) {
      // ---- the rotation: digits d0, d1 in registers, d2, d3 over the block's 16 threads
#pragma unroll
      for (int i = 0; i < 4; ++i) h4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], 1.0f);
#pragma unroll
      for (int i = 0; i < 4; ++i) h4(v[i], v[i + 4], v[i + 8], v[i + 12], 1.0f);
      float4* wr = reinterpret_cast<float4*>(gbuf + t16 * XROW);
#pragma unroll
      for (int i = 0; i < 8; ++i) wr[i] = make_float4(v[2 * i].x, v[2 * i].y, v[2 * i + 1].x, v[2 * i + 1].y);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = gbuf[i * XROW + t16];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) h4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], 1.0f);
#pragma unroll
      for (int i = 0; i < 4; ++i) h4(v[i], v[i + 4], v[i + 8], v[i + 12], 0.0625f);
      // ---- the largest magnitude, as bits: a NaN's are above infinity's and stay
      uint2 top = make_uint2(0u, 0u);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        top.x = max(top.x, __float_as_uint(v[i].x) & 0x7FFFFFFFu);
        top.y = max(top.y, __float_as_uint(v[i].y) & 0x7FFFFFFFu);
      }
#pragma unroll
      for (int o = 8; o; o >>= 1) {
        top.x = max(top.x, __shfl_xor_sync(0xffffffffu, top.x, o));
        top.y = max(top.y, __shfl_xor_sync(0xffffffffu, top.y, o));
      }
      if (t16 == 0) tops[half] = top;
      __syncthreads();
#pragma unroll 4
      for (int i = 0; i < parts; ++i) top.x = max(top.x, tops[first + i].x), top.y = max(top.y, tops[first + i].y);
      const float2 amax = make_float2(__uint_as_float(top.x), __uint_as_float(top.y));
      if (tr == 0) {
        if (r0 < a.M) a.scales[r0] = __fdiv_rn(amax.x, 127.f);
        if (r0 + 1 < a.M) a.scales[r0 + 1] = __fdiv_rn(amax.y, 127.f);
      }
      // ---- codes: 0 for rows of zeros and rows without a finite largest magnitude
      const float2 inv = make_float2(amax.x > 0.f && amax.x < INFINITY ? fminf(__fdiv_rn(127.f, amax.x), 3e38f) : 0.f,
                                     amax.y > 0.f && amax.y < INFINITY ? fminf(__fdiv_rn(127.f, amax.y), 3e38f) : 0.f);
      unsigned char* const cbuf = reinterpret_cast<unsigned char*>(gbuf);  // 16 chunks of 16 byte pairs, CSTRIDE apart
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 q = __fmul2_rn(v[i], inv);
        uint32_t c;
        asm("{\n\t.reg .s32 k0, k1;\n\tcvt.rni.s32.f32 k0, %1;\n\tcvt.rni.s32.f32 k1, %2;\n\t"
            "cvt.pack.sat.s8.s32.b32 %0, k1, k0, 0;\n\t}"
            : "=r"(c) : "f"(q.x), "f"(q.y));
        *reinterpret_cast<uint16_t*>(cbuf + i * CSTRIDE + 2 * t16) = static_cast<uint16_t>(c);  // element t + 16 i of the block
      }
      __syncwarp();
      const uint4* rd = reinterpret_cast<const uint4*>(cbuf + t16 * CSTRIDE);
      const uint4 u0 = rd[0], u1 = rd[1];
      const uint32_t w8[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
      uint32_t o[2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[0][i] = __byte_perm(w8[2 * i], w8[2 * i + 1], 0x6420);
        o[1][i] = __byte_perm(w8[2 * i], w8[2 * i + 1], 0x7531);
      }
      __syncwarp();
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (n[h] > 0) *reinterpret_cast<uint4*>(a.codes + (r0 + h) * a.ldc + col) = make_uint4(o[h][0], o[h][1], o[h][2], o[h][3]);
    } else {
      __syncthreads();  // the next rows' sums
    }
  }
}

// Gradients: a group has one row at a time; its threads keep their channels' part of dw over all its rows.
template <int DT, bool FAST, bool AHEAD>
__global__ void __launch_bounds__(AHEAD ? RN_AHEAD : 1024) resnorm_grad_kernel(const ResNormArgs a, int T, int G, bool wide, float* dw) {
  extern __shared__ __align__(16) unsigned char rn_smem[];
  const int tid = threadIdx.x, unit = tid / T, tr = tid - unit * T, col = 16 * tr, left = unit < G ? a.K - col : 0;
  const int half = tid >> 4, halves = blockDim.x >> 4, first = unit < G ? unit * (T >> 4) : 0, parts = unit < G ? T >> 4 : 0;
  float* const part = reinterpret_cast<float*>(rn_smem);  // two rows' sums in turn: one barrier a row
  const int64_t step = static_cast<int64_t>(gridDim.x) * G;
  int64_t r = static_cast<int64_t>(blockIdx.x) * G + unit;
  if (unit >= G) r = a.M;
  const float over_k = 1.f / static_cast<float>(a.K);
  uint32_t td[8], hd[8], ts[8];
  auto load = [&](int64_t row) {
    const int n = row < a.M ? left : 0;
    rn_load(rn_at(a.dh, row, a.lddh, col), n, wide, hd);
    rn_load(rn_at(a.t, row, a.ldt, col), n, wide, ts);
    rn_load(rn_at(a.dt, row, a.lddt, col), a.dt ? n : 0, wide, td);
  };
  float sum[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) sum[i] = 0.f;
  if (AHEAD) load(r);
  int turn = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * G; base < a.M; base += step, r += step, turn ^= 1) {
    if (!AHEAD) load(r);
    const int n = r < a.M ? left : 0;
    const int mrow = rn_mod_row(a, r);
    const float rs = r < a.M ? a.rstd[r] : 0.f;
    float g[16], x[16], d[16], p[16];
    rn_unpack<DT>(hd, g);
    rn_unpack<DT>(ts, x);
    rn_unpack<DT>(td, d);
    if (AHEAD && base + step < a.M) load(r + step);
    if (a.scale && mrow >= 0) {
      rn_param<DT, FAST>(a.scale, mrow * a.ldm + col, a.m_dtype, left, p);
#pragma unroll
      for (int i = 0; i < 16; ++i) g[i] *= 1.f + p[i];
    }
    rn_param<DT, FAST>(a.w, col, a.w_dtype, left, p);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] *= rs;
      sum[i] = fmaf(g[i], x[i], sum[i]);
      g[i] *= p[i];
      dot = fmaf(g[i], x[i], dot);
    }
#pragma unroll
    for (int o = 8; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if ((tid & 15) == 0) part[turn * halves + half] = dot;
    __syncthreads();
    dot = 0.f;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) dot += part[turn * halves + first + i];
    dot *= over_k;
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 16; ++i) d[i] = fmaf(rs, g[i] - x[i] * dot, d[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = pack2<DT>(make_float2(d[2 * i], d[2 * i + 1]));
    rn_store(rn_at(a.dx, r, a.lddx, col), n, wide, o);
    if (a.dy) {
      if (mrow >= 0) {
        rn_param<DT, FAST>(a.gate, mrow * a.ldm + col, a.m_dtype, left, p);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = pack2<DT>(make_float2(d[2 * i] * p[2 * i], d[2 * i + 1] * p[2 * i + 1]));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = 0u;
      }
      rn_store(rn_at(a.dy, r, a.lddy, col), n, wide, o);
    }
  }
  if (dw && unit < G) {
    float* to = dw + (static_cast<int64_t>(blockIdx.x) * G + unit) * a.K + col;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (left > 4 * i) *reinterpret_cast<float4*>(to + 4 * i) = make_float4(sum[4 * i], sum[4 * i + 1], sum[4 * i + 2], sum[4 * i + 3]);
  }
}
// dw: the groups' parts, eight stretches of them by a warp each, then these in order.  A CTA has 32 channels.
__global__ void __launch_bounds__(256) resnorm_dw_kernel(const float* part, int64_t lines, int K, void* dw, int w_dtype) {
  __shared__ float sums[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  const int64_t per = (lines + 7) / 8, to = (w + 1) * per < lines ? (w + 1) * per : lines;
  float s = 0.f;
  if (c < K) {
#pragma unroll 8
    for (int64_t i = w * per; i < to; ++i) s += part[i * K + c];
  }
  sums[w][lane] = s;
  __syncthreads();
  if (w != 0 || c >= K) return;
  for (int i = 1; i < 8; ++i) s += sums[i][lane];
  if (w_dtype == H3B_FP32) static_cast<float*>(dw)[c] = s;
  else if (w_dtype == H3B_FP16) static_cast<__half*>(dw)[c] = __float2half_rn(s);
  else static_cast<__nv_bfloat16*>(dw)[c] = __float2bfloat16_rn(s);
}

// Groups of a CTA and CTAs of the launch.  CTAs of about 256 threads, as many to an SM as give it 1024 (768 from 257 threads on).
struct RnShape {
  int T, G, threads, blocks;
};
static int rn_sms() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}
static RnShape rn_shape(int64_t groups, int K) {
  RnShape s{};
  s.T = (K + 255) / 256 * 16;
  s.G = s.T >= 256 ? 1 : 256 / s.T;
  s.threads = (s.T * s.G + 31) / 32 * 32;
  const int64_t want = (groups + s.G - 1) / s.G, cap = static_cast<int64_t>(rn_sms()) * (s.threads >= 1024 ? 1 : 1024 / s.threads);
  s.blocks = static_cast<int>(want < cap ? want : cap);
  return s;
}
size_t resnorm_workspace(int64_t M, int K, bool backward) {
  if (!backward || M == 0) return 0;
  const RnShape s = rn_shape(M, K);
  return static_cast<size_t>(s.blocks) * s.G * K * 4;
}
static bool rn_wide(const void* p, int64_t ld) { return !p || (ld % 16 == 0 && reinterpret_cast<uintptr_t>(p) % 32 == 0); }

template <int DT, bool CODES, bool FAST, bool AHEAD>
static int resnorm_forward_t(const ResNormArgs& a, cudaStream_t st) {
  const RnShape s = rn_shape((a.M + 1) / 2, a.K);
  auto kernel = resnorm_kernel<DT, CODES, FAST, AHEAD>;
  const int halves = s.threads / 16;
  const int smem = (16 * halves + 15) / 16 * 16 + (CODES ? halves * xgrp(16) * 8 : 0);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(resnorm)");
  }
  const bool wide = rn_wide(a.x, a.ldx) && rn_wide(a.y, a.ldy) && rn_wide(a.t, a.ldt) && rn_wide(a.h, a.ldh);
  kernel<<<s.blocks, s.threads, smem, st>>>(a, s.T, s.G, wide);
  return check_launch("resnorm_kernel");
}
template <int DT, bool FAST, bool AHEAD>
static int resnorm_backward_t(const ResNormArgs& a, cudaStream_t st) {
  const RnShape s = rn_shape(a.M, a.K);
  const bool wide = rn_wide(a.dt, a.lddt) && rn_wide(a.dh, a.lddh) && rn_wide(a.t, a.ldt) && rn_wide(a.dx, a.lddx) && rn_wide(a.dy, a.lddy);
  float* part = a.dw ? static_cast<float*>(a.ws) : nullptr;
  resnorm_grad_kernel<DT, FAST, AHEAD><<<s.blocks, s.threads, 2 * s.threads / 16 * 4, st>>>(a, s.T, s.G, wide, part);
  if (int rc = check_launch("resnorm_grad_kernel")) return rc;
  if (!a.dw) return H3B_OK;
  resnorm_dw_kernel<<<(a.K + 31) / 32, 256, 0, st>>>(part, static_cast<int64_t>(s.blocks) * s.G, a.K, a.dw, a.w_dtype);
  return check_launch("resnorm_dw_kernel");
}
template <int DT>
static int resnorm_t(const ResNormArgs& a, bool backward, cudaStream_t st) {
  constexpr int CODE = DT == DT_BF16 ? H3B_BF16 : H3B_FP16;
  const bool fast = a.w_dtype == CODE && ((!a.gate && !a.scale) || a.m_dtype == CODE), ahead = (a.K + 255) / 256 * 16 <= RN_AHEAD;
  if (backward) {
    if (fast) return ahead ? resnorm_backward_t<DT, true, true>(a, st) : resnorm_backward_t<DT, true, false>(a, st);
    return ahead ? resnorm_backward_t<DT, false, true>(a, st) : resnorm_backward_t<DT, false, false>(a, st);
  }
  if (a.codes) {
    if (fast) return ahead ? resnorm_forward_t<DT, true, true, true>(a, st) : resnorm_forward_t<DT, true, true, false>(a, st);
    return ahead ? resnorm_forward_t<DT, true, false, true>(a, st) : resnorm_forward_t<DT, true, false, false>(a, st);
  }
  if (fast) return ahead ? resnorm_forward_t<DT, false, true, true>(a, st) : resnorm_forward_t<DT, false, true, false>(a, st);
  return ahead ? resnorm_forward_t<DT, false, false, true>(a, st) : resnorm_forward_t<DT, false, false, false>(a, st);
}
int resnorm_launch(const ResNormArgs& a, bool backward, cudaStream_t st) {
  if (backward && a.M == 0) {  // nothing to add up
    const cudaError_t e = a.dw ? cudaMemsetAsync(a.dw, 0, static_cast<size_t>(a.K) * (a.w_dtype == H3B_FP32 ? 4 : 2), st) : cudaSuccess;
    return e == cudaSuccess ? H3B_OK : cuda_fail(e, "cudaMemsetAsync(dw)");
  }
  return a.dtype == H3B_FP16 ? resnorm_t<DT_FP16>(a, backward, st) : resnorm_t<DT_BF16>(a, backward, st);
}

}  // namespace h3b
