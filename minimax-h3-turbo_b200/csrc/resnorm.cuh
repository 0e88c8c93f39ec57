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
// channels of two rows (or 16 and 16 of one row, SPLIT, where a row is long), the halves of packed fp32 instructions, from their
// arrival to their codes.  16 threads have a block of 256: four times 4 channels each, 64 apart, so that every access of theirs is 128
// bytes in a row (16 channels in a row to a thread: 502 us where this takes 448, 59440 x 5120 into codes; the floor is 326).  The
// rotation's four butterfly digits are then two in registers and two over the 16 threads, through shared memory as in rotq.cuh.  The
// gradients need no rotation and have twice 8 channels, 128 apart (four times 4: 160 us where this takes 130, 12090 x 5376).  CTAs are
// persistent; while rows are worked on, the next ones come into shared memory as bulk copies of whole rows (held in registers instead,
// they left room for 10 warps to an SM: 763 us).  What is left above the floor: some 29 instructions a channel take
// 59 % of the issue slots, and the CTA's two barriers a round are the largest stall of its 20 warps to an SM (30 warps of 64 registers
// spill: 580 us).  w, gate, scale and shift come from L1 every time: 4 bytes a channel and pair of rows.
#pragma once
#include <atomic>
#include <type_traits>

#include "rotq.cuh"

namespace h3b {

// W channels of the stream's type, 4 or 8, that one load brings
template <int W>
using RnWord = std::conditional_t<W == 4, uint2, uint4>;
template <int DT, int W>
__device__ __forceinline__ void rn_unpack(const RnWord<W>& u, float (&f)[W]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {
    const float2 v = unpack2<DT>(w[i]);
    f[2 * i] = v.x, f[2 * i + 1] = v.y;
  }
}
template <int DT, int W>
__device__ __forceinline__ RnWord<W> rn_pack(const float (&f)[W]) {
  RnWord<W> u;
  uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
  for (int i = 0; i < W / 2; ++i) w[i] = pack2<DT>(make_float2(f[2 * i], f[2 * i + 1]));
  return u;
}
template <int W>
__device__ __forceinline__ RnWord<W> rn_load(const unsigned char* p, bool ok) {
  return ok ? *reinterpret_cast<const RnWord<W>*>(p) : RnWord<W>{};
}
__device__ __forceinline__ void rn_bulk(void* dst, const void* src, int bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// Address of number `col` of the weight or of a modulation row, of the stream's type (FAST) or of any
template <bool FAST>
__device__ __forceinline__ const char* rn_param_at(const void* p, int64_t at, int dt) {
  return static_cast<const char*>(p) + (FAST || dt != H3B_FP32 ? 2 : 4) * at;
}
// The k-th W numbers of a thread from there: 16 W apart
template <int DT, bool FAST, int W>
__device__ __forceinline__ void rn_param(const char* p, int k, int dt, bool ok, float (&f)[W]) {
#pragma unroll
  for (int i = 0; i < W; ++i) f[i] = 0.f;
  if (!ok) return;
  if (!FAST && dt == H3B_FP32) {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const float4 u = __ldg(reinterpret_cast<const float4*>(p + 64 * W * k) + i / 4);
      f[i] = u.x, f[i + 1] = u.y, f[i + 2] = u.z, f[i + 3] = u.w;
    }
  } else {
    const RnWord<W> u = __ldg(reinterpret_cast<const RnWord<W>*>(p + 32 * W * k));
    if (FAST || dt == (DT == DT_BF16 ? H3B_BF16 : H3B_FP16)) rn_unpack<DT, W>(u, f);
    else rn_unpack<DT == DT_BF16 ? DT_FP16 : DT_BF16, W>(u, f);
  }
}
__device__ __forceinline__ int rn_mod_row(const ResNormArgs& a, int64_t row) {
  int m = -1;
  if (row >= a.M) return m;
  if (a.token_rows) {
    m = a.token_rows[row];
    return m < a.n_rows ? m : -1;
  }
  const int r = static_cast<int>(row);  // below 2^30
#pragma unroll 2
  for (int s = 0; s < a.segs.n; ++s)
    if (r >= a.segs.first[s] && r < a.segs.end[s]) m = a.segs.row[s];
  return m;
}
__device__ __forceinline__ char* rn_at(const void* p, int64_t row, int64_t ld, int col) {
  return static_cast<char*>(const_cast<void*>(p)) + 2 * (row * ld + col);
}
__device__ __forceinline__ float rn_sum16(float v) {
#pragma unroll
  for (int o = 8; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sums (or largest numbers) of two rows: every 16 threads leave theirs in `part`; behind the barrier (the CTA's) every 16 threads add
// up the rows' n <= 32.  Threads 0-7 of the 16 have the first row, 8-15 the second.
template <typename N, typename N2, typename F>
__device__ __forceinline__ N2 rn_over_rows(N2 v, N2* part, int mine, int first, int n, F&& f) {
  const int t = threadIdx.x & 7, up = (threadIdx.x >> 3) & 1;
  auto eight = [&](N w) {
#pragma unroll
    for (int o = 4; o; o >>= 1) w = f(w, __shfl_xor_sync(0xffffffffu, w, o));
    return w;
  };
  N* const flat = reinterpret_cast<N*>(part);
  const N s = eight(f(up ? v.y : v.x, __shfl_xor_sync(0xffffffffu, up ? v.x : v.y, 8)));
  if (t == 0) flat[2 * mine + up] = s;
  __syncthreads();
  N w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (t + 8 * i < n) w = f(w, flat[2 * (first + t + 8 * i) + up]);
  w = eight(w);
  const N other = __shfl_xor_sync(0xffffffffu, w, 8);
  N2 out;
  out.x = up ? other : w, out.y = up ? w : other;
  return out;
}

// Four codes: rounded to the nearest, saturated, the first in the lowest byte
__device__ __forceinline__ uint32_t rn_codes(float x0, float x1, float x2, float x3) {
  uint32_t c;
  asm("{\n\t.reg .s32 k0, k1, k2, k3;\n\t.reg .b32 up;\n\tcvt.rni.s32.f32 k0, %1;\n\tcvt.rni.s32.f32 k1, %2;\n\t"
      "cvt.rni.s32.f32 k2, %3;\n\tcvt.rni.s32.f32 k3, %4;\n\tcvt.pack.sat.s8.s32.b32 up, k3, k2, 0;\n\t"
      "cvt.pack.sat.s8.s32.b32 %0, k1, k0, up;\n\t}"
      : "=r"(c) : "f"(x0), "f"(x1), "f"(x2), "f"(x3));
  return c;
}

// What a launch is made of: groups of T threads, G to a CTA (rounded up to whole warps); a group has two rows, or one (SPLIT: its lanes'
// columns are `off` apart, half the row rounded up to whole blocks of 256, so that both are at the same place of theirs).
struct RnShape {
  int T, G, threads, blocks, off, smem, ahead;
  bool split, more;
};
// Threads of a CTA at most: 320 with 96 registers each and 20 warps to an SM; 384 with 80 and 24, for groups of more than 320 and,
// without codes, where it lets more warps onto an SM (16000 x 4096: 88 us, with 96 registers 94; with codes 114 and 109); 512 with 128
// and 16 for groups of more than 384.  Rows of up to 8192 channels are worked on in pairs, since the weight's and the modulation's
// numbers then serve both (in halves of one row: 12090 x 5376 without codes 128 us where pairs take 106, with codes and h 177 and 148).
constexpr int RN_THREADS = 320, RN_MORE = 384, RN_LARGE = 512;
// Shared memory: barriers and abort flag (32 bytes), the groups' modulation rows (at most RN_GRAD_THREADS / 16 pairs of them), their
// sums, their rows, the rotation's exchange
constexpr int RN_HEAD = 256;
__host__ __device__ inline int rn_rows_at(int threads) { return RN_HEAD + threads; }  // threads / 16 half-warps x (8 + 8) bytes
__host__ __device__ inline int rn_group_bytes(int K, bool split) { return (split ? 2 : 4) * 2 * K; }

template <int DT, bool CODES, bool FAST, bool SPLIT, int MOST>
__global__ void __launch_bounds__(MOST, MOST == RN_LARGE ? 1 : 2) resnorm_kernel(const ResNormArgs a, const RnShape s) {
  constexpr int W = 4, PIECES = 16 / W;  // with or without codes, so that the sums are the same
  extern __shared__ __align__(128) unsigned char rn_smem[];
  const int tid = threadIdx.x, T = s.T, G = s.G, unit = tid / T, tr = tid - unit * T, K = a.K;
  const int half = tid >> 4, halves = blockDim.x >> 4, t16 = tid & 15, parts = unit < G ? T >> 4 : 0, first = unit * parts;
  const int col[2] = {(tr & ~15) * 16 + W * t16, (tr & ~15) * 16 + W * t16 + (SPLIT ? s.off : 0)};  // and PIECES times 16 W further
  const int from[2] = {col[0], SPLIT && col[1] >= K ? col[0] : col[1]};
  uint64_t* const bar = reinterpret_cast<uint64_t*>(rn_smem);
  volatile int* const abort = reinterpret_cast<volatile int*>(rn_smem + 8);
  float2* const part = reinterpret_cast<float2*>(rn_smem + RN_HEAD);
  int2* const rows_of = reinterpret_cast<int2*>(rn_smem + 32) + (unit < G ? unit : 0);
  uint2* const tops = reinterpret_cast<uint2*>(part + halves);
  unsigned char* const mine = rn_smem + rn_rows_at(blockDim.x) + (unit < G ? unit : 0) * rn_group_bytes(K, SPLIT);
  float2* const gbuf = reinterpret_cast<float2*>(rn_smem + rn_rows_at(blockDim.x) + G * rn_group_bytes(K, SPLIT)) + half * xgrp(16);
  constexpr int ROWS = SPLIT ? 1 : 2;
  const int64_t groups = (a.M + ROWS - 1) / ROWS, step = static_cast<int64_t>(gridDim.x) * G;
  int64_t r0 = ROWS * (static_cast<int64_t>(blockIdx.x) * G + unit);
  if (unit >= G) r0 = a.M;  // threads behind the last group: no rows, but every barrier
  if (tid == 0) {
    mbar_init(bar, G);
    mbar_fence_init();
    *abort = 0;
  }
  // a group's first thread finds the modulation rows of the next round too (a row that is not there has its neighbour's)
  auto find = [&](int64_t r) {
    int2 m;
    m.x = m.y = rn_mod_row(a, r);
    if (!SPLIT && r + 1 < a.M) m.y = rn_mod_row(a, r + 1);
    *rows_of = m;
  };
  const bool leads = tr == 0 && unit < G;
  if (leads) find(r0);
  __syncthreads();
  auto bring = [&](int64_t r) {  // by a group's first thread
    int n = 0;
    for (int h = 0; h < ROWS; ++h) n += r + h < a.M ? 4 * K : 0;
    mbar_arrive_expect_tx(bar, n);
    for (int h = 0; h < ROWS; ++h)
      if (r + h < a.M) {
        rn_bulk(mine + h * 4 * K, rn_at(a.x, r + h, a.ldx, 0), 2 * K, bar);
        rn_bulk(mine + h * 4 * K + 2 * K, rn_at(a.y, r + h, a.ldy, 0), 2 * K, bar);
      }
  };
  if (leads) bring(r0);
  const bool mods = FAST && a.gate && a.scale && K % 256 == 0 && unit < G;
  const float over_k = 1.f / static_cast<float>(K);
  uint32_t turn = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * G; base < groups; base += step, r0 += ROWS * step, turn ^= 1) {
    const int64_t row[2] = {r0, r0 + ROWS - 1};
    const int n[2] = {row[0] < a.M ? K - col[0] : 0, row[1] < a.M ? K - col[1] : 0};
    const int2 both = *rows_of;
    const int mrow[2] = {both.x, both.y};
    const bool same = !SPLIT && mrow[0] == mrow[1];  // one load of a modulation row serves both lanes
    // the ordinary case by itself, without a branch inside: modulation rows of the stream's type, 16 channels to every thread.  Where a
    // split row's second half ends before (off, above), its threads go through the first half's channels with zeros.
    const bool plain = mods && mrow[0] >= 0 && (SPLIT || same);
    mbar_wait(bar, turn, abort);
    // ---- the stream
    float2 v[16], ss = make_float2(0.f, 0.f);
    auto stream = [&](auto is_plain) {
      constexpr bool P = decltype(is_plain)::value;
      const unsigned char* at[2];
      const char* pg[2];
      char* to[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        at[h] = mine + (SPLIT ? 0 : h) * 4 * K + 2 * from[h];
        pg[h] = rn_param_at<FAST>(a.gate, mrow[h] * a.ldm + from[h], a.m_dtype);
        to[h] = rn_at(a.t, row[h], a.ldt, col[h]);
      }
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {  // W channels at a time
        float p[W];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float f[W], y[W];
          const bool ok = P || n[h] > 16 * W * k;
          rn_unpack<DT, W>(rn_load<W>(at[h] + 32 * W * k, ok), f);
          rn_unpack<DT, W>(rn_load<W>(at[h] + 2 * K + 32 * W * k, ok), y);
          if (P || a.gate) {
            if (P || mrow[h] >= 0) {
              if (h == 0 || SPLIT || !(P || same)) rn_param<DT, FAST, W>(pg[h], k, a.m_dtype, ok, p);
#pragma unroll
              for (int i = 0; i < W; ++i)  // P: the product of two numbers of 16 bits is exact
                f[i] = P ? fmaf(y[i], p[i], f[i]) : __fadd_rn(f[i], __fmul_rn(y[i], p[i]));
            }
          } else {
#pragma unroll
            for (int i = 0; i < W; ++i) f[i] = __fadd_rn(f[i], y[i]);
          }
          const RnWord<W> t = rn_pack<DT, W>(f);
          if (P ? n[h] > 0 : ok) *reinterpret_cast<RnWord<W>*>(to[h] + 32 * W * k) = t;
          rn_unpack<DT, W>(t, f);
#pragma unroll
          for (int i = 0; i < W; ++i) {
            if (h == 0) v[W * k + i].x = f[i];
            else v[W * k + i].y = P && SPLIT && n[1] <= 0 ? 0.f : f[i];
          }
        }
      }
    };
    if (plain) stream(std::true_type{});
    else stream(std::false_type{});
#pragma unroll
    for (int i = 0; i < 16; ++i) ss = __ffma2_rn(v[i], v[i], ss);
    if (SPLIT) ss.x = ss.y = ss.x + ss.y;
    ss = rn_over_rows<float>(ss, part, half, first, parts, [](float b, float c) { return b + c; });
    // everyone has read the rows: the next ones may come
    if (leads && base + step < groups) bring(r0 + ROWS * step), find(r0 + ROWS * step);
    const float2 rs = make_float2(rsqrtf(fmaf(ss.x, over_k, a.eps)), rsqrtf(fmaf(ss.y, over_k, a.eps)));
    if (a.rstd && leads) {
      if (row[0] < a.M) a.rstd[row[0]] = rs.x;
      if (!SPLIT && row[1] < a.M) a.rstd[row[1]] = rs.y;
    }
    // ---- the norm and its modulation
    auto norm = [&](auto is_plain) {
      constexpr bool P = decltype(is_plain)::value;
      const char *pw[2], *ps[2], *pt[2];
      char* to[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        pw[h] = rn_param_at<FAST>(a.w, from[h], a.w_dtype);
        ps[h] = rn_param_at<FAST>(a.scale, mrow[h] * a.ldm + from[h], a.m_dtype);
        pt[h] = rn_param_at<FAST>(a.shift, mrow[h] * a.ldm + from[h], a.m_dtype);
        to[h] = rn_at(a.h, row[h], a.ldh, col[h]);
      }
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        float p[W], q[W];
        rn_param<DT, FAST, W>(pw[0], k, a.w_dtype, P || (unit < G && K - col[0] > 16 * W * k), p);
        if (SPLIT) rn_param<DT, FAST, W>(pw[1], k, a.w_dtype, P || (unit < G && K - col[1] > 16 * W * k), q);
#pragma unroll
        for (int i = 0; i < W; ++i)
          v[W * k + i] = __fmul2_rn(__fmul2_rn(v[W * k + i], rs), make_float2(p[i], SPLIT ? q[i] : p[i]));
        if (P || a.scale) {
          if (!SPLIT && (P || same)) {
            if (P || mrow[0] >= 0) {
              rn_param<DT, FAST, W>(ps[0], k, a.m_dtype, P || n[0] > 16 * W * k, p);
              rn_param<DT, FAST, W>(pt[0], k, a.m_dtype, P || n[0] > 16 * W * k, q);
#pragma unroll
              for (int i = 0; i < W; ++i) {
                const float u = 1.f + p[i];
                v[W * k + i] = __ffma2_rn(v[W * k + i], make_float2(u, u), make_float2(q[i], q[i]));
              }
            }
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (!P && mrow[h] < 0) continue;
              rn_param<DT, FAST, W>(ps[h], k, a.m_dtype, P || n[h] > 16 * W * k, p);
              rn_param<DT, FAST, W>(pt[h], k, a.m_dtype, P || n[h] > 16 * W * k, q);
#pragma unroll
              for (int i = 0; i < W; ++i) {
                if (h == 0) v[W * k + i].x = fmaf(v[W * k + i].x, 1.f + p[i], q[i]);
                else v[W * k + i].y = fmaf(v[W * k + i].y, 1.f + p[i], q[i]);
              }
            }
          }
        }
        if (a.h) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < W; ++i) p[i] = h == 0 ? v[W * k + i].x : v[W * k + i].y;
            if (n[h] > (P ? 0 : 16 * W * k)) *reinterpret_cast<RnWord<W>*>(to[h] + 32 * W * k) = rn_pack<DT, W>(p);
          }
        }
      }
    };
    if (plain) norm(std::true_type{});
    else norm(std::false_type{});
    if constexpr (CODES) {
      // ---- the rotation: digits d0, d3 in registers, d1, d2 over the block's 16 threads; then thread 4 d3 + d0 has number d1 + 4 d2
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
      // ---- the largest magnitude.  max leaves NaN out, but every number of a block is a sum over all of it: one that is not finite
      // makes them all so, and then the first one's bits (infinity's and NaN's are above the others') say it
      float2 m = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 16; i += 2) m.x = max3f(m.x, fabsf(v[i].x), fabsf(v[i + 1].x)), m.y = max3f(m.y, fabsf(v[i].y), fabsf(v[i + 1].y));
      uint2 top = make_uint2(max(__float_as_uint(m.x), __float_as_uint(v[0].x) & 0x7FFFFFFFu),
                             max(__float_as_uint(m.y), __float_as_uint(v[0].y) & 0x7FFFFFFFu));
      if (SPLIT) top.x = top.y = n[1] > 0 ? max(top.x, top.y) : top.x;
      top = rn_over_rows<uint32_t>(top, tops, half, first, parts, [](uint32_t b, uint32_t c) { return max(b, c); });
      const float2 amax = make_float2(__uint_as_float(top.x), __uint_as_float(top.y));
      if (leads) {
        if (row[0] < a.M) a.scales[row[0]] = __fdiv_rn(amax.x, 127.f);
        if (!SPLIT && row[1] < a.M) a.scales[row[1]] = __fdiv_rn(amax.y, 127.f);
      }
      // ---- codes: 0 for rows of zeros and rows without a finite largest magnitude
      const float2 inv = make_float2(amax.x > 0.f && amax.x < INFINITY ? fminf(__fdiv_rn(127.f, amax.x), 3e38f) : 0.f,
                                     amax.y > 0.f && amax.y < INFINITY ? fminf(__fdiv_rn(127.f, amax.y), 3e38f) : 0.f);
      // a thread's 16 codes of a row, channels 64 d3 + d0 + 4 i, as four words; every four threads change words to have 16 channels
      // that follow one another (lines of 4 threads are 16 bytes further apart, which keeps the reads off each other's banks)
      unsigned char* const cbuf = reinterpret_cast<unsigned char*>(gbuf);
      uint32_t c[2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = __fmul2_rn(v[4 * i + j], inv);
        c[0][i] = rn_codes(q[0].x, q[1].x, q[2].x, q[3].x), c[1][i] = rn_codes(q[0].y, q[1].y, q[2].y, q[3].y);
      }
      const int line = 80 * (t16 >> 2);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<uint4*>(cbuf + 320 * h + line + 16 * (t16 & 3)) = make_uint4(c[h][0], c[h][1], c[h][2], c[h][3]);
      __syncwarp();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c[h][j] = *reinterpret_cast<const uint32_t*>(cbuf + 320 * h + line + 16 * j + 4 * (t16 & 3));
        const uint32_t a0 = __byte_perm(c[h][0], c[h][1], 0x5140), a1 = __byte_perm(c[h][0], c[h][1], 0x7362);
        const uint32_t b0 = __byte_perm(c[h][2], c[h][3], 0x5140), b1 = __byte_perm(c[h][2], c[h][3], 0x7362);
        if (n[h] > 0)
          *reinterpret_cast<uint4*>(a.codes + row[h] * a.ldc + 16 * tr + (SPLIT && h ? s.off : 0)) =
              make_uint4(__byte_perm(a0, b0, 0x5410), __byte_perm(a0, b0, 0x7632), __byte_perm(a1, b1, 0x5410), __byte_perm(a1, b1, 0x7632));
      }
      __syncwarp();
    } else {
      __syncthreads();  // the next rows' sums
    }
  }
}

// Gradients: a group has one row at a time, a thread 16 channels (or 16 and 16, SPLIT) of it; its part of dw over all its rows stays in
// registers.  Rows come as bulk copies two rows ahead, into three buffers in turn (one ahead and two buffers where three do not fit).
constexpr int RN_AHEAD = 3;
constexpr int RN_GRAD_THREADS = 384;  // of a row that is not split, with 80 registers each and 24 warps to an SM; split ones have up to 512 with 128
template <int DT, bool FAST, bool SPLIT>
__global__ void __launch_bounds__(SPLIT ? 512 : RN_GRAD_THREADS, SPLIT ? 1 : 2) resnorm_grad_kernel(const ResNormArgs a, const RnShape s,
                                                                                           float* dw) {
  constexpr int L = SPLIT ? 2 : 1, W = 8, PIECES = 16 / W;
  extern __shared__ __align__(128) unsigned char rn_smem[];
  const int tid = threadIdx.x, T = s.T, G = s.G, unit = tid / T, tr = tid - unit * T, K = a.K;
  const int half = tid >> 4, halves = blockDim.x >> 4, parts = unit < G ? T >> 4 : 0, first = unit * parts;
  const int col0 = (tr & ~15) * 16 + W * (tid & 15);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(rn_smem);  // three
  volatile int* const abort = reinterpret_cast<volatile int*>(rn_smem + 24);
  float* const part = reinterpret_cast<float*>(rn_smem + RN_HEAD);  // two rows' sums in turn: one barrier a row
  const int bytes = (a.dt ? 6 : 4) * K;  // dh, t, dt
  unsigned char* const mine = rn_smem + rn_rows_at(blockDim.x) + (unit < G ? unit : 0) * s.ahead * bytes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * G;
  int64_t r = static_cast<int64_t>(blockIdx.x) * G + unit;
  if (unit >= G) r = a.M;
  if (tid == 0) {
    for (int i = 0; i < RN_AHEAD; ++i) mbar_init(bars + i, G);
    mbar_fence_init();
    *abort = 0;
  }
  __syncthreads();
  auto bring = [&](int64_t row, int i) {  // by a group's first thread, into buffer i
    const bool ok = row < a.M;
    mbar_arrive_expect_tx(bars + i, ok ? bytes : 0);
    if (!ok) return;
    unsigned char* const to = mine + i * bytes;
    rn_bulk(to, rn_at(a.dh, row, a.lddh, 0), 2 * K, bars + i);
    rn_bulk(to + 2 * K, rn_at(a.t, row, a.ldt, 0), 2 * K, bars + i);
    if (a.dt) rn_bulk(to + 4 * K, rn_at(a.dt, row, a.lddt, 0), 2 * K, bars + i);
  };
  const bool leads = tr == 0 && unit < G;
  const int64_t left = (a.M - static_cast<int64_t>(blockIdx.x) * G + step - 1) / step;  // rounds of this CTA
  if (leads)
    for (int i = 0; i < s.ahead - 1 && i < left; ++i) bring(r + i * step, i);
  const float over_k = 1.f / static_cast<float>(K);
  const bool mods = FAST && a.dy && a.scale && K % 256 == 0 && unit < G, second = SPLIT && col0 + s.off < K;
  float sum[L][16];
#pragma unroll
  for (int l = 0; l < L; ++l)
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[l][i] = 0.f;
  int buf = 0;
  uint32_t phase = 0;
  for (int64_t k = 0; k < left; ++k, r += step) {
    const int mrow = rn_mod_row(a, r);
    const float rs = r < a.M ? a.rstd[r] : 0.f;
    mbar_wait(bars + buf, phase, abort);
    const unsigned char* const at = mine + buf * bytes;
    float g[L][16], x[L][16], dot = 0.f;
    // the ordinary case by itself, as above
    const bool plain = mods && mrow >= 0;
    auto dots = [&](auto is_plain) {
      constexpr bool P = decltype(is_plain)::value;
#pragma unroll
      for (int l = 0; l < L; ++l) {
        const bool live = !P || l == 0 || second;
        const int col = live ? col0 + l * s.off : col0;
        const char* const ps = rn_param_at<FAST>(a.scale, mrow * a.ldm + col, a.m_dtype);
        const char* const pw = rn_param_at<FAST>(a.w, col, a.w_dtype);
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
          const bool ok = P || (r < a.M && col + 16 * W * k < K);
          float p[W], f[W];
          rn_unpack<DT, W>(rn_load<W>(at + 2 * col + 32 * W * k, ok), f);
          if (P || (a.scale && mrow >= 0)) {
            rn_param<DT, FAST, W>(ps, k, a.m_dtype, ok, p);
#pragma unroll
            for (int i = 0; i < W; ++i) f[i] *= 1.f + p[i];
          }
#pragma unroll
          for (int i = 0; i < W; ++i) g[l][W * k + i] = live ? f[i] : 0.f;
          rn_unpack<DT, W>(rn_load<W>(at + 2 * K + 2 * col + 32 * W * k, ok), f);
          rn_param<DT, FAST, W>(pw, k, a.w_dtype, ok, p);
#pragma unroll
          for (int i = 0; i < W; ++i) {
            const int e = W * k + i;
            x[l][e] = f[i] * rs;
            sum[l][e] = fmaf(g[l][e], x[l][e], sum[l][e]);
            g[l][e] *= p[i];
            dot = fmaf(g[l][e], x[l][e], dot);
          }
        }
      }
    };
    if (plain) dots(std::true_type{});
    else dots(std::false_type{});
    dot = rn_sum16(dot);
    float* const here = part + (k & 1) * halves;
    if ((tid & 15) == 0) here[half] = dot;
    __syncthreads();
    // everyone is through with the row before: its buffer is free
    const int free = buf == 0 ? s.ahead - 1 : buf - 1;
    if (leads && k + s.ahead - 1 < left) bring(r + (s.ahead - 1) * step, free);
    const int t16 = tid & 15;
    dot = rn_sum16((t16 < parts ? here[first + t16] : 0.f) + (t16 + 16 < parts ? here[first + 16 + t16] : 0.f)) * over_k;
    auto write = [&](auto is_plain) {
      constexpr bool P = decltype(is_plain)::value;
#pragma unroll
      for (int l = 0; l < L; ++l) {
        const bool live = !P || l == 0 || second;
        const int col = live ? col0 + l * s.off : col0;
        const char* const pg = rn_param_at<FAST>(a.gate, mrow * a.ldm + col, a.m_dtype);
        char* const to_x = rn_at(a.dx, r, a.lddx, col);
        char* const to_y = rn_at(a.dy, r, a.lddy, col);
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
          const bool ok = P || (r < a.M && col + 16 * W * k < K);
          float d[W];
          rn_unpack<DT, W>(rn_load<W>(at + 4 * K + 2 * col + 32 * W * k, ok && a.dt), d);
#pragma unroll
          for (int i = 0; i < W; ++i) d[i] = fmaf(rs, g[l][W * k + i] - x[l][W * k + i] * dot, d[i]);
          if (ok && live) *reinterpret_cast<RnWord<W>*>(to_x + 32 * W * k) = rn_pack<DT, W>(d);
          if (P || a.dy) {
            float p[W];
            rn_param<DT, FAST, W>(pg, k, a.m_dtype, ok && (P || mrow >= 0), p);
#pragma unroll
            for (int i = 0; i < W; ++i) d[i] = P || mrow >= 0 ? d[i] * p[i] : 0.f;
            if (ok && live) *reinterpret_cast<RnWord<W>*>(to_y + 32 * W * k) = rn_pack<DT, W>(d);
          }
        }
      }
    };
    if (plain) write(std::true_type{});
    else write(std::false_type{});
    if (++buf == s.ahead) buf = 0, phase ^= 1;
  }
  if (dw && unit < G) {
#pragma unroll
    for (int l = 0; l < L; ++l) {
      const int col = col0 + l * s.off;
      float* to = dw + (static_cast<int64_t>(blockIdx.x) * G + unit) * K + col;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = i / (W / 4) * 16 * W + i % (W / 4) * 4;
        if (K - col > e) *reinterpret_cast<float4*>(to + e) = make_float4(sum[l][4 * i], sum[l][4 * i + 1], sum[l][4 * i + 2], sum[l][4 * i + 3]);
      }
    }
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

// SM count, and whether a kernel's shared memory has been asked for: once per device (a call spends microseconds on them otherwise)
constexpr int RN_DEVICES = 64;
static int rn_device() {
  int dev = 0;
  cudaGetDevice(&dev);
  return dev;
}
static int rn_sms() {
  static std::atomic<int> known[RN_DEVICES];
  const int dev = rn_device();
  int sms = dev < RN_DEVICES ? known[dev].load(std::memory_order_relaxed) : 0;
  if (sms == 0) {
    sms = 148;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (dev < RN_DEVICES) known[dev].store(sms, std::memory_order_relaxed);
  }
  return sms;
}
// CTAs of up to RN_THREADS, RN_MORE or RN_LARGE threads, as many to an SM as its registers and its shared memory allow
static RnShape rn_shape(int64_t M, int K, bool codes, bool backward) {
  RnShape s{};
  s.T = (K + 255) / 256 * 16;
  s.split = s.T > (backward ? RN_GRAD_THREADS : RN_LARGE);
  if (s.split) s.off = (K + 511) / 512 * 256, s.T = s.off / 16;
  const int most = backward ? RN_GRAD_THREADS : RN_THREADS;
  s.G = s.T > most ? 1 : most / s.T;
  const int64_t groups = backward || s.split ? M : (M + 1) / 2;
  if (groups < 2 * rn_sms() && s.G > 1) s.G = 1;  // few rows: spread over the SMs
  s.threads = (s.T * s.G + 31) / 32 * 32;
  s.ahead = RN_AHEAD * 6 * K > 220 * 1024 ? 2 : RN_AHEAD;
  s.smem = rn_rows_at(s.threads) + s.G * (backward ? s.ahead * 6 * K : rn_group_bytes(K, s.split)) +
           (codes ? s.threads / 16 * xgrp(16) * 8 : 0);
  const int w = s.threads / 32;
  s.more = s.threads <= RN_MORE && (s.threads > RN_THREADS || (!codes && 24 / w * w > 20 / w * w));
  int per = (backward ? (s.split ? 16 : 24) : s.threads > RN_MORE ? 16 : s.more ? 24 : 20) / w;
  if (per > 225 * 1024 / (s.smem + 1024)) per = 225 * 1024 / (s.smem + 1024);
  if (per < 1) per = 1;
  const int64_t want = (groups + s.G - 1) / s.G, cap = static_cast<int64_t>(rn_sms()) * per;
  s.blocks = static_cast<int>(want < cap ? want : cap);
  return s;
}
size_t resnorm_workspace(int64_t M, int K, bool backward) {
  if (!backward || M == 0) return 0;
  const RnShape s = rn_shape(M, K, false, true);
  return static_cast<size_t>(s.blocks) * s.G * K * 4;
}
template <typename F>
static int rn_ready(F* kernel, int smem, std::atomic<bool> (&done)[RN_DEVICES]) {
  if (smem <= 48 * 1024) return H3B_OK;
  const int dev = rn_device();
  if (dev < RN_DEVICES && done[dev].load(std::memory_order_acquire)) return H3B_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(resnorm)");
  if (dev < RN_DEVICES) done[dev].store(true, std::memory_order_release);
  return H3B_OK;
}

template <int DT, bool FAST, bool SPLIT, int MOST>
static int resnorm_forward_s(const ResNormArgs& a, const RnShape& s, cudaStream_t st) {
  auto kernel = a.codes ? resnorm_kernel<DT, true, FAST, SPLIT, MOST> : resnorm_kernel<DT, false, FAST, SPLIT, MOST>;
  static std::atomic<bool> ready[2][RN_DEVICES];
  if (int rc = rn_ready(kernel, s.smem, ready[a.codes != nullptr])) return rc;
  kernel<<<s.blocks, s.threads, s.smem, st>>>(a, s);
  return check_launch("resnorm_kernel");
}
template <int DT, bool FAST, bool SPLIT>
static int resnorm_forward_t(const ResNormArgs& a, const RnShape& s, cudaStream_t st) {
  if (s.more) return resnorm_forward_s<DT, FAST, SPLIT, RN_MORE>(a, s, st);
  return s.threads > RN_MORE ? resnorm_forward_s<DT, FAST, SPLIT, RN_LARGE>(a, s, st) : resnorm_forward_s<DT, FAST, SPLIT, RN_THREADS>(a, s, st);
}
template <int DT, bool FAST>
static int resnorm_backward_t(const ResNormArgs& a, const RnShape& s, cudaStream_t st) {
  auto kernel = s.split ? resnorm_grad_kernel<DT, FAST, true> : resnorm_grad_kernel<DT, FAST, false>;
  static std::atomic<bool> ready[2][RN_DEVICES];
  if (int rc = rn_ready(kernel, s.smem, ready[s.split])) return rc;
  kernel<<<s.blocks, s.threads, s.smem, st>>>(a, s, a.dw ? static_cast<float*>(a.ws) : nullptr);
  if (int rc = check_launch("resnorm_grad_kernel")) return rc;
  if (!a.dw) return H3B_OK;
  resnorm_dw_kernel<<<(a.K + 31) / 32, 256, 0, st>>>(static_cast<float*>(a.ws), static_cast<int64_t>(s.blocks) * s.G, a.K, a.dw, a.w_dtype);
  return check_launch("resnorm_dw_kernel");
}
template <int DT>
static int resnorm_t(const ResNormArgs& a, bool backward, cudaStream_t st) {
  constexpr int CODE = DT == DT_BF16 ? H3B_BF16 : H3B_FP16;
  const bool fast = a.w_dtype == CODE && ((!a.gate && !a.scale) || a.m_dtype == CODE);
  const RnShape s = rn_shape(a.M, a.K, !backward && a.codes, backward);
  if (backward) return fast ? resnorm_backward_t<DT, true>(a, s, st) : resnorm_backward_t<DT, false>(a, s, st);
  if (fast) return s.split ? resnorm_forward_t<DT, true, true>(a, s, st) : resnorm_forward_t<DT, true, false>(a, s, st);
  return s.split ? resnorm_forward_t<DT, false, true>(a, s, st) : resnorm_forward_t<DT, false, false>(a, s, st);
}
int resnorm_launch(const ResNormArgs& a, bool backward, cudaStream_t st) {
  if (backward && a.M == 0) {  // nothing to add up
    const cudaError_t e = a.dw ? cudaMemsetAsync(a.dw, 0, static_cast<size_t>(a.K) * (a.w_dtype == H3B_FP32 ? 4 : 2), st) : cudaSuccess;
    return e == cudaSuccess ? H3B_OK : cuda_fail(e, "cudaMemsetAsync(dw)");
  }
  return a.dtype == H3B_FP16 ? resnorm_t<DT_FP16>(a, backward, st) : resnorm_t<DT_BF16>(a, backward, st);
}

}  // namespace h3b
