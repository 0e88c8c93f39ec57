// Rotary embedding of q and k from their positions on several axes, out of place: y = R(theta) x, or R(-theta) x.
//
//   theta[b, s, j] = pos[b, s, axis(j)] * inv_freq[j]            j < F = sum of the sections, axis(j) the section of j
//   pair (a, b) of j: channels (j, j + F) "half" or (2 j, 2 j + 1) "adjacent"
//   (a, b) -> (a cos - b sin, a sin + b cos);  channels >= 2 F are copied
// The rotation is orthogonal, so its gradient is the rotation back (inverse: sin -> -sin).
//
// Angles: theta in turns (theta / 2 pi) is computed and reduced to [-1/2, 1/2] in fp64, and sincospif takes the remainder: no slow
// large-argument path.  Position times frequency is exact there for fp32 positions and for integers below 2^29; with the roundings
// of larger ones, of 1 / (2 pi) and of the product with it the angle is off by at most 4 * 2^-53 |theta|, which is below the
// error of cos and sin in fp32 up to |theta| = 2^28 and 5e-4 at 2^40.
// One rounding per output element, from fp32 products.
//
// HBM-bound: every element is read once and written once.  A CTA owns a few tokens of q or k: its threads fill a table
// of the tokens' (cos, sin) in shared memory -- one evaluation per token and pair, not per head -- then go through the
// tokens' rows in 16-byte units.  What hides the latency is full occupancy: eight CTAs of 256 threads per SM at 32 registers;
// with the registers left to the compiler (41, six CTAs) it is 1.15 to 1.2 times slower, with four units loaded ahead per
// thread 1.9 times.  59440 tokens x 2 x 40 heads of 128 channels, bf16 (2.43 GB): 400 us, 6.1 TB/s, at 1965 MHz; 442 us, 5.5 TB/s,
// in a row under the power limit.  Partners off the 16-byte grid ("half" with F not a multiple of the unit) are bound by
// instructions: 2.1 to 2.5 TB/s in 16 bits, 4.4 to 4.9 in 32 (two aligned units and a shift instead of element loads measured slower: both paths run in most warps).
// Few tokens: one token per CTA, so that the heads of a handful of tokens spread over the SMs.
#include "fastdiv.cuh"
#include "h3b_common.cuh"
#include "launch.h"

namespace h3b {

constexpr int RA_THREADS = 256;
constexpr int RA_MAX_TOKENS = 8;  // tokens per CTA

struct RopeSide {
  const char* x;
  char* y;
  const char* pos;
  int64_t xb, xs, xh, yb, ys, yh, pb, ps;  // strides in elements (channels contiguous)
  int64_t S, tiles;                        // tokens per batch entry; CTAs of this side
  int heads;
  FastDiv by_row;  // units of a token
};

struct RopeParams {
  RopeSide side[2];
  const float* inv_freq;
  int64_t B;
  int D, F, ld, axes, pos_dtype, inverse, tokens;  // ld: F rounded up to even; tokens: per CTA
  int section_end[H3B_MAX_AXES];
  FastDiv by_units, by_pairs;  // units of a head; F
};

enum { RA_HALF = 0, RA_HALF_ANY = 1, RA_ADJACENT = 2 };

template <typename T>
__device__ __forceinline__ float ra_f(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same_v<T, __half>) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T ra_t(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

template <typename T>
struct alignas(16) RaVec {
  T e[16 / sizeof(T)];
};

// n channels of a row (n <= 16 / sizeof(T)): one 16-byte access when the rows allow it
template <typename T, bool VEC>
__device__ __forceinline__ RaVec<T> ra_load(const T* p, int n) {
  RaVec<T> v;
  if constexpr (VEC) {
    v = *reinterpret_cast<const RaVec<T>*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i)
      if (i < n) v.e[i] = p[i];
      else v.e[i] = ra_t<T>(0.f);
  }
  return v;
}
template <typename T, bool VEC>
__device__ __forceinline__ void ra_store(T* p, const RaVec<T>& v, int n) {
  if constexpr (VEC) {
    *reinterpret_cast<RaVec<T>*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i)
      if (i < n) p[i] = v.e[i];
  }
}

// One unit of a head's row, V = 16 / sizeof(T) channels wide:
//   RA_HALF      (F a multiple of V) unit u < F / V: channels u V .. and their partners u V + F ..; the rest are copies
//   RA_HALF_ANY  output chunk u; partners are read one by one (the second read of a line comes from L1)
//   RA_ADJACENT  output chunk u, its pairs are inside
template <typename T, bool VEC, int MODE>
__device__ __forceinline__ void ra_unit(const T* x, T* y, int u, int D, int F, const float2* cs) {
  constexpr int V = 16 / sizeof(T);
  if constexpr (MODE == RA_HALF) {
    if (u < F / V) {
      RaVec<T> a = ra_load<T, VEC>(x + u * V, V), b = ra_load<T, VEC>(x + u * V + F, V);
      const float4* t4 = reinterpret_cast<const float4*>(cs + u * V);
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        const float4 t = t4[i / 2];
        const float a0 = ra_f(a.e[i]), b0 = ra_f(b.e[i]), a1 = ra_f(a.e[i + 1]), b1 = ra_f(b.e[i + 1]);
        a.e[i] = ra_t<T>(a0 * t.x - b0 * t.y);
        b.e[i] = ra_t<T>(a0 * t.y + b0 * t.x);
        a.e[i + 1] = ra_t<T>(a1 * t.z - b1 * t.w);
        b.e[i + 1] = ra_t<T>(a1 * t.w + b1 * t.z);
      }
      ra_store<T, VEC>(y + u * V, a, V);
      ra_store<T, VEC>(y + u * V + F, b, V);
    } else {
      const int c = F + u * V, n = min(V, D - c);
      ra_store<T, VEC>(y + c, ra_load<T, VEC>(x + c, n), n);
    }
  } else {
    const int c = u * V, n = min(V, D - c);
    RaVec<T> a = ra_load<T, VEC>(x + c, n);
    if constexpr (MODE == RA_HALF_ANY) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int ch = c + i;
        if (i < n && ch < 2 * F) {
          const bool lo = ch < F;
          const float2 t = cs[lo ? ch : ch - F];
          const float mine = ra_f(a.e[i]), other = ra_f(x[lo ? ch + F : ch - F]);
          a.e[i] = ra_t<T>(lo ? mine * t.x - other * t.y : other * t.y + mine * t.x);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        if (c + i < 2 * F) {
          const float2 t = cs[(c + i) / 2];
          const float fa = ra_f(a.e[i]), fb = ra_f(a.e[i + 1]);
          a.e[i] = ra_t<T>(fa * t.x - fb * t.y);
          a.e[i + 1] = ra_t<T>(fa * t.y + fb * t.x);
        }
      }
    }
    ra_store<T, VEC>(y + c, a, n);
  }
}

__device__ __forceinline__ double ra_pos(const char* p, int64_t i, int dt) {
  if (dt == H3B_FP32) return reinterpret_cast<const float*>(p)[i];
  if (dt == H3B_INT32) return reinterpret_cast<const int32_t*>(p)[i];
  return static_cast<double>(reinterpret_cast<const int64_t*>(p)[i]);
}

template <typename T, bool VEC, int MODE>
__global__ void __launch_bounds__(RA_THREADS, 2048 / RA_THREADS) rope_axes_kernel(const RopeParams P) {
  extern __shared__ __align__(16) float2 cs_table[];  // [tokens][ld]
  __shared__ int64_t x_at[RA_MAX_TOKENS], y_at[RA_MAX_TOKENS];
  const bool second = static_cast<int64_t>(blockIdx.x) >= P.side[0].tiles;
  const RopeSide& sd = P.side[second];
  const int64_t tile = static_cast<int64_t>(blockIdx.x) - (second ? P.side[0].tiles : 0);
  const int64_t total = P.B * sd.S, tok0 = tile * P.tokens;
  const int ntok = static_cast<int>(total - tok0 < P.tokens ? total - tok0 : P.tokens);
  if (threadIdx.x < ntok) {
    const int64_t tok = tok0 + threadIdx.x, b = tok / sd.S, s = tok - b * sd.S;
    x_at[threadIdx.x] = b * sd.xb + s * sd.xs;
    y_at[threadIdx.x] = b * sd.yb + s * sd.ys;
  }
  for (int i = threadIdx.x; i < ntok * P.F; i += RA_THREADS) {
    int j, axis = 0;
    const int t = P.by_pairs.divmod(i, j);
    while (j >= P.section_end[axis]) ++axis;
    const int64_t tok = tok0 + t, b = tok / sd.S, s = tok - b * sd.S;
    double turns = ra_pos(sd.pos, b * sd.pb + s * sd.ps + axis, P.pos_dtype) * static_cast<double>(__ldg(P.inv_freq + j)) *
                   0.15915494309189533577;  // 1 / (2 pi)
    turns -= rint(turns);
    float sn, c;
    sincospif(2.f * static_cast<float>(turns), &sn, &c);
    cs_table[t * P.ld + j] = make_float2(c, P.inverse ? -sn : sn);
  }
  __syncthreads();
  const T* x = reinterpret_cast<const T*>(sd.x);
  T* y = reinterpret_cast<T*>(sd.y);
  const int n = ntok * static_cast<int>(sd.by_row.d);
  for (int i = threadIdx.x; i < n; i += RA_THREADS) {
    int w, u;
    const int t = sd.by_row.divmod(i, w), h = P.by_units.divmod(w, u);
    ra_unit<T, VEC, MODE>(x + x_at[t] + h * sd.xh, y + y_at[t] + h * sd.yh, u, P.D, P.F, cs_table + t * P.ld);
  }
}

template <typename T>
static int rope_axes_launch_t(RopeParams& P, int pairing, bool vec, int sms, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int mode = pairing == H3B_PAIR_ADJACENT ? RA_ADJACENT : P.F % V == 0 ? RA_HALF : RA_HALF_ANY;
  const int units = mode == RA_HALF ? P.F / V + (P.D - 2 * P.F + V - 1) / V : (P.D + V - 1) / V;
  P.by_units.set(units);
  P.by_pairs.set(P.F);
  P.ld = (P.F + 1) & ~1;
  int64_t tokens = 0, blocks = 0;
  for (const auto& sd : P.side) tokens += sd.x ? P.B * sd.S : 0;
  const int64_t per = tokens / (8 * static_cast<int64_t>(sms));  // eight CTAs per SM before a CTA takes several tokens
  P.tokens = static_cast<int>(per < 1 ? 1 : per > RA_MAX_TOKENS ? RA_MAX_TOKENS : per);
  for (auto& sd : P.side) {
    sd.tiles = sd.x ? (P.B * sd.S + P.tokens - 1) / P.tokens : 0;
    sd.by_row.set(units * (sd.x ? sd.heads : 1));
    blocks += sd.tiles;
  }
  if (blocks == 0) return H3B_OK;
  if (blocks > 0x7FFFFFFF) return fail(H3B_ERR_UNSUPPORTED, "rope_axes: too many tokens for one launch");
  const size_t smem = static_cast<size_t>(P.tokens) * P.ld * sizeof(float2);
#define H3B_RA(VEC, MODE) rope_axes_kernel<T, VEC, MODE><<<static_cast<int>(blocks), RA_THREADS, smem, st>>>(P)
  if (vec) {
    if (mode == RA_HALF) H3B_RA(true, RA_HALF);
    else if (mode == RA_HALF_ANY) H3B_RA(true, RA_HALF_ANY);
    else H3B_RA(true, RA_ADJACENT);
  } else {
    if (mode == RA_HALF) H3B_RA(false, RA_HALF);
    else if (mode == RA_HALF_ANY) H3B_RA(false, RA_HALF_ANY);
    else H3B_RA(false, RA_ADJACENT);
  }
#undef H3B_RA
  return check_launch("rope_axes_kernel");
}

int rope_axes_launch(const h3b_rope_operand* q, const h3b_rope_operand* k, int x_dtype, int64_t B, int D,
                     const float* inv_freq, const int32_t* sections, int axes, int pos_dtype, int pairing, int inverse,
                     cudaStream_t st) {
  RopeParams P{};
  P.inv_freq = inv_freq;
  P.B = B;
  P.D = D;
  P.axes = axes;
  P.pos_dtype = pos_dtype;
  P.inverse = inverse;
  for (int a = 0; a < axes; ++a) P.section_end[a] = P.F += sections[a];
  const int es = x_dtype == H3B_FP32 ? 4 : 2, vw = 16 / es;
  bool vec = D % vw == 0;  // 16-byte accesses: every row of every tensor starts on a 16-byte boundary
  const h3b_rope_operand* ops[2] = {q, k};
  for (int i = 0; i < 2; ++i) {
    const h3b_rope_operand* o = ops[i];
    RopeSide& sd = P.side[i];
    if (!o) continue;
    sd.x = static_cast<const char*>(o->x), sd.y = static_cast<char*>(o->y), sd.pos = static_cast<const char*>(o->pos);
    sd.xb = o->x_stride_b, sd.xs = o->x_stride_s, sd.xh = o->x_stride_h;
    sd.yb = o->y_stride_b, sd.ys = o->y_stride_s, sd.yh = o->y_stride_h;
    sd.pb = o->pos_stride_b, sd.ps = o->pos_stride_s;
    sd.S = o->S, sd.heads = static_cast<int>(o->heads);
    for (int64_t v : {sd.xb, sd.xs, sd.xh, sd.yb, sd.ys, sd.yh}) vec = vec && v % vw == 0;
    vec = vec && reinterpret_cast<uintptr_t>(sd.x) % 16 == 0 && reinterpret_cast<uintptr_t>(sd.y) % 16 == 0;
  }
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (x_dtype == H3B_BF16) return rope_axes_launch_t<__nv_bfloat16>(P, pairing, vec, sms, st);
  if (x_dtype == H3B_FP16) return rope_axes_launch_t<__half>(P, pairing, vec, sms, st);
  return rope_axes_launch_t<float>(P, pairing, vec, sms, st);
}

}  // namespace h3b
