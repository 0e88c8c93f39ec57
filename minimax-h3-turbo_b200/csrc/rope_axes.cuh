// Rotary embedding of q and k from their positions on several axes, out of place: y = R(theta) x, or R(-theta) x.
//
//   theta[b, s, j] = pos[b, s, axis(j)] * inv_freq[j]            j < F = sum of the sections, axis(j) the section of j
//   pair (a, b) of j: channels (j, j + F) "half" or (2 j, 2 j + 1) "adjacent"
//   (a, b) -> (a cos - b sin, a sin + b cos);  channels >= 2 F are copied
// The rotation is orthogonal, so its gradient is the rotation back (inverse: sin -> -sin).
//
// Angles: the product of a 32-bit position and a 32-bit frequency is exact in fp64, turns (theta / 2 pi) are reduced to
// [-1/2, 1/2] there, and sincospif takes the remainder: full fp32 accuracy at any position, no slow large-argument path.
// One rounding per output element, from fp32 products.
//
// HBM-bound: every element is read once and written once.  A CTA owns a few tokens of q or k: its threads fill a table
// of the tokens' (cos, sin) in shared memory -- one evaluation per token and pair, not per head -- then walk the heads
// with 16-byte accesses.
#include "h3b_common.cuh"
#include "launch.h"

namespace h3b {

constexpr int RA_THREADS = 256;
constexpr int RA_MAX_TOKENS = 8;   // tokens per CTA
constexpr int RA_MAX_PAIRS = 512;  // F: pairs of one head

struct RopeSide {
  const char* x;
  char* y;
  const char* pos;
  int64_t xb, xs, xh, yb, ys, yh, pb, ps;  // strides in elements (channels contiguous)
  int64_t S, tiles;                        // tokens per batch entry; CTAs of this side
  int heads;
};

struct RopeParams {
  RopeSide side[2];
  const float* inv_freq;
  int64_t B;
  int D, F, axes, pos_dtype, inverse, tokens;  // tokens: per CTA
  int section_end[H3B_MAX_AXES];
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
__device__ __forceinline__ void ra_unit(const T* xr, T* yr, int u, int D, int F, const float2* cs) {
  constexpr int V = 16 / sizeof(T);
  if constexpr (MODE == RA_HALF) {
    if (u < F / V) {
      const RaVec<T> a = ra_load<T, VEC>(xr + u * V, V), b = ra_load<T, VEC>(xr + u * V + F, V);
      RaVec<T> oa, ob;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 t = cs[u * V + i];
        const float fa = ra_f(a.e[i]), fb = ra_f(b.e[i]);
        oa.e[i] = ra_t<T>(fa * t.x - fb * t.y);
        ob.e[i] = ra_t<T>(fa * t.y + fb * t.x);
      }
      ra_store<T, VEC>(yr + u * V, oa, V);
      ra_store<T, VEC>(yr + u * V + F, ob, V);
    } else {
      const int c = 2 * F + (u - F / V) * V;
      ra_store<T, VEC>(yr + c, ra_load<T, VEC>(xr + c, min(V, D - c)), min(V, D - c));
    }
  } else {
    const int c = u * V, n = min(V, D - c);
    const RaVec<T> a = ra_load<T, VEC>(xr + c, n);
    RaVec<T> o = a;
    if constexpr (MODE == RA_HALF_ANY) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int ch = c + i;
        if (i < n && ch < 2 * F) {
          const bool lo = ch < F;
          const float2 t = cs[lo ? ch : ch - F];
          const float mine = ra_f(a.e[i]), other = ra_f(xr[lo ? ch + F : ch - F]);
          o.e[i] = ra_t<T>(lo ? mine * t.x - other * t.y : other * t.y + mine * t.x);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        if (c + i < 2 * F) {
          const float2 t = cs[(c + i) / 2];
          const float fa = ra_f(a.e[i]), fb = ra_f(a.e[i + 1]);
          o.e[i] = ra_t<T>(fa * t.x - fb * t.y);
          o.e[i + 1] = ra_t<T>(fa * t.y + fb * t.x);
        }
      }
    }
    ra_store<T, VEC>(yr + c, o, n);
  }
}

__device__ __forceinline__ double ra_pos(const char* p, int64_t i, int dt) {
  if (dt == H3B_FP32) return reinterpret_cast<const float*>(p)[i];
  if (dt == H3B_INT32) return reinterpret_cast<const int32_t*>(p)[i];
  return static_cast<double>(reinterpret_cast<const int64_t*>(p)[i]);
}

template <typename T, bool VEC, int MODE>
__global__ void __launch_bounds__(RA_THREADS) rope_axes_kernel(const RopeParams P) {
  constexpr int V = 16 / sizeof(T);
  extern __shared__ float2 cs_table[];  // [tokens][F]
  const bool second = static_cast<int64_t>(blockIdx.x) >= P.side[0].tiles;
  const RopeSide& sd = P.side[second];
  const int64_t tile = static_cast<int64_t>(blockIdx.x) - (second ? P.side[0].tiles : 0);
  const int64_t total = P.B * sd.S, tok0 = tile * P.tokens;
  const int ntok = static_cast<int>(total - tok0 < P.tokens ? total - tok0 : P.tokens);
  for (int i = threadIdx.x; i < ntok * P.F; i += RA_THREADS) {
    const int t = i / P.F, j = i - t * P.F;
    int axis = 0;
    while (j >= P.section_end[axis]) ++axis;
    const int64_t tok = tok0 + t, b = tok / sd.S, s = tok - b * sd.S;
    double turns = ra_pos(sd.pos, b * sd.pb + s * sd.ps + axis, P.pos_dtype) * static_cast<double>(__ldg(P.inv_freq + j)) *
                   0.15915494309189533577;  // 1 / (2 pi)
    turns -= rint(turns);
    float sn, c;
    sincospif(2.f * static_cast<float>(turns), &sn, &c);
    cs_table[i] = make_float2(c, P.inverse ? -sn : sn);
  }
  __syncthreads();
  const int units = MODE == RA_HALF ? P.F / V + (P.D - 2 * P.F + V - 1) / V : (P.D + V - 1) / V;
  const int per_tok = units * sd.heads;
  for (int t = 0; t < ntok; ++t) {
    const int64_t tok = tok0 + t, b = tok / sd.S, s = tok - b * sd.S;
    const T* xt = reinterpret_cast<const T*>(sd.x) + b * sd.xb + s * sd.xs;
    T* yt = reinterpret_cast<T*>(sd.y) + b * sd.yb + s * sd.ys;
    for (int i = threadIdx.x; i < per_tok; i += RA_THREADS) {
      const int h = i / units, u = i - h * units;
      ra_unit<T, VEC, MODE>(xt + h * sd.xh, yt + h * sd.yh, u, P.D, P.F, cs_table + t * P.F);
    }
  }
}

template <typename T>
static int rope_axes_launch_t(RopeParams& P, int pairing, bool vec, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  P.tokens = RA_MAX_TOKENS;
  int64_t blocks = 0;
  for (auto& sd : P.side) {
    sd.tiles = sd.x ? (P.B * sd.S + P.tokens - 1) / P.tokens : 0;
    blocks += sd.tiles;
  }
  if (blocks == 0) return H3B_OK;
  if (blocks > 0x7FFFFFFF) return fail(H3B_ERR_UNSUPPORTED, "rope_axes: too many tokens for one launch");
  const size_t smem = static_cast<size_t>(P.tokens) * P.F * sizeof(float2);
  const int mode = pairing == H3B_PAIR_ADJACENT ? RA_ADJACENT : P.F % V == 0 ? RA_HALF : RA_HALF_ANY;
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
    sd = RopeSide{static_cast<const char*>(o->x), static_cast<char*>(o->y), static_cast<const char*>(o->pos),
                  o->x_stride_b, o->x_stride_s, o->x_stride_h, o->y_stride_b, o->y_stride_s, o->y_stride_h,
                  o->pos_stride_b, o->pos_stride_s, o->S, 0, static_cast<int>(o->heads)};
    for (int64_t v : {sd.xb, sd.xs, sd.xh, sd.yb, sd.ys, sd.yh}) vec = vec && v % vw == 0;
    vec = vec && reinterpret_cast<uintptr_t>(sd.x) % 16 == 0 && reinterpret_cast<uintptr_t>(sd.y) % 16 == 0;
  }
  if (x_dtype == H3B_BF16) return rope_axes_launch_t<__nv_bfloat16>(P, pairing, vec, st);
  if (x_dtype == H3B_FP16) return rope_axes_launch_t<__half>(P, pairing, vec, st);
  return rope_axes_launch_t<float>(P, pairing, vec, st);
}

}  // namespace h3b
