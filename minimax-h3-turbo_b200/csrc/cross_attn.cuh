// Cross attention: the gradients, simple kernels in fp32 (four lanes own a row, 32 channels each; the other side's rows are
// staged in shared memory 32 at a time), and the host side of both directions.
#include "cross_fwd.cuh"

namespace h3b {

constexpr int CA_ROWS = 32;      // rows a CTA owns
constexpr int CA_TILE = 32;      // rows of the other side staged at a time
constexpr int CA_LANES = 4;      // lanes per row
constexpr int CA_CH = 32;        // channels per lane
constexpr int CA_MAXD = CA_LANES * CA_CH;

template <typename T>
__device__ __forceinline__ float ca_f(T v) {
  if constexpr (std::is_same_v<T, __half>) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T ca_t(float v) {
  if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

template <typename T>
__device__ __forceinline__ const T* ca_row(const h3b_attn_tensor& t, int b, int64_t s, int h) {
  return static_cast<const T*>(t.ptr) + b * t.stride_b + s * t.stride_s + h * t.stride_h;
}

// stage rows [s0, s0 + CA_TILE) of head h as fp32 [CA_TILE][CA_MAXD] (zero outside the tensor)
template <typename T>
__device__ __forceinline__ void ca_stage(float (*dst)[CA_MAXD], const h3b_attn_tensor& t, int b, int64_t s0, int64_t S, int h, int D) {
  for (int i = threadIdx.x; i < CA_TILE * CA_MAXD; i += blockDim.x) {
    const int r = i / CA_MAXD, c = i % CA_MAXD;
    dst[r][c] = (s0 + r < S && c < D) ? ca_f<T>(ca_row<T>(t, b, s0 + r, h)[c]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void ca_own(float (&x)[CA_CH], const h3b_attn_tensor& t, int b, int64_t s, bool valid, int h, int D, int sub) {
#pragma unroll
  for (int i = 0; i < CA_CH; ++i) {
    const int c = sub + CA_LANES * i;
    x[i] = (valid && c < D) ? ca_f<T>(ca_row<T>(t, b, s, h)[c]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void ca_put(const h3b_attn_tensor& t, int b, int64_t s, int h, int D, int sub, const float (&x)[CA_CH], float w) {
  T* row = const_cast<T*>(ca_row<T>(t, b, s, h));
#pragma unroll
  for (int i = 0; i < CA_CH; ++i) {
    const int c = sub + CA_LANES * i;
    if (c < D) row[c] = ca_t<T>(x[i] * w);
  }
}
__device__ __forceinline__ float ca_dot(const float (&x)[CA_CH], const float* row, int sub) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < CA_CH; ++i) s = fmaf(x[i], row[sub + CA_LANES * i], s);
  s += __shfl_xor_sync(0xffffffffu, s, 1);
  s += __shfl_xor_sync(0xffffffffu, s, 2);
  return s;
}

// dq and delta.  grid (row tiles of Sq, Hq, B)
__device__ __forceinline__ float ca_bias(const CrossParams& P, int b, int64_t j, int64_t len) {
  return j >= len ? -INFINITY : P.bias2 ? P.bias2[b * P.Skp + j] : 0.f;
}
template <typename T>
__global__ void __launch_bounds__(CA_ROWS* CA_LANES) cross_rows_kernel(const CrossParams P) {
  __shared__ float ks[CA_TILE][CA_MAXD], vs[CA_TILE][CA_MAXD];
  __shared__ float bias[CA_TILE];
  const int sub = threadIdx.x % CA_LANES, h = blockIdx.y, b = blockIdx.z, hk = h / P.G;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * CA_ROWS + threadIdx.x / CA_LANES;
  const bool valid = row < P.Sq;
  const int64_t len = ca_len(P.kv_lens, b, P.Sk), stat = (static_cast<int64_t>(b) * P.Hq + h) * P.Sq + row;
  float q[CA_CH], acc[CA_CH] = {}, g[CA_CH], o[CA_CH];
  ca_own<T>(q, P.q, b, row, valid, h, P.D, sub);
  float lse = INFINITY, delta = 0.f;
  ca_own<T>(g, P.go, b, row, valid, h, P.D, sub);
  ca_own<T>(o, P.o, b, row, valid, h, P.D, sub);
#pragma unroll
  for (int i = 0; i < CA_CH; ++i) delta = fmaf(g[i], o[i], delta);
  delta += __shfl_xor_sync(0xffffffffu, delta, 1);
  delta += __shfl_xor_sync(0xffffffffu, delta, 2);
  if (valid) lse = P.lse[stat] * CA_LOG2E;
  if (lse == -INFINITY) lse = INFINITY;  // a row without keys: every p is 0
  if (valid && sub == 0) P.delta[stat] = delta;
  for (int64_t j0 = 0; j0 < len; j0 += CA_TILE) {
    __syncthreads();
    ca_stage<T>(ks, P.k, b, j0, len, hk, P.D);
    ca_stage<T>(vs, P.v, b, j0, len, hk, P.D);
    if (threadIdx.x < CA_TILE) bias[threadIdx.x] = ca_bias(P, b, j0 + threadIdx.x, len);
    __syncthreads();
    for (int j = 0; j < CA_TILE; ++j) {
      const float bj = bias[j];
      if (bj == -INFINITY) continue;  // what a masked key holds is never looked at
      const float s = fmaf(ca_dot(q, ks[j], sub), P.scale2, bj);
      const float ds = exp2f(s - lse) * (ca_dot(g, vs[j], sub) - delta);
#pragma unroll
      for (int i = 0; i < CA_CH; ++i) acc[i] = fmaf(ds, ks[j][sub + CA_LANES * i], acc[i]);
    }
  }
  if (valid) ca_put<T>(P.dq, b, row, h, P.D, sub, acc, P.scale);
}

// dk and dv.  grid (row tiles of Sk, Hkv, B)
template <typename T>
__global__ void __launch_bounds__(CA_ROWS* CA_LANES) cross_keys_kernel(const CrossParams P) {
  __shared__ float qs[CA_TILE][CA_MAXD], gs[CA_TILE][CA_MAXD];
  __shared__ float lse[CA_TILE], delta[CA_TILE];
  const int sub = threadIdx.x % CA_LANES, hk = blockIdx.y, b = blockIdx.z;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * CA_ROWS + threadIdx.x / CA_LANES;
  const int64_t len = ca_len(P.kv_lens, b, P.Sk);
  const float bj = row < len ? ca_bias(P, b, row, len) : -INFINITY;
  const bool live = bj != -INFINITY;
  float k[CA_CH], v[CA_CH], dk[CA_CH] = {}, dv[CA_CH] = {};
  ca_own<T>(k, P.k, b, row, live, hk, P.D, sub);
  ca_own<T>(v, P.v, b, row, live, hk, P.D, sub);
  for (int h = hk * P.G; h < (hk + 1) * P.G; ++h) {
    const int64_t stat = (static_cast<int64_t>(b) * P.Hq + h) * P.Sq;
    for (int64_t i0 = 0; i0 < P.Sq; i0 += CA_TILE) {
      __syncthreads();
      ca_stage<T>(qs, P.q, b, i0, P.Sq, h, P.D);
      ca_stage<T>(gs, P.go, b, i0, P.Sq, h, P.D);
      if (threadIdx.x < CA_TILE) {
        const bool in = i0 + threadIdx.x < P.Sq;
        const float e = in ? P.lse[stat + i0 + threadIdx.x] * CA_LOG2E : INFINITY;
        lse[threadIdx.x] = e == -INFINITY ? INFINITY : e;
        delta[threadIdx.x] = in ? P.delta[stat + i0 + threadIdx.x] : 0.f;
      }
      __syncthreads();
      for (int i = 0; i < CA_TILE; ++i) {
        const float s = fmaf(ca_dot(k, qs[i], sub), P.scale2, bj), dp = ca_dot(v, gs[i], sub);
        const float p = live ? exp2f(s - lse[i]) : 0.f, ds = p * (dp - delta[i]);
#pragma unroll
        for (int c = 0; c < CA_CH; ++c) {
          dv[c] = fmaf(p, gs[i][sub + CA_LANES * c], dv[c]);
          dk[c] = fmaf(ds, qs[i][sub + CA_LANES * c], dk[c]);
        }
      }
    }
  }
  if (row >= P.Sk) return;
  ca_put<T>(P.dk, b, row, hk, P.D, sub, dk, P.scale);
  ca_put<T>(P.dv, b, row, hk, P.D, sub, dv, 1.f);
}

template <typename T>
static int cross_launch_t(const CrossParams& P, bool backward, cudaStream_t st) {
  if (!backward) return fwd_launch<T>(P, st);
  const dim3 qgrid(static_cast<unsigned>((P.Sq + CA_ROWS - 1) / CA_ROWS), P.Hq, P.B);
  const dim3 kgrid(static_cast<unsigned>((P.Sk + CA_ROWS - 1) / CA_ROWS), P.Hkv, P.B);
  const int threads = CA_ROWS * CA_LANES;
  if (P.Sq > 0) cross_rows_kernel<T><<<qgrid, threads, 0, st>>>(P);
  if (P.Sk > 0) cross_keys_kernel<T><<<kgrid, threads, 0, st>>>(P);
  return check_launch("cross_keys_kernel");
}

// Workspace, parts 256-byte aligned: the prepared mask [B, Skp] and its key counts [B]; delta [B, Hq, Sq] (backward);
// partial outputs and log-sum-exps of the key splits (forward).
struct CrossWs {
  size_t bias2 = 0, lens = 0, delta = 0, part_o = 0, part_lse = 0, total = 0;
};
static CrossWs cross_plan(CrossParams& P, int mask_kind, bool backward) {
  P.G = P.Hq / P.Hkv;
  P.nq = CT / P.G;
  P.Skp = (P.Sk + CT - 1) / CT * CT;
  P.q_tiles = static_cast<int>((P.Sq + P.nq - 1) / P.nq);
  P.units = (P.q_tiles + 1) / 2;
  P.splits = backward ? 1 : fwd_splits(static_cast<int64_t>(P.units) * P.Hkv * P.B, P.Skp / CT);
  CrossWs w;
  auto take = [&](size_t bytes) {
    const size_t at = w.total;
    w.total += (bytes + 255) / 256 * 256;
    return at;
  };
  const size_t rows = static_cast<size_t>(P.B) * P.Hq * P.Sq;
  if (mask_kind != H3B_MASK_NONE) {
    w.bias2 = take(static_cast<size_t>(P.B) * P.Skp * 4);
    w.lens = take(static_cast<size_t>(P.B) * 4);
  }
  if (backward) w.delta = take(rows * 4);
  if (P.splits > 1) {
    w.part_o = take(rows * P.splits * P.D * 4);
    w.part_lse = take(rows * P.splits * 4);
  }
  return w;
}
static CrossParams cross_sizes(int64_t B, int64_t Sq, int64_t Sk, int Hq, int Hkv, int D) {
  CrossParams P{};
  P.B = static_cast<int>(B), P.Sq = Sq, P.Sk = Sk, P.Hq = Hq, P.Hkv = Hkv, P.D = D;
  return P;
}

size_t cross_workspace(int64_t B, int64_t Sq, int64_t Sk, int Hq, int Hkv, int D, int mask_kind, bool backward) {
  CrossParams P = cross_sizes(B, Sq, Sk, Hq, Hkv, D);
  return cross_plan(P, Sk > 0 ? mask_kind : H3B_MASK_NONE, backward).total;
}

int cross_launch(const h3b_attn_tensor* t, int dtype, int64_t B, int64_t Sq, int64_t Sk, int Hq, int Hkv, int D, float scale,
                 const int32_t* kv_lens, const void* mask, int mask_kind, int64_t ldm, float* lse, void* ws, bool backward,
                 cudaStream_t st) {
  CrossParams P = cross_sizes(B, Sq, Sk, Hq, Hkv, D);
  const CrossWs w = cross_plan(P, mask_kind, backward);
  P.q = t[0], P.k = t[1], P.v = t[2], P.o = t[3];
  if (backward) P.go = t[4], P.dq = t[5], P.dk = t[6], P.dv = t[7];
  P.lse = lse;
  char* base = static_cast<char*>(ws);
  P.delta = reinterpret_cast<float*>(base + w.delta);
  P.part_o = reinterpret_cast<float*>(base + w.part_o);
  P.part_lse = reinterpret_cast<float*>(base + w.part_lse);
  P.kv_lens = kv_lens;
  P.scale = scale, P.scale2 = scale * CA_LOG2E;
  if (mask_kind != H3B_MASK_NONE) {
    float* bias2 = reinterpret_cast<float*>(base + w.bias2);
    int32_t* lens = reinterpret_cast<int32_t*>(base + w.lens);
    cross_mask_kernel<<<P.B, CA_PREP, 0, st>>>(mask, mask_kind, ldm, kv_lens, Sk, P.Skp, bias2, lens);
    const int rc = check_launch("cross_mask_kernel");
    if (rc) return rc;
    P.bias2 = bias2;
    P.kv_lens = lens;
  }
  return dtype == H3B_BF16 ? cross_launch_t<__nv_bfloat16>(P, backward, st) : cross_launch_t<__half>(P, backward, st);
}

}  // namespace h3b
