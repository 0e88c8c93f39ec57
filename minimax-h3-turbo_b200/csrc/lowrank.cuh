// Low-rank adapters of many requests beside a shared projection, and their gradients.
//
//   out_i = base_i + s_g (x_i A_g^T) B_g^T        g: the adapter of row i; rows without one keep base_i
//   h_i = s_g x_i A_g^T                           [rank], held in 32 bits until it is an operand of the second product
//   dh_i = s_g go_i B_g,   dx_i = dh_i A_g,   dA_g = sum_i dh_i^T x_i,   dB_g = sum_i go_i^T h_i
//
// The rows are gone through in the plan's order (by adapter, then by row), in tiles of one adapter's rows.
#pragma once
#include <type_traits>
#include <utility>

#include "h3b_common.cuh"
#include "launch.h"

namespace h3b {

template <typename T>
__device__ __forceinline__ float lr_f(T v) {
  if constexpr (std::is_same_v<T, __half>) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T lr_t(float v) {
  if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// ----------------------------------------------------------------------------------------------- plan
// A plan is one int32 array: order [M], the rows by adapter, those without one last; offset [R + 2], where each adapter's rows
// begin in it (group R: rows without one); then tables of four numbers a tile (adapter, first place in order, rows, 0): tiles of
// up to LR_TILE rows, tiles of up to LR_FEW rows.  Unused lines of a table have no rows.
constexpr int LR_TILE = 128, LR_FEW = 8;
struct LrPlan {
  const int32_t* order;
  const int32_t* offset;
  const int4* tiles;
  const int4* few;
  int64_t n_tiles, n_few;  // lines of the tables, used or not
};
static int64_t lr_up4(int64_t v) { return (v + 3) / 4 * 4; }
static int64_t lr_lines(int64_t M, int64_t R, int rows) { return M / rows + (R + 1 < M ? R + 1 : M); }
static int64_t lr_plan_ints(int64_t M, int64_t R) {
  return lr_up4(M) + lr_up4(R + 2) + 4 * (lr_lines(M, R, LR_TILE) + lr_lines(M, R, LR_FEW));
}
static LrPlan lr_plan(const int32_t* p, int64_t M, int64_t R) {
  LrPlan pl{};
  pl.order = p;
  pl.offset = p + lr_up4(M);
  pl.tiles = reinterpret_cast<const int4*>(pl.offset + lr_up4(R + 2));
  pl.n_tiles = lr_lines(M, R, LR_TILE);
  pl.few = pl.tiles + pl.n_tiles;
  pl.n_few = lr_lines(M, R, LR_FEW);
  return pl;
}

constexpr int LR_PLAN_THREADS = 1024;
__device__ __forceinline__ int lr_group(const int32_t* rows, int64_t i, int R) {
  const int g = rows[i];
  return g < 0 || g >= R ? R : g;
}
// CTA g finds the places of adapter g's rows: as many rows as have a smaller group come before.  Every warp counts a stretch of
// the rows, then writes its own in order.
static __global__ void __launch_bounds__(LR_PLAN_THREADS) lr_order_kernel(const int32_t* __restrict__ rows, int64_t M, int R,
                                                                        int32_t* __restrict__ order,
                                                                        int32_t* __restrict__ offset) {
  constexpr int W = LR_PLAN_THREADS / 32;
  __shared__ int mine[W], below[W];
  const int g = blockIdx.x, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t per = ((M + W - 1) / W + 31) / 32 * 32, from = w * per, to = from + per < M ? from + per : M;
  int n = 0, b = 0;
  for (int64_t i = from + lane; i < to; i += 32) {
    const int v = lr_group(rows, i, R);
    n += v == g;
    b += v < g;
  }
  n = __reduce_add_sync(0xffffffffu, n);
  b = __reduce_add_sync(0xffffffffu, b);
  if (lane == 0) mine[w] = n, below[w] = b;
  __syncthreads();
  int at = 0, total = 0;
  for (int i = 0; i < W; ++i) {
    at += below[i] + (i < w ? mine[i] : 0);
    total += below[i];
  }
  if (threadIdx.x == 0) {
    offset[g] = total;
    if (g == R) offset[R + 1] = static_cast<int32_t>(M);
  }
  for (int64_t i = from; i < to; i += 32) {
    const bool hit = i + lane < to && lr_group(rows, i + lane, R) == g;
    const unsigned m = __ballot_sync(0xffffffffu, hit);
    if (hit) order[at + __popc(m & ((1u << lane) - 1))] = static_cast<int32_t>(i + lane);
    at += __popc(m);
  }
}
// One CTA: the tables of tiles, from the offsets.
static __global__ void __launch_bounds__(LR_PLAN_THREADS) lr_tiles_kernel(const int32_t* __restrict__ offset, int R,
                                                                        int4* __restrict__ tiles, int64_t n_tiles,
                                                                        int4* __restrict__ few, int64_t n_few) {
  constexpr int W = LR_PLAN_THREADS / 32;
  __shared__ int sums[W];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int table = 0; table < 2; ++table) {
    int4* t = table ? few : tiles;
    const int64_t lines = table ? n_few : n_tiles;
    const int size = table ? LR_FEW : LR_TILE;
    int base = 0;
    for (int g0 = 0; g0 <= R; g0 += LR_PLAN_THREADS) {
      const int g = g0 + static_cast<int>(threadIdx.x);
      const int first = g <= R ? offset[g] : 0, n = g <= R ? offset[g + 1] - first : 0, mine = (n + size - 1) / size;
      int inc = mine;
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (lane == 31) sums[w] = inc;
      __syncthreads();
      int at = base + inc - mine, total = 0;
      for (int i = 0; i < W; ++i) {
        if (i < w) at += sums[i];
        total += sums[i];
      }
      for (int i = 0; i < mine; ++i) t[at + i] = make_int4(g, first + i * size, min(size, n - i * size), 0);
      base += total;
      __syncthreads();
    }
    for (int64_t i = base + threadIdx.x; i < lines; i += LR_PLAN_THREADS) t[i] = make_int4(R, 0, 0, 0);
  }
}
int lr_plan_launch(const int32_t* rows, int64_t M, int64_t R, int32_t* plan, cudaStream_t st) {
  const LrPlan p = lr_plan(plan, M, R);
  lr_order_kernel<<<static_cast<int>(R) + 1, LR_PLAN_THREADS, 0, st>>>(rows, M, static_cast<int>(R), const_cast<int32_t*>(p.order),
                                                                      const_cast<int32_t*>(p.offset));
  if (int rc = check_launch("lr_order_kernel")) return rc;
  lr_tiles_kernel<<<1, LR_PLAN_THREADS, 0, st>>>(p.offset, static_cast<int>(R), const_cast<int4*>(p.tiles), p.n_tiles,
                                                const_cast<int4*>(p.few), p.n_few);
  return check_launch("lr_tiles_kernel");
}
int64_t lr_plan_size(int64_t M, int64_t R) { return lr_plan_ints(M, R); }

// ----------------------------------------------------------------------------------------------- hidden rows
// h (or dh) of every row in the plan's order: rows of rp = rank rounded up to 16 values of the operands' type, and a power of
// two per row that they are to be multiplied by (1 in bf16): fp16 holds products of fp16 numbers only after scaling.
static int lr_rp(int rank) { return (rank + 15) / 16 * 16; }
static size_t lr_up256(size_t v) { return (v + 255) / 256 * 256; }
size_t lr_hidden_bytes(int64_t M, int rank) {
  return lr_up256(static_cast<size_t>(M) * lr_rp(rank) * 2) + lr_up256(static_cast<size_t>(M) * 4);
}
struct LrHidden {
  void* h;      // [M][rp]
  float* mult;  // [M]
};
static LrHidden lr_hidden(void* p, int64_t M, int rank) {
  return LrHidden{p, reinterpret_cast<float*>(static_cast<char*>(p) + lr_up256(static_cast<size_t>(M) * lr_rp(rank) * 2))};
}
// The power of two that brings a row whose largest magnitude is `top` into [1, 2); 1 for rows of zeros, infinities or NaN.
__device__ __forceinline__ float lr_power(float top) {
  const int e = (__float_as_int(top) >> 23) & 0xFF;
  return e == 0 || e >= 253 ? 1.f : __int_as_float(e << 23);
}

template <typename T>
__global__ void __launch_bounds__(256) lr_shrink_kernel(const LrPlan p, const T* __restrict__ x, int64_t ldx, int64_t C,
                                                        const T* __restrict__ w, bool w_rows, int rank, int rp, int R,
                                                        const float* __restrict__ scales, const LrHidden out) {
  __shared__ float h[128];
  const int4 t = p.few[blockIdx.x];
  if (t.z == 0 || t.x >= R) return;
  const float s = scales ? scales[t.x] : 1.f;
  w += static_cast<int64_t>(t.x) * rank * C;
  for (int i = 0; i < t.z; ++i) {
    const T* xr = x + p.order[t.y + i] * ldx;
    for (int j = threadIdx.x >> 5; j < rp; j += 8) {
      float sum = 0.f;
      if (j < rank)
        for (int64_t c = threadIdx.x & 31; c < C; c += 32) sum += lr_f(xr[c]) * lr_f(w_rows ? w[j * C + c] : w[c * rank + j]);
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if ((threadIdx.x & 31) == 0) h[j] = sum * s;
    }
    __syncthreads();
    float mult = 1.f;
    if (std::is_same_v<T, __half>) {
      float top = 0.f;
      for (int j = 0; j < rp; ++j) top = fmaxf(top, fabsf(h[j]));
      mult = lr_power(top);
    }
    const int64_t at = t.y + i;
    if (threadIdx.x < rp) static_cast<T*>(out.h)[at * rp + threadIdx.x] = lr_t<T>(h[threadIdx.x] / mult);
    if (threadIdx.x == 0) out.mult[at] = mult;
    __syncthreads();
  }
}
template <typename T>
__global__ void __launch_bounds__(256) lr_expand_kernel(const LrPlan p, const LrHidden hid, const T* __restrict__ w, bool w_rows,
                                                        int rank, int rp, int R, const T* __restrict__ base, int64_t ldb,
                                                        T* __restrict__ out, int64_t ldo, int64_t N) {
  const int4 t = p.few[blockIdx.x];
  for (int i = 0; i < t.z; ++i) {
    const int64_t row = p.order[t.y + i], at = t.y + i;
    const T* wg = w + static_cast<int64_t>(t.x) * rank * N;
    for (int64_t n = threadIdx.x; n < N; n += 256) {
      float sum = 0.f;
      if (t.x < R) {
        for (int j = 0; j < rank; ++j) sum += lr_f(static_cast<const T*>(hid.h)[at * rp + j]) * lr_f(w_rows ? wg[n * rank + j] : wg[j * N + n]);
        sum *= hid.mult[at];
      }
      out[row * ldo + n] = lr_t<T>(sum + (base ? lr_f(base[row * ldb + n]) : 0.f));
    }
  }
}
// grad [rank][C] (by_rank) or [C][rank] of adapter blockIdx.y
template <typename T>
__global__ void __launch_bounds__(256) lr_wgrad_kernel(const LrPlan p, const LrHidden hid, const T* __restrict__ x, int64_t ldx,
                                                       int64_t C, int rank, int rp, bool by_rank, T* __restrict__ grad) {
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, c = e / rank;
  const int j = static_cast<int>(e - c * rank), g = blockIdx.y;
  if (c >= C) return;
  float sum = 0.f;
  for (int i = p.offset[g]; i < p.offset[g + 1]; ++i)
    sum += lr_f(static_cast<const T*>(hid.h)[static_cast<int64_t>(i) * rp + j]) * hid.mult[i] * lr_f(x[p.order[i] * ldx + c]);
  grad[static_cast<int64_t>(g) * rank * C + (by_rank ? j * C + c : c * rank + j)] = lr_t<T>(sum);
}

size_t lr_workspace(int64_t M, int64_t K, int64_t N, int rank, int64_t R, bool backward) {
  return lr_hidden_bytes(M, rank);
}

template <typename T>
static int lr_forward_t(const LrArgs& a, cudaStream_t st) {
  const LrPlan p = lr_plan(a.plan, a.M, a.R);
  const LrHidden h = lr_hidden(a.hidden ? a.hidden : a.ws, a.M, a.rank);
  const int rp = lr_rp(a.rank), R = static_cast<int>(a.R), grid = static_cast<int>(p.n_few);
  lr_shrink_kernel<T><<<grid, 256, 0, st>>>(p, static_cast<const T*>(a.x), a.ldx, a.K, static_cast<const T*>(a.a), true, a.rank, rp,
                                           R, a.scales, h);
  if (int rc = check_launch("lr_shrink_kernel")) return rc;
  lr_expand_kernel<T><<<grid, 256, 0, st>>>(p, h, static_cast<const T*>(a.b), true, a.rank, rp, R, static_cast<const T*>(a.base),
                                           a.ldbase, static_cast<T*>(a.out), a.ldo, a.N);
  return check_launch("lr_expand_kernel");
}
template <typename T>
static int lr_backward_t(const LrArgs& a, cudaStream_t st) {
  const LrPlan p = lr_plan(a.plan, a.M, a.R);
  const LrHidden h = lr_hidden(a.hidden, a.M, a.rank), dh = lr_hidden(a.ws, a.M, a.rank);
  const int rp = lr_rp(a.rank), R = static_cast<int>(a.R), grid = static_cast<int>(p.n_few);
  const T *x = static_cast<const T*>(a.x), *go = static_cast<const T*>(a.go);
  if (a.dx || a.da) {
    lr_shrink_kernel<T><<<grid, 256, 0, st>>>(p, go, a.ldgo, a.N, static_cast<const T*>(a.b), false, a.rank, rp, R, a.scales, dh);
    if (int rc = check_launch("lr_shrink_kernel")) return rc;
  }
  if (a.dx) {
    lr_expand_kernel<T><<<grid, 256, 0, st>>>(p, dh, static_cast<const T*>(a.a), false, a.rank, rp, R, nullptr, 0,
                                             static_cast<T*>(a.dx), a.lddx, a.K);
    if (int rc = check_launch("lr_expand_kernel")) return rc;
  }
  if (a.da) {
    lr_wgrad_kernel<T><<<dim3(static_cast<unsigned>((a.K * a.rank + 255) / 256), R), 256, 0, st>>>(p, dh, x, a.ldx, a.K, a.rank, rp, true, static_cast<T*>(a.da));
    if (int rc = check_launch("lr_wgrad_kernel")) return rc;
  }
  if (a.db) {
    lr_wgrad_kernel<T><<<dim3(static_cast<unsigned>((a.N * a.rank + 255) / 256), R), 256, 0, st>>>(p, h, go, a.ldgo, a.N, a.rank, rp, false, static_cast<T*>(a.db));
    if (int rc = check_launch("lr_wgrad_kernel")) return rc;
  }
  return H3B_OK;
}
int lr_forward(const LrArgs& a, cudaStream_t st) {
  return a.dtype == H3B_FP16 ? lr_forward_t<__half>(a, st) : lr_forward_t<__nv_bfloat16>(a, st);
}
int lr_backward(const LrArgs& a, cudaStream_t st) {
  if (a.M == 0) {  // no plan to read: nothing has rows
    for (auto [p, n] : {std::make_pair(a.da, a.K), std::make_pair(a.db, a.N)}) {
      const cudaError_t e = p ? cudaMemsetAsync(p, 0, static_cast<size_t>(a.R) * a.rank * n * 2, st) : cudaSuccess;
      if (e != cudaSuccess) return cuda_fail(e, "cudaMemsetAsync(gradients of adapters without rows)");
    }
    return H3B_OK;
  }
  return a.dtype == H3B_FP16 ? lr_backward_t<__half>(a, st) : lr_backward_t<__nv_bfloat16>(a, st);
}

}  // namespace h3b
