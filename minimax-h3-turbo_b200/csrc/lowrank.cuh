// Low-rank adapters of many requests beside a shared projection, and their gradients.
//
//   out_i = base_i + s_g (x_i A_g^T) B_g^T        g: the adapter of row i; rows without one keep base_i
//   h_i = s_g x_i A_g^T                           [rank], held in 32 bits until it is an operand of the second product
//   dh_i = s_g go_i B_g,   dx_i = dh_i A_g,   dA_g = sum_i dh_i^T x_i,   dB_g = sum_i go_i^T h_i
//
// The rows are gone through in the plan's order (by adapter, then by row), in tiles of one adapter's rows; rows are gathered by their
// numbers, so a batch may hold its requests in any order.
#pragma once
#include <type_traits>
#include <utility>

#include "cross_common.cuh"

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
// begin in it (group R: rows without one); slot [R + 1], below; then tables of four numbers a line:
//   tiles  (adapter, first place in order, rows, 0), up to LR_TILE rows each
//   few    the same, up to LR_FEW rows each
//   units  (adapter, first tile, tiles, slot), up to lr_unit_tiles(M) tiles each: what a CTA of the weight gradients adds up.  The
//          units of an adapter that has several have a slot each, slot[g] to slot[g + 1], for their partial sums; else -1
// Unused lines of a table have no rows (no tiles).
constexpr int LR_TILE = 128, LR_FEW = 8;
constexpr int LR_SPLITS = 16;  // units that all rows are dealt out to, if they are one adapter's
struct LrPlan {
  const int32_t* order;
  const int32_t* offset;
  const int32_t* slot;
  const int4* tiles;
  const int4* few;
  const int4* units;
  int64_t n_tiles, n_few, n_units;  // lines of the tables, used or not
  int unit_tiles;
};
static int64_t lr_up4(int64_t v) { return (v + 3) / 4 * 4; }
static int64_t lr_lines(int64_t M, int64_t R, int rows) { return M / rows + (R + 1 < M ? R + 1 : M); }
static int lr_unit_tiles(int64_t M) { return static_cast<int>((M + LR_TILE * LR_SPLITS - 1) / (LR_TILE * LR_SPLITS)); }
static int64_t lr_unit_lines(int64_t M, int64_t R) { return lr_lines(M, R, LR_TILE) / lr_unit_tiles(M) + (R < M ? R : M); }
// An adapter with several units has more than lr_unit_tiles(M) >= M / (LR_TILE LR_SPLITS) tiles, of which all but one are full: there
// are at most LR_SPLITS of them, and their units are at most (M / LR_TILE + LR_SPLITS) / lr_unit_tiles(M) + LR_SPLITS.
static int64_t lr_slots(int64_t M) { return (M / LR_TILE + LR_SPLITS) / lr_unit_tiles(M) + LR_SPLITS; }
static LrPlan lr_plan(const int32_t* p, int64_t M, int64_t R) {
  LrPlan pl{};
  pl.order = p;
  pl.offset = p + lr_up4(M);
  pl.slot = pl.offset + lr_up4(R + 2);
  pl.tiles = reinterpret_cast<const int4*>(pl.slot + lr_up4(R + 1));
  pl.n_tiles = lr_lines(M, R, LR_TILE);
  pl.few = pl.tiles + pl.n_tiles;
  pl.n_few = lr_lines(M, R, LR_FEW);
  pl.units = pl.few + pl.n_few;
  pl.n_units = lr_unit_lines(M, R);
  pl.unit_tiles = lr_unit_tiles(M);
  return pl;
}
int64_t lr_plan_size(int64_t M, int64_t R) {
  return M == 0 ? 0 : lr_up4(M) + lr_up4(R + 2) + lr_up4(R + 1) +
                          4 * (lr_lines(M, R, LR_TILE) + lr_lines(M, R, LR_FEW) + lr_unit_lines(M, R));
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
// One CTA: the tables, from the offsets.  1024 adapters at a time: their numbers of lines are added up, then every warp writes
// those of its 32 adapters, a lane per line.
static __global__ void __launch_bounds__(LR_PLAN_THREADS) lr_tables_kernel(const LrPlan p, int R) {
  constexpr int W = LR_PLAN_THREADS / 32;
  __shared__ int4 sums[W];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, per = p.unit_tiles;
  int4* const tiles = const_cast<int4*>(p.tiles);
  int4* const few = const_cast<int4*>(p.few);
  int4* const units = const_cast<int4*>(p.units);
  int32_t* const slot = const_cast<int32_t*>(p.slot);
  int4 base = make_int4(0, 0, 0, 0);  // lines of tiles, few, units; slots
  for (int g0 = 0; g0 <= R; g0 += LR_PLAN_THREADS) {
    const int g = g0 + static_cast<int>(threadIdx.x);
    const int first = g <= R ? p.offset[g] : 0, n = g <= R ? p.offset[g + 1] - first : 0;
    int4 mine;
    mine.x = (n + LR_TILE - 1) / LR_TILE;
    mine.y = (n + LR_FEW - 1) / LR_FEW;
    mine.z = g < R ? (mine.x + per - 1) / per : 0;
    mine.w = mine.z > 1 ? mine.z : 0;
    int4 inc = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const int4 v = make_int4(__shfl_up_sync(0xffffffffu, inc.x, o), __shfl_up_sync(0xffffffffu, inc.y, o),
                               __shfl_up_sync(0xffffffffu, inc.z, o), __shfl_up_sync(0xffffffffu, inc.w, o));
      if (lane >= o) inc.x += v.x, inc.y += v.y, inc.z += v.z, inc.w += v.w;
    }
    if (lane == 31) sums[w] = inc;
    __syncthreads();
    int4 at = make_int4(base.x + inc.x - mine.x, base.y + inc.y - mine.y, base.z + inc.z - mine.z, base.w + inc.w - mine.w);
    for (int i = 0; i < W; ++i) {
      const int4 v = sums[i];
      if (i < w) at.x += v.x, at.y += v.y, at.z += v.z, at.w += v.w;
      base.x += v.x, base.y += v.y, base.z += v.z, base.w += v.w;
    }
    if (g <= R) slot[g] = at.w;
    for (int l = 0; l < 32; ++l) {
      const int rows = __shfl_sync(0xffffffffu, n, l), from = __shfl_sync(0xffffffffu, first, l), who = g0 + 32 * w + l;
      const int4 t = make_int4(__shfl_sync(0xffffffffu, at.x, l), __shfl_sync(0xffffffffu, at.y, l),
                               __shfl_sync(0xffffffffu, at.z, l), __shfl_sync(0xffffffffu, at.w, l));
      const int nt = (rows + LR_TILE - 1) / LR_TILE, nu = who < R ? (nt + per - 1) / per : 0;
      for (int i = lane; i < nt; i += 32) tiles[t.x + i] = make_int4(who, from + i * LR_TILE, min(LR_TILE, rows - i * LR_TILE), 0);
      for (int i = lane; i < (rows + LR_FEW - 1) / LR_FEW; i += 32)
        few[t.y + i] = make_int4(who, from + i * LR_FEW, min(LR_FEW, rows - i * LR_FEW), 0);
      for (int i = lane; i < nu; i += 32) units[t.z + i] = make_int4(who, t.x + i * per, min(per, nt - i * per), nu > 1 ? t.w + i : -1);
    }
    __syncthreads();
  }
  for (int64_t i = base.x + threadIdx.x; i < p.n_tiles; i += LR_PLAN_THREADS) tiles[i] = make_int4(R, 0, 0, 0);
  for (int64_t i = base.y + threadIdx.x; i < p.n_few; i += LR_PLAN_THREADS) few[i] = make_int4(R, 0, 0, 0);
  for (int64_t i = base.z + threadIdx.x; i < p.n_units; i += LR_PLAN_THREADS) units[i] = make_int4(R, 0, 0, -1);
}
int lr_plan_launch(const int32_t* rows, int64_t M, int64_t R, int32_t* plan, cudaStream_t st) {
  const LrPlan p = lr_plan(plan, M, R);
  lr_order_kernel<<<static_cast<int>(R) + 1, LR_PLAN_THREADS, 0, st>>>(rows, M, static_cast<int>(R), const_cast<int32_t*>(p.order),
                                                                      const_cast<int32_t*>(p.offset));
  if (int rc = check_launch("lr_order_kernel")) return rc;
  lr_tables_kernel<<<1, LR_PLAN_THREADS, 0, st>>>(p, static_cast<int>(R));
  return check_launch("lr_tables_kernel");
}

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
// ----------------------------------------------------------------------------------------------- common parts of the tile kernels
// 16 bytes from global to shared memory without passing through registers; zeros where ok is false (nothing is read then)
__device__ __forceinline__ void lr_copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void lr_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void lr_copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Instruction descriptor of tcgen05.mma kind::f16: a_mn / b_mn: the operand's M or N index is the contiguous one
template <typename T>
__host__ __device__ constexpr uint32_t lr_idesc(int m, int n, bool a_mn, bool b_mn) {
  return idesc_f16<T>(m, n, b_mn) | static_cast<uint32_t>(a_mn) << 15;
}
// Low word of the descriptor of a tile whose rows are K and whose columns are M or N (desc_chan for parts of another size)
__device__ __forceinline__ uint32_t lr_desc_mn(uint32_t tile, uint32_t part_bytes) {
  return (tile & 0x3FFFFu) >> 4 | (part_bytes >> 4) << 16;
}
__device__ __forceinline__ uint32_t lr_tmem_cols(int n) { return n <= 32 ? 32u : n <= 64 ? 64u : 128u; }
// the warp's copies of a stage have arrived: visible to the tensor cores, then counted
__device__ __forceinline__ void lr_arrive_full(uint64_t* bar) {
  fence_proxy_async_smem();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// ----------------------------------------------------------------------------------------------- first product: hidden rows
// H [128 rows, rp] of a tile = X [128, C] W, C the contraction: W is A_g [rank, C] (W_ROWS) or B_g [C, rank].  HBM-bound: X is read
// once, 2 rank flops a byte.  The CTAs of a cluster share a tile's C (95 tiles of 12090 rows would leave a third of the SMs idle)
// and add their parts up through distributed shared memory in a fixed order.  Copies are cp.async of 16 bytes, since rows are
// gathered.  Warps 0-3 copy, then read the accumulators; warp 4 issues the products.
constexpr int LR_XPART = LR_TILE * 128;  // 64 channels of 128 rows
constexpr int LR_SHRINK_THREADS = 160;
template <int STAGES>  // 5 with W_ROWS only: B_g's parts are 64 channels wide
struct LrShrinkCfg {
  static constexpr int RP = STAGES == 5 ? 32 : STAGES == 4 ? 64 : 128;  // the largest rp of this variant
  static constexpr int WBYTES = RP * 128;
  static constexpr int STAGE = LR_XPART + WBYTES;
  static constexpr int SMEM = STAGES * STAGE + 1024;
};
// The power of two that brings a row whose largest magnitude is `top` into [1, 2); the smallest for rows of zeros (which
// then has no say in the largest of several rows), 1 for infinities and NaN.
__device__ __forceinline__ float lr_power(float top) {
  const int e = (__float_as_int(top) >> 23) & 0xFF;
  return e >= 253 ? 1.f : __int_as_float(max(e, 1) << 23);
}

template <typename T, bool W_ROWS, int STAGES>
__global__ void __launch_bounds__(LR_SHRINK_THREADS) lr_shrink_kernel(const LrPlan p, const T* x, int64_t ldx, int64_t C,
                                                                      const T* w, int rank, int ldw, int rp, int R, const float* scales, const LrHidden out,
                                                                      int splits) {
  using Cfg = LrShrinkCfg<STAGES>;
  extern __shared__ unsigned char lr_smem[];
  __shared__ uint64_t full[STAGES], empty[STAGES], done;
  __shared__ uint32_t tmem_at;
  __shared__ int abort_flag;
  after_previous();
  const int tile = blockIdx.x / splits, split = blockIdx.x - tile * splits;
  const int4 t = p.tiles[tile];
  if (t.z == 0 || t.x >= R) return;  // the same for every CTA of the cluster
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned char* const base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(lr_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  volatile int* abort = &abort_flag;
  const int chunks = static_cast<int>((C + 63) / 64), per = (chunks + splits - 1) / splits;
  const int c0 = min(split * per, chunks), n = min(per, chunks - c0);
  if (warp == 4) {
    if (lane == 0) {
      for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 4), mbar_init(&empty[i], 1);
      mbar_init(&done, 1);
      mbar_fence_init();
      abort_flag = 0;
    }
    tmem_alloc(&tmem_at, lr_tmem_cols(rp));
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  if (warp == 4) {
    const uint32_t idesc = lr_idesc<T>(LR_TILE, rp, false, !W_ROWS);
    for (int i = 0; i < n; ++i) {
      const int s = i % STAGES;
      warp_wait(&full[s], (i / STAGES) & 1, abort);
      tc_fence_after();
      const uint32_t xs = smem_u32(base + s * Cfg::STAGE), ws = xs + LR_XPART;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_f16_ss(tmem, desc_rows(xs) + kk * 2, W_ROWS ? desc_rows(ws) + kk * 2 : lr_desc_mn(ws, 64 * 128) + kk * 128, idesc,
                     i > 0 || kk > 0);
      }
      __syncwarp();
      commit_one(&empty[s]);
    }
    commit_one(&done);
  } else {
    const int r0 = tid >> 3, ch = tid & 7;  // rows r0, r0 + 16, ...; 16-byte chunk of the part
    const T* xr[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = r0 + 16 * i;
      xr[i] = r < t.z ? x + static_cast<int64_t>(p.order[t.y + r]) * ldx + ch * 8 : nullptr;
    }
    const T* wg = w + static_cast<int64_t>(t.x) * (W_ROWS ? rank * C : C * ldw);
    const uint32_t at = static_cast<uint32_t>(r0 * 128 + ((ch ^ (r0 & 7)) << 4));
    for (int i = 0; i < n + STAGES - 1; ++i) {
      if (i < n) {
        const int s = i % STAGES;
        mbar_wait(&empty[s], ((i / STAGES) & 1) ^ 1, abort);
        const uint32_t xs = smem_u32(base + s * Cfg::STAGE) + at, ws = xs + LR_XPART;
        const int64_t c = static_cast<int64_t>(c0 + i) * 64;
        const bool in = c + ch * 8 < C;
#pragma unroll
        for (int j = 0; j < 8; ++j) lr_copy16(xs + j * 2048, xr[j] && in ? xr[j] + c : x, xr[j] && in);
        if constexpr (W_ROWS) {
#pragma unroll
          for (int j = 0; j < Cfg::RP / 16; ++j) {
            const int r = r0 + 16 * j;
            if (16 * j < rp) lr_copy16(ws + j * 2048, r < rank && in ? wg + r * C + c + ch * 8 : w, r < rank && in);
          }
        } else {
#pragma unroll
          for (int part = 0; part < (Cfg::RP + 63) / 64; ++part) {
            const int k = part * 64 + ch * 8;
            if (k < rp) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int64_t r = c + r0 + 16 * j;
                const bool ok = r < C && k < ldw;
                lr_copy16(ws + part * 8192 + j * 2048, ok ? wg + r * ldw + k : w, ok);
              }
            }
          }
        }
      }
      lr_copy_commit();
      if (i >= STAGES - 1) {
        lr_copy_wait<STAGES - 1>();
        lr_arrive_full(&full[(i - (STAGES - 1)) % STAGES]);
      }
    }
    warp_wait(&done, 0, abort);
    tc_fence_after();
  }
  // the parts of the cluster's CTAs through shared memory (the stages are free: every product has read its operands)
  const float scale = scales ? scales[t.x] : 1.f;
  float* const red = reinterpret_cast<float*>(base);
  const int ld = rp + 4;
  if (warp < 4) {
    for (int c = 0; c < rp; c += 16) {
      uint32_t v[16];
      if (n > 0) {
        tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + c, v);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4*>(red + tid * ld + c + 4 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
    tc_fence_before();
  }
  if (splits > 1) cluster_sync();
  else __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, lr_tmem_cols(rp));
  } else {
    // `splits` lanes to a row, rp / splits values each (an even number)
    const int row = split * (LR_TILE / splits) + tid / splits, w0 = rp / splits, cols = tid % splits * w0;
    float top = 0.f;
    for (int c = cols; c < cols + w0; c += 2) {
      float2 sum = make_float2(0.f, 0.f);
      const uint32_t mine = smem_u32(red + row * ld + c);
      for (int k = 0; k < splits; ++k) {
        float2 v;
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(mapa_rank(mine, k)) : "memory");
        sum.x += v.x, sum.y += v.y;
      }
      sum.x *= scale, sum.y *= scale;
      top = fmaxf(top, fmaxf(fabsf(sum.x), fabsf(sum.y)));
      *reinterpret_cast<float2*>(red + row * ld + c) = sum;  // read by this thread alone
    }
    float mult = 1.f;
    if constexpr (std::is_same_v<T, __half>) {
      for (int o = splits / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      mult = lr_power(top);
    }
    if (row < t.z) {
      const int64_t pos = t.y + row;
      const float inv = 1.f / mult;  // a power of two
      uint32_t* h = reinterpret_cast<uint32_t*>(static_cast<T*>(out.h) + pos * rp + cols);
      for (int c = 0; c < w0; c += 2) {
        const float2 v = *reinterpret_cast<const float2*>(red + row * ld + cols + c);
        h[c / 2] = pack2<T>(v.x * inv, v.y * inv);
      }
      if (cols == 0) out.mult[pos] = mult;
    }
  }
  if (splits > 1) cluster_sync();  // the others have read this CTA's part
}

// ----------------------------------------------------------------------------------------------- second product: out or dx
// out [128 rows, N] of a tile = base + H W^T: W is B_g [N, rank] (W_ROWS) or A_g [rank, N].  HBM-bound: base and out are touched once,
// 32 bytes of a row per thread and instruction (full sectors), the next 128 columns' base on the way while these are added.  Warps
// 0-7 read the accumulators (a row per lane, 64 columns per warp), 8-11 copy, 12 issues the products.
constexpr int LR_NT = 128;  // columns of a step
constexpr int LR_EXPAND_THREADS = 416;
template <int RPM>  // the largest rp of this variant: 64 or 128
struct LrExpandCfg {
  static constexpr int PARTS = RPM / 64, STAGES = RPM == 64 ? 3 : 2;
  static constexpr int TILE = PARTS * LR_XPART;
  static constexpr int SMEM = TILE + STAGES * TILE + 1024;
};
// 16 columns of a row, `left` of them in the tensor (a multiple of 8)
template <typename T>
__device__ __forceinline__ void lr_load16(const T* p, int64_t left, bool wide, uint32_t (&v)[8]) {
  if (left >= 16 && wide) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "l"(p)
                 : "memory");
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (left > 8 * i) u = *reinterpret_cast<const uint4*>(p + 8 * i);
    v[4 * i] = u.x, v[4 * i + 1] = u.y, v[4 * i + 2] = u.z, v[4 * i + 3] = u.w;
  }
}
template <typename T>
__device__ __forceinline__ void lr_store16(T* p, int64_t left, bool wide, const uint32_t (&v)[8]) {
  if (left >= 16 && wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (left > 8 * i) *reinterpret_cast<uint4*>(p + 8 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}
template <typename T>
__device__ __forceinline__ float2 lr_unpack2(uint32_t w) {
  if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

template <typename T, bool W_ROWS, int RPM>
__global__ void __launch_bounds__(LR_EXPAND_THREADS, 2) lr_expand_kernel(const LrPlan p, const LrHidden hid, const T* w,
                                                                         int rank, int ldw, int rp, int R, const T* base, int64_t ldb,
                                                                         T* out, int64_t ldo, int64_t N, int per, int parts, bool wide) {
  using Cfg = LrExpandCfg<RPM>;
  constexpr int ST = Cfg::STAGES;
  extern __shared__ unsigned char lr_smem[];
  __shared__ uint64_t full[ST], empty[ST], h_full, acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_at;
  __shared__ int abort_flag;
  after_previous();
  const int tile = blockIdx.x / parts;  // `parts` CTAs to a tile, `per` steps of columns each
  const int4 t = p.tiles[tile];
  if (t.z == 0) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int steps = static_cast<int>((N + LR_NT - 1) / LR_NT), s0 = (blockIdx.x - tile * parts) * per, n = min(per, steps - s0);
  if (t.x >= R) {  // rows without an adapter
    if (base == out) return;
    const int64_t from = static_cast<int64_t>(s0) * LR_NT, cols = min(static_cast<int64_t>(n) * LR_NT, N - from) / 8;
    for (int r = warp; r < t.z; r += LR_EXPAND_THREADS / 32) {
      const int64_t row = p.order[t.y + r];
      for (int64_t c = lane; c < cols; c += 32)
        *reinterpret_cast<uint4*>(out + row * ldo + from + 8 * c) =
            base ? *reinterpret_cast<const uint4*>(base + row * ldb + from + 8 * c) : make_uint4(0, 0, 0, 0);
    }
    return;
  }
  unsigned char* const hs = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(lr_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* const wsm = hs + Cfg::TILE;
  volatile int* abort = &abort_flag;
  if (warp == 12) {
    if (lane == 0) {
      for (int i = 0; i < ST; ++i) mbar_init(&full[i], 4), mbar_init(&empty[i], 1);
      for (int i = 0; i < 2; ++i) mbar_init(&acc_full[i], 1), mbar_init(&acc_empty[i], 8);
      mbar_init(&h_full, 4);
      mbar_fence_init();
      abort_flag = 0;
    }
    tmem_alloc(&tmem_at, 2 * LR_NT);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  if (warp < 8) {
    const int r = 32 * (warp & 3) + lane, half = warp >> 2;
    const bool valid = r < t.z;
    const int64_t row = valid ? p.order[t.y + r] : 0;
    const float mult = std::is_same_v<T, __half> && valid ? hid.mult[t.y + r] : 1.f;
    int64_t c = static_cast<int64_t>(s0) * LR_NT + half * 64;
    const T* b = base + row * ldb + c;
    T* o = out + row * ldo + c;
    int64_t left = valid ? N - c : 0;
    uint32_t v[4][8];
#pragma unroll
    for (int k = 0; k < 4; ++k) lr_load16(b + 16 * k, base ? left - 16 * k : 0, wide, v[k]);
    for (int i = 0; i < n; ++i) {
      const int buf = i & 1;
      warp_wait(&acc_full[buf], (i >> 1) & 1, abort);
      tc_fence_after();
      const bool more = i + 1 < n && base;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t a[16];
        tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + buf * LR_NT + half * 64 + 16 * k, a);
        tmem_ld_wait();
        if (k == 3) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[buf]);
        }
        uint32_t res[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 f = lr_unpack2<T>(v[k][j]);
          res[j] = pack2<T>(fmaf(__uint_as_float(a[2 * j]), mult, f.x), fmaf(__uint_as_float(a[2 * j + 1]), mult, f.y));
        }
        if (more) lr_load16(b + LR_NT + 16 * k, left - LR_NT - 16 * k, wide, v[k]);
        lr_store16(o + 16 * k, left - 16 * k, wide, res);
      }
      b += LR_NT, o += LR_NT, left -= LR_NT;
    }
  } else if (warp < 12) {
    const int pt = tid - 256, r0 = pt >> 3, ch = pt & 7;
    const uint32_t at = static_cast<uint32_t>(r0 * 128 + ((ch ^ (r0 & 7)) << 4));
    const T* h = static_cast<const T*>(hid.h);
#pragma unroll
    for (int part = 0; part < Cfg::PARTS; ++part) {
      const int k = part * 64 + ch * 8;
      if (k < rp) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = r0 + 16 * j;
          lr_copy16(smem_u32(hs + part * LR_XPART) + at + j * 2048, r < t.z ? h + static_cast<int64_t>(t.y + r) * rp + k : h, r < t.z);
        }
      }
    }
    lr_copy_commit();
    const T* wg = w + static_cast<int64_t>(t.x) * (W_ROWS ? N * ldw : rank * N);
    for (int i = 0; i < n + ST - 1; ++i) {
      if (i < n) {
        const int s = i % ST;
        mbar_wait(&empty[s], ((i / ST) & 1) ^ 1, abort);
        const uint32_t dst = smem_u32(wsm + s * Cfg::TILE) + at;
        const int64_t c = static_cast<int64_t>(s0 + i) * LR_NT;
        if constexpr (W_ROWS) {
#pragma unroll
          for (int part = 0; part < Cfg::PARTS; ++part) {
            const int k = part * 64 + ch * 8;
            if (k < rp) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const int64_t r = c + r0 + 16 * j;
                const bool ok = r < N && k < ldw;
                lr_copy16(dst + part * LR_XPART + j * 2048, ok ? wg + r * ldw + k : w, ok);
              }
            }
          }
        } else {
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            const int64_t k = c + part * 64 + ch * 8;
#pragma unroll
            for (int j = 0; j < RPM / 16; ++j) {
              const int r = r0 + 16 * j;
              const bool ok = r < rank && k < N;
              if (16 * j < rp) lr_copy16(dst + part * rp * 128 + j * 2048, ok ? wg + r * N + k : w, ok);
            }
          }
        }
      }
      lr_copy_commit();
      if (i == 0) {
        lr_copy_wait<1>();
        lr_arrive_full(&h_full);
      }
      if (i >= ST - 1) {
        lr_copy_wait<ST - 1>();
        lr_arrive_full(&full[(i - (ST - 1)) % ST]);
      }
    }
  } else {
    const uint32_t idesc = lr_idesc<T>(LR_TILE, LR_NT, false, !W_ROWS), ha = desc_rows(smem_u32(hs));
    warp_wait(&h_full, 0, abort);
    for (int i = 0; i < n; ++i) {
      const int s = i % ST, buf = i & 1;
      warp_wait(&full[s], (i / ST) & 1, abort);
      warp_wait(&acc_empty[buf], ((i >> 1) & 1) ^ 1, abort);
      tc_fence_after();
      const uint32_t ws = smem_u32(wsm + s * Cfg::TILE);
      if (elect_one())
        for (int kk = 0; kk < rp / 16; ++kk)
          mma_f16_ss(tmem + buf * LR_NT, ha + rows_step(kk), W_ROWS ? desc_rows(ws) + rows_step(kk) : lr_desc_mn(ws, rp * 128) + kk * 128,
                     idesc, kk > 0);
      __syncwarp();
      commit_one(&empty[s]);
      commit_one(&acc_full[buf]);
    }
  }
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * LR_NT);
  }
}

// ----------------------------------------------------------------------------------------------- weight gradients
// D [128 channels, rp] = X^T H over the rows of a unit (a stretch of one adapter's rows): X's columns are M, H's are N, rows are K,
// all read as they lie in memory.  HBM-bound: X is read once; H comes from L2.  Rows behind the last are zeros in both operands.  One
// launch does dA (x with dh) and dB (grad_out with h).  fp16: a row's power of two is taken out against the largest of the unit.
// Warps 0-3 copy, then read the accumulators; warp 4 issues the products.
constexpr int LR_KROWS = 64;  // rows of a stage
template <int RPM>
struct LrWgradCfg {
  static constexpr int PARTS = RPM / 64, STAGES = RPM == 64 ? 4 : 3;
  static constexpr int XBYTES = 2 * LR_KROWS * 128, STAGE = XBYTES + PARTS * LR_KROWS * 128;
  static constexpr int SMEM = STAGES * STAGE + 1024;
};
template <typename T>
struct LrWgradSide {
  const T* x;
  int64_t ldx, C;
  LrHidden hid;
  T* grad;       // [rank][C] (by_rank) or [C][rank] of every adapter
  float* part;   // [slots][C][rp]
  int blocks;    // of 128 channels
  bool by_rank;
};
template <typename T, int RPM>
__global__ void __launch_bounds__(160) lr_wgrad_kernel(const LrPlan p, const LrWgradSide<T> sa, const LrWgradSide<T> sb, int rank, int rp,
                                                       int R) {
  using Cfg = LrWgradCfg<RPM>;
  constexpr int ST = Cfg::STAGES;
  extern __shared__ unsigned char lr_smem[];
  __shared__ uint64_t full[ST], empty[ST], done;
  __shared__ uint32_t tmem_at;
  __shared__ int abort_flag;
  __shared__ float tops[4];
  after_previous();
  const int both = sa.blocks + sb.blocks, unit = blockIdx.x / both, block = blockIdx.x - unit * both;
  const int4 u = p.units[unit];
  if (u.z == 0 || u.x >= R) return;
  const bool second = block >= sa.blocks;
  const LrWgradSide<T>& sd = second ? sb : sa;
  const int64_t col = static_cast<int64_t>(second ? block - sa.blocks : block) * 128;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int4 first = p.tiles[u.y], last = p.tiles[u.y + u.z - 1];
  const int p0 = first.y, rows = last.y + last.z - p0, n = (rows + LR_KROWS - 1) / LR_KROWS;
  unsigned char* const base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(lr_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  volatile int* abort = &abort_flag;
  if (warp == 4) {
    if (lane == 0) {
      for (int i = 0; i < ST; ++i) mbar_init(&full[i], 4), mbar_init(&empty[i], 1);
      mbar_init(&done, 1);
      mbar_fence_init();
      abort_flag = 0;
    }
    tmem_alloc(&tmem_at, lr_tmem_cols(rp));
    tmem_relinquish();
  } else if (std::is_same_v<T, __half>) {
    float top = 0.f;
    for (int i = tid; i < rows; i += 128) top = fmaxf(top, sd.hid.mult[p0 + i]);
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) tops[warp] = top;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  if (warp == 4) {
    const uint32_t idesc = lr_idesc<T>(128, rp, true, true);
    for (int i = 0; i < n; ++i) {
      const int s = i % ST;
      warp_wait(&full[s], (i / ST) & 1, abort);
      tc_fence_after();
      const uint32_t xs = smem_u32(base + s * Cfg::STAGE), hs = xs + Cfg::XBYTES;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < LR_KROWS / 16; ++kk)
          mma_f16_ss(tmem, lr_desc_mn(xs, LR_KROWS * 128) + kk * 128, lr_desc_mn(hs, LR_KROWS * 128) + kk * 128, idesc, i > 0 || kk > 0);
      }
      __syncwarp();
      commit_one(&empty[s]);
    }
    commit_one(&done);
  } else {
    const float top = std::is_same_v<T, __half> ? fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) : 1.f;
    const int r0 = tid >> 3, ch = tid & 7;
    const uint32_t at = static_cast<uint32_t>(r0 * 128 + ((ch ^ (r0 & 7)) << 4));
    const T* h = static_cast<const T*>(sd.hid.h);
    int next[4];  // numbers of the next stage's rows
    auto numbers = [&](int i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = i * LR_KROWS + r0 + 16 * j;
        next[j] = r < rows ? p.order[p0 + r] : -1;
      }
    };
    numbers(0);
    for (int i = 0; i < n + ST - 1; ++i) {
      if (i < n) {
        const int s = i % ST;
        const T* xr[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) xr[j] = next[j] >= 0 ? sd.x + next[j] * sd.ldx + col : nullptr;
        if (i + 1 < n) numbers(i + 1);
        mbar_wait(&empty[s], ((i / ST) & 1) ^ 1, abort);
        const uint32_t dst = smem_u32(base + s * Cfg::STAGE) + at;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          const int k = part * 64 + ch * 8;
          const bool in = col + k < sd.C;
#pragma unroll
          for (int j = 0; j < 4; ++j) lr_copy16(dst + part * (LR_KROWS * 128) + j * 2048, xr[j] && in ? xr[j] + k : sd.x, xr[j] && in);
        }
#pragma unroll
        for (int part = 0; part < Cfg::PARTS; ++part) {
          const int k = part * 64 + ch * 8;
          if (k < rp) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int r = i * LR_KROWS + r0 + 16 * j;
              const uint32_t to = dst + Cfg::XBYTES + part * (LR_KROWS * 128) + j * 2048;
              const T* src = h + static_cast<int64_t>(p0 + r) * rp + k;
              if constexpr (std::is_same_v<T, __half>) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (r < rows) {
                  v = *reinterpret_cast<const uint4*>(src);
                  const __half2 f = __float2half2_rn(sd.hid.mult[p0 + r] / top);
                  __half2* e = reinterpret_cast<__half2*>(&v);
#pragma unroll
                  for (int q = 0; q < 4; ++q) e[q] = __hmul2(e[q], f);
                }
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
              } else {
                lr_copy16(to, r < rows ? src : h, r < rows);
              }
            }
          }
        }
      }
      lr_copy_commit();
      if (i >= ST - 1) {
        lr_copy_wait<ST - 1>();
        lr_arrive_full(&full[(i - (ST - 1)) % ST]);
      }
    }
    warp_wait(&done, 0, abort);
    tc_fence_after();
    const int64_t c = col + tid;  // a channel per lane
    for (int j = 0; j < rp; j += 16) {
      uint32_t v[16];
      tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + j, v);
      tmem_ld_wait();
      if (c >= sd.C) {
      } else if (u.w >= 0) {
        store_cols_f32(sd.part + (u.w * sd.C + c) * rp + j, v, top, 16);
      } else {
        T* g = sd.grad + static_cast<int64_t>(u.x) * rank * sd.C;
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (j + k < rank) g[sd.by_rank ? (j + k) * sd.C + c : c * rank + j + k] = lr_t<T>(__uint_as_float(v[k]) * top);
      }
      __syncwarp();
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, lr_tmem_cols(rp));
  }
}
// The parts of an adapter's units, added up in their order; zeros for adapters without rows.  A CTA: 32 channels of one adapter.
template <typename T>
__global__ void __launch_bounds__(256) lr_join_kernel(const LrPlan p, const LrWgradSide<T> sa, const LrWgradSide<T> sb, int blocks_a,
                                                      int rank, int rp) {
  __shared__ float sums[32][H3B_MAX_RANK + 1];
  after_previous();
  const int g = blockIdx.y;
  const int s0 = p.slot[g], s1 = p.slot[g + 1];
  const bool none = p.offset[g] == p.offset[g + 1];
  if (s0 == s1 && !none) return;
  const bool second = static_cast<int>(blockIdx.x) >= blocks_a;
  const LrWgradSide<T>& sd = second ? sb : sa;
  const int64_t col = static_cast<int64_t>(second ? blockIdx.x - blocks_a : blockIdx.x) * 32;
  const int cols = static_cast<int>(min(static_cast<int64_t>(32), sd.C - col));
  for (int e = threadIdx.x; e < cols * rp; e += 256) {
    const float* from = sd.part + col * rp + e;
    float sum = 0.f;
#pragma unroll 8
    for (int s = s0; s < s1; ++s) sum += from[s * sd.C * rp];
    sums[e / rp][e % rp] = sum;
  }
  __syncthreads();
  T* out = sd.grad + static_cast<int64_t>(g) * rank * sd.C;
  for (int e = threadIdx.x; e < cols * rank; e += 256) {
    const int c = sd.by_rank ? e % cols : e / rank, j = sd.by_rank ? e / cols : e % rank;
    out[sd.by_rank ? j * sd.C + col + c : (col + c) * rank + j] = lr_t<T>(sums[c][j]);
  }
}

// b [R, N, rank] with rows of ld = rank rounded up to 8 (zeros behind): rows of other ranks do not start on 16-byte boundaries
template <typename T>
__global__ void __launch_bounds__(256) lr_pad_kernel(const T* __restrict__ b, T* __restrict__ to, int64_t rows, int rank, int ld) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < rows * ld; i += gridDim.x * 256ll) {
    const int64_t r = i / ld;
    const int j = static_cast<int>(i - r * ld);
    to[i] = j < rank ? b[r * rank + j] : lr_t<T>(0.f);
  }
}

// ----------------------------------------------------------------------------------------------- launches
static int lr_ldw(int rank) { return (rank + 7) / 8 * 8; }
// A workspace: hidden rows, padded b, parts of the weight gradients
struct LrSpace {
  size_t hidden, pad, part_a, part_b, total;
};
static LrSpace lr_space(int64_t M, int64_t K, int64_t N, int rank, int64_t R, bool backward) {
  LrSpace s{};
  s.pad = lr_hidden_bytes(M, rank);
  s.part_a = s.pad + (rank % 8 ? lr_up256(static_cast<size_t>(R) * N * lr_ldw(rank) * 2) : 0);
  const size_t slot = backward ? static_cast<size_t>(lr_slots(M)) * lr_rp(rank) * 4 : 0;
  s.part_b = s.part_a + lr_up256(slot * K);
  s.total = s.part_b + lr_up256(slot * N);
  return s;
}
size_t lr_workspace(int64_t M, int64_t K, int64_t N, int rank, int64_t R, bool backward) {
  return M == 0 ? 0 : lr_space(M, K, N, rank, R, backward).total;
}
// CTAs of a cluster that share a tile's contraction: as many as fill the SMs twice, at most a fourth of the steps
static int lr_splits(int64_t tiles, int64_t C) {
  const int64_t chunks = (C + 63) / 64;
  int s = 1;
  while (s < 8 && tiles * s < 2 * cross_sms() && chunks >= 8 * s) s *= 2;
  return s;
}
template <typename... KA, typename... A>
static int lr_launch(const char* what, void (*kernel)(KA...), std::atomic<bool> (&ready)[CA_DEVICES], dim3 grid, int threads, int smem,
                     int cluster, cudaStream_t st, A&&... args) {
  if (int rc = cross_smem(reinterpret_cast<const void*>(kernel), smem, ready, what)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<KA>(args)...);
  return e == cudaSuccess ? check_launch(what) : cuda_fail(e, what);
}
template <typename T, bool W_ROWS, int STAGES>
static int lr_shrink_s(const LrPlan& p, const T* x, int64_t ldx, int64_t C, const T* w, int rank, int ldw, int rp, int R,
                       const float* scales, const LrHidden& h, cudaStream_t st) {
  static std::atomic<bool> ready[CA_DEVICES];
  const int splits = lr_splits(p.n_tiles, C);
  return lr_launch("lr_shrink_kernel", lr_shrink_kernel<T, W_ROWS, STAGES>, ready, dim3(static_cast<unsigned>(p.n_tiles * splits)),
                   LR_SHRINK_THREADS, LrShrinkCfg<STAGES>::SMEM, splits, st, p, x, ldx, C, w, rank, ldw, rp, R, scales, h, splits);
}
template <typename T, bool W_ROWS>
static int lr_shrink(const LrPlan& p, const T* x, int64_t ldx, int64_t C, const T* w, int rank, int ldw, int R, const float* scales,
                     const LrHidden& h, cudaStream_t st) {
  const int rp = lr_rp(rank);
  if constexpr (W_ROWS)
    if (rp <= 32) return lr_shrink_s<T, W_ROWS, 5>(p, x, ldx, C, w, rank, ldw, rp, R, scales, h, st);
  if (rp <= 64) return lr_shrink_s<T, W_ROWS, 4>(p, x, ldx, C, w, rank, ldw, rp, R, scales, h, st);
  return lr_shrink_s<T, W_ROWS, 3>(p, x, ldx, C, w, rank, ldw, rp, R, scales, h, st);
}
template <typename T, bool W_ROWS, int RPM>
static int lr_expand_s(const LrPlan& p, const LrHidden& h, const T* w, int rank, int ldw, int rp, int R, const T* base, int64_t ldb, T* out,
                       int64_t ldo, int64_t N, cudaStream_t st) {
  static std::atomic<bool> ready[CA_DEVICES];
  const int64_t steps = (N + LR_NT - 1) / LR_NT;
  // eight CTAs to an SM in all, of two steps at least (a CTA's start costs about as much as one)
  int64_t per = p.n_tiles * steps / (8 * cross_sms());
  per = per < 2 ? 2 : per > 16 ? 16 : per;
  const int parts = static_cast<int>((steps + per - 1) / per);
  const bool wide = ldo % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 32 == 0 &&
                    (!base || (ldb % 16 == 0 && reinterpret_cast<uintptr_t>(base) % 32 == 0));
  return lr_launch("lr_expand_kernel", lr_expand_kernel<T, W_ROWS, RPM>, ready,
                   dim3(static_cast<unsigned>(p.n_tiles * parts)), LR_EXPAND_THREADS, LrExpandCfg<RPM>::SMEM, 1, st, p, h, w, rank, ldw,
                   rp, R, base, ldb, out, ldo, N, static_cast<int>(per), parts, wide);
}
template <typename T, bool W_ROWS>
static int lr_expand(const LrPlan& p, const LrHidden& h, const T* w, int rank, int ldw, int R, const T* base, int64_t ldb, T* out, int64_t ldo,
                     int64_t N, cudaStream_t st) {
  const int rp = lr_rp(rank);
  if (rp <= 64) return lr_expand_s<T, W_ROWS, 64>(p, h, w, rank, ldw, rp, R, base, ldb, out, ldo, N, st);
  return lr_expand_s<T, W_ROWS, 128>(p, h, w, rank, ldw, rp, R, base, ldb, out, ldo, N, st);
}
template <typename T, int RPM>
static int lr_wgrad(const LrPlan& p, const LrWgradSide<T>& a, const LrWgradSide<T>& b, int rank, int R, cudaStream_t st) {
  static std::atomic<bool> ready[CA_DEVICES], joined[CA_DEVICES];
  const int rp = lr_rp(rank);
  const int64_t grid = p.n_units * (a.blocks + b.blocks);
  if (int rc = lr_launch("lr_wgrad_kernel", lr_wgrad_kernel<T, RPM>, ready, dim3(static_cast<unsigned>(grid)), 160, LrWgradCfg<RPM>::SMEM,
                         1, st, p, a, b, rank, rp, R))
    return rc;
  const int ja = static_cast<int>((a.blocks ? a.C + 31 : 0) / 32), jb = static_cast<int>((b.blocks ? b.C + 31 : 0) / 32);
  return lr_launch("lr_join_kernel", lr_join_kernel<T>, joined, dim3(ja + jb, R), 256, 0, 1, st, p, a, b, ja, rank, rp);
}
template <typename T>
static int lr_pad(const LrArgs& a, const LrSpace& s, const T*& b, cudaStream_t st) {
  if (a.rank % 8 == 0) return H3B_OK;
  T* to = reinterpret_cast<T*>(static_cast<char*>(a.ws) + s.pad);
  const int64_t rows = a.R * a.N, blocks = (rows * lr_ldw(a.rank) + 1023) / 1024, cap = 8ll * cross_sms();
  lr_pad_kernel<T><<<static_cast<unsigned>(blocks < cap ? blocks : cap), 256, 0, st>>>(b, to, rows, a.rank, lr_ldw(a.rank));
  b = to;
  return check_launch("lr_pad_kernel");
}

template <typename T>
static int lr_forward_t(const LrArgs& a, cudaStream_t st) {
  const LrPlan p = lr_plan(a.plan, a.M, a.R);
  const LrSpace s = lr_space(a.M, a.K, a.N, a.rank, a.R, false);
  const LrHidden h = lr_hidden(a.hidden ? a.hidden : a.ws, a.M, a.rank);
  const int R = static_cast<int>(a.R);
  const T* b = static_cast<const T*>(a.b);
  if (int rc = lr_pad<T>(a, s, b, st)) return rc;
  if (int rc = lr_shrink<T, true>(p, static_cast<const T*>(a.x), a.ldx, a.K, static_cast<const T*>(a.a), a.rank, 0, R, a.scales, h, st))
    return rc;
  return lr_expand<T, true>(p, h, b, a.rank, lr_ldw(a.rank), R, static_cast<const T*>(a.base), a.ldbase, static_cast<T*>(a.out), a.ldo,
                            a.N, st);
}
template <typename T>
static int lr_backward_t(const LrArgs& a, cudaStream_t st) {
  const LrPlan p = lr_plan(a.plan, a.M, a.R);
  const LrSpace s = lr_space(a.M, a.K, a.N, a.rank, a.R, true);
  const LrHidden h = lr_hidden(a.hidden, a.M, a.rank), dh = lr_hidden(a.ws, a.M, a.rank);
  const int R = static_cast<int>(a.R);
  const T *x = static_cast<const T*>(a.x), *go = static_cast<const T*>(a.go), *b = static_cast<const T*>(a.b);
  if (a.dx || a.da) {
    if (int rc = lr_pad<T>(a, s, b, st)) return rc;
    if (int rc = lr_shrink<T, false>(p, go, a.ldgo, a.N, b, a.rank, lr_ldw(a.rank), R, a.scales, dh, st)) return rc;
  }
  if (a.dx)
    if (int rc = lr_expand<T, false>(p, dh, static_cast<const T*>(a.a), a.rank, 0, R, nullptr, 0, static_cast<T*>(a.dx), a.lddx, a.K, st))
      return rc;
  if (!a.da && !a.db) return H3B_OK;
  char* ws = static_cast<char*>(a.ws);
  const int blocks_k = static_cast<int>((a.K + 127) / 128), blocks_n = static_cast<int>((a.N + 127) / 128);
  const LrWgradSide<T> sa{x, a.ldx, a.K, dh, static_cast<T*>(a.da), reinterpret_cast<float*>(ws + s.part_a), a.da ? blocks_k : 0, true};
  const LrWgradSide<T> sb{go, a.ldgo, a.N, h, static_cast<T*>(a.db), reinterpret_cast<float*>(ws + s.part_b), a.db ? blocks_n : 0, false};
  return lr_rp(a.rank) <= 64 ? lr_wgrad<T, 64>(p, sa, sb, a.rank, R, st) : lr_wgrad<T, 128>(p, sa, sb, a.rank, R, st);
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
