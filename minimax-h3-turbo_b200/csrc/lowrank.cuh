// Low-rank adapters of many requests beside a shared projection, and their gradients.
//
//   out_i = base_i + s_g (x_i A_g^T) B_g^T        g: the adapter of row i; rows without one keep base_i
//   h_i = s_g x_i A_g^T                           [rank], summed in 32 bits; an operand of the second product
//   dh_i = s_g go_i B_g,   dx_i = dh_i A_g,   dA_g = sum_i dh_i^T x_i,   dB_g = sum_i go_i^T h_i
//
// As operands, h and dh are rounded once: to tf32 beside fp16 operands, to bf16 beside bf16 ones (few rows: to tf32).  fp16 itself does
// not hold them: its numbers span 2^40, products of two of them twice that, and rows, ranks and the other operand may each have a size
// of their own, so that no power of two per row or rank keeps a number's digits in every sum that it is part of.  tf32 has fp16's 11
// digits over fp32's range, and every fp16 and bf16 number is one: the products of fp16 operands with h and dh are tf32 products.
// (Operands scaled into fp16 by a power of two per row lost what is 2^-25 of the row's largest number and below, and in the gradients
// of A and B 2^-25 of the largest of all rows that are added up.  They took 301 us for 12090 rows 5120 -> 15360 of rank 128 where tf32
// takes 451, at rank 16 167 and 164; training steps of 12090 rows 5120 -> 5120 269 and 277 at rank 32, 597 and 671 at rank 128.)
// bf16's 8 digits for h are a choice for speed, which results of 8 digits allow: these are 1.9e-3 to 2.3e-3 off in all, their own
// rounding alone being 1.65e-3.  tf32 products come to 1.67e-3, but take 172 us instead of 148 for 12090 rows 5120 -> 15360 of rank 16, 570
// instead of 359 for 59440 rows 5120 -> 5120 of rank 64, and 273 instead of 205 for a training step of 12090 rows 5120 -> 5120 of rank
// 32.  Few rows wait for weights and cost the same either way (64 rows of 64 adapters of rank 64, 5120 -> 15360, 30 us and 33).
//
// The rows are gone through in the plan's order (by adapter, then by row), in tiles of one adapter's rows; rows are gathered by their
// numbers, so a batch may hold its requests in any order.
#pragma once
#include <type_traits>
#include <utility>

#include "cross_common.cuh"

namespace h3b {

template <typename T>
__device__ __forceinline__ T lr_t(float v) {
  if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// ----------------------------------------------------------------------------------------------- plan
// A plan is one int32 array: order [M], the rows by adapter, those without one last; offset [R + 2], where each adapter's rows
// begin in it (group R: rows without one); slot [R + 1], below; then tables of four numbers a line:
//   tiles  (adapter, first place in order, rows, first row if they follow one another, else -1), up to LR_TILE rows each
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
// n rows make at most (n - 1) / rows of a unit + 1 of them
static int64_t lr_unit_lines(int64_t M, int64_t R) { return M / (LR_TILE * lr_unit_tiles(M)) + (R < M ? R : M); }
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
// rows of an adapter are in ascending order: they follow one another where the last is as far from the first as their number says
__device__ __forceinline__ int4 lr_line(const int32_t* order, int who, int from, int n) {
  const int first = order[from], last = order[from + n - 1];
  return make_int4(who, from, n, last - first == n - 1 ? first : -1);
}
// row i of a tile
__device__ __forceinline__ int lr_row(const LrPlan& p, const int4& t, int i) { return t.w >= 0 ? t.w + i : p.order[t.y + i]; }
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
      for (int i = lane; i < nt; i += 32) tiles[t.x + i] = lr_line(p.order, who, from + i * LR_TILE, min(LR_TILE, rows - i * LR_TILE));
      for (int i = lane; i < (rows + LR_FEW - 1) / LR_FEW; i += 32)
        few[t.y + i] = lr_line(p.order, who, from + i * LR_FEW, min(LR_FEW, rows - i * LR_FEW));
      for (int i = lane; i < nu; i += 32) units[t.z + i] = make_int4(who, t.x + i * per, min(per, nt - i * per), nu > 1 ? t.w + i : -1);
    }
    __syncthreads();
  }
  for (int64_t i = base.x + threadIdx.x; i < p.n_tiles; i += LR_PLAN_THREADS) tiles[i] = make_int4(R, 0, 0, -1);
  for (int64_t i = base.y + threadIdx.x; i < p.n_few; i += LR_PLAN_THREADS) few[i] = make_int4(R, 0, 0, -1);
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
// h (or dh) of every row in the plan's order: rows of rp = rank rounded up to 16 numbers, bf16, or tf32 in 32 bits (WIDE)
template <typename T>
constexpr bool LR_WIDE = std::is_same_v<T, __half>;
template <typename T>
using LrHid = std::conditional_t<LR_WIDE<T>, float, T>;
static int lr_rp(int rank) { return (rank + 15) / 16 * 16; }
static size_t lr_up256(size_t v) { return (v + 255) / 256 * 256; }
size_t lr_hidden_bytes(int64_t M, int rank) { return lr_up256(static_cast<size_t>(M) * lr_rp(rank) * 4); }  // of the wider type
__device__ __forceinline__ float lr_tf32(float v) {  // to the nearest; infinities and NaN stay
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
  return __uint_as_float(r);
}
// 8 numbers of a hidden row
template <typename T>
__device__ __forceinline__ void lr_store_hidden(LrHid<T>* to, const float4& u, const float4& v) {
  if constexpr (LR_WIDE<T>) {
    *reinterpret_cast<float4*>(to) = make_float4(lr_tf32(u.x), lr_tf32(u.y), lr_tf32(u.z), lr_tf32(u.w));
    *reinterpret_cast<float4*>(to + 4) = make_float4(lr_tf32(v.x), lr_tf32(v.y), lr_tf32(v.z), lr_tf32(v.w));
  } else {
    *reinterpret_cast<uint4*>(to) = make_uint4(pack2<T>(u.x, u.y), pack2<T>(u.z, u.w), pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
  }
}
// ----------------------------------------------------------------------------------------------- common parts of the tile kernels
// 16 bytes from global to shared memory without passing through registers; zeros where ok is false (nothing is read then)
__device__ __forceinline__ void lr_copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16u : 0u) : "memory");
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

// ----------------------------------------------------------------------------------------------- rows through registers
// The second product has 2 rank flops to a byte of base and out and is HBM-bound, so what counts is how these bytes travel.  They go
// between global memory and the registers of mma.sync directly, 32 bytes to a lane and 128 to a row (four lanes) an instruction.
// Fragments of m16n8k16 would have a lane touch 4 bytes of a row; but which numbers a product calls its n (or its k) is free as long
// as all operands agree, so lane t of a row takes 16 numbers in one piece as the n = 2 t, 2 t + 1 of eight products; the small
// operand W is put in that order in shared memory.  (tcgen05, out by way of tensor memory and shared memory: 220 us for base and out
// of 12090 x 15360 where this takes 115 and their bytes 113.)  The same goes for the products of few rows.
template <typename T>
__device__ __forceinline__ void lr_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// two numbers of each operand's row (k = t, t + 4 of the instruction; which numbers of the sum these are is free, as above): a0, a2 of
// row g, a1, a3 of row g + 8
__device__ __forceinline__ void lr_mma_tf32(float (&d)[4], float a0, float a1, float a2, float a3, float2 b) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(a2)), "r"(__float_as_uint(a3)),
        "r"(__float_as_uint(b.x)), "r"(__float_as_uint(b.y)));
}
// four 8 x 8 matrices of 16-bit numbers, each transposed on the way: lane l gives the address of row l % 8 of matrix l / 8
__device__ __forceinline__ void lr_ldmatrix_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 16 numbers of a row from p on, `left` of them there (a multiple of 8, also negative); wide: rows start on 32-byte boundaries and are
// multiples of 16 long
template <typename T>
__device__ __forceinline__ void lr_load16(const T* p, int64_t left, bool wide, uint32_t (&v)[8]) {
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
    if (left > 8 * i) u = *reinterpret_cast<const uint4*>(p + 8 * i);
    v[4 * i] = u.x, v[4 * i + 1] = u.y, v[4 * i + 2] = u.z, v[4 * i + 3] = u.w;
  }
}
template <typename T>
__device__ __forceinline__ void lr_store16(T* p, int64_t left, bool wide, const uint32_t (&v)[8]) {
  if (wide) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %9, 0;\n\t@p st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n\t}" ::"l"(p),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                 "r"(static_cast<uint32_t>(left >= 16))
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
// 8 numbers of a row of `rank`, from j on, into shared memory; zeros behind the rank and where ok is false.  Rows of ranks that are no
// multiples of 8 do not start on 16-byte boundaries and are read number by number.
template <typename T>
__device__ __forceinline__ void lr_stage8(uint32_t dst, const T* row, int j, int rank, bool ok) {
  if (rank % 8 == 0) {
    lr_copy16(dst, ok && j < rank ? row + j : row, ok && j < rank);
  } else {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = ok && j + 2 * i < rank ? *reinterpret_cast<const uint16_t*>(row + j + 2 * i) : 0u;
      const uint32_t hi = ok && j + 2 * i + 1 < rank ? *reinterpret_cast<const uint16_t*>(row + j + 2 * i + 1) : 0u;
      v[i] = lo | hi << 16;
    }
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
  }
}

// ----------------------------------------------------------------------------------------------- first product: hidden rows
// H [128 rows, rp] of a tile = X [128, C] W, C the contraction: W is A_g [rank, C] (W_ROWS) or B_g [C, rank].  HBM-bound: X is read
// once, 2 rank flops a byte.  The CTAs of a cluster share a tile's C (95 tiles of 12090 rows would leave a third of the SMs idle)
// and add their parts up through distributed shared memory in a fixed order.  Copies are cp.async of 16 bytes, since rows are
// gathered.  Warps 0-3 copy, then read the accumulators; warp 4 issues the products.  12090 x 5120 of rank 16: 30 us, 4.1 TB/s (its
// bytes take 19; the rest is the pipeline's start and the parts' way through the cluster); 59440 x 5120 of rank 64: 124 us, 4.9 TB/s.
// Letting the second product's CTAs in early, to have base on the way at the end of this one, made both slower (together 150 -> 192
// us for 12090 rows 5120 -> 15360).
constexpr int LR_XPART = LR_TILE * 128;  // 64 channels of 128 rows
constexpr int LR_FIRST_THREADS = 160;
template <int RPM, bool W_ROWS>  // the largest rp of this variant: 64 or 128
struct LrFirstCfg {
  // A stage has PB parts of 64 channels: 256 bytes of every row at a time where they fit (59440 rows 5120 -> 5120 of rank 64, both
  // products: 356 us, with 128 bytes 404)
  static constexpr int PB = RPM == 64 ? 2 : 1, STAGES = RPM == 64 ? 2 : 3, CTAS = 2, KC = 64 * PB;
  static constexpr int WPART = W_ROWS ? RPM * 128 : KC * 128;  // of W: [RPM ranks][64 channels], or [KC channels][64 ranks]
  static constexpr int STAGE = PB * LR_XPART + (W_ROWS ? PB : RPM / 64) * WPART;
  static constexpr int SMEM = STAGES * STAGE + 1024;
};
// This CTA's rows of a tile: the parts of the cluster's S CTAs added up in their order, into its own; by warps 0-3
template <int S>
__device__ __forceinline__ void lr_gather(float* red, int ld, int row0, int rp) {
  const int n4 = rp / 4;
#pragma unroll 2
  for (int e = threadIdx.x; e < LR_TILE / S * n4; e += 128) {
    const int r = e / n4;
    float* const own = red + (row0 + r) * ld + (e - r * n4) * 4;
    const uint32_t at = smem_u32(own);
    float4 v[S];
#pragma unroll
    for (int k = 0; k < S; ++k)
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(v[k].x), "=f"(v[k].y), "=f"(v[k].z), "=f"(v[k].w) : "r"(mapa_rank(at, k)) : "memory");
    float4 sum = v[0];
#pragma unroll
    for (int k = 1; k < S; ++k) sum.x += v[k].x, sum.y += v[k].y, sum.z += v[k].z, sum.w += v[k].w;
    *reinterpret_cast<float4*>(own) = sum;  // read by this thread alone
  }
}

template <typename T, bool W_ROWS, int RPM>
__global__ void __launch_bounds__(LR_FIRST_THREADS) lr_first_kernel(const LrPlan p, const T* x, int64_t ldx, int64_t C,
                                                                      const T* w, int rank, int rp, int R, const float* scales, LrHid<T>* out,
                                                                      int splits) {
  using Cfg = LrFirstCfg<RPM, W_ROWS>;
  constexpr int STAGES = Cfg::STAGES, PB = Cfg::PB, KC = Cfg::KC;
  extern __shared__ __align__(1024) unsigned char lr_smem[];
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
  const int chunks = static_cast<int>((C + KC - 1) / KC), per = (chunks + splits - 1) / splits;
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
      const uint32_t xs = smem_u32(base + s * Cfg::STAGE), ws = xs + PB * LR_XPART;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 4 * PB; ++kk)
          mma_f16_ss(tmem, desc_rows(xs) + rows_step(kk),
                     W_ROWS ? desc_rows(ws + kk / 4 * Cfg::WPART) + kk % 4 * 2 : lr_desc_mn(ws, Cfg::WPART) + kk * 128, idesc, i > 0 || kk > 0);
      }
      __syncwarp();
      commit_one(&empty[s]);
    }
    commit_one(&done);
  } else {
    // 8 PB lanes have a row's 128 PB bytes; rows r0, r0 + RS, ...
    constexpr int LANES = 8 * PB, RS = 128 / LANES, NR = LR_TILE / RS;
    const int r0 = tid / LANES, ch = tid % LANES, part = ch >> 3, c8 = ch & 7;
    int row[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) row[i] = r0 + RS * i < t.z ? lr_row(p, t, r0 + RS * i) : -1;
    const T* wg = w + static_cast<int64_t>(t.x) * rank * C;
    const uint32_t at = static_cast<uint32_t>(r0 * 128 + ((c8 ^ (r0 & 7)) << 4));  // RS is 16 or 8: the same chunk in all rows
    const T* const xc = x + ch * 8;
    for (int i = 0; i < n + STAGES - 1; ++i) {
      if (i < n) {
        const int s = i % STAGES;
        mbar_wait(&empty[s], ((i / STAGES) & 1) ^ 1, abort);
        const uint32_t xs = smem_u32(base + s * Cfg::STAGE), ws = xs + PB * LR_XPART;
        const int64_t c = static_cast<int64_t>(c0 + i) * KC;
        const bool in = c + ch * 8 < C;
#pragma unroll
        for (int j = 0; j < NR; ++j) {
          const bool ok = row[j] >= 0 && in;
          lr_copy16(xs + part * LR_XPART + at + j * RS * 128, ok ? xc + row[j] * ldx + c : x, ok);
        }
        if constexpr (W_ROWS) {
#pragma unroll
          for (int j = 0; j < RPM / RS; ++j) {
            const int r = r0 + RS * j;
            if (RS * j < rp) lr_copy16(ws + part * Cfg::WPART + at + j * RS * 128, r < rank && in ? wg + r * C + c + ch * 8 : w, r < rank && in);
          }
        } else {
          const int k0 = tid >> 3, k8 = tid & 7;  // 16 channels at a time, eight lanes to 64 ranks of one
          const uint32_t wat = ws + k0 * 128 + ((k8 ^ (k0 & 7)) << 4);
#pragma unroll
          for (int q = 0; q < RPM / 64; ++q) {
            const int k = q * 64 + k8 * 8;
            if (k < rp) {
#pragma unroll
              for (int j = 0; j < KC / 16; ++j) {
                const int64_t r = c + k0 + 16 * j;
                lr_stage8(wat + q * Cfg::WPART + j * 2048, r < C ? wg + r * rank : w, k, rank, r < C);
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
      if (c + 16 > rank) {  // an infinity in X times a rank that is not there: NaN, which would reach every sum over the row
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = c + i < rank ? v[i] : 0u;
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
    const int rows = LR_TILE / splits, row0 = split * rows;  // this CTA's share of the tile's rows
    if (splits == 2) lr_gather<2>(red, ld, row0, rp);
    if (splits == 4) lr_gather<4>(red, ld, row0, rp);
    if (splits == 8) lr_gather<8>(red, ld, row0, rp);
    group_sync(1, 128);
    const int lanes = rp / 8;  // 8 numbers to a lane
    for (int e = tid; e < rows * lanes; e += 128) {
      const int r = e / lanes, c = (e - r * lanes) * 8, row = row0 + r;
      if (row >= t.z) break;
      const float* from = red + row * ld + c;
      const float4 u = *reinterpret_cast<const float4*>(from), v = *reinterpret_cast<const float4*>(from + 4);
      lr_store_hidden<T>(out + static_cast<int64_t>(t.y + row) * rp + c, make_float4(u.x * scale, u.y * scale, u.z * scale, u.w * scale),
                         make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale));
    }
  }
  if (splits > 1) cluster_sync();  // the others have read this CTA's part
}

// ----------------------------------------------------------------------------------------------- second product: out or dx
// out [128 rows, N] of a tile = base + H W^T: W is B_g [N, rank] (W_ROWS) or A_g [rank, N].  A CTA has 64 CB columns of a tile, a warp 16
// rows of them: all of its base is asked for at once, then W goes to shared memory, then the products are added and stored.
//   block of 64 columns: lane t has columns 16 t .. 16 t + 15; 2 j, 2 j + 1 of these are product j's n = 2 t, 2 t + 1
// Ranks are filled up with zeros to 16 NQ: leaving products out by the rank cost 13 instructions to a product.  12090 x 15360 of
// rank 16 with base: 115 us, 6.5 TB/s; 59440 x 5120 of rank 64: 241 us, 5.1 TB/s; dx of 12090 x 5120, rank 32: 26 us, its bytes 19.
// WIDE products take twice the tensor cores' time and H's fragments come from L1: 59440 x 5120 of rank 64 410 us, dx 43 us.
constexpr int LR_THREADS = 256;
template <int NQ, bool W_ROWS, bool BASE, bool WIDE>  // 16 NQ: the largest rp of this variant
struct LrSecondCfg {
  // Columns of a CTA: 128 with base, whose numbers wait in registers.  256 where that does not count (no base), or counts less than what W
  // and H take of L2 (ranks from 33 on: 59440 rows 5120 -> 5120 of rank 64 in all 411 us, with 128 columns 430).  WIDE with base: 256,
  // and two CTAs to an SM instead of three, up to rank 64 (12090 rows 5120 -> 15360 of rank 16 164 us, with 128 and three 172; 59440 of
  // rank 64 522 and 528), then 128 and three (12090 rows of rank 128 451 us, with 256 and two 488)
  static constexpr int CB = !BASE ? 4 : WIDE ? (NQ <= 4 ? 4 : 2) : NQ <= 2 ? 2 : 4, COLS = 64 * CB;
  // rows of W: [COLS][16 NQ], 32 bytes apart from a multiple of 64; or [16 NQ][COLS], 16 from a multiple of 128: no bank conflicts
  static constexpr int LDW = W_ROWS ? (32 * NQ + 31) / 64 * 64 + 32 : 2 * COLS + 16;
  static constexpr int SMEM = LDW * (W_ROWS ? COLS : 16 * NQ);
  static constexpr int CTAS = !BASE ? (NQ <= 4 ? 3 : 2) : WIDE ? (NQ <= 4 ? 2 : 3) : NQ <= 2 ? 3 : 2;
};
template <typename T, bool W_ROWS, bool BASE, int NQ>
__global__ void __launch_bounds__(LR_THREADS, LrSecondCfg<NQ, W_ROWS, BASE, LR_WIDE<T>>::CTAS)
    lr_second_kernel(const LrPlan p, const LrHid<T>* hid, const T* w, int rank, int rp, int R, const T* base, int64_t ldb, T* out,
                     int64_t ldo, int64_t N, int parts, bool wide) {
  using Cfg = LrSecondCfg<NQ, W_ROWS, BASE, LR_WIDE<T>>;
  constexpr int CB = Cfg::CB, COLS = Cfg::COLS, LDW = Cfg::LDW;
  constexpr bool WIDE = LR_WIDE<T>;
  extern __shared__ __align__(1024) unsigned char lr_smem[];
  after_previous();
  const int tile = blockIdx.x / parts;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x - tile * parts) * COLS;
  const int4 t = p.tiles[tile];
  if (t.z == 0 || (t.x >= R && base == out)) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
  const int r0 = 16 * warp + g;
  const int64_t c = c0 + 16 * q4;
  int row[2];  // on their way while the small operands are asked for
#pragma unroll
  for (int h = 0; h < 2; ++h) row[h] = r0 + 8 * h < t.z ? lr_row(p, t, r0 + 8 * h) : -1;
  uint32_t v[BASE ? CB : 1][2][8];
  auto ask = [&] {
    if constexpr (BASE) {
#pragma unroll
      for (int b = 0; b < CB; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) lr_load16(base + row[h] * ldb + c + 64 * b, row[h] >= 0 ? N - c - 64 * b : 0, wide, v[b][h]);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[0][h][j] = 0u;
    }
  };
  if (t.x >= R) {  // rows without an adapter
    ask();
#pragma unroll
    for (int b = 0; b < CB; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h) lr_store16(out + row[h] * ldo + c + 64 * b, row[h] >= 0 ? N - c - 64 * b : 0, wide, v[BASE ? b : 0][h]);
    return;
  }
  const uint32_t sm = smem_u32(lr_smem);
  const T* wg = w + static_cast<int64_t>(t.x) * rank * N;
  if constexpr (W_ROWS) {
    // column 16 a + 2 j + i of a block of 64 lies at 8 j + 2 a + i: the eight columns of a product in a piece
#pragma unroll
    for (int e = tid; e < COLS * 2 * NQ; e += LR_THREADS) {
      const int n = e / (2 * NQ), j = e % (2 * NQ) * 8, b = n & 63;
      const int at = (n & ~63) + (b >> 1 & 7) * 8 + (b >> 4) * 2 + (b & 1);
      const bool ok = c0 + n < N;
      lr_stage8(sm + at * LDW + 2 * j, ok ? wg + (c0 + n) * rank : w, j, rank, ok);
    }
    lr_copy_commit();
  } else {
    // the same order of columns; pairs of columns stay together
#pragma unroll
    for (int e = tid; e < 16 * NQ * (COLS / 8); e += LR_THREADS) {
      const int r = e / (COLS / 8), n = e % (COLS / 8) * 8, b = n & 63;
      uint4 u = make_uint4(0, 0, 0, 0);
      if (r < rank && c0 + n < N) u = *reinterpret_cast<const uint4*>(wg + r * N + c0 + n);
      const uint32_t to = sm + r * LDW + 2 * ((n & ~63) + (b >> 1 & 7) * 8 + (b >> 4) * 2);
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(to), "r"(u.x) : "memory");
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + 16), "r"(u.y) : "memory");
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + 32), "r"(u.z) : "memory");
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + 48), "r"(u.w) : "memory");
    }
  }
  // H: this lane's k are 4 t .. 4 t + 3 of every 16 (W_ROWS), or 2 t, 2 t + 1, 2 t + 8, 2 t + 9.  Beside fp16 they take twice the
  // registers and come from L1 at their product instead.
  const LrHid<T>* hr[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) hr[h] = hid + static_cast<int64_t>(t.y + min(r0 + 8 * h, t.z - 1)) * rp + (W_ROWS ? 4 : 2) * q4;
  uint32_t a[NQ][4];
  if constexpr (!WIDE) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        uint2 u = make_uint2(0, 0);
        if (16 * q < rp) {
          if constexpr (W_ROWS) u = *reinterpret_cast<const uint2*>(hr[h] + 16 * q);
          else u = make_uint2(*reinterpret_cast<const uint32_t*>(hr[h] + 16 * q), *reinterpret_cast<const uint32_t*>(hr[h] + 16 * q + 8));
        }
        a[q][h] = u.x, a[q][2 + h] = u.y;
      }
  }
  ask();
  lr_copy_wait<0>();
  __syncthreads();
#pragma unroll
  for (int b = 0; b < CB; ++b) {
    float d[8][4];  // the sums begin with base
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 f = BASE ? lr_unpack2<T>(v[BASE ? b : 0][h][j]) : make_float2(0.f, 0.f);
        d[j][2 * h] = f.x, d[j][2 * h + 1] = f.y;
      }
    if constexpr (WIDE) {
      constexpr int AT_ONCE = NQ <= 4 ? 4 : 2;
#pragma unroll AT_ONCE
      for (int q = 0; q < NQ; ++q) {
        if (16 * q >= rp) break;
        float4 f[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (W_ROWS) {
            f[h] = *reinterpret_cast<const float4*>(hr[h] + 16 * q);
          } else {
            const float2 lo = *reinterpret_cast<const float2*>(hr[h] + 16 * q), hi = *reinterpret_cast<const float2*>(hr[h] + 16 * q + 8);
            f[h] = make_float4(lo.x, lo.y, hi.x, hi.y);
          }
        }
        auto product = [&](float (&to)[4], uint32_t w0, uint32_t w1) {
          lr_mma_tf32(to, f[0].x, f[1].x, f[0].y, f[1].y, lr_unpack2<T>(w0));
          lr_mma_tf32(to, f[0].z, f[1].z, f[0].w, f[1].w, lr_unpack2<T>(w1));
        };
        if constexpr (W_ROWS) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint2 u = *reinterpret_cast<const uint2*>(lr_smem + (64 * b + 8 * j + g) * LDW + 32 * q + 8 * q4);
            product(d[j], u.x, u.y);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            uint32_t m[4];
            lr_ldmatrix_t(m, sm + (16 * q + (lane & 15)) * LDW + 2 * (64 * b + 8 * j) + (lane >> 4) * 16);
            product(d[j], m[0], m[1]);
            product(d[j + 1], m[2], m[3]);
          }
        }
      }
    } else if constexpr (W_ROWS) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const uint2 u = *reinterpret_cast<const uint2*>(lr_smem + (64 * b + 8 * j + g) * LDW + 32 * q + 8 * q4);
          lr_mma<T>(d[j], a[q][0], a[q][1], a[q][2], a[q][3], u.x, u.y);
        }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j += 2)
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          uint32_t m[4];
          lr_ldmatrix_t(m, sm + (16 * q + (lane & 15)) * LDW + 2 * (64 * b + 8 * j) + (lane >> 4) * 16);
          lr_mma<T>(d[j], a[q][0], a[q][1], a[q][2], a[q][3], m[0], m[1]);
          lr_mma<T>(d[j + 1], a[q][0], a[q][1], a[q][2], a[q][3], m[2], m[3]);
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t res[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) res[j] = pack2<T>(d[j][2 * h], d[j][2 * h + 1]);
      lr_store16(out + row[h] * ldo + c + 64 * b, row[h] >= 0 ? N - c - 64 * b : 0, wide, res);
    }
  }
}

// ----------------------------------------------------------------------------------------------- few rows
// Up to eight rows of one adapter, as single tokens of many requests have them: everything is the adapters' weights, read once, and
// latency.  Weights go from memory straight to fragments; K is dealt out to `splits` CTAs of a tile, whose parts the second kernel adds
// up in a fixed order (4 rows of rank 16, 5120 -> 5120: 4.3 us; 64 rows of 49 adapters of rank 64, 5120 -> 15360: 30 us, 4.3 TB/s of the
// weights in use, base and out).  The second kernel is let in when every CTA of the first has begun, and asks for its weights and base
// before it waits for the parts: the two products' weights come in one stream.  (A cluster of eight CTAs for both products, its parts
// in distributed shared memory: 16.2 us for one row of rank 64, 91 us for 64 rows of 64 adapters 5120 -> 15360.)
//   32 columns (ranks) of a row: lane t has 8 t .. 8 t + 7, which are k = 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of two products
constexpr int LR_FEW_THREADS = 128;
__device__ __forceinline__ void lr_let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void lr_prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
template <typename T>
__device__ __forceinline__ uint4 lr_row8(const T* row, int64_t j, int64_t n, bool aligned) {  // numbers j .. j + 7 of n, zeros behind
  uint4 v = make_uint4(0, 0, 0, 0);
  if (aligned) {
    if (j < n) v = *reinterpret_cast<const uint4*>(row + j);
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (j + i < n) w[i / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(row + j + i)) << (16 * (i & 1));
  }
  return v;
}
// part[tile][split][row of 8][rp] = x A_g^T over the split's columns: 16 ranks x 8 rows a product
template <typename T, int RB>  // 16 RB: the largest rp of this variant
__global__ void __launch_bounds__(LR_FEW_THREADS) lr_few_down_kernel(const LrPlan p, const T* x, int64_t ldx, int64_t K, const T* a, int rank,
                                                                     int rp, int R, int splits, float* part) {
  constexpr int W = LR_FEW_THREADS / 32;
  __shared__ float red[W][8][16 * RB + 4];
  after_previous();
  lr_let_next();
  const int tile = blockIdx.x / splits, split = blockIdx.x - tile * splits;
  const int4 t = p.few[tile];
  if (t.z == 0 || t.x >= R) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
  const int row = g < t.z ? lr_row(p, t, g) : -1;  // this lane's row
  const T* ag = a + static_cast<int64_t>(t.x) * rank * K;
  float acc[RB][4];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  const int blocks = static_cast<int>((K + 31) / 32), b0 = split * blocks / splits, b1 = (split + 1) * blocks / splits;
#pragma unroll 2
  for (int i = b0 + warp; i < b1; i += W) {
    const int64_t k = i * 32 + 8 * q4;
    const uint4 xv = lr_row8(x + row * ldx, k, row >= 0 ? K : 0, true);
    uint4 w[RB][2];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = 16 * r + 8 * h + g;
        w[r][h] = lr_row8(ag + j * K, k, j < rank ? K : 0, true);
      }
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      lr_mma<T>(acc[r], w[r][0].x, w[r][1].x, w[r][0].y, w[r][1].y, xv.x, xv.y);
      lr_mma<T>(acc[r], w[r][0].z, w[r][1].z, w[r][0].w, w[r][1].w, xv.z, xv.w);
    }
  }
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[warp][2 * q4 + (e & 1)][16 * r + g + 8 * (e >> 1)] = acc[r][e];
  __syncthreads();
  float* to = part + static_cast<int64_t>(blockIdx.x) * 8 * rp;
  for (int e = tid; e < t.z * rp; e += LR_FEW_THREADS) {
    const int m = e / rp, j = e - m * rp;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) sum += red[w][m][j];
    to[e] = sum;
  }
}
// out [rows, 64 columns of a warp]: lane t has columns 16 t .. 16 t + 15, of which 2 j, 2 j + 1 are product j's n = 2 t, 2 t + 1
template <typename T, int RB>
__global__ void __launch_bounds__(LR_FEW_THREADS) lr_few_up_kernel(const LrPlan p, const T* b, int rank, int rp, int R, const float* scales,
                                                                   const T* base, int64_t ldb, T* out, int64_t ldo, int64_t N, int columns,
                                                                   bool wide, const float* part, int splits, LrHid<T>* hid, bool keep) {
  constexpr int KB = (RB + 1) / 2, AT_ONCE = KB > 2 ? 4 : 8;  // blocks of 32 ranks; products whose weights are held
  __shared__ __align__(16) float hs[8][32 * KB + 8];
  const int tile = blockIdx.x / columns, at = blockIdx.x - tile * columns;
  const int4 t = p.few[tile];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
  if (t.z == 0 || (t.x >= R && base == out)) {
    after_previous();
    return;
  }
  const int row = g < t.z ? lr_row(p, t, g) : -1;  // this lane's row
  const int64_t c0 = (static_cast<int64_t>(at) * (LR_FEW_THREADS / 32) + warp) * 64, c = c0 + 16 * q4, n0 = c0 + 16 * (g >> 1) + (g & 1);
  uint32_t v[8];
  lr_load16(base + row * ldb + c, base && row >= 0 ? N - c : 0, wide, v);
  if (t.x >= R) {  // rows without an adapter
    after_previous();
    lr_store16(out + row * ldo + c, row >= 0 ? N - c : 0, wide, v);
    return;
  }
  const T* bg = b + static_cast<int64_t>(t.x) * rank * N;
  const bool aligned = rank % 8 == 0;
  uint4 w[AT_ONCE][KB];
  auto weights = [&](int j0) {
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        const int64_t n = n0 + 2 * (j0 + j);
        w[j][k] = lr_row8(bg + n * rank, 32 * k + 8 * q4, n < N ? rank : 0, aligned);
      }
  };
  weights(0);
  if (AT_ONCE < 8) {
#pragma unroll
    for (int j = AT_ONCE; j < 8; ++j)
      if (n0 + 2 * j < N && q4 * 64 < rank) lr_prefetch(bg + (n0 + 2 * j) * rank + q4 * 64);
  }
  after_previous();
  // ---- h: the splits' parts added up, in tf32 for this product; zeros for rows and ranks that are not there
  const float scale = scales ? scales[t.x] : 1.f;
  const bool first = keep && at == 0;
  for (int e = tid; e < 8 * 32 * KB; e += LR_FEW_THREADS) {
    const int m = e / (32 * KB), j = e % (32 * KB);
    float sum = 0.f;
    if (m < t.z && j < rank) {
      const float* from = part + static_cast<int64_t>(tile) * splits * 8 * rp + m * rp + j;
#pragma unroll 8
      for (int s = 0; s < splits; ++s) sum += from[static_cast<int64_t>(s) * 8 * rp];
    }
    const float u = lr_tf32(sum * scale);
    hs[m][j] = u;
    if (first && m < t.z && j < rp) {
      LrHid<T>* const to = hid + static_cast<int64_t>(t.y + m) * rp + j;
      if constexpr (LR_WIDE<T>) *to = u;
      else *to = lr_t<T>(sum * scale);
    }
  }
  __syncthreads();
#pragma unroll
  for (int j0 = 0; j0 < 8; j0 += AT_ONCE) {
    if (j0 > 0) weights(j0);
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        const float4* const hk = reinterpret_cast<const float4*>(&hs[g][32 * k + 8 * q4]);
        const float4 lo = hk[0], hi = hk[1];
        lr_mma_tf32(d, lo.x, 0.f, lo.y, 0.f, lr_unpack2<T>(w[j][k].x));
        lr_mma_tf32(d, lo.z, 0.f, lo.w, 0.f, lr_unpack2<T>(w[j][k].y));
        lr_mma_tf32(d, hi.x, 0.f, hi.y, 0.f, lr_unpack2<T>(w[j][k].z));
        lr_mma_tf32(d, hi.z, 0.f, hi.w, 0.f, lr_unpack2<T>(w[j][k].w));
      }
      const float2 f = lr_unpack2<T>(v[j0 + j]);
      v[j0 + j] = pack2<T>(d[0] + f.x, d[1] + f.y);
    }
  }
  lr_store16(out + row * ldo + c, row >= 0 ? N - c : 0, wide, v);
}

// ----------------------------------------------------------------------------------------------- weight gradients
// D [128 channels, rp] = X^T H over the rows of a unit (a stretch of one adapter's rows): X's columns are M, H's are N, rows are K,
// all read as they lie in memory.  HBM-bound: X is read once; H comes from L2.  Rows behind the last are zeros in both operands.  One
// launch does dA (x with dh) and dB (grad_out with h).
// bf16: warps 0-3 copy, then read the accumulators; warp 4 issues the products.  12090 rows of 5120 and 5120, rank 32: 58 us, 4.3 TB/s (5.0
// by itself; in a training step dx's way out of L2 is in it), and 7 to 11 us for the sum of the units' parts.  Fewer, longer units
// took longer (two of these 16 in one CTA 58, four 60, eight 74).
constexpr int LR_KROWS = 64;  // rows of a stage
// ST stages: three, or one where the adapters have no more rows than that on average, so that more CTAs fit an SM (training steps 5120
// -> 5120: 512 rows of 64 adapters, rank 64, 171 us, with three 180; 61 rows of 24, rank 128, 102, with three 116)
template <int RPM, int ST>
struct LrWgradCfg {
  static constexpr int PARTS = RPM / 64;
  static constexpr int XBYTES = 2 * LR_KROWS * 128, STAGE = XBYTES + PARTS * LR_KROWS * 128, OUT = 128 * (RPM + 8) * 2 + 1024;
  static constexpr int SMEM = (ST * STAGE > OUT ? ST * STAGE : OUT) + 1024;
};
template <typename T>
struct LrWgradSide {
  const T* x;
  int64_t ldx, C;
  const LrHid<T>* hid;
  T* grad;       // [rank][C] (by_rank) or [C][rank] of every adapter
  float* part;   // [slots][C][rp]
  int blocks;    // of 128 channels
  bool by_rank;
};
// Where a CTA of the weight gradients works: its unit's rows (places in order), its side and its first channel
template <typename T>
struct LrWgradPart {
  const LrWgradSide<T>* sd;
  int64_t col;
  int adapter, slot, p0, rows;
  __device__ LrWgradPart(const LrPlan& p, const LrWgradSide<T>& sa, const LrWgradSide<T>& sb, int R) {
    const int both = sa.blocks + sb.blocks, unit = blockIdx.x / both, block = blockIdx.x - unit * both;
    const int4 u = p.units[unit];
    const bool second = block >= sa.blocks;
    sd = second ? &sb : &sa, col = static_cast<int64_t>(second ? block - sa.blocks : block) * 128;
    adapter = u.x, slot = u.w, p0 = rows = 0;
    if (u.z == 0 || u.x >= R) return;  // no rows
    const int4 first = p.tiles[u.y], last = p.tiles[u.y + u.z - 1];
    p0 = first.y, rows = last.y + last.z - p0;
  }
};
// A whole gradient of 128 channels from shared memory (`out`: [rank][136] by rank, else [128][rank + 8])
// to memory, 16 bytes at a time in the order of memory, by 128 threads.  Lanes that wrote their channel's ranks one by one took 223 us
// for 24 adapters of rank 128 beside 1112 -> 7680.
__device__ __forceinline__ int lr_grad_ld(bool by_rank, int rank) { return by_rank ? 136 : rank + 8; }
template <typename T>
__device__ __forceinline__ void lr_put_gradient(const LrWgradPart<T>& w, const T* out, int rank) {
  const LrWgradSide<T>& sd = *w.sd;
  const int tid = threadIdx.x, ld = lr_grad_ld(sd.by_rank, rank);
  T* const g = sd.grad + static_cast<int64_t>(w.adapter) * rank * sd.C + w.col * (sd.by_rank ? 1 : rank);
  if (sd.by_rank) {
    for (int e = tid; e < rank * 16; e += 128) {
      const int j = e >> 4, i = (e & 15) * 8;
      if (w.col + i < sd.C) *reinterpret_cast<uint4*>(g + j * sd.C + i) = *reinterpret_cast<const uint4*>(out + j * ld + i);
    }
  } else {
    const bool eights = rank % 8 == 0;
    const int total = static_cast<int>(min(static_cast<int64_t>(128), sd.C - w.col)) * rank;
    for (int i = tid * 8; i < total; i += 128 * 8) {
      const int r = i / rank, k = i - r * rank;
      if (eights) {
        *reinterpret_cast<uint4*>(g + i) = *reinterpret_cast<const uint4*>(out + r * ld + k);
      } else {
        uint4 u;
        T* const e = reinterpret_cast<T*>(&u);
        for (int q = 0, rr = r, kk = k; q < 8; ++q) {
          e[q] = out[rr * ld + kk];
          if (++kk == rank) kk = 0, ++rr;
        }
        *reinterpret_cast<uint4*>(g + i) = u;
      }
    }
  }
}
template <typename T, int RPM, int ST>
__global__ void __launch_bounds__(160) lr_wgrad_kernel(const LrPlan p, const LrWgradSide<T> sa, const LrWgradSide<T> sb, int rank, int rp,
                                                       int R) {
  using Cfg = LrWgradCfg<RPM, ST>;
  extern __shared__ __align__(1024) unsigned char lr_smem[];
  __shared__ uint64_t full[ST], empty[ST], done;
  __shared__ uint32_t tmem_at;
  __shared__ int abort_flag;
  after_previous();
  const LrWgradPart<T> w(p, sa, sb, R);
  if (w.rows == 0) return;
  const LrWgradSide<T>& sd = *w.sd;
  const int64_t col = w.col;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, p0 = w.p0, rows = w.rows, n = (rows + LR_KROWS - 1) / LR_KROWS;
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
    const int r0 = tid >> 3, ch = tid & 7;
    const uint32_t at = static_cast<uint32_t>(r0 * 128 + ((ch ^ (r0 & 7)) << 4));
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
              lr_copy16(to, r < rows ? sd.hid + static_cast<int64_t>(p0 + r) * rp + k : sd.hid, r < rows);
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
    // a channel per lane; a whole gradient by way of shared memory (every product has read the stages)
    const int64_t c = col + tid;
    const int ld = lr_grad_ld(sd.by_rank, rank);
    T* const out = reinterpret_cast<T*>(base);
    for (int j = 0; j < rp; j += 16) {
      uint32_t v[16];
      tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + j, v);
      tmem_ld_wait();
      if (w.slot >= 0) {
        if (c < sd.C) store_cols_f32(sd.part + (w.slot * sd.C + c) * rp + j, v, 1.f, 16);
      } else if (!sd.by_rank && rank % 8 == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) o[k] = pack2<T>(__uint_as_float(v[8 * h + 2 * k]), __uint_as_float(v[8 * h + 2 * k + 1]));
          if (j + 8 * h < rank) *reinterpret_cast<uint4*>(out + tid * ld + j + 8 * h) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (j + k < rank) out[sd.by_rank ? (j + k) * ld + tid : tid * ld + j + k] = lr_t<T>(__uint_as_float(v[k]));
      }
      __syncwarp();
    }
    if (w.slot < 0) {
      group_sync(1, 128);
      lr_put_gradient(w, out, rank);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, lr_tmem_cols(rp));
  }
}
// fp16: H is tf32, which tcgen05 takes with the contraction contiguous alone; X and H lie the other way.  So the products are those of
// mma.sync: a warp has 32 channels, ldmatrix turns X on the way to the fragments, its numbers become tf32 there (they all are), and a
// lane takes two neighbouring ranks as the n of two products.  Rows in stages of 32, three of them, or one where the adapters have no
// more rows than that on average.  12090 rows of 5120 and 5120, rank 32: 103 us (tcgen05 with bf16 operands 49, their bytes 38), by 16
// warps to an SM that take turns at copies, conversions and products; training steps of 512 rows of 64 adapters, rank 64, 5120 -> 5120
// take 153 us, bf16 144.
constexpr int LR_WROWS = 32;
template <int RPM, int ST>
struct LrWgradWideCfg {
  static constexpr int LDX = 136 * 2;  // bytes of a row of X: 16 from a multiple of 128, no bank conflicts
  static constexpr int XBYTES = LR_WROWS * LDX, STAGE = XBYTES + LR_WROWS * (RPM + 4) * 4, OUT = 128 * (RPM + 8) * 2 + 1024;
  static constexpr int SMEM = ST * STAGE > OUT ? ST * STAGE : OUT;
  static constexpr int CTAS = RPM == 64 ? 4 : 3;
};
template <typename T, int RPM, int ST>
__global__ void __launch_bounds__(128, LrWgradWideCfg<RPM, ST>::CTAS)
    lr_wgrad_wide_kernel(const LrPlan p, const LrWgradSide<T> sa, const LrWgradSide<T> sb, int rank, int rp, int R) {
  using Cfg = LrWgradWideCfg<RPM, ST>;
  extern __shared__ __align__(1024) unsigned char lr_smem[];
  after_previous();
  const LrWgradPart<T> w(p, sa, sb, R);
  if (w.rows == 0) return;
  const LrWgradSide<T>& sd = *w.sd;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
  const int rows = w.rows, n = (rows + LR_WROWS - 1) / LR_WROWS, ldh = rp + 4;  // numbers of a row of H: its reads touch every bank once
  const uint32_t sm = smem_u32(lr_smem);
  float acc[2][RPM / 16][2][4];  // [16 channels][16 ranks][product]
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int b = 0; b < RPM / 16; ++b)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[m][b][e / 4][e % 4] = 0.f;
  const int r0 = tid >> 4, ch = (tid & 15) * 8;  // 16 lanes have a row's 256 bytes; rows r0, r0 + 8, ...
  const bool in = w.col + ch < sd.C;
  int next[4];
  auto numbers = [&](int i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = i * LR_WROWS + r0 + 8 * j;
      next[j] = r < rows ? p.order[w.p0 + r] : -1;
    }
  };
  auto bring = [&](int i) {  // stage i, and the numbers of the next one's rows
    if (i < n) {
      const uint32_t xs = sm + i % ST * Cfg::STAGE, hs = xs + Cfg::XBYTES;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool ok = next[j] >= 0 && in;
        lr_copy16(xs + (r0 + 8 * j) * Cfg::LDX + ch * 2, ok ? sd.x + next[j] * sd.ldx + w.col + ch : sd.x, ok);
      }
      const int fours = rp / 4;
      for (int e = tid; e < LR_WROWS * fours; e += 128) {
        const int r = e / fours, k = (e - r * fours) * 4, at = i * LR_WROWS + r;
        lr_copy16(hs + (r * ldh + k) * 4, at < rows ? sd.hid + static_cast<int64_t>(w.p0 + at) * rp + k : sd.hid, at < rows);
      }
      if (i + 1 < n) numbers(i + 1);
    }
    lr_copy_commit();
  };
  numbers(0);
  for (int i = 0; i < ST - 1; ++i) bring(i);
  for (int i = 0; i < n; ++i) {
    if (ST == 1) bring(i);
    lr_copy_wait<ST == 1 ? 0 : ST - 2>();
    __syncthreads();  // stage i is there, and everyone is through with the one before
    if (ST > 1) bring(i + ST - 1);
    const uint32_t xs = sm + i % ST * Cfg::STAGE + (warp * 32) * 2;
    const float* hs = reinterpret_cast<const float*>(lr_smem + i % ST * Cfg::STAGE + Cfg::XBYTES);
#pragma unroll
    for (int k = 0; k < LR_WROWS; k += 16) {
      if (i * LR_WROWS + k >= rows) break;
      float2 a[2][4];  // rows 2 t, 2 t + 1 of channel g; of g + 8; rows 2 t + 8, 2 t + 9 of both
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        uint32_t u[4];
        lr_ldmatrix_t(u, xs + (k + (lane >> 4) * 8 + (lane & 7)) * Cfg::LDX + (16 * m + (lane >> 3 & 1) * 8) * 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[m][e] = lr_unpack2<T>(u[e]);
      }
      const float* const h = hs + (k + 2 * q4) * ldh + 2 * g;
#pragma unroll
      for (int b = 0; b < RPM / 16; ++b) {
        if (16 * b >= rp) break;
        auto ranks = [&](int row) { return *reinterpret_cast<const float2*>(h + row * ldh + 16 * b); };
        const float2 h0 = ranks(0), h1 = ranks(1), h8 = ranks(8), h9 = ranks(9);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          lr_mma_tf32(acc[m][b][0], a[m][0].x, a[m][1].x, a[m][0].y, a[m][1].y, make_float2(h0.x, h1.x));
          lr_mma_tf32(acc[m][b][1], a[m][0].x, a[m][1].x, a[m][0].y, a[m][1].y, make_float2(h0.y, h1.y));
          lr_mma_tf32(acc[m][b][0], a[m][2].x, a[m][3].x, a[m][2].y, a[m][3].y, make_float2(h8.x, h9.x));
          lr_mma_tf32(acc[m][b][1], a[m][2].x, a[m][3].x, a[m][2].y, a[m][3].y, make_float2(h8.y, h9.y));
        }
      }
    }
    if (ST == 1) __syncthreads();
  }
  lr_copy_wait<0>();
  __syncthreads();
  // a lane has ranks 16 b + 4 t .. + 3 of channels g and g + 8: product 0 the even ones, 1 the odd ones
  T* const out = reinterpret_cast<T*>(lr_smem);
  const int ld = lr_grad_ld(sd.by_rank, rank);
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int b = 0; b < RPM / 16; ++b)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const float v[4] = {acc[m][b][0][2 * s], acc[m][b][1][2 * s], acc[m][b][0][2 * s + 1], acc[m][b][1][2 * s + 1]};
        const int c = warp * 32 + 16 * m + 8 * s + g, j = 16 * b + 4 * q4;
        if (w.slot >= 0) {
          if (j < rp && w.col + c < sd.C)
            *reinterpret_cast<float4*>(sd.part + (w.slot * sd.C + w.col + c) * rp + j) = make_float4(v[0], v[1], v[2], v[3]);
        } else if (!sd.by_rank && rank % 8 == 0) {
          if (j < rank) *reinterpret_cast<uint2*>(out + c * ld + j) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (j + e < rank) out[sd.by_rank ? (j + e) * ld + c : c * ld + j + e] = lr_t<T>(v[e]);
        }
      }
  if (w.slot >= 0) return;
  __syncthreads();
  lr_put_gradient(w, out, rank);
}
// The parts of an adapter's units, added up in their order; zeros for adapters without rows.  A CTA adds up to 1024 numbers (lr_chans(rp)
// channels) of one adapter at a time, four to a thread, so that the loads of 16 parts are on the way at once, and stores them 16 bytes
// at a time.  Most adapters of many have nothing to add up: they share so many CTAs as fill the SMs.
__host__ __device__ inline int lr_chans(int rp) { return 1024 / rp / 8 * 8; }
template <typename T>
__global__ void __launch_bounds__(256) lr_join_kernel(const LrPlan p, const LrWgradSide<T> sa, const LrWgradSide<T> sb, int blocks_a,
                                                      int blocks, int rank, int rp) {
  __shared__ float sums[1024 + 64];  // a line of rp + 1 numbers to a channel
  after_previous();
  const int g = blockIdx.y, tid = threadIdx.x;
  const int s0 = p.slot[g], s1 = p.slot[g + 1];
  if (p.offset[g] == p.offset[g + 1]) {
    for (const LrWgradSide<T>* sd : {&sa, &sb}) {
      const int64_t size = static_cast<int64_t>(rank) * sd->C;  // a multiple of 8
      if (sd->blocks)
        for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + tid) * 8; i < size; i += static_cast<int64_t>(gridDim.x) * 256 * 8)
          *reinterpret_cast<uint4*>(sd->grad + g * size + i) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  if (s0 == s1) return;
  const int chans = lr_chans(rp), e = tid * 4, c = e / rp, j = e - c * rp;
  for (int block = blockIdx.x; block < blocks; block += gridDim.x) {
    const bool second = block >= blocks_a;
    const LrWgradSide<T>& sd = second ? sb : sa;
    const int64_t col = static_cast<int64_t>(second ? block - blocks_a : block) * chans;
    const int cols = static_cast<int>(min(static_cast<int64_t>(chans), sd.C - col));  // a multiple of 8
    if (c < cols) {
      const float4* from = reinterpret_cast<const float4*>(sd.part + col * rp + e);
      const int64_t step = sd.C * rp / 4;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int s = s0; s < s1; s += 16) {
        float4 v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = s + k < s1 ? from[(s + k) * step] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 16; ++k) sum.x += v[k].x, sum.y += v[k].y, sum.z += v[k].z, sum.w += v[k].w;
      }
      float* to = sums + c * (rp + 1) + j;
      to[0] = sum.x, to[1] = sum.y, to[2] = sum.z, to[3] = sum.w;
    }
    __syncthreads();
    T* const out = sd.grad + static_cast<int64_t>(g) * rank * sd.C;
    if (tid < rank * cols / 8) {
      float w[8];
      T* to;
      if (sd.by_rank) {  // eight channels of a rank
        const int jj = tid / (cols / 8), cc = (tid - jj * (cols / 8)) * 8;
#pragma unroll
        for (int q = 0; q < 8; ++q) w[q] = sums[(cc + q) * (rp + 1) + jj];
        to = out + jj * sd.C + col + cc;
      } else {  // eight numbers in the order of memory
        int cc = tid * 8 / rank, jj = tid * 8 - cc * rank;
        to = out + (col + cc) * rank + jj;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          w[q] = sums[cc * (rp + 1) + jj];
          if (++jj == rank) jj = 0, ++cc;
        }
      }
      *reinterpret_cast<uint4*>(to) = make_uint4(pack2<T>(w[0], w[1]), pack2<T>(w[2], w[3]), pack2<T>(w[4], w[5]), pack2<T>(w[6], w[7]));
    }
    __syncthreads();
  }
}

// ----------------------------------------------------------------------------------------------- launches
// Whether a batch's rows go by eights or by 128: while the weights that every eight rows read again cost less than the other kernels'
// fixed times (5120 -> 5120, us by eights and by 128: rank 16 512 rows 9.5, 13.5, 1024 rows 19.3, 14.5; rank 64 128 rows 13.8, 19.4,
// 512 rows 19.9, 20.8; rank 128 64 rows 23, 27, 256 rows 34, 28), and where most adapters have no more than eight rows anyway.
static bool lr_are_few(int64_t M, int64_t R, int rank) { return M <= 8 * R || (M <= 512 && M * lr_rp(rank) <= 12288); }
// CTAs that share the first product of a tile of few rows: some four to an SM in all, of four blocks of 32 columns at least,
// and 16 at most (their parts are added up by every CTA of the second product).  The SMs are B200's number, not the device's: the
// workspace goes by it, whose size is asked with any device current.
static int lr_few_splits(int64_t tiles, int64_t K) {
  const int64_t most = K / 128 < 16 ? K / 128 : 16, want = 4 * 148 / tiles;
  return static_cast<int>(want > most ? (most < 1 ? 1 : most) : want < 1 ? 1 : want);
}
// A workspace: hidden rows, then parts of the weight gradients or of few rows' first product
struct LrSpace {
  size_t part_a, part_b, total;
};
static LrSpace lr_space(int64_t M, int64_t K, int64_t N, int rank, int64_t R, bool backward) {
  LrSpace s{};
  s.part_a = lr_hidden_bytes(M, rank);
  if (!backward) {
    const int64_t tiles = lr_lines(M, R, LR_FEW);
    s.part_b = s.total = s.part_a + (lr_are_few(M, R, rank) ? lr_up256(static_cast<size_t>(tiles) * lr_few_splits(tiles, K) * 8 * lr_rp(rank) * 4) : 0);
    return s;
  }
  const size_t slot = static_cast<size_t>(lr_slots(M)) * lr_rp(rank) * 4;
  s.part_b = s.part_a + lr_up256(slot * K);
  s.total = s.part_b + lr_up256(slot * N);
  return s;
}
size_t lr_workspace(int64_t M, int64_t K, int64_t N, int rank, int64_t R, bool backward) {
  return M == 0 ? 0 : lr_space(M, K, N, rank, R, backward).total;
}
// How many CTAs share a tile's steps, 1, 2, 4 or 8: the fewest rounds of resident CTAs times the steps that each takes, with what a
// CTA's start and end cost (`extra` steps; about what 768 columns do: 97 tiles x 5120 columns go in two parts, 189 and 467 tiles whole,
// up to 33 tiles in eight).  Powers of two alone: a training step of
// 12090 rows takes 204 us with two parts, 227 with three (and 214 with four, 211 with five).
static int64_t lr_cost(int64_t tiles, int64_t steps, int64_t parts, int64_t slots, int64_t extra) {
  return ((tiles * parts + slots - 1) / slots) * ((steps + parts - 1) / parts + extra);
}
static int lr_splits(int64_t tiles, int64_t chunks, int extra, int ctas) {
  const int64_t slots = static_cast<int64_t>(ctas) * cross_sms();
  int best = 1;
  for (int n = 2; n <= 8; n *= 2)
    if (lr_cost(tiles, chunks, n, slots, extra) < lr_cost(tiles, chunks, best, slots, extra)) best = n;
  return best;
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
static bool lr_wide(const void* p, int64_t ld) { return !p || (ld % 16 == 0 && reinterpret_cast<uintptr_t>(p) % 32 == 0); }
template <typename T, bool W_ROWS, int RPM>
static int lr_first_s(const LrPlan& p, const T* x, int64_t ldx, int64_t C, const T* w, int rank, int rp, int R, const float* scales,
                       LrHid<T>* h, cudaStream_t st) {
  using Cfg = LrFirstCfg<RPM, W_ROWS>;
  static std::atomic<bool> ready[CA_DEVICES];
  const int splits = lr_splits(p.n_tiles, (C + Cfg::KC - 1) / Cfg::KC, 768 / Cfg::KC, Cfg::CTAS);
  return lr_launch("lr_first_kernel", lr_first_kernel<T, W_ROWS, RPM>, ready, dim3(static_cast<unsigned>(p.n_tiles * splits)),
                   LR_FIRST_THREADS, Cfg::SMEM, splits, st, p, x, ldx, C, w, rank, rp, R, scales, h, splits);
}
template <typename T, bool W_ROWS>
static int lr_first(const LrPlan& p, const T* x, int64_t ldx, int64_t C, const T* w, int rank, int R, const float* scales,
                     LrHid<T>* h, cudaStream_t st) {
  const int rp = lr_rp(rank);
  if (rp <= 64) return lr_first_s<T, W_ROWS, 64>(p, x, ldx, C, w, rank, rp, R, scales, h, st);
  return lr_first_s<T, W_ROWS, 128>(p, x, ldx, C, w, rank, rp, R, scales, h, st);
}
template <typename T, bool W_ROWS, bool BASE, int NQ>
static int lr_second_s(const LrPlan& p, const LrHid<T>* h, const T* w, int rank, int rp, int R, const T* base, int64_t ldb, T* out,
                       int64_t ldo, int64_t N, cudaStream_t st) {
  using Cfg = LrSecondCfg<NQ, W_ROWS, BASE, LR_WIDE<T>>;
  static std::atomic<bool> ready[CA_DEVICES];
  const int parts = static_cast<int>((N + Cfg::COLS - 1) / Cfg::COLS);
  return lr_launch("lr_second_kernel", lr_second_kernel<T, W_ROWS, BASE, NQ>, ready, dim3(static_cast<unsigned>(p.n_tiles * parts)), LR_THREADS,
                   Cfg::SMEM, 1, st, p, h, w, rank, rp, R, base, ldb, out, ldo, N, parts,
                   N % 16 == 0 && lr_wide(base, ldb) && lr_wide(out, ldo));
}
// W_ROWS: with or without base; else (dx) without
template <typename T, bool W_ROWS, int NQ>
static int lr_second_b(const LrPlan& p, const LrHid<T>* h, const T* w, int rank, int rp, int R, const T* base, int64_t ldb, T* out,
                       int64_t ldo, int64_t N, cudaStream_t st) {
  if constexpr (W_ROWS)
    if (base) return lr_second_s<T, W_ROWS, true, NQ>(p, h, w, rank, rp, R, base, ldb, out, ldo, N, st);
  return lr_second_s<T, W_ROWS, false, NQ>(p, h, w, rank, rp, R, nullptr, 0, out, ldo, N, st);
}
template <typename T, bool W_ROWS>
static int lr_second(const LrPlan& p, const LrHid<T>* h, const T* w, int rank, int R, const T* base, int64_t ldb, T* out, int64_t ldo,
                     int64_t N, cudaStream_t st) {
  const int rp = lr_rp(rank);
  if (rp <= 16) return lr_second_b<T, W_ROWS, 1>(p, h, w, rank, rp, R, base, ldb, out, ldo, N, st);
  if (rp <= 32) return lr_second_b<T, W_ROWS, 2>(p, h, w, rank, rp, R, base, ldb, out, ldo, N, st);
  if (rp <= 64) return lr_second_b<T, W_ROWS, 4>(p, h, w, rank, rp, R, base, ldb, out, ldo, N, st);
  return lr_second_b<T, W_ROWS, 8>(p, h, w, rank, rp, R, base, ldb, out, ldo, N, st);
}
template <typename T, int RPM, int ST>
static int lr_wgrad_s(const LrPlan& p, const LrWgradSide<T>& a, const LrWgradSide<T>& b, int rank, int R, cudaStream_t st) {
  static std::atomic<bool> ready[CA_DEVICES];
  const dim3 grid(static_cast<unsigned>(p.n_units * (a.blocks + b.blocks)));
  if constexpr (LR_WIDE<T>)
    return lr_launch("lr_wgrad_wide_kernel", lr_wgrad_wide_kernel<T, RPM, ST>, ready, grid, 128, LrWgradWideCfg<RPM, ST>::SMEM, 1, st, p, a, b,
                     rank, lr_rp(rank), R);
  else
    return lr_launch("lr_wgrad_kernel", lr_wgrad_kernel<T, RPM, ST>, ready, grid, 160, LrWgradCfg<RPM, ST>::SMEM, 1, st, p, a, b, rank,
                     lr_rp(rank), R);
}
template <typename T, int RPM>
static int lr_wgrad(const LrPlan& p, const LrWgradSide<T>& a, const LrWgradSide<T>& b, int rank, int64_t M, int R, cudaStream_t st) {
  static std::atomic<bool> joined[CA_DEVICES];
  const int rp = lr_rp(rank);
  const bool one = M <= (LR_WIDE<T> ? LR_WROWS : LR_KROWS) * R;
  if (int rc = one ? lr_wgrad_s<T, RPM, 1>(p, a, b, rank, R, st) : lr_wgrad_s<T, RPM, 3>(p, a, b, rank, R, st)) return rc;
  const int chans = lr_chans(rp);
  const int ja = static_cast<int>((a.blocks ? a.C + chans - 1 : 0) / chans), jb = static_cast<int>((b.blocks ? b.C + chans - 1 : 0) / chans);
  const int each = (8 * cross_sms() + R - 1) / R;
  return lr_launch("lr_join_kernel", lr_join_kernel<T>, joined, dim3(ja + jb < each ? ja + jb : each, R), 256, 0, 1, st, p, a, b, ja, ja + jb,
                   rank, rp);
}
template <typename T, int RB>
static int lr_few_s(const LrPlan& p, const LrArgs& a, int rp, LrHid<T>* h, float* part, cudaStream_t st) {
  static std::atomic<bool> ready[2][CA_DEVICES];
  const T* base = static_cast<const T*>(a.base);
  T* out = static_cast<T*>(a.out);
  const int splits = lr_few_splits(p.n_few, a.K), R = static_cast<int>(a.R);
  const int columns = static_cast<int>((a.N + 2 * LR_FEW_THREADS - 1) / (2 * LR_FEW_THREADS));
  if (int rc = lr_launch("lr_few_down_kernel", lr_few_down_kernel<T, RB>, ready[0], dim3(static_cast<unsigned>(p.n_few * splits)),
                         LR_FEW_THREADS, 0, 1, st, p, static_cast<const T*>(a.x), a.ldx, a.K, static_cast<const T*>(a.a), a.rank, rp, R,
                         splits, part))
    return rc;
  return lr_launch("lr_few_up_kernel", lr_few_up_kernel<T, RB>, ready[1], dim3(static_cast<unsigned>(p.n_few * columns)), LR_FEW_THREADS, 0, 1,
                   st, p, static_cast<const T*>(a.b), a.rank, rp, R, a.scales, base, a.ldbase, out, a.ldo, a.N, columns,
                   a.N % 16 == 0 && lr_wide(base, a.ldbase) && lr_wide(out, a.ldo), part, splits, h, a.hidden != nullptr);
}
template <typename T>
static int lr_few(const LrPlan& p, const LrArgs& a, LrHid<T>* h, float* part, cudaStream_t st) {
  const int rp = lr_rp(a.rank);
  if (rp <= 16) return lr_few_s<T, 1>(p, a, rp, h, part, st);
  if (rp <= 32) return lr_few_s<T, 2>(p, a, rp, h, part, st);
  if (rp <= 64) return lr_few_s<T, 4>(p, a, rp, h, part, st);
  return lr_few_s<T, 8>(p, a, rp, h, part, st);
}
template <typename T>
static int lr_forward_t(const LrArgs& a, cudaStream_t st) {
  const LrPlan p = lr_plan(a.plan, a.M, a.R);
  LrHid<T>* const h = static_cast<LrHid<T>*>(a.hidden ? a.hidden : a.ws);
  const int R = static_cast<int>(a.R);
  if (lr_are_few(a.M, a.R, a.rank))
    return lr_few<T>(p, a, h, reinterpret_cast<float*>(static_cast<char*>(a.ws) + lr_space(a.M, a.K, a.N, a.rank, a.R, false).part_a), st);
  if (int rc = lr_first<T, true>(p, static_cast<const T*>(a.x), a.ldx, a.K, static_cast<const T*>(a.a), a.rank, R, a.scales, h, st))
    return rc;
  return lr_second<T, true>(p, h, static_cast<const T*>(a.b), a.rank, R, static_cast<const T*>(a.base), a.ldbase, static_cast<T*>(a.out),
                            a.ldo, a.N, st);
}
template <typename T>
static int lr_backward_t(const LrArgs& a, cudaStream_t st) {
  const LrPlan p = lr_plan(a.plan, a.M, a.R);
  const LrSpace s = lr_space(a.M, a.K, a.N, a.rank, a.R, true);
  LrHid<T> *const h = static_cast<LrHid<T>*>(a.hidden), *const dh = static_cast<LrHid<T>*>(a.ws);
  const int R = static_cast<int>(a.R);
  const T *x = static_cast<const T*>(a.x), *go = static_cast<const T*>(a.go);
  if (a.dx || a.da)
    if (int rc = lr_first<T, false>(p, go, a.ldgo, a.N, static_cast<const T*>(a.b), a.rank, R, a.scales, dh, st)) return rc;
  if (a.dx)
    if (int rc = lr_second<T, false>(p, dh, static_cast<const T*>(a.a), a.rank, R, nullptr, 0, static_cast<T*>(a.dx), a.lddx, a.K, st))
      return rc;
  if (!a.da && !a.db) return H3B_OK;
  char* ws = static_cast<char*>(a.ws);
  const int blocks_k = static_cast<int>((a.K + 127) / 128), blocks_n = static_cast<int>((a.N + 127) / 128);
  const LrWgradSide<T> sa{x, a.ldx, a.K, dh, static_cast<T*>(a.da), reinterpret_cast<float*>(ws + s.part_a), a.da ? blocks_k : 0, true};
  const LrWgradSide<T> sb{go, a.ldgo, a.N, h, static_cast<T*>(a.db), reinterpret_cast<float*>(ws + s.part_b), a.db ? blocks_n : 0, false};
  return lr_rp(a.rank) <= 64 ? lr_wgrad<T, 64>(p, sa, sb, a.rank, a.M, R, st) : lr_wgrad<T, 128>(p, sa, sb, a.rank, a.M, R, st);
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
