// Shared parts of the cross-attention kernels (cross_fwd.cuh, cross_bwd.cuh): argument block, tensor maps, the bf16/fp16
// tcgen05 wrappers, and the mask preparation.
//
//   s_ij = scale q_i . k_j + bias_j          bias_j: 0, the additive key bias (less its largest value), -inf if masked
//   p_ij = exp(s_ij - lse_i),  lse_i = log sum_j exp(s_ij),  o_i = sum_j p_ij v_j;   no key left: o_i = 0, lse_i = -inf
//   backward, with g = dL/do:  delta_i = g_i . o_i,  ds_ij = p_ij (g_i . v_j - delta_i)
//     dv_j = sum_i p_ij g_i,  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
//   Hq / Hkv query heads share a key head; their gradients add up in dk and dv.
//
// Query tiles: 128 rows are (128 / G) queries x the G = Hq / Hkv query heads of one key head, row = query * G + head, so
// heads that share keys read them once; a 5-D tensor map (channel, head of the group, key head, query, batch) loads and
// stores such a tile in one copy per 64 channels.  Channels are padded to 64 or 128 (DP) by the copy's zero fill.
#pragma once

#include <atomic>
#include <mutex>
#include <type_traits>

#include "fastdiv.cuh"
#include "h3b_common.cuh"
#include "launch.h"

namespace h3b {

constexpr int CT = 128;  // rows of a query tile, keys of a key tile
constexpr float CA_LOG2E = 1.4426950408889634f, CA_LN2 = 0.6931471805599453f;

struct CrossParams {
  h3b_attn_tensor q, k, v, o, go, dq, dk, dv;
  float* lse;              // [B, Hq, Sq]
  const int32_t* kv_lens;  // [B] keys in use, or null: all
  const float* bias2;      // [B, Skp] what is added to the scores, in units of log2; or null
  float* part_o;           // [splits, B * Hq * Sq, D] partial outputs, each normalised by its own sum
  float* part_lse;         // [splits, B * Hq * Sq] their log-sum-exps in units of log2
  float* stats;            // backward: [B, Hkv, q_tiles][-lse log2(e), delta][128 tile rows]
  float* g_norm2;          // backward, fp16: [B, Hkv, q_tiles][128 tile rows] squared norms of g
  float* g_top2;           // [B, Hkv, q_tiles] the largest of a tile's
  float* v_top2;           // [B, Hkv, Skp / 128] the largest squared norm of the values in use of a key tile
  float* v_all2;           // [B, Hkv] the largest of all tiles
  float* part_dq;          // [splits, B * Hq * Sq, D] partial dQ
  float* part_dk;          // [kv_splits][dK, dV][B * Hkv * Sk, D] partial dK and dV
  int64_t Sq, Sk, Skp;
  int B, Hq, Hkv, G, D, nq;  // nq: queries of a tile
  int q_tiles, units;  // query tiles; pairs of them
  int splits;          // key splits of a unit (forward, dQ)
  int ragged;          // forward: 0, or how many splits of all entries there are at most, of a size chosen from the lengths
  int kv_splits;       // query splits of a unit (dK, dV)
  float scale, scale2;         // scale2 = scale log2(e)
  bool wide;                   // backward: rows of dq, dk and dv start on 32-byte boundaries and are multiples of 32 bytes
  FastDiv by_g, by_hkv, by_units, by_splits, by_q_tiles, by_k_tiles, by_kv_splits, by_batch;
};

__device__ __forceinline__ int64_t ca_len(const int32_t* lens, int b, int64_t Sk) {
  if (!lens) return Sk;
  const int64_t n = lens[b];
  return n < 0 ? 0 : n > Sk ? Sk : n;
}

// ----------------------------------------------------------------------------------------------- PTX wrappers
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tma_store_5d(const void* src, const CUtensorMap* map, int c0, int c1, int c2, int c3, int c4) {
  asm volatile("cp.async.bulk.tensor.5d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5, %6}], [%1];" ::"l"(map),
               "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// bring a tile into L2
__device__ __forceinline__ void tma_prefetch_5d(const CUtensorMap* map, int c0, int c1, int c2, int c3, int c4) {
  asm volatile("cp.async.bulk.prefetch.tensor.5d.L2.global [%0, {%1, %2, %3, %4, %5}];" ::"l"(map), "r"(c0), "r"(c1), "r"(c2),
               "r"(c3), "r"(c4)
               : "memory");
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// D[tmem] (+)= A B, bf16/fp16 operands, fp32 accumulator; A from shared memory or from tensor memory.  Operands in shared memory
// are given by the low words of their descriptors (desc_rows, desc_chan): the high word is the same constant for all of them
// (groups of 8 rows 1024 bytes apart, descriptor version 1, 128-byte swizzle) and is joined here, next to its use.  As 64-bit
// values kept through the loops, the compiler (12.9) lost their swizzle bits in one variant of the gradient kernels after an edit
// elsewhere in the kernel: the product then read the tile as if it were not swizzled.
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 h;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b32 h, %5;\n\t"
      "mov.b64 a, {%1, h};\n\tmov.b64 b, {%2, h};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(DESC_HI)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 h;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b32 h, %5;\n\t"
      "mov.b64 b, {%2, h};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(DESC_HI)
      : "memory");
}
// 32 lanes x 16 consecutive 32-bit columns: thread i of the warp gets its lane's 16 columns.
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// 32 lanes x 32 consecutive 32-bit columns: thread i of the warp writes its lane's 32 columns.
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One lane of a converged warp, the same one every time.  The MMA warp runs its loop as a whole and elects a lane only around
// the tcgen05 instructions: what they take from registers stays warp-uniform.  (With the loop inside `if (lane == 0)` every
// operand of every product was moved to a uniform register by itself: 67 cycles a product, and 4550 instead of ~3200 cycles
// for two query tiles x one key tile of the forward kernel.)
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void commit_one(uint64_t* bar) {
  if (elect_one()) mma_commit(bar);
}
// Instruction descriptor of tcgen05.mma kind::f16: A and B of one type, fp32 accumulator, M x N tile, A K-major,
// B K-major or (b_mn) with its N index contiguous.
template <typename T>
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool b_mn) {
  const uint32_t fmt = std::is_same_v<T, __nv_bfloat16> ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
// A tile of shared memory: 128 rows, DP channels, in parts of 64 channels (128 rows x 128 bytes, 128-byte swizzle).
constexpr uint32_t SUB_BYTES = CT * 128;
// Descriptor (its low word: start address, leading offset) of a tile whose rows are the operand's M or N index (K-major); step kk
// (16 channels) adds rows_step(kk).  Offsets are in units of 16 bytes and stay inside the 14-bit address field (shared memory is
// under 256 KB).
__device__ __forceinline__ uint32_t desc_rows(uint32_t tile) { return (tile & 0x3FFFFu) >> 4 | 1u << 16; }
__host__ __device__ constexpr uint32_t rows_step(int kk) { return ((kk >> 2) * SUB_BYTES + (kk & 3) * 32) >> 4; }
// Descriptor of a tile whose channels are the operand's N index and whose rows are K (MN-major): 64-channel parts
// SUB_BYTES apart (leading offset), groups of 8 rows 1024 bytes apart (stride offset); step kk (16 rows) adds chan_step(kk).
__device__ __forceinline__ uint32_t desc_chan(uint32_t tile) { return (tile & 0x3FFFFu) >> 4 | (SUB_BYTES >> 4) << 16; }
__host__ __device__ constexpr uint32_t chan_step(int kk) { return (kk * 2048) >> 4; }
// the products of one tile, in steps of 16: D (+)= A B^T with A and B K-major in shared memory
template <int STEPS>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  if (elect_one())
#pragma unroll
    for (int kk = 0; kk < STEPS; ++kk) mma_f16_ss(d, a + rows_step(kk), b + rows_step(kk), idesc, kk > 0);
}
// D = A B^T with A [128 rows, STEPS x 16 channels] in tensor memory (16-bit columns side by side), B K-major in shared memory
template <int STEPS>
__device__ __forceinline__ void mma_rows_ta(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  if (elect_one())
#pragma unroll
    for (int kk = 0; kk < STEPS; ++kk) mma_f16_ts(d, a + kk * 8, b + rows_step(kk), idesc, kk > 0);
}
// D (+)= A B with A [128 rows x 128] in tensor memory and B's 128 rows in shared memory.  A's 16-bit columns lie side by
// side (PARTS 1), or in PARTS parts at the first columns of the fp32 values that one group of warps each read.
template <int PARTS>
__device__ __forceinline__ void mma_chan(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  constexpr int PER = CT / 16 / PARTS;
  if (elect_one())
#pragma unroll
    for (int kk = 0; kk < CT / 16; ++kk)
      mma_f16_ts(d, a + kk / PER * (CT / PARTS) * (PARTS > 1) + (PARTS > 1 ? kk % PER : kk) * 8, b + chan_step(kk), idesc, acc | (kk > 0));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// wait for the kernel before this one in the stream (and its writes)
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int R>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}
// every lane of the warp waits; one outcome for all (what follows are whole-warp instructions)
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort));
}
// Barriers of some warps of a CTA.  They have no bound: every warp of the group reaches each of them whatever its waits on
// mbarriers came to (after a wait that gave up, a role goes through its loops without waiting).
__device__ __forceinline__ void group_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ bool group_any(int id, int threads, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbar.red.or.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"(static_cast<uint32_t>(v))
      : "memory");
  return r != 0;
}
// write 8 packed values (16 bytes, chunk c of 8) of row r into a 64-channel part with the 128-byte swizzle
__device__ __forceinline__ void put_swizzled(unsigned char* part, int r, int c, uint4 v) {
  *reinterpret_cast<uint4*>(part + r * 128 + ((c ^ (r & 7)) << 4)) = v;
}

// pairs of fp32 in one 64-bit register: one instruction per two sums or products
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 f2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_split(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 f2_fma(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 f2_add(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 f2_mul(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// exp2 of two numbers <= 16 on the FMA pipe (the special function unit's 4 results per cycle and scheduler are the bound of
// softmax loops): x = n + f, |f| <= 1/2 by adding and taking off 1.5 * 2^23; 2^f by a degree-4 polynomial fitted to the least
// largest relative error (2.6e-6; 2.7e-6 as evaluated in fp32).  Range reduction and minimax polynomials are textbook (Muller,
// Elementary Functions); taking part of a softmax's exponentials so is a published technique of attention kernels.  TAIL false: n is added to the exponent; below 2^-126 that is 2^-126, and NaN may come out
// as any number.  TAIL true, one instruction more: times 2^n, with 0 below 2^-126 (the bits of 2^n end at n = -127, and x is
// held there); NaN stays.
template <bool TAIL>
__device__ __forceinline__ f32x2 f2_exp2(float xa, float xb) {
  const f32x2 x = TAIL ? f2(max_nan(xa, -127.f), max_nan(xb, -127.f)) : f2(fmaxf(xa, -126.f), fmaxf(xb, -126.f));
  const f32x2 t = f2_add(x, f2(12582912.f, 12582912.f));
  const f32x2 f = f2_fma(f2_add(t, f2(-12582912.f, -12582912.f)), f2(-1.f, -1.f), x);
  f32x2 p = f2_fma(f2(0.009570101946812917f, 0.009570101946812917f), f, f2(0.05591786158553334f, 0.05591786158553334f));
  p = f2_fma(p, f, f2(0.24024744837984488f, 0.24024744837984488f));
  p = f2_fma(p, f, f2(0.6931218145829676f, 0.6931218145829676f));
  p = f2_fma(p, f, f2(0.9999992614392343f, 0.9999992614392343f));
  float ta, tb, pa, pb;
  f2_split(t, ta, tb);  // the low bits of t are n
  const int na = __float_as_int(ta) << 23, nb = __float_as_int(tb) << 23;
  if constexpr (TAIL) return f2_mul(p, f2(__int_as_float(na + (127 << 23)), __int_as_float(nb + (127 << 23))));
  f2_split(p, pa, pb);
  return f2(__int_as_float(__float_as_int(pa) + na), __int_as_float(__float_as_int(pb) + nb));
}

// 16 columns of a row of results (n: valid columns from here on, a multiple of 8): one 32-byte store where every row allows it
// (`wide`), else 16-byte ones.  A lane per row: an instruction touches 32 lines either way, so half the instructions count.
template <typename T>
__device__ __forceinline__ void store_cols(T* dst, const uint32_t (&o)[16], float w, int n, bool wide) {
  uint32_t v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = pack2<T>(__uint_as_float(o[2 * i]) * w, __uint_as_float(o[2 * i + 1]) * w);
  if (wide) {
    if (n > 0)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                   "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                   : "memory");
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (8 * i < n) *reinterpret_cast<uint4*>(dst + 8 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}
__device__ __forceinline__ void store_cols_f32(float* dst, const uint32_t (&o)[16], float w, int n) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (4 * i < n)
      *reinterpret_cast<float4*>(dst + 4 * i) =
          make_float4(__uint_as_float(o[4 * i]) * w, __uint_as_float(o[4 * i + 1]) * w, __uint_as_float(o[4 * i + 2]) * w,
                      __uint_as_float(o[4 * i + 3]) * w);
}

// ----------------------------------------------------------------------------------------------- mask preparation
// One CTA per batch entry turns a key mask into what the kernels add to the scores: bias2[j] = log2(e) (bias_j - top),
// top the largest bias in use (softmax does not change, and an entry whose keys all carry a large negative value keeps
// its scores' digits and its log-sum-exp), -inf for keys that are out; and the number of keys up to the last one in use.
struct MaskArgs {
  const void* mask;  // null: none
  const int32_t* kv_lens;
  float* bias2;
  int32_t* lens;
  int64_t ldm, Sk, Skp;
  int kind;
};
__device__ __forceinline__ float ca_mask_value(const MaskArgs& a, int64_t i) {
  return a.kind == H3B_MASK_BOOL ? (static_cast<const uint8_t*>(a.mask)[i] ? 0.f : -INFINITY) : static_cast<const float*>(a.mask)[i];
}
template <int THREADS>
__device__ __forceinline__ void prepare_mask(const MaskArgs& a, int b) {
  constexpr int W = THREADS / 32;
  __shared__ float top_s[W];
  __shared__ int last_s[W];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t len = ca_len(a.kv_lens, b, a.Sk);
  float top = -INFINITY;
  int last = 0;
  for (int64_t j = threadIdx.x; j < len; j += THREADS) {
    const float v = ca_mask_value(a, b * a.ldm + j);
    if (v != -INFINITY) last = static_cast<int>(j) + 1;
    top = fmaxf(top, v);
  }
  for (int o = 16; o; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
  }
  if (lane == 0) top_s[w] = top, last_s[w] = last;
  __syncthreads();
  top = top_s[lane % W], last = last_s[lane % W];
  for (int o = W / 2; o; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
  }
  if (threadIdx.x == 0) a.lens[b] = last;
  for (int64_t j = threadIdx.x; j < a.Skp; j += THREADS) {
    const float v = j < len ? ca_mask_value(a, b * a.ldm + j) : -INFINITY;
    a.bias2[b * a.Skp + j] = v == -INFINITY ? v : (v - top) * CA_LOG2E;
  }
}
constexpr int CA_PREP = 1024;
static __global__ void __launch_bounds__(CA_PREP) cross_mask_kernel(const MaskArgs a) {
  after_previous();
  prepare_mask<CA_PREP>(a, blockIdx.x);
}

// ----------------------------------------------------------------------------------------------- tensor maps
typedef CUresult (*CrossEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static CrossEncodeFn cross_encode_fn() {
  static CrossEncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<CrossEncodeFn>(p);
  });
  return fn;
}
// dims / strides (elements; strides of dims 1..) of a 2-byte tensor; box: 64 channels x the given extents
static int cross_map(CUtensorMap* map, const void* base, bool half, int rank, const int64_t* ext, const int64_t* str,
                     const int* box_ext) {
  CrossEncodeFn fn = cross_encode_fn();
  if (!fn) return fail(H3B_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable (driver too old?)");
  cuuint64_t dims[5], strides[4];
  cuuint32_t box[5], one[5];
  for (int i = 0; i < rank; ++i) {
    dims[i] = static_cast<cuuint64_t>(ext[i] > 0 ? ext[i] : 1);  // an empty side is never loaded
    box[i] = static_cast<cuuint32_t>(box_ext[i]);
    one[i] = 1;
    // the stride of an extent of one is never used; any valid value will do
    if (i) strides[i - 1] = ext[i] > 1 ? static_cast<cuuint64_t>(str[i]) * 2 : 16;
  }
  const CUresult r = fn(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
                        const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(H3B_ERR_CUDA, "cuTensorMapEncodeTiled failed (code " + std::to_string(int(r)) + ")");
  return H3B_OK;
}
// What the map of an empty side is made of (nothing loads from it): a pointer and strides that a map may have.
static h3b_attn_tensor cross_stand_in(const h3b_attn_tensor& t) { return h3b_attn_tensor{t.ptr, 8, 8, 8}; }
// (channel, head of the group, key head, query, batch), a box of 64 channels x G heads x nq queries
static int cross_map_q(CUtensorMap* map, const CrossParams& P, const h3b_attn_tensor& t, bool half) {
  const int64_t ext[5] = {P.D, P.G, P.Hkv, P.Sq, P.B};
  const int64_t str[5] = {1, t.stride_h, t.stride_h * P.G, t.stride_s, t.stride_b};
  const int box[5] = {64, P.G, 1, P.nq, 1};
  return cross_map(map, t.ptr, half, 5, ext, str, box);
}
// (channel, key head, key, batch), a box of 64 channels x 128 keys
static int cross_map_k(CUtensorMap* map, const CrossParams& P, const h3b_attn_tensor& t, bool half) {
  const int64_t ext[4] = {P.D, P.Hkv, P.Sk, P.B};
  const int64_t str[4] = {1, t.stride_h, t.stride_s, t.stride_b};
  const int box[4] = {64, 1, CT, 1};
  return cross_map(map, t.ptr, half, 4, ext, str, box);
}

// Launch that may begin while the kernel before it in the stream finishes: set-up (barriers, tensor memory, descriptors)
// overlaps its tail.  (The kernel before gives no early signal: CTAs of the next one that wait on an SM cost the running one
// a tenth of its time.)  Every kernel launched so calls after_previous() before it touches global memory, and reads it with
// plain loads: the read-only path (__ldg) is for data that nobody writes while the kernel runs, its waiting part included.
template <typename... KA, typename... A>
static int cross_launch_after(const char* what, void (*kernel)(KA...), dim3 grid, int threads, int smem, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<KA>(args)...);
  return e == cudaSuccess ? check_launch(what) : cuda_fail(e, what);
}

// SM count and what a kernel needs set before its first launch: asked for and set once per device (a property of the
// device and of the kernel; a call spends over a microsecond on them otherwise).
constexpr int CA_DEVICES = 64;
static int cross_device() {
  int dev = 0;
  cudaGetDevice(&dev);
  return dev;
}
static int cross_sms() {
  static std::atomic<int> known[CA_DEVICES];
  const int dev = cross_device();
  int sms = dev < CA_DEVICES ? known[dev].load(std::memory_order_relaxed) : 0;
  if (sms == 0) {
    sms = 148;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (dev < CA_DEVICES) known[dev].store(sms, std::memory_order_relaxed);
  }
  return sms;
}
// `done`: one flag per device of this kernel
static int cross_smem(const void* kernel, int bytes, std::atomic<bool> (&done)[CA_DEVICES], const char* what) {
  const int dev = cross_device();
  if (dev < CA_DEVICES && done[dev].load(std::memory_order_acquire)) return H3B_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return cuda_fail(e, what);
  if (dev < CA_DEVICES) done[dev].store(true, std::memory_order_release);
  return H3B_OK;
}

}  // namespace h3b
