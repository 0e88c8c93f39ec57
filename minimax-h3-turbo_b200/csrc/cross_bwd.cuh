// Cross attention gradients on the tcgen05 tensor cores, two kernels after one for the row vectors, no atomics.
//
// cross_dq_kernel: a unit is one query tile (128 rows) over a range of key tiles:
//     S = Q K^T, dP = G V^T, dS = P (dP - delta), dQ += dS K           (rows of tensor memory are queries)
//   delta = g . o comes from cross_stats_kernel, which writes it and -lse of every tile row in tile order (inside this
//   kernel it cost over 3 us a unit).  When all keys fit one tile delta = sum_j p_j dP_j instead: the same number without
//   the rounding of o, which is all there is to dS when one key takes the whole weight.
// cross_dkv_kernel: a unit is one key tile over a range of query tiles of all heads that share it:
//     S^T = K Q^T, dP^T = V G^T, dV += P^T G, dK += dS^T Q             (rows of tensor memory are keys)
// Each computes S and dP: 7 products of the scores' size instead of 5.  The price of sharing them (dQ summed over key tiles
// by atomics, in a changing order, through fp32 buffers in memory) is not paid: results have the same bits every time.
// P and dS are rounded to the operand type for the second products (8 or 11 bits, relative to each element); sums are fp32.
// fp16 has few exponents: P of 12090 keys lies where its steps are absolute, and so does dS of a gradient of ordinary size, or
// past its range (do of 1e-3 over 12090 keys: dq off by 1.6e-2 if rounded as they are).  So both are held times a power of two
// that the fp32 results are divided by: P times 2^14, dS times what keeps its bound |g| max |v| / 2 below 2^15, |g| of the row for
// dQ, the largest of the unit's rows for dK (there rows are what is summed over).  cross_stats_kernel takes the norms, for which it
// reads the values once more: 2 x 12090 queries x 512 keys x 40 heads x 64 697 -> 737 us, 3 x 5 queries x 12090 keys, 56 over 8
// heads x 128 108 -> 129 us, against the same kernels without the factors.
//
// Warps of both: 0-15 elementwise work, thread = row, four warps to the same 32 rows with 32 columns each; 16-19 epilogue
// (accumulators -> global memory); 20 MMA issue; 21 copies; 22 (dQ) zeroes K rows of masked
// keys before their product.  P and dS go back to tensor memory over the columns that their own warps read S or dP from.
//
// bf16, 40 heads x 128 channels, both with the row vectors, at 1965 MHz / in a row under the power limit: 2 x 4096 queries x 512 keys
// 340 / 375 us (885 / 800 TFLOP/s of 7 products), 12090 x 1600 1200 / 1380 us (1160 / 1005).  Tensor pipe 65 % (dQ)
// and 74 % (dK, dV) active; neither HBM (8 %) nor the FMA pipe (40 %) is near its limit: the chain scores -> elementwise work ->
// second product is.
#include "cross_common.cuh"

namespace h3b {

struct BwdTile {
  int it, b, hk, split, tile, t0, t1, t;  // `tile`: the unit's own tile; t: the tile of the other side
  __device__ __forceinline__ bool first() const { return t == t0; }
  __device__ __forceinline__ bool last() const { return t == t1 - 1; }
};

// Walks the units of this CTA.  DQ: own tiles are query tiles, the other side key tiles; else the other way round.
template <bool DQ>
struct BwdWalk {
  const CrossParams& P;
  int n, splits;
  BwdTile c;
  bool valid;
  __device__ __forceinline__ BwdWalk(const CrossParams& p) : P(p) {
    splits = DQ ? p.splits : p.kv_splits;
    n = (DQ ? p.q_tiles : static_cast<int>(p.Skp / CT)) * splits * p.Hkv * p.B;
    c.it = blockIdx.x;
    seek();
  }
  __device__ __forceinline__ void unit(int it, BwdTile& u) const {
    const FastDiv &by_own = DQ ? P.by_q_tiles : P.by_k_tiles, &by_split = DQ ? P.by_splits : P.by_kv_splits;
    const int r = by_split.divmod(by_own.divmod(it, u.tile), u.split);
    u.b = P.by_hkv.divmod(r, u.hk);
    const int64_t len = ca_len(P.kv_lens, u.b, P.Sk);
    const int other = DQ ? static_cast<int>((len + CT - 1) / CT) : static_cast<int64_t>(u.tile) * CT < len ? P.q_tiles : 0;
    const int per = by_split.div(other + splits - 1);
    u.t0 = min(u.split * per, other);
    u.t1 = min(u.t0 + per, other);
    u.t = u.t0;
  }
  __device__ __forceinline__ void seek() {  // the first unit from c.it on with work
    for (valid = false; c.it < n; c.it += gridDim.x) {
      unit(c.it, c);
      if (c.t1 > c.t0) {
        valid = true;
        return;
      }
    }
  }
  __device__ __forceinline__ void next() {
    if (++c.t < c.t1) return;
    c.it += gridDim.x;
    seek();
  }
};

// The same walk for the MMA warp, which needs only how many tiles a unit has.
template <bool DQ>
struct BwdCount {
  const CrossParams& P;
  int it, left;
  bool first;
  __device__ __forceinline__ BwdCount(const CrossParams& p) : P(p), it(blockIdx.x) { seek(); }
  __device__ __forceinline__ bool valid() const { return left > 0; }
  __device__ __forceinline__ bool last() const { return left == 1; }
  __device__ __forceinline__ void seek() {
    const int splits = DQ ? P.splits : P.kv_splits;
    const int n = (DQ ? P.q_tiles : static_cast<int>(P.Skp / CT)) * splits * P.Hkv * P.B;
    first = true;
    for (left = 0; it < n; it += gridDim.x) {
      const FastDiv &by_own = DQ ? P.by_q_tiles : P.by_k_tiles, &by_split = DQ ? P.by_splits : P.by_kv_splits;
      int tile, split;
      const int b = P.by_hkv.div(by_split.divmod(by_own.divmod(it, tile), split));
      const int64_t len = ca_len(P.kv_lens, b, P.Sk);
      const int other = DQ ? static_cast<int>((len + CT - 1) / CT) : static_cast<int64_t>(tile) * CT < len ? P.q_tiles : 0;
      const int per = by_split.div(other + splits - 1);
      left = min(per, other - min(split * per, other));
      if (left > 0) return;
    }
  }
  __device__ __forceinline__ void next() {
    first = false;
    if (--left > 0) return;
    it += gridDim.x;
    seek();
  }
};

template <int DP>
struct BwdCfg {
  static constexpr int NSUB = DP / 64;
  static constexpr int TILE = NSUB * static_cast<int>(SUB_BYTES);
  static constexpr int SMEM = 7 * TILE + 4 * CT * 4 + 512;  // 7 tiles, small vectors, barriers and exponents (472 bytes)
  static constexpr int THREADS = 768;
  static constexpr uint32_t TMEM_COLS = 512;
};

// ------------------------------------------------------------------------------------------------ fp16's range
constexpr int P_EXP = 14;  // fp16: P is held times 2^P_EXP
template <typename T>
constexpr bool scaled = std::is_same_v<T, __half>;
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }
// e of the factor 2^e for dS.  dP_j - delta = (1 - p_j) (dP_j - mean of the others), so |dS| <= p (1 - p) 2 |g| |v| <= |g| |v| / 2;
// 2^e times that is below 2^15, which leaves a factor of two for what roundings add.  Norms that are not finite, or 0, give the ends
// of the range: the results are not numbers, or 0, whatever the factor.
__device__ __forceinline__ int ds_exp(float g2, float v2) {
  const int k = ((__float_as_int(0.25f * g2 * v2) >> 23) & 255) - 127;  // the bound's square is below 2^(k + 1)
  return min(60, 15 - ((k + 2) >> 1));
}
// the largest of n numbers >= 0; called by whole warps
__device__ __forceinline__ float warp_top(const float* p, int n) {
  float top = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x & 31; i < n; i += 32) top = fmaxf(top, p[i]);
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  return top;
}
// of all key tiles of a head; the dQ kernel leaves it for the dK/dV kernel, whose units may be shorter than that list
__device__ __forceinline__ float values_top(const CrossParams& P, int b, int hk) {
  const int n = static_cast<int>(P.Skp / CT), at = b * P.Hkv + hk;
  const float top = warp_top(P.v_top2 + static_cast<int64_t>(at) * n, n);
  if (threadIdx.x == 0) P.v_all2[at] = top;  // (every unit of the head writes the same number)
  return top;
}
__device__ __forceinline__ float rows_top(const CrossParams& P, int b, int hk) {
  return warp_top(P.g_top2 + (static_cast<int64_t>(b) * P.Hkv + hk) * P.q_tiles, P.q_tiles);
}

// ------------------------------------------------------------------------------------------------ row vectors
// -lse in units of log2 (-inf for tile rows outside the tensor and rows without keys; fp16: P_EXP more, so that what the kernels
// take from it is P 2^P_EXP) and delta = g . o, in tile order.  One row is DP / 8 lanes x 16 bytes; reads o and g once: HBM-bound.
// delta is left out (0) where the dQ kernel surely takes it from P and dP.  With a key mask the first B CTAs prepare it instead
// (a launch less).  fp16: also the squared norms of g, and in CTAs before these those of the values in use, which it reads once.
template <int N>
__device__ __forceinline__ float lanes_sum(float d) {
#pragma unroll
  for (int o = N / 2; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  return d;
}
// largest squared norm of a tile's values that are in use and finite (one that is not makes its results so by itself)
template <typename T, int DP>
__device__ __forceinline__ void tile_values_top(const CrossParams& P, const MaskArgs& mask, int unit) {
  constexpr int PER_ROW = DP / 8, ROWS = 256 / PER_ROW, PASSES = CT / ROWS;
  __shared__ float tops[8];
  int tile, hk;
  const int b = P.by_k_tiles.divmod(P.by_hkv.divmod(unit, hk), tile);
  const int64_t len = ca_len(mask.kv_lens, b, P.Sk);
  const int ch = threadIdx.x % PER_ROW * 8;
  const T* vb = static_cast<const T*>(P.v.ptr) + b * P.v.stride_b + hk * P.v.stride_h + ch;
  uint4 x[PASSES];
#pragma unroll
  for (int a = 0; a < PASSES; ++a) {
    const int64_t key = static_cast<int64_t>(tile) * CT + a * ROWS + threadIdx.x / PER_ROW;
    x[a] = make_uint4(0, 0, 0, 0);
    if (key < len && ch < P.D && !(mask.mask && ca_mask_value(mask, b * mask.ldm + key) == -INFINITY))
      x[a] = *reinterpret_cast<const uint4*>(vb + key * P.v.stride_s);
  }
  float top = 0.f;
#pragma unroll
  for (int a = 0; a < PASSES; ++a) {
    const T* xe = reinterpret_cast<const T*>(&x[a]);
    float d = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) d = fmaf(static_cast<float>(xe[e]), static_cast<float>(xe[e]), d);
    d = lanes_sum<PER_ROW>(d);
    if (d < INFINITY) top = fmaxf(top, d);
  }
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (float t : tops) top = fmaxf(top, t);
    P.v_top2[(static_cast<int64_t>(b) * P.Hkv + hk) * (P.Skp / CT) + tile] = top;
  }
}
template <typename T, int DP>
__global__ void __launch_bounds__(256) cross_stats_kernel(const CrossParams P, const MaskArgs mask) {
  constexpr int PER_ROW = DP / 8, ROWS = 256 / PER_ROW, PASSES = CT / ROWS;
  after_previous();
  int unit = blockIdx.x;
  if (mask.mask) {
    if (unit < P.B) {
      prepare_mask<256>(mask, unit);
      return;
    }
    unit -= P.B;
  }
  if constexpr (scaled<T>) {
    const int n = static_cast<int>(P.Skp / CT) * P.Hkv * P.B;
    if (unit < n) {
      tile_values_top<T, DP>(P, mask, unit);
      return;
    }
    unit -= n;
  }
  int tile, hk;  // key heads next to one another: CTAs that run together read the same stretch of memory
  const int b = P.by_q_tiles.divmod(P.by_hkv.divmod(unit, hk), tile);
  const bool need = P.splits > 1 || ca_len(mask.kv_lens, b, P.Sk) > CT;  // the lengths before the mask
  const int ch = threadIdx.x % PER_ROW * 8;
  const int64_t at = (static_cast<int64_t>(b) * P.Hkv + hk) * P.q_tiles + tile;
  float* st = P.stats + at * (2 * CT);
  const T* ob = static_cast<const T*>(P.o.ptr) + b * P.o.stride_b + ch;
  const T* gb = static_cast<const T*>(P.go.ptr) + b * P.go.stride_b + ch;
  uint4 ov[PASSES], gv[PASSES];
#pragma unroll
  for (int a = 0; a < PASSES; ++a) {
    int h;
    const int q = P.by_g.divmod(a * ROWS + threadIdx.x / PER_ROW, h);
    h += hk * P.G;
    const int64_t s = static_cast<int64_t>(tile) * P.nq + q;
    ov[a] = gv[a] = make_uint4(0, 0, 0, 0);
    if ((need || scaled<T>) && q < P.nq && s < P.Sq && ch < P.D) {
      if (need) ov[a] = *reinterpret_cast<const uint4*>(ob + s * P.o.stride_s + h * P.o.stride_h);
      gv[a] = *reinterpret_cast<const uint4*>(gb + s * P.go.stride_s + h * P.go.stride_h);
    }
  }
  float e = -INFINITY;  // of this thread's row, below
  if (threadIdx.x < CT) {
    int h;
    const int q = P.by_g.divmod(threadIdx.x, h);
    const int64_t s = static_cast<int64_t>(tile) * P.nq + q;
    if (q < P.nq && s < P.Sq) e = P.lse[(static_cast<int64_t>(b) * P.Hq + hk * P.G + h) * P.Sq + s];
    st[threadIdx.x] = e == -INFINITY ? -INFINITY : fmaf(-e, CA_LOG2E, scaled<T> ? P_EXP : 0.f);
  }
  __shared__ float norms[CT], tops[CT / 32];
#pragma unroll
  for (int a = 0; a < PASSES; ++a) {
    const T* oe = reinterpret_cast<const T*>(&ov[a]);
    const T* ge = reinterpret_cast<const T*>(&gv[a]);
    const int row = a * ROWS + threadIdx.x / PER_ROW;
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) d = fmaf(static_cast<float>(oe[i]), static_cast<float>(ge[i]), d);
    d = lanes_sum<PER_ROW>(d);
    if (threadIdx.x % PER_ROW == 0) st[CT + row] = d;
    if constexpr (scaled<T>) {
      float n = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) n = fmaf(static_cast<float>(ge[i]), static_cast<float>(ge[i]), n);
      n = lanes_sum<PER_ROW>(n);
      if (threadIdx.x % PER_ROW == 0) norms[row] = n;
    }
  }
  if constexpr (scaled<T>) {
    __syncthreads();
    if (threadIdx.x < CT) {
      const float n = norms[threadIdx.x];
      P.g_norm2[at * CT + threadIdx.x] = n;
      float top = e != -INFINITY && n < INFINITY ? n : 0.f;  // of rows that have keys
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    }
    __syncthreads();
    if (threadIdx.x == 0) P.g_top2[at] = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  }
}

// ------------------------------------------------------------------------------------------------ dQ
// What bounds the products here is the shared memory's bandwidth (two K-major operands there take all of it at N = 128), so a
// unit's Q and G tiles, the A operands of S and dP, are moved to tensor memory once: S dP dQ Q G = 512 columns.  dS goes over
// dP; the next S is issued as soon as S has been read, so it and the next dP run under the elementwise work.
template <typename T, int DP, bool BIAS>
__global__ void __launch_bounds__(BwdCfg<DP>::THREADS, 1)
    cross_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmG,
                    const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const CrossParams P) {
  using C = BwdCfg<DP>;
  constexpr int KS = 3, VS = 2;  // ring stages
  extern __shared__ __align__(1024) unsigned char ca_smem[];
  unsigned char* sQ = ca_smem;
  unsigned char* sG = sQ + C::TILE;
  unsigned char* sK = sG + C::TILE;
  unsigned char* sV = sK + KS * C::TILE;
  float* part = reinterpret_cast<float*>(sV + VS * C::TILE);  // [4][128] quarters of a row's delta
  uint64_t* q_full = reinterpret_cast<uint64_t*>(part + 4 * CT);
  uint64_t* q_empty = q_full + 1;
  uint64_t* g_full = q_empty + 1;
  uint64_t* g_empty = g_full + 1;
  uint64_t* k_full = g_empty + 1;
  uint64_t* k_empty = k_full + KS;
  uint64_t* k_clean = k_empty + KS;
  uint64_t* v_full = k_clean + KS;
  uint64_t* v_empty = v_full + VS;
  uint64_t* s_full = v_empty + VS;
  uint64_t* s_read = s_full + 1;
  uint64_t* qg_tmem = s_read + 1;
  uint64_t* dp_full = qg_tmem + 1;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* part_full = ds_full + 1;
  uint64_t* dq_full = part_full + 1;
  uint64_t* dq_empty = dq_full + 1;
  uint64_t* done = dq_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  signed char* row_exp = reinterpret_cast<signed char*>(tmem_slot + 2);  // fp16: [unit & 1][128] ds_exp of the rows

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const bool masked = BIAS || P.kv_lens != nullptr;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 16);
    mbar_init(g_full, 1);
    mbar_init(g_empty, 16);
    for (int s = 0; s < KS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&k_clean[s], 1);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_read, 16);
    mbar_init(qg_tmem, 16);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 16);
    mbar_init(part_full, 16);
    mbar_init(dq_full, 1);
    mbar_init(dq_empty, 4);
    mbar_init(done, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmG);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 20) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  after_previous();
  const uint32_t tDP = tmem + CT, tDQ = tmem + 2 * CT, tQ = tmem + 3 * CT, tG = tQ + 64;  // S dP dQ Q G

  if (warp < 16) {
    // ------------------------------------------------------------------------------------------ P, dS
    regs_inc<96>();
    const int quarter = warp >> 2, row = threadIdx.x & (CT - 1);
    const uint32_t at = (static_cast<uint32_t>(warp & 3) << 21) + quarter * 32;  // this warp's lanes and columns
    uint32_t ph = 0, xph = 0, uph = 0;
    float nlse2 = -INFINITY, delta = 0.f;
    float c = 1.f;  // fp16: what P 2^P_EXP (dP - delta) is multiplied by
    int exp = 0, slot = 0;
    bool ok = true;
    int64_t len = 0;
    float* stat = nullptr;
    for (BwdWalk<true> w(P); ok && w.valid; w.next()) {
      const BwdTile& u = w.c;
      const bool one_tile = P.splits == 1 && u.t1 - u.t0 == 1;
      if (u.first()) {
        len = ca_len(P.kv_lens, u.b, P.Sk);
        stat = P.stats + ((static_cast<int64_t>(u.b) * P.Hkv + u.hk) * P.q_tiles + u.tile) * (2 * CT);
        nlse2 = stat[row];  // -inf for rows outside and rows without keys: every p is 0
        delta = stat[CT + row];
        if constexpr (scaled<T>) {
          const float g2 = P.g_norm2[((static_cast<int64_t>(u.b) * P.Hkv + u.hk) * P.q_tiles + u.tile) * CT + row];
          exp = ds_exp(g2, values_top(P, u.b, u.hk));
          c = pow2(exp - P_EXP);
        }
        // Q and G to tensor memory, this warp's 32 rows and quarter of the channels; the products of the unit before that
        // read them there are complete (its last S and dP have been waited for)
#pragma unroll 1
        for (int m = 0; m < 2; ++m) {
          if (!(ok = warp_wait(m ? g_full : q_full, uph, abort_flag))) break;
          const unsigned char* tile = m ? sG : sQ;
          uint32_t v[DP / 8];
#pragma unroll
          for (int i = 0; i < DP / 32; ++i) {
            const int ch = quarter * (DP / 4) + 8 * i;
            const uint4 x = *reinterpret_cast<const uint4*>(tile + (ch >> 6) * SUB_BYTES + row * 128 + ((((ch & 63) >> 3) ^ (row & 7)) << 4));
            v[4 * i] = x.x, v[4 * i + 1] = x.y, v[4 * i + 2] = x.z, v[4 * i + 3] = x.w;
          }
          const uint32_t dst = (m ? tG : tQ) + (static_cast<uint32_t>(warp & 3) << 21) + quarter * (DP / 8);
          if constexpr (DP == 128) tmem_st_32x32b_x16(dst, v);
          else tmem_st_32x32b_x8(dst, v);
          __syncwarp();
          if (lane == 0) mbar_arrive(m ? g_empty : q_empty);
        }
        if (!ok) break;
        uph ^= 1;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(qg_tmem);
      }
      if (!(ok = warp_wait(s_full, ph, abort_flag))) break;
      tc_fence_after();
      if (scaled<T> && u.first()) {  // (this S was issued after the epilogue had taken the unit before the last, and with it its slot)
        if (quarter == 0) row_exp[slot * CT + row] = static_cast<signed char>(exp);
        slot ^= 1;
      }
      float p[32];
      uint32_t r[32];
      tmem_ld_32x32b_x32(tmem + at, r);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_read);
      if constexpr (BIAS) {
        const float4* b4 = reinterpret_cast<const float4*>(P.bias2 + u.b * P.Skp + static_cast<int64_t>(u.t) * CT + quarter * 32);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 bb = b4[i];
          const float bv[4] = {bb.x, bb.y, bb.z, bb.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = ex2(fmaf(__uint_as_float(r[4 * i + e]), P.scale2, bv[e] + nlse2));
            p[4 * i + e] = bv[e] == -INFINITY ? 0.f : x;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; i += 4) {  // every other pair through the FMA pipe's exp2
          const f32x2 sc = f2(P.scale2, P.scale2), n2 = f2(nlse2, nlse2);
          float xa, xb, xc, xd;
          f2_split(f2_fma(f2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), sc, n2), xa, xb);
          f2_split(f2_fma(f2(__uint_as_float(r[i + 2]), __uint_as_float(r[i + 3])), sc, n2), xc, xd);
          p[i] = ex2(xa), p[i + 1] = ex2(xb);
          f2_split(f2_exp2<true>(xc, xd), p[i + 2], p[i + 3]);
        }
        const int64_t lim = len - (static_cast<int64_t>(u.t) * CT + quarter * 32);  // columns in use, from this warp's first
        if (lim < 32) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (i >= lim) p[i] = 0.f;
        }
      }
      if (nlse2 == -INFINITY) {  // also when the row's own scores are not numbers
#pragma unroll
        for (int i = 0; i < 32; ++i) p[i] = 0.f;
      }
      if (!(ok = warp_wait(dp_full, ph, abort_flag))) break;
      ph ^= 1;
      tc_fence_after();
      tmem_ld_32x32b_x32(tDP + at, r);
      tmem_ld_wait();
      if (masked) {  // a masked key's dP may be anything
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (p[i] == 0.f) r[i] = 0;
      }
      if (u.first()) {
        if (one_tile) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 32; ++i) d[i & 3] = fmaf(p[i], __uint_as_float(r[i]), d[i & 3]);
          // (the next unit's dP, which its quarters come from, is issued after every warp has handed in this unit's dS)
          part[quarter * CT + row] = (d[0] + d[1]) + (d[2] + d[3]);
          __syncwarp();
          if (lane == 0) mbar_arrive(part_full);
          if (!(ok = warp_wait(part_full, xph, abort_flag))) break;
          xph ^= 1;
          delta = (part[row] + part[CT + row]) + (part[2 * CT + row] + part[3 * CT + row]);
          if constexpr (scaled<T>) delta *= pow2(-P_EXP);
          // (rows that no query fills have 0 x whatever shared memory held; the dK/dV kernel multiplies by what is written here)
          if (nlse2 == -INFINITY) delta = 0.f;
          if (quarter == 0) stat[CT + row] = delta;
        }
      }
      uint32_t pk[16];
      const float cd = -delta * c;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if constexpr (scaled<T>) {  // c is a power of two: the same rounding as of dP - delta
          float da, db;
          const f32x2 d = f2_fma(f2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), f2(c, c), f2(cd, cd));
          f2_split(f2_mul(f2(p[2 * i], p[2 * i + 1]), d), da, db);
          pk[i] = pack2<T>(da, db);
        } else {
          pk[i] = pack2<T>(p[2 * i] * (__uint_as_float(r[2 * i]) - delta), p[2 * i + 1] * (__uint_as_float(r[2 * i + 1]) - delta));
        }
      }
      tmem_st_32x32b_x16(tDP + at, pk);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
  } else if (warp < 20) {
    // ------------------------------------------------------------------------------------------ epilogue
    regs_dec<48>();
    const int row = threadIdx.x & (CT - 1);
    int hg;
    const int qr = P.by_g.divmod(row, hg);
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
    uint32_t ph = 0;
    int slot = 0;
    bool ok = true;
    BwdWalk<true> w(P);
    BwdTile u;
    for (int it = blockIdx.x; ok && it < w.n; it += gridDim.x) {
      w.unit(it, u);
      const int64_t s = static_cast<int64_t>(u.tile) * P.nq + qr;
      const bool valid = qr < P.nq && s < P.Sq, any = u.t1 > u.t0;
      if (any) {
        if (!(ok = warp_wait(dq_full, ph, abort_flag))) break;
        ph ^= 1;
        tc_fence_after();
      }
      const int64_t rid = (static_cast<int64_t>(u.b) * P.Hq + u.hk * P.G + hg) * P.Sq + s;
      T* dst = static_cast<T*>(P.dq.ptr) + u.b * P.dq.stride_b + s * P.dq.stride_s + (u.hk * P.G + hg) * P.dq.stride_h;
      float* dst32 = P.part_dq + (static_cast<int64_t>(u.split) * P.B * P.Hq * P.Sq + rid) * P.D;
      float f = P.scale;
      if (scaled<T> && any) {
        f *= pow2(-row_exp[slot * CT + row]);
        slot ^= 1;
      }
#pragma unroll 1
      for (int c = 0; c < DP / 16; ++c) {
        uint32_t o[16];
        if (any) {
          tmem_ld_32x32b_x16(tDQ + lanes + 16 * c, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = 0;
        }
        if (!valid) continue;
        if (P.splits > 1) store_cols_f32(dst32 + 16 * c, o, f, P.D - 16 * c);
        else store_cols<T>(dst + 16 * c, o, f, P.D - 16 * c, P.wide);
      }
      if (any) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dq_empty);
      }
    }
  } else {
    regs_dec<48>();
    if (warp == 20) {
      // -------------------------------------------------------------------------------------- MMA issue
      constexpr uint32_t idS = idesc_f16<T>(CT, CT, false), idD = idesc_f16<T>(CT, DP, true);
      constexpr uint32_t TILE16 = C::TILE >> 4;
      const uint32_t rK = desc_rows(smem_u32(sK)), rV = desc_rows(smem_u32(sV)), cK = desc_chan(smem_u32(sK));
      BwdCount<true> ws(P), wp(P), wd(P);  // the next S, dP and dQ product
      int sk = 0, pv = 0, dk = 0;
      uint32_t skph = 0, pvph = 0, srph = 1, uph = 0, dsph = 0, dqph = 1;
      bool ok = true;
      auto do_s = [&] {
        if (!ok) return;
        if (!(ok = warp_wait(&k_full[sk], skph, abort_flag))) return;
        if (masked && !(ok = warp_wait(&k_clean[sk], skph, abort_flag))) return;
        if (!(ok = warp_wait(s_read, srph, abort_flag))) return;  // the S before has been read
        srph ^= 1;
        if (ws.first) {
          if (!(ok = warp_wait(qg_tmem, uph, abort_flag))) return;
          uph ^= 1;
        }
        tc_fence_after();
        mma_rows_ta<DP / 16>(tmem, tQ, rK + sk * TILE16, idS);
        commit_one(s_full);
        if (++sk == KS) sk = 0, skph ^= 1;
        ws.next();
      };
      auto do_dp = [&] {
        if (!ok) return;
        if (!(ok = warp_wait(&v_full[pv], pvph, abort_flag))) return;
        tc_fence_after();
        mma_rows_ta<DP / 16>(tDP, tG, rV + pv * TILE16, idS);
        commit_one(dp_full);
        commit_one(&v_empty[pv]);
        if (++pv == VS) pv = 0, pvph ^= 1;
        wp.next();
      };
      while (ok && wd.valid()) {
        if (wd.first) {  // a unit begins: its Q and G are in tensor memory once the one before is through
          do_s();
          do_dp();
          if (ws.valid() && ws.it == wd.it) do_s();
        }
        if (!ok || !(ok = warp_wait(ds_full, dsph, abort_flag))) break;  // dS is written, dP has been read
        dsph ^= 1;
        if (wd.first) {
          if (!(ok = warp_wait(dq_empty, dqph, abort_flag))) break;
          dqph ^= 1;
        }
        tc_fence_after();
        mma_chan<4>(tDQ, tDP, cK + dk * TILE16, idD, !wd.first);
        commit_one(&k_empty[dk]);
        if (wd.last()) commit_one(dq_full);
        if (++dk == KS) dk = 0;
        wd.next();
        if (wd.valid() && !wd.first) {
          do_dp();
          if (ws.valid() && ws.it == wd.it) do_s();
        }
      }
    } else if (warp == 21) {
      if (lane == 0) {
        // -------------------------------------------------------------------------------------- copies
        int k = 0, v = 0, kfills = 0, vfills = 0, qfills = 0, gfills = 0;
        uint32_t kph = 1, vph = 1, qph = 1, gph = 1;
        bool ok = true;
        const uint32_t q_bytes = static_cast<uint32_t>(C::NSUB * 128 * P.G * P.nq);
        BwdWalk<true> w(P);
        auto prefetch = [&](int it) {  // Q and G tiles of a unit to come into L2
          if (it >= w.n) return;
          BwdTile nx;
          w.unit(it, nx);
          for (int p = 0; p < C::NSUB; ++p) {
            tma_prefetch_5d(&tmG, 64 * p, 0, nx.hk, nx.tile * P.nq, nx.b);
            tma_prefetch_5d(&tmQ, 64 * p, 0, nx.hk, nx.tile * P.nq, nx.b);
          }
        };
        for (; ok && w.valid; w.next()) {
          const BwdTile& u = w.c;
          if (u.first()) {
            if (!(ok = mbar_wait(q_empty, qph, abort_flag))) break;
            qph ^= 1;
            mbar_arrive_expect_tx(q_full, q_bytes);
            for (int p = 0; p < C::NSUB; ++p) tma_load_5d(sQ + p * SUB_BYTES, &tmQ, q_full, 64 * p, 0, u.hk, u.tile * P.nq, u.b);
            ++qfills;
          }
          if (!(ok = mbar_wait(&k_empty[k], kph, abort_flag))) break;
          mbar_arrive_expect_tx(&k_full[k], C::TILE);
          for (int p = 0; p < C::NSUB; ++p) tma_load_4d(sK + k * C::TILE + p * SUB_BYTES, &tmK, &k_full[k], 64 * p, u.hk, u.t * CT, u.b);
          ++kfills;
          if (++k == KS) k = 0, kph ^= 1;
          if (u.first()) {
            if (!(ok = mbar_wait(g_empty, gph, abort_flag))) break;
            gph ^= 1;
            mbar_arrive_expect_tx(g_full, q_bytes);
            for (int p = 0; p < C::NSUB; ++p) tma_load_5d(sG + p * SUB_BYTES, &tmG, g_full, 64 * p, 0, u.hk, u.tile * P.nq, u.b);
            ++gfills;
            prefetch(u.it + static_cast<int>(gridDim.x));
          }
          if (!(ok = mbar_wait(&v_empty[v], vph, abort_flag))) break;
          mbar_arrive_expect_tx(&v_full[v], C::TILE);
          for (int p = 0; p < C::NSUB; ++p) tma_load_4d(sV + v * C::TILE + p * SUB_BYTES, &tmV, &v_full[v], 64 * p, u.hk, u.t * CT, u.b);
          ++vfills;
          if (++v == VS) v = 0, vph ^= 1;
        }
        auto drain = [](uint64_t* bars, int stages, int fills) {  // copies in flight land before the memory goes away
          for (int j = fills > stages ? fills - stages : 0; j < fills; ++j)
            if (!mbar_wait_drain(&bars[j % stages], static_cast<uint32_t>((j / stages) & 1))) break;
        };
        drain(k_full, KS, kfills);
        drain(v_full, VS, vfills);
        drain(q_full, 1, qfills);
        drain(g_full, 1, gfills);
      }
      __syncwarp();
    } else if (warp == 22 && masked) {
      // ---------------------------------------------------------------------------------------- rows of masked keys
      int k = 0;
      uint32_t kph = 0;
      for (BwdWalk<true> w(P); w.valid; w.next()) {
        const BwdTile& u = w.c;
        if (!warp_wait(&k_full[k], kph, abort_flag)) break;
        const int64_t len = ca_len(P.kv_lens, u.b, P.Sk);
        if (BIAS || (len < P.Sk && static_cast<int64_t>(u.t + 1) * CT > len)) {
          for (int j = lane; j < CT; j += 32) {
            const int64_t key = static_cast<int64_t>(u.t) * CT + j;
            if (key >= len || (BIAS && P.bias2[u.b * P.Skp + key] == -INFINITY))
              for (int p = 0; p < C::NSUB; ++p)
                for (int c = 0; c < 8; ++c)
                  *reinterpret_cast<uint4*>(sK + k * C::TILE + p * SUB_BYTES + j * 128 + c * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(&k_clean[k]);
        if (++k == KS) k = 0, kph ^= 1;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 20) {
    tc_fence_after();
    commit_one(done);
    mbar_wait_drain(done, 0);
    __syncwarp();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------------------------ dK, dV
// Q and G arrive in rings (K and V stay): Q 3 stages, because dK's product, the last of a query tile, reads it; G 2.  11840
// queries x 40 heads x 128 channels: 122 us over 256 keys, 795 over 2048 (4 products: 1250 TFLOP/s); dQ there 112 and 605
// (3 products: 1230).
template <typename T, int DP, bool BIAS>
__global__ void __launch_bounds__(BwdCfg<DP>::THREADS, 1)
    cross_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmG,
                     const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const CrossParams P) {
  using C = BwdCfg<DP>;
  constexpr int QS = 3, GS = 2, TS = 2;  // ring stages: Q and G tiles, row vectors
  extern __shared__ __align__(1024) unsigned char ca_smem[];
  unsigned char* sK = ca_smem;
  unsigned char* sV = sK + C::TILE;
  unsigned char* sQ = sV + C::TILE;
  unsigned char* sG = sQ + QS * C::TILE;
  float* sT = reinterpret_cast<float*>(sG + GS * C::TILE);  // [TS][-lse, delta][128]
  uint64_t* k_full = reinterpret_cast<uint64_t*>(sT + TS * 2 * CT);
  uint64_t* k_empty = k_full + 1;
  uint64_t* v_full = k_empty + 1;
  uint64_t* v_empty = v_full + 1;
  uint64_t* q_full = v_empty + 1;
  uint64_t* q_empty = q_full + QS;
  uint64_t* g_full = q_empty + QS;
  uint64_t* g_empty = g_full + GS;
  uint64_t* t_full = g_empty + GS;
  uint64_t* t_empty = t_full + TS;
  uint64_t* s_full = t_empty + TS;
  uint64_t* p_full = s_full + 1;
  uint64_t* dp_full = p_full + 1;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* acc_full = ds_full + 1;
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* done = acc_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* unit_exp = reinterpret_cast<int*>(tmem_slot + 2);  // fp16: [unit & 1] ds_exp of a unit

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(k_full, 1);
    mbar_init(k_empty, 1);
    mbar_init(v_full, 1);
    mbar_init(v_empty, 1);
    for (int s = 0; s < QS; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
    }
    for (int s = 0; s < GS; ++s) {
      mbar_init(&g_full[s], 1);
      mbar_init(&g_empty[s], 1);
    }
    for (int s = 0; s < TS; ++s) {
      mbar_init(&t_full[s], 1);
      mbar_init(&t_empty[s], 16);
    }
    mbar_init(s_full, 1);
    mbar_init(p_full, 16);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 16);
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 4);
    mbar_init(done, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmG);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  // rows of the query tiles that no copy writes (128 is not a multiple of G): their products have weight 0, but 0 x NaN
  for (int i = threadIdx.x; i < (QS + GS) * C::NSUB * (CT - P.G * P.nq) * 8; i += blockDim.x) {
    const int rows = CT - P.G * P.nq, c = i & 7, r = (i >> 3) % rows, p = (i >> 3) / rows;
    *reinterpret_cast<uint4*>(sQ + p * SUB_BYTES + (P.G * P.nq + r) * 128 + c * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  if (warp == 20) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  after_previous();
  const uint32_t tDP = tmem + CT, tDV = tmem + 2 * CT, tDK = tmem + 3 * CT;  // S dP dV dK

  if (warp < 16) {
    // ------------------------------------------------------------------------------------------ P^T, dS^T
    regs_inc<96>();
    const int quarter = warp >> 2, row = threadIdx.x & (CT - 1);
    const uint32_t at = (static_cast<uint32_t>(warp & 3) << 21) + quarter * 32;
    uint32_t ph = 0, tph = 0;
    int ts = 0;
    bool ok = true, live = false;
    float rb = 0.f, c = 1.f;  // c: as for dQ, one for all rows
    int exp = 0, slot = 0;
    for (BwdWalk<false> w(P); ok && w.valid; w.next()) {
      const BwdTile& u = w.c;
      if (u.first()) {
        const int64_t key = static_cast<int64_t>(u.tile) * CT + row;
        live = key < ca_len(P.kv_lens, u.b, P.Sk);
        if constexpr (BIAS) {
          rb = P.bias2[u.b * P.Skp + key];
          live = live && rb != -INFINITY;
        }
        if constexpr (scaled<T>) {
          exp = ds_exp(rows_top(P, u.b, u.hk), P.v_all2[u.b * P.Hkv + u.hk]);
          c = pow2(exp - P_EXP);
        }
      }
      if (!(ok = warp_wait(&t_full[ts], tph, abort_flag))) break;
      if (!(ok = warp_wait(s_full, ph, abort_flag))) break;
      tc_fence_after();
      if (scaled<T> && u.first()) {  // (as for dQ)
        if (threadIdx.x == 0) unit_exp[slot] = exp;
        slot ^= 1;
      }
      const float4* nl = reinterpret_cast<const float4*>(sT + ts * 2 * CT + quarter * 32);
      const float4* dl = reinterpret_cast<const float4*>(sT + ts * 2 * CT + CT + quarter * 32);
      float p[32];
      uint32_t r[32], pk[16];
      const f32x2 sc = f2(P.scale2, P.scale2);
      tmem_ld_32x32b_x32(tmem + at, r);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // every other pair through the FMA pipe's exp2: this phase is what the products wait for
        const float4 n4 = nl[i];
        f32x2 na = f2(n4.x, n4.y), nb = f2(n4.z, n4.w);
        if constexpr (BIAS) na = f2_add(na, f2(rb, rb)), nb = f2_add(nb, f2(rb, rb));
        float xa, xb, xc, xd;
        f2_split(f2_fma(f2(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1])), sc, na), xa, xb);
        f2_split(f2_fma(f2(__uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3])), sc, nb), xc, xd);
        p[4 * i] = ex2(xa), p[4 * i + 1] = ex2(xb);
        f2_split(f2_exp2<true>(xc, xd), p[4 * i + 2], p[4 * i + 3]);
      }
      if (!live) {  // this row's key is out: whatever its scores were
#pragma unroll
        for (int i = 0; i < 32; ++i) p[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) pk[i] = pack2<T>(p[2 * i], p[2 * i + 1]);
      tmem_st_32x32b_x16(tmem + at, pk);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
      if (!(ok = warp_wait(dp_full, ph, abort_flag))) break;
      tc_fence_after();
      tmem_ld_32x32b_x32(tDP + at, r);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 d4 = dl[i];
        const float dv[4] = {d4.x, d4.y, d4.z, d4.w};
        if constexpr (scaled<T>) {  // c is a power of two: the same rounding as of dP - delta
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const int k = 4 * i + e;
            const f32x2 d = f2_fma(f2(__uint_as_float(r[k]), __uint_as_float(r[k + 1])), f2(c, c), f2_mul(f2(dv[e], dv[e + 1]), f2(-c, -c)));
            f2_split(f2_mul(f2(p[k], p[k + 1]), d), p[k], p[k + 1]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) p[4 * i + e] *= __uint_as_float(r[4 * i + e]) - dv[e];
        }
      }
      if (!live) {
#pragma unroll
        for (int i = 0; i < 32; ++i) p[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) pk[i] = pack2<T>(p[2 * i], p[2 * i + 1]);
      tmem_st_32x32b_x16(tDP + at, pk);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(ds_full);
        mbar_arrive(&t_empty[ts]);
      }
      ph ^= 1;
      if (++ts == TS) ts = 0, tph ^= 1;
    }
  } else if (warp < 20) {
    // ------------------------------------------------------------------------------------------ epilogue
    regs_dec<48>();
    const int row = threadIdx.x & (CT - 1);
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
    uint32_t ph = 0;
    int slot = 0;
    BwdWalk<false> w(P);
    BwdTile u;
    bool ok = true;
    const int64_t part = static_cast<int64_t>(P.B) * P.Hkv * P.Sk * P.D;  // elements of one split's dK or dV
    for (int it = blockIdx.x; ok && it < w.n; it += gridDim.x) {
      w.unit(it, u);
      const int64_t key = static_cast<int64_t>(u.tile) * CT + row;
      const bool valid = key < P.Sk, any = u.t1 > u.t0;
      if (any) {
        if (!(ok = warp_wait(acc_full, ph, abort_flag))) break;
        ph ^= 1;
        tc_fence_after();
      }
      T* dk = static_cast<T*>(P.dk.ptr) + u.b * P.dk.stride_b + key * P.dk.stride_s + u.hk * P.dk.stride_h;
      T* dv = static_cast<T*>(P.dv.ptr) + u.b * P.dv.stride_b + key * P.dv.stride_s + u.hk * P.dv.stride_h;
      float f_k = P.scale, f_v = 1.f;
      if (scaled<T> && any) {
        f_k *= pow2(-unit_exp[slot]);
        slot ^= 1;
        f_v = pow2(-P_EXP);
      }
      float* dk32 = P.part_dk + u.split * 2 * part + ((static_cast<int64_t>(u.b) * P.Hkv + u.hk) * P.Sk + key) * P.D;
#pragma unroll 1
      for (int c = 0; c < 2 * (DP / 16); ++c) {
        const bool is_k = c >= DP / 16;
        const int col = 16 * (is_k ? c - DP / 16 : c);
        uint32_t o[16];
        if (any) {
          tmem_ld_32x32b_x16((is_k ? tDK : tDV) + lanes + col, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = 0;
        }
        if (!valid) continue;
        const float f = is_k ? f_k : f_v;
        if (P.kv_splits > 1) store_cols_f32(dk32 + (is_k ? 0 : part) + col, o, f, P.D - col);
        else store_cols<T>((is_k ? dk : dv) + col, o, f, P.D - col, P.wide);
      }
      if (any) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty);
      }
    }
  } else {
    regs_dec<48>();
    if (warp == 20) {
      // -------------------------------------------------------------------------------------- MMA issue
      constexpr uint32_t idS = idesc_f16<T>(CT, CT, false), idD = idesc_f16<T>(CT, DP, true);
      constexpr uint32_t TILE16 = C::TILE >> 4;
      const uint32_t rQ = desc_rows(smem_u32(sQ)), rG = desc_rows(smem_u32(sG)), rK = desc_rows(smem_u32(sK)),
                     rV = desc_rows(smem_u32(sV));
      const uint32_t cQ = desc_chan(smem_u32(sQ)), cG = desc_chan(smem_u32(sG));
      BwdCount<false> ws(P), wp(P), wd(P);  // the next S^T, dP^T, and the tile in hand
      int sq = 0, pg = 0, dq = 0, dg = 0;
      uint32_t sqph = 0, pgph = 0, kph = 0, vph = 0, ph = 0, aph = 1;
      bool ok = true;
      auto do_s = [&] {
        if (!ok || !ws.valid()) return;
        if (ws.first) {
          if (!(ok = warp_wait(k_full, kph, abort_flag))) return;
          kph ^= 1;
        }
        if (!(ok = warp_wait(&q_full[sq], sqph, abort_flag))) return;
        tc_fence_after();
        mma_rows<DP / 16>(tmem, rK, rQ + sq * TILE16, idS);
        commit_one(s_full);
        if (ws.last()) commit_one(k_empty);
        if (++sq == QS) sq = 0, sqph ^= 1;
        ws.next();
      };
      auto do_dp = [&] {
        if (!ok || !wp.valid()) return;
        if (wp.first) {
          if (!(ok = warp_wait(v_full, vph, abort_flag))) return;
          vph ^= 1;
        }
        if (!(ok = warp_wait(&g_full[pg], pgph, abort_flag))) return;
        tc_fence_after();
        mma_rows<DP / 16>(tDP, rV, rG + pg * TILE16, idS);
        commit_one(dp_full);
        if (wp.last()) commit_one(v_empty);
        if (++pg == GS) pg = 0, pgph ^= 1;
        wp.next();
      };
      do_s();
      do_dp();
      while (ok && wd.valid()) {
        const uint32_t acc = !wd.first;
        const bool last = wd.last();
        if (!(ok = warp_wait(p_full, ph, abort_flag))) break;
        if (!acc) {
          if (!(ok = warp_wait(acc_empty, aph, abort_flag))) break;
          aph ^= 1;
        }
        tc_fence_after();
        mma_chan<4>(tDV, tmem, cG + dg * TILE16, idD, acc);
        commit_one(&g_empty[dg]);
        if (++dg == GS) dg = 0;
        do_s();
        if (!ok || !(ok = warp_wait(ds_full, ph, abort_flag))) break;
        tc_fence_after();
        mma_chan<4>(tDK, tDP, cQ + dq * TILE16, idD, acc);
        commit_one(&q_empty[dq]);
        if (last) commit_one(acc_full);
        if (++dq == QS) dq = 0;
        do_dp();
        ph ^= 1;
        wd.next();
      }
    } else if (warp == 21) {
      if (lane == 0) {
        // -------------------------------------------------------------------------------------- copies
        int q = 0, g = 0, ts = 0, qfills = 0, gfills = 0, tfills = 0, kfills = 0, vfills = 0;
        uint32_t qph = 1, gph = 1, tph = 1, uph = 1;
        bool ok = true;
        const uint32_t q_bytes = static_cast<uint32_t>(C::NSUB * 128 * P.G * P.nq);
        for (BwdWalk<false> w(P); ok && w.valid; w.next()) {
          const BwdTile& u = w.c;
          if (u.first()) {
            if (!(ok = mbar_wait(k_empty, uph, abort_flag))) break;
            mbar_arrive_expect_tx(k_full, C::TILE);
            for (int p = 0; p < C::NSUB; ++p) tma_load_4d(sK + p * SUB_BYTES, &tmK, k_full, 64 * p, u.hk, u.tile * CT, u.b);
            ++kfills;
          }
          if (!(ok = mbar_wait(&q_empty[q], qph, abort_flag))) break;
          mbar_arrive_expect_tx(&q_full[q], q_bytes);
          for (int p = 0; p < C::NSUB; ++p) tma_load_5d(sQ + q * C::TILE + p * SUB_BYTES, &tmQ, &q_full[q], 64 * p, 0, u.hk, u.t * P.nq, u.b);
          ++qfills;
          if (++q == QS) q = 0, qph ^= 1;
          if (!(ok = mbar_wait(&t_empty[ts], tph, abort_flag))) break;
          mbar_arrive_expect_tx(&t_full[ts], 2 * CT * 4);
          bulk_load(sT + ts * 2 * CT, P.stats + ((static_cast<int64_t>(u.b) * P.Hkv + u.hk) * P.q_tiles + u.t) * (2 * CT), 2 * CT * 4,
                    &t_full[ts]);
          ++tfills;
          if (++ts == TS) ts = 0, tph ^= 1;
          if (u.first()) {
            if (!(ok = mbar_wait(v_empty, uph, abort_flag))) break;
            uph ^= 1;
            mbar_arrive_expect_tx(v_full, C::TILE);
            for (int p = 0; p < C::NSUB; ++p) tma_load_4d(sV + p * SUB_BYTES, &tmV, v_full, 64 * p, u.hk, u.tile * CT, u.b);
            ++vfills;
          }
          if (!(ok = mbar_wait(&g_empty[g], gph, abort_flag))) break;
          mbar_arrive_expect_tx(&g_full[g], q_bytes);
          for (int p = 0; p < C::NSUB; ++p) tma_load_5d(sG + g * C::TILE + p * SUB_BYTES, &tmG, &g_full[g], 64 * p, 0, u.hk, u.t * P.nq, u.b);
          ++gfills;
          if (++g == GS) g = 0, gph ^= 1;
        }
        auto drain = [](uint64_t* bars, int stages, int fills) {  // copies in flight land before the memory goes away
          for (int j = fills > stages ? fills - stages : 0; j < fills; ++j)
            if (!mbar_wait_drain(&bars[j % stages], static_cast<uint32_t>((j / stages) & 1))) break;
        };
        drain(q_full, QS, qfills);
        drain(g_full, GS, gfills);
        drain(t_full, TS, tfills);
        drain(k_full, 1, kfills);
        drain(v_full, 1, vfills);
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 20) {
    tc_fence_after();
    commit_one(done);
    mbar_wait_drain(done, 0);
    __syncwarp();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// Adds up the splits' partial gradients in order and rounds once.  Four channels per thread; `rows` rows of D channels,
// row -> (b, h, s) with H heads and S rows (dQ: Hq, Sq; dK and dV: Hkv, Sk); the second tensor (blockIdx.y = 1) follows the
// first in every split.  HBM-bound: reads the splits' sums (fp32) once.
template <typename T>
__global__ void __launch_bounds__(256) cross_join_kernel(const float* part, int64_t stride, int splits, int64_t rows, int D,
                                                         int64_t S, int H, h3b_attn_tensor out0, h3b_attn_tensor out1) {
  after_previous();
  const int per = D / 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= rows * per) return;
  const h3b_attn_tensor& out = blockIdx.y ? out1 : out0;
  const int64_t row = i / per;
  const int c = static_cast<int>(i - row * per) * 4;
  const float* src = part + (blockIdx.y * rows + row) * D + c;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < splits; ++s) {
    const float4 v = *reinterpret_cast<const float4*>(src + s * stride);
    a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
  }
  const int64_t s = row % S, bh = row / S, h = bh % H, b = bh / H;
  *reinterpret_cast<uint2*>(static_cast<T*>(out.ptr) + b * out.stride_b + s * out.stride_s + h * out.stride_h + c) =
      make_uint2(pack2<T>(a.x, a.y), pack2<T>(a.z, a.w));
}
template <typename T>
static int join_launch(const float* part, int splits, int64_t rows, int D, int64_t S, int H, const h3b_attn_tensor& out0,
                       const h3b_attn_tensor* out1, cudaStream_t st) {
  const int n = out1 ? 2 : 1;
  const dim3 grid(static_cast<unsigned>((rows * (D / 4) + 255) / 256), n);
  return cross_launch_after("cross_join_kernel", cross_join_kernel<T>, grid, 256, 0, st, part, n * rows * D, splits, rows, D, S,
                            H, out0, out1 ? *out1 : out0);
}

// Splits of the other side's tiles for `units` units of `tiles` tiles each: least time of the busiest SM, in tiles (a unit
// costs about two more to fill and drain; splitting at all about three for the second kernel).
static int bwd_splits(int64_t units, int64_t tiles) {
  const int sms = cross_sms();
  if (units >= 2 * sms || tiles <= 1) return 1;
  int best = 1;
  int64_t best_cost = (units + sms - 1) / sms * (tiles + 2);
  for (int s = 2; s <= 64 && s <= tiles; ++s) {
    const int64_t cost = (units * s + sms - 1) / sms * ((tiles + s - 1) / s + 2) + 3;
    if (cost < best_cost) best = s, best_cost = cost;
  }
  return best;
}

template <typename T, int DP, bool BIAS>
static int bwd_launch_cfg(const CrossParams& P, const MaskArgs& mask, cudaStream_t st) {
  using C = BwdCfg<DP>;
  CUtensorMap q, g, k, v;
  const bool half = std::is_same_v<T, __half>;
  int rc = cross_map_q(&q, P, P.Sq > 0 ? P.q : cross_stand_in(P.k), half);
  if (!rc) rc = cross_map_q(&g, P, P.Sq > 0 ? P.go : cross_stand_in(P.k), half);
  if (!rc) rc = cross_map_k(&k, P, P.Sk > 0 ? P.k : cross_stand_in(P.q), half);
  if (!rc) rc = cross_map_k(&v, P, P.Sk > 0 ? P.v : cross_stand_in(P.q), half);
  if (rc) return rc;
  const int sms = cross_sms();
  auto kq = cross_dq_kernel<T, DP, BIAS>;
  auto kkv = cross_dkv_kernel<T, DP, BIAS>;
  static std::atomic<bool> ready_q[CA_DEVICES], ready_kv[CA_DEVICES];
  rc = cross_smem(reinterpret_cast<const void*>(kq), C::SMEM, ready_q, "cross_dq_kernel shared memory");
  if (!rc) rc = cross_smem(reinterpret_cast<const void*>(kkv), C::SMEM, ready_kv, "cross_dkv_kernel shared memory");
  if (rc) return rc;
  if (P.Sq > 0) {
    const int64_t n = static_cast<int64_t>(P.q_tiles) * P.splits * P.Hkv * P.B, rows = static_cast<int64_t>(P.B) * P.Hq * P.Sq;
    const int64_t tiles = (P.q_tiles + (scaled<T> ? P.Skp / CT : 0)) * P.Hkv * P.B;
    if (n >= (1 << 30) || tiles >= (1 << 30)) return fail(H3B_ERR_UNSUPPORTED, "cross_attention_backward: too many tiles");
    rc = cross_launch_after("cross_stats_kernel", cross_stats_kernel<T, DP>, dim3(static_cast<unsigned>(tiles + (mask.mask ? P.B : 0))), 256, 0,
                            st, P, mask);
    if (rc) return rc;
    rc = cross_launch_after("cross_dq_kernel", kq, dim3(static_cast<unsigned>(n < sms ? n : sms)), C::THREADS, C::SMEM, st, q, g, k, v, P);
    if (!rc && P.splits > 1) rc = join_launch<T>(P.part_dq, P.splits, rows, P.D, P.Sq, P.Hq, P.dq, nullptr, st);
    if (rc) return rc;
  }
  if (P.Sk > 0) {
    const int64_t n = P.Skp / CT * P.kv_splits * P.Hkv * P.B, rows = static_cast<int64_t>(P.B) * P.Hkv * P.Sk;
    if (n >= (1 << 30)) return fail(H3B_ERR_UNSUPPORTED, "cross_attention_backward: too many key tiles");
    rc = cross_launch_after("cross_dkv_kernel", kkv, dim3(static_cast<unsigned>(n < sms ? n : sms)), C::THREADS, C::SMEM, st, q, g, k, v, P);
    if (!rc && P.kv_splits > 1) rc = join_launch<T>(P.part_dk, P.kv_splits, rows, P.D, P.Sk, P.Hkv, P.dk, &P.dv, st);
  }
  return rc;
}

template <typename T>
static int bwd_launch(const CrossParams& P, const MaskArgs& mask, cudaStream_t st) {
  if (P.D <= 64) return P.bias2 ? bwd_launch_cfg<T, 64, true>(P, mask, st) : bwd_launch_cfg<T, 64, false>(P, mask, st);
  return P.bias2 ? bwd_launch_cfg<T, 128, true>(P, mask, st) : bwd_launch_cfg<T, 128, false>(P, mask, st);
}

}  // namespace h3b
