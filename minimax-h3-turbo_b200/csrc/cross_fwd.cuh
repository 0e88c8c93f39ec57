// Cross attention forward on the tcgen05 tensor cores.
//
// A work unit is a pair of query tiles (slots 0 and 1, 128 rows each) of one key head, over a range of key tiles.  One
// persistent CTA per SM walks the units; its warps:
//   0-7, 8-15  softmax of slot 0 and 1: two threads per row, 64 scores each.  S (128 fp32 columns of tensor memory) ->
//              registers, running maximum and sum in fp32, P = exp2(S scale2 - m) rounded to the operand type, back to
//              tensor memory (over S).  P rounded to 8 (bf16) or 11 (fp16) bits, relative to each probability: the product's
//              operand type; the sum uses the unrounded values.  (Running maximum and sum in one pass: Milakov and
//              Gimelshein, Online normalizer calculation for softmax, 2018; rescaling only past a bound is a published
//              refinement of it.)  m is an exact maximum of the tiles so far, but taken anew
//              only when a tile exceeds it by more than 8 (a factor 2^8: far from overflow in fp32 sums and fp16 P): P of a
//              tile is computed with the m at hand, without a pass for the maximum before it, and only such a tile is gone
//              over again, after its threads have rescaled O in tensor memory.  A unit's first tile, if all its keys are in use,
//              is tried with m = 0, which does for normalised q and k: kept if the largest of every 64 scores is between 0
//              and 8, as it may be for any later tile.
//              After a unit's last tile the same threads take O / l through swizzled staging to a bulk tensor store, while
//              the next unit's first scores are on their way; and the log-sum-exp.
//   16         MMA issue: S = Q K^T (both from shared memory), O += P V (P from tensor memory, V channel-major)
//   17         copies: Q tiles, and a ring of pairs (V of a key tile, K of the next): what one step of both slots reads,
//              one barrier each way
//   18         zeroes the rows of V tiles whose keys are left out, before their product (0 x NaN would reach the sums)
//   19         stores
// Tensor memory: S0 S1 O0 O1, 128 columns each.  While one slot's softmax runs, the tensor cores work for the other.
// Units with few query tiles split the keys over CTAs; cross_combine_kernel joins the partial results by their
// log-sum-exps in a fixed order.
//
// Bound by the chain scores -> softmax -> second product: 3150 cycles for two query tiles x one key tile, of which the
// products alone take 2048 (tensor pipe 60 % active; exponentials 45 %).  Two threads per row and two slots, because one
// thread per row takes longer for a softmax than the other slot's products last.
// bf16, 40 heads x 128 channels, normalised q and k, at 1965 MHz / in a row under the power limit: 57840 queries x 1600 keys 1650 /
// 1915 us (1150 / 990 TFLOP/s), 2 x 12090 x 512 260 / 302 us (975 / 840), one query x 57840 keys 205 / 235 us (HBM, 5.8 / 5.0 TB/s).
// Scores of a larger spread are gone over twice more often: 2 x 12090 x 512 at standard deviations 1, 1.4, 2, 4, 8: 259, 368, 304,
// 391, 407 us.
#include "cross_common.cuh"

namespace h3b {

template <int DP>
struct FwdCfg {
  static constexpr int NSUB = DP / 64;
  static constexpr int TILE = NSUB * static_cast<int>(SUB_BYTES);  // bytes of a 128-row tile
  static constexpr int STAGES = DP == 128 ? 2 : 4;                 // ring of (V, next K) pairs
  static constexpr int SMEM = 2 * TILE + STAGES * 2 * TILE + TILE + 4 * CT * 4 + 512;
  static constexpr int THREADS = 640;
  static constexpr uint32_t TMEM_COLS = 512;
};

struct FwdUnit {
  int b, hk, split, tile0, t0, t1;  // batch, key head, key split, first query tile, key tiles [t0, t1)
  bool two;                         // the second query tile exists
};

__device__ __forceinline__ int key_tiles(const CrossParams& P, int b) {
  return static_cast<int>((ca_len(P.kv_lens, b, P.Sk) + CT - 1) / CT);
}
// Where entries differ in length (P.ragged), splits have the same number of key tiles in all entries, the smallest that makes
// no more splits than P.ragged, so that a short entry takes few SMs instead of many for a short while; an entry without keys
// has one.  Sets `per`, and `first` to this CTA's only unit (n_items: none).  Called by whole warps.  5 queries over 12090, 8059
// and 4028 keys, 56 over 8 heads x 128: 29.5 us, 34.9 with as many splits for every entry; equal lengths pay 2 to 3 us.
__device__ __forceinline__ int ragged_splits(const CrossParams& P, int b, int per) { return max(1, (key_tiles(P, b) + per - 1) / per); }
__device__ __forceinline__ void ragged_unit(const CrossParams& P, int n_items, int& per, int& first) {
  const int lane = threadIdx.x & 31, equal = P.ragged / P.B;  // (as many splits for each entry are surely not too many)
  int most = 1;
  for (int b = lane; b < P.B; b += 32) most = max(most, key_tiles(P, b));
  most = __reduce_max_sync(0xffffffffu, most);
  per = (most + P.splits - 1) / P.splits;
  for (int hi = max(per, (most + equal - 1) / equal); per < hi;) {
    const int mid = (per + hi) / 2;
    int n = 0;
    for (int b = lane; b < P.B; b += 32) n += ragged_splits(P, b, mid);
    if (__reduce_add_sync(0xffffffffu, n) <= P.ragged) hi = mid;
    else per = mid + 1;
  }
  int pair, hk, r = P.by_hkv.divmod(P.by_units.divmod(blockIdx.x, pair), hk);  // the r-th split of all entries
  first = n_items;
  for (int b0 = 0; b0 < P.B; b0 += 32) {
    const int n = b0 + lane < P.B ? ragged_splits(P, b0 + lane, per) : 0;
    int upto = n;
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned after = __ballot_sync(0xffffffffu, upto > r);
    if (after) {
      const int at = __ffs(after) - 1, split = r - __shfl_sync(0xffffffffu, upto - n, at);
      first = ((split * P.B + b0 + at) * P.Hkv + hk) * P.units + pair;
      return;
    }
    r -= __shfl_sync(0xffffffffu, upto, 31);
  }
}

// `per`: 0, or the key tiles of a split (ragged_unit).
__device__ __forceinline__ FwdUnit fwd_unit(const CrossParams& P, int it, int per) {
  FwdUnit u;
  int pair;
  u.split = P.by_batch.divmod(P.by_hkv.divmod(P.by_units.divmod(it, pair), u.hk), u.b);
  u.tile0 = pair * 2;
  u.two = u.tile0 + 1 < P.q_tiles;
  const int nt = key_tiles(P, u.b);
  if (!per) per = P.by_splits.div(nt + P.splits - 1);
  u.t0 = min(u.split * per, nt);
  u.t1 = min(u.t0 + per, nt);
  return u;
}
// the next unit with key tiles
template <bool RAGGED>
__device__ __forceinline__ bool fwd_next(const CrossParams& P, int per, int& it, int n, FwdUnit& u) {
  for (; it < n; it += RAGGED ? n : gridDim.x) {
    u = fwd_unit(P, it, per);
    if (u.t1 > u.t0) {
      it += RAGGED ? n : gridDim.x;
      return true;
    }
  }
  return false;
}
// V rows of tile t must be zeroed before use: a mask, or a length that ends inside the tile and before the tensor's end
__device__ __forceinline__ bool needs_zeroing(const CrossParams& P, int64_t len, int t) {
  return P.bias2 != nullptr || (len < P.Sk && static_cast<int64_t>(t + 1) * CT > len);
}

// 16 scores of a row -> probabilities: x = s scale2 + nm (nm = -m), p = exp2(x).  MASK 0: all keys in use; 1: keys from
// `lim` on are out; 2: `bias` is what each key adds, -inf: out, whatever its score.  Of unmasked keys every POLY-th pair goes
// through the FMA pipe's exp2.  Adds to the row's sums, raises `top` (NaN stays).
template <typename T, int MASK>
__device__ __forceinline__ void soft_chunk(const uint32_t (&r)[16], float scale2, float nm, int lim, const float4 (&bias)[4],
                                           uint32_t* pk, f32x2 (&sum)[2], float (&top)[2]) {
  const f32x2 sc = f2(scale2, scale2), n2 = f2(nm, nm);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = 2 * (i + h);
      float xa, xb;
      const f32x2 sv = f2(__uint_as_float(r[k]), __uint_as_float(r[k + 1]));
      if constexpr (MASK == 2) {
        const float ba = h ? bias[i / 2].z : bias[i / 2].x, bc = h ? bias[i / 2].w : bias[i / 2].y;
        f2_split(f2_fma(sv, sc, f2_add(f2(ba, bc), n2)), xa, xb);
        if (ba == -INFINITY) xa = -INFINITY;
        if (bc == -INFINITY) xb = -INFINITY;
      } else {
        f2_split(f2_fma(sv, sc, n2), xa, xb);
        if constexpr (MASK == 1) {
          if (k >= lim) xa = -INFINITY;
          if (k + 1 >= lim) xb = -INFINITY;
        }
      }
      top[h] = max_nan(top[h], xa, xb);
      const f32x2 p = MASK == 0 && h && (i & 2) ? f2_exp2<false>(xa, xb) : f2(ex2(xa), ex2(xb));
      sum[h] = f2_add(sum[h], p);
      float pa, pb;
      f2_split(p, pa, pb);
      pk[i + h] = pack2<T>(pa, pb);
    }
  }
}
// the largest of 32 scores (MASK 2: of s scale2 + bias).  Runs once a unit: from a cold instruction cache, at some nine cycles
// per instruction, so it is kept short (two scores per maximum, the scale once at the end).
template <int MASK>
__device__ __forceinline__ float max_chunk(const uint32_t (&r)[32], float scale2, int lim, const float4 (&bias)[8], float top) {
  float tp[2] = {top, -INFINITY};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float x[4];
    if constexpr (MASK == 2) {
      const float bv[4] = {bias[i].x, bias[i].y, bias[i].z, bias[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = fmaf(__uint_as_float(r[4 * i + e]), scale2, bv[e]);
        if (bv[e] == -INFINITY) x[e] = -INFINITY;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = __uint_as_float(r[4 * i + e]);
        if (MASK == 1 && 4 * i + e >= lim) x[e] = -INFINITY;
      }
    }
    tp[0] = fmaxf(tp[0], fmaxf(x[0], x[1]));
    tp[1] = fmaxf(tp[1], fmaxf(x[2], x[3]));
  }
  return fmaxf(tp[0], tp[1]);
}

// RAGGED: one unit per CTA, chosen from the lengths (a variant of its own: inside the other one it cost 2 %)
template <typename T, int DP, bool BIAS, bool RAGGED>
__global__ void __launch_bounds__(FwdCfg<DP>::THREADS, 1)
    cross_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO, const CrossParams P) {
  using C = FwdCfg<DP>;
  extern __shared__ __align__(1024) unsigned char ca_smem[];
  unsigned char* sQ = ca_smem;
  unsigned char* sV = sQ + 2 * C::TILE;  // stage: V tile, K tile
  unsigned char* sO = sV + C::STAGES * 2 * C::TILE;
  float* halves = reinterpret_cast<float*>(sO + C::TILE);  // [slot][half][row] maxima or sums of a row's halves
  uint64_t* q_full = reinterpret_cast<uint64_t*>(halves + 4 * CT);
  uint64_t* q_empty = q_full + 2;
  uint64_t* kv_full = q_empty + 2;
  uint64_t* kv_empty = kv_full + C::STAGES;
  uint64_t* v_clean = kv_empty + C::STAGES;
  uint64_t* s_full = v_clean + C::STAGES;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* out_full = o_full + 2;  // the staging holds a slot's output
  uint64_t* out_free = out_full + 1;  // [use & 1] and has been read
  uint64_t* done = out_free + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int n_items = P.units * P.splits * P.Hkv * P.B;
  // with any mask every V tile passes warp 18 (in step with the ring: a phase it skipped could be taken for another)
  const bool masked = BIAS || P.kv_lens != nullptr;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 8);
      mbar_init(&o_full[s], 1);
    }
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
      mbar_init(&v_clean[s], 1);
    }
    mbar_init(out_full, 8);
    mbar_init(&out_free[0], 1);
    mbar_init(&out_free[1], 1);
    mbar_init(done, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmO);
  }
  if (warp == 16) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  after_previous();
  int per = 0, first = blockIdx.x;  // this CTA's first unit
  if constexpr (RAGGED) ragged_unit(P, n_items, per, first);

  if (warp < 16) {
    // ------------------------------------------------------------------------------------------ softmax
    regs_inc<104>();
    const int slot = warp >> 3, half = (warp >> 2) & 1, row = threadIdx.x & (CT - 1);
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // lane offset (32 per warp) in bits 16..
    const uint32_t tS = tmem + slot * CT + lanes, tO = tmem + 2 * CT + slot * CT + lanes;
    const int bar = 1 + slot * 4 + (warp & 3);  // the two warps of the same 32 rows
    float* mine = halves + (slot * 2 + half) * CT + row;
    const float* other = halves + (slot * 2 + 1 - half) * CT + row;
    int hg;
    const int qr = P.by_g.divmod(row, hg);
    const int64_t rows = static_cast<int64_t>(P.B) * P.Hq * P.Sq;
    uint32_t sph = 0, oph = 0, uses = slot;  // uses: of the staging by both slots before this one
    bool dead = false;
    FwdUnit u, nxt;
    int it = first;
    for (bool have = fwd_next<RAGGED>(P, per, it, n_items, u), more; have; u = nxt, have = more) {
      if (slot == 1 && !u.two) {
        ++uses;
        more = fwd_next<RAGGED>(P, per, it, n_items, nxt);
        continue;
      }
      const int64_t len = ca_len(P.kv_lens, u.b, P.Sk);
      const int64_t s = static_cast<int64_t>(u.tile0 + slot) * P.nq + qr;
      const bool valid = qr < P.nq && s < P.Sq;
      const bool idle = !__any_sync(0xffffffffu, valid);  // none of these 32 rows exists: with few queries most warps
      float m = -INFINITY;
      f32x2 l = f2(0.f, 0.f);
      if (idle) {  // their P is whatever the columns hold: nobody reads what comes of it
        for (int t = u.t0; t < u.t1; ++t, sph ^= 1) {
          dead = dead || !warp_wait(&s_full[slot], sph, abort_flag);
          if (lane == 0) mbar_arrive(&p_full[slot]);
        }
        more = fwd_next<RAGGED>(P, per, it, n_items, nxt);
      }
      for (int t = idle ? u.t1 : u.t0; t < u.t1; ++t) {
        dead = dead || !warp_wait(&s_full[slot], sph, abort_flag);
        sph ^= 1;
        tc_fence_after();
        const int64_t left = len - static_cast<int64_t>(t) * CT - half * 64;
        const int lim = left < 64 ? static_cast<int>(left) : 64;  // keys in use, of this thread's
        const float4* b4 = BIAS ? reinterpret_cast<const float4*>(P.bias2 + u.b * P.Skp + static_cast<int64_t>(t) * CT + half * 64) : nullptr;
        uint32_t pk[32];
        f32x2 sum[2];
        const bool guess = !BIAS && t == u.t0 && len - static_cast<int64_t>(t) * CT >= CT;
        for (bool exact = t == u.t0 && !guess;; exact = true) {
          if (exact) {
            float top = -INFINITY;
            {
              uint32_t r[2][32];
              float4 bias[8];
              tmem_ld_32x32b_x32(tS + half * 64, r[0]);
              if constexpr (!BIAS) tmem_ld_32x32b_x32(tS + half * 64 + 32, r[1]);
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                if constexpr (BIAS) {  // on its way while the scores are; 32 of either at a time
                  if (c) tmem_ld_32x32b_x32(tS + half * 64 + 32, r[1]);
#pragma unroll
                  for (int i = 0; i < 8; ++i) bias[i] = b4[8 * c + i];
                }
                if (BIAS || c == 0) tmem_ld_wait();
                if constexpr (BIAS) top = max_chunk<2>(r[c], P.scale2, 0, bias, top);
                else if (lim < 64) top = max_chunk<1>(r[c], P.scale2, lim - 32 * c, bias, top);
                else top = max_chunk<0>(r[c], P.scale2, 0, bias, top);
              }
            }
            *mine = top;
            group_sync(bar, 64);  // (both have read by the barrier after the probabilities)
            top = fmaxf(top, *other);
            top = fmaxf(m, BIAS ? top : top * P.scale2);
            if (t > u.t0) {  // the product of the tile before is complete: its commit came before that of these scores
              const float f = top == -INFINITY ? 1.f : ex2(m - top);
              float la, lb;
              f2_split(l, la, lb);
              l = f2(la * f, lb * f);
#pragma unroll 1
              for (int c = half * (DP / 32); c < (half + 1) * (DP / 32); ++c) {
                uint32_t o[16];
                tmem_ld_32x32b_x16(tO + 16 * c, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_st_32x32b_x16(tO + 16 * c, o);
              }
            }
            m = top;
          }
          const float nm = m == -INFINITY ? 0.f : -m;  // no key so far: the guess, or every probability is exp2(-inf) = 0
          float over[2] = {-INFINITY, -INFINITY};
          sum[0] = sum[1] = f2(0.f, 0.f);
          uint32_t r[2][16];
          tmem_ld_32x32b_x16(tS + half * 64, r[0]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float4 bias[4];  // on its way while the scores are
            if constexpr (BIAS) {
#pragma unroll
              for (int i = 0; i < 4; ++i) bias[i] = b4[4 * c + i];
            }
            tmem_ld_wait();
            if (c < 3) tmem_ld_32x32b_x16(tS + half * 64 + 16 * (c + 1), r[(c + 1) & 1]);
            if constexpr (BIAS) soft_chunk<T, 2>(r[c & 1], P.scale2, nm, 0, bias, pk + 8 * c, sum, over);
            else if (lim < 64) soft_chunk<T, 1>(r[c & 1], P.scale2, nm, lim - 16 * c, bias, pk + 8 * c, sum, over);
            else soft_chunk<T, 0>(r[c & 1], P.scale2, nm, 0, bias, pk + 8 * c, sum, over);
          }
          over[0] = max_nan(over[0], over[1]);
          if (over[0] != over[0]) sum[0] = f2(over[0], over[0]);  // a score that is not a number: so is the row
          // past this barrier both warps have read S
          // (rows that no query fills have no say: what they hold is left from another tile or kernel, and a maximum taken
          // anew changes how every row's P is rounded)
          const bool far = guess ? !(over[0] >= 0.f && over[0] <= 8.f) : over[0] > (m == -INFINITY ? -INFINITY : 8.f);
          const bool again = group_any(bar, 64, valid & far);
          if (exact) break;
          if (!again) {
            if (guess) m = 0.f;
            break;
          }
        }
        l = f2_add(l, f2_add(sum[0], sum[1]));
        tmem_st_32x32b_x32(tS + half * 32, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[slot]);
        if (t == u.t0) more = fwd_next<RAGGED>(P, per, it, n_items, nxt);  // while the next scores are on their way
      }
      // ---- the unit's output
      float la, lb;
      f2_split(l, la, lb);
      *mine = la + lb;
      group_sync(bar, 64);
      const float total = halves[slot * 2 * CT + row] + halves[(slot * 2 + 1) * CT + row];
      const bool none = total == 0.f;  // no key took part: zero, whatever the products hold
      const float inv = none ? 0.f : 1.f / total;
      const int64_t rid = (static_cast<int64_t>(u.b) * P.Hq + u.hk * P.G + hg) * P.Sq + s;
      if (half == 0 && valid) {
        const float lse2 = none ? -INFINITY : m + log2f(total);
        if (P.splits > 1) P.part_lse[u.split * rows + rid] = lse2;
        else if (P.lse) P.lse[rid] = lse2 * CA_LN2;
      }
      dead = dead || !warp_wait(&o_full[slot], oph, abort_flag);
      oph ^= 1;
      tc_fence_after();
      // this thread's columns: half of DP
      if (P.splits > 1) {
        float* dst = P.part_o + (u.split * rows + rid) * P.D;
#pragma unroll 1
        for (int c = half * (DP / 32); !idle && c < (half + 1) * (DP / 32); ++c) {
          uint32_t o[16];
          tmem_ld_32x32b_x16(tO + 16 * c, o);
          tmem_ld_wait();
          if (!valid) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * c + 4 * i < P.D)
              *reinterpret_cast<float4*>(dst + 16 * c + 4 * i) =
                  none ? make_float4(0.f, 0.f, 0.f, 0.f)
                       : make_float4(__uint_as_float(o[4 * i]) * inv, __uint_as_float(o[4 * i + 1]) * inv,
                                     __uint_as_float(o[4 * i + 2]) * inv, __uint_as_float(o[4 * i + 3]) * inv);
        }
      } else {
        // the use before this one (uses - 1) has left the staging.  Two barriers in turn: a slot gets here only after the use
        // three before was read (its own last wait, or the other slot's, which the products in between came after), so a
        // phase cannot be taken for the one before it
        if (uses) dead = dead || !warp_wait(&out_free[(uses - 1) & 1], ((uses - 1) >> 1) & 1, abort_flag);
        const f32x2 inv2 = f2(inv, inv);
#pragma unroll 1
        for (int c = idle ? DP / 64 : 0; c < DP / 64; ++c) {  // (a loop: see max_chunk)
          const int col = half * (DP / 2) + 32 * c;
          uint32_t o[32];
          tmem_ld_32x32b_x32(tO + col, o);
          tmem_ld_wait();
          unsigned char* part = sO + (col >> 6) * SUB_BYTES;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint4 v;
            uint32_t* vv = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float oa, ob;
              f2_split(f2_fma(f2(__uint_as_float(o[8 * i + 2 * e]), __uint_as_float(o[8 * i + 2 * e + 1])), inv2, f2(0.f, 0.f)), oa, ob);
              vv[e] = pack2<T>(oa, ob);
            }
            if (none) v = make_uint4(0, 0, 0, 0);
            put_swizzled(part, row, ((col & 63) >> 3) + i, v);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(out_full);
      }
      tc_fence_before();
      group_sync(bar, 64);  // both have read the sums before the next unit's maxima
      uses += u.two ? 2 : 1;
    }
  } else {
    regs_dec<64>();
    if (warp == 16) {
      // -------------------------------------------------------------------------------------- MMA issue
      constexpr uint32_t idQK = idesc_f16<T>(CT, CT, false), idPV = idesc_f16<T>(CT, DP, true);
      constexpr uint32_t TILE16 = C::TILE >> 4;
      const uint32_t dQ = desc_rows(smem_u32(sQ)), dK = desc_rows(smem_u32(sV) + C::TILE), dV = desc_chan(smem_u32(sV));
      int st = 0;
      uint32_t kph = 0, qph[2] = {0, 0}, pph[2] = {0, 0};
      FwdUnit cur, nxt;
      int it = first;
      bool have = fwd_next<RAGGED>(P, per, it, n_items, cur), ok = true;
      auto qk = [&](int slot, int kst, bool first, bool last) {  // S of a slot; its Q tile arrives with the unit's first
        if (first) {
          if (!(ok = warp_wait(&q_full[slot], qph[slot], abort_flag))) return;
          qph[slot] ^= 1;
          tc_fence_after();
        }
        mma_rows<DP / 16>(tmem + slot * CT, dQ + slot * TILE16, dK + kst * 2 * TILE16, idQK);
        commit_one(&s_full[slot]);
        if (last) commit_one(&q_empty[slot]);
      };
      auto advance = [&] {
        commit_one(&kv_empty[st]);
        if (++st == C::STAGES) st = 0, kph ^= 1;
      };
      if (have) {
        ok = warp_wait(&kv_full[st], kph, abort_flag);
        tc_fence_after();
        if (ok) qk(0, st, true, cur.t1 - cur.t0 == 1);
        if (ok && cur.two) qk(1, st, true, cur.t1 - cur.t0 == 1);
        advance();
      }
      while (have && ok) {
        const bool more = fwd_next<RAGGED>(P, per, it, n_items, nxt);
        for (int t = cur.t0; ok && t < cur.t1; ++t) {
          const bool last = t == cur.t1 - 1, then_qk = !last || more;
          const bool qk_last = last ? nxt.t1 - nxt.t0 == 1 : t + 2 == cur.t1;
          if (!(ok = warp_wait(&kv_full[st], kph, abort_flag))) break;
          if (masked && !(ok = warp_wait(&v_clean[st], kph, abort_flag))) break;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (s == 0 || cur.two) {
              if (!(ok = warp_wait(&p_full[s], pph[s], abort_flag))) break;
              pph[s] ^= 1;
              tc_fence_after();  // (a unit's first P comes after its threads have read the O before)
              mma_chan<1>(tmem + 2 * CT + s * CT, tmem + s * CT, dV + st * 2 * TILE16, idPV, t > cur.t0);
              if (last) commit_one(&o_full[s]);
            }
            if (then_qk && (s == 0 || (last ? nxt.two : cur.two))) qk(s, st, last, qk_last);
            if (!ok) break;
          }
          if (ok) advance();
        }
        cur = nxt;
        have = more;
      }
    } else if (warp == 17) {
      if (lane == 0) {
        // -------------------------------------------------------------------------------------- copies
        int st = 0, fills = 0, qfills[2] = {0, 0};
        uint32_t kph = 1, qph[2] = {1, 1};
        FwdUnit u, nxt;
        bool ok = true;
        const uint32_t q_bytes = static_cast<uint32_t>(C::NSUB * 128 * P.G * P.nq);
        auto load_q = [&](const FwdUnit& w, int s) {
          if (!ok || !(ok = mbar_wait(&q_empty[s], qph[s], abort_flag))) return;
          qph[s] ^= 1;
          mbar_arrive_expect_tx(&q_full[s], q_bytes);
          for (int p = 0; p < C::NSUB; ++p)
            tma_load_5d(sQ + s * C::TILE + p * SUB_BYTES, &tmQ, &q_full[s], 64 * p, 0, w.hk, (w.tile0 + s) * P.nq, w.b);
          ++qfills[s];
        };
        // one stage: V of tile tv (if >= 0) of unit uv, K of tile tk (if >= 0) of unit uk
        auto load_kv = [&](const FwdUnit& uv, int tv, const FwdUnit& uk, int tk) {
          if (!ok || !(ok = mbar_wait(&kv_empty[st], kph, abort_flag))) return;
          mbar_arrive_expect_tx(&kv_full[st], ((tv >= 0) + (tk >= 0)) * C::TILE);
          unsigned char* dst = sV + st * 2 * C::TILE;
          for (int p = 0; tv >= 0 && p < C::NSUB; ++p)
            tma_load_4d(dst + p * SUB_BYTES, &tmV, &kv_full[st], 64 * p, uv.hk, tv * CT, uv.b);
          for (int p = 0; tk >= 0 && p < C::NSUB; ++p)
            tma_load_4d(dst + C::TILE + p * SUB_BYTES, &tmK, &kv_full[st], 64 * p, uk.hk, tk * CT, uk.b);
          ++fills;
          if (++st == C::STAGES) st = 0, kph ^= 1;
        };
        int it = first;
        bool have = fwd_next<RAGGED>(P, per, it, n_items, u);
        if (have) {
          load_kv(u, -1, u, u.t0);
          load_q(u, 0);
          if (u.two) load_q(u, 1);
        }
        while (have && ok) {
          const bool more = fwd_next<RAGGED>(P, per, it, n_items, nxt);
          for (int s = 0; more && s < (nxt.two ? 2 : 1); ++s)
            for (int p = 0; p < C::NSUB; ++p) tma_prefetch_5d(&tmQ, 64 * p, 0, nxt.hk, (nxt.tile0 + s) * P.nq, nxt.b);
          for (int t = u.t0; ok && t < u.t1; ++t) {
            const bool last = t == u.t1 - 1;
            if (!last) load_kv(u, t, u, t + 1);
            else load_kv(u, t, nxt, more ? nxt.t0 : -1);
          }
          // the next unit's Q tiles come in while this one's last key tile is in hand
          if (more) load_q(nxt, 0);
          if (more && nxt.two) load_q(nxt, 1);
          u = nxt;
          have = more;
        }
        // copies in flight land in this CTA's shared memory: wait for the last ones before it goes away
        for (int j = fills > C::STAGES ? fills - C::STAGES : 0; j < fills; ++j)
          if (!mbar_wait_drain(&kv_full[j % C::STAGES], static_cast<uint32_t>((j / C::STAGES) & 1))) break;
        for (int s = 0; s < 2; ++s)
          if (qfills[s]) mbar_wait_drain(&q_full[s], static_cast<uint32_t>((qfills[s] - 1) & 1));
      }
      __syncwarp();
    } else if (warp == 18 && masked) {
      // ---------------------------------------------------------------------------------------- rows of masked keys
      if (lane == 0) mbar_arrive(&v_clean[0]);  // the first stage holds a K tile only
      int st = 1;
      uint32_t kph = 0;
      FwdUnit u;
      bool ok = true;
      for (int it = first; ok && fwd_next<RAGGED>(P, per, it, n_items, u);) {
        const int64_t len = ca_len(P.kv_lens, u.b, P.Sk);
        for (int t = u.t0; ok && t < u.t1; ++t) {
          if (!(ok = warp_wait(&kv_full[st], kph, abort_flag))) break;
          if (needs_zeroing(P, len, t)) {
            for (int j = lane; j < CT; j += 32) {
              const int64_t key = static_cast<int64_t>(t) * CT + j;
              if (key >= len || (BIAS && P.bias2[u.b * P.Skp + key] == -INFINITY))
                for (int p = 0; p < C::NSUB; ++p)
                  for (int c = 0; c < 8; ++c)
                    *reinterpret_cast<uint4*>(sV + st * 2 * C::TILE + p * SUB_BYTES + j * 128 + c * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (lane == 0) mbar_arrive(&v_clean[st]);
          if (++st == C::STAGES) st = 0, kph ^= 1;
        }
      }
    } else if (warp == 19) {
      // ---------------------------------------------------------------------------------------- stores
      uint32_t ph = 0, uses = 0;
      bool ok = true;
      for (int it = first; ok && it < n_items; it += RAGGED ? n_items : gridDim.x) {
        const FwdUnit u = fwd_unit(P, it, per);
        // the splits that this entry has not got
        for (int r = lane; RAGGED && u.split == 0 && r < (u.two ? 2 : 1) * P.nq * P.G; r += 32) {
          int h;
          const int64_t q = static_cast<int64_t>(u.tile0) * P.nq + P.by_g.divmod(r, h), rows = static_cast<int64_t>(P.B) * P.Hq * P.Sq;
          for (int x = ragged_splits(P, u.b, per); x < P.splits && q < P.Sq; ++x)
            P.part_lse[x * rows + (static_cast<int64_t>(u.b) * P.Hq + u.hk * P.G + h) * P.Sq + q] = -INFINITY;
        }
        for (int s = 0; ok && s < (u.two ? 2 : 1); ++s) {
          const int64_t s0 = static_cast<int64_t>(u.tile0 + s) * P.nq;
          if (u.t1 > u.t0) {
            if (P.splits > 1) continue;
            if (lane == 0 && (ok = mbar_wait(out_full, ph, abort_flag))) {
              for (int p = 0; p < C::NSUB; ++p) tma_store_5d(sO + p * SUB_BYTES, &tmO, 64 * p, 0, u.hk, static_cast<int>(s0), u.b);
              bulk_commit();
              bulk_wait_read();
              mbar_arrive(&out_free[uses & 1]);
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
            ph ^= 1;
            ++uses;
            continue;
          }
          for (int r = lane; r < P.nq * P.G; r += 32) {  // a unit without keys: zero rows
            const int64_t q = s0 + r / P.G, h = u.hk * P.G + r % P.G;
            if (q >= P.Sq) break;
            const int64_t rid = (u.b * static_cast<int64_t>(P.Hq) + h) * P.Sq + q;
            if (P.splits > 1) {
              P.part_lse[u.split * static_cast<int64_t>(P.B) * P.Hq * P.Sq + rid] = -INFINITY;
              continue;
            }
            if (P.lse) P.lse[rid] = -INFINITY;
            T* dst = static_cast<T*>(P.o.ptr) + u.b * P.o.stride_b + q * P.o.stride_s + h * P.o.stride_h;
            for (int c = 0; c < P.D; c += 8) *reinterpret_cast<uint4*>(dst + c) = make_uint4(0, 0, 0, 0);
          }
        }
      }
      if (lane == 0) bulk_wait_all();
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    commit_one(done);  // every product issued (after a wait that gave up some may still run) and its arrivals are over
    mbar_wait_drain(done, 0);
    __syncwarp();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// Joins the key splits of every row: weights exp2(lse_s - lse), always in the same order.  One warp per row, eight splits on
// their way at a time.  No shared memory: with four warps per row that add up there, the attention kernels around this one took
// 7 us longer each (33 us launches, measured).
template <typename T>
__global__ void __launch_bounds__(32) cross_combine_kernel(const CrossParams P) {
  after_previous();
  const int64_t rows = static_cast<int64_t>(P.B) * P.Hq * P.Sq, row = blockIdx.x;
  const int lane = threadIdx.x;
  float e[2], top = -INFINITY, sum = 0.f;  // at most 64 splits
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    e[i] = lane + 32 * i < P.splits ? P.part_lse[(lane + 32 * i) * rows + row] : -INFINITY;
    top = fmaxf(top, e[i]);
  }
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    e[i] = ex2(e[i] - base);
    sum += e[i];
  }
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int s = 0; s < P.splits; ++s) {
    const float w = __shfl_sync(0xffffffffu, s < 32 ? e[0] : e[1], s & 31);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);  // a split without keys wrote nothing
    if (w != 0.f && 4 * lane < P.D) o = *reinterpret_cast<const float4*>(P.part_o + (s * rows + row) * P.D + 4 * lane);
    acc.x = fmaf(w, o.x, acc.x), acc.y = fmaf(w, o.y, acc.y), acc.z = fmaf(w, o.z, acc.z), acc.w = fmaf(w, o.w, acc.w);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t s = row % P.Sq, bh = row / P.Sq, h = bh % P.Hq, b = bh / P.Hq;
  if (4 * lane < P.D) {
    uint2 v = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
    *reinterpret_cast<uint2*>(static_cast<T*>(P.o.ptr) + b * P.o.stride_b + s * P.o.stride_s + h * P.o.stride_h + 4 * lane) = v;
  }
  if (P.lse && lane == 0) P.lse[row] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * CA_LN2;
}

// Key splits of the forward: enough that every SM has work, at the least time of the busiest SM, counted in key tiles
// (a unit costs about two tiles to fill and drain, splitting at all about three for the second kernel).
static int fwd_splits(int64_t units, int64_t key_tiles) {
  const int sms = cross_sms();
  if (units >= sms || key_tiles <= 1) return 1;
  int best = 1;
  int64_t best_cost = key_tiles + 2;
  for (int s = 2; s <= 64 && s <= key_tiles; ++s) {
    const int64_t waves = (units * s + sms - 1) / sms, cost = waves * ((key_tiles + s - 1) / s + 2) + 3;
    if (cost < best_cost) best = s, best_cost = cost;
  }
  return best;
}

template <typename T, int DP, bool BIAS, bool RAGGED>
static int fwd_launch_cfg(const CrossParams& P, cudaStream_t st) {
  using C = FwdCfg<DP>;
  CUtensorMap q, k, v, o;
  const bool half = std::is_same_v<T, __half>;
  int rc = cross_map_q(&q, P, P.q, half);
  if (!rc) rc = cross_map_k(&k, P, P.Sk > 0 ? P.k : cross_stand_in(P.q), half);
  if (!rc) rc = cross_map_k(&v, P, P.Sk > 0 ? P.v : cross_stand_in(P.q), half);
  if (!rc) rc = cross_map_q(&o, P, P.o, half);
  if (rc) return rc;
  auto kern = cross_fwd_kernel<T, DP, BIAS, RAGGED>;
  static std::atomic<bool> ready[CA_DEVICES];
  rc = cross_smem(reinterpret_cast<const void*>(kern), C::SMEM, ready, "cross_fwd_kernel shared memory");
  if (rc) return rc;
  const int64_t items = static_cast<int64_t>(P.units) * P.splits * P.Hkv * P.B;
  if (items >= (1 << 30)) return fail(H3B_ERR_UNSUPPORTED, "cross_attention: too many query tiles");
  const int grid = RAGGED ? P.ragged * P.units * P.Hkv : static_cast<int>(items < cross_sms() ? items : cross_sms());
  rc = cross_launch_after("cross_fwd_kernel", kern, dim3(grid), C::THREADS, C::SMEM, st, q, k, v, o, P);
  if (rc || P.splits == 1) return rc;
  const int64_t rows = static_cast<int64_t>(P.B) * P.Hq * P.Sq;
  return cross_launch_after("cross_combine_kernel", cross_combine_kernel<T>, dim3(static_cast<unsigned>(rows)), 32, 0, st, P);
}

template <typename T, int DP>
static int fwd_launch_dp(const CrossParams& P, cudaStream_t st) {
  if (P.bias2) return P.ragged ? fwd_launch_cfg<T, DP, true, true>(P, st) : fwd_launch_cfg<T, DP, true, false>(P, st);
  return P.ragged ? fwd_launch_cfg<T, DP, false, true>(P, st) : fwd_launch_cfg<T, DP, false, false>(P, st);
}
template <typename T>
static int fwd_launch(const CrossParams& P, cudaStream_t st) {
  return P.D <= 64 ? fwd_launch_dp<T, 64>(P, st) : fwd_launch_dp<T, 128>(P, st);
}

}  // namespace h3b
