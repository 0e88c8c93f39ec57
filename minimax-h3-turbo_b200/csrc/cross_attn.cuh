// Cross attention: the host side of both directions (kernels: cross_fwd.cuh, cross_bwd.cuh).
#include "cross_bwd.cuh"
#include "cross_fwd.cuh"

namespace h3b {

// Workspace, parts 256-byte aligned: the prepared mask [B, Skp] and its key counts [B]; the forward's
// partial outputs and log-sum-exps; the backward's row vectors in tile order, norms (used in fp16) and partial gradients.
struct CrossWs {
  size_t bias2 = 0, lens = 0, part_o = 0, part_lse = 0, stats = 0, g_norm2 = 0, g_top2 = 0, v_top2 = 0, v_all2 = 0, part_dq = 0, part_dk = 0, total = 0;
  int room = 1;  // splits that the forward's partial outputs have room for
};
static CrossWs cross_plan(CrossParams& P, int mask_kind, bool backward) {
  P.G = P.Hq / P.Hkv;
  P.nq = CT / P.G;
  P.Skp = (P.Sk + CT - 1) / CT * CT;
  P.q_tiles = static_cast<int>((P.Sq + P.nq - 1) / P.nq);
  P.units = (P.q_tiles + 1) / 2;
  const int64_t heads = static_cast<int64_t>(P.Hkv) * P.B, key_tiles = P.Skp / CT;
  P.splits = backward ? bwd_splits(P.q_tiles * heads, key_tiles) : fwd_splits(P.units * heads, key_tiles);
  P.kv_splits = backward ? bwd_splits(key_tiles * heads, P.q_tiles) : 1;
  P.by_g.set(P.G), P.by_hkv.set(P.Hkv), P.by_units.set(max(1, P.units)), P.by_splits.set(P.splits);
  P.by_batch.set(max(1, P.B));
  P.by_q_tiles.set(max(1, P.q_tiles)), P.by_k_tiles.set(max(1, static_cast<int>(key_tiles))), P.by_kv_splits.set(P.kv_splits);
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
  if (!backward && P.splits > 1) {
    w.room = static_cast<int>(min(static_cast<int64_t>(min(64, 2 * P.splits)), key_tiles));
    w.part_o = take(rows * w.room * P.D * 4);
    w.part_lse = take(rows * w.room * 4);
  }
  if (backward) {
    w.stats = take(static_cast<size_t>(heads) * P.q_tiles * 2 * CT * 4);
    w.g_norm2 = take(static_cast<size_t>(heads) * P.q_tiles * CT * 4);
    w.g_top2 = take(static_cast<size_t>(heads) * P.q_tiles * 4);
    w.v_top2 = take(static_cast<size_t>(heads) * key_tiles * 4);
    w.v_all2 = take(static_cast<size_t>(heads) * 4);
    if (P.splits > 1) w.part_dq = take(rows * P.splits * P.D * 4);
    if (P.kv_splits > 1) w.part_dk = take(static_cast<size_t>(heads) * P.Sk * P.kv_splits * 2 * P.D * 4);
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
  if (backward) {
    P.go = t[4], P.dq = t[5], P.dk = t[6], P.dv = t[7];
    P.wide = D % 16 == 0;
    for (const h3b_attn_tensor* g : {&P.dq, &P.dk, &P.dv})
      P.wide = P.wide && reinterpret_cast<uintptr_t>(g->ptr) % 32 == 0 && (g->stride_b | g->stride_s | g->stride_h) % 16 == 0;
  }
  P.lse = lse;
  char* base = static_cast<char*>(ws);
  P.stats = reinterpret_cast<float*>(base + w.stats);
  P.g_norm2 = reinterpret_cast<float*>(base + w.g_norm2);
  P.g_top2 = reinterpret_cast<float*>(base + w.g_top2);
  P.v_top2 = reinterpret_cast<float*>(base + w.v_top2);
  P.v_all2 = reinterpret_cast<float*>(base + w.v_all2);
  P.part_dq = reinterpret_cast<float*>(base + w.part_dq);
  P.part_dk = reinterpret_cast<float*>(base + w.part_dk);
  P.part_o = reinterpret_cast<float*>(base + w.part_o);
  P.part_lse = reinterpret_cast<float*>(base + w.part_lse);
  P.kv_lens = kv_lens;
  P.scale = scale, P.scale2 = scale * CA_LOG2E;
  MaskArgs m{};
  m.kv_lens = kv_lens;
  if (mask_kind != H3B_MASK_NONE) {
    m = MaskArgs{mask, kv_lens, reinterpret_cast<float*>(base + w.bias2), reinterpret_cast<int32_t*>(base + w.lens), ldm, Sk, P.Skp, mask_kind};
    P.bias2 = m.bias2;
    P.kv_lens = m.lens;
    if (!backward || Sq == 0) {  // the backward pass prepares it with its row vectors
      const int rc = cross_launch_after("cross_mask_kernel", cross_mask_kernel, dim3(P.B), CA_PREP, 0, st, m);
      if (rc) return rc;
    }
  }
  if (!backward && P.splits > 1 && P.kv_lens) {  // entries of different length: see ragged_unit
    const int heads = P.units * P.Hkv;
    P.ragged = max(cross_sms() / heads, P.splits * P.B);
    P.splits = w.room;
    P.by_splits.set(P.splits);
  }
  if (dtype == H3B_BF16) return backward ? bwd_launch<__nv_bfloat16>(P, m, st) : fwd_launch<__nv_bfloat16>(P, st);
  return backward ? bwd_launch<__half>(P, m, st) : fwd_launch<__half>(P, st);
}

}  // namespace h3b
