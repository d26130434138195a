// Attention of a tree of drafted tokens over a paged KV cache (fxb_tree_attn).
// No reference counterpart: its sampler keeps no cache (ml/fxlm/sample.py:63-73).
//
// o = softmax(scale * q k^T) v over the context slots and the visible nodes,
// computed online: a running maximum m, sum l and output O are rescaled by
// exp(m_old - m_new) when the maximum rises, in fp32.
#include "common.cuh"
#include "internal.h"

namespace {

constexpr int kMaxTree = 64;

template <typename T>
struct Params {
  int B, T_, Hq, Hkv, G, page_shift, P, W;
  float scale_log2;
  const T *q, *k, *v;
  T *o, *kp, *vp;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, o_sb, o_st, o_sh;
  int64_t kp_sp, kp_sh, kp_st, vp_sp, vp_sh, vp_st;
  const int32_t* table;
  int64_t table_sb;
  const int32_t *lens, *n_nodes;
  const int64_t* mask;
  int64_t mask_sb;
  int* err;
};

// One warp per (row b, node t, query head): lanes hold D / 32 elements each.
template <typename T, int D>
__global__ void __launch_bounds__(128) tree_attn_simple(const Params<T> a) {
  constexpr int E = D / 32;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= (int64_t)a.B * a.T_ * a.Hq) return;
  const int h = (int)(w % a.Hq);
  const int t = (int)(w / a.Hq % a.T_), b = (int)(w / a.Hq / a.T_);
  const int hk = h / a.G, page = 1 << a.page_shift;
  T* o = a.o + b * a.o_sb + t * a.o_st + h * a.o_sh + lane * E;
  const int n_in = a.n_nodes[b], n = min(max(n_in, 0), a.T_);
  if (n != n_in && lane == 0) atomicOr(a.err, FXB_DERR_PAGES);
  float acc[E] = {}, q[E];
  float m = -INFINITY, l = 0.f;
  if (t < n) {
    int64_t len = a.lens[b];
    if (len < 0 || len > ((int64_t)a.W << a.page_shift)) {
      if (lane == 0) atomicOr(a.err, FXB_DERR_PAGES);
      len = len < 0 ? 0 : (int64_t)a.W << a.page_shift;
    }
    const int32_t* table = a.table + b * a.table_sb;
    const T* k = a.k + b * a.k_sb + hk * a.k_sh + lane * E;
    const T* v = a.v + b * a.v_sb + hk * a.v_sh + lane * E;
    if (h == hk * a.G) {  // this node's key and value go into the cache
      const int64_t at = len + t, pi = at >> a.page_shift;
      const int pg = pi < a.W ? table[pi] : -1;
      if (pg < 0 || pg >= a.P) {
        if (lane == 0) atomicOr(a.err, FXB_DERR_PAGES);
      } else {
        T* kd = a.kp + pg * a.kp_sp + hk * a.kp_sh + (at & (page - 1)) * a.kp_st + lane * E;
        T* vd = a.vp + pg * a.vp_sp + hk * a.vp_sh + (at & (page - 1)) * a.vp_st + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          kd[e] = k[t * a.k_st + e];
          vd[e] = v[t * a.v_st + e];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      q[e] = to_f<T>(a.q[b * a.q_sb + t * a.q_st + h * a.q_sh + lane * E + e]) * a.scale_log2;
    const uint64_t see = (uint64_t)a.mask[b * a.mask_sb + t];
    for (int64_t j = 0; j < len + n; ++j) {
      const T *kj, *vj;
      if (j < len) {
        const int pg = table[j >> a.page_shift];
        if (pg < 0 || pg >= a.P) {
          if (lane == 0) atomicOr(a.err, FXB_DERR_PAGES);
          continue;
        }
        kj = a.kp + pg * a.kp_sp + hk * a.kp_sh + (j & (page - 1)) * a.kp_st + lane * E;
        vj = a.vp + pg * a.vp_sp + hk * a.vp_sh + (j & (page - 1)) * a.vp_st + lane * E;
      } else {
        const int i = (int)(j - len);
        if (!((see >> i) & 1)) continue;
        kj = k + i * a.k_st;
        vj = v + i * a.v_st;
      }
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(q[e], to_f<T>(kj[e]), s);
      s = warp_sum(s);
      if (s == -INFINITY) continue;  // weight 0
      const float mn = fmaxf(m, s);
      const float r = m == mn ? 1.f : exp2f(m - mn), p = exp2f(s - mn);
      m = mn;
      l = fmaf(l, r, p);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(acc[e], r, p * to_f<T>(vj[e]));
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no visible key: zeros; NaN stays
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = from_f<T>(acc[e] * inv);
}

template <typename T, int D>
int launch(const fxb_tree_attn_args* a, int shift, int* err, void* stream) {
  Params<T> p = {a->B, a->T, a->Hq, a->Hkv, a->Hq / a->Hkv, shift, a->P, a->W, a->scale * 1.4426950408889634f,
                 static_cast<const T*>(a->q), static_cast<const T*>(a->k), static_cast<const T*>(a->v),
                 static_cast<T*>(a->o), static_cast<T*>(a->k_pages), static_cast<T*>(a->v_pages),
                 a->q_sb, a->q_st, a->q_sh, a->k_sb, a->k_st, a->k_sh, a->v_sb, a->v_st, a->v_sh,
                 a->o_sb, a->o_st, a->o_sh, a->kp_sp, a->kp_sh, a->kp_st, a->vp_sp, a->vp_sh, a->vp_st,
                 a->table, a->table_sb, a->lens, a->n_nodes, a->mask, a->mask_sb, err};
  const int64_t warps = (int64_t)a->B * a->T * a->Hq;
  fxb::pdl_launch(tree_attn_simple<T, D>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, fxb::as_stream(stream), p);
  return fxb::check_launch("fxb_tree_attn");
}

}  // namespace

extern "C" {

size_t fxb_tree_attn_workspace(int32_t, int32_t, int32_t, int32_t, int32_t, int32_t) { return 0; }
size_t fxb_tree_attn_workspace_zeroed(int32_t, int32_t, int32_t, int32_t, int32_t, int32_t) { return 0; }

int fxb_tree_attn(const fxb_tree_attn_args* a, void* stream) {
  if (!a) return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: args is NULL");
  const int e = fxb::dtype_size(a->dtype);
  if (!e) return fxb::set_error(FXB_EUNSUPPORTED, "fxb_tree_attn: dtype %d", a->dtype);
  if (a->D != 64 && a->D != 128) return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: head_dim %d (64 or 128)", a->D);
  if (a->B < 1 || a->T < 1 || a->T > kMaxTree || a->Hkv < 1 || a->Hq < 1 || a->Hq % a->Hkv)
    return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: B=%d T=%d (1..%d) Hq=%d Hkv=%d", a->B, a->T, kMaxTree, a->Hq,
                          a->Hkv);
  int shift = 0;
  for (int s = 4; s <= 8; ++s)
    if (a->page == 1 << s) shift = s;
  if (!shift) return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: page %d (16, 32, 64, 128 or 256)", a->page);
  if (a->P < 1 || a->W < 1 || a->table_sb < a->W || a->mask_sb < a->T)
    return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: P=%d W=%d, or a row stride of table or mask too small", a->P,
                          a->W);
  const void* ptr[6] = {a->q, a->k, a->v, a->o, a->k_pages, a->v_pages};
  for (const void* p : ptr)
    if (!p || !fxb::aligned16(p))
      return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: q, k, v, o and the pages must be 16-byte aligned");
  if (!a->table || !a->lens || !a->n_nodes || !a->mask)
    return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: table, lens, n_nodes or mask is NULL");
  const int64_t st[18] = {a->q_sb, a->q_st, a->q_sh, a->k_sb, a->k_st, a->k_sh, a->v_sb, a->v_st, a->v_sh,
                          a->o_sb, a->o_st, a->o_sh, a->kp_sp, a->kp_sh, a->kp_st, a->vp_sp, a->vp_sh, a->vp_st};
  for (int64_t s : st)
    if (s < 0 || (s * e) % 16)
      return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: strides must be multiples of 16 bytes");
  if (!(a->scale > 0.f) || !(a->scale < INFINITY))
    return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: scale must be positive and finite");
  int* err = fxb::dev_error_ptr();
  if (!err) return FXB_ECUDA;
  if (a->dtype == FXB_DTYPE_F32)
    return a->D == 64 ? launch<float, 64>(a, shift, err, stream) : launch<float, 128>(a, shift, err, stream);
  if (a->dtype == FXB_DTYPE_F16)
    return a->D == 64 ? launch<__half, 64>(a, shift, err, stream) : launch<__half, 128>(a, shift, err, stream);
  return a->D == 64 ? launch<__nv_bfloat16, 64>(a, shift, err, stream)
                    : launch<__nv_bfloat16, 128>(a, shift, err, stream);
}

}  // extern "C"
