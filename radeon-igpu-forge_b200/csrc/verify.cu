// Verification of a tree of drafted tokens against the target's probabilities
// (fxb_verify_tree). No reference counterpart: its sampler drafts nothing
// (ml/fxlm/sample.py:63-73).
//
// The walk over the tree needs a few probabilities of single tokens; whole
// rows are needed only where a residual is formed: the sum of max(w - q, 0)
// after a rejection, and the draw of the next token at the node where the walk
// ends. Every sum is taken over floor(w * 2^36) in 64-bit integers, so it does
// not depend on how the row is divided, and every other step is one rounded
// fp32 operation per element in a fixed order.
#include "common.cuh"
#include "internal.h"

namespace {

constexpr int kMaxTree = 64;
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr float kFix = 68719476736.f;  // 2^36

struct VerifyParams {
  const int64_t* tokens;
  const int32_t *parents, *n_nodes;
  const float *p, *q;
  int64_t p_sb, p_st, q_sb, q_st;
  const float* u;
  int32_t *path, *n_path;
  int64_t* next;
  int B, T, V;
};

FXB_DEV long long fixed(float w) { return __float2ll_rz((w > 0.f ? fminf(w, 1.f) : 0.f) * kFix); }

// what is left of probability w after its node's row lost `k` drawn children:
// the residual is not yet divided by its sum (scale[j] = 1 / sum of step j)
FXB_DEV float residual(float w, float q, const float* scale, int k) {
  for (int j = 0; j < k; ++j) {
    const float r = __fsub_rn(__fmul_rn(w, scale[j]), q);
    w = r > 0.f ? r : 0.f;
  }
  return w;
}

struct Shared {
  int par[kMaxTree];
  int64_t tok[kMaxTree];
  float u[kMaxTree], pv[kMaxTree], qv[kMaxTree];
  float scale[kMaxTree + 1];   // with q: 1, then 1 / sum after each rejection at the current node
  int64_t gone[kMaxTree];      // without q: rejected tokens of the current node, each once
  long long part[kWarps];
  int cur, child, rejected, n_gone, done;
  long long total;
};

// Sum over the row of what the current node has left, per warp in s.part
// (warp w owns the w-th run of `run` tokens); returns after a barrier.
FXB_DEV void row_sums(const VerifyParams& a, Shared& s, const float* p, const float* q, int run, int k, int n_gone) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lo = min(a.V, warp * run), hi = min(a.V, lo + run);
  long long sum = 0;
#pragma unroll 4
  for (int i = lo + lane; i < hi; i += 32) sum += fixed(k ? residual(p[i], q[i], s.scale, k) : p[i]);
  for (int j = lane; j < n_gone; j += 32) {
    const int64_t x = s.gone[j];
    if (x >= lo && x < hi) sum -= fixed(p[x]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s.part[warp] = sum;
  __syncthreads();
}

template <bool DRAFT>
__global__ void __launch_bounds__(kThreads) verify_tree_kernel(const VerifyParams a) {
  __shared__ Shared s;
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  const int n = min(max(a.n_nodes[b], 0), a.T);
  int32_t* path = a.path + (int64_t)b * a.T;
  for (int i = tid; i < a.T; i += kThreads) path[i] = i == 0 && n > 0 ? 0 : -1;
  if (n == 0) {
    if (tid == 0) {
      a.n_path[b] = 0;
      a.next[b] = -1;
    }
    return;
  }
  const float* P = a.p + b * a.p_sb;
  const float* Q = DRAFT ? a.q + b * a.q_sb : nullptr;
  if (tid < n) {
    const int par = tid ? a.parents[(int64_t)b * a.T + tid] : -1;
    const int64_t x = a.tokens[(int64_t)b * a.T + tid];
    const bool in = x >= 0 && x < a.V && par >= 0 && par < tid;
    s.par[tid] = par;
    s.tok[tid] = x;
    s.u[tid] = a.u[(int64_t)b * a.T + tid];
    s.pv[tid] = in ? P[par * a.p_st + x] : 0.f;
    s.qv[tid] = DRAFT && in ? Q[par * a.q_st + x] : 0.f;
  }
  if (tid == 0) {
    s.cur = s.rejected = s.n_gone = s.done = 0;
    s.child = 1;
    s.scale[0] = 1.f;
  }
  __syncthreads();
  const int run = (a.V + kWarps - 1) / kWarps;
  int n_path = 1;
  while (true) {
    if (tid == 0) {
      // one sweep in index order: the children of a node the walk reaches come after it
      int c = s.child, cur = s.cur, k = s.rejected, ng = s.n_gone;
      float mass = 1.f;  // without q: what the current node has left (one sweep does it all)
      bool stop = false;
      for (; c < n && !stop; ++c) {
        if (s.par[c] != cur) continue;
        bool take;
        if (DRAFT) {
          float w = residual(s.pv[c], s.qv[c], s.scale, k);
          w = w > 0.f ? w : 0.f;
          take = __fmul_rn(s.u[c], s.qv[c]) < __fmul_rn(w, s.scale[k]);
          if (!take) {
            ++k;
            stop = true;  // the sum of the residual is needed
          }
        } else {
          float w = s.pv[c] > 0.f ? fminf(s.pv[c], 1.f) : 0.f;
          bool seen = false;
          for (int j = 0; j < ng; ++j) seen |= s.gone[j] == s.tok[c];
          if (seen) w = 0.f;
          take = __fmul_rn(s.u[c], mass) < w;
          if (!take) {
            mass = fmaxf(__fsub_rn(mass, w), 0.f);
            if (!seen && s.tok[c] >= 0 && s.tok[c] < a.V) s.gone[ng++] = s.tok[c];
          }
        }
        if (take) {
          cur = c;
          path[n_path++] = c;
          k = ng = 0;
          mass = 1.f;
        }
      }
      s.child = c;
      s.cur = cur;
      s.rejected = k;
      s.n_gone = ng;
      s.done = !stop;
    }
    __syncthreads();
    if (s.done) break;
    // the sum of what is left after rejection number s.rejected
    const int k = s.rejected;
    row_sums(a, s, P + s.cur * a.p_st, Q + s.cur * a.q_st, run, k, 0);
    if (tid == 0) {
      long long total = 0;
      for (int w = 0; w < kWarps; ++w) total += s.part[w];
      if (total == 0) {
        s.child = n;  // nothing left: no further child can be accepted
      } else {
        s.scale[k] = __fdiv_rn(1.f, __fmul_rn(__ll2float_rn(total), 1.f / kFix));
      }
    }
    __syncthreads();
  }
  // the next token, from what is left of the last node's row
  const float* p = P + s.cur * a.p_st;
  const float* q = DRAFT ? Q + s.cur * a.q_st : nullptr;
  int k = s.rejected, n_gone = s.n_gone;
  for (int attempt = 0;; ++attempt) {
    row_sums(a, s, p, q, run, k, n_gone);
    if (tid == 0) {
      long long total = 0;
      for (int w = 0; w < kWarps; ++w) total += s.part[w];
      s.total = total;
    }
    __syncthreads();
    if (s.total || attempt || (k == 0 && n_gone == 0)) break;
    k = n_gone = 0;  // nothing left: the row itself
    __syncthreads();
  }
  if (tid == 0) a.n_path[b] = n_path;
  const long long total = s.total;
  if (total == 0) {
    if (tid == 0) a.next[b] = -1;
    return;
  }
  // floor(total * u) with u in 2^-24ths, without the 64-bit product's overflow
  const float uf = __fmul_rn(s.u[0], 16777216.f);
  const long long ku = uf > 0.f ? (uf < 16777215.f ? __float2ll_rz(uf) : 16777215LL) : 0LL;
  const long long thr = (total >> 24) * ku + (((total & 0xffffff) * ku) >> 24);
  if (tid < 32) {
    int w = 0;
    long long before = 0;
    while (before + s.part[w] <= thr) before += s.part[w++];
    const int lo = w * run, hi = min(a.V, lo + run);
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const int i = i0 + lane;
      long long f = 0;
      if (i < hi) {
        f = fixed(DRAFT && k ? residual(p[i], q[i], s.scale, k) : p[i]);
        for (int j = 0; j < n_gone; ++j)
          if (s.gone[j] == i) f = 0;
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, f, o);
        if (lane >= o) f += y;
      }
      const unsigned m = __ballot_sync(0xffffffffu, before + f > thr);
      if (m) {
        if (lane == 0) a.next[b] = i0 + __ffs(m) - 1;
        break;
      }
      before += __shfl_sync(0xffffffffu, f, 31);
    }
  }
}

}  // namespace

extern "C" int fxb_verify_tree(const int64_t* tokens, const int32_t* parents, const int32_t* n_nodes, const float* p,
                               int64_t p_sb, int64_t p_st, const float* q, int64_t q_sb, int64_t q_st, const float* u,
                               int32_t* path, int32_t* n_path, int64_t* next, int32_t B, int32_t T, int32_t V,
                               void* stream) {
  if (B < 1 || T < 1 || T > kMaxTree || V < 1)
    return fxb::set_error(FXB_EINVAL, "fxb_verify_tree: B=%d T=%d (1..%d) V=%d", B, T, kMaxTree, V);
  if (!tokens || !parents || !n_nodes || !p || !u || !path || !n_path || !next)
    return fxb::set_error(FXB_EINVAL, "fxb_verify_tree: a required array is NULL");
  if (p_st < 0 || p_sb < 0 || (q && (q_st < 0 || q_sb < 0)))
    return fxb::set_error(FXB_EINVAL, "fxb_verify_tree: negative stride");
  const VerifyParams a = {tokens, parents, n_nodes, p, q, p_sb, p_st, q_sb, q_st, u, path, n_path, next, B, T, V};
  if (q)
    fxb::pdl_launch(verify_tree_kernel<true>, dim3(B), dim3(kThreads), 0, fxb::as_stream(stream), a);
  else
    fxb::pdl_launch(verify_tree_kernel<false>, dim3(B), dim3(kThreads), 0, fxb::as_stream(stream), a);
  return fxb::check_launch("fxb_verify_tree");
}
