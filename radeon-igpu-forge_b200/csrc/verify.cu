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
//
// What bounds it: latency. One row of 8 nodes and 32768 tokens takes 4.9 us
// (131 kB), 64 rows of 32 nodes and 50257 tokens 21.4 us (25.8 MB, 3.9 us at a
// copy's rate): up to four rejections in a row, each of which needs the sum
// that the one before it left, and the same row again, from L2.
#include "common.cuh"
#include "internal.h"

namespace {

constexpr int kMaxTree = 64;
constexpr int kMaxThreads = 512, kMaxWarps = kMaxThreads / 32;
constexpr int kMaxCluster = 8;
constexpr float kFix = 68719476736.f;  // 2^36

struct VerifyParams {
  const int64_t* tokens;
  const int32_t *parents, *n_nodes;
  const float *p, *q;
  int64_t p_sb, p_st, q_sb, q_st;
  const float* u;
  int32_t *path, *n_path;
  int64_t* next;
  int B, T, V, cluster;
  int* err;
};

// floor(w * 2^36) of w in [0, 1] (clamped; NaN is 0) in two halves of 18 bits: adding 2^23 with rounding
// towards zero leaves the whole part of a number below it in the low bits. All steps are exact; the 64-bit
// conversion would go through a pipe of a sixteenth of the rate.
FXB_DEV void fixed_add(float w, int& hi, int& lo) {
  const float t = (w > 0.f ? fminf(w, 1.f) : 0.f) * 262144.f;
  const float h = __fadd_rz(t, 8388608.f);
  const float l = __fadd_rz((t - (h - 8388608.f)) * 262144.f, 8388608.f);
  hi += __float_as_int(h) - 0x4b000000;
  lo += __float_as_int(l) - 0x4b000000;
}
FXB_DEV long long fixed(float w) {
  int hi = 0, lo = 0;
  fixed_add(w, hi, lo);
  return ((long long)hi << 18) + lo;
}

// one rejection's step: what is left of probability w * f (f: 1 / the sum of what was left before) without q
FXB_DEV float less(float w, float f, float q) {
  const float r = __fsub_rn(__fmul_rn(w, f), q);
  return r > 0.f ? r : 0.f;
}

// One cluster of thread blocks a row: each block sums a slice of the
// vocabulary. Block 0 alone decides (its first warp walks the tree) and tells
// the others, so all blocks take the same steps. Decisions and sums go into the
// other blocks' shared memory by st.async, which completes on a barrier there:
// a cluster-wide barrier took 0.9 us a time.
struct Shared {
  int par[kMaxTree];
  int64_t tok[kMaxTree];
  float u[kMaxTree], pv[kMaxTree], qv[kMaxTree];
  float scale[kMaxTree + 1];  // with q: 1, then 1 / sum after each rejection at the current node
  long long part[kMaxWarps];     // sums of this block's warps
  // what block 0 decided (current node, rejections at it, whether the walk is over), and without q the nodes
  // whose tokens the current node has lost, each token once
  uint64_t told[2];
  long long slice[2][kMaxCluster];  // sums of all blocks, in turn
  uint64_t told_bar, slice_bar[2];
  int failed;                 // a wait has expired
};

FXB_DEV void put(void* local, int rank, uint64_t value, uint64_t* bar) {  // into the same place of another block
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(
                   mapa_shared(smem_u32(local), rank)),
               "l"(value), "r"(mapa_shared(smem_u32(bar), rank))
               : "memory");
}

constexpr int kAtOnce = 16;  // elements of a thread under way

template <bool DRAFT>
__global__ void __launch_bounds__(kMaxThreads, 2) verify_tree_kernel(const VerifyParams a) {
  __shared__ Shared s;
  const int rank = cluster_ctarank(), ranks = a.cluster, b = blockIdx.x / ranks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  if (tid == 0) {
    mbar_init(smem_u32(&s.told_bar), 1);
    mbar_init(smem_u32(&s.slice_bar[0]), 1);
    mbar_init(smem_u32(&s.slice_bar[1]), 1);
    fence_mbar_init();
    mbar_expect_tx(smem_u32(&s.told_bar), 16);
    mbar_expect_tx(smem_u32(&s.slice_bar[0]), 8 * ranks);
    mbar_expect_tx(smem_u32(&s.slice_bar[1]), 8 * ranks);
    s.scale[0] = 1.f;
    s.failed = 0;
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  pdl_trigger();
  pdl_wait();
  const float* P = a.p + b * a.p_sb;
  const float* Q = DRAFT ? a.q + b * a.q_sb : nullptr;
  int32_t* path = a.path + (int64_t)b * a.T;
  const int n_in = a.n_nodes[b];
  if (tid < a.T) {
    const int64_t x = a.tokens[(int64_t)b * a.T + tid];
    s.tok[tid] = x;
    if (rank == 0) {
      const int par = tid ? a.parents[(int64_t)b * a.T + tid] : -1;
      const bool in = x >= 0 && x < a.V && par >= 0 && par < tid;
      s.par[tid] = par;
      s.u[tid] = a.u[(int64_t)b * a.T + tid];
      s.pv[tid] = in ? P[par * a.p_st + x] : 0.f;
      s.qv[tid] = DRAFT && in ? Q[par * a.q_st + x] : 0.f;
    }
  }
  const int n = min(max(n_in, 0), a.T);
  const int per = (a.V + ranks - 1) / ranks, run = (per + warps - 1) / warps;
  const int first = min(a.V, rank * per), count = min(a.V, first + per) - first;
  __syncthreads();
  // all blocks run and their barriers are ready
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  // the walk's state, in the registers of block 0's first warp: the nodes' parents, a lane two
  int par0 = -2, par1 = -2, n_path = 1, cur = 0, k = 0;
  uint64_t later = ~1ull;  // nodes not yet met: the children of a node come after it
  uint64_t gone = 0;
  if (rank == 0 && warp == 0) {
    if (lane && lane < n) par0 = s.par[lane];
    if (lane + 32 < n) par1 = s.par[lane + 32];
    for (int i = lane; i < a.T; i += 32) path[i] = i == 0 && n > 0 ? 0 : -1;
    __syncwarp();
  }
  int turn = 0;
  unsigned told_phase = 0, slice_phase = 0;  // parities (slice: bit `turn`)
  const float *p = nullptr, *q = nullptr;
  bool ok = true;

  // One thread polls, the block's others wait at its barrier and leave the SM to blocks with work.
  auto wait = [&](uint64_t* bar, unsigned parity) {
    if (tid == 0 && !mbar_wait(smem_u32(bar), parity, a.err, FXB_DERR_VERIFY_WAIT)) s.failed = 1;
    __syncthreads();
    ok = !s.failed;
  };
  // The sum over the row of what the current node has left: of this block's warps in s.part (warp w owns the
  // w-th run of the slice), of the blocks in s.slice[turn], and in all.
  auto row_sum = [&]() -> long long {
    const int lo = first + min(count, warp * run), hi = first + min(count, warp * run + run);
    long long sum = 0;
#pragma unroll 1
    for (int i0 = lo + lane; i0 < hi; i0 += 32 * kAtOnce) {
      float w[kAtOnce], d[kAtOnce];
      // past the end: 0, which adds nothing
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) w[x] = i0 + 32 * x < hi ? p[i0 + 32 * x] : 0.f;
      if (DRAFT && k) {
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) d[x] = i0 + 32 * x < hi ? q[i0 + 32 * x] : 0.f;
#pragma unroll 1
        for (int j = 0; j < k; ++j) {
          const float f = s.scale[j];
#pragma unroll
          for (int x = 0; x < kAtOnce; ++x) w[x] = less(w[x], f, d[x]);
        }
      }
      int h = 0, l = 0;
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) fixed_add(w[x], h, l);
      sum += ((long long)h << 18) + l;
    }
    if (!DRAFT)
      for (uint64_t g = gone; g; g &= g - 1) {
        const int64_t x = s.tok[__ffsll(g) - 1];
        if (lane == 0 && x >= lo && x < hi) sum -= fixed(p[x]);
      }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s.part[warp] = sum;
    __syncthreads();
    if (tid < 32) {
      long long all = tid < warps ? s.part[tid] : 0;
#pragma unroll
      for (int o = kMaxWarps / 2; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      all = __shfl_sync(0xffffffffu, all, 0);
      if (tid < ranks) put(&s.slice[turn][rank], tid, all, &s.slice_bar[turn]);
    }
    wait(&s.slice_bar[turn], (slice_phase >> turn) & 1);
    slice_phase ^= 1u << turn;
    long long total = 0;
    for (int c = 0; c < ranks; ++c) total += s.slice[turn][c];
    return total;
  };

  while (true) {
    if (rank == 0 && warp == 0) {
      float mass = 1.f;  // without q: what the current node has left (one sweep does it all)
      bool more = false;
      while (true) {
        const uint64_t kids = (((uint64_t)__ballot_sync(0xffffffffu, par1 == cur) << 32) |
                               __ballot_sync(0xffffffffu, par0 == cur)) & later;
        if (!kids) break;
        const int c = __ffsll(kids) - 1;
        later = c == 63 ? 0 : ~0ull << (c + 1);
        bool take;
        if (DRAFT) {
          float w = s.pv[c];
          for (int j = 0; j < k; ++j) w = less(w, s.scale[j], s.qv[c]);
          w = w > 0.f ? w : 0.f;
          take = __fmul_rn(s.u[c], s.qv[c]) < __fmul_rn(w, s.scale[k]);
          if (!take) {
            ++k;
            more = (kids & later) != 0;  // the sum of the residual is needed, if another child is to be tried
          }
        } else {
          const int64_t x = s.tok[c];
          float w = s.pv[c] > 0.f ? fminf(s.pv[c], 1.f) : 0.f;
          bool seen = false;
          for (uint64_t g = gone; g; g &= g - 1) seen |= s.tok[__ffsll(g) - 1] == x;
          if (seen) w = 0.f;
          take = __fmul_rn(s.u[c], mass) < w;
          if (!take) {
            mass = fmaxf(__fsub_rn(mass, w), 0.f);
            if (!seen && x >= 0 && x < a.V) gone |= 1ull << c;
          }
        }
        if (take) {
          cur = c;
          if (lane == 0) path[n_path] = c;
          ++n_path;
          k = 0;
          gone = 0;
          mass = 1.f;
        } else if (DRAFT) {
          break;
        }
      }
      if (lane < ranks) {
        put(&s.told[0], lane, (uint64_t)cur | (uint64_t)k << 8 | (uint64_t)(more ? 0 : 1) << 16, &s.told_bar);
        put(&s.told[1], lane, gone, &s.told_bar);
      }
    }
    wait(&s.told_bar, told_phase);
    told_phase ^= 1;
    const uint64_t told = s.told[0];
    k = (int)(told >> 8) & 255;
    gone = s.told[1];
    p = P + (told & 255) * a.p_st;
    q = DRAFT ? Q + (told & 255) * a.q_st : nullptr;
    if (!ok || (told >> 16)) break;
    const long long total = row_sum();
    // everyone has read what was told and summed (row_sum's barriers are armed again by then)
    __syncthreads();
    if (tid == 0) {
      mbar_expect_tx(smem_u32(&s.told_bar), 16);
      mbar_expect_tx(smem_u32(&s.slice_bar[turn]), 8 * ranks);
      s.scale[k] = total ? __fdiv_rn(1.f, __fmul_rn(__ll2float_rn(total), 1.f / kFix)) : 0.f;
    }
    __syncthreads();
    turn ^= 1;
    if (total == 0) later = 0;  // nothing left: no further child can be accepted
  }
  // the next token, from what is left of the last node's row, or from the row itself where nothing is left
  long long total = n && ok ? row_sum() : 0;
  if (n && ok && total == 0 && (k || gone)) {
    turn ^= 1;
    k = 0;
    gone = 0;
    __syncthreads();  // s.part has been read
    total = row_sum();
  }
  if (rank == 0 && tid == 0) {
    a.n_path[b] = n ? n_path : 0;
    if (n != n_in) atomicOr(a.err, FXB_DERR_PAGES);
  }
  if (total == 0 || !ok) {
    if (rank == 0 && tid == 0) a.next[b] = -1;
    return;
  }
  // floor(total * u) with u in 2^-24ths, without the 64-bit product's overflow
  const float uf = __fmul_rn(a.u[(int64_t)b * a.T], 16777216.f);
  const long long ku = uf > 0.f ? (uf < 16777215.f ? __float2ll_rz(uf) : 16777215LL) : 0LL;
  long long rest = (total >> 24) * ku + (((total & 0xffffff) * ku) >> 24);
  for (int c = 0; c < rank; ++c) rest -= s.slice[turn][c];
  if (rest < 0 || rest >= s.slice[turn][rank]) return;  // another block's slice
  int w = 0;
  while (rest >= s.part[w]) rest -= s.part[w++];
  // the run of warp w, divided over the warps again
  const int run_lo = first + min(count, w * run), run_hi = first + min(count, w * run + run);
  const int sub = (run_hi - run_lo + warps - 1) / warps;
  const int lo = min(run_hi, run_lo + warp * sub), hi = min(run_hi, lo + sub);
  auto left = [&](int i) -> long long {
    if (i >= hi) return 0;
    float x = p[i];
    if (DRAFT && k) {
      const float d = q[i];
      for (int j = 0; j < k; ++j) x = less(x, s.scale[j], d);
    }
    if (!DRAFT)
      for (uint64_t g = gone; g; g &= g - 1)
        if (s.tok[__ffsll(g) - 1] == i) x = 0.f;
    return fixed(x);
  };
  long long sum = 0;
#pragma unroll 4
  for (int i = lo + lane; i < hi; i += 32) sum += left(i);
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();  // s.part has been read
  if (lane == 0) s.part[warp] = sum;
  __syncthreads();
  for (int x = 0; x < warp; ++x) rest -= s.part[x];
  if (rest < 0 || rest >= s.part[warp]) return;
  for (int i0 = lo; i0 < hi; i0 += 32) {
    long long f = left(i0 + lane);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, f, o);
      if (lane >= o) f += y;
    }
    const unsigned m = __ballot_sync(0xffffffffu, f > rest);
    if (m) {
      if (lane == 0) a.next[b] = i0 + __ffs(m) - 1;
      return;
    }
    rest -= __shfl_sync(0xffffffffu, f, 31);
  }
}

// Thread blocks of a cluster: one for every 4096 tokens of the vocabulary, at
// most 8 (a portable cluster; 64 rows of 50257: 21.4 us with 8 blocks of 256
// threads, 27.1 with 4, 36.8 with 2, 55.8 with 1). Threads of a block: 256,
// four blocks an SM, and a thread's 16 elements of 32768 all under way at once
// (one row: 4.9 us, 5.6 with 512 threads); 512 for longer slices while every
// block has an SM to itself.
int cluster_of(int V) {
  int c = 1;
  while (c < kMaxCluster && V > c * 4096) c *= 2;
  return c;
}

template <bool DRAFT> int launch(const VerifyParams& a, void* stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.B * a.cluster));
  const bool alone = (int64_t)a.B * a.cluster <= fxb::num_sms();
  cfg.blockDim = dim3(alone && a.V > a.cluster * kAtOnce * kMaxThreads / 2 ? kMaxThreads : kMaxThreads / 2);
  cfg.stream = fxb::as_stream(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = fxb::pdl_enabled() ? 2 : 1;
  (void)cudaLaunchKernelEx(&cfg, verify_tree_kernel<DRAFT>, a);
  return fxb::check_launch("fxb_verify_tree");
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
  if ((int64_t)B * kMaxCluster > 0x7fffffff) return fxb::set_error(FXB_EINVAL, "fxb_verify_tree: B=%d", B);
  int* err = fxb::dev_error_ptr();
  if (!err) return FXB_ECUDA;
  const VerifyParams a = {tokens, parents, n_nodes, p, q, p_sb, p_st, q_sb, q_st, u, path, n_path, next,
                          B, T, V, cluster_of(V), err};
  return q ? launch<true>(a, stream) : launch<false>(a, stream);
}
