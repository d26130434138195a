// Pages of a KV cache: committing accepted tokens, making room, forking and
// freeing sequences (fxb_kv_commit, fxb_kv_fork). No reference counterpart:
// its sampler keeps no cache (ml/fxlm/sample.py:63-73).
//
// Both operators move whole token rows (D elements, a multiple of 16 bytes)
// between slots of the pool, in every layer, and update the page table. They
// are bound by latency for a few sequences (commit of 8 tokens of one sequence
// in 12 layers 3.0 us; four samples of one prompt 6.3 us, two kernels) and by
// HBM for many (commit of 64 sequences in 32 layers, 67 MB: 12.8 us, 0.80 of a
// copy's rate; 48 beams in 32 layers, 291 MB: 52.5 us, 0.85).
#include "common.cuh"
#include "internal.h"

namespace {

constexpr int kThreads = 512;
constexpr int kMaxTree = 64;    // tokens of a path (nodes of a tree)
constexpr int kMaxRows = 4096;  // rows of the page table (their offsets stand in shared memory)

struct Pool {  // strides in bytes
  uint8_t* p;
  int64_t sl, sp, sh, st;
};

struct KvParams {
  Pool k, v;
  int L, P, H, page_shift, chunks;  // chunks: 16-byte pieces of a token row
  int S, W;
  int32_t* table;
  int64_t table_ss;
  int32_t *n_pages, *lens, *ref;
  int* err;
};

// Exclusive prefix sum over the block (kThreads threads); *total for everyone.
FXB_DEV int block_scan(int v, int* total) {
  __shared__ int warp_sum_[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the previous use of warp_sum_ is over
  if (lane == 31) warp_sum_[warp] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const int s = warp_sum_[w];
    before += w < warp ? s : 0;
    all += s;
  }
  *total = all;
  return before + x - v;
}

// Hands out the `total` lowest-numbered free pages: give(rank, page) once for
// every rank in [0, total). False, and no call, if fewer are free. Each thread
// scans a run of pages of its own, so that all loads are in flight at once.
template <typename Give>
FXB_DEV bool lowest_free_pages(const int32_t* ref, int P, int total, Give give) {
  const int run = ((P + kThreads * 4 - 1) / (kThreads * 4)) * 4;
  const int lo = min(P, (int)threadIdx.x * run), hi = min(P, lo + run);
  int mine = 0;
#pragma unroll 4
  for (int i = lo; i < hi; ++i) mine += ref[i] == 0;
  int all;
  int rank = block_scan(mine, &all);
  if (all < total) return false;
  if (mine && rank < total)
    for (int i = lo; i < hi && rank < total; ++i)
      if (ref[i] == 0) give(rank++, i);
  return true;
}

// ------------------------------------------------------------------ commit
// Blocks [0, gx * S) move tokens, gx blocks a row of the table: a thread owns
// one 16-byte piece of a token row in one (layer, key or value, head) and takes
// the path's tokens in ascending order, kBatch loads before their stores. Since
// path[i] >= i, what a store overwrites was read before it, by this thread.
// The last block updates lengths and pages; the movers read the old lengths
// and only table entries that were there before, so nothing waits for it.
constexpr int kBatch = 8;

__global__ void __launch_bounds__(kThreads) kv_commit_kernel(KvParams c, const int32_t* path, int64_t path_ss,
                                                             int T, const int32_t* n_path, const int32_t* room,
                                                             int32_t* lens_out, int gx) {
  pdl_trigger();
  pdl_wait();
  const int page = 1 << c.page_shift;
  if ((int)blockIdx.x < gx * c.S) {
    __shared__ int64_t from[2][kMaxTree], to[2][kMaxTree];
    __shared__ int moves;
    const int s = blockIdx.x / gx, bx = blockIdx.x - s * gx;
    const int n = min(max(n_path[s], 0), T), len = c.lens[s], held = min(max(c.n_pages[s], 0), c.W);
    if (threadIdx.x < 32) {  // the list of moves: tokens that change place, in order
      int count = 0;
      for (int i0 = 0; i0 < n; i0 += 32) {
        const int i = i0 + threadIdx.x;
        bool move = false, bad = false;
        int64_t src = 0, dst = 0;
        int sp = -1, dp = -1;
        if (i < n) {
          const int p = path[s * path_ss + i];
          const int before = i ? path[s * path_ss + i - 1] : -1;
          bad = p <= before || p < i || p >= T;
          if (!bad && p != i) {
            src = (int64_t)len + p;
            dst = (int64_t)len + i;
            bad = len < 0 || (src >> c.page_shift) >= held;
            if (!bad) {
              sp = c.table[s * c.table_ss + (src >> c.page_shift)];
              dp = c.table[s * c.table_ss + (dst >> c.page_shift)];
              bad = sp < 0 || sp >= c.P || dp < 0 || dp >= c.P;
              move = !bad;
            }
          }
        }
        if (bad) atomicOr(c.err, FXB_DERR_PAGES);
        const unsigned m = __ballot_sync(0xffffffffu, move);
        if (move) {
          const int at = count + __popc(m & ((1u << threadIdx.x) - 1));
          const int so = (int)(src & (page - 1)), d = (int)(dst & (page - 1));
          from[0][at] = sp * c.k.sp + so * c.k.st;
          from[1][at] = sp * c.v.sp + so * c.v.st;
          to[0][at] = dp * c.k.sp + d * c.k.st;
          to[1][at] = dp * c.v.sp + d * c.v.st;
        }
        count += __popc(m);
      }
      if (threadIdx.x == 0) moves = count;
    }
    __syncthreads();
    const int nm = moves;
    const int64_t x = (int64_t)bx * kThreads + threadIdx.x;
    const int ch = (int)(x % c.chunks);
    int64_t y = x / c.chunks;
    const int h = (int)(y % c.H);
    y /= c.H;
    const int kv = (int)(y & 1), l = (int)(y >> 1);
    if (l >= c.L) return;
    const Pool& pool = kv ? c.v : c.k;
    uint8_t* base = pool.p + l * pool.sl + h * pool.sh + ch * 16;
    for (int i0 = 0; i0 < nm; i0 += kBatch) {
      uint4 r[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + j < nm) r[j] = *reinterpret_cast<const uint4*>(base + from[kv][i0 + j]);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + j < nm) *reinterpret_cast<uint4*>(base + to[kv][i0 + j]) = r[j];
    }
    return;
  }
  // lengths, and pages for the rows that want room
  __shared__ int off[kMaxRows];
  int total = 0;
  for (int s0 = 0; s0 < c.S; s0 += kThreads) {
    const int s = s0 + threadIdx.x;
    int add = 0;
    if (s < c.S) {
      const int n_in = path ? n_path[s] : 0, n = min(max(n_in, 0), T);
      if (n != n_in) atomicOr(c.err, FXB_DERR_PAGES);
      const int len = c.lens[s] + n;
      lens_out[s] = len;
      const int want = room ? room[s] : 0;
      if (want > 0) {
        int64_t need = ((int64_t)len + want + page - 1) >> c.page_shift;
        if (need > c.W) {
          atomicOr(c.err, FXB_DERR_PAGES);
          need = c.W;
        }
        add = max(0, (int)need - max(c.n_pages[s], 0));
      }
    }
    int all;
    const int before = block_scan(add, &all);
    if (s < c.S) off[s] = total + before;
    total = all > c.P - total ? c.P + 1 : total + all;  // more than the pool has: stays so (every length is written)
  }
  if (total == 0) return;
  __syncthreads();
  bool ok = total <= c.P;
  if (ok)
    ok = lowest_free_pages(c.ref, c.P, total, [&](int rank, int pg) {
      int lo = 0, hi = c.S - 1;  // the last row whose pages start at or before rank
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (off[mid] <= rank) lo = mid;
        else hi = mid - 1;
      }
      c.table[lo * c.table_ss + max(c.n_pages[lo], 0) + rank - off[lo]] = pg;
      c.ref[pg] = 1;
    });
  if (!ok) {
    if (threadIdx.x == 0) atomicOr(c.err, FXB_DERR_PAGES);
    return;
  }
  __syncthreads();  // every n_pages above has been read
  for (int s = threadIdx.x; s < c.S; s += kThreads) {
    const int end = s + 1 < c.S ? off[s + 1] : total;
    if (end > off[s]) c.n_pages[s] = max(c.n_pages[s], 0) + end - off[s];
  }
}

// ------------------------------------------------------------------ fork
// Workspace: a copy of the table (S x W), then per row what the plan says.
struct ForkPlan {
  int32_t* snap;   // S x W
  int32_t* old_n;  // pages held before
  int32_t* from;   // the row it forks from, -1: emptied
  int32_t* held;   // its length
  int32_t* fresh;  // its own copy of the last page, -1: none
  int32_t* ok;     // 1: the plan holds
};
__host__ __device__ inline ForkPlan fork_plan(void* ws, int S, int W) {
  ForkPlan f;
  f.snap = static_cast<int32_t*>(ws);
  f.old_n = f.snap + (int64_t)S * W;
  f.from = f.old_n + S;
  f.held = f.from + S;
  f.fresh = f.held + S;
  f.ok = f.fresh + S;
  return f;
}

// First kernel: block 0 plans, the others copy the table (rows are read by
// other rows after they have been overwritten).
__global__ void __launch_bounds__(kThreads) kv_fork_plan_kernel(KvParams c, const int32_t* parents, ForkPlan f) {
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x > 0) {
    const int64_t n = (int64_t)c.S * c.W;
    for (int64_t i = (int64_t)(blockIdx.x - 1) * kThreads + threadIdx.x; i < n;
         i += (int64_t)(gridDim.x - 1) * kThreads)
      f.snap[i] = c.table[(i / c.W) * c.table_ss + i % c.W];
    return;
  }
  __shared__ int heir[kMaxRows];   // who keeps a row's last page; -1: the row itself
  __shared__ int taker[kMaxRows];  // the row that gets the page of this rank
  __shared__ int bad;
  if (threadIdx.x == 0) bad = 0;
  for (int s = threadIdx.x; s < c.S; s += kThreads) heir[s] = 0x7fffffff;
  __syncthreads();
  for (int s = threadIdx.x; s < c.S; s += kThreads) {
    const int p = parents[s];
    if (p < -1 || p >= c.S) atomicOr(&bad, 1);
    else if (p >= 0) atomicMin(&heir[p], p == s ? -1 : s);
  }
  __syncthreads();
  bool ok = !bad;
  int total = 0;
  if (ok) {
    for (int s0 = 0; s0 < c.S; s0 += kThreads) {
      const int s = s0 + threadIdx.x;
      int copy = 0;
      if (s < c.S) {
        const int p = parents[s];
        const int held = p >= 0 ? max(c.lens[p], 0) : 0;
        const int keeper = p >= 0 ? (heir[p] < 0 ? p : heir[p]) : s;
        copy = (held & ((1 << c.page_shift) - 1)) != 0 && keeper != s;
        f.from[s] = p;
        f.held[s] = held;
        f.old_n[s] = min(max(c.n_pages[s], 0), c.W);
        f.fresh[s] = -1;
        // a length beyond the pages that its row holds
        if (p >= 0 && ((held + (1 << c.page_shift) - 1) >> c.page_shift) > min(max(c.n_pages[p], 0), c.W))
          atomicOr(&bad, 1);
      }
      int all;
      const int before = block_scan(copy, &all);
      if (copy) taker[total + before] = s;
      total += all;
    }
    __syncthreads();
    ok = !bad;
  }
  if (ok && total) ok = lowest_free_pages(c.ref, c.P, total, [&](int rank, int pg) { f.fresh[taker[rank]] = pg; });
  if (threadIdx.x == 0) {
    *f.ok = ok ? 1 : 0;
    if (!ok) atomicOr(c.err, FXB_DERR_PAGES);
  }
}

// Second kernel: blocks [0, tb) write the table, the lengths and the counts
// (integer atomics: any order gives the same counts); the other warps copy the
// filled slots of one (row, layer, key or value, head) each. Sources were held
// before the call and destinations were free, so no copy reads what another
// one writes.
__global__ void __launch_bounds__(kThreads) kv_fork_kernel(KvParams c, ForkPlan f, int tb) {
  pdl_trigger();
  pdl_wait();
  if (!*f.ok) return;
  const int page = 1 << c.page_shift;
  if ((int)blockIdx.x < tb) {
    const int64_t n = (int64_t)c.S * c.W;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)tb * kThreads) {
      const int s = (int)(i / c.W), j = (int)(i - (int64_t)s * c.W);
      const int p = f.from[s], count = (f.held[s] + page - 1) >> c.page_shift;
      const int was = j < f.old_n[s] ? f.snap[i] : -1;
      int now = -1;
      if (j < count) now = j == count - 1 && f.fresh[s] >= 0 ? f.fresh[s] : f.snap[(int64_t)p * c.W + j];
      if (was != now) {
        if (was >= 0 && was < c.P) atomicSub(&c.ref[was], 1);
        if (now >= 0 && now < c.P) atomicAdd(&c.ref[now], 1);
      }
      c.table[s * c.table_ss + j] = now;
      if (j == 0) {
        c.n_pages[s] = count;
        c.lens[s] = f.held[s];
      }
    }
    return;
  }
  const int lane = threadIdx.x & 31;
  const int64_t units = (int64_t)c.S * c.L * 2 * c.H;
  const int64_t warps = (int64_t)(gridDim.x - tb) * (kThreads / 32);
  for (int64_t u = (int64_t)(blockIdx.x - tb) * (kThreads / 32) + (threadIdx.x >> 5); u < units; u += warps) {
    int64_t y = u;
    const int h = (int)(y % c.H);
    y /= c.H;
    const int kv = (int)(y & 1);
    y >>= 1;
    const int l = (int)(y % c.L), s = (int)(y / c.L);
    const int dst = f.fresh[s];
    if (dst < 0) continue;
    const int held = f.held[s];
    const int src = f.snap[(int64_t)f.from[s] * c.W + ((held - 1) >> c.page_shift)];
    if (src < 0 || src >= c.P) {
      if (lane == 0) atomicOr(c.err, FXB_DERR_PAGES);
      continue;
    }
    const Pool& pool = kv ? c.v : c.k;
    const uint8_t* a = pool.p + l * pool.sl + src * pool.sp + h * pool.sh;
    uint8_t* b = pool.p + l * pool.sl + dst * pool.sp + h * pool.sh;
    const int n = (held & (page - 1)) * c.chunks;
    for (int i0 = lane; i0 < n; i0 += 32 * kBatch) {
      uint4 r[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + 32 * j, t = i / c.chunks, ch = i - t * c.chunks;
        if (i < n) r[j] = *reinterpret_cast<const uint4*>(a + t * pool.st + ch * 16);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + 32 * j, t = i / c.chunks, ch = i - t * c.chunks;
        if (i < n) *reinterpret_cast<uint4*>(b + t * pool.st + ch * 16) = r[j];
      }
    }
  }
}

int page_shift_of(int page) {
  for (int s = 4; s <= 8; ++s)
    if (page == 1 << s) return s;
  return -1;
}

// `pools`: whether the call touches keys and values
int params(const char* fn, const fxb_kv_args* a, bool pools, KvParams* c) {
  if (!a) return fxb::set_error(FXB_EINVAL, "%s: args is NULL", fn);
  const int sh = page_shift_of(a->page);
  if (sh < 0) return fxb::set_error(FXB_EINVAL, "%s: page %d (16, 32, 64, 128 or 256)", fn, a->page);
  if (a->S < 1 || a->S > kMaxRows || a->W < 1 || a->P < 1)
    return fxb::set_error(FXB_EINVAL, "%s: S=%d (1..%d) W=%d P=%d", fn, a->S, kMaxRows, a->W, a->P);
  if (!a->table || !a->n_pages || !a->lens || !a->ref)
    return fxb::set_error(FXB_EINVAL, "%s: table, n_pages, lens or ref is NULL", fn);
  if (a->table_ss < a->W) return fxb::set_error(FXB_EINVAL, "%s: table row stride below W", fn);
  c->chunks = 1;
  if (pools) {
    const int e = a->elem_size;
    if (e != 2 && e != 4) return fxb::set_error(FXB_EINVAL, "%s: elem_size %d (2 or 4)", fn, e);
    if (a->L < 1 || a->H < 1 || a->D < 1 || (a->D * (int64_t)e) % 16)
      return fxb::set_error(FXB_EINVAL, "%s: L=%d H=%d D=%d (rows of a multiple of 16 bytes)", fn, a->L, a->H, a->D);
    if (!a->k || !a->v || !fxb::aligned16(a->k) || !fxb::aligned16(a->v))
      return fxb::set_error(FXB_EINVAL, "%s: k and v must be 16-byte aligned", fn);
    const struct { int64_t entries, stride; } st[8] = {  // the stride of an axis of one entry is not used
        {a->L, a->k_sl}, {a->P, a->k_sp}, {a->H, a->k_sh}, {a->page, a->k_st},
        {a->L, a->v_sl}, {a->P, a->v_sp}, {a->H, a->v_sh}, {a->page, a->v_st}};
    for (const auto& x : st)
      if (x.entries > 1 && (x.stride < 0 || (x.stride * e) % 16))
        return fxb::set_error(FXB_EINVAL, "%s: strides must be multiples of 16 bytes", fn);
    c->k = {static_cast<uint8_t*>(a->k), a->k_sl * e, a->k_sp * e, a->k_sh * e, a->k_st * e};
    c->v = {static_cast<uint8_t*>(a->v), a->v_sl * e, a->v_sp * e, a->v_sh * e, a->v_st * e};
    c->chunks = (int)(a->D * (int64_t)e / 16);
  }
  c->L = a->L;
  c->P = a->P;
  c->H = a->H;
  c->page_shift = sh;
  c->S = a->S;
  c->W = a->W;
  c->table = a->table;
  c->table_ss = a->table_ss;
  c->n_pages = a->n_pages;
  c->lens = a->lens;
  c->ref = a->ref;
  return FXB_OK;
}

}  // namespace

extern "C" {

int fxb_kv_commit(const fxb_kv_args* args, const int32_t* path, int64_t path_ss, int32_t T, const int32_t* n_path,
                  const int32_t* room, int32_t* lens_out, void* stream) {
  KvParams c = {};
  if (int r = params("fxb_kv_commit", args, path != nullptr, &c)) return r;
  if (path && (T < 1 || T > kMaxTree || path_ss < T || !n_path))
    return fxb::set_error(FXB_EINVAL, "fxb_kv_commit: path needs n_path, 1 <= T=%d <= %d and a row stride >= T", T,
                          kMaxTree);
  for (const int32_t* x : {(const int32_t*)args->lens, (const int32_t*)args->n_pages, (const int32_t*)args->ref,
                           (const int32_t*)args->table, path, n_path, room})
    if (!lens_out || lens_out == x)  // (the token movers read these while the lengths are written)
      return fxb::set_error(FXB_EINVAL, "fxb_kv_commit: lens_out must be an array of its own");
  if (!(c.err = fxb::dev_error_ptr())) return FXB_ECUDA;
  int64_t gx = 0;
  if (path) {
    gx = ((int64_t)c.L * 2 * c.H * c.chunks + kThreads - 1) / kThreads;
    if (gx * c.S > 0x7ffffffe) return fxb::set_error(FXB_EINVAL, "fxb_kv_commit: cache too large");
  }
  fxb::pdl_launch(kv_commit_kernel, dim3((unsigned)(gx * c.S + 1)), dim3(kThreads), 0, fxb::as_stream(stream), c, path,
                  path_ss, T, n_path, room, lens_out, (int)gx);
  return fxb::check_launch("fxb_kv_commit");
}

size_t fxb_kv_fork_workspace(int32_t S, int32_t W) {
  if (S < 1 || W < 1) return 0;
  return ((size_t)S * W + 4 * (size_t)S + 1) * sizeof(int32_t);
}

int fxb_kv_fork(const fxb_kv_args* args, const int32_t* parents, void* workspace, void* stream) {
  KvParams c = {};
  if (int r = params("fxb_kv_fork", args, true, &c)) return r;
  if (!parents || !workspace || !fxb::aligned16(workspace))
    return fxb::set_error(FXB_EINVAL, "fxb_kv_fork: parents or workspace missing (16-byte aligned)");
  if (!(c.err = fxb::dev_error_ptr())) return FXB_ECUDA;
  const ForkPlan f = fork_plan(workspace, c.S, c.W);
  const int64_t entries = (int64_t)c.S * c.W;
  const int tb = (int)min((entries + kThreads - 1) / kThreads, (int64_t)fxb::num_sms());
  const int64_t units = (int64_t)c.S * c.L * 2 * c.H;
  const int cb = (int)min((units + kThreads / 32 - 1) / (kThreads / 32), (int64_t)fxb::num_sms() * 4);
  fxb::pdl_launch(kv_fork_plan_kernel, dim3(1 + tb), dim3(kThreads), 0, fxb::as_stream(stream), c, parents, f);
  if (int r = fxb::check_launch("fxb_kv_fork")) return r;
  fxb::pdl_launch(kv_fork_kernel, dim3(tb + cb), dim3(kThreads), 0, fxb::as_stream(stream), c, f, tb);
  return fxb::check_launch("fxb_kv_fork");
}

}  // extern "C"
