// What the two kernels of fxb_tree_attn share: their parameters, the division
// of the work over thread blocks and the joining of states.
//
// o = softmax(scale * q k^T) v over the context slots and the visible nodes,
// computed in one pass over the keys: a running maximum m, sum l and output O
// per row, rescaled by 2^(m_old - m_new) when the maximum rises. States of
// different parts of the keys join the same way, so a sequence can be divided
// at will.
//
// Work. An item is (batch row, key head, row tile): the R = T * G query rows
// of a key head (G query heads share it; row r is node r / G, head r % G),
// cut into tiles of rows. An item's keys are its context in blocks of
// BLOCK_KEYS slots and one block of nodes. The blocks are shared out evenly
// over the thread blocks, whatever the sequences' lengths (see Shares); an
// item that several thread blocks share is joined from their states in the
// workspace, in a fixed order: by the thread block that finishes last
// (few rows), or by a second kernel (many rows, whose states are large).
#pragma once
#include "common.cuh"
#include "internal.h"

namespace fxb_tree {

constexpr int kMaxTree = 64;
constexpr int kMaxGrid = 1024;        // arrival counters in the workspace
constexpr size_t kCounters = kMaxGrid * sizeof(unsigned);  // the same place for both kernels: it stays zero
constexpr float kRescaleLog2 = 8.f;   // how far a row's reference maximum may lag behind, in powers of two

FXB_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Params {
  int B, T, Hq, Hkv, G, R, RT, NT, page_shift, P, W;  // RT row tiles of an item's rows; NT: nodes of one (many rows)
  float scale_log2;
  const void *q, *k, *v;  // k, v: of the nodes
  void *o, *kp, *vp;
  int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh;
  int64_t k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  int64_t kp_sp, kp_sh, kp_st, vp_sp, vp_sh, vp_st;
  const int32_t* table;
  int64_t table_sb;
  const int32_t *lens, *n_nodes;
  const int64_t* mask;
  int64_t mask_sb;
  // workspace: kMaxGrid counters of arrivals (few rows; an item's is that of the block that begins it),
  unsigned* arrived;
  int2* owners;  // then the first and last thread block of each item (many rows),
  float* parts;  // then two states for every thread block
  int* err;
};

// ------------------------------------------------------------------ division of the work
struct Row {  // a batch row; one without nodes has no blocks (its zeros are written apart)
  int len, n, blocks;
};
template <int BLOCK_KEYS> FXB_DEV Row row_of(const Params& a, int b) {
  const int len_in = a.lens[b], n_in = a.n_nodes[b];
  const int64_t most = (int64_t)a.W << a.page_shift;
  Row r;
  r.len = len_in < 0 ? 0 : (len_in > most ? (int)most : len_in);
  r.n = min(max(n_in, 0), a.T);
  if (r.len != len_in || r.n != n_in) atomicOr(a.err, FXB_DERR_PAGES);
  r.blocks = r.n ? r.len / BLOCK_KEYS + (r.len % BLOCK_KEYS != 0) + 1 : 0;
  return r;
}

struct Scratch {  // of share(), in shared memory
  int64_t warp_total[12], rest;
  int b;
};
// inclusive prefix sum over the block's threads; *total for everyone
template <int THREADS> FXB_DEV int64_t block_scan(int64_t v, int64_t* total, int64_t* warp_total) {
  constexpr int kWarps = THREADS / 32;
  static_assert(kWarps <= 12, "Scratch");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) warp_total[warp] = v;
  __syncthreads();
  int64_t all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) v += warp_total[w];
    all += warp_total[w];
  }
  *total = all;
  return v;
}

// Position in the sequence of all blocks: block j of item (b, hk, rt), and how
// many of the thread block's share are left, this one among them.
struct Cursor {
  int left, b, hk, rt, j;
  Row row;
};
template <int BLOCK_KEYS> FXB_DEV void next(const Params& a, Cursor& c) {
  --c.left;
  if (++c.j < c.row.blocks) return;
  c.j = 0;
  if (++c.rt < a.RT) return;
  c.rt = 0;
  if (++c.hk < a.Hkv) return;
  c.hk = 0;
  if (c.left > 0) do
      c.row = row_of<BLOCK_KEYS>(a, ++c.b);
    while (c.row.blocks == 0);
}

// How the blocks are shared out. Even: the sequence of all blocks is cut into
// equal shares, the first `more` of them one block longer; a share may end one
// item and begin the next. Whole: every item is cut into `pieces` equal parts
// by itself, a thread block each, so that no thread block has two parts to hand
// over (about 2.5 us each); taken where items are few, shares longer than two
// blocks, and the longest part not much longer than an even share (8 rows of
// 16 nodes at 1008 slots: 18.2 -> 15.5 us). WHOLE: the kernel for few rows; the
// other joins its states in a kernel of its own and gains nothing.
struct Shares {
  int64_t total, each, more;  // even: blocks in all, of a share, shares with one more
  int first, pieces;          // whole: the item's thread blocks (pieces > 0)
  FXB_DEV void even(int64_t n) {
    total = n;
    const int64_t g = n < 1 ? 1 : (n < (int64_t)gridDim.x ? n : (int64_t)gridDim.x);
    // (a 64-bit division takes some hundred instructions)
    each = n >> 32 ? n / g : (int64_t)((uint32_t)n / (uint32_t)g);
    more = n - each * g;
    pieces = 0;
  }
  FXB_DEV int64_t begin(int cta) const {
    const int64_t u = each * cta + (cta < more ? cta : more);
    return u < total ? u : total;
  }
  FXB_DEV int owner(int64_t u) const {  // the thread block that has block u
    const int64_t big = more * (each + 1), v = u < big ? u : u - big, d = u < big ? each + 1 : each;
    const int q = v >> 32 ? (int)(v / d) : (int)((uint32_t)v / (uint32_t)d);
    return u < big ? q : (int)more + q;
  }
  // the thread blocks of the item whose first block is u and that has n blocks
  FXB_DEV int2 owners(int64_t u, int n) const {
    return pieces ? make_int2(first, first + pieces - 1) : make_int2(owner(u), owner(u + n - 1));
  }
};
// Up to 32 batch rows: every warp finds the share by itself, a lane a batch
// row, without a barrier (1.0 us of 1.9 at the start of a call).
FXB_DEV int64_t warp_scan(int64_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}
template <int BLOCK_KEYS, bool WHOLE>
FXB_DEV Cursor share_small(const Params& a, int64_t* start, Shares* shares) {
  const int per = a.Hkv * a.RT, lane = threadIdx.x & 31, G = gridDim.x;
  Row row = {0, 0, 0};
  if (lane < a.B) row = row_of<BLOCK_KEYS>(a, lane);
  int unit = row.blocks;  // of an item, in what u counts
  int64_t incl = warp_scan((int64_t)unit * per);
  shares->even(__shfl_sync(0xffffffffu, incl, 31));
  int64_t u = *start = shares->begin(blockIdx.x);
  Cursor c;
  c.left = (int)(shares->begin(blockIdx.x + 1) - u);
  int part = 0;
  const int least = (int)shares->each + (shares->more != 0);
  if (WHOLE && (int64_t)a.B * per <= G / 2 && least > 2) {
    for (int more = 0; more <= 4 && !part; more = more ? 2 * more : 1) {
      const int q = least + more, cuts = (row.blocks + q - 1) / q;
      const int64_t x = warp_scan((int64_t)cuts * per), all = __shfl_sync(0xffffffffu, x, 31);
      if (all <= G) {
        part = q;
        unit = cuts;
        incl = x;
        u = blockIdx.x;
        c.left = u < all;
      }
    }
  }
  if (c.left == 0) return c;
  const int at = __popc(__ballot_sync(0xffffffffu, incl <= u));  // rows that end at or before u
  c.b = at;
  c.row.len = __shfl_sync(0xffffffffu, row.len, at);
  c.row.n = __shfl_sync(0xffffffffu, row.n, at);
  c.row.blocks = __shfl_sync(0xffffffffu, row.blocks, at);
  unit = __shfl_sync(0xffffffffu, unit, at);
  const int64_t rest = u - (__shfl_sync(0xffffffffu, incl, at) - (int64_t)unit * per);
  const int hr = rest >> 32 ? (int)(rest / unit) : (int)((uint32_t)rest / (uint32_t)unit);
  c.j = (int)(rest - (int64_t)hr * unit);
  if (part) {
    const int k = c.j;
    shares->first = blockIdx.x - k;
    shares->pieces = unit;
    c.j = (int)((int64_t)c.row.blocks * k / unit);
    c.left = (int)((int64_t)c.row.blocks * (k + 1) / unit) - c.j;
    *start = c.j;
  }
  c.hk = hr / a.RT;
  c.rt = hr - c.hk * a.RT;
  return c;
}

// This thread block's share. Its first block has number *start: in all (even),
// or in its item (whole).
template <int BLOCK_KEYS, int THREADS, bool WHOLE> FXB_DEV Cursor share(const Params& a, int64_t* start, Shares* shares, Scratch& s) {
  if (a.B <= 32) return share_small<BLOCK_KEYS, WHOLE>(a, start, shares);
  const int per = a.Hkv * a.RT, tid = threadIdx.x, G = gridDim.x;
  int64_t n = 0, mine = 0, incl = 0;
  int blocks = 0;
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {
    const int b = b0 + tid;
    blocks = b < a.B ? row_of<BLOCK_KEYS>(a, b).blocks : 0;
    mine = (int64_t)blocks * per;
    int64_t all;
    incl = block_scan<THREADS>(mine, &all, s.warp_total) + n;
    n += all;
  }
  shares->even(n);
  int64_t u = *start = shares->begin(blockIdx.x);
  Cursor c;
  c.left = (int)(shares->begin(blockIdx.x + 1) - u);
  int part = 0;  // whole: the longest part that is allowed
  const int least = (int)shares->each + (shares->more != 0);
  if (WHOLE && a.B <= THREADS && (int64_t)a.B * per <= G / 2 && least > 2) {
    for (int more = 0; more <= 4 && !part; more = more ? 2 * more : 1) {
      const int q = least + more, cuts = (blocks + q - 1) / q;
      int64_t all;
      const int64_t x = block_scan<THREADS>((int64_t)cuts * per, &all, s.warp_total);
      if (all <= G) {
        part = q;
        mine = (int64_t)cuts * per;
        incl = x;
        u = blockIdx.x;
        c.left = u < all;
      }
    }
  }
  if (c.left == 0) return c;
  if (a.B > THREADS) n = 0;
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {
    const int b = b0 + tid;
    if (a.B > THREADS) {
      mine = b < a.B ? (int64_t)row_of<BLOCK_KEYS>(a, b).blocks * per : 0;
      int64_t all;
      incl = block_scan<THREADS>(mine, &all, s.warp_total) + n;
      n += all;
    }
    if (u < incl && u >= incl - mine) {
      s.b = b;
      s.rest = u - (incl - mine);
    }
    if (a.B > THREADS && n > u) break;
  }
  __syncthreads();
  c.b = s.b;
  c.row = row_of<BLOCK_KEYS>(a, c.b);
  const int64_t rest = s.rest;
  const int unit = part ? (c.row.blocks + part - 1) / part : c.row.blocks;  // of an item, in what u counts
  const int hr = rest >> 32 ? (int)(rest / unit) : (int)((uint32_t)rest / (uint32_t)unit);
  c.j = (int)(rest - (int64_t)hr * unit);
  if (part) {
    const int k = c.j;
    shares->first = blockIdx.x - k;
    shares->pieces = unit;
    c.j = (int)((int64_t)c.row.blocks * k / unit);
    c.left = (int)((int64_t)c.row.blocks * (k + 1) / unit) - c.j;
    *start = c.j;
  }
  c.hk = hr / a.RT;
  c.rt = hr - c.hk * a.RT;
  return c;
}

// Zeros for the batch rows without nodes, dealt out to the thread blocks.
// `nodes`: those of the first such row, read ahead.
template <typename T, int D, int THREADS> FXB_DEV void idle_rows(const Params& a, int nodes) {
  constexpr int kPer = 16 / sizeof(T);
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    if ((b == (int)blockIdx.x ? nodes : a.n_nodes[b]) > 0) continue;
    const int n = a.T * a.Hq * (D / kPer);
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const int d = i % (D / kPer), x = i / (D / kPer), t = x / a.Hq, h = x - t * a.Hq;
      *reinterpret_cast<uint4*>(static_cast<T*>(a.o) + b * a.o_sb + t * a.o_st + h * a.o_sh + d * kPer) =
          make_uint4(0, 0, 0, 0);
    }
  }
}

// ------------------------------------------------------------------ joining states
template <typename T, int D>
FXB_DEV void write_out(const Params& a, int b, int hk, int r, int d, float4 o, float l) {
  if (r >= a.R) return;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no visible key: zeros; NaN stays
  const int t = r / a.G, h = hk * a.G + (r - t * a.G);
  T* p = static_cast<T*>(a.o) + b * a.o_sb + t * a.o_st + h * a.o_sh + d;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
  }
}
FXB_DEV void axpy4(float4& o, float w, const float4& x) {
  o.x = fmaf(w, x.x, o.x);
  o.y = fmaf(w, x.y, o.y);
  o.z = fmaf(w, x.z, o.z);
  o.w = fmaf(w, x.w, o.w);
}
// weight of a state with maximum m in a join with maximum mx
FXB_DEV float weight(float m, float mx) { return m == -INFINITY ? 0.f : ex2(m - mx); }

// State of an item's part in the workspace: m and l of each row, then O as
// [D / 4][ROWS] float4. A thread block has two places: 1 for an item that it
// begins, 0 for one that it continues.
template <int ROWS, int D> FXB_DEV float* part_of(const Params& a, int cta, int place) {
  return a.parts + ((int64_t)cta * 2 + place) * ROWS * (D + 2);
}

// Joins the parts [lo, hi] of an item (those of thread blocks lo to hi), in a
// fixed order: row r of the tile at row0, its quads d4, d4 + step,
// ... `slices` lanes, LANES apart, take every slices-th part each and exchange
// their states (slices a power of two, all lanes of the warp call). A part
// costs a trip to L2 whatever is read of it, so U are under way at once.
template <typename T, int ROWS, int D, int NQ, int U>
FXB_DEV void join_row(const Params& a, int b, int hk, int row0, int r, int d4, int step, int lo, int hi, int slice = 0,
                      int slices = 1, int lanes = 32) {
  float m = -INFINITY, l = 0.f;
  float4 o[NQ];
#pragma unroll
  for (int x = 0; x < NQ; ++x) o[x] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int k0 = lo + slice; k0 <= hi; k0 += U * slices) {
    float mk[U], lk[U];
    float4 ok[U][NQ];
#pragma unroll
    for (int y = 0; y < U; ++y) {
      const int k = k0 + y * slices;
      mk[y] = -INFINITY;
      if (k <= hi) {
        const float* p = part_of<ROWS, D>(a, k, k == lo);
        mk[y] = __ldcg(p + r);
        lk[y] = __ldcg(p + ROWS + r);
#pragma unroll
        for (int x = 0; x < NQ; ++x)
          ok[y][x] = __ldcg(reinterpret_cast<const float4*>(p + 2 * ROWS) + (d4 + x * step) * ROWS + r);
      }
    }
    float mn = m;
#pragma unroll
    for (int y = 0; y < U; ++y) mn = fmaxf(mn, mk[y]);
    const float f = weight(m, mn);
    l *= f;
#pragma unroll
    for (int x = 0; x < NQ; ++x) o[x] = make_float4(o[x].x * f, o[x].y * f, o[x].z * f, o[x].w * f);
#pragma unroll
    for (int y = 0; y < U; ++y) {
      if (k0 + y * slices > hi) break;
      const float w = weight(mk[y], mn);
      l = fmaf(w, lk[y], l);
#pragma unroll
      for (int x = 0; x < NQ; ++x) axpy4(o[x], w, ok[y][x]);
    }
    m = mn;
  }
  for (int s = 1; s < slices; s <<= 1) {
    const float m1 = __shfl_xor_sync(0xffffffffu, m, s * lanes), mn = fmaxf(m, m1);
    const float f = weight(m, mn), f1 = weight(m1, mn);
    l = l * f + __shfl_xor_sync(0xffffffffu, l, s * lanes) * f1;
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      float4& y = o[x];
      y.x = y.x * f + __shfl_xor_sync(0xffffffffu, y.x, s * lanes) * f1;
      y.y = y.y * f + __shfl_xor_sync(0xffffffffu, y.y, s * lanes) * f1;
      y.z = y.z * f + __shfl_xor_sync(0xffffffffu, y.z, s * lanes) * f1;
      y.w = y.w * f + __shfl_xor_sync(0xffffffffu, y.w, s * lanes) * f1;
    }
    m = mn;
  }
  if (slice == 0) {
#pragma unroll
    for (int x = 0; x < NQ; ++x) write_out<T, D>(a, b, hk, row0 + r, (d4 + x * step) * 4, o[x], l);
  }
}

// ------------------------------------------------------------------ host
// (outer, mid, rows, D) view with element strides, 128-byte swizzle; boxes of
// box_rows x box_mid rows of 128 bytes. The stride of an axis of one entry is
// not used and may be anything.
inline int encode_rows(CUtensorMap* m, CUtensorMapDataType type, int size, const void* base, int D, int rows,
                       int64_t s_rows, int mid, int64_t s_mid, int outer, int64_t s_outer, int box_rows, int box_mid) {
  const uint64_t e = size, one = D * e;
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)rows, (uint64_t)mid, (uint64_t)outer};
  const uint64_t strides[3] = {rows > 1 ? s_rows * e : one, mid > 1 ? s_mid * e : one, outer > 1 ? s_outer * e : one};
  const uint32_t box[4] = {(uint32_t)(128 / e), (uint32_t)box_rows, (uint32_t)box_mid, 1};
  return fxb::encode_tiled(m, type, 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
// thread blocks: `most`, but no more than there can be blocks of keys
inline int grid_of(const fxb_tree_attn_args* x, const Params& a, int block_keys, int most) {
  const int64_t keys = (int64_t)a.W << a.page_shift;
  const int64_t n = (int64_t)a.B * a.Hkv * a.RT * ((keys + block_keys - 1) / block_keys + 1);
  return (int)(n < most ? n : most);
}
// the kernel for many rows (tree_attn_wide.cu): 16-bit types, G <= 128
size_t wide_workspace(const fxb_tree_attn_args* x);
int launch_wide(const fxb_tree_attn_args* x, Params& a, void* stream);

}  // namespace fxb_tree
