// Attention of a tree of drafted tokens over a paged KV cache: the kernel for
// many rows (16-bit types), on tcgen05 tensor cores.
//
// A row tile is up to 128 rows (whole nodes: 128 / G of them) against tiles of
// 128 keys; the block of nodes is one tile of 64. Persistent thread blocks, one
// an SM, walk their share of all tiles. Roles (384 threads):
//   warps 0-3, 4-7  softmax: a thread owns a row and one half of a tile's keys;
//                   the two threads of a row exchange its maximum;
//   warp 8          issues S = Q K^T, up to two tiles ahead of the softmax;
//   warp 11         issues O += P V (a warp of its own: when keys are late it
//                   still takes what the softmax has finished);
//   warp 9          copies Q, keys and values by TMA, a lane a page;
//   warp 10         writes the nodes' keys and values into the cache.
// Tensor memory (512 columns): scores of two tiles at 0 and 128 (fp32),
// probabilities of two tiles at 256 and 320 (16 bits, the A operand of P V), O
// at 384. Scores are free as soon as they are in registers, so that the tensor
// cores and the softmax run side by side.
// Keys and values go through one ring of operands in the order of their use
// (K0 K1 V0 K2 V1 ...). A wait tells a phase from the one before it by parity
// alone, so whoever waits for a slot has to know that its previous use is over.
// The ring's length is even: a slot is used by keys only or by values only (but
// for the first keys and the last values), so each of the two issuing warps
// waits for every use of its slots. With an odd length the warp that issues S
// took a slot for filled whose older values were still under way.
//
// What bounds it: HBM with one row tile (one row of 8 nodes x 4 heads at 100003
// slots, D = 128: 82 us, 5.0 TB/s at 1965 MHz; 96 us, 4.3 TB/s in calls without
// a pause, for which the power limit leaves 1720 MHz); with several, which read the cache from L2,
// the softmax's chain of short waits (4 rows of 63 nodes x 8 heads at up to
// 12001 slots: 60 us, 595 TFLOP/s; about 2600 cycles a tile, of which the
// exponentials take 1024 of their unit and the products 1024 of theirs). Without
// the copies that case takes 57.9 us, without the exponentials 55.8, without
// seven of eight products 57.9, without all three 46.8: no unit is the limit.
// The copying warp (1300 cycles an operand) and the softmax warps (2500 a tile)
// keep the same pace. Not faster: a group of warps for each of two tiles in
// flight (63.7 us), 16 softmax warps with 32 keys a thread (62.1), packed fp32
// pairs and three-way maxima (59.8), one arrival a warp (61.2), a ring and a
// copying warp each for keys and values (59.7 to 63.1: the softmax's pace).
#include "tree_attn.cuh"

namespace {

using namespace fxb_tree;

constexpr int kTileRows = 128;
constexpr int kBlockKeys = 128;
constexpr int kThreads = 384;
constexpr int kWarpS = 8, kWarpTma = 9, kWarpStore = 10, kWarpPV = 11;
constexpr int kSoftmax = 256;  // threads of both groups

constexpr int kSmall = 3 * 1024; // shared memory behind the operands
template <int D> struct Wide {
  static constexpr int kBoxes = D / 64;
  static constexpr int kOperand = kTileRows * D * 2;  // Q, K or V of a tile: D / 64 blocks of [128 rows][128 bytes]
  static constexpr int kSlots = D == 128 ? 6 : 12;    // ring of keys and values: an even number, see the top
  static constexpr int kSmem = (1 + kSlots) * kOperand + kSmall;
  static constexpr int kPart = kTileRows * (D + 2);   // floats of a state in the workspace
};
static_assert(Wide<128>::kSmem <= 232448 && Wide<64>::kSmem <= 232448, "shared memory of a block");

// byte offset of 16-byte piece c of row r of an operand (128-byte swizzle)
FXB_DEV uint32_t sw(int r, int c) { return (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4); }
// steps of 16 along K of an operand whose rows are M or N (K-major) or K (MN-major)
constexpr uint32_t kmajor_off(int kk) { return (kk >> 2) * 16384 + (kk & 3) * 32; }
constexpr uint32_t mnmajor_off(int kk) { return kk * 2048; }

// completes loads from tensor memory; the registers pass through it, so that nothing that uses them moves before it
FXB_DEV void tmem_wait_ld32(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

struct Small {
  float x[2][2][kTileRows];  // [tile parity][half]: a row's maximum over half a tile; its sum at an item's end
  uint64_t bars[36];
  Scratch scratch;
  int odd_value[3];          // an item's node has a value that is not finite (items in turn)
  uint32_t tmem_slot;
};
static_assert(sizeof(Small) <= kSmall, "shared memory behind the operands");

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
tree_attn_wide(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
               const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmNK,
               const __grid_constant__ CUtensorMap tmNV, const Params a) {
  using W = Wide<D>;
  constexpr int NS = W::kSlots, NBOX = W::kBoxes;
  constexpr int FMT = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  // All of it dynamic, so that six operands fit beside Q: it begins on a 1024-byte boundary, as the swizzle needs
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = smem_u32(smem_raw);
  uint8_t* gbase = smem_raw;
  Small& sm = *reinterpret_cast<Small*>(smem_raw + (1 + NS) * W::kOperand);
  if (base & 1023) {  // (not met: there is no static shared memory)
    if (threadIdx.x == 0) atomicOr(a.err, FXB_DERR_ATTN_WAIT);
    return;
  }
  const uint32_t sQ = base, sKV = base + W::kOperand;
  const uint32_t bar0 = smem_u32(sm.bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (NS + s); };
  const uint32_t q_full = bar0 + 8u * (2 * NS), q_empty = bar0 + 8u * (2 * NS + 1);
  auto s_full = [&](int i) { return bar0 + 8u * (2 * NS + 2 + i); };   // of tile parity i
  auto s_empty = [&](int i) { return bar0 + 8u * (2 * NS + 4 + i); };
  auto p_full = [&](int i) { return bar0 + 8u * (2 * NS + 6 + i); };
  auto pv_done = [&](int i) { return bar0 + 8u * (2 * NS + 8 + i); };
  const uint32_t o_free = bar0 + 8u * (2 * NS + 10), final_bar = bar0 + 8u * (2 * NS + 11);  // all products are complete
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full(i), 1);
      mbar_init(s_empty(i), kSoftmax);
      mbar_init(p_full(i), kSoftmax);
      mbar_init(pv_done(i), 1);
    }
    sm.odd_value[0] = sm.odd_value[1] = sm.odd_value[2] = 0;
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(o_free, kSoftmax);
    mbar_init(final_bar, 2);
    fence_mbar_init();
  }
  if (warp == kWarpS) {
    tmem_alloc(smem_u32(&sm.tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_slot;
  pdl_wait();
  pdl_trigger();  // (the joining kernel waits before its first read)

  int64_t start;
  Shares shares;
  const int nodes = (int)blockIdx.x < a.B ? a.n_nodes[blockIdx.x] : 1;
  Cursor c = share<kBlockKeys, kThreads, false>(a, &start, &shares, sm.scratch);
  idle_rows<T, D, kThreads>(a, nodes);
  const int n_tiles = c.left;
  // places in the ring's order of use
  auto k_index = [&](int q) { return q == 0 ? 0 : 2 * q - 1; };
  auto v_index = [&](int q) { return q + 1 < n_tiles ? 2 * q + 2 : 2 * q + 1; };
  bool ok = true;

  if (warp == kWarpTma) {
    // ------------------------------------------------ copies; lane i takes page i of a tile
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      tma_prefetch_desc(&tmNK);
      tma_prefetch_desc(&tmNV);
    }
    const int page = 1 << a.page_shift, box_rows = min(page, kBlockKeys), per_tile = kBlockKeys / box_rows;
    int items = -1, issued = 0;
    // this lane's page of the tile at f, as the table has it. Nothing may depend on it here: it is read a step
    // ahead of its use, and the warp waits at the first instruction that needs it
    auto page_of = [&](const Cursor& f) {
      const int slot0 = f.j * kBlockKeys + lane * box_rows;
      const bool has = f.left > 0 && f.j < f.row.blocks - 1 && lane < per_tile && slot0 < f.row.len;
      return has ? a.table[f.b * a.table_sb + (slot0 >> a.page_shift)] : 0;
    };
    auto load = [&](bool values, const Cursor& f, int pg) -> bool {
      const int s = issued % NS;
      if (!mbar_wait_warp(empty(s), ((issued / NS) & 1) ^ 1, a.err, FXB_DERR_ATTN_WAIT)) return false;
      const bool tree = f.j == f.row.blocks - 1;
      const int pages = tree ? 1 : (min(f.row.len - f.j * kBlockKeys, kBlockKeys) + box_rows - 1) / box_rows;
      if (lane == 0) mbar_expect_tx(full(s), pages * (tree ? kMaxTree : box_rows) * 128 * NBOX);
      __syncwarp();
      if (lane < pages) {
        if (!tree && (pg < 0 || pg >= a.P)) {  // outside the pool: reported, page 0 is read instead
          atomicOr(a.err, FXB_DERR_PAGES);
          pg = 0;
        }
        const CUtensorMap* map = values ? (tree ? &tmNV : &tmV) : (tree ? &tmNK : &tmK);
        const uint32_t dst = sKV + s * W::kOperand + (tree ? 0 : lane * box_rows * 128);
        const int row = tree ? 0 : (f.j * kBlockKeys) & (page - 1);  // 0 unless a page holds several tiles
#pragma unroll
        for (int x = 0; x < NBOX; ++x) tma_load_4d(dst + x * 16384, map, full(s), x * 64, row, f.hk, tree ? f.b : pg);
      }
      ++issued;
      return true;
    };
    // step q: keys of tile q, then values of tile q - 1
    if (n_tiles) {
      Cursor f = c, fv = c;
      int pg = page_of(f), pv = -1;
#pragma unroll 1
      for (int q = 0; q <= n_tiles && ok; ++q) {
        if (q < n_tiles && (q == 0 || f.j == 0)) {  // the item's rows of Q
          ++items;
          ok = mbar_wait_warp(q_empty, (items & 1) ^ 1, a.err, FXB_DERR_ATTN_WAIT);
          if (!ok) break;
          if (lane == 0) {
            mbar_expect_tx(q_full, a.NT * a.G * 128 * NBOX);
#pragma unroll
            for (int x = 0; x < NBOX; ++x)
              tma_load_4d(sQ + x * 16384, &tmQ, q_full, x * 64, f.hk * a.G,
                          f.rt * a.NT, f.b);
          }
        }
        const Cursor fk = f;
        const int pk = pg;
        if (q < n_tiles) {
          next<kBlockKeys>(a, f);
          pg = page_of(f);  // used in the next step
        }
#pragma unroll 1
        for (int kv = q < n_tiles ? 0 : 1; kv < (q ? 2 : 1) && ok; ++kv)
          ok = load(kv != 0, kv ? fv : fk, kv ? pv : pk);
        fv = fk;
        pv = pk;
      }
      // what is under way lands before shared memory goes
      for (int i = max(0, issued - NS); i < issued; ++i)
        mbar_wait_warp(full(i % NS), (i / NS) & 1, a.err, FXB_DERR_ATTN_WAIT);
      if (items >= 0) mbar_wait_warp(q_full, items & 1, a.err, FXB_DERR_ATTN_WAIT);
    }
  } else if (warp == kWarpS || warp == kWarpPV) {
    // ------------------------------------------------ products. The whole warp keeps together and polls (a
    // completed wait costs an instruction, not an exchange between lanes); an elected lane issues, and the
    // operands of a product are known to be uniform
    auto uwait = [&](uint32_t bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, a.err, FXB_DERR_ATTN_WAIT));
    };
    int items = -1;  // items begun
    if (warp == kWarpS) {
      constexpr uint32_t IS = umma_idesc_f16(FMT, 0, 0, kTileRows, kBlockKeys);
      constexpr uint32_t IST = umma_idesc_f16(FMT, 0, 0, kTileRows, kMaxTree);
      const uint64_t qd = umma_desc_sw128(sQ, 16, 1024);
#pragma unroll 1
      for (int q = 0; q < n_tiles; ++q) {
        const int i = k_index(q), st = i % NS, par = q & 1;
        const bool tree = c.j == c.row.blocks - 1;
        if (q == 0 || c.j == 0) {
          ++items;
          if (!uwait(q_full, items & 1)) break;
        }
        if (!uwait(s_empty(par), ((q >> 1) & 1) ^ 1)) break;
        if (!uwait(full(st), (i / NS) & 1)) break;
        tc_fence_after();
        const uint64_t kd = umma_desc_sw128(sKV + st * W::kOperand, 16, 1024);
        const uint32_t is = tree ? IST : IS, d = tmem + par * 128;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_f16(d, desc_add(qd, kmajor_off(kk)), desc_add(kd, kmajor_off(kk)), is, kk > 0);
          umma_commit(s_full(par));
          umma_commit(empty(st));
          if (tree || q + 1 == n_tiles) umma_commit(q_empty);  // the item's last S has read Q
        }
        __syncwarp();
        next<kBlockKeys>(a, c);
      }
    } else {
      constexpr uint32_t IPV = umma_idesc_f16(FMT, 0, 1, kTileRows, D);
      const uint32_t o = tmem + 384;
#pragma unroll 1
      for (int q = 0; q < n_tiles; ++q) {
        const int i = v_index(q), st = i % NS, par = q & 1;
        const bool tree = c.j == c.row.blocks - 1, first = q == 0 || c.j == 0;
        if (first) ++items;
        if (!uwait(full(st), (i / NS) & 1)) break;
        // the item's first product overwrites O: that of the previous item has been read
        if (first && items > 0 && !uwait(o_free, (items - 1) & 1)) break;
        if (!uwait(p_full(par), (q >> 1) & 1)) break;
        tc_fence_after();
        const uint64_t vd = umma_desc_sw128(sKV + st * W::kOperand, 16384, 1024);
        const uint32_t pr = tmem + 256 + par * 64;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kMaxTree / 16; ++kk)
            umma_f16_ta(o, pr + kk * 8, desc_add(vd, mnmajor_off(kk)), IPV, kk > 0 || !first ? 1u : 0u);
          if (!tree) {
#pragma unroll
            for (int kk = kMaxTree / 16; kk < kBlockKeys / 16; ++kk)
              umma_f16_ta(o, pr + kk * 8, desc_add(vd, mnmajor_off(kk)), IPV, 1u);
          }
          umma_commit(pv_done(par));
          umma_commit(empty(st));
        }
        __syncwarp();
        next<kBlockKeys>(a, c);
      }
    }
    if (elect_one()) umma_commit(final_bar);
    uwait(final_bar, 0);
  } else if (warp == kWarpStore) {
    // ------------------------------------------------ the nodes' keys and values into the cache
    constexpr int CH = D / 8;
    for (Cursor f = c; f.left > 0; next<kBlockKeys>(a, f)) {
      if (f.j != f.row.blocks - 1 || f.rt) continue;
      const int hk = f.hk, n = f.row.n * CH;
#pragma unroll 1
      for (int i0 = lane; i0 < n; i0 += 32 * 4) {
        uint4 xk[4], xv[4];
        int64_t to[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = i0 + 32 * u, t = i / CH, ch = i % CH;
          to[u] = -1;
          if (i < n) {
            const int64_t pos = (int64_t)f.row.len + t, pi = pos >> a.page_shift;
            const int pg = pi < a.W ? a.table[f.b * a.table_sb + pi] : -1;
            if (pg < 0 || pg >= a.P) atomicOr(a.err, FXB_DERR_PAGES);
            else to[u] = ((int64_t)pg << a.page_shift) | (pos & ((1 << a.page_shift) - 1));
            xk[u] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.k) + f.b * a.k_sb + t * a.k_st + hk * a.k_sh +
                                                    ch * 8);
            xv[u] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.v) + f.b * a.v_sb + t * a.v_st + hk * a.v_sh +
                                                    ch * 8);
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (to[u] < 0) continue;
          const int ch = (i0 + 32 * u) % CH;
          const int64_t pg = to[u] >> a.page_shift, off = to[u] & ((1 << a.page_shift) - 1);
          *reinterpret_cast<uint4*>(static_cast<T*>(a.kp) + pg * a.kp_sp + hk * a.kp_sh + off * a.kp_st + ch * 8) = xk[u];
          *reinterpret_cast<uint4*>(static_cast<T*>(a.vp) + pg * a.vp_sp + hk * a.vp_sh + off * a.vp_st + ch * 8) = xv[u];
        }
      }
    }
  } else {
    // ------------------------------------------------ softmax
    const int g = warp >> 2, r = (warp & 3) * 32 + lane;  // half of the keys, row of the tile
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_off, tP = tmem + lane_off + 256, tO = tmem + lane_off + 384 + g * (D / 2);
    int item = 0;
    auto uwait = [&](uint32_t bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, a.err, FXB_DERR_ATTN_WAIT));
    };
    float m = -INFINITY, l = 0.f;
    bool live = false, dead = true;  // this row is a node's; no row of this warp is
    uint64_t see = 0;
    int64_t u_first = 0;
#pragma unroll 1
    for (int q = 0; q < n_tiles; ++q) {
      const int hk = c.hk, t0 = c.rt * a.NT, par = q & 1;
      const bool tree = c.j == c.row.blocks - 1, begins = q == 0 || c.j == 0;
      if (begins) {
        u_first = start + q - c.j;
        m = -INFINITY;
        l = 0.f;
        const int t = t0 + r / a.G;
        live = r < a.NT * a.G && t < c.row.n;
        see = live ? (uint64_t)a.mask[c.b * a.mask_sb + t] : 0;
        dead = !__any_sync(0xffffffffu, live);
      }
      if (ok && !uwait(s_full(par), (q >> 1) & 1)) ok = false;
      const int cols = tree ? kMaxTree : kBlockKeys;
      const int c0 = g * (cols / 2);  // this thread's columns: 64, or 32 of the nodes
      uint32_t v[64];
      float mx = -INFINITY;
      // After an expired wait a warp goes on through the tiles without work, so that every barrier is met.
      if (ok) {
        tc_fence_after();
        const int valid = tree ? c.row.n : min(c.row.len - c.j * kBlockKeys, kBlockKeys);
        const bool some = valid < cols || tree;
        tmem_ld32(tS + par * 128 + c0, v);
        tmem_ld32(tS + par * 128 + min(c0 + 32, 96), v + 32);
        tmem_wait_ld32(v);
        tmem_wait_ld32(v + 32);
        tc_fence_before();
        mbar_arrive(s_empty(par));
        if (some) {  // tail of the context, or nodes
          const int in = min(max(valid - c0, 0), 64);
          uint64_t w = in == 64 ? ~0ull : (1ull << in) - 1;
          if (tree) w &= (see >> c0) & 0xffffffffull;
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (!((w >> i) & 1)) v[i] = __float_as_uint(-INFINITY);
          // values that no row may count are zeroed (0 * NaN is NaN): behind the sequence, or nodes that
          // do not exist; infinities and NaN of nodes too: who sees them adds them at the item's end
          const int vi = v_index(q), vslot = vi % NS;
          if (!uwait(full(vslot), (vi / NS) & 1)) ok = false;
          uint8_t* vs = gbase + (sKV - base) + vslot * W::kOperand;
          bool odd = false;
#pragma unroll 1
          for (int i = threadIdx.x; i < cols * (D / 8); i += kSoftmax) {
            const int row = i / (D / 8);
            uint4* p = reinterpret_cast<uint4*>(vs + sw(row, i % (D / 8)));
            if (row >= valid) {
              *p = make_uint4(0, 0, 0, 0);
            } else if (tree) {
              float f[8];
              unpack8<T>(*p, f);
              bool any = false;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const bool fin = fabsf(f[e]) < INFINITY;
                any |= !fin;
                f[e] = fin ? f[e] : 0.f;
              }
              if (any) *p = pack8<T>(f);
              odd |= any;
            }
          }
          if (odd) atomicExch(&sm.odd_value[item % 3], 1);
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (!dead) {
          float mv[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 32; ++i)
            mv[i & 3] = fmaxf(fmaxf(mv[i & 3], __uint_as_float(v[i])), __uint_as_float(v[32 + i]));
          mx = fmaxf(fmaxf(mv[0], mv[1]), fmaxf(mv[2], mv[3]));
          sm.x[par][g][r] = mx;
        }
      }
      if (!dead) {
        __syncwarp();
        named_bar_sync(2 + (warp & 3), 64);  // the row's two threads
      }
      if (ok) {
        if (!dead) {
          // (a row that is no node's holds whatever was in shared memory: it must not ask for a rescaling)
          mx = live ? fmaxf(mx, sm.x[par][g ^ 1][r]) * a.scale_log2 : -INFINITY;
          // the reference maximum m moves only when a tile exceeds it by more than 2^8: probabilities stay
          // below 2^8, which 16 bits hold as well as [0, 1], and O is rarely rescaled
          if (begins) {
            m = mx;  // the item's first P V overwrites O
          } else if (__any_sync(0xffffffffu, mx > m + kRescaleLog2)) {
            if (!uwait(pv_done(par ^ 1), ((q - 1) >> 1) & 1)) ok = false;
            tc_fence_after();
            const bool up = mx > m + kRescaleLog2;
            const float f = up ? ex2(m - mx) : 1.f;
#pragma unroll 1
            for (int i = 0; i < D / 2 / 16; ++i) {
              uint32_t o[16];
              tmem_ld16(tO + i * 16, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st16(tO + i * 16, o);
            }
            tmem_wait_st();
            l *= f;
            if (up) m = mx;
          }
        }
        // the place of the probabilities is free once P V of tile q - 2 is complete
        if (q >= 2 && !uwait(pv_done(par), ((q - 2) >> 1) & 1)) ok = false;
        __syncwarp();
        if (!dead) {
          const float z = m == -INFINITY ? 0.f : m;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          // Probabilities enter the second product in the inputs' type, as both of its operands have one type: the
          // error against 64 bits is 1.35 times that of fp32 probabilities (bf16 2.3e-3 for 1.7e-3). A second
          // product with what the rounding leaves brings it to 1.0 times for 71.2 us instead of 59.7 (4 rows of 63
          // nodes x 8 heads) and 94 instead of 82 (one row at 100003 slots), and makes NaN of an infinite value
          // where nothing, or less than 0, is left.
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h == 1 && tree) break;
            uint32_t p[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float p0 = ex2(fmaf(__uint_as_float(v[32 * h + 2 * i]), a.scale_log2, -z));
              const float p1 = ex2(fmaf(__uint_as_float(v[32 * h + 2 * i + 1]), a.scale_log2, -z));
              sum[(2 * i) & 3] += p0;
              sum[(2 * i + 1) & 3] += p1;
              p[i] = pack2<T>(p0, p1);
            }
            tmem_st16(tP + par * 64 + c0 / 2 + 16 * h, p);
          }
          tmem_wait_st();
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
        tc_fence_before();
        mbar_arrive(p_full(par));
      }
      const Cursor cur = c;
      next<kBlockKeys>(a, c);
      if (!tree && q + 1 < n_tiles) continue;
      // ---- the item ends here
      if (ok && !uwait(pv_done(par), (q >> 1) & 1)) ok = false;
      if (!dead) sm.x[par ^ 1][g][r] = live ? l : 0.f;  // (the maxima of tile q - 1 have been read)
      // the next item's flag, last read two items ago (every thread has passed the barrier since)
      if (threadIdx.x == 0) sm.odd_value[(item + 1) % 3] = 0;
      __syncwarp();
      named_bar_sync(1, kSoftmax);
      const bool begun = u_first >= start, whole = begun && tree;
      const float mj = live ? m : -INFINITY, lj = live ? sm.x[par ^ 1][0][r] + sm.x[par ^ 1][1][r] : 0.f;
      if (!dead) named_bar_sync(2 + (warp & 3), 64);  // both have read: tile q + 1 writes there
      const int rows = min(a.NT, a.T - t0) * a.G;
      float* part = part_of<kTileRows, D>(a, blockIdx.x, begun);
      // 16 columns at a time, rolled (this code runs once an item, out of a cold instruction cache). Accesses to
      // tensor memory are collective: the warp is brought together before each, and the lanes' own condition is
      // kept opaque, so that the loop cannot be split by lanes.
      const int t = (t0 * a.G + r) / a.G, h = hk * a.G + (t0 * a.G + r - t * a.G);
      T* out = static_cast<T*>(a.o) + cur.b * a.o_sb + t * a.o_st + h * a.o_sh + g * (D / 2);
      float4* to = reinterpret_cast<float4*>(part + 2 * kTileRows) + g * (D / 8) * kTileRows + r;
      const float inv = lj > 0.f ? 1.f / lj : (lj == 0.f ? 0.f : lj);  // no visible key: zeros; NaN stays
      const bool odd = tree && sm.odd_value[item % 3];
      int mine = r < rows && ok;
      tc_fence_after();
#pragma unroll 1
      for (int i = 0; i < D / 2; i += 16) {
        asm volatile("" : "+r"(mine));
        __syncwarp();
        uint32_t ov[16];
        tmem_ld16(tO + i, ov);
        tmem_wait_ld();
        float o[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = live ? __uint_as_float(ov[e]) : 0.f;
        if (odd && live)
#pragma unroll 1
          for (int j = 0; j < cur.row.n; ++j)
            if ((see >> j) & 1)
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float y = to_f<T>(
                    static_cast<const T*>(a.v)[cur.b * a.v_sb + j * a.v_st + hk * a.v_sh + g * (D / 2) + i + e]);
                if (!(fabsf(y) < INFINITY)) o[e] += y;
              }
        if (mine) {
          if (whole) {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] *= inv;
            store8<T>(out + i, o);
            store8<T>(out + i + 8, o + 8);
          } else {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              to[(i + e) / 4 * kTileRows] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      mbar_arrive(o_free);
      if (!whole && g == 0 && r < rows) {
        part[r] = mj;
        part[kTileRows + r] = lj;
      }
      if (begun && threadIdx.x == 0)
        a.owners[((int64_t)cur.b * a.Hkv + cur.hk) * a.RT + cur.rt] =
            shares.owners(u_first, cur.row.blocks);
      ++item;
      __syncwarp();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kWarpS) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the items that several thread blocks share: a block takes 32 rows of
// an item, a lane a row, a warp a sixteenth of its columns.
constexpr int kJoinThreads = 512;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) tree_attn_join(const Params a) {
  pdl_trigger();
  pdl_wait();
  const int hr = blockIdx.x % (a.Hkv * a.RT), b = blockIdx.x / (a.Hkv * a.RT);
  const int2 own = a.owners[blockIdx.x];
  if (a.n_nodes[b] <= 0 || own.x == own.y) return;  // (no nodes: no owners either)
  const int hk = hr / a.RT, t0 = (hr % a.RT) * a.NT;
  const int r = blockIdx.y * 32 + (threadIdx.x & 31), warp = threadIdx.x >> 5;
  if (r >= min(a.NT, a.T - t0) * a.G) return;
  constexpr int kStep = kJoinThreads / 32;
  join_row<T, kTileRows, D, D / 4 / kStep, 4>(a, b, hk, t0 * a.G, r, warp, kStep, own.x, own.y);
}

template <typename T> constexpr CUtensorMapDataType map_type() {
  return std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

template <typename T, int D>
int launch(const fxb_tree_attn_args* x, Params& a, int grid, void* stream) {
  CUtensorMap q, k, v, nk, nv;
  const auto t = map_type<T>();
  if (int r = encode_rows(&q, t, 2, x->q, D, x->Hq, x->q_sh, x->T, x->q_st, x->B, x->q_sb, a.G, a.NT)) return r;
  const int box = x->page < kBlockKeys ? x->page : kBlockKeys;
  if (int r = encode_rows(&k, t, 2, x->k_pages, D, x->page, x->kp_st, x->Hkv, x->kp_sh, x->P, x->kp_sp, box, 1)) return r;
  if (int r = encode_rows(&v, t, 2, x->v_pages, D, x->page, x->vp_st, x->Hkv, x->vp_sh, x->P, x->vp_sp, box, 1)) return r;
  if (int r = encode_rows(&nk, t, 2, x->k, D, x->T, x->k_st, x->Hkv, x->k_sh, x->B, x->k_sb, kMaxTree, 1)) return r;
  if (int r = encode_rows(&nv, t, 2, x->v, D, x->T, x->v_st, x->Hkv, x->v_sh, x->B, x->v_sb, kMaxTree, 1)) return r;
  if (int r = fxb::check_cuda(
          cudaFuncSetAttribute(tree_attn_wide<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Wide<D>::kSmem),
          "fxb_tree_attn"))
    return r;
  fxb::pdl_launch(tree_attn_wide<T, D>, dim3(grid), dim3(kThreads), Wide<D>::kSmem, fxb::as_stream(stream), q, k, v,
                  nk, nv, a);
  if (int r = fxb::check_launch("fxb_tree_attn")) return r;
  const int chunks = (a.NT * a.G + 31) / 32;
  fxb::pdl_launch(tree_attn_join<T, D>, dim3((unsigned)(a.B * a.Hkv * a.RT), chunks), dim3(kJoinThreads), 0,
                  fxb::as_stream(stream), a);
  return fxb::check_launch("fxb_tree_attn");
}

}  // namespace

namespace fxb_tree {

// nodes of a row tile, row tiles
static int nodes_of(int T, int G) { return T < kTileRows / G ? T : kTileRows / G; }
static size_t owners_bytes(int B, int Hkv, int RT) { return ((size_t)B * Hkv * RT * sizeof(int2) + 255) / 256 * 256; }

size_t wide_workspace(const fxb_tree_attn_args* x) {
  const int NT = nodes_of(x->T, x->Hq / x->Hkv), RT = (x->T + NT - 1) / NT;
  return kCounters + owners_bytes(x->B, x->Hkv, RT) +
         (size_t)fxb::num_sms() * 2 * (x->D == 64 ? Wide<64>::kPart : Wide<128>::kPart) * sizeof(float);
}

int launch_wide(const fxb_tree_attn_args* x, Params& a, void* stream) {
  a.NT = nodes_of(a.T, a.G);
  a.RT = (a.T + a.NT - 1) / a.NT;
  char* ws = static_cast<char*>(x->workspace) + kCounters;
  a.owners = reinterpret_cast<int2*>(ws);
  a.parts = reinterpret_cast<float*>(ws + owners_bytes(a.B, a.Hkv, a.RT));
  const int grid = grid_of(x, a, kBlockKeys, fxb::num_sms());
  if (x->dtype == FXB_DTYPE_F16)
    return x->D == 64 ? launch<__half, 64>(x, a, grid, stream) : launch<__half, 128>(x, a, grid, stream);
  return x->D == 64 ? launch<__nv_bfloat16, 64>(x, a, grid, stream) : launch<__nv_bfloat16, 128>(x, a, grid, stream);
}

}  // namespace fxb_tree
