// Attention of a tree of drafted tokens over a paged KV cache (fxb_tree_attn):
// the kernel for few rows and the entry point. No reference counterpart: its
// sampler keeps no cache (ml/fxlm/sample.py:63-73).
//
// Every warp works by itself on its own keys of each block (16 of 64; 8 in
// fp32 with D = 128), from copies that it starts by itself, so that nothing but
// an item's end makes one warp wait for another. What bounds it: HBM while the
// cache is long (48 rows of 4 nodes x 32 heads over 8 key heads, up to 8192
// slots, D = 128: 191 us, 6.1 TB/s, 0.94 of the rate of a copy); a chain of
// latencies where it is short (one token of 12 heads at 1023 slots: 8.6 us: the
// launch, the share of the work, the first copies, the join of the parts); in
// fp32 from 16 rows on the issue of FMA and shared-memory loads by two warps a
// scheduler (8 rows of 24 at 39062 slots, D = 64: 141 us, 16.5 TFLOP/s).
#include "tree_attn.cuh"

namespace {

using namespace fxb_tree;

constexpr int kBlockKeys = 64;          // keys of a block, dealt out to the warps
constexpr int kRows = 16;               // rows of a tile

// ------------------------------------------------------------------ few rows
template <typename T, int D> struct Shape {
  static constexpr int kTile = sizeof(T) == 4 && D == 128 ? 8 : 16;  // keys a warp takes at once
  static constexpr int kWarps = kBlockKeys / kTile, kThreads = kWarps * 32;
  static constexpr int kBoxCols = 128 / sizeof(T);           // columns of a 128-byte swizzled row
  static constexpr int kBoxes = D / kBoxCols;
  static constexpr int kOperand = kTile * D * sizeof(T);      // one warp's keys (or values)
  static constexpr int kSlot = 2 * kOperand;                  // of one stage; >= 16 rows of O in fp32
  static constexpr int kStages = sizeof(T) == 4 || D == 128 ? 3 : 6;
  static constexpr int kQPitch = D + 4;                       // fp32: rows of Q in shared memory
  static constexpr int kQBytes = sizeof(T) == 4 ? kRows * kQPitch * 4 : 0;
  static constexpr int kPBytes = sizeof(T) == 4 ? kWarps * (kTile * kRows + kRows) * 4 : 0;
  static constexpr int kSmem = 1024 + kWarps * kStages * kSlot + kQBytes + kPBytes;
  // 98 KB under way in a thread block, two blocks an SM; fp32 with D = 128 takes 196 KB for as many keys
  static constexpr int kCtas = kSmem <= 112 * 1024 ? 2 : 1;   // thread blocks of an SM
};
// offset of element d of row r of O in a slot: 32-byte pieces exchanged by row, so that the
// eight rows that a warp's accumulators hold at once fall into different banks
template <int D> FXB_DEV int o_at(int r, int d) { return r * D + ((((d >> 3) ^ (r & 7)) << 3) | (d & 7)); }

FXB_DEV void ldmatrix4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
FXB_DEV void ldmatrix4t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T> FXB_DEV void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <> FXB_DEV void mma16816<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> FXB_DEV void mma16816<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// byte offset of 16-byte piece c of row r of an operand in shared memory (128-byte swizzle)
template <int ROWS> FXB_DEV uint32_t sw(int r, int c) {
  return (c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// 16-bit types: m16n8k16 products. A lane holds, of rows lane / 4 and lane / 4
// + 8, two columns of every eight.
template <typename T, int D>
struct Rows16 {
  static constexpr int kHeld = kRows, kTile = Shape<T, D>::kTile;
  uint32_t q[D / 16][4];
  float o[D / 8][4];
  float m[2], l[2];
  uint64_t see[2];
  bool live[2];  // rows of nodes that exist; the others see nothing

  FXB_DEV void begin(const Params& a, int b, int hk, int row0, int n, float*) {
    const int lane = threadIdx.x & 31;
    const T* base = static_cast<const T*>(a.q) + b * a.q_sb + 2 * (lane & 3);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = row0 + (lane >> 2) + 8 * i, t = r / a.G;
      live[i] = r < a.R && t < n;
      see[i] = live[i] ? (uint64_t)a.mask[b * a.mask_sb + t] : 0;
      const T* p = base + t * a.q_st + (hk * a.G + (r - t * a.G)) * a.q_sh;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        q[k][i] = live[i] ? *reinterpret_cast<const uint32_t*>(p + k * 16) : 0u;
        q[k][i + 2] = live[i] ? *reinterpret_cast<const uint32_t*>(p + k * 16 + 8) : 0u;
      }
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  }

  // context tile: keys [0, valid) count. Tree tile (tree): the nodes
  // node0 + j, j < valid, each for the rows that see it.
  FXB_DEV void tile(const Params& a, uint8_t* slot, int valid, bool tree, int node0, const float*, float*) {
    const int lane = threadIdx.x & 31;
    const uint32_t sk = smem_u32(slot), sv = sk + Shape<T, D>::kOperand;
    // scores of 16 rows x 16 keys; even and odd slices of D apart, for two shorter chains of products
    const bool full = valid == kTile && !tree;
    float s[2][4] = {}, s1[2][4] = {};
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      uint32_t f[4];
      ldmatrix4(sk + sw<kTile>((lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)), f);
      mma16816<T>(k & 1 ? s1[0] : s[0], q[k], f[0], f[1]);
      mma16816<T>(k & 1 ? s1[1] : s[1], q[k], f[2], f[3]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] += s1[i][e];
    if (!full) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = i * 8 + 2 * (lane & 3) + (e & 1);
          if (j >= valid || (tree && !((see[e >> 1] >> (node0 + j)) & 1))) s[i][e] = -INFINITY;
        }
    }
    // The reference maximum m of a row moves only when a tile exceeds it by
    // more than 2^8: probabilities then stay below 2^8, which fp32 sums and
    // 16-bit probabilities hold as well as [0, 1], and O is rarely rescaled.
    float mx[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      mx[h] = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2)) * a.scale_log2;
    }
    const bool up0 = mx[0] > m[0] + kRescaleLog2, up1 = mx[1] > m[1] + kRescaleLog2;
    if (__any_sync(0xffffffffu, up0 || up1)) {
      const float m0 = up0 ? mx[0] : m[0], m1 = up1 ? mx[1] : m[1];
      const float r0 = up0 ? ex2(m[0] - m0) : 1.f, r1 = up1 ? ex2(m[1] - m1) : 1.f;
      m[0] = m0;
      m[1] = m1;
      l[0] *= r0;
      l[1] *= r1;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][0] *= r0;
        o[i][1] *= r0;
        o[i][2] *= r1;
        o[i][3] *= r1;
      }
    }
    const float z0 = m[0] == -INFINITY ? 0.f : m[0], z1 = m[1] == -INFINITY ? 0.f : m[1];
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float p0 = ex2(fmaf(s[i][0], a.scale_log2, -z0)), p1 = ex2(fmaf(s[i][1], a.scale_log2, -z0));
      const float p2 = ex2(fmaf(s[i][2], a.scale_log2, -z1)), p3 = ex2(fmaf(s[i][3], a.scale_log2, -z1));
      l[0] += p0 + p1;
      l[1] += p2 + p3;
      // The probabilities enter the second product in the inputs' type, as both of its operands have one type: the
      // error against 64 bits is 1.35 times that of fp32 probabilities (bf16 2.3e-3 for 1.7e-3). A second product
      // with what the rounding leaves brings it to 1.0 times, but takes 200 us for 190 (48 rows of up to 8192 slots,
      // without a pause, at the clock of the power limit), and makes NaN of an infinite value where nothing, or less than 0, is left.
      p[2 * i] = pack2<T>(p0, p1);
      p[2 * i + 1] = pack2<T>(p2, p3);
    }
    if (!full) {
      // values that no row may count are zeroed (0 * NaN is NaN): those behind
      // the sequence, and infinities and NaN in nodes, which are then added
      // to the rows that see them
      uint8_t* vs = slot + Shape<T, D>::kOperand;
      bool odd = false;
      for (int i = lane; i < kTile * (D / 8); i += 32) {
        const int r = i / (D / 8), c = i - r * (D / 8);
        uint4* x = reinterpret_cast<uint4*>(vs + sw<kTile>(r, c));
        if (r >= valid) {
          *x = make_uint4(0, 0, 0, 0);
        } else if (tree) {
          float f[8];
          unpack8<T>(*x, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) odd |= !(fabsf(f[e]) < INFINITY);
        }
      }
      __syncwarp();
      if (__any_sync(0xffffffffu, odd)) {
        for (int j = 0; j < valid; ++j)
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            const float2 f = unpack2<T>(*reinterpret_cast<const uint32_t*>(vs + sw<kTile>(j, i) + 4 * (lane & 3)));
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if ((see[h] >> (node0 + j)) & 1) {
                if (!(fabsf(f.x) < INFINITY)) o[i][2 * h] += f.x;
                if (!(fabsf(f.y) < INFINITY)) o[i][2 * h + 1] += f.y;
              }
          }
        __syncwarp();
        for (int i = lane; i < valid * D; i += 32) {
          T* x = reinterpret_cast<T*>(vs + sw<kTile>(i / D, (i % D) / 8)) + i % 8;
          if (!(fabsf(to_f<T>(*x)) < INFINITY)) *x = from_f<T>(0.f);
        }
      }
      fence_proxy_async_smem();  // these writes come before the next copy into the stage
      __syncwarp();
    }
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      uint32_t f[4];
      ldmatrix4t(sv + sw<kTile>((lane & 7) + (((lane >> 3) & 1) << 3), 2 * c + (lane >> 4)), f);
      mma16816<T>(o[2 * c], p, f[0], f[1]);
      mma16816<T>(o[2 * c + 1], p, f[2], f[3]);
    }
  }

  FXB_DEV void end(float* slot, float* sm, float* sl) {
    const int lane = threadIdx.x & 31, r = lane >> 2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x = l[h] + __shfl_xor_sync(0xffffffffu, l[h], 1);
      x += __shfl_xor_sync(0xffffffffu, x, 2);
      if ((lane & 3) == 0) {
        sm[r + 8 * h] = live[h] ? m[h] : -INFINITY;
        sl[r + 8 * h] = live[h] ? x : 0.f;
      }
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<float2*>(slot + o_at<D>(r + 8 * h, i * 8 + 2 * (lane & 3))) =
            live[h] ? make_float2(o[i][2 * h], o[i][2 * h + 1]) : make_float2(0.f, 0.f);
    }
  }
};

// fp32: FMA, two at once (fma.rn.f32x2). A warp holds the first N rows of a
// tile: 4, 8 or 16, the fewest that hold the call's rows (4 rows of 2 nodes x
// 13 heads at 6009 slots, D = 128: 61 us with 4, 107 with 16; 3 rows of 5 nodes
// at 517 slots, D = 64: 9.8 us with 8, 11.8 with 16). The scores, summed in
// parts of D, lie four rows and every eighth key to a lane (with N < 16 in
// kSplit copies). For O a lane has all N rows, two to a register pair, and
// D / 32 columns. 8 keys a warp and eight warps for D = 128 (that case with 16
// keys and four warps: 84 us), 16 keys and two blocks of four warps for D = 64
// (8 rows of 24 at 39062 slots: 159 us, 237 with 8 keys and eight warps; 141 us
// now that the swizzle's places are found once a tile).
FXB_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
FXB_DEV uint64_t pair_of(float x, float y) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
FXB_DEV float2 halves(uint64_t x) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(x));
  return d;
}
FXB_DEV ulonglong2 load2(const uint8_t* p) { return *reinterpret_cast<const ulonglong2*>(p); }
template <int D, int N>
struct Rows32 {
  static constexpr int kHeld = N, kTile = Shape<float, D>::kTile;
  static constexpr int C = D / 32, kKeys = kTile / 8, kGroups = N / 4, kSplit = 4 / kGroups;
  uint64_t o[N / 2][C];
  float m[4], l[4];
  uint64_t see[4];
  bool live[4];

  // place of a piece of a key's row in a box (128-byte swizzle); a tile's few places are found once, everything
  // else is a constant
  FXB_DEV static uint32_t key_at(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }
  FXB_DEV static int group() { return (threadIdx.x & 31) / 8 % kGroups; }
  FXB_DEV static int split() { return (threadIdx.x & 31) / 8 / kGroups; }
  // Probabilities lie by key, pieces of four rows exchanged by key: a lane's stores then fall into different banks
  FXB_DEV static float* p_at(float* sp, int j, int r) { return sp + j * N + ((r / 4) ^ (j / (32 / N) & (N / 4 - 1))) * 4; }

  FXB_DEV void begin(const Params& a, int b, int hk, int row0, int n, float* sq) {
    __syncthreads();  // the previous item's Q has been read
    for (int i = threadIdx.x; i < N * (D / 4); i += Shape<float, D>::kThreads) {
      const int rr = i / (D / 4), d = (i - rr * (D / 4)) * 4, r = row0 + rr, t = r / a.G;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < a.R && t < n)
        x = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + b * a.q_sb + t * a.q_st +
                                             (hk * a.G + (r - t * a.G)) * a.q_sh + d);
      *reinterpret_cast<float4*>(sq + rr * (D + 4) + d) = x;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = row0 + group() * 4 + i, t = r / a.G;
      live[i] = r < a.R && t < n;
      see[i] = live[i] ? (uint64_t)a.mask[b * a.mask_sb + t] : 0;
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < N / 2; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c) o[r][c] = 0;
    __syncthreads();
  }

  FXB_DEV void tile(const Params& a, uint8_t* slot, int valid, bool tree, int node0, const float* sq, float* sp) {
    const int lane = threadIdx.x & 31, rg = group() * 4, kg = lane & 7;
    const uint8_t* vs = slot + Shape<float, D>::kOperand;
    float s[4][kKeys];
    if constexpr (kKeys == 2) {  // four rows x keys kg and kg + 8 x every kSplit-th piece of D
      uint64_t acc[4][2] = {};
      const float* qs = sq + rg * (D + 4) + split() * 4;
      uint32_t at[8 / kSplit];
#pragma unroll
      for (int x = 0; x < 8 / kSplit; ++x) at[x] = key_at(kg, x * kSplit + split());
#pragma unroll
      for (int x = 0; x < D / 4 / kSplit; ++x) {
        const int box = x * kSplit / 8;
        const ulonglong2 k0 = load2(slot + at[x % (8 / kSplit)] + box * kTile * 128);
        const ulonglong2 k1 = load2(slot + at[x % (8 / kSplit)] + box * kTile * 128 + 8 * 128);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(qs + i * (D + 4) + x * kSplit * 4);
          acc[i][0] = fma2(q.y, k0.y, fma2(q.x, k0.x, acc[i][0]));
          acc[i][1] = fma2(q.y, k1.y, fma2(q.x, k1.x, acc[i][1]));
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 h = halves(acc[i][e]);
          s[i][e] = h.x + h.y;
#pragma unroll
          for (int w = 8 * kGroups; w < 32; w *= 2) s[i][e] += __shfl_xor_sync(0xffffffffu, s[i][e], w);
        }
    } else {
      // kIn rows x keys lane % 4 and + 4 x one of kParts parts of D; bit 2 of the lane is bit 2 of the piece,
      // which keeps eight lanes' pieces of K in different banks
      constexpr int kIn = N < 8 ? N : 8, kParts = 8 * kIn / N < 8 ? 4 : 8, kPieces = D / 4 / kParts;
      const int s0 = (lane >> 2) & 1, s1 = (lane >> 3) & 1, hi = lane >> 4;
      const int c0 = 4 * s0 + 8 * s1 + (kParts == 8 ? hi * 16 : 0);
      const float* rows = sq + (kParts == 8 ? 0 : hi * 8) * (D + 4) + c0 * 4;
      uint32_t at[4];
#pragma unroll
      for (int x = 0; x < 4; ++x)
        at[x] = (c0 >> 3) * kTile * 128 + key_at(lane & 3, (c0 & 7) + x);
      uint64_t acc[kIn][2] = {};
#pragma unroll
      for (int x = 0; x < kPieces; ++x) {
        const int c = (x & 3) + (x >> 2) * 16;  // behind c0
        const ulonglong2 k0 = load2(slot + at[x & 3] + (x >> 2) * 2 * kTile * 128);
        const ulonglong2 k1 = load2(slot + (at[x & 3] ^ 64) + 4 * 128 + (x >> 2) * 2 * kTile * 128);
#pragma unroll
        for (int i = 0; i < kIn; ++i) {
          const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(rows + i * (D + 4) + c * 4);
          acc[i][0] = fma2(q.y, k0.y, fma2(q.x, k0.x, acc[i][0]));
          acc[i][1] = fma2(q.y, k1.y, fma2(q.x, k1.x, acc[i][1]));
        }
      }
      // the parts add up: a lane keeps one of its two keys, then four of its rows
      float w[kIn];
#pragma unroll
      for (int i = 0; i < kIn; ++i) {
        const float2 x0 = halves(acc[i][0]), x1 = halves(acc[i][1]);
        const float y0 = x0.x + x0.y, y1 = x1.x + x1.y;
        w[i] = (s0 ? y1 : y0) + __shfl_xor_sync(0xffffffffu, s0 ? y0 : y1, 4);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (kIn == 8)
          s[i][0] = (s1 ? w[4 + i] : w[i]) + __shfl_xor_sync(0xffffffffu, s1 ? w[i] : w[4 + i], 8);
        else
          s[i][0] = w[i] + __shfl_xor_sync(0xffffffffu, w[i], 8);
        if constexpr (kParts == 8) s[i][0] += __shfl_xor_sync(0xffffffffu, s[i][0], 16);
      }
    }
    float r[4], p[4][kKeys];
    bool moved = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = -INFINITY;
#pragma unroll
      for (int e = 0; e < kKeys; ++e) {
        const int j = kg + 8 * e;
        const bool in = j < valid && (tree ? (see[i] >> (node0 + j)) & 1 : live[i]);
        s[i][e] = in ? s[i][e] * a.scale_log2 : -INFINITY;
        x = fmaxf(x, s[i][e]);
      }
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
      const bool up = x > m[i] + kRescaleLog2;  // (as in Rows16: O is rarely rescaled)
      r[i] = up ? ex2(m[i] - x) : 1.f;
      if (up) m[i] = x;
      moved |= up;
      l[i] *= r[i];
#pragma unroll
      for (int e = 0; e < kKeys; ++e) {
        p[i][e] = ex2(s[i][e] - (m[i] == -INFINITY ? 0.f : m[i]));
        l[i] += p[i][e];
      }
    }
    float* factors = sp + kTile * N;
    if (split() == 0) {
#pragma unroll
      for (int e = 0; e < kKeys; ++e)
        *reinterpret_cast<float4*>(p_at(sp, kg + 8 * e, rg)) = make_float4(p[0][e], p[1][e], p[2][e], p[3][e]);
    }
    moved = __any_sync(0xffffffffu, moved);
    if (moved && kg == 0 && split() == 0) *reinterpret_cast<float4*>(factors + rg) = make_float4(r[0], r[1], r[2], r[3]);
    __syncwarp();
    if (moved) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(factors + i);
#pragma unroll
        for (int c = 0; c < C; ++c) {
          o[i / 2][c] = fma2(o[i / 2][c], f.x, 0);
          o[i / 2 + 1][c] = fma2(o[i / 2 + 1][c], f.y, 0);
        }
      }
    }
    const int piece = C == 4 ? lane : lane >> 1;
    const uint8_t* vp = vs + (piece >> 3) * (kTile * 128) + (C == 4 ? 0 : 8 * (lane & 1));
    auto values = [&](const uint8_t* at, float* v) {
      if constexpr (C == 4) {
        const float4 x = *reinterpret_cast<const float4*>(at);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(at);
        v[0] = x.x; v[1] = x.y;
      }
    };
    if (valid == kTile && !tree) {
      uint32_t at[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) at[j] = ((piece & 7) ^ j) << 4;
#pragma unroll
      for (int j = 0; j < kTile; ++j) {
        float v[C];
        values(vp + at[j & 7] + j * 128, v);
        uint64_t vv[C];
#pragma unroll
        for (int c = 0; c < C; ++c) vv[c] = pair_of(v[c], v[c]);
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(p_at(sp, j, i));
#pragma unroll
          for (int c = 0; c < C; ++c) {
            o[i / 2][c] = fma2(w.x, vv[c], o[i / 2][c]);
            o[i / 2 + 1][c] = fma2(w.y, vv[c], o[i / 2 + 1][c]);
          }
        }
      }
    } else {  // values that count for some rows only: weight 0 is no product
#pragma unroll 1
      for (int j = 0; j < valid; ++j) {
        float v[C];
        values(vp + (((piece & 7) ^ (j & 7)) << 4) + j * 128, v);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
          const float2 w = *reinterpret_cast<const float2*>(p_at(sp, j, i) + (i & 2));
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const float2 x = halves(o[i / 2][c]);
            o[i / 2][c] = pair_of(w.x != 0.f ? fmaf(w.x, v[c], x.x) : x.x, w.y != 0.f ? fmaf(w.y, v[c], x.y) : x.y);
          }
        }
      }
    }
    __syncwarp();
  }

  FXB_DEV void end(float* slot, float* sm, float* sl) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = l[i] + __shfl_xor_sync(0xffffffffu, l[i], 1);
      x += __shfl_xor_sync(0xffffffffu, x, 2);
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      if ((lane & 7) == 0 && split() == 0) {
        sm[group() * 4 + i] = m[i];
        sl[group() * 4 + i] = x;
      }
    }
    __syncwarp();
#pragma unroll
    for (int r = 0; r < N; r += 2) {
      const bool any0 = sm[r] != -INFINITY, any1 = sm[r + 1] != -INFINITY;  // (weights of 0 times infinity are NaN)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float2 x = halves(o[r / 2][c]);
        slot[o_at<D>(r, lane * C + c)] = any0 ? x.x : 0.f;
        slot[o_at<D>(r + 1, lane * C + c)] = any1 ? x.y : 0.f;
      }
    }
  }
};

// The nodes' keys and values into the cache. Nodes that one warp takes
// leave the first to the products: the others copy.
template <typename T, int D>
FXB_DEV void store_nodes(const Params& a, int b, int hk, const Row& row) {
  constexpr int kPer = 16 / sizeof(T), CH = D / kPer;  // 16-byte pieces of a row
  constexpr int kThreads = Shape<T, D>::kThreads;
  const int skip = row.n <= Shape<T, D>::kTile ? 32 : 0, tid = (int)threadIdx.x - skip;
  if (tid < 0) return;
  const T* k = static_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh;
  const T* v = static_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh;
  for (int i = tid; i < row.n * CH; i += kThreads - skip) {
    const int t = i / CH, d = (i % CH) * kPer;
    const uint4 xk = *reinterpret_cast<const uint4*>(k + t * a.k_st + d);
    const uint4 xv = *reinterpret_cast<const uint4*>(v + t * a.v_st + d);
    const int64_t pos = (int64_t)row.len + t, pi = pos >> a.page_shift;
    const int pg = pi < a.W ? a.table[b * a.table_sb + pi] : -1;
    if (pg < 0 || pg >= a.P) {
      atomicOr(a.err, FXB_DERR_PAGES);
      continue;
    }
    const int64_t off = pos & ((1 << a.page_shift) - 1);
    *reinterpret_cast<uint4*>(static_cast<T*>(a.kp) + pg * a.kp_sp + hk * a.kp_sh + off * a.kp_st + d) = xk;
    *reinterpret_cast<uint4*>(static_cast<T*>(a.vp) + pg * a.vp_sp + hk * a.vp_sh + off * a.vp_st + d) = xv;
  }
}

template <typename T, int D, int N> struct RowsOf { using type = Rows16<T, D>; };
template <int D, int N> struct RowsOf<float, D, N> { using type = Rows32<D, N>; };

template <typename T, int D, int N>
__global__ void __launch_bounds__(Shape<T, D>::kThreads, Shape<T, D>::kCtas)
tree_attn_rows(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
               const __grid_constant__ CUtensorMap tmNK, const __grid_constant__ CUtensorMap tmNV, const Params a) {
  using S = Shape<T, D>;
  constexpr int ST = S::kStages, kTile = S::kTile, kWarps = S::kWarps, kThreads = S::kThreads;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[kWarps][ST];
  __shared__ float sm[kWarps][kRows], sl[kWarps][kRows];
  __shared__ int s_last;
  __shared__ Scratch scratch;
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = smem + warp * ST * S::kSlot;
  float* sq = reinterpret_cast<float*>(smem + kWarps * ST * S::kSlot);
  float* sp = sq + S::kQBytes / 4 + warp * (kTile * kRows + kRows);
  if (lane == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(smem_u32(&bars[warp][i]), 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmNK);
    tma_prefetch_desc(&tmNV);
  }
  __syncwarp();
  pdl_trigger();
  pdl_wait();

  int64_t start;
  Shares shares;
  const int nodes = (int)blockIdx.x < a.B ? a.n_nodes[blockIdx.x] : 1;
  Cursor c = share<kBlockKeys, kThreads, true>(a, &start, &shares, scratch);
  idle_rows<T, D, kThreads>(a, nodes);
  if (c.left == 0) return;
  Cursor f = c;          // the next block to fetch
  int f_stage = 0;       // and its stage
  unsigned armed = 0;    // bit s: the copy in stage s is under way, or there and not yet used
  // Page ids, read ahead: lane i has those of this warp's keys in block base + i of f's row (window), in block
  // base + 32 + i (ahead), and in block i (front: where every key head of the row begins again)
  const int in_block = warp * kTile;
  auto pages_at = [&](int base) {
    const int64_t at = ((int64_t)(base + lane) * kBlockKeys + in_block) >> a.page_shift;
    return at < a.W ? a.table[f.b * a.table_sb + at] : -1;
  };
  int base = f.j, window = pages_at(base), ahead = pages_at(base + 32), front = pages_at(0);
  auto fetch = [&]() {  // block f into its stage; moves f on
    if (f.left == 0) return;
    if (f.j >= base + 32) {
      base += 32;
      window = ahead;
      ahead = pages_at(base + 32);
    }
    const bool tree = f.j == f.row.blocks - 1;
    const int at = tree ? in_block : f.j * kBlockKeys + in_block;
    const int pg = __shfl_sync(0xffffffffu, window, f.j - base);
    bool go = at < (tree ? f.row.n : f.row.len);
    if (go && !tree && (pg < 0 || pg >= a.P)) {
      if (lane == 0) atomicOr(a.err, FXB_DERR_PAGES);
      go = false;
    }
    if (go) armed |= 1u << f_stage;
    if (go && lane == 0) {
      const uint32_t bar = smem_u32(&bars[warp][f_stage]), dst = smem_u32(ring + f_stage * S::kSlot);
      const int row = tree ? at : at & ((1 << a.page_shift) - 1), d3 = tree ? f.b : pg;
      mbar_expect_tx(bar, S::kSlot);
#pragma unroll
      for (int x = 0; x < S::kBoxes; ++x) {
        tma_load_4d(dst + x * kTile * 128, tree ? &tmNK : &tmK, bar, x * S::kBoxCols, row, f.hk, d3);
        tma_load_4d(dst + S::kOperand + x * kTile * 128, tree ? &tmNV : &tmV, bar, x * S::kBoxCols, row, f.hk, d3);
      }
    }
    f_stage = f_stage + 1 == ST ? 0 : f_stage + 1;
    const int b = f.b;
    next<kBlockKeys>(a, f);
    if (f.j == 0 && f.left) {
      if (f.b != b) front = pages_at(0);
      if (f.b != b || base) ahead = pages_at(32);
      base = 0;
      window = front;
    }
  };
  typename RowsOf<T, D, N>::type rows;
  rows.begin(a, c.b, c.hk, c.rt * kRows, c.row.n, sq);  // the loads of Q are under way while the ring fills
  for (int i = 0; i < ST; ++i) fetch();

  unsigned phase = 0;    // bit s: parity of stage s
  bool ok = true, fresh = false;
  int64_t u_begin = start - c.j;   // the item's first block
  for (int s = 0, done = 0; c.left; s = s + 1 == ST ? 0 : s + 1, ++done) {
    const int hk = c.hk, row0 = c.rt * kRows;
    uint8_t* slot = ring + s * S::kSlot;
    if (fresh) {
      rows.begin(a, c.b, hk, row0, c.row.n, sq);
      u_begin = start + done - c.j;
      fresh = false;
    }
    const bool tree = c.j == c.row.blocks - 1;
    if (tree && row0 == 0) store_nodes<T, D>(a, c.b, hk, c.row);
    if (ok && ((armed >> s) & 1)) {
      ok = mbar_wait_warp(smem_u32(&bars[warp][s]), (phase >> s) & 1, a.err, FXB_DERR_ATTN_WAIT);
      if (ok) {
        armed &= ~(1u << s);
        phase ^= 1u << s;
        const int at = tree ? in_block : c.j * kBlockKeys + in_block;
        const int valid = min(kTile, (tree ? c.row.n : c.row.len) - at);
        rows.tile(a, slot, valid, tree, at, sq, sp);
      }
    }
    const Cursor cur = c;
    next<kBlockKeys>(a, c);
    if (tree || c.left == 0) {
      // the warps' states join; each lies in the stage that its warp has just used up
      __syncwarp();
      rows.end(reinterpret_cast<float*>(slot), sm[warp], sl[warp]);
      __syncthreads();
      const bool begun = u_begin >= start;  // this block has the item's first keys
      const bool whole = begun && tree;
      float* part = part_of<kRows, D>(a, blockIdx.x, begun);
      constexpr int kHeld = decltype(rows)::kHeld;
      for (int i = threadIdx.x; i < kHeld * (D / 4); i += kThreads) {
        const int r = i % kHeld, d = i / kHeld * 4;
        float mx = sm[0][r];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, sm[w][r]);
        float l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float wt = weight(sm[w][r], mx);
          const float* so = reinterpret_cast<const float*>(smem + w * ST * S::kSlot + s * S::kSlot);
          axpy4(o, wt, *reinterpret_cast<const float4*>(so + o_at<D>(r, d)));
          l = fmaf(sl[w][r], wt, l);
        }
        if (whole) {
          write_out<T, D>(a, cur.b, hk, row0 + r, d, o, l);
        } else {
          if (d == 0) {
            part[r] = mx;
            part[kRows + r] = l;
          }
          reinterpret_cast<float4*>(part + 2 * kRows)[(d / 4) * kRows + r] = o;
        }
      }
      if (!whole) {  // the last thread block to arrive joins the parts
        const int2 own = shares.owners(u_begin, cur.row.blocks);
        const int lo = own.x, hi = own.y;
        __syncthreads();
        if (threadIdx.x == 0) {
          __threadfence();  // after the barrier: for the whole block's writes
          const unsigned before = atomicAdd(&a.arrived[lo], 1u);
          s_last = before == (unsigned)(hi - lo);
          if (s_last) a.arrived[lo] = 0;  // for the next call
        }
        __syncthreads();
        if (s_last) {
          __threadfence();
          // 16 lanes of a row's quad: few rows leave several lanes for the parts of one
          constexpr int kStep = kThreads / kRows;
          const int live = min(kRows, a.R - row0);
          const int lanes = live > 8 ? 16 : (live > 4 ? 8 : (live > 2 ? 4 : live));
          const int x = threadIdx.x % kRows;
          join_row<T, kRows, D, D / 4 / kStep, 128 / D * 2>(a, cur.b, hk, row0, x % lanes, threadIdx.x / kRows, kStep, lo, hi,
                                               x / lanes, kRows / lanes, lanes);
        }
      }
      __syncthreads();
      fence_proxy_async_smem();  // what was written here comes before the copies into it
      fresh = true;
    }
    __syncwarp();
    if (ok) fetch();
  }
  // after an expired wait copies may be under way: they land before shared memory goes
  for (int s = 0; s < ST; ++s)
    if ((armed >> s) & 1) mbar_wait_warp(smem_u32(&bars[warp][s]), (phase >> s) & 1, a.err, FXB_DERR_ATTN_WAIT);
}

// ------------------------------------------------------------------ host
template <typename T> constexpr CUtensorMapDataType map_type() {
  return sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
         : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                          : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}
// Few or many rows of a key head. The first kernel reads the cache once for
// every 16 rows and leaves 16 x 16 products to a warp; the second takes up to
// 128 rows with one reading, in tiles of 128 whatever the number of rows. From
// 17 rows on the second reading costs more than the empty rows (16 rows of 24
// at 6000 slots, D = 128: 57.5 us against 84.8; 4 rows of 32 at 30000: 78
// against 125; 8 rows of 48 at 1000, D = 64: 20.1 against 22.5), but for short
// caches, where both are near a launch (2 rows of 18 at 100 slots: 9.3 against
// 8.6). The lengths lie on the device, so the rule cannot ask for them. More
// than 128 query heads a key head do not fit a tile of whole nodes.
bool many_rows(int dtype, int T, int G) { return dtype != FXB_DTYPE_F32 && T * G > kRows && G <= 128; }

template <typename T, int D> constexpr int rows_ctas() { return Shape<T, D>::kCtas; }
int rows_grid(int dtype, int D) {
  const int ctas = dtype == FXB_DTYPE_F32 ? (D == 64 ? rows_ctas<float, 64>() : rows_ctas<float, 128>())
                                          : (D == 64 ? rows_ctas<__half, 64>() : rows_ctas<__half, 128>());
  return ctas * fxb::num_sms();
}

size_t workspace_bytes(const fxb_tree_attn_args* x) {
  if (many_rows(x->dtype, x->T, x->Hq / x->Hkv)) return wide_workspace(x);
  return kCounters + (size_t)rows_grid(x->dtype, x->D) * 2 * kRows * (x->D + 2) * sizeof(float);
}

template <typename T, int D, int N = kRows>
int launch(const fxb_tree_attn_args* x, Params& a, void* stream) {
  using S = Shape<T, D>;
  CUtensorMap k, v, nk, nv;
  const auto t = map_type<T>();
  const int e = sizeof(T);
  if (int r = encode_rows(&k, t, e, x->k_pages, D, x->page, x->kp_st, x->Hkv, x->kp_sh, x->P, x->kp_sp, S::kTile, 1)) return r;
  if (int r = encode_rows(&v, t, e, x->v_pages, D, x->page, x->vp_st, x->Hkv, x->vp_sh, x->P, x->vp_sp, S::kTile, 1)) return r;
  if (int r = encode_rows(&nk, t, e, x->k, D, x->T, x->k_st, x->Hkv, x->k_sh, x->B, x->k_sb, S::kTile, 1)) return r;
  if (int r = encode_rows(&nv, t, e, x->v, D, x->T, x->v_st, x->Hkv, x->v_sh, x->B, x->v_sb, S::kTile, 1)) return r;
  a.RT = (a.R + kRows - 1) / kRows;
  const int grid = grid_of(x, a, kBlockKeys, rows_grid(x->dtype, D));
  if (int r = fxb::check_cuda(
          cudaFuncSetAttribute(tree_attn_rows<T, D, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem),
          "fxb_tree_attn"))
    return r;
  fxb::pdl_launch(tree_attn_rows<T, D, N>, dim3(grid), dim3(S::kThreads), S::kSmem, fxb::as_stream(stream), k, v, nk, nv, a);
  return fxb::check_launch("fxb_tree_attn");
}

}  // namespace

extern "C" {

size_t fxb_tree_attn_workspace(int32_t dtype, int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t D) {
  if ((D != 64 && D != 128) || !fxb::dtype_size(dtype) || B < 1 || T < 1 || Hkv < 1 || Hq < Hkv) return 0;
  fxb_tree_attn_args x = {};
  x.dtype = dtype;
  x.B = B;
  x.T = T;
  x.Hq = Hq;
  x.Hkv = Hkv;
  x.D = D;
  return workspace_bytes(&x);
}
size_t fxb_tree_attn_workspace_zeroed(int32_t dtype, int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t D) {
  return fxb_tree_attn_workspace(dtype, B, T, Hq, Hkv, D) ? kCounters : 0;
}

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
  // a mask's row stride of 0: one tree for all batch rows (a table's would put all rows' nodes into the same slots)
  if (a->P < 1 || a->W < 1 || a->table_sb < a->W || (a->mask_sb < a->T && a->mask_sb != 0))
    return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: P=%d W=%d, or a row stride of table or mask too small", a->P,
                          a->W);
  const void* ptr[6] = {a->q, a->k, a->v, a->o, a->k_pages, a->v_pages};
  for (const void* p : ptr)
    if (!p || !fxb::aligned16(p))
      return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: q, k, v, o and the pages must be 16-byte aligned");
  if (!a->table || !a->lens || !a->n_nodes || !a->mask)
    return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: table, lens, n_nodes or mask is NULL");
  const struct { int64_t entries, stride; } st[18] = {  // the stride of an axis of one entry is not used
      {a->B, a->q_sb}, {a->T, a->q_st}, {a->Hq, a->q_sh}, {a->B, a->k_sb}, {a->T, a->k_st}, {a->Hkv, a->k_sh},
      {a->B, a->v_sb}, {a->T, a->v_st}, {a->Hkv, a->v_sh}, {a->B, a->o_sb}, {a->T, a->o_st}, {a->Hq, a->o_sh},
      {a->P, a->kp_sp}, {a->Hkv, a->kp_sh}, {a->page, a->kp_st}, {a->P, a->vp_sp}, {a->Hkv, a->vp_sh}, {a->page, a->vp_st}};
  for (const auto& s : st)
    if (s.entries > 1 && (s.stride < 0 || (s.stride * e) % 16))
      return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: strides must be multiples of 16 bytes");
  if (!(a->scale > 0.f) || !(a->scale < INFINITY))
    return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: scale must be positive and finite");
  const int G = a->Hq / a->Hkv;
  if (!a->workspace || !fxb::aligned16(a->workspace) ||
      a->workspace_bytes < (int64_t)workspace_bytes(a))
    return fxb::set_error(FXB_EINVAL, "fxb_tree_attn: workspace of fxb_tree_attn_workspace bytes, 16-byte aligned");
  if (rows_grid(a->dtype, a->D) > kMaxGrid)
    return fxb::set_error(FXB_EUNSUPPORTED, "fxb_tree_attn: device with too many SMs");
  int* err = fxb::dev_error_ptr();
  if (!err) return FXB_ECUDA;
  Params p = {};
  p.B = a->B;
  p.T = a->T;
  p.Hq = a->Hq;
  p.Hkv = a->Hkv;
  p.G = G;
  p.R = p.T * p.G;
  p.page_shift = shift;
  p.P = a->P;
  p.W = a->W;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.o = a->o;
  p.kp = a->k_pages;
  p.vp = a->v_pages;
  p.q_sb = a->q_sb; p.q_st = a->q_st; p.q_sh = a->q_sh;
  p.o_sb = a->o_sb; p.o_st = a->o_st; p.o_sh = a->o_sh;
  p.k_sb = a->k_sb; p.k_st = a->k_st; p.k_sh = a->k_sh;
  p.v_sb = a->v_sb; p.v_st = a->v_st; p.v_sh = a->v_sh;
  p.kp_sp = a->kp_sp; p.kp_sh = a->kp_sh; p.kp_st = a->kp_st;
  p.vp_sp = a->vp_sp; p.vp_sh = a->vp_sh; p.vp_st = a->vp_st;
  p.table = a->table;
  p.table_sb = a->table_sb;
  p.lens = a->lens;
  p.n_nodes = a->n_nodes;
  p.mask = a->mask;
  p.mask_sb = a->mask_sb;
  p.arrived = static_cast<unsigned*>(a->workspace);
  p.parts = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + kCounters);
  p.err = err;
  if (many_rows(a->dtype, a->T, G)) return launch_wide(a, p, stream);
  if (a->dtype == FXB_DTYPE_F32) {
    if (p.R <= 4) return a->D == 64 ? launch<float, 64, 4>(a, p, stream) : launch<float, 128, 4>(a, p, stream);
    if (p.R <= 8) return a->D == 64 ? launch<float, 64, 8>(a, p, stream) : launch<float, 128, 8>(a, p, stream);
    return a->D == 64 ? launch<float, 64>(a, p, stream) : launch<float, 128>(a, p, stream);
  }
  if (a->dtype == FXB_DTYPE_F16)
    return a->D == 64 ? launch<__half, 64>(a, p, stream) : launch<__half, 128>(a, p, stream);
  return a->D == 64 ? launch<__nv_bfloat16, 64>(a, p, stream)
                    : launch<__nv_bfloat16, 128>(a, p, stream);
}

}  // extern "C"
