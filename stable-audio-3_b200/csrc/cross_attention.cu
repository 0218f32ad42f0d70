// Attention of queries to an encoder's states of another length, forward and backward, on tcgen05 for sm_100a:
// key heads shared by groups of query heads, heads of 64 or 128 columns, packed or uniform batches, per-sequence
// key lengths and a key mask.
//
//   S = scale * Q K^T, hidden keys -inf;  P = softmax(S);  O = P V;  lse = log sum exp S
//   delta = rowsum(dO * O);  dP = dO V^T;  dS = P * (dP - delta)
//   dQ = scale * dS K;  dK = scale * dS^T Q;  dV = P^T dO      (dK, dV summed over the query heads of the group)
//
// A row without visible keys gives O = 0, lse = -inf and no gradient. What stands in hidden keys and behind the
// ends of sequences may be anything, NaN included: scores of hidden keys are replaced, never scaled, and rows that
// a contraction would multiply by a zero probability (V and K of hidden keys, Q and dO behind a sequence's end)
// are zeroed in shared memory before the tensor core reads them.
//
// Sums, softmax statistics and accumulators are fp32; P and dS are rounded once to the operands' 16-bit type, the
// type of the matrix instructions.
#include <type_traits>

#include "attn_tile.cuh"
#include "common.cuh"
#include "cross_attention.cuh"
#include "host_util.h"

namespace sa3 {
SA3_DEFINE_ERROR_READER(read_error_cross)

constexpr int XA_BM = 128;  // rows of the wide side of a tile: queries (forward, dQ) or keys (dK / dV)
constexpr int XA_BN = 64;   // rows of the walked side: keys (forward, dQ) or queries (dK / dV)
constexpr float XA_LOG2E = 1.4426950408889634f;
constexpr float XA_MOST = 32768.f;  // largest sum of a step's exponentials that keeps a row's reference maximum
constexpr int XA_SUB_M = XA_BM * 128;   // bytes of a 64-column sub-tile of the wide side
constexpr int XA_SUB_N = XA_BN * 128;   // ... of the walked side

// the lowest min(n, 64) bits
__device__ __forceinline__ uint64_t low_bits64(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// Bit i: key j0 + i of the sequence is visible (i < 64). All lanes of a warp call it and get the same word.
__device__ __forceinline__ uint64_t visible64(const XParams& p, const XSeq& s, int j0, int lane) {
  const int n = s.seen - j0;
  if (!p.key_mask) return low_bits64(n);
  const uint8_t* m = p.key_mask + s.ks + j0;
  const bool a = lane < n && __ldg(m + lane) != 0, b = lane + 32 < n && __ldg(m + lane + 32) != 0;
  const uint32_t lo = __ballot_sync(0xffffffffu, a), hi = __ballot_sync(0xffffffffu, b);
  return ((uint64_t)hi << 32) | lo;
}

// A whole warp zeroes those of `rows` <= 64 rows of a tile (subs sub-tiles of 64 columns, `sub` bytes apart) whose bit in
// `keep` is clear. A row is 128 contiguous bytes of a sub-tile: the 128-byte swizzle only permutes its 16-byte chunks.
__device__ __forceinline__ void zero_rows(uint8_t* tile, int subs, int sub, int rows, uint64_t keep, int lane) {
  const int chunk = lane & 7;
  for (int r = lane >> 3; r < rows; r += 4)
    if (!((keep >> r) & 1))
      for (int c = 0; c < subs; ++c)
        *reinterpret_cast<uint4*>(tile + c * sub + r * 128 + chunk * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
}

// 4 bytes from global to shared memory, or zeros
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}

__device__ __forceinline__ float unpack_lo(uint32_t w, bool f16) {
  return f16 ? __half2float(__ushort_as_half((unsigned short)(w & 0xffffu))) : __uint_as_float(w << 16);
}
__device__ __forceinline__ float unpack_hi(uint32_t w, bool f16) {
  return f16 ? __half2float(__ushort_as_half((unsigned short)(w >> 16))) : __uint_as_float(w & 0xffff0000u);
}

__device__ __forceinline__ float max32(const uint32_t (&s)[32]) {
  float m[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) m[e] = -INFINITY;
  max_chunk(s, m);
  return fmaxf(fmax3(fmax3(m[0], m[1], m[2]), m[3], m[4]), fmax3(m[5], m[6], m[7]));
}

// scores of hidden columns become -inf
__device__ __forceinline__ void hide32(uint32_t (&s)[32], uint32_t vis) {
#pragma unroll
  for (int e = 0; e < 32; ++e) s[e] = (vis >> e) & 1u ? s[e] : NEG_INF_BITS;
}

// A softmax warp's 32 TMEM lanes x NC columns, times f (0 where !keep), rounded to 16 bits, to the first `rows` of 32
// rows at dst. A lane holds one row: CW columns at a time go through 64 * CW bytes of shared memory (16-byte chunks
// exchanged within a row so that neither side has bank conflicts), so that a store instruction writes CW consecutive
// columns of several rows and not 8 of 32.
template <int NC, int CW>
__device__ __forceinline__ void store_rows16(uint32_t t_src, float f, bool keep, bool f16, uint8_t* stage, int lane,
                                             int rows, uint16_t* dst, long long ld) {
  constexpr int LPR = CW / 8, RPI = 32 / LPR;  // lanes a row, rows an instruction
  auto slot = [](int r, int c) {
    return r * (CW * 2) + ((c ^ (CW == 64 ? r & 7 : CW == 32 ? (r >> 1) & 3 : (r >> 2) & 1)) << 4);
  };
  uint16_t* out = dst + (lane / LPR) * ld + (lane % LPR) * 8;
#pragma unroll
  for (int c = 0; c < NC / CW; ++c) {
    uint32_t w[CW / 2];
#pragma unroll
    for (int x = 0; x < CW / 16; ++x) {
      uint32_t o[16];
      tmem_ld16(t_src + CW * c + 16 * x, o);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        w[8 * x + e] = keep ? pack_2(__uint_as_float(o[2 * e]) * f, __uint_as_float(o[2 * e + 1]) * f, f16) : 0u;
    }
#pragma unroll
    for (int e = 0; e < LPR; ++e)
      *reinterpret_cast<uint4*>(stage + slot(lane, e)) = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
    __syncwarp();
#pragma unroll
    for (int e = 0; e < LPR; ++e) {
      const int r = RPI * e + lane / LPR;
      const uint4 v = *reinterpret_cast<const uint4*>(stage + slot(r, lane % LPR));
      if (r < rows) *reinterpret_cast<uint4*>(out + RPI * e * ld + CW * c) = v;
    }
    __syncwarp();
  }
}
constexpr int XA_STAGE = 32 * 32;  // bytes of a warp's pass of 16 columns
// one lane's row, directly
template <int NC>
__device__ __forceinline__ void store_row16(uint32_t t_src, float f, bool f16, bool store, uint16_t* dst) {
#pragma unroll
  for (int c = 0; c < NC / 32; ++c) {
    uint32_t o[32], w[16];
    tmem_ld32_async(t_src + 32 * c, o);
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 16; ++e)
      w[e] = pack_2(__uint_as_float(o[2 * e]) * f, __uint_as_float(o[2 * e + 1]) * f, f16);
    if (store) {
      uint4* d = reinterpret_cast<uint4*>(dst) + 4 * c;
#pragma unroll
      for (int e = 0; e < 4; ++e) d[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
    }
  }
}
// The swizzled tiles need a base on a 1024-byte boundary. Dynamic shared memory starts on one when a kernel has no
// static shared memory; if it ever did not, the kernel would report that and do nothing.
__device__ __forceinline__ bool aligned_base(const uint8_t* smem) {
  if ((smem_u32(smem) & 1023) == 0) return true;
  if (threadIdx.x == 0) record_error(SA3_DEVERR_TIMEOUT, 119);
  return false;
}
template <int D>
__device__ __forceinline__ void zero_row16(void* dst) {
#pragma unroll
  for (int e = 0; e < D / 8; ++e) reinterpret_cast<uint4*>(dst)[e] = make_uint4(0, 0, 0, 0);
}

// one lane's NC columns in fp32
template <int NC>
__device__ __forceinline__ void store_rows32(uint32_t t_src, float f, bool keep, bool store, float* dst) {
#pragma unroll
  for (int c = 0; c < NC / 32; ++c) {
    uint32_t o[32];
    tmem_ld32_async(t_src + 32 * c, o);
    tmem_wait_ld();
    if (store)
#pragma unroll
      for (int e = 0; e < 32; e += 4)
        *reinterpret_cast<float4*>(dst + 32 * c + e) =
            keep ? make_float4(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f, __uint_as_float(o[e + 2]) * f,
                               __uint_as_float(o[e + 3]) * f)
                 : make_float4(0.f, 0.f, 0.f, 0.f);
  }
}

// The walk of a persistent CTA over work items: query rows (fastest), head, part of the keys, sequence. Every role of
// the CTA walks by itself. Uniform batches step by the grid without divisions, which would delay each item's first
// product. Packed ones number only the tiles that their sequences have: numbering the tiles up to the longest sequence
// leaves some CTAs with few that exist (4 sequences of 1255 .. 2500 queries: 111 -> 69 us forward, 172 -> 106 us dQ).
// XA_SCAN sequences at most, since a CTA orders them first and finding an item's sequence takes a step for each: 64 of
// 75 .. 435 queries, 24 heads of 64 columns: 123 -> 105 us forward, 476 -> 413 backward, and 69 -> 73, 358 -> 362 where
// all are alike; 128 of half the length, without the order: 121 -> 143, 652 -> 638.
constexpr int XA_SCAN = 64;
// The sequences of a packed batch in the order of their items: longest keys first, so that no CTA begins with a long
// item when the others are done. Where the key tiles differ, the CTAs take every other round of items backwards: the
// one with a round's longest has the next round's shortest (337 -> 315 us for the four sequences, both passes; with
// equal keys that only costs, 67 -> 72 us forward for 16384 queries x 257 keys x 24 heads).
struct XOrder {
  int back;                 // whether
  int starts[XA_SCAN + 1];  // items before the sequence, and all items
  uint8_t seq[XA_SCAN];
};
constexpr int XA_ORDER = sizeof(XOrder);
// By one warp, for batches of 1 .. XA_SCAN.
template <int ROWS, int KEYS>
__device__ __forceinline__ void make_order(XOrder* o, const XParams& p, int lane) {
  static_assert(XA_SCAN == 64, "two sequences a lane");
  int keys[2], items[2], rank[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int b = 32 * e + lane;
    keys[e] = items[e] = 0;
    if (b < p.batch) {
      const XSeq s = make_seq(p, b);
      keys[e] = s.seen;
      items[e] = (s.lq + ROWS - 1) / ROWS * p.heads * p.parts;
    }
  }
  int most = 0, least = 0x7fffffff;
  for (int b = 0; b < p.batch; ++b) {
    const int x = __shfl_sync(0xffffffffu, b < 32 ? keys[0] : keys[1], b & 31);
    most = max(most, x);
    least = min(least, x);
#pragma unroll
    for (int e = 0; e < 2; ++e) rank[e] += x > keys[e] || (x == keys[e] && b < 32 * e + lane);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (32 * e + lane < p.batch) {
      o->seq[rank[e]] = (uint8_t)(32 * e + lane);
      o->starts[rank[e] + 1] = items[e];
    }
  }
  __syncwarp();
  const int at = 2 * lane;
  const int x = at < p.batch ? o->starts[at + 1] : 0, y = at + 1 < p.batch ? o->starts[at + 2] : 0;
  int sum = x + y;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += up;
  }
  if (lane == 0) {
    o->starts[0] = 0;
    o->back = (most + KEYS - 1) / KEYS != (least + KEYS - 1) / KEYS;
  }
  if (at < p.batch) o->starts[at + 1] = sum - y;
  if (at + 1 < p.batch) o->starts[at + 2] = sum;
}
template <int ROWS, int KEYS, bool SCAN>  // query rows of an item, keys of a tile, packed numbering
struct XWalk {
  XSeq s;
  int tile, h, part, b;  // the item; b: packed, its place in the order
  int j0, T;             // its keys: from j0, in T tiles; T = 0 also for a tile behind the end of its sequence
  bool live;             // there is an item
  int item, dt, dh, dp, db, qtiles;
  const XOrder* order;
  __device__ __forceinline__ void load(const XParams& p) {
    const int all = tile * ROWS < s.lq ? (s.seen + KEYS - 1) / KEYS : 0;
    T = all;
    j0 = 0;
    if (p.parts > 1) {
      const int t0 = (int)((long long)all * part / p.parts);
      T = (int)((long long)all * (part + 1) / p.parts) - t0;
      j0 = t0 * KEYS;
    }
  }
  // packed: the sequence, tile, head and part of `item`
  __device__ __forceinline__ void find(const XParams& p) {
    const int was = b;
    if (b < 0) b = 0;
    while (item >= order->starts[b + 1]) {
      if (++b == p.batch) {
        live = false;
        return;
      }
    }
    if (b != was) s = make_seq(p, order->seq[b]);
    const int tiles = (s.lq + ROWS - 1) / ROWS;
    int x = item - order->starts[b];
    tile = x % tiles, x /= tiles, h = x % p.heads, part = x / p.heads;
    load(p);
  }
  __device__ __forceinline__ XWalk(const XParams& p, int qt, int num_items, const XOrder* o) {
    qtiles = qt;
    int x = item = blockIdx.x;
    live = item < num_items;
    if (SCAN) {
      order = o;
      b = -1;
      dt = o->back ? 2 * (int)(gridDim.x - blockIdx.x) - 1 : gridDim.x;
      if (live) find(p);
      return;
    }
    tile = x % qt, x /= qt, h = x % p.heads, x /= p.heads, part = x % p.parts, b = x / p.parts;
    x = gridDim.x;
    dt = x % qt, x /= qt, dh = x % p.heads, x /= p.heads, dp = x % p.parts, db = x / p.parts;
    if (live) {
      s = make_seq(p, b);
      load(p);
    }
  }
  __device__ __forceinline__ void next(const XParams& p, int num_items) {
    if (SCAN) {
      item += dt;
      dt = 2 * (int)gridDim.x - dt;
    } else {
      item += gridDim.x;
    }
    live = item < num_items;
    if (!live) return;
    if (SCAN) {
      find(p);
      return;
    }
    tile += dt;
    int c = tile >= qtiles;
    tile -= c ? qtiles : 0;
    h += dh + c;
    c = h >= p.heads;
    h -= c ? p.heads : 0;
    part += dp + c;
    c = part >= p.parts;
    part -= c ? p.parts : 0;
    const int was = b;
    b += db + c;
    if (b != was) s = make_seq(p, b);
    load(p);
  }
};

// A CTA's softmax warps come first, then a warp that loads and two that issue products: in the forward one a unit, in
// dQ one for the scores and one for dS K. A warp alone takes some ten cycles an instruction; with one issuer for all,
// its loop set the time of a tile (dQ of 2 x 8247 queries x 257 keys x 24 heads: 162 -> 113 us).
constexpr int XA_THREADS = 384;
constexpr int XA_SOFTMAX = 8;      // softmax warps of the dQ kernel: arrivals on the barriers that they release
constexpr int XA_REGS_LAUNCH = 80;  // two CTAs an SM
constexpr int XA_REGS_LOW = 48;     // loads and MMA after the split
constexpr int XA_REGS_HIGH = 96;    // softmax after the split
static_assert(XA_REGS_LOW * 128 + XA_REGS_HIGH * 256 <= XA_REGS_LAUNCH * XA_THREADS,
              "register split exceeds the block's launch allocation");
__device__ __forceinline__ void regs_low() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(XA_REGS_LOW)); }
__device__ __forceinline__ void regs_high() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(XA_REGS_HIGH)); }
// the two softmax warps that share a lane quarter (64 threads)
__device__ __forceinline__ void pair_sync(int quarter) { asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory"); }

// ------------------------------------------------------------------------------------------------ forward
// Persistent, two CTAs an SM. A unit is a query tile of 128 rows with four softmax warps (a thread a row) and an issuing
// warp; D = 64 has two units a CTA, which share the key tiles, D = 128 one. A unit owns 128 or 256 columns of TMEM:
// two score buffers of SB = 32 or 64 columns and O. It works in steps of SB keys: S = Q K^T, the softmax (which writes
// P over its S), O (+)= P V. The next step's S is ready before the softmax gets to it; S of step n + 2 is sent right
// behind P V of step n, whose P it overwrites: one thread's products run in order, so nothing has to come back in
// between. Bound by the chain barrier - TMEM load - exponentials - TMEM store - barrier - products of a step, of which
// an SM has four (D = 64) or two (D = 128) to run past each other: 68 us on 2 x 8247 queries x 257 keys x 24 heads (23
// for the exponentials alone), 1034 TFLOP/s on 4099 x 6001 with 16 heads of 128 columns (62 % of the measured peak).
// Work item = (query rows of the CTA's units, head, part of the keys, sequence), query rows fastest, so CTAs that run
// together share K/V in L2. The softmax takes a row's maximum over its first visible step only, as the reference of
// the exponentials, and moves it when a step's sum shows that a score lies far above.
template <int D>
struct XFwd {
  static constexpr int SUBS = D / 64;
  static constexpr int UNITS = D == 64 ? 2 : 1, BN = 64, COLS = 256 / UNITS;
  static constexpr int SB = (COLS - D) / 2, SPT = BN / SB;  // keys of a step, steps of a key tile
  static constexpr int SOFTMAX = 4 * UNITS, THREADS = 32 * (SOFTMAX + 4);
  static constexpr int QS = D == 64 ? 2 : 1, KS = 2;
  static constexpr int SUB_N = BN * 128;  // bytes of 64 columns of a key tile
  static constexpr int Q_BYTES = SUBS * XA_SUB_M, T_BYTES = SUBS * SUB_N;
  static constexpr int TILES = UNITS * QS * Q_BYTES + 2 * KS * T_BYTES;
  static constexpr int CW = D == 64 ? 32 : 64, STAGE = 64 * CW;  // columns of a store pass, bytes of a warp's
  static constexpr int SMEM = TILES + SOFTMAX * STAGE + 320 + XA_ORDER;
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two CTAs an SM");
};

template <int D, bool F16, bool SCAN>
__global__ void __launch_bounds__(XFwd<D>::THREADS, 2)
    cross_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const XParams p, int num_items, int qtiles) {
  using C = XFwd<D>;
  using Walk = XWalk<C::UNITS * XA_BM, C::BN, SCAN>;
  constexpr int U = C::UNITS, BN = C::BN, SB = C::SB;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  if (!aligned_base(smem)) return;
  auto sQ = [&](int u, int s) { return smem + (u * C::QS + s) * C::Q_BYTES; };
  auto sK = [&](int s) { return smem + U * C::QS * C::Q_BYTES + s * C::T_BYTES; };
  auto sV = [&](int s) { return smem + U * C::QS * C::Q_BYTES + (C::KS + s) * C::T_BYTES; };
  uint8_t* stage = smem + C::TILES;  // STAGE bytes a softmax warp
  uint64_t* bars = reinterpret_cast<uint64_t*>(stage + C::SOFTMAX * C::STAGE);
  uint64_t* q_full = bars;        // [unit][QS]
  uint64_t* q_empty = bars + 4;   // [unit][QS]
  uint64_t* k_full = bars + 8;    // [KS]
  uint64_t* k_empty = bars + 10;  // [KS] (an arrival of each unit)
  uint64_t* v_full = bars + 12;   // [KS]
  uint64_t* v_empty = bars + 14;  // [KS] (an arrival of each unit)
  uint64_t* s_full = bars + 16;   // [unit][2] scores of a step are in TMEM
  uint64_t* p_full = bars + 20;   // [unit][2] its probabilities are (4 arrivals)
  // [unit][2] P V of a step is done. Two, since the softmax skips most of these phases: when it waits for step n's it
  // knows that step n - 2's is over, so the parity on the step's own barrier cannot be that of an older phase.
  uint64_t* o_full = bars + 24;
  uint64_t* o_empty = bars + 28;  // [unit] the softmax has read an item's O (4 arrivals)
  uint64_t* done = bars + 30;     // [unit]
  constexpr int NBARS = 32;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + NBARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert(NBARS * 8 + 8 <= 320, "barriers");
  XOrder* order = reinterpret_cast<XOrder*>(bars + 40);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NBARS; ++i)
      mbar_init(&bars[i], (i >= 20 && i < 24) || i == 28 || i == 29 ? 4 : i == 10 || i == 11 || i == 14 || i == 15 ? U : 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dep_wait();
  if (SCAN) {
    if (warp == 0) make_order<U * XA_BM, BN>(order, p, lane);
    __syncthreads();
  }
  // units of an item that have query rows
  auto units_of = [&](const Walk& it) { return U == 1 || (it.tile * U + 1) * XA_BM >= it.s.lq ? 1 : U; };

  if (U == 2 && warp >= C::SOFTMAX) regs_low();
  if (warp == C::SOFTMAX) {
    if (lane == 0) {
      int g = 0, qc[2] = {0, 0};
      bool ok = true, v_out = true;  // v_out: V of the last counted tile was issued
      for (Walk it(p, qtiles, num_items, order); it.live && ok; it.next(p, num_items)) {
        if (it.T == 0) continue;
        const XSeq& s = it.s;
        const int cq = it.h * D, ck = (it.h / p.group) * D, nu = units_of(it);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u >= nu || !ok) break;
          const int qs = qc[u] % C::QS;
          uint64_t* full = &q_full[u * 2 + qs];
          if (qc[u] >= C::QS && !bar_wait(&q_empty[u * 2 + qs], ((qc[u] / C::QS) - 1) & 1, abort_flag, 100)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(full, C::Q_BYTES);
          for (int c = 0; c < C::SUBS; ++c)
            tma_load_2d(sQ(u, qs) + c * XA_SUB_M, &tmQ, full, cq + 64 * c, s.qs + (it.tile * U + u) * XA_BM);
          qc[u]++;
        }
        for (int t = 0; t < it.T && ok; ++t, ++g) {
          const int ks = g % C::KS, row = s.ks + it.j0 + t * BN;
          if (g >= C::KS && !bar_wait(&k_empty[ks], ((g / C::KS) - 1) & 1, abort_flag, 101)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&k_full[ks], C::T_BYTES);
          for (int c = 0; c < C::SUBS; ++c) tma_load_2d(sK(ks) + c * C::SUB_N, &tmK, &k_full[ks], ck + 64 * c, row);
          if (g >= C::KS && !bar_wait(&v_empty[ks], ((g / C::KS) - 1) & 1, abort_flag, 102)) {
            g++;
            ok = v_out = false;
            break;
          }
          mbar_arrive_expect_tx(&v_full[ks], C::T_BYTES);
          for (int c = 0; c < C::SUBS; ++c) tma_load_2d(sV(ks) + c * C::SUB_N, &tmV, &v_full[ks], ck + 64 * c, row);
        }
      }
      if (*abort_flag) {
        // wait (bounded, ignoring the abort flag) for the last loads this thread issued
        volatile int never = 0;
        for (int u = 0; u < U; ++u)
          for (int c = max(qc[u] - C::QS, 0); c < qc[u]; ++c)
            bar_wait(&q_full[u * 2 + c % C::QS], (c / C::QS) & 1, &never, 103);
        for (int c = max(g - C::KS, 0); c < g; ++c) {
          bar_wait(&k_full[c % C::KS], (c / C::KS) & 1, &never, 103);
          if (c + 1 < g || v_out) bar_wait(&v_full[c % C::KS], (c / C::KS) & 1, &never, 103);
        }
      }
    }
  } else if (warp > C::SOFTMAX && warp <= C::SOFTMAX + U) {
    // ------------------------------------------------------------------ products of unit u
    const int u = uniform_int(warp) - C::SOFTMAX - 1;
    const int fmt = F16 ? 0 : 1;
    const uint32_t base = uniform_int(smem_u32(smem));
    const uint64_t dk = sdesc_kmajor_sw128(base), dv = sdesc_mnmajor_sw128(base + U * C::QS * C::Q_BYTES + C::KS * C::T_BYTES, C::SUB_N);
    const uint32_t k_hi = (uint32_t)(dk >> 32), k_lo = (uint32_t)dk;
    const uint32_t v_hi = (uint32_t)(dv >> 32), v_lo = (uint32_t)dv;
    const uint32_t idesc_full = make_idesc(128, SB, fmt, fmt, 0, 0), idesc_o = make_idesc(128, D, fmt, fmt, 0, 1);
    const uint32_t tm = uniform_int(tmem), t_s = tm + C::COLS * u, t_o = t_s + 2 * SB;
    uint64_t *my_s = &s_full[2 * u], *my_p = &p_full[2 * u], *my_o = &o_full[2 * u];
    int g = 0, gn = 0, qc = 0;  // key tiles seen, steps of this unit's items, its items
    bool ok = true;
    for (Walk it(p, qtiles, num_items, order); it.live && ok; it.next(p, num_items)) {
      const int T = uniform_int(it.T);
      if (T == 0) continue;
      if (u >= uniform_int(units_of(it))) {
        // the other unit's item: hand its tiles back
        for (int t = 0; t < T && ok; ++t, ++g) {
          ok = warp_bar_wait(&k_full[g % C::KS], (g / C::KS) & 1, abort_flag, 105) &&
               warp_bar_wait(&v_full[g % C::KS], (g / C::KS) & 1, abort_flag, 106);
          if (ok && lane == 0) {
            mbar_arrive(&k_empty[g % C::KS]);
            mbar_arrive(&v_empty[g % C::KS]);
          }
        }
        continue;
      }
      const int qs = qc % C::QS;
      const uint32_t qlo = k_lo + (((u * C::QS + qs) * C::Q_BYTES) >> 4);
      const int keys = uniform_int(min(it.s.seen - it.j0, T * BN)), N = (keys + SB - 1) / SB;  // keys and steps of the item
      auto scores = [&](int n) {
        const int tile = g + n / C::SPT, ks = tile % C::KS;
        if (n % C::SPT == 0 && !warp_bar_wait(&k_full[ks], (tile / C::KS) & 1, abort_flag, 105)) return false;
        tc_fence_after();
        const int left = keys - n * SB;
        const uint32_t idesc = left >= SB ? idesc_full : make_idesc(128, (left + 15) & ~15, fmt, fmt, 0, 0);
        const uint32_t klo = k_lo + ((U * C::QS * C::Q_BYTES + ks * C::T_BYTES + (n % C::SPT) * SB * 128) >> 4);
        const int b = (gn + n) & 1;
#pragma unroll
        for (int c = 0; c < C::SUBS; ++c)
          mma4_ss(t_s + SB * b, qlo + c * (XA_SUB_M >> 4), klo + c * (C::SUB_N >> 4), k_hi, idesc, c != 0);
        if (n % C::SPT == C::SPT - 1 || n == N - 1)
          commit2_elect(&my_s[b], &k_empty[ks]);
        else
          commit_elect(&my_s[b]);
        if (n == N - 1) commit_elect(&q_empty[u * 2 + qs]);
        return true;
      };
      ok = warp_bar_wait(&q_full[u * 2 + qs], (qc / C::QS) & 1, abort_flag, 104) && scores(0) && (N < 2 || scores(1)) &&
           (qc == 0 || warp_bar_wait(&o_empty[u], (qc - 1) & 1, abort_flag, 108));
      for (int n = 0; n < N && ok; ++n) {
        const int tile = g + n / C::SPT, vs = tile % C::KS, left = keys - n * SB;
        if (n % C::SPT == 0) {
          ok = warp_bar_wait(&v_full[vs], (tile / C::KS) & 1, abort_flag, 106);
          if (!ok) break;
          if (p.key_mask || left < BN) {
            // V of hidden keys, which P V multiplies by zero (the CTA's other unit may write the same zeros)
            const int rows = min(BN, (left + 15) & ~15);
            const uint64_t vis = visible64(p, it.s, it.j0 + n * SB, lane), all = low_bits64(rows);
            if ((vis & all) != all) zero_rows(sV(vs), C::SUBS, C::SUB_N, rows, vis, lane);
          }
        }
        const int b = (gn + n) & 1;
        ok = warp_bar_wait(&my_p[b], ((gn + n) >> 1) & 1, abort_flag, 107);
        if (!ok) break;
        tc_fence_after();
        const uint32_t vlo = v_lo + ((vs * C::T_BYTES + (n % C::SPT) * SB * 128) >> 4), t_p = t_s + SB * b;
        if (SB == 64 && left >= SB) {
          mma4_ts(t_o, t_p, t_p + 16, vlo, v_hi, idesc_o, n > 0);
        } else {
#pragma unroll
          for (int k = 0; k < SB / 16; ++k)
            if (left > 16 * k)
              mma_ts_lo(t_o, t_p + 8 * k, vlo + k * (2048 >> 4), v_hi, idesc_o, (n > 0 || k > 0) ? 1u : 0u);
        }
        if (n % C::SPT == C::SPT - 1 || n == N - 1)
          commit2_elect(&my_o[b], &v_empty[vs]);
        else
          commit_elect(&my_o[b]);
        if (n + 2 < N) ok = scores(n + 2);
      }
      g += T;
      gn += N;
      qc++;
    }
    commit_elect(&done[u]);
    volatile int never = 0;
    warp_bar_wait(&done[u], 0, &never, 109);
  } else if (warp < C::SOFTMAX) {
    if (U == 2) regs_high();
    const int u = warp >> 2, quarter = warp & 3;
    const uint32_t t_u = tmem + ((uint32_t)(quarter * 32) << 16) + C::COLS * u, t_o = t_u + 2 * SB;
    uint64_t *my_s = &s_full[2 * u], *my_p = &p_full[2 * u], *my_o = &o_full[2 * u];
    const float NEG_INF = -INFINITY;
    const uint64_t scale2 = f2(p.scale_log2, p.scale_log2);
    int gn = 0;
    for (Walk it(p, qtiles, num_items, order); it.live; it.next(p, num_items)) {
      const XSeq& s = it.s;
      const int T = it.T, i0 = (it.tile * U + u) * XA_BM;
      if (i0 >= s.lq) continue;
      const int rows = min(32, s.lq - i0 - quarter * 32);  // of this warp that exist
      bool bad = false;
      float m = NEG_INF, l = 0.f;
      int left = min(s.seen - it.j0, T * BN);  // keys of this step and the following ones
      const int N = (left + SB - 1) / SB;
      for (int n = 0; n < N; ++n, ++gn, left -= SB) {
        const bool masked = p.key_mask != nullptr || left < SB;
        uint64_t vis = ~0ull;
        if (masked) vis = visible64(p, s, it.j0 + n * SB, lane);
        const int b = gn & 1;
        const uint32_t t_s = t_u + SB * b;
        if (!bar_wait(&my_s[b], (gn >> 1) & 1, abort_flag, 110)) bad = true;
        tc_fence_after();
        if (rows > 0) {  // else no row of this warp exists: what P holds there is multiplied and never stored
          uint32_t sc[SB / 32][32], w[SB / 2];
#pragma unroll
          for (int c = 0; c < SB / 32; ++c) tmem_ld32_async(t_s + 32 * c, sc[c]);
          tmem_wait_ld();
          if (masked) {
#pragma unroll
            for (int c = 0; c < SB / 32; ++c) hide32(sc[c], (uint32_t)(vis >> (32 * c)));
          }
          float sum;
          auto exponentials = [&]() {
            const float mu = m == NEG_INF ? 0.f : m;
            const uint64_t negm2 = f2(-mu, -mu);
            uint64_t acc[4] = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < SB / 32; ++c)
              exp_chunk(sc[c], scale2, negm2, acc, reinterpret_cast<uint32_t(&)[16]>(w[16 * c]), F16);
            const float2 r = f2_split(fadd2(fadd2(acc[0], acc[1]), fadd2(acc[2], acc[3])));
            sum = r.x + r.y;
          };
          // m becomes the maximum of the visible scores so far (scale > 0); what was summed with the old one is scaled
          auto move = [&]() {
            float mx = max32(sc[0]);
            if (SB == 64) mx = fmaxf(mx, max32(sc[SB / 32 - 1]));
            const float top = fmaxf(m, mx * p.scale_log2);
            const float alpha = top > m ? fast_exp2(m - top) : 1.f;
            m = top;
            l *= alpha;
            if (n > 0) {
              if (!bar_wait(&my_o[b ^ 1], ((gn - 1) >> 1) & 1, abort_flag, 111)) bad = true;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 16; ++c) {
                uint32_t o[16];
                tmem_ld16(t_o + 16 * c, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tmem_st16(t_o + 16 * c, o);
              }
            }
          };
          if (__any_sync(0xffffffffu, m == NEG_INF)) move();
          exponentials();
          // A later step is tried with the reference that is there: its sum tells whether a score lies too far above it
          // (P stays below fp16's largest number). Then the reference moves and the step is done again.
          if (__any_sync(0xffffffffu, !(sum <= XA_MOST))) {
            move();
            exponentials();
          }
          l += sum;
#pragma unroll
          for (int c = 0; c < SB / 32; ++c) tmem_st16(t_s + 16 * c, reinterpret_cast<uint32_t(&)[16]>(w[16 * c]));
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&my_p[b]);
      }
      const long long row0 = s.qs + i0 + quarter * 32;
      const long long at = ((long long)it.part * p.heads + it.h) * p.total_q + row0;  // one part: of lse itself
      float* lse = p.parts > 1 ? p.part_lse + at : p.lse ? p.lse + at : nullptr;
      uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + row0 * p.ldo + it.h * D;
      if (T == 0) {
        if (lane < rows) {
          if (p.parts == 1) zero_row16<D>(dst + lane * p.ldo);  // else a part of weight zero: its output is not read
          if (lse) lse[lane] = NEG_INF;
        }
        continue;
      }
      if (!bar_wait(&my_o[(gn - 1) & 1], ((gn - 1) >> 1) & 1, abort_flag, 112)) bad = true;
      tc_fence_after();
      const int put = bad || *abort_flag ? 0 : rows;
      const float inv = l > 0.f ? 1.f / l : 0.f;
      if (rows > 0) {
        if (p.parts > 1)
          store_rows32<D>(t_o, inv, true, lane < put, p.part_o + (at + lane) * D);
        else
          store_rows16<D, C::CW>(t_o, inv, true, F16, stage + warp * C::STAGE, lane, put, dst, p.ldo);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_empty[u]);
      if (lane < put && lse) lse[lane] = l > 0.f ? (m + __log2f(l)) * 0.6931471805599453f : NEG_INF;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 256);
}

// ------------------------------------------------------------------------------------------------ dQ
// The forward's walk again: a CTA holds Q and dO of a query tile, walks the keys, recomputes P from the stored lse
// and accumulates dQ in TMEM. It also forms delta (rowsum(dO * O), or with a single key tile the equal sum of P * dP)
// and stores it for the dK / dV kernel, so delta needs no launch of its own. TMEM (256 columns): S, dP, dQ, and dS (packed pairs) in two
// buffers of its own where they fit (D = 64); at D = 128 dS lies over dP. S of the next tile is multiplied as soon as
// the softmax has read this one's, dP with it at D = 64, and after this tile's dS K at D = 128. 106 us on 2 x 8247
// queries x 257 keys x 24 heads: some 1050 cycles a key tile and SM, and 5000 for an item's start and end, where its
// 64 KB come from DRAM (31 us in all).
template <int D>
struct XDq {
  static constexpr int SUBS = D / 64;
  static constexpr bool SEP = D == 64;
  static constexpr int QS = SEP ? 2 : 1, KS = 2, VS = SEP ? 2 : 1;
  static constexpr int Q_BYTES = SUBS * XA_SUB_M, T_BYTES = SUBS * XA_SUB_N;
  static constexpr int TILES = 2 * QS * Q_BYTES + (KS + VS) * T_BYTES;
  // at D = 128 there is no room to stage the stores
  static constexpr int STAGE = SEP ? XA_SOFTMAX * XA_STAGE : 0;
  static constexpr int SMEM = TILES + STAGE + XA_BM * 4 + 176 + XA_ORDER;
  static constexpr int COL_DQ = 128, COL_DS = SEP ? 192 : 64;
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two CTAs an SM");
};

template <int D, bool F16, bool SCAN>
__global__ void __launch_bounds__(XA_THREADS, 2)
    cross_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                    const __grid_constant__ CUtensorMap tmO, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const XParams p, const XGrad gr, int num_items,
                    int qtiles) {
  using C = XDq<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  if (!aligned_base(smem)) return;
  auto sQ = [&](int s) { return smem + s * C::Q_BYTES; };
  auto sDO = [&](int s) { return smem + (C::QS + s) * C::Q_BYTES; };
  auto sK = [&](int s) { return smem + 2 * C::QS * C::Q_BYTES + s * C::T_BYTES; };
  auto sV = [&](int s) { return smem + 2 * C::QS * C::Q_BYTES + (C::KS + s) * C::T_BYTES; };
  uint8_t* stage = smem + C::TILES;                                   // XA_STAGE bytes a softmax warp
  float* sh_delta = reinterpret_cast<float*>(stage + C::STAGE);       // [rows] of the item
  uint64_t* bars = reinterpret_cast<uint64_t*>(sh_delta + XA_BM);
  uint64_t* q_full = bars;          // [QS] Q and dO
  uint64_t* q_empty = bars + 2;     // [QS]
  uint64_t* k_full = bars + 4;      // [KS]
  uint64_t* k_empty = bars + 6;     // [KS]
  uint64_t* v_full = bars + 8;      // [VS]
  uint64_t* v_empty = bars + 10;    // [VS]
  uint64_t* sdp_full = bars + 12;   // S and dP of a tile are in TMEM
  uint64_t* sdp_empty = bars + 13;  // the softmax holds them in registers (XA_SOFTMAX arrivals)
  uint64_t* ds_full = bars + 14;    // [2] dS is in TMEM (XA_SOFTMAX arrivals)
  uint64_t* dq_full = bars + 16;    // [2] dS K of a tile is done
  uint64_t* dq_empty = bars + 18;   // the softmax has read an item's dQ (XA_SOFTMAX arrivals)
  uint64_t* done = bars + 19;       // [2]
  constexpr int NBARS = 21;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + NBARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert(NBARS * 8 + 8 <= 176, "barriers");
  XOrder* order = reinterpret_cast<XOrder*>(bars + 22);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NBARS; ++i) mbar_init(&bars[i], (i == 13 || i == 14 || i == 15 || i == 18) ? XA_SOFTMAX : 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmDO);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dep_wait();
  if (SCAN) {
    if (warp == 0) make_order<XA_BM, XA_BN>(order, p, lane);
    __syncthreads();
  }

  if (warp >= XA_SOFTMAX) regs_low();
  if (warp == 8) {
    if (lane == 0) {
      int g = 0, qc = 0;
      bool ok = true, v_out = true;  // v_out: V of the last counted tile was issued
      for (XWalk<XA_BM, XA_BN, SCAN> it(p, qtiles, num_items, order); it.live && ok; it.next(p, num_items)) {
        if (it.T == 0) continue;
        const XSeq& s = it.s;
        const int cq = it.h * D, ck = (it.h / p.group) * D;
        const int qs = qc % C::QS;
        if (qc >= C::QS && !bar_wait(&q_empty[qs], ((qc / C::QS) - 1) & 1, abort_flag, 120)) break;
        mbar_arrive_expect_tx(&q_full[qs], 2 * C::Q_BYTES);
        for (int c = 0; c < C::SUBS; ++c) {
          tma_load_2d(sQ(qs) + c * XA_SUB_M, &tmQ, &q_full[qs], cq + 64 * c, s.qs + it.tile * XA_BM);
          tma_load_2d(sDO(qs) + c * XA_SUB_M, &tmDO, &q_full[qs], cq + 64 * c, s.qs + it.tile * XA_BM);
          // O of these rows, which the softmax warps read for delta when they get to the item
          if (it.T > 1) tma_prefetch_l2_2d(&tmO, cq + 64 * c, s.qs + it.tile * XA_BM);
        }
        qc++;
        for (int t = 0; t < it.T; ++t, ++g) {
          const int ks = g % C::KS, vs = g % C::VS, row = s.ks + t * XA_BN;
          if (g >= C::KS && !bar_wait(&k_empty[ks], ((g / C::KS) - 1) & 1, abort_flag, 121)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&k_full[ks], C::T_BYTES);
          for (int c = 0; c < C::SUBS; ++c) tma_load_2d(sK(ks) + c * XA_SUB_N, &tmK, &k_full[ks], ck + 64 * c, row);
          if (g >= C::VS && !bar_wait(&v_empty[vs], ((g / C::VS) - 1) & 1, abort_flag, 122)) {
            g++;
            ok = v_out = false;
            break;
          }
          mbar_arrive_expect_tx(&v_full[vs], C::T_BYTES);
          for (int c = 0; c < C::SUBS; ++c) tma_load_2d(sV(vs) + c * XA_SUB_N, &tmV, &v_full[vs], ck + 64 * c, row);
        }
      }
      if (*abort_flag) {
        volatile int never = 0;
        for (int c = max(qc - C::QS, 0); c < qc; ++c) bar_wait(&q_full[c % C::QS], (c / C::QS) & 1, &never, 123);
        for (int c = max(g - C::KS, 0); c < g; ++c) bar_wait(&k_full[c % C::KS], (c / C::KS) & 1, &never, 123);
        const int gv = v_out ? g : g - 1;
        for (int c = max(gv - C::VS, 0); c < gv; ++c) bar_wait(&v_full[c % C::VS], (c / C::VS) & 1, &never, 123);
      }
    }
  } else if (warp == 9) {
    // S = Q K^T and dP = dO V^T
    const int fmt = F16 ? 0 : 1;
    const uint32_t base = uniform_int(smem_u32(smem)), tm = uniform_int(tmem);
    const uint64_t dk = sdesc_kmajor_sw128(base);
    const uint32_t k_hi = (uint32_t)(dk >> 32), k_lo = (uint32_t)dk;
    const uint32_t idesc_full = make_idesc(128, XA_BN, fmt, fmt, 0, 0);
    int g = 0, qc = 0;
    bool ok = true;
    for (XWalk<XA_BM, XA_BN, SCAN> it(p, qtiles, num_items, order); it.live && ok; it.next(p, num_items)) {
      const int T = uniform_int(it.T), seen = uniform_int(it.s.seen);
      if (T == 0) continue;
      const int qs = qc % C::QS;
      const uint32_t qlo = k_lo + ((qs * C::Q_BYTES) >> 4), dlo = k_lo + (((C::QS + qs) * C::Q_BYTES) >> 4);
      ok = warp_bar_wait(&q_full[qs], (qc / C::QS) & 1, abort_flag, 124);
      for (int t = 0; t < T && ok; ++t, ++g) {
        const int ks = g % C::KS, vs = g % C::VS, left = seen - t * XA_BN;
        ok = warp_bar_wait(&k_full[ks], (g / C::KS) & 1, abort_flag, 125);
        if (!ok) break;
        const int cols = min(XA_BN, (left + 15) & ~15);
        if (p.key_mask || left < XA_BN) {
          const uint64_t vis = visible64(p, it.s, t * XA_BN, lane), all = low_bits64(cols);
          if ((vis & all) != all) zero_rows(sK(ks), C::SUBS, XA_SUB_N, cols, vis, lane);  // dS K multiplies them by zero
        }
        ok = g == 0 || warp_bar_wait(sdp_empty, (g - 1) & 1, abort_flag, 126);
        if (!ok) break;
        tc_fence_after();
        const uint32_t idesc = left >= XA_BN ? idesc_full : make_idesc(128, cols, fmt, fmt, 0, 0);
        const uint32_t klo = k_lo + ((2 * C::QS * C::Q_BYTES + ks * C::T_BYTES) >> 4);
        const uint32_t vlo = k_lo + ((2 * C::QS * C::Q_BYTES + (C::KS + vs) * C::T_BYTES) >> 4);
#pragma unroll
        for (int c = 0; c < C::SUBS; ++c)
          mma4_ss(tm, qlo + c * (XA_SUB_M >> 4), klo + c * (XA_SUB_N >> 4), k_hi, idesc, c != 0);
        ok = warp_bar_wait(&v_full[vs], (g / C::VS) & 1, abort_flag, 125) &&
             (C::SEP || g == 0 || warp_bar_wait(&dq_full[(g - 1) & 1], ((g - 1) >> 1) & 1, abort_flag, 125));
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < C::SUBS; ++c)
          mma4_ss(tm + 64, dlo + c * (XA_SUB_M >> 4), vlo + c * (XA_SUB_N >> 4), k_hi, idesc, c != 0);
        commit2_elect(sdp_full, &v_empty[vs]);
        if (t == T - 1) commit_elect(&q_empty[qs]);
      }
      qc++;
    }
    commit_elect(&done[0]);
    volatile int never = 0;
    warp_bar_wait(&done[0], 0, &never, 129);
  } else if (warp == 10) {
    // dQ (+)= dS K
    const int fmt = F16 ? 0 : 1;
    const uint32_t tm = uniform_int(tmem);
    const uint64_t dm = sdesc_mnmajor_sw128(uniform_int(smem_u32(sK(0))), XA_SUB_N);
    const uint32_t m_hi = (uint32_t)(dm >> 32), m_lo = (uint32_t)dm;
    const uint32_t idesc = make_idesc(128, D, fmt, fmt, 0, 1);
    const uint32_t t_dq = tm + C::COL_DQ;
    int g = 0, qc = 0;
    bool ok = true;
    for (XWalk<XA_BM, XA_BN, SCAN> it(p, qtiles, num_items, order); it.live && ok; it.next(p, num_items)) {
      const int T = uniform_int(it.T), seen = uniform_int(it.s.seen);
      if (T == 0) continue;
      ok = qc == 0 || warp_bar_wait(dq_empty, (qc - 1) & 1, abort_flag, 128);
      for (int t = 0; t < T && ok; ++t, ++g) {
        const int ks = g % C::KS;
        ok = warp_bar_wait(&ds_full[g & 1], (g >> 1) & 1, abort_flag, 127);
        if (!ok) break;
        tc_fence_after();
        const int steps = min(XA_BN / 16, (seen - t * XA_BN + 15) >> 4);
        const uint32_t mlo = m_lo + ((ks * C::T_BYTES) >> 4);
        const uint32_t t_ds = tm + C::COL_DS + (C::SEP ? 32 * (g & 1) : 0);
        if (steps == XA_BN / 16) {
          mma4_ts(t_dq, t_ds, t_ds + (C::SEP ? 16 : 32), mlo, m_hi, idesc, t > 0);
        } else {
          for (int k = 0; k < steps; ++k)
            mma_ts_lo(t_dq, t_ds + (C::SEP ? 16 : 32) * (k >> 1) + 8 * (k & 1), mlo + k * (2048 >> 4), m_hi, idesc, (t > 0 || k > 0) ? 1u : 0u);
        }
        commit2_elect(&dq_full[g & 1], &k_empty[ks]);
      }
      qc++;
    }
    commit_elect(&done[1]);
    volatile int never = 0;
    warp_bar_wait(&done[1], 0, &never, 129);
  } else if (warp < XA_SOFTMAX) {
    regs_high();
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t t_s = tmem + lane_off + 32 * half, t_dq = tmem + lane_off + C::COL_DQ + half * (D / 2);
    const uint64_t scale2 = f2(p.scale_log2, p.scale_log2);
    int g = 0;
    for (XWalk<XA_BM, XA_BN, SCAN> it(p, qtiles, num_items, order); it.live; it.next(p, num_items)) {
      const XSeq& s = it.s;
      if (it.tile * XA_BM >= s.lq) continue;
      const int h = it.h, T = it.T;
      const int rows = min(32, s.lq - it.tile * XA_BM - quarter * 32);  // of this warp that exist
      const long long row0 = s.qs + it.tile * XA_BM + quarter * 32;
      const long long stat = (long long)h * p.total_q + row0;
      float lse = -INFINITY;
      if (lane < rows) lse = __ldg(p.lse + stat + lane);
      // One key tile: delta = sum P * dP over the row's scores below, without O's rounding, which is felt where few keys
      // are averaged, and without reading O and dO. Else delta = rowsum(dO * O).
      const bool single = T == 1;
      float delta = 0.f;
      if (T > 1) {
        // this warp's 16 of the pair's 32 rows, D / 8 lanes a row, 16 bytes each
        constexpr int LPR = D / 8, RPI = 32 / LPR;
        const int c = lane % LPR, first = 16 * half + lane / LPR;
        const uint16_t* po = reinterpret_cast<const uint16_t*>(p.out) + (row0 + first) * p.ldo + h * D + 8 * c;
        const uint16_t* pd = reinterpret_cast<const uint16_t*>(gr.dout) + (row0 + first) * gr.lddo + h * D + 8 * c;
#pragma unroll 1
        for (int n = 0; n < 16; n += 4 * RPI) {
          uint4 o4[4], d4[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = n + e * RPI;
            o4[e] = d4[e] = make_uint4(0, 0, 0, 0);
            if (first + r < rows) {
              o4[e] = __ldg(reinterpret_cast<const uint4*>(po + r * p.ldo));
              d4[e] = __ldg(reinterpret_cast<const uint4*>(pd + r * gr.lddo));
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t ow[4] = {o4[e].x, o4[e].y, o4[e].z, o4[e].w}, dw[4] = {d4[e].x, d4[e].y, d4[e].z, d4[e].w};
            float sum = 0.f;
#pragma unroll
            for (int x = 0; x < 4; ++x)
              sum = fmaf(unpack_hi(ow[x], F16), unpack_hi(dw[x], F16),
                         fmaf(unpack_lo(ow[x], F16), unpack_lo(dw[x], F16), sum));
#pragma unroll
            for (int x = LPR / 2; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            if (c == 0) sh_delta[quarter * 32 + n + e * RPI + first] = sum;
          }
        }
        pair_sync(quarter);
        delta = sh_delta[quarter * 32 + lane];
        pair_sync(quarter);  // both have read it before the next item's is written
      }
      uint16_t* dst = reinterpret_cast<uint16_t*>(gr.dq) + row0 * gr.lddq + h * D + half * (D / 2);
      if (T == 0) {
        if (lane < rows) zero_row16<D / 2>(dst + lane * gr.lddq);
        continue;
      }
      // a row that saw no key has lse = -inf, which stays -inf here: its probabilities come out as zero
      const float nl = lse == -INFINITY ? -INFINITY : -lse * XA_LOG2E;
      const uint64_t negl2 = f2(nl, nl);
      if (half == 0 && lane < rows) gr.stats[stat + lane] = nl;
      bool bad = false;
      int left = s.seen;
      for (int t = 0; t < T; ++t, ++g, left -= XA_BN) {
        uint32_t vis = (uint32_t)(low_bits64(left) >> (32 * half));
        if (p.key_mask) vis = (uint32_t)(visible64(p, s, t * XA_BN, lane) >> (32 * half));
        const uint32_t t_ds = tmem + lane_off + C::COL_DS + (C::SEP ? 32 * (g & 1) + 16 * half : 32 * half);
        if (!bar_wait(sdp_full, g & 1, abort_flag, 130)) bad = true;
        // the dS that last lay in this tile's columns has been multiplied (D = 128: dP was multiplied after it)
        if (C::SEP && g > 1 && !bar_wait(&dq_full[g & 1], ((g - 2) >> 1) & 1, abort_flag, 131)) bad = true;
        tc_fence_after();
        const bool some = rows > 0 && left > 32 * half;  // else no row of this warp exists, or no column
        // the sum of both halves of a row
        auto pair_sum = [&](float x) {
          float* c = sh_delta + quarter * 32 + lane;
          if (half) *c = x;
          pair_sync(quarter);
          if (!half) *c = x += *c;
          pair_sync(quarter);
          x = *c;
          pair_sync(quarter);  // before the next item's is written
          return x;
        };
        auto keep = [&](uint32_t(&w)[16]) {
          if (vis != 0xffffffffu) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              w[e] &= ((vis >> (2 * e)) & 1u ? 0x0000ffffu : 0u) | ((vis >> (2 * e + 1)) & 1u ? 0xffff0000u : 0u);
          }
        };
        if (some) {
          uint32_t sc[32], dp[32], w[16];
          tmem_ld32_async(t_s, sc);
          tmem_ld32_async(t_s + 64, dp);
          tmem_wait_ld();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(sdp_empty);
          if (single) {
            float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 x = f2_split(ffma2(f2(__uint_as_float(sc[e]), __uint_as_float(sc[e + 1])), scale2, negl2));
              const float p0 = fast_exp2(x.x), p1 = fast_exp2(x.y);
              sc[e] = __float_as_uint(p0);
              sc[e + 1] = __float_as_uint(p1);
              // hidden columns may hold anything
              if ((vis >> e) & 1u) part[(e >> 1) & 3] = fmaf(p0, __uint_as_float(dp[e]), part[(e >> 1) & 3]);
              if ((vis >> (e + 1)) & 1u) part[(e >> 1) & 3] = fmaf(p1, __uint_as_float(dp[e + 1]), part[(e >> 1) & 3]);
            }
            delta = pair_sum((part[0] + part[1]) + (part[2] + part[3]));
#pragma unroll
            for (int e = 0; e < 32; e += 2)
              w[e >> 1] = pack_2(__uint_as_float(sc[e]) * (__uint_as_float(dp[e]) - delta),
                                 __uint_as_float(sc[e + 1]) * (__uint_as_float(dp[e + 1]) - delta), F16);
          } else {
            const uint64_t negd2 = f2(-delta, -delta);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 x = f2_split(ffma2(f2(__uint_as_float(sc[e]), __uint_as_float(sc[e + 1])), scale2, negl2));
              const uint64_t pr = f2(fast_exp2(x.x), fast_exp2(x.y));
              const float2 d =
                  f2_split(fmul2(pr, fadd2(f2(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1])), negd2)));
              w[e >> 1] = pack_2(d.x, d.y, F16);
            }
          }
          keep(w);
          tmem_st16(t_ds, w);
          tmem_wait_st();
        } else {
          if (lane == 0) mbar_arrive(sdp_empty);
          if (single && rows > 0) delta = pair_sum(0.f);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_full[g & 1]);
      }
      if (half == 0 && lane < rows) gr.stats[(long long)p.heads * p.total_q + stat + lane] = -delta;
      if (!bar_wait(&dq_full[(g - 1) & 1], ((g - 1) >> 1) & 1, abort_flag, 132)) bad = true;
      tc_fence_after();
      const int put = bad || *abort_flag ? 0 : rows;
      if (rows > 0) {
        if (C::SEP)
          store_rows16<D / 2, 16>(t_dq, p.scale, true, F16, stage + warp * XA_STAGE, lane, put, dst, gr.lddq);
        else
          store_row16<D / 2>(t_dq, p.scale, F16, lane < put, dst + lane * gr.lddq);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dq_empty);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 256);
}

// ------------------------------------------------------------------------------------------------ dK, dV
// A CTA (one an SM) holds K and V of 128 keys of one key head and walks the query tiles of 64 rows of every head of
// the group, or a part of them when there are fewer key tiles than SMs: the parts are then written in fp32 and added
// in a fixed order by a second launch, so results never depend on the order in which CTAs finish. The products are
// taken transposed (S^T = K Q^T, dP^T = V dO^T), which puts P^T and dS^T into TMEM in the form of the A operand of
// dV += P^T dO and dK += dS^T Q, with dO and Q read as they lie. Two score buffers, each with eight softmax warps of its
// own (two to a row): they form P and dS while the tensor core works on the other. TMEM (512 columns): 2 x (S^T 64,
// dP^T 64), dV, dK. Bound by the issuing warp's loop at D = 64 (16 products and two waits a tile: some 1500 cycles for
// 656 of products; 105 us on 2 x 8247 queries x 257 keys x 24 heads), by the products at D = 128.
constexpr int XB_THREADS = 576;  // warps 0..15 softmax (8 to a score buffer, two to a row), 16 loads, 17 MMA
constexpr int XB_SOFTMAX = 8;
template <int D>
struct XDkv {
  static constexpr int SUBS = D / 64;
  static constexpr int STAGES = 4;
  static constexpr int K_BYTES = SUBS * XA_SUB_M, T_BYTES = SUBS * XA_SUB_N;
  static constexpr int TILES = 2 * K_BYTES + STAGES * 2 * T_BYTES;
  static constexpr int STATS = STAGES * 2 * XA_BN * 4;
  static constexpr int SMEM = TILES + STATS + 1024 + 512;  // the stores go through the tiles of Q and dO
  static constexpr int COL_DV = 256, COL_DK = 256 + D;
};

// The n-th sequence of a packed batch of at most XA_SCAN by its queries, longest first: by one warp. CTAs start in that
// order, so that the long walks do not come last (8 sequences of 50 .. 2000 queries and 30 .. 600 keys, 16 heads of 128
// columns: 104 -> 98 us, 48 such: 666 -> 624, dQ included).
__device__ __forceinline__ int nth_longest(const XParams& p, int n, int lane) {
  int rows[2], rank[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 2; ++e) rows[e] = 32 * e + lane < p.batch ? make_seq(p, 32 * e + lane).lq : -1;
  for (int b = 0; b < p.batch; ++b) {
    const int x = __shfl_sync(0xffffffffu, b < 32 ? rows[0] : rows[1], b & 31);
#pragma unroll
    for (int e = 0; e < 2; ++e) rank[e] += x > rows[e] || (x == rows[e] && b < 32 * e + lane);
  }
  const unsigned lo = __ballot_sync(0xffffffffu, lane < p.batch && rank[0] == n);
  const unsigned hi = __ballot_sync(0xffffffffu, 32 + lane < p.batch && rank[1] == n);
  return lo ? __ffs(lo) - 1 : 31 + __ffs(hi);
}

template <int D, bool F16>
__global__ void __launch_bounds__(XB_THREADS, 1)
    cross_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                     const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const XParams p,
                     const XGrad gr, int ktiles, int splits) {
  using C = XDkv<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = smem + C::K_BYTES;
  auto sQ = [&](int s) { return smem + 2 * C::K_BYTES + 2 * s * C::T_BYTES; };
  auto sDO = [&](int s) { return smem + 2 * C::K_BYTES + (2 * s + 1) * C::T_BYTES; };
  float* stats = reinterpret_cast<float*>(smem + C::TILES);  // per stage: -lse * log2(e) [64], -delta [64]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::TILES + C::STATS);
  uint64_t* kv_full = bars;
  uint64_t* full = bars + 1;      // [STAGES] (33 arrivals: the tiles, and each lane's copies)
  uint64_t* empty = bars + 5;     // [STAGES]
  uint64_t* sdp_full = bars + 9;  // [2]
  uint64_t* ds_full = bars + 11;  // [2] XB_SOFTMAX arrivals
  uint64_t* done = bars + 13;
  constexpr int NBARS = 14;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + NBARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* seq_slot = reinterpret_cast<int*>(tmem_slot + 2);

  static_assert(2 * XB_SOFTMAX * XA_STAGE <= C::STAGES * 2 * C::T_BYTES, "room for the stores");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NBARS; ++i) mbar_init(&bars[i], (i == 11 || i == 12) ? XB_SOFTMAX : (i >= 1 && i < 5) ? 33 : 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmDO);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dep_wait();

  const int part = blockIdx.x % splits;
  const int kt = (blockIdx.x / splits) % ktiles;
  const int rest = blockIdx.x / splits / ktiles;
  const int hk = rest % p.kv_heads;
  int b = rest / p.kv_heads;
  if (p.cu_q && p.batch <= XA_SCAN) {
    if (warp == 0) {
      const int x = nth_longest(p, b, lane);
      if (lane == 0) *seq_slot = x;
    }
    __syncthreads();
    b = *seq_slot;
  }
  const XSeq s = make_seq(p, b);
  const int j0 = kt * XA_BM;
  const int qtiles = (s.lq + XA_BN - 1) / XA_BN;
  const long long steps_all = (long long)p.group * qtiles;
  const int t0 = (int)(steps_all * part / splits);
  const int t1 = j0 < s.seen ? (int)(steps_all * (part + 1) / splits) : t0;  // hidden keys get zeros
  const int T = j0 < s.lk ? t1 - t0 : 0;

  if (warp == 16) {
    if (T > 0) {
      if (lane == 0) {
        mbar_arrive_expect_tx(kv_full, 2 * C::K_BYTES);
        for (int c = 0; c < C::SUBS; ++c) {
          tma_load_2d(sK + c * XA_SUB_M, &tmK, kv_full, hk * D + 64 * c, s.ks + j0);
          tma_load_2d(sV + c * XA_SUB_M, &tmV, kv_full, hk * D + 64 * c, s.ks + j0);
        }
      }
      int t = 0, h = hk * p.group + t0 / qtiles, i0 = (t0 % qtiles) * XA_BN;
      const long long both = (long long)p.heads * p.total_q;  // from -lse * log2(e) to -delta of a row
      for (; t < T; ++t) {
        const int st = t % C::STAGES;
        if (t >= C::STAGES && !warp_bar_wait(&empty[st], ((t / C::STAGES) - 1) & 1, abort_flag, 140)) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[st], 2 * C::T_BYTES);
          for (int c = 0; c < C::SUBS; ++c) {
            tma_load_2d(sQ(st) + c * XA_SUB_N, &tmQ, &full[st], h * D + 64 * c, s.qs + i0);
            tma_load_2d(sDO(st) + c * XA_SUB_N, &tmDO, &full[st], h * D + 64 * c, s.qs + i0);
          }
        }
        // The row statistics travel with the tile, copied asynchronously: a load that the warp waited for, and divisions
        // for the tile's place, made its loop slower than the products. Rows behind the end get zeros: with their Q and
        // dO zeroed below, their probability is one and they add nothing.
        const float* src = gr.stats + (long long)h * p.total_q + s.qs + i0;
        const uint32_t dst = smem_u32(stats + st * 2 * XA_BN);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = lane + 32 * e;
          const bool on = i0 + i < s.lq;
          copy4(dst + 4 * i, on ? src + i : gr.stats, on);
          copy4(dst + 4 * (XA_BN + i), on ? src + both + i : gr.stats, on);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[st])) : "memory");
        i0 += XA_BN;
        if (i0 >= s.lq) {
          i0 = 0;
          ++h;
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (*abort_flag && lane == 0) {
        volatile int never = 0;
        bar_wait(kv_full, 0, &never, 141);
        for (int c = max(t - C::STAGES, 0); c < t; ++c) bar_wait(&full[c % C::STAGES], (c / C::STAGES) & 1, &never, 141);
      }
    }
  } else if (warp == 17) {
    // S^T = K Q^T and dP^T = V dO^T, dV += P^T dO and dK += dS^T Q. The scores of tile t + 2 are sent right behind the
    // products that read tile t's P and dS, which they overwrite: one thread's products run in order.
    const int fmt = F16 ? 0 : 1;
    const uint32_t tm = uniform_int(tmem), base = uniform_int(smem_u32(smem));
    const int n = uniform_int(T), first = uniform_int(t0), per = uniform_int(qtiles), lq = uniform_int(s.lq);
    const uint64_t dk = sdesc_kmajor_sw128(base), dm = sdesc_mnmajor_sw128(base + 2 * C::K_BYTES, XA_SUB_N);
    const uint32_t k_hi = (uint32_t)(dk >> 32), k_lo = (uint32_t)dk, v_lo = k_lo + (C::K_BYTES >> 4);
    const uint32_t m_hi = (uint32_t)(dm >> 32), m_lo = (uint32_t)dm;
    const uint32_t idesc_s = make_idesc(128, XA_BN, fmt, fmt, 0, 0), idesc_g = make_idesc(128, D, fmt, fmt, 0, 1);
    bool ok = n > 0 && warp_bar_wait(kv_full, 0, abort_flag, 142);
    int i0 = n > 0 ? (first % per) * XA_BN : 0;  // first row of the next scores' tile in its sequence
    auto ready = [&](int t) {
      const int st = t % C::STAGES;
      if (!warp_bar_wait(&full[st], (t / C::STAGES) & 1, abort_flag, 143)) return false;
      const int rows = lq - i0;
      if (rows < XA_BN) {
        // rows behind the end: whatever stands there must not enter the sums
        zero_rows(sQ(st), C::SUBS, XA_SUB_N, XA_BN, low_bits64(rows), lane);
        zero_rows(sDO(st), C::SUBS, XA_SUB_N, XA_BN, low_bits64(rows), lane);
      }
      i0 = rows > XA_BN ? i0 + XA_BN : 0;
      return true;
    };
    auto scores = [&](int t) {
      const int st = t % C::STAGES;
      const uint32_t qlo = k_lo + ((2 * C::K_BYTES + 2 * st * C::T_BYTES) >> 4), dlo = qlo + (C::T_BYTES >> 4);
      const uint32_t t_s = tm + 128 * (t & 1);
#pragma unroll
      for (int c = 0; c < C::SUBS; ++c)
        mma4_ss(t_s, k_lo + c * (XA_SUB_M >> 4), qlo + c * (XA_SUB_N >> 4), k_hi, idesc_s, c != 0);
#pragma unroll
      for (int c = 0; c < C::SUBS; ++c)
        mma4_ss(t_s + 64, v_lo + c * (XA_SUB_M >> 4), dlo + c * (XA_SUB_N >> 4), k_hi, idesc_s, c != 0);
      commit_elect(&sdp_full[t & 1]);
    };
    for (int t = 0; t < 2 && t < n && ok; ++t) {
      ok = ready(t);
      if (!ok) break;
      tc_fence_after();
      scores(t);
    }
    for (int t = 0; t < n && ok; ++t) {
      // D = 64: both waits lie before the products, while those of the last tile still run, since a wait takes a few
      // hundred cycles here even for a phase that is over (127 -> 110 us). At D = 128 a tile is twice the bytes and may
      // not be there yet: it is waited for behind this tile's products (214 against 225 us).
      ok = (D == 128 || t + 2 >= n || ready(t + 2)) && warp_bar_wait(&ds_full[t & 1], (t >> 1) & 1, abort_flag, 144);
      if (!ok) break;
      tc_fence_after();
      const int st = t % C::STAGES;
      const uint32_t qlo = m_lo + ((2 * st * C::T_BYTES) >> 4), dlo = qlo + (C::T_BYTES >> 4);
      const uint32_t t_s = tm + 128 * (t & 1);
      mma4_ts(tm + C::COL_DV, t_s, t_s + 32, dlo, m_hi, idesc_g, t > 0);
      mma4_ts(tm + C::COL_DK, t_s + 64, t_s + 96, qlo, m_hi, idesc_g, t > 0);
      commit_elect(&empty[st]);
      if (t + 2 < n) {
        if (D == 128) {
          ok = ready(t + 2);
          if (!ok) break;
          tc_fence_after();
        }
        scores(t + 2);
      }
    }
    commit_elect(done);
    volatile int never = 0;
    warp_bar_wait(done, 0, &never, 145);
  } else {
    const int grp = warp >> 3, half = (warp >> 2) & 1, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t t_s = tmem + lane_off + 128 * grp + 32 * half;
    const int j = j0 + r;
    const long long row = s.ks + j;
    bool vis = j < s.seen;
    if (vis && p.key_mask) vis = __ldg(p.key_mask + row) != 0;
    const bool some = __any_sync(0xffffffffu, vis);  // else the rows of this warp are not stored, or stored as zeros
    const uint64_t scale2 = f2(p.scale_log2, p.scale_log2);
    bool bad = false;
    for (int t = grp; t < T; t += 2) {
      const int st = t % C::STAGES;
      const float* sp = stats + st * 2 * XA_BN + 32 * half;
      if (!bar_wait(&full[st], (t / C::STAGES) & 1, abort_flag, 146)) bad = true;
      if (!bar_wait(&sdp_full[grp], (t >> 1) & 1, abort_flag, 147)) bad = true;
      tc_fence_after();
      if (some) {
        uint32_t sc[32], dp[32], wp[16], wd[16];
        tmem_ld32_async(t_s, sc);
        tmem_ld32_async(t_s + 64, dp);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 l4 = *reinterpret_cast<const float4*>(sp + e);
          const float4 d4 = *reinterpret_cast<const float4*>(sp + XA_BN + e);
#pragma unroll
          for (int f = 0; f < 4; f += 2) {
            const uint64_t nl = f ? f2(l4.z, l4.w) : f2(l4.x, l4.y), nd = f ? f2(d4.z, d4.w) : f2(d4.x, d4.y);
            const float2 x =
                f2_split(ffma2(f2(__uint_as_float(sc[e + f]), __uint_as_float(sc[e + f + 1])), scale2, nl));
            const float p0 = fast_exp2(x.x), p1 = fast_exp2(x.y);
            const float2 d = f2_split(
                fmul2(f2(p0, p1), fadd2(f2(__uint_as_float(dp[e + f]), __uint_as_float(dp[e + f + 1])), nd)));
            wp[(e + f) >> 1] = pack_2(p0, p1, F16);
            wd[(e + f) >> 1] = pack_2(d.x, d.y, F16);
          }
        }
        tmem_st16(t_s, wp);
        tmem_st16(t_s + 64, wd);
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ds_full[grp]);
    }
    // Warps 0..7 store dV, 8..15 dK, half of the columns each. The row of a hidden key has accumulated whatever its K
    // and V gave (rows of the products do not mix): it is stored as zeros.
    if (!bar_wait(done, 0, abort_flag, 148)) bad = true;
    tc_fence_after();
    const int rows = bad || *abort_flag ? 0 : s.lk - j0 - quarter * 32;  // of this warp that exist, if positive
    const uint32_t t_g = tmem + lane_off + (grp ? C::COL_DK : C::COL_DV) + half * (D / 2);
    const float f = grp ? p.scale : 1.f;
    if (splits == 1) {
      const long long ld = grp ? gr.lddk : gr.lddv;
      uint16_t* dst = reinterpret_cast<uint16_t*>(grp ? gr.dk : gr.dv) + (row - lane) * ld + hk * D + half * (D / 2);
      if (T > 0)
        store_rows16<D / 2, 16>(t_g, f, vis, F16, sQ(0) + warp * XA_STAGE, lane, rows, dst, ld);
      else if (lane < rows)
        zero_row16<D / 2>(dst + lane * ld);
    } else {
      const long long width = (long long)p.kv_heads * D;
      float* dst = gr.partial + ((long long)(part * 2 + grp) * p.total_k + row) * width + hk * D + half * (D / 2);
      if (T > 0)
        store_rows32<D / 2>(t_g, f, vis, lane < rows, dst);
      else if (lane < rows)
#pragma unroll
        for (int e = 0; e < D / 2; e += 4) *reinterpret_cast<float4*>(dst + e) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// dK and dV from the parts of the walk, in part order: grid (rows of a sequence x vectors, sequence).
__global__ void __launch_bounds__(256) cross_join_kernel(const XParams p, const XGrad gr, int splits, int width) {
  grid_dep_wait();
  const XSeq s = make_seq(p, blockIdx.y);
  const int vecs = width / 4;
  const long long n = (long long)s.lk * vecs;
  for (long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x; at < 2 * n;
       at += (long long)gridDim.x * blockDim.x) {
    const int w = at >= n;
    const long long i = at - w * n, row = s.ks + i / vecs, c = (i % vecs) * 4;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int sp = 0; sp < splits; ++sp) {
      const float4 v = *reinterpret_cast<const float4*>(gr.partial + ((long long)(sp * 2 + w) * p.total_k + row) * width + c);
      a.x += v.x;
      a.y += v.y;
      a.z += v.z;
      a.w += v.w;
    }
    uint16_t* dst = reinterpret_cast<uint16_t*>(w ? gr.dk : gr.dv) + row * (w ? gr.lddk : gr.lddv) + c;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_2(a.x, a.y, p.f16), pack_2(a.z, a.w, p.f16));
  }
}

// The forward's output from the parts of the keys: out = sum_s exp(lse_s - lse) out_s, lse = log sum_s exp(lse_s).
// WARPS warps take a row of a head: each reads every WARPS-th part, its loads in flight at once, and they join in shared
// memory. grid (rows of a sequence x heads, sequence).
template <int D, int WARPS>
__global__ void __launch_bounds__(256) cross_merge_kernel(const XParams p) {
  constexpr int ROWS = 8 / WARPS, E = D / 32;
  using V = typename std::conditional<E == 2, float2, float4>::type;
  __shared__ float sh[8][D];
  __shared__ float sh_l[8];
  grid_dep_wait();
  const XSeq s = make_seq(p, blockIdx.y);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % WARPS;
  const long long n = (long long)s.lq * p.heads, one = (long long)p.heads * p.total_q;
  for (long long first = (long long)blockIdx.x * ROWS; first < n; first += (long long)gridDim.x * ROWS) {
    const long long at = first + warp / WARPS;
    const bool on = at < n;
    const int h = on ? (int)(at % p.heads) : 0;
    const long long row = s.qs + (on ? at / p.heads : 0), src = (long long)h * p.total_q + row;
    float top = -INFINITY;
    if (on)
      for (int sp = lane; sp < p.parts; sp += 32) top = fmaxf(top, p.part_lse[sp * one + src]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    float a[E], l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) a[e] = 0.f;
    if (on) {
#pragma unroll 4
      for (int sp = sub; sp < p.parts; sp += WARPS) {
        // a part of weight zero may hold anything
        const float e = p.part_lse[sp * one + src];
        const float f = e == -INFINITY ? 0.f : fast_exp2((e - top) * XA_LOG2E);
        const V v = *reinterpret_cast<const V*>(p.part_o + (sp * one + src) * D + E * lane);
        const float* o = reinterpret_cast<const float*>(&v);
        l += f;
#pragma unroll
        for (int x = 0; x < E; ++x) a[x] = fmaf(f, f != 0.f ? o[x] : 0.f, a[x]);
      }
    }
    if (WARPS > 1) {
#pragma unroll
      for (int x = 0; x < E; ++x) sh[warp][E * lane + x] = a[x];
      if (lane == 0) sh_l[warp] = l;
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int w = 1; w < WARPS; ++w) {
#pragma unroll
          for (int x = 0; x < E; ++x) a[x] += sh[warp + w][E * lane + x];
          l += sh_l[warp + w];
        }
      }
    }
    if (on && sub == 0) {
      const float inv = l > 0.f ? 1.f / l : 0.f;
      uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(p.out) + row * p.ldo + h * D + E * lane);
#pragma unroll
      for (int x = 0; x < E; x += 2) dst[x / 2] = pack_2(a[x] * inv, a[x + 1] * inv, p.f16);
      if (lane == 0 && p.lse) p.lse[src] = l > 0.f ? top + __log2f(l) * 0.6931471805599453f : -INFINITY;
    }
    if (WARPS > 1) __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ host
// Parts of the dK / dV walk: the number that ends soonest, in tiles of 1.2 us (D = 128) or 0.8. A part's set-up and
// epilogue cost about 12 tiles, the joining launch 8 and its bytes (`bytes` a part, written and read) at 3 TB/s. One part
// writes its result at once. (The device alone would have it at 4 tiles: 3 x 77 queries x 33 keys, 8 heads on 2, take 18.1
// us with one part and 14.7 with four; but such calls wait for the host, for which the launch is 1.3 us more.)
static double join_tiles(long long bytes, int head_dim) { return bytes / 3e6 / (head_dim == 128 ? 1.2 : 0.8); }
// Uniform batches: every wave of CTAs costs its longest walk. Backward in all with 1, 2, 4, 8 parts: 24 heads of 64, 2 x
// 8247 queries x 128 keys 167, 129, 139, 141 us and 115 with 3; x 257 keys 206, 225, 242, 269; 8 heads on one of 128, 700
// queries x 64 keys 94, 57, 37, 27 and 23 with 32.
static int dkv_splits(long long ctas, long long tiles, long long bytes, int head_dim, int sms) {
  const double join = join_tiles(bytes, head_dim);
  long long best = 1;
  double cost = -1.;
  for (long long n = 1; n <= 32 && n <= tiles; ++n) {
    const long long waves = (ctas * n + sms - 1) / sms;
    const double c = (double)waves * ((tiles + n - 1) / n + 12) + (n > 1 ? 8. + n * join : 0.);
    if (cost < 0. || c < cost) {
      cost = c;
      best = n;
    }
  }
  return (int)best;
}
// Packed batches: the lengths are on the device, the totals are not. The SMs share the work of all CTAs, which start with
// the longest walk, and the end is ragged by a quarter of one; no walk can be shorter than the longest. Backward in all of
// 4 sequences of 1255 .. 2500 queries and 528 .. 2111 keys, 16 heads of 128 columns, with 1, 2, 3, 4 parts: 329, 357, 365,
// 374 us; 8 of 50 .. 2000 and 30 .. 600: 132, 98, 107, 111; 2 such: 144, 94, 75, 65, and 52 with 8.
static int dkv_splits_packed(long long ctas, long long tiles_mean, long long tiles_most, long long bytes, int head_dim,
                             int sms) {
  long long best = 1;
  double cost = -1.;
  const double join = join_tiles(bytes, head_dim);
  for (long long n = 1; n <= 32 && n <= tiles_most; ++n) {
    const double all = (double)ctas * (tiles_mean + 12. * n) / sms + tiles_most / (4. * n), walk = tiles_most / (double)n + 12.;
    const double c = (all > walk ? all : walk) + (n > 1 ? 8. + n * join : 0.);
    if (cost < 0. || c < cost) {
      cost = c;
      best = n;
    }
  }
  return (int)best;
}

static int check_common(const void* q, const void* k, const void* v, const void* out, const int* cu_q, const int* cu_k,
                        int batch, int max_q, int max_k, int total_q, int total_k, int heads, int kv_heads, int head_dim,
                        long long ldq, long long ldk, long long ldv, long long ldo, float scale, int dtype) {
  if (batch < 0 || max_q < 0 || max_k < 0 || total_q < 0 || total_k < 0 || heads <= 0 || kv_heads <= 0 ||
      heads % kv_heads != 0)
    return SA3_ERR_ARG;
  if (!(scale > 0.f) || !(scale * XA_LOG2E <= 3.4e38f)) return SA3_ERR_ARG;  // NaN and infinity fail both
  if (head_dim != 64 && head_dim != 128) return SA3_ERR_UNSUPPORTED;
  if (dtype != SA3_DT_BF16 && dtype != SA3_DT_F16) return SA3_ERR_DTYPE;
  if (!cu_q && (long long)batch * max_q != total_q) return SA3_ERR_ARG;
  if (!cu_k && (long long)batch * max_k != total_k) return SA3_ERR_ARG;
  const long long wq = (long long)heads * head_dim, wk = (long long)kv_heads * head_dim;
  if (ldq < wq || ldo < wq || ldk < wk || ldv < wk) return SA3_ERR_ARG;
  if (total_q > 0 && (!q || !out)) return SA3_ERR_ARG;
  if (total_k > 0 && (!k || !v)) return SA3_ERR_ARG;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || ((ldq | ldk | ldv | ldo) & 7))
    return SA3_ERR_ALIGN;
  if ((reinterpret_cast<uintptr_t>(cu_q) | reinterpret_cast<uintptr_t>(cu_k)) & 3) return SA3_ERR_ALIGN;
  // grid and item counts stay in 32 bits
  const long long items = ((long long)max_q / XA_BM + 1) * heads * (batch > 0 ? batch : 1);
  const long long kitems = ((long long)max_k / XA_BM + 1) * kv_heads * (batch > 0 ? batch : 1);
  if (heads > 65535 || batch > 65535 || items > (1LL << 30) || kitems > (1LL << 25)) return SA3_ERR_UNSUPPORTED;
  return SA3_OK;
}

static XParams make_params(void* out, float* lse, const int* cu_q, const int* cu_k, const int* k_lens,
                           const unsigned char* key_mask, int batch, int max_q, int max_k, int total_q, int total_k,
                           int heads, int kv_heads, long long ldo, float scale, int dtype) {
  XParams p = {};
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.k_lens = k_lens;
  p.key_mask = key_mask;
  p.batch = batch;
  p.Lq = max_q;
  p.Lk = max_k;
  p.total_q = total_q;
  p.total_k = total_k;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = heads / kv_heads;
  p.scale = scale;
  p.scale_log2 = scale * XA_LOG2E;
  p.f16 = dtype == SA3_DT_F16;
  p.out = out;
  p.ldo = ldo;
  p.lse = lse;
  p.parts = 1;
  return p;
}

// Tensor map of a token-row buffer with boxes of 64 columns x `box` rows. A buffer without rows is never read:
// its map is taken over `other`.
static int token_map(CUtensorMap* m, const void* x, const void* other, int f16, long long width, long long rows,
                     long long ld, int box) {
  const auto dt = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return make_tmap_2d(m, rows > 0 ? x : other, dt, 2, width, rows > 0 ? rows : 1, ld, 64, box);
}

static bool scans(const XParams& p) { return p.cu_q && p.batch <= XA_SCAN; }

// Grid of the joining kernels: enough blocks of 256 threads for `n` elements of a sequence, about 8 an SM in all.
static dim3 rows_grid(long long n, int batch, int sms) {
  const long long need = (n + 255) / 256, most = (8LL * sms + batch - 1) / batch;
  return dim3((unsigned)(need < most ? need : most), (unsigned)batch);
}

template <int D, bool F16>
static int launch_fwd(const XParams& p, const void* q, const void* k, const void* v, long long ldq, long long ldk,
                      long long ldv, int sms, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  int rc;
  const long long wq = (long long)p.heads * D, wk = (long long)p.kv_heads * D;
  if ((rc = token_map(&mq, q, q, p.f16, wq, p.total_q, ldq, XA_BM))) return rc;
  using C = XFwd<D>;
  if ((rc = token_map(&mk, k, q, p.f16, wk, p.total_k, ldk, C::BN))) return rc;
  if ((rc = token_map(&mv, v, q, p.f16, wk, p.total_k, ldv, C::BN))) return rc;
  const int qtiles = (p.Lq + C::UNITS * XA_BM - 1) / (C::UNITS * XA_BM);
  const int items = qtiles * p.heads * p.batch * p.parts;
  auto kern = scans(p) ? cross_fwd_kernel<D, F16, true> : cross_fwd_kernel<D, F16, false>;
  if ((rc = ensure_smem(kern, C::SMEM))) return rc;
  launch_ex(kern, dim3(items < 2 * sms ? items : 2 * sms), dim3(C::THREADS), C::SMEM, st, 1, mq,
            mk, mv, p, items, qtiles);
  return launch_status();
}

template <int D, bool F16>
static int launch_bwd(const XParams& p, const XGrad& g, const void* q, const void* k, const void* v, long long ldq,
                      long long ldk, long long ldv, int splits, int sms, cudaStream_t st) {
  CUtensorMap q128, do128, o128, q64, do64, k64, v64, k128, v128;
  int rc;
  const long long wq = (long long)p.heads * D, wk = (long long)p.kv_heads * D;
  const void* any = p.total_q > 0 ? q : k;
  if ((rc = token_map(&q128, q, any, p.f16, wq, p.total_q, ldq, XA_BM))) return rc;
  if ((rc = token_map(&q64, q, any, p.f16, wq, p.total_q, ldq, XA_BN))) return rc;
  if ((rc = token_map(&do128, g.dout, any, p.f16, wq, p.total_q, g.lddo, XA_BM))) return rc;
  if ((rc = token_map(&o128, p.out, any, p.f16, wq, p.total_q, p.ldo, XA_BM))) return rc;
  if ((rc = token_map(&do64, g.dout, any, p.f16, wq, p.total_q, g.lddo, XA_BN))) return rc;
  if ((rc = token_map(&k64, k, any, p.f16, wk, p.total_k, ldk, XA_BN))) return rc;
  if ((rc = token_map(&v64, v, any, p.f16, wk, p.total_k, ldv, XA_BN))) return rc;
  if ((rc = token_map(&k128, k, any, p.f16, wk, p.total_k, ldk, XA_BM))) return rc;
  if ((rc = token_map(&v128, v, any, p.f16, wk, p.total_k, ldv, XA_BM))) return rc;
  if (p.total_q > 0 && p.Lq > 0) {
    const int qtiles = (p.Lq + XA_BM - 1) / XA_BM;
    const int items = qtiles * p.heads * p.batch;
    auto kern = scans(p) ? cross_dq_kernel<D, F16, true> : cross_dq_kernel<D, F16, false>;
    if ((rc = ensure_smem(kern, XDq<D>::SMEM))) return rc;
    launch_ex(kern, dim3(items < 2 * sms ? items : 2 * sms), dim3(XA_THREADS), XDq<D>::SMEM, st, 1, q128,
              do128, o128, k64, v64, p, g, items, qtiles);
    if ((rc = launch_status())) return rc;
  }
  if (p.total_k > 0 && p.Lk > 0) {
    const int ktiles = (p.Lk + XA_BM - 1) / XA_BM;
    if ((rc = ensure_smem(cross_dkv_kernel<D, F16>, XDkv<D>::SMEM))) return rc;
    launch_ex(cross_dkv_kernel<D, F16>, dim3((unsigned)(ktiles * p.kv_heads * p.batch * splits)), dim3(XB_THREADS),
              XDkv<D>::SMEM, st, 1, q64, do64, k128, v128, p, g, ktiles, splits);
    if ((rc = launch_status())) return rc;
    if (splits > 1) {
      launch_ex(cross_join_kernel, rows_grid(2LL * p.Lk * p.kv_heads * D / 4, p.batch, sms), dim3(256), 0, st, 1, p, g,
                splits, p.kv_heads * D);
      if ((rc = launch_status())) return rc;
    }
  }
  return SA3_OK;
}

// the parts' lse first, their outputs behind it at a 16-byte boundary
static long long fwd_bytes(int parts, int heads, int total_q, int head_dim) {
  const long long rows = (long long)parts * heads * total_q;
  return 4 * (((rows + 3) & ~3LL) + rows * head_dim);
}

// the row statistics first, the parts of dK and dV behind them at a 16-byte boundary
static long long stats_bytes(int heads, int total_q) { return (((long long)heads * total_q * 8) + 15) & ~15LL; }

// Parts of the keys in the forward (one CTA each, joined by a second launch) while the query tiles alone leave CTA slots
// empty: the number that ends soonest by these measured times. A step of 64 keys takes 1.3 us (D = 64; 1.6 with both
// units at work) or 0.9 us (D = 128) alone on an SM, 1.45 / 2.8 / 1.4 us with two CTAs there, an item 2 us besides;
// the joining launch 3 us, 0.1 us a part, and its bytes at 3 TB/s. 8 heads of 64 columns, 64 queries, 8192 keys: 168,
// 89, 49, 29, 20, 19 us with 1, 2, 4, .. 32 parts; 148 heads of 128 columns, 128 queries: 137, 114, 127 with 1, 2, 4.
static int fwd_parts(int batch, int max_q, int max_k, int heads, int kv_heads, int head_dim, int sms) {
  if (batch <= 0 || max_q <= 0) return 1;
  if ((long long)max_q * (heads / kv_heads) <= XT_MAX_ROWS) return cross_token_parts(batch, kv_heads, max_k, sms);
  const bool narrow = head_dim == 64, pair = narrow && max_q > XA_BM;
  const int rows = pair ? 2 * XA_BM : XA_BM;
  const long long items = (long long)((max_q + rows - 1) / rows) * heads * batch, fill = 2LL * sms / items;
  const int tiles = (max_k + XA_BN - 1) / XA_BN;
  const float alone = narrow ? pair ? 1.6f : 1.3f : 0.9f, both = narrow ? pair ? 2.8f : 1.45f : 1.4f;
  const float join = (float)heads * batch * max_q * head_dim * 8e-6f / 3.f;
  int best = 1;
  float cost = 0.f;
  for (int n = 1; n <= fill && n <= 64 && (n == 1 || 2 * n <= tiles); ++n) {
    const float c = (tiles + n - 1) / n * (items * n > sms ? both : alone) + 2.f + (n > 1 ? 3.f + n * (0.1f + join) : 0.f);
    if (n == 1 || c < cost) {
      cost = c;
      best = n;
    }
  }
  return best;
}

static int bwd_splits(int batch, int max_q, int max_k, int total_q, int total_k, int heads, int kv_heads, int head_dim,
                      int sms) {
  if (batch <= 0) return 1;
  const long long most = (long long)(heads / kv_heads) * ((max_q + XA_BN - 1) / XA_BN);
  const long long ctas = (long long)((max_k + XA_BM - 1) / XA_BM) * kv_heads * batch;
  if (ctas <= 0 || most <= 0) return 1;
  const long long bytes = 16LL * total_k * kv_heads * head_dim;
  if ((long long)batch * max_q == total_q && (long long)batch * max_k == total_k)
    return dkv_splits(ctas, most, bytes, head_dim, sms);
  const long long some = (total_k / XA_BM + batch) * kv_heads;
  const long long mean = (long long)(heads / kv_heads) * (total_q / XA_BN / batch + 1);
  return dkv_splits_packed(some < ctas ? some : ctas, mean < most ? mean : most, most, bytes, head_dim, sms);
}

}  // namespace sa3

using namespace sa3;

extern "C" int sa3_cross_attention(const void* q, const void* k, const void* v, void* out, float* lse,
                                   const int* cu_seqlens_q, const int* cu_seqlens_k, const int* k_lens,
                                   const unsigned char* key_mask, int batch, int max_seqlen_q, int max_seqlen_k,
                                   int total_q, int total_k, int heads, int kv_heads, int head_dim, long long ldq,
                                   long long ldk, long long ldv, long long ldo, float softmax_scale, int dtype,
                                   void* workspace, long long workspace_bytes, void* stream) {
  int rc = check_common(q, k, v, out, cu_seqlens_q, cu_seqlens_k, batch, max_seqlen_q, max_seqlen_k, total_q, total_k,
                        heads, kv_heads, head_dim, ldq, ldk, ldv, ldo, softmax_scale, dtype);
  if (rc) return rc;
  if ((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(k_lens)) & 3) return SA3_ERR_ALIGN;
  if (batch == 0 || total_q == 0 || max_seqlen_q == 0) return SA3_OK;
  if (out == q || (total_k > 0 && (out == k || out == v))) return SA3_ERR_ARG;
  const int sms = sm_count();
  if (sms <= 0) return SA3_ERR_LAUNCH;
  XParams p = make_params(out, lse, cu_seqlens_q, cu_seqlens_k, k_lens, key_mask, batch, max_seqlen_q, max_seqlen_k,
                          total_q, total_k, heads, kv_heads, ldo, softmax_scale, dtype);
  p.parts = fwd_parts(batch, max_seqlen_q, max_seqlen_k, heads, kv_heads, head_dim, sms);
  if (p.parts > 1) {
    if (!workspace || workspace_bytes < fwd_bytes(p.parts, heads, total_q, head_dim)) return SA3_ERR_ARG;
    if (!aligned16(workspace)) return SA3_ERR_ALIGN;
    p.part_lse = static_cast<float*>(workspace);
    p.part_o = p.part_lse + (((long long)p.parts * heads * total_q + 3) & ~3LL);
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if ((long long)max_seqlen_q * p.group <= XT_MAX_ROWS)
    rc = cross_token(p, q, k, v, ldq, ldk, ldv, head_dim, sms, st);
  else
    rc = (head_dim == 64 ? p.f16 ? launch_fwd<64, true> : launch_fwd<64, false>
                         : p.f16 ? launch_fwd<128, true> : launch_fwd<128, false>)(p, q, k, v, ldq, ldk, ldv, sms, st);
  if (rc || p.parts == 1) return rc;
  // 8 warps a row where there are many parts and no more rows than blocks that run at once (32 parts of 136 rows: 52.4
  // against 55.5 us with one warp, in all); else a warp a row (8 parts of 8192 rows: 51.6 against 81.3 us).
  const long long all_rows = (long long)max_seqlen_q * heads * batch;
  const bool few = p.parts <= 16 || all_rows > 8LL * sms;
  const dim3 grid = rows_grid((long long)max_seqlen_q * heads * (few ? 32 : 256), batch, sms);
  launch_ex(head_dim == 64 ? few ? cross_merge_kernel<64, 1> : cross_merge_kernel<64, 8>
                           : few ? cross_merge_kernel<128, 1> : cross_merge_kernel<128, 8>,
            grid, dim3(256), 0, st, 1, p);
  return launch_status();
}

extern "C" int sa3_cross_attention_workspace(int batch, int max_seqlen_q, int max_seqlen_k, int total_q, int heads,
                                             int kv_heads, int head_dim, long long* bytes) {
  if (!bytes || batch < 0 || max_seqlen_q < 0 || max_seqlen_k < 0 || total_q < 0 || heads <= 0 || kv_heads <= 0 ||
      heads % kv_heads != 0)
    return SA3_ERR_ARG;
  if (head_dim != 64 && head_dim != 128) return SA3_ERR_UNSUPPORTED;
  const int sms = sm_count();
  if (sms <= 0) return SA3_ERR_LAUNCH;
  const int n = fwd_parts(batch, max_seqlen_q, max_seqlen_k, heads, kv_heads, head_dim, sms);
  *bytes = n > 1 ? fwd_bytes(n, heads, total_q, head_dim) : 0;
  return SA3_OK;
}

extern "C" int sa3_cross_attention_bwd_workspace(int batch, int max_seqlen_q, int max_seqlen_k, int total_q, int total_k,
                                                 int heads, int kv_heads, int head_dim, long long* bytes) {
  if (!bytes || batch < 0 || max_seqlen_q < 0 || max_seqlen_k < 0 || total_q < 0 || total_k < 0 || heads <= 0 ||
      kv_heads <= 0 || heads % kv_heads != 0)
    return SA3_ERR_ARG;
  if (head_dim != 64 && head_dim != 128) return SA3_ERR_UNSUPPORTED;
  const int sms = sm_count();
  if (sms <= 0) return SA3_ERR_LAUNCH;
  const int n = bwd_splits(batch, max_seqlen_q, max_seqlen_k, total_q, total_k, heads, kv_heads, head_dim, sms);
  *bytes = stats_bytes(heads, total_q) + (n > 1 ? 8LL * n * total_k * kv_heads * head_dim : 0);
  return SA3_OK;
}

extern "C" int sa3_cross_attention_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out,
                                       const float* lse, void* dq, void* dk, void* dv, const int* cu_seqlens_q,
                                       const int* cu_seqlens_k, const int* k_lens, const unsigned char* key_mask,
                                       int batch, int max_seqlen_q, int max_seqlen_k, int total_q, int total_k, int heads,
                                       int kv_heads, int head_dim, long long lddo, long long ldq, long long ldk,
                                       long long ldv, long long ldo, long long lddq, long long lddk, long long lddv,
                                       float softmax_scale, int dtype, void* workspace, long long workspace_bytes,
                                       void* stream) {
  int rc = check_common(q, k, v, out, cu_seqlens_q, cu_seqlens_k, batch, max_seqlen_q, max_seqlen_k, total_q, total_k,
                        heads, kv_heads, head_dim, ldq, ldk, ldv, ldo, softmax_scale, dtype);
  if (rc) return rc;
  const long long wq = (long long)heads * head_dim, wk = (long long)kv_heads * head_dim;
  if (lddo < wq || lddq < wq || lddk < wk || lddv < wk) return SA3_ERR_ARG;
  if (total_q > 0 && (!dout || !dq || !lse)) return SA3_ERR_ARG;
  if (total_k > 0 && (!dk || !dv)) return SA3_ERR_ARG;
  if (!aligned16(dout) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) || !aligned16(workspace) ||
      ((lddo | lddq | lddk | lddv) & 7))
    return SA3_ERR_ALIGN;
  if ((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(k_lens)) & 3) return SA3_ERR_ALIGN;
  if (batch == 0 || (total_q == 0 && total_k == 0)) return SA3_OK;
  // the dK / dV kernel reads q and dout after dq is written
  const void* rows_q[] = {dout, q, out, dq};
  const void* rows_k[] = {k, v, dk, dv};
  for (const void* y : {(const void*)dq, (const void*)dk, (const void*)dv}) {
    int same = 0;
    for (int i = 0; i < 4; ++i) same += (total_q > 0 && rows_q[i] == y) + (total_k > 0 && rows_k[i] == y);
    if (same > 1) return SA3_ERR_ARG;
  }
  const int sms = sm_count();
  if (sms <= 0) return SA3_ERR_LAUNCH;
  const int splits = bwd_splits(batch, max_seqlen_q, max_seqlen_k, total_q, total_k, heads, kv_heads, head_dim, sms);
  const long long at = stats_bytes(heads, total_q);
  const long long need = at + (splits > 1 ? 8LL * splits * total_k * kv_heads * head_dim : 0);
  if (workspace_bytes < need || (need > 0 && !workspace)) return SA3_ERR_ARG;
  const XParams p = make_params(const_cast<void*>(out), const_cast<float*>(lse), cu_seqlens_q, cu_seqlens_k, k_lens,
                                key_mask, batch, max_seqlen_q, max_seqlen_k, total_q, total_k, heads, kv_heads, ldo,
                                softmax_scale, dtype);
  XGrad g = {};
  g.dout = dout;
  g.lddo = lddo;
  g.dq = dq;
  g.lddq = lddq;
  g.dk = dk;
  g.lddk = lddk;
  g.dv = dv;
  g.lddv = lddv;
  g.stats = static_cast<float*>(workspace);
  g.partial = splits > 1 ? reinterpret_cast<float*>(static_cast<char*>(workspace) + at) : nullptr;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return (head_dim == 64 ? p.f16 ? launch_bwd<64, true> : launch_bwd<64, false>
                         : p.f16 ? launch_bwd<128, true> : launch_bwd<128, false>)(p, g, q, k, v, ldq, ldk, ldv,
                                                                                   splits, sms, st);
}
