// Attention of a few query rows (one decoded token of every sequence, times the query heads that share a key head)
// to an encoder's states: out = softmax(scale * q K^T) V over the visible keys.
//
// Bound by reading K and V once. All query rows of a key head (at most 16: query tokens x heads of the group) are the
// N side of warp matrix instructions m16n8k16, so K and V of the head are read once for the whole group and no row of
// the instruction is wasted up to 8 (tcgen05 would leave 112 of its 128 rows empty):
//   S^T (16 keys x rows) = K Q^T          A = K by ldmatrix, B = Q^T, kept in registers
//   O^T (16 columns x rows) += V^T P^T    A = V^T by ldmatrix.trans, B = P^T: the S^T fragment, transposed by movmatrix
// The keys are split over the warps of a cluster of CTAs, 16 keys a step. Each warp copies its steps asynchronously
// into a ring of its own in shared memory (16-byte chunk c of key j at chunk c ^ (j & 7): no bank conflicts on either
// side), several steps ahead, so the bytes in flight take no registers and no warp waits for another: 5.6 TB/s for 64
// sequences of 375 .. 1500 keys, 8 key heads of 128 columns (45 us). Hidden keys are
// not read: their rows are filled with zeros and their scores are -inf.
// The reference maximum of a row moves only when a score exceeds it by more than 2^8; one vote a step finds out, and
// the usual step has no reduction over lanes. The warps of a CTA join through shared memory and the CTAs of the
// cluster through distributed shared memory, in a fixed order: one launch, no workspace.
#include <cooperative_groups.h>

#include "attn_tile.cuh"
#include "common.cuh"
#include "cross_attention.cuh"
#include "host_util.h"

namespace sa3 {
namespace cg = cooperative_groups;

constexpr int XT_WARPS = 4;
constexpr int XT_THREADS = XT_WARPS * 32;
constexpr int XT_KEYS = 16;          // keys of a step of a warp
constexpr int XT_MAX_CLUSTER = 8;
constexpr int XT_PART_KEYS = 256;    // least keys of a part of the split without clusters: 4 steps of a warp
constexpr int XT_MAX_PARTS = 128;
constexpr int XT_MAX_ORDER = 64;     // sequences that are ordered: two a lane
constexpr int XT_ORDER_KEYS = 1280;  // longest keys from which that is worth it
constexpr int XT_SPLIT_KEYS = 8192;  // keys from which that split is worth its second launch
constexpr float XT_RESCALE_LOG2 = 8.f;
// Steps in flight: 96 KB a CTA at either width, two CTAs an SM.
template <int D>
constexpr int XT_STAGES = D == 64 ? 6 : 3;

struct XTokenParams {
  XParams p;
  const void *q, *k, *v;
  long long ldq, ldk, ldv;
};

template <bool F16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// 16 bytes from global to shared memory, or zeros
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}

// The n-th of at most XT_MAX_ORDER sequences by its visible keys, most first; every warp finds it by itself.
__device__ __forceinline__ int nth_most_keys(const XParams& p, int n, int lane) {
  int keys[2], rank[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 2; ++e) keys[e] = make_seq(p, min(32 * e + lane, p.batch - 1)).seen;
  if (__reduce_max_sync(0xffffffffu, max(keys[0], keys[1])) == __reduce_min_sync(0xffffffffu, min(keys[0], keys[1])))
    return n;
#pragma unroll 8
  for (int b = 0; b < p.batch; ++b) {
    const int x = __shfl_sync(0xffffffffu, b < 32 ? keys[0] : keys[1], b & 31);
#pragma unroll
    for (int e = 0; e < 2; ++e) rank[e] += x > keys[e] || (x == keys[e] && b < 32 * e + lane);
  }
  const unsigned lo = __ballot_sync(0xffffffffu, lane < p.batch && rank[0] == n);
  const unsigned hi = __ballot_sync(0xffffffffu, 32 + lane < p.batch && rank[1] == n);
  return lo ? __ffs(lo) - 1 : 31 + __ffs(hi);
}

// NT: tiles of 8 query rows (1 or 2).
template <int D, bool F16, int NT>
__global__ void __launch_bounds__(XT_THREADS, 2) cross_token_kernel(const XTokenParams a, int csize, bool ordered) {
  constexpr int ROWS = 8 * NT;
  constexpr int CH = D / 8;                 // 16-byte chunks of a key
  constexpr int KPI = 32 / CH;              // keys that one copy instruction of a warp covers
  constexpr int ST = XT_STAGES<D>, HALF = XT_KEYS * D * 2, STEP = 2 * HALF;  // K, then V, of a step
  // the warps' rings; afterwards [warps][ROWS][D] partial outputs and their [warps][ROWS] maxima and sums
  extern __shared__ __align__(128) float sh[];
  float* sh_m = sh + XT_WARPS * ROWS * D;
  float* sh_l = sh_m + XT_WARPS * ROWS;
  const XParams& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % csize, part = blockIdx.x / csize % p.parts, unit = blockIdx.x / csize / p.parts;
  const int hk = unit % p.kv_heads;
  int b = unit / p.kv_heads;
  grid_dep_wait();
  if (ordered) b = nth_most_keys(p, b, lane);
  const XSeq sq = make_seq(p, b);
  const int qs = sq.qs, lq = sq.lq, ks = sq.ks, seen = sq.seen;
  const int rows = lq * p.group;  // row m: token m / group, head hk * group + m % group

  const int first = ((part * csize + rank) * XT_WARPS + warp) * XT_KEYS, stride = p.parts * csize * XT_WARPS * XT_KEYS;
  const int steps = first < seen ? (seen - first - 1) / stride + 1 : 0;
  const uint32_t ring = smem_u32(sh) + warp * ST * STEP;
  // copies: lane -> key lane / CH of a group of KPI keys, chunk lane % CH
  const int ck = lane / CH, cc = lane % CH;
  const long long row0 = (long long)ks + first + ck;
  const uint16_t* kp = reinterpret_cast<const uint16_t*>(a.k) + row0 * a.ldk + hk * D + 8 * cc;
  const uint16_t* vp = reinterpret_cast<const uint16_t*>(a.v) + row0 * a.ldv + hk * D + 8 * cc;
  const long long k_step = (long long)stride * a.ldk, v_step = (long long)stride * a.ldv;
  // issue the copies of step c, at which kp and vp stand, into its slot; the mask of its visible keys
  auto fetch = [&](int c) -> uint32_t {
    uint32_t vis = 0;
    if (c < steps) {
      const int j0 = first + c * stride;
      vis = seen - j0 >= XT_KEYS ? 0xffffu : (1u << (seen - j0)) - 1u;
      if (p.key_mask) {
        const bool on = lane < XT_KEYS && ((vis >> lane) & 1u) && __ldg(p.key_mask + (long long)ks + j0 + lane) != 0;
        vis = __ballot_sync(0xffffffffu, on);
      }
      const uint32_t slot = ring + (c % ST) * STEP;
#pragma unroll
      for (int i = 0; i < XT_KEYS / KPI; ++i) {
        const int j = i * KPI + ck;
        const bool on = (vis >> j) & 1u;
        const uint32_t dst = slot + j * (D * 2) + ((cc ^ (j & 7)) << 4);
        // a hidden key's address is not formed: it may lie behind the buffer
        copy16(dst, on ? kp + i * KPI * a.ldk : a.k, on);
        copy16(dst + HALF, on ? vp + i * KPI * a.ldv : a.v, on);
      }
      kp += k_step;
      vp += v_step;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    return vis;
  };
  uint32_t ahead[ST];
#pragma unroll
  for (int c = 0; c < ST; ++c) ahead[c] = fetch(c);

  // B fragments of Q^T: columns 16 i + 2 t, + 1 (first), + 8 (second) of row 8 n + g
  uint32_t qf[NT][D / 16][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int m = 8 * n + g;
    const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) +
                          (m < rows ? (long long)(qs + m / p.group) * a.ldq + (hk * p.group + m % p.group) * D : 0);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      qf[n][i][0] = m < rows ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * i + 2 * t)) : 0u;
      qf[n][i][1] = m < rows ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * i + 2 * t + 8)) : 0u;
    }
  }
  // O^T tiles: (column 16 i + g, rows 8 n + 2t and + 1), (column + 8, the same)
  float o[NT][D / 16][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
  float mr[NT][2], lr[NT][2];  // rows 8 n + 2t, + 1: reference maximum (uniform over g) and this lane's part of the sum
#pragma unroll
  for (int n = 0; n < NT; ++n) mr[n][0] = mr[n][1] = -INFINITY, lr[n][0] = lr[n][1] = 0.f;

  // ldmatrix: lane l gives the row address of matrix l / 8. K: keys (l & 15), chunk 2 i + (l >> 4).
  // V^T: keys (l & 7) + 8 * (l >> 4), chunk 2 i + ((l >> 3) & 1).
  const int kj = lane & 15, kc = lane >> 4, vj = (lane & 7) + 8 * (lane >> 4), vc = (lane >> 3) & 1;
  for (int step = 0; step < steps; ++step) {
    const uint32_t vis = ahead[0];
    asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
    __syncwarp();
    const uint32_t slot = ring + (step % ST) * STEP;
    float s[NT][2][4];  // two chains of the sum over a head's columns
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][0][e] = s[n][1][e] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      uint32_t ka[4];
      ldmatrix4(ka, slot + kj * (D * 2) + (((2 * i + kc) ^ (kj & 7)) << 4));
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_16816<F16>(s[n][i & 1], ka, qf[n][i][0], qf[n][i][1]);
    }
    // lane (g, t): keys g and g + 8 of rows 8 n + 2 t, + 1
    const bool on0 = (vis >> g) & 1u, on1 = (vis >> (g + 8)) & 1u;
    bool move = false;
    float x[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[n][e] = (e < 2 ? on0 : on1) ? (s[n][0][e] + s[n][1][e]) * p.scale_log2 : -INFINITY;
      move = move || fmaxf(x[n][0], x[n][2]) > mr[n][0] + XT_RESCALE_LOG2 ||
             fmaxf(x[n][1], x[n][3]) > mr[n][1] + XT_RESCALE_LOG2;
    }
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(x[n][e], x[n][e + 2]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float top = fmaxf(mr[n][e], mx);
          const float f = top > mr[n][e] ? fast_exp2(mr[n][e] - top) : 1.f;
          mr[n][e] = top;
          lr[n][e] *= f;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            o[n][i][e] *= f;
            o[n][i][e + 2] *= f;
          }
        }
      }
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float u0 = mr[n][0] == -INFINITY ? 0.f : mr[n][0], u1 = mr[n][1] == -INFINITY ? 0.f : mr[n][1];
      const float p0 = fast_exp2(x[n][0] - u0), p1 = fast_exp2(x[n][1] - u1);
      const float p2 = fast_exp2(x[n][2] - u0), p3 = fast_exp2(x[n][3] - u1);
      lr[n][0] += p0 + p2;
      lr[n][1] += p1 + p3;
      pb[n][0] = transpose8(pack_2(p0, p1, F16));
      pb[n][1] = transpose8(pack_2(p2, p3, F16));
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      uint32_t va[4];
      ldmatrix4_trans(va, slot + HALF + vj * (D * 2) + (((2 * i + vc) ^ (vj & 7)) << 4));
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_16816<F16>(o[n][i], va, pb[n][0], pb[n][1]);
    }
    __syncwarp();  // every lane has read the slot
#pragma unroll
    for (int c = 0; c + 1 < ST; ++c) ahead[c] = ahead[c + 1];
    ahead[ST - 1] = fetch(step + ST);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // the rings become the joining buffers

#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      lr[n][e] += __shfl_xor_sync(0xffffffffu, lr[n][e], 4);
      lr[n][e] += __shfl_xor_sync(0xffffffffu, lr[n][e], 8);
      lr[n][e] += __shfl_xor_sync(0xffffffffu, lr[n][e], 16);
      const int r = warp * ROWS + 8 * n + 2 * t + e;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        sh[r * D + 16 * i + g] = o[n][i][e];
        sh[r * D + 16 * i + g + 8] = o[n][i][e + 2];
      }
      if (g == 0) {
        sh_m[r] = mr[n][e];
        sh_l[r] = lr[n][e];
      }
    }
  __syncthreads();
  // the CTA's, in warp 0's place: an element is read and written by the same thread
  float keep_m = -INFINITY, keep_l = 0.f;
  if (tid < ROWS) {
#pragma unroll
    for (int w = 0; w < XT_WARPS; ++w) keep_m = fmaxf(keep_m, sh_m[w * ROWS + tid]);
#pragma unroll
    for (int w = 0; w < XT_WARPS; ++w)
      if (keep_m != -INFINITY) keep_l += sh_l[w * ROWS + tid] * fast_exp2(sh_m[w * ROWS + tid] - keep_m);
  }
  const int live = min(rows, ROWS);
  for (int i = tid; i < live * (D / 4); i += XT_THREADS) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < XT_WARPS; ++w) mx = fmaxf(mx, sh_m[w * ROWS + r]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mx != -INFINITY) {
#pragma unroll
      for (int w = 0; w < XT_WARPS; ++w) {
        const float f = fast_exp2(sh_m[w * ROWS + r] - mx);
        const float4 x = *reinterpret_cast<const float4*>(sh + (w * ROWS + r) * D + d);
        acc.x = fmaf(x.x, f, acc.x);
        acc.y = fmaf(x.y, f, acc.y);
        acc.z = fmaf(x.z, f, acc.z);
        acc.w = fmaf(x.w, f, acc.w);
      }
    }
    *reinterpret_cast<float4*>(sh + r * D + d) = acc;
  }
  __syncthreads();
  if (tid < ROWS) {
    sh_m[tid] = keep_m;
    sh_l[tid] = keep_l;
  }
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  // the cluster's: CTA `rank` finishes its share of the elements
  for (int i = rank * XT_THREADS + tid; i < live * (D / 4); i += csize * XT_THREADS) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    float mx = -INFINITY, l = 0.f;
    for (int c = 0; c < csize; ++c) mx = fmaxf(mx, cl.map_shared_rank(sh_m, c)[r]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mx != -INFINITY) {
      for (int c = 0; c < csize; ++c) {
        const float f = fast_exp2(cl.map_shared_rank(sh_m, c)[r] - mx);
        l = fmaf(cl.map_shared_rank(sh_l, c)[r], f, l);
        const float4 x = *reinterpret_cast<const float4*>(cl.map_shared_rank(sh, c) + r * D + d);
        acc.x = fmaf(x.x, f, acc.x);
        acc.y = fmaf(x.y, f, acc.y);
        acc.z = fmaf(x.z, f, acc.z);
        acc.w = fmaf(x.w, f, acc.w);
      }
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const long long row = qs + r / p.group;
    const int h = hk * p.group + r % p.group;
    acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    const float lse = l > 0.f ? (mx + __log2f(l)) * 0.6931471805599453f : -INFINITY;
    if (p.parts > 1) {
      const long long at = ((long long)part * p.heads + h) * p.total_q + row;
      *reinterpret_cast<float4*>(p.part_o + at * D + d) = acc;
      if (d == 0) p.part_lse[at] = lse;
    } else {
      uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + row * p.ldo + h * D + d;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_2(acc.x, acc.y, F16), pack_2(acc.z, acc.w, F16));
      if (d == 0 && p.lse) p.lse[(long long)h * p.total_q + row] = lse;
    }
  }
  cl.sync();  // no CTA leaves while another reads its shared memory
}

template <int D, bool F16, int NT>
static int launch_token(const XTokenParams& a, int csize, int sms, cudaStream_t st) {
  constexpr int ROWS = 8 * NT;
  constexpr int RING = XT_WARPS * XT_STAGES<D> * 2 * XT_KEYS * D * 2;
  constexpr int JOIN = (XT_WARPS * ROWS * D + 2 * XT_WARPS * ROWS) * 4;
  constexpr int NEED = RING > JOIN ? RING : JOIN;
  constexpr int ALONE = 120 * 1024;  // no second CTA fits beside it
  static_assert(NEED <= ALONE && 2 * (NEED + 1024) <= 228 * 1024, "two CTAs an SM");
  const long long ctas = (long long)a.p.batch * a.p.kv_heads * a.p.parts * csize;
  // The CTAs of a cluster are packed two to an SM where two fit, even when SMs are left empty. A launch that has an
  // SM for every CTA asks for so much shared memory that they spread.
  const int SMEM = ctas <= sms ? ALONE : NEED;
  // Between one and two waves of CTAs with lengths of their own the long ones start first: 64 sequences of 187 .. 1500
  // keys, 8 key heads: 25.2 -> 23.9 us (64 columns), 39.9 -> 36.8 (128), 40 of 500 .. 4000: 45.9 -> 37.7, 72.3 -> 65.9.
  // With shorter keys finding the place costs more (75 .. 600: 15.4 -> 17.5, 21.5 -> 23.6), with more waves the last ones
  // are of short sequences alone (16 key heads, 128 .. 1024 keys: 33.4 -> 42.8).
  const bool ordered = (a.p.k_lens || a.p.cu_k) && a.p.batch <= XT_MAX_ORDER && a.p.Lk >= XT_ORDER_KEYS &&
                       ctas > 2LL * sms && ctas <= 4LL * sms;
  auto kern = cross_token_kernel<D, F16, NT>;
  int rc;
  if ((rc = ensure_smem(kern, ALONE))) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(XT_THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = csize;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  int n = 1;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  if (cudaLaunchKernelEx(&cfg, kern, a, csize, ordered) != cudaSuccess) {
    cudaGetLastError();
    return SA3_ERR_LAUNCH;
  }
  return launch_status();
}

// Parts of the keys that are joined by a second launch: when even clusters of 8 leave SMs empty and the keys are
// long enough to pay for that launch. Two CTAs an SM. 8 key heads of 64 columns, cluster against parts: 7.5 and 7.9 us
// at 4096 keys, 10.4 and 10.0 at 8192, 49.9 and 27.0 at 65536; one key head of 128 columns and 8192 keys: 13.2 us in a
// cluster, 11.4, 8.6, 8.0 with 16, 32, 64 parts; 65536 keys: 13.9 with 128, 15.1 with 256.
int cross_token_parts(int batch, int kv_heads, int max_k, int sms) {
  const long long units = (long long)batch * kv_heads;
  if (units * XT_MAX_CLUSTER >= sms || max_k < XT_SPLIT_KEYS) return 1;
  const long long fill = 2LL * sms / units, most = max_k / XT_PART_KEYS;
  const long long n = fill < most ? fill : most;
  return (int)(n < XT_MAX_PARTS ? n : XT_MAX_PARTS);
}

// Cluster size: more CTAs to a key head while the launch leaves room for them and every warp still has a step of keys
// (8 key heads of 64 columns, 4096 keys: 26.6, 15.5, 10.3, 7.5 us with 1, 2, 4, 8; 16 sequences of 1024 keys: 10.7,
// 10.0, 14.7, 22.8).
int cross_token(const XParams& p, const void* q, const void* k, const void* v, long long ldq, long long ldk,
                long long ldv, int head_dim, int sms, cudaStream_t st) {
  XTokenParams a = {p, q, k, v, ldq, ldk, ldv};
  const long long units = (long long)p.batch * p.kv_heads;
  int csize = 1;
  while (p.parts == 1 && csize < XT_MAX_CLUSTER && units * csize * 2 <= 2LL * sms &&
         (long long)csize * 2 * XT_WARPS * XT_KEYS <= p.Lk)
    csize *= 2;
  const bool two = (long long)p.Lq * p.group > 8;
#define SA3_TOKEN(D, F) \
  return two ? launch_token<D, F, 2>(a, csize, sms, st) : launch_token<D, F, 1>(a, csize, sms, st)
  if (head_dim == 64) {
    if (p.f16) {
      SA3_TOKEN(64, true);
    }
    SA3_TOKEN(64, false);
  }
  if (p.f16) {
    SA3_TOKEN(128, true);
  }
  SA3_TOKEN(128, false);
#undef SA3_TOKEN
}

}  // namespace sa3
