// Attention of a few query rows (one decoded token of every sequence, times the query heads that share a key head)
// to an encoder's states: out = softmax(scale * q K^T) V over the visible keys.
//
// Bound by reading K and V once. All query rows of a key head (at most 16: query tokens x heads of the group) form
// one 16-row A operand, so K and V of the head are read once for the whole group. The keys are split over the warps
// of a cluster of CTAs, 16 keys a step; K and V go from global memory straight into the B fragments of the warp
// matrix instructions (the tensor cores' tcgen05 form would leave 112 of its 128 rows empty, and it needs the tiles
// in shared memory first), 16 bytes a lane:
//   K: lane (g, t) = (lane / 4, lane % 4) reads columns 32 c + 8 t .. + 7 of key g. They serve as the k indices
//      {2t, 2t+1, 2t+8, 2t+9} of two steps; the sum over a head's columns may run in any order, so Q's fragments are
//      read in the same order.
//   V: lane (g, t) reads columns 64 c + 8 g .. + 7 of keys 2t, 2t+1, 2t+8, 2t+9; column e of the eight belongs to
//      the n-tile e, whose column g is thus d = 64 c + 8 g + e.
// Hidden keys are not read: their registers are zero and their scores -inf.
// Each warp keeps its own running maximum, sum and fp32 accumulators; the warps of a CTA join through shared memory
// and the CTAs of the cluster through distributed shared memory, in a fixed order: one launch, no workspace.
#include <cooperative_groups.h>

#include "attn_tile.cuh"
#include "common.cuh"
#include "cross_attention.h"
#include "host_util.h"

namespace sa3 {
namespace cg = cooperative_groups;

constexpr int XT_WARPS = 8;
constexpr int XT_THREADS = XT_WARPS * 32;
constexpr int XT_KEYS = 16;  // keys of a step of a warp

struct XTokenParams {
  XParams p;
  const void *q, *k, *v;
  long long ldq, ldk, ldv;
};

__device__ __forceinline__ int clamp_to(int v, int lo, int hi) { return min(max(v, lo), hi); }

template <bool F16>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// R16: 9..16 query rows, else at most 8 (the upper half of every fragment is zero and is not kept).
template <int D, bool F16, bool R16>
__global__ void __launch_bounds__(XT_THREADS, R16 ? 1 : 2) cross_token_kernel(const XTokenParams a, int csize) {
  constexpr int ROWS = R16 ? 16 : 8;
  constexpr int KC = D / 32, VC = D / 64;  // 16-byte column chunks of a lane
  extern __shared__ float sh[];            // [warps][ROWS][D] partial outputs, then [warps][ROWS] maxima and sums
  float* sh_m = sh + XT_WARPS * ROWS * D;
  float* sh_l = sh_m + XT_WARPS * ROWS;
  const XParams& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % csize, unit = blockIdx.x / csize;
  const int hk = unit % p.kv_heads, b = unit / p.kv_heads;
  grid_dep_wait();
  int qs = b * p.Lq, lq = p.Lq, ks = b * p.Lk, lk = p.Lk;
  if (p.cu_q) {
    qs = clamp_to(__ldg(p.cu_q + b), 0, p.total_q);
    lq = clamp_to(__ldg(p.cu_q + b + 1) - qs, 0, min(p.total_q - qs, p.Lq));
  }
  if (p.cu_k) {
    ks = clamp_to(__ldg(p.cu_k + b), 0, p.total_k);
    lk = clamp_to(__ldg(p.cu_k + b + 1) - ks, 0, min(p.total_k - ks, p.Lk));
  }
  const int seen = p.k_lens ? clamp_to(__ldg(p.k_lens + b), 0, lk) : lk;
  const int rows = lq * p.group;  // row m: token m / group, head hk * group + m % group

  // Q fragments in the column order of the K loads
  uint32_t qa[KC][2][2], qb[KC][2][2];  // [chunk][step][a0, a2] of row g, [a1, a3] of row g + 8
  auto q_row = [&](int m) {
    return reinterpret_cast<const uint16_t*>(a.q) + (long long)(qs + m / p.group) * a.ldq +
           (hk * p.group + m % p.group) * D;
  };
#pragma unroll
  for (int c = 0; c < KC; ++c) {
    uint4 x = make_uint4(0, 0, 0, 0), y = x;
    if (g < rows) x = __ldg(reinterpret_cast<const uint4*>(q_row(g) + 32 * c + 8 * t));
    if (R16 && g + 8 < rows) y = __ldg(reinterpret_cast<const uint4*>(q_row(g + 8) + 32 * c + 8 * t));
    qa[c][0][0] = x.x, qa[c][0][1] = x.y, qa[c][1][0] = x.z, qa[c][1][1] = x.w;
    qb[c][0][0] = y.x, qb[c][0][1] = y.y, qb[c][1][0] = y.z, qb[c][1][1] = y.w;
  }

  float o[VC * 8][R16 ? 4 : 2];
#pragma unroll
  for (int n = 0; n < VC * 8; ++n)
#pragma unroll
    for (int e = 0; e < (R16 ? 4 : 2); ++e) o[n][e] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

  const uint16_t* kb = reinterpret_cast<const uint16_t*>(a.k) + hk * D + 8 * t;
  const uint16_t* vb = reinterpret_cast<const uint16_t*>(a.v) + hk * D + 8 * g;
  const int stride = csize * XT_WARPS * XT_KEYS;
  for (int j0 = (rank * XT_WARPS + warp) * XT_KEYS; j0 < seen; j0 += stride) {
    uint32_t vis = seen - j0 >= XT_KEYS ? 0xffffu : (1u << (seen - j0)) - 1u;
    if (p.key_mask) {
      const bool on = lane < XT_KEYS && ((vis >> lane) & 1u) && __ldg(p.key_mask + ks + j0 + lane) != 0;
      vis = __ballot_sync(0xffffffffu, on);
    }
    uint4 kf[2][KC], vf[4][VC];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const bool on = (vis >> (8 * n + g)) & 1u;
      const uint16_t* src = kb + (long long)(ks + j0 + 8 * n + g) * a.ldk;
#pragma unroll
      for (int c = 0; c < KC; ++c) kf[n][c] = on ? ld_stream(src + 32 * c) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int j = 2 * t + (r & 1) + 8 * (r >> 1);
      const bool on = (vis >> j) & 1u;
      const uint16_t* src = vb + (long long)(ks + j0 + j) * a.ldv;
#pragma unroll
      for (int c = 0; c < VC; ++c) vf[r][c] = on ? ld_stream(src + 64 * c) : make_uint4(0, 0, 0, 0);
    }
    float s[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        mma_16816<F16>(s[n], qa[c][0][0], R16 ? qb[c][0][0] : 0u, qa[c][0][1], R16 ? qb[c][0][1] : 0u, kf[n][c].x,
                       kf[n][c].y);
        mma_16816<F16>(s[n], qa[c][1][0], R16 ? qb[c][1][0] : 0u, qa[c][1][1], R16 ? qb[c][1][1] : 0u, kf[n][c].z,
                       kf[n][c].w);
      }
      // lane (g, t) holds keys 8 n + 2 t, + 1 of rows g and g + 8
      const bool on0 = (vis >> (8 * n + 2 * t)) & 1u, on1 = (vis >> (8 * n + 2 * t + 1)) & 1u;
      s[n][0] = on0 ? s[n][0] * p.scale_log2 : -INFINITY;
      s[n][1] = on1 ? s[n][1] * p.scale_log2 : -INFINITY;
      s[n][2] = on0 ? s[n][2] * p.scale_log2 : -INFINITY;
      s[n][3] = on1 ? s[n][3] * p.scale_log2 : -INFINITY;
    }
    auto quad_max = [](float x) {
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
    };
    const float n0 = fmaxf(m0, quad_max(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]))));
    const float n1 = R16 ? fmaxf(m1, quad_max(fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3])))) : 0.f;
    if (__any_sync(0xffffffffu, n0 > m0 || (R16 && n1 > m1))) {
      const float f0 = n0 > m0 ? fast_exp2(m0 - n0) : 1.f, f1 = R16 && n1 > m1 ? fast_exp2(m1 - n1) : 1.f;
      l0 *= f0;
      l1 *= f1;
#pragma unroll
      for (int n = 0; n < VC * 8; ++n) {
        o[n][0] *= f0;
        o[n][1] *= f0;
        if (R16) {
          o[n][2] *= f1;
          o[n][3] *= f1;
        }
      }
      m0 = n0;
      m1 = n1;
    }
    const float u0 = m0 == -INFINITY ? 0.f : m0, u1 = m1 == -INFINITY ? 0.f : m1;
    uint32_t pa[2], pb[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const float e0 = fast_exp2(s[n][0] - u0), e1 = fast_exp2(s[n][1] - u0);
      l0 += e0 + e1;
      pa[n] = pack_2(e0, e1, F16);
      pb[n] = 0u;
      if (R16) {
        const float e2 = fast_exp2(s[n][2] - u1), e3 = fast_exp2(s[n][3] - u1);
        l1 += e2 + e3;
        pb[n] = pack_2(e2, e3, F16);
      }
    }
#pragma unroll
    for (int c = 0; c < VC; ++c) {
      const uint32_t w0[4] = {vf[0][c].x, vf[0][c].y, vf[0][c].z, vf[0][c].w};
      const uint32_t w1[4] = {vf[1][c].x, vf[1][c].y, vf[1][c].z, vf[1][c].w};
      const uint32_t w2[4] = {vf[2][c].x, vf[2][c].y, vf[2][c].z, vf[2][c].w};
      const uint32_t w3[4] = {vf[3][c].x, vf[3][c].y, vf[3][c].z, vf[3][c].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t sel = e & 1 ? 0x7632u : 0x5410u;
        const uint32_t b0 = __byte_perm(w0[e >> 1], w1[e >> 1], sel), b1 = __byte_perm(w2[e >> 1], w3[e >> 1], sel);
        float x[4] = {o[8 * c + e][0], o[8 * c + e][1], R16 ? o[8 * c + e][R16 ? 2 : 0] : 0.f,
                      R16 ? o[8 * c + e][R16 ? 3 : 0] : 0.f};
        mma_16816<F16>(x, pa[0], pb[0], pa[1], pb[1], b0, b1);
        o[8 * c + e][0] = x[0];
        o[8 * c + e][1] = x[1];
        if (R16) {
          o[8 * c + e][R16 ? 2 : 0] = x[2];
          o[8 * c + e][R16 ? 3 : 0] = x[3];
        }
      }
    }
  }

  // the warp's partial result: lane (g, t) has d = 64 c + 16 t + e (first of a pair) and + 8 (second)
  auto quad_sum = [](float x) {
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    return x + __shfl_xor_sync(0xffffffffu, x, 2);
  };
  l0 = quad_sum(l0);
  l1 = quad_sum(l1);
#pragma unroll
  for (int hh = 0; hh < (R16 ? 2 : 1); ++hh) {
    float* dst = sh + (warp * ROWS + g + 8 * hh) * D + 16 * t;
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int n = 8 * c + (e & 7), x = 2 * hh + (e >> 3);
        *reinterpret_cast<float4*>(dst + 64 * c + e) = make_float4(o[n][x], o[n + 1][x], o[n + 2][x], o[n + 3][x]);
      }
    if (t == 0) {
      sh_m[warp * ROWS + g + 8 * hh] = hh ? m1 : m0;
      sh_l[warp * ROWS + g + 8 * hh] = hh ? l1 : l0;
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
    uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + row * p.ldo + h * D + d;
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(pack_2(acc.x * inv, acc.y * inv, F16), pack_2(acc.z * inv, acc.w * inv, F16));
    if (d == 0 && p.lse)
      p.lse[(long long)h * p.total_q + row] = l > 0.f ? (mx + __log2f(l)) * 0.6931471805599453f : -INFINITY;
  }
  cl.sync();  // no CTA leaves while another reads its shared memory
}

template <int D, bool F16, bool R16>
static int launch_token(const XTokenParams& a, int csize, cudaStream_t st) {
  constexpr int ROWS = R16 ? 16 : 8;
  constexpr int SMEM = (XT_WARPS * ROWS * D + 2 * XT_WARPS * ROWS) * 4;
  auto kern = cross_token_kernel<D, F16, R16>;
  int rc;
  if ((rc = ensure_smem(kern, SMEM))) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)a.p.batch * a.p.kv_heads * csize));
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
  if (cudaLaunchKernelEx(&cfg, kern, a, csize) != cudaSuccess) {
    cudaGetLastError();
    return SA3_ERR_LAUNCH;
  }
  return launch_status();
}

// Cluster size: more CTAs to a key head while the launch leaves SMs idle and every warp still has a step of keys.
int cross_token(const XParams& p, const void* q, const void* k, const void* v, long long ldq, long long ldk,
                long long ldv, int head_dim, int sms, cudaStream_t st) {
  XTokenParams a = {p, q, k, v, ldq, ldk, ldv};
  const long long units = (long long)p.batch * p.kv_heads;
  int csize = 1;
  while (csize < 8 && units * csize < 2LL * sms && (long long)csize * 2 * XT_WARPS * XT_KEYS <= p.Lk) csize *= 2;
  const bool r16 = (long long)p.Lq * p.group > 8;
#define SA3_TOKEN(D, F)                                                              \
  return r16 ? launch_token<D, F, true>(a, csize, st) : launch_token<D, F, false>(a, csize, st)
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
