// Rotary positions on token rows, in the general form: half or interleaved pairs, any even part of the head,
// any frequencies (long-context scalings change the frequencies and a common factor), 16-bit or fp32 data,
// queries and keys of different head counts in one launch, and the inverse rotation (the gradient).
//
// With theta(p, i) = p * inv_freq[i] a pair (a, b) becomes scale * (a cos - b sin, b cos + a sin); the inverse
// has -sin. The map is linear and scale * R(theta) transposed is scale * R(-theta), so the inverse is the
// backward pass. The pairs are (i, i + r/2) in the half layout, (2i, 2i + 1) in the interleaved one; columns
// r.. of a head pass through.
//
// Angles: p * inv_freq in fp32 is wrong by 0.06 rad at p = 1e6, so the turn count p * (inv_freq / 2 pi) is formed
// in fp64 and reduced to its fraction there; the fraction (|x| <= 1/2) goes to fp32, where sincospif is exact to
// 2 ulp: the angle is within 1e-7 rad for every 32-bit position, without a table to read or to run past.
//
// Bound by memory: each element is read and written once. A block takes `rpb` rows; it first computes their
// rpb * r/2 cosines and sines into shared memory (once for all heads), while each thread's first data loads are
// already in flight. A thread keeps one unit of the head (2 * VEC elements: VEC pairs, or 2 * VEC columns that
// pass through) and walks heads and rows. VEC is the widest vector that the alignment of every pointer, stride
// and part of the head allows, up to 16 bytes (16494 rows x 48 heads x 64 of bf16: 32.6, 43.2, 56.2, 99.6 us with
// 16, 8, 4, 2 bytes).
#include "common.cuh"
#include "host_util.h"

namespace sa3 {

constexpr int ROT_THREADS = 256;
constexpr int ROT_MAX_DIM = 512;
constexpr int ROT_MAX_RPB = 4;
constexpr int ROT_BATCH = 2;

struct RotaryParams {
  const void* x[2];  // q, k
  void* y[2];  // may be x: a thread reads an element before it writes it, and no other thread touches it
  long long ldx[2], ldy[2];
  int heads[2];
  int dim, rot;           // columns of a head, rotated ones
  int units;              // units of a head that are visited
  int heads_par;          // heads a block takes side by side
  long long rows;
  int rpb;                // rows of a block
  const double* inv_freq;
  const int* row_pos;
  long long rows_per_batch, offset;
  float scale;
  float sign;
  bool stream;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// stream: evicted first, for outputs that L2 could not keep for their reader anyway
template <typename T, int VEC>
__device__ __forceinline__ void put(T* dst, const Pack<T, VEC>& v, bool stream) {
  if constexpr (sizeof(Pack<T, VEC>) == 16) {
    if (stream) {
      __stcs(reinterpret_cast<uint4*>(dst), *reinterpret_cast<const uint4*>(&v));
      return;
    }
  }
  *reinterpret_cast<Pack<T, VEC>*>(dst) = v;
}

template <typename T, int VEC, bool IL>
__global__ void __launch_bounds__(ROT_THREADS) rotary_kernel(RotaryParams p) {
  __shared__ float2 cs[ROT_MAX_RPB * ROT_MAX_DIM / 2];
  using V = Pack<T, VEC>;
  const int tid = threadIdx.x;
  const long long row0 = (long long)blockIdx.x * p.rpb;
  const int nrows = (int)min((long long)p.rpb, p.rows - row0);
  const int half = p.rot >> 1;
  grid_dep_wait();

  const int u = tid % p.units, hq = tid / p.units;
  const bool rotates = u * 2 * VEC < p.rot;
  // element offsets of the unit's two vectors within a head
  const int c0 = IL || !rotates ? u * 2 * VEC : u * VEC;
  const int c1 = IL || !rotates ? c0 + VEC : half + u * VEC;
  const bool has1 = VEC > 1 || c1 < p.dim;  // an odd width leaves the last one-element unit without its second half
  const int total = p.heads[0] + p.heads[1];
  auto at = [&](int r, int h, const void* const* base, const long long* ld) {
    const int w = h >= p.heads[0];
    return reinterpret_cast<const T*>(base[w]) + (row0 + r) * ld[w] + (long long)(h - (w ? p.heads[0] : 0)) * p.dim;
  };
  // The thread's steps: heads hq, hq + heads_par, .. of the first row, then of the next. ROT_BATCH steps are loaded
  // before the first of them is stored.
  V a[ROT_BATCH], b[ROT_BATCH];
  auto fetch = [&](int r, int h) {
#pragma unroll
    for (int n = 0; n < ROT_BATCH; ++n) {
      if (r < nrows) {
        const T* x = at(r, h, p.x, p.ldx);
        a[n] = *reinterpret_cast<const V*>(x + c0);
        b[n] = a[n];
        if (has1) b[n] = *reinterpret_cast<const V*>(x + c1);
      }
      h += p.heads_par;
      if (h >= total) h = hq, ++r;
    }
  };
  fetch(0, hq);  // in flight while the angles are computed

  for (int i = tid; i < nrows * half; i += blockDim.x) {
    const int rr = i / half, f = i - rr * half;
    const long long row = row0 + rr;
    const long long pos = p.row_pos ? (long long)__ldg(p.row_pos + row)
                                    : p.offset + (p.rows_per_batch > 0 ? row % p.rows_per_batch : row);
    double t = (double)pos * (__ldg(p.inv_freq + f) * 0.15915494309189533577);  // 1 / (2 pi)
    t -= rint(t);
    float s, c;
    sincospif(2.f * (float)t, &s, &c);
    cs[i] = make_float2(c * p.scale, s * p.scale * p.sign);
  }
  __syncthreads();

  int r = 0, h = hq;
  while (true) {
#pragma unroll
    for (int n = 0; n < ROT_BATCH; ++n) {
      if (r < nrows) {
        V &x = a[n], &y = b[n];
        if (rotates) {
          const float2* w = cs + r * half + u * VEC;
          if (IL) {
            // VEC pairs in 2 * VEC consecutive elements: pair e sits at elements 2e and 2e + 1
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              T& lo = 2 * e < VEC ? x.v[(2 * e) % VEC] : y.v[(2 * e) % VEC];
              T& hi = 2 * e + 1 < VEC ? x.v[(2 * e + 1) % VEC] : y.v[(2 * e + 1) % VEC];
              const float f = to_f32(lo), g = to_f32(hi);
              lo = from_f32<T>(f * w[e].x - g * w[e].y);
              hi = from_f32<T>(g * w[e].x + f * w[e].y);
            }
          } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float f = to_f32(x.v[e]), g = to_f32(y.v[e]);
              x.v[e] = from_f32<T>(f * w[e].x - g * w[e].y);
              y.v[e] = from_f32<T>(g * w[e].x + f * w[e].y);
            }
          }
        }
        T* dst = const_cast<T*>(at(r, h, p.y, p.ldy));
        put(dst + c0, x, p.stream);
        if (has1) put(dst + c1, y, p.stream);
      }
      h += p.heads_par;
      if (h >= total) h = hq, ++r;
    }
    if (r >= nrows) break;
    fetch(r, h);
  }
}

template <typename T, int VEC>
int launch_rotary(RotaryParams p, bool il, bool in_place, cudaStream_t st) {
  const int unit = 2 * VEC;
  p.units = ((in_place ? p.rot : p.dim) + unit - 1) / unit;
  const int total = p.heads[0] + p.heads[1];
  const int most = ROT_THREADS / p.units;  // >= 1: units <= ROT_MAX_DIM / 2
  const int turns = (total + most - 1) / most;
  p.heads_par = (total + turns - 1) / turns;
  const int threads = p.units * p.heads_par;
  // More rows to a block save blocks and overlap one's angles with another's data once every SM has several blocks; below
  // that one row each spreads the work. 1, 2, 4 rows: 2.1, 2.2, 3.0 us for 256 rows of 48 heads x 64, 6.2, 6.0, 6.1 for
  // 2400, 38.0, 33.4, 32.6 for 16494; 3.8, 3.6, 4.5 for 2400 rows of 8 heads x 128, 13.4, 13.2, 13.7 for 16494.
  const bool wide = p.rows >= 148 * 64 && total * p.dim * (int)sizeof(T) > 4096;
  p.rpb = p.rows < 148 * 16 ? 1 : wide ? ROT_MAX_RPB : 2;
  // Outputs above a quarter of L2 are stored evict-first: 39.7 -> 33.5 us for 101 MB out of a fused buffer (16494 rows x
  // 48 heads x 64), 69 -> 65 us for 210 MB. Smaller ones are left for the attention that reads them next.
  p.stream = p.rows * total * p.dim * (long long)sizeof(T) > (32LL << 20);
  const long long blocks = (p.rows + p.rpb - 1) / p.rpb;
  if (blocks > 0x7fffffffLL) return SA3_ERR_UNSUPPORTED;
  auto kern = il ? rotary_kernel<T, VEC, true> : rotary_kernel<T, VEC, false>;
  launch_ex(kern, dim3((unsigned)blocks), dim3(threads), 0, st, 1, p);
  return launch_status();
}

}  // namespace sa3

using namespace sa3;

extern "C" int sa3_rotary(const void* q, void* q_out, const void* k, void* k_out, int dtype, long long rows, int heads,
                          int kv_heads, int head_dim, int rot_dim, long long ldq, long long ldqo, long long ldk,
                          long long ldko, const double* inv_freq, const int* row_pos, long long rows_per_batch,
                          long long offset, int interleaved, int inverse, float scale, void* stream) {
  if (rows < 0 || heads <= 0 || head_dim <= 0 || rot_dim <= 0 || rot_dim > head_dim || (rot_dim & 1) ||
      rows_per_batch < 0)
    return SA3_ERR_ARG;
  if (k ? kv_heads <= 0 || !k_out : kv_heads != 0 || k_out) return SA3_ERR_ARG;
  if (head_dim > ROT_MAX_DIM || heads > 65535 || kv_heads > 65535) return SA3_ERR_UNSUPPORTED;
  int esz = 0;
  if (dtype == SA3_DT_F32) esz = 4;
  else if (dtype == SA3_DT_BF16 || dtype == SA3_DT_F16) esz = 2;
  else return SA3_ERR_DTYPE;
  const long long wq = (long long)heads * head_dim, wk = (long long)kv_heads * head_dim;
  if (ldq < wq || ldqo < wq || (k && (ldk < wk || ldko < wk))) return SA3_ERR_ARG;
  if (rows == 0) return SA3_OK;
  if (!q || !q_out || !inv_freq) return SA3_ERR_ARG;
  const uintptr_t any = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) |
                        reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out);
  if ((q == q_out && ldq != ldqo && rows > 1) || (k && k == k_out && ldk != ldko && rows > 1)) return SA3_ERR_ARG;
  if (k && (q_out == k_out || q_out == k || k_out == q)) return SA3_ERR_ARG;
  if (any % esz || (reinterpret_cast<uintptr_t>(inv_freq) & 7) || (reinterpret_cast<uintptr_t>(row_pos) & 3))
    return SA3_ERR_ALIGN;

  RotaryParams p = {};
  p.x[0] = q;
  p.x[1] = k;
  p.y[0] = q_out;
  p.y[1] = k_out;
  p.ldx[0] = ldq;
  p.ldx[1] = k ? ldk : 0;
  p.ldy[0] = ldqo;
  p.ldy[1] = k ? ldko : 0;
  p.heads[0] = heads;
  p.heads[1] = k ? kv_heads : 0;
  p.dim = head_dim;
  p.rot = rot_dim;
  p.rows = rows;
  p.inv_freq = inv_freq;
  p.row_pos = row_pos;
  p.rows_per_batch = rows_per_batch;
  p.offset = offset;
  p.scale = scale;
  p.sign = inverse ? -1.f : 1.f;
  const bool il = interleaved != 0;
  // in place the columns that pass through need not be touched
  const bool in_place = q == q_out && ldq == ldqo && (!k || (k == k_out && ldk == ldko));
  auto fits = [&](int vec) {
    const int unit = 2 * vec;
    const bool parts = (il ? rot_dim % unit : (rot_dim / 2) % vec) == 0 && (head_dim - rot_dim) % unit == 0;
    const long long lds = p.ldx[0] | p.ldx[1] | p.ldy[0] | p.ldy[1];
    return parts && any % ((uintptr_t)vec * esz) == 0 && lds % vec == 0 && head_dim % vec == 0;
  };
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == SA3_DT_F32) {
    if (fits(4)) return launch_rotary<float, 4>(p, il, in_place, st);
    if (fits(2)) return launch_rotary<float, 2>(p, il, in_place, st);
    return launch_rotary<float, 1>(p, il, in_place, st);
  }
#define SA3_ROTARY(T)                                                  \
  if (fits(8)) return launch_rotary<T, 8>(p, il, in_place, st);        \
  if (fits(4)) return launch_rotary<T, 4>(p, il, in_place, st);        \
  if (fits(2)) return launch_rotary<T, 2>(p, il, in_place, st);        \
  return launch_rotary<T, 1>(p, il, in_place, st)
  if (dtype == SA3_DT_F16) {
    SA3_ROTARY(__half);
  }
  SA3_ROTARY(__nv_bfloat16);
#undef SA3_ROTARY
}
