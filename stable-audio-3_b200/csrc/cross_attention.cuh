// Arguments of the cross-attention kernels, the clamped sequence offsets and the split over the keys.
#pragma once
#include "common.cuh"

namespace sa3 {

struct XParams {
  const int* cu_q;  // packed batches: row offsets of the sequences, else NULL and Lq / Lk rows each
  const int* cu_k;
  const int* k_lens;              // keys that may be seen, per sequence, or NULL
  const unsigned char* key_mask;  // one byte a key row, zero = hidden, or NULL
  int batch, Lq, Lk, total_q, total_k;
  int heads, kv_heads, group;
  float scale, scale_log2;
  int f16;  // fp16 operands and outputs, else bf16
  void* out;
  long long ldo;
  float* lse;  // [heads, total_q] natural logarithms, or NULL
  // Forward with the keys split over CTAs that do not meet (parts > 1): each part's normalised output and lse, joined
  // by a second launch. part_o [parts][heads][total_q][head_dim], part_lse [parts][heads][total_q].
  int parts;
  float* part_o;
  float* part_lse;
};

struct XGrad {
  const void* dout;
  void *dq, *dk, *dv;
  long long lddo, lddq, lddk, lddv;
  float* stats;    // [-lse * log2(e), -delta][heads, total_q]
  float* partial;  // [parts][dV, dK][total_k, kv_heads * head_dim], NULL for one part
};

// One sequence: row offsets and lengths, clamped to the buffers so that no offset reaches outside them.
struct XSeq {
  int qs, lq, ks, lk, seen;  // seen: keys before the sequence's key length (a key mask may hide more)
};

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

__device__ __forceinline__ XSeq make_seq(const XParams& p, int b) {
  XSeq s;
  if (p.cu_q) {
    s.qs = clampi(__ldg(p.cu_q + b), 0, p.total_q);
    s.lq = clampi(__ldg(p.cu_q + b + 1) - s.qs, 0, min(p.total_q - s.qs, p.Lq));
  } else {
    s.qs = b * p.Lq;
    s.lq = p.Lq;
  }
  if (p.cu_k) {
    s.ks = clampi(__ldg(p.cu_k + b), 0, p.total_k);
    s.lk = clampi(__ldg(p.cu_k + b + 1) - s.ks, 0, min(p.total_k - s.ks, p.Lk));
  } else {
    s.ks = b * p.Lk;
    s.lk = p.Lk;
  }
  s.seen = p.k_lens ? clampi(__ldg(p.k_lens + b), 0, s.lk) : s.lk;
  return s;
}

// Query rows (tokens x heads of a group) of a key head up to which the few-row kernel is taken: what its two
// instruction tiles hold. Against the tile kernel, 8 key heads: 8 rows of one token 7.8 to 29.9 us (64 columns, 4096
// keys), 14.6 to 164.7 (32 sequences of 1024 keys); 16 tokens of single heads 8.8 to 17.4, 16.7 to 28.0, and at 128
// columns 11.5 to 14.8, 28.2 to 26.1.
constexpr int XT_MAX_ROWS = 16;
int cross_token_parts(int batch, int kv_heads, int max_k, int sms);
int cross_token(const XParams& p, const void* q, const void* k, const void* v, long long ldq, long long ldk,
                long long ldv, int head_dim, int sms, cudaStream_t st);

}  // namespace sa3
