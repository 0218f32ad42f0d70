// Arguments of the cross-attention kernels.
#pragma once
#include <cuda_runtime.h>

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
};

struct XGrad {
  const void* dout;
  void *dq, *dk, *dv;
  long long lddo, lddq, lddk, lddv;
  float* delta;    // [heads, total_q]
  float* partial;  // [parts][dV, dK][total_k, kv_heads * head_dim], NULL for one part
};

// Query rows (tokens x heads of a group) of a key head up to which the few-row kernel is taken.
constexpr int XT_MAX_ROWS = 16;
int cross_token(const XParams& p, const void* q, const void* k, const void* v, long long ldq, long long ldk,
                long long ldv, int head_dim, int sms, cudaStream_t st);

}  // namespace sa3
