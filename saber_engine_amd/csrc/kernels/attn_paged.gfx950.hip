// The code object `attn_paged`: what stands between a decoder layer's qkv linear and its output gate. No counterpart among the
// objects this library stands in for (the reference's attention kernels are outside the linear's path).
//
//   kv_append_{bf16,e4m3}_d{64,128,256}              new tokens into the paged cache, position rotation on the way (attn_append.h)
//   attn_few_{bf16,e4m3}_d{64,128,256}_r{16,32}      attention of up to 16 / 32 rows a kv head and sequence (attn_few.h)
//   attn_many_{bf16,e4m3}_d{64,128,256}              attention of many rows, 128 a workgroup (attn_many.h)
#include "attn_append.h"
#include "attn_few.h"
#include "attn_many.h"

#define KV_APPEND(name, D, F8)                                                                                                    \
  extern "C" __global__ __launch_bounds__(256) void kv_append_##name##_d##D(                                                      \
      const unsigned short *__restrict__ q, const unsigned short *__restrict__ k, const unsigned short *__restrict__ v,           \
      unsigned short *__restrict__ q_out, unsigned char *__restrict__ kc, unsigned char *__restrict__ vc,                         \
      const float *__restrict__ k_scale, const float *__restrict__ v_scale, const int *__restrict__ table,                        \
      const int *__restrict__ kv_len, const int *__restrict__ cu_q, const unsigned short *__restrict__ q_norm,                    \
      const unsigned short *__restrict__ k_norm, const double *__restrict__ inv_freq, int q_row, int q_head, int kv_row,          \
      int tokens, int seqs, int shape, int form, int pages, int table_stride, float eps) {                                       \
    kv_append_body<D, F8>(q, k, v, q_out, kc, vc, k_scale, v_scale, table, kv_len, cu_q, q_norm, k_norm, inv_freq, q_row, q_head, \
                          kv_row, tokens, seqs, shape, form, pages, table_stride, eps);                                           \
  }
#define ATTN_FEW(name, D, F8, RT, R)                                                                                              \
  extern "C" __global__ __launch_bounds__(256, RT == 1 && (D < 256 || F8) ? 2 : 1) void attn_few_##name##_d##D##_r##R(                                                \
      const unsigned short *__restrict__ q, const unsigned char *__restrict__ kc, const unsigned char *__restrict__ vc,           \
      const float *__restrict__ k_scale, const float *__restrict__ v_scale, const int *__restrict__ table,                        \
      const int *__restrict__ kv_len, const int *__restrict__ cu_q, unsigned short *__restrict__ out, float *__restrict__ partial, \
      int *__restrict__ counter, int q_row, int tokens, int seqs, int shape, int page_shift, int pages, int table_stride,         \
      int unit_shift, int qtiles, float scale) {                                                                                  \
    attn_few_body<D, F8, RT>(q, kc, vc, k_scale, v_scale, table, kv_len, cu_q, out, partial, counter, q_row, tokens, seqs, shape, \
                             page_shift, pages, table_stride, unit_shift, qtiles, scale);                                             \
  }
#define ATTN_MANY(name, D, F8)                                                                                                    \
  extern "C" __global__ __launch_bounds__(256, 2) void attn_many_##name##_d##D(                                                      \
      const unsigned short *__restrict__ q, const unsigned char *__restrict__ kc, const unsigned char *__restrict__ vc,           \
      const float *__restrict__ k_scale, const float *__restrict__ v_scale, const int *__restrict__ table,                        \
      const int *__restrict__ kv_len, const int *__restrict__ cu_q, unsigned short *__restrict__ out, float *__restrict__ partial, \
      int *__restrict__ counter, int q_row, int tokens, int shape, int page_shift, int pages, int table_stride, int chunk,        \
      int splits, int qtiles, float scale) {                                                                                      \
    attn_many_body<D, F8>(q, kc, vc, k_scale, v_scale, table, kv_len, cu_q, out, partial, counter, q_row, tokens, shape,          \
                          page_shift, pages, table_stride, chunk, splits, qtiles, scale);                                         \
  }
#define ATTN_ALL(D)            \
  KV_APPEND(bf16, D, false)    \
  KV_APPEND(e4m3, D, true)     \
  ATTN_FEW(bf16, D, false, 1, 16) \
  ATTN_FEW(bf16, D, false, 2, 32) \
  ATTN_FEW(e4m3, D, true, 1, 16)  \
  ATTN_FEW(e4m3, D, true, 2, 32)  \
  ATTN_MANY(bf16, D, false)    \
  ATTN_MANY(e4m3, D, true)
ATTN_ALL(64)
ATTN_ALL(128)
ATTN_ALL(256)
