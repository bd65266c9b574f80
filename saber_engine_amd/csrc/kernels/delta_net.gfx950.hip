// The code object `delta_net`: what stands between a delta-net layer's projections and its norm and output gate, and the copies that fork a
// sequence. No counterpart among the objects this library stands in for (the reference's delta-net kernels are outside the linear's path).
//
//   delta_conv_w{2,3,4}     short causal convolution and SiLU of new rows (delta_conv.h)
//   delta_step_c{16,32}     the gated delta rule a row at a time (delta_step.h)
//   delta_prep, delta_scan_w{2,4}  ... in chunks of 64 rows (delta_chunk.h)
//   block_copy              blocks of two arrays to other blocks (block_copy.h)
#include "block_copy.h"
#include "delta_chunk.h"
#include "delta_conv.h"
#include "delta_step.h"

#define DELTA_CONV(W)                                                                                                                      \
  extern "C" __global__ __launch_bounds__(256) void delta_conv_w##W(                                                                       \
      const unsigned short *__restrict__ x, const unsigned short *__restrict__ weight, const unsigned short *__restrict__ bias,            \
      unsigned short *__restrict__ tail, const int *__restrict__ slot, const int *__restrict__ cu_q, const int *__restrict__ kept,         \
      unsigned short *__restrict__ out, int x_row, int out_row, int tokens, int seqs, int channels, int slots, int run) {                  \
    delta_conv_body<W>(x, weight, bias, tail, slot, cu_q, kept, out, x_row, out_row, tokens, seqs, channels, slots, run);                  \
  }
DELTA_CONV(2)
DELTA_CONV(3)
DELTA_CONV(4)

#define DELTA_STEP(C)                                                                                                                            \
  extern "C" __global__ __launch_bounds__(64 * 128 / C) void delta_step_c##C(                                                                    \
      const unsigned short *__restrict__ q, const unsigned short *__restrict__ k, const unsigned short *__restrict__ v,                          \
      const unsigned short *__restrict__ a, const unsigned short *__restrict__ b, const float *__restrict__ a_log,                               \
      const float *__restrict__ dt_bias, float *__restrict__ state, const int *__restrict__ slot, const int *__restrict__ cu_q,                  \
      const int *__restrict__ kept, unsigned short *__restrict__ out, int row, int ab_row, int tokens, int seqs, int shape, int slots, float eps, \
      float scale) {                                                                                                                             \
    delta_step_body<C>(q, k, v, a, b, a_log, dt_bias, state, slot, cu_q, kept, out, row, ab_row, tokens, seqs, shape, slots, eps, scale);        \
  }
DELTA_STEP(16)
DELTA_STEP(32)

extern "C" __global__ __launch_bounds__(256, 4) void delta_prep(
    const unsigned short *__restrict__ q, const unsigned short *__restrict__ k, const unsigned short *__restrict__ a, const unsigned short *__restrict__ b,
    const float *__restrict__ a_log, const float *__restrict__ dt_bias, const int *__restrict__ slot, const int *__restrict__ cu_q,
    unsigned char *__restrict__ keys, unsigned char *__restrict__ work, int row, int ab_row, int tokens, int seqs, int shape, int slots, int places, int many,
    float eps) {
  delta_prep_body(q, k, a, b, a_log, dt_bias, slot, cu_q, keys, work, row, ab_row, tokens, seqs, shape, slots, places, many, eps);
}

#define DELTA_SCAN(W)                                                                                                                         \
  extern "C" __global__ __launch_bounds__(128 * W) void delta_scan_w##W(                                                                      \
      const unsigned short *__restrict__ v, const unsigned char *__restrict__ keys, const unsigned char *__restrict__ work,                   \
      float *__restrict__ state, const int *__restrict__ slot, const int *__restrict__ cu_q, unsigned short *__restrict__ out, int row,        \
      int tokens, int seqs, int shape, int slots, float scale) {                                                                              \
    delta_scan_body<W>(v, keys, work, state, slot, cu_q, out, row, tokens, seqs, shape, slots, scale);                                        \
  }
DELTA_SCAN(2)
DELTA_SCAN(4)

extern "C" __global__ __launch_bounds__(BLOCK_THREADS) void block_copy(unsigned char *__restrict__ a, unsigned char *__restrict__ b, const int *__restrict__ src,
                                                             const int *__restrict__ dst, long long a_bytes, long long b_bytes, int blocks) {
  block_copy_body(a, b, src, dst, a_bytes, b_bytes, blocks);
}
