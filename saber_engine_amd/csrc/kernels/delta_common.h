// Shared device helpers of a delta-net layer's core: the short causal convolution, the gated delta rule, the copies of a sequence.
//
// THE RULE, a value head's state S f32 [128 of the key][128 of the value], key head h / (heads / key_heads):
//   k^ = k / sqrt(|k|^2 + eps), q^ likewise, decay = exp(-exp(a_log) softplus(a + dt_bias)), beta = sigmoid(b)
//   S <- decay S + k^ (beta (v - (decay S)^T k^))^T,   o = scale S^T q^
// States lie [slots][heads][128][128], sequence s's in slot[s] (no table: s); a slot outside the pool: the sequence is passed over.
#pragma once
#include "attn_common.h"

constexpr int DN = 128;         // a head's keys, and its values
constexpr int DN_CHUNK = 64;    // rows that the chunked form takes at once
// exp(-120) is no f32: a decay stronger than that is the same zero, and sums of such logarithms keep the digits of the others
constexpr float DN_LEAST = -120.f;

struct dn_rows {
  int s, t0, n, slot;  // a sequence, its first row, its rows (of `tokens`), its slot
};

// Sequence s of packed rows (cu), or row s alone; n <= 0 where there is nothing to do.
static __device__ __forceinline__ dn_rows dn_sequence(const int *__restrict__ cu, const int *__restrict__ slot, int s, int tokens, int slots) {
  dn_rows x;
  x.s = s;
  x.t0 = cu ? cu[s] : s;
  x.n = (cu ? min(cu[s + 1], tokens) : min(s + 1, tokens)) - x.t0;
  x.slot = slot ? slot[s] : s;
  if (x.t0 < 0 || (unsigned)x.slot >= (unsigned)slots) x.n = 0;
  return x;
}

// The logarithm of a row's decay, and its beta.
static __device__ __forceinline__ float dn_log_decay(float a, float a_log, float dt_bias) {
  const float x = a + dt_bias, g = -expf(a_log) * (x > 20.f ? x : log1pf(expf(x)));
  return g < DN_LEAST ? DN_LEAST : g;
}
static __device__ __forceinline__ float dn_beta(float b) { return 1.f / (1.f + expf(-b)); }

// f32 as a sum of bf16: the first N terms, 8 bits of the mantissa each (three are all 24), of a pair of values at a time.
template <int N>
static __device__ __forceinline__ void dn_split(float x, float y, unsigned (&t)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    t[i] = iu8_bf16_pack(x, y);
    x -= __uint_as_float(t[i] << 16), y -= __uint_as_float(t[i] & 0xFFFF0000u);
  }
}
// Two result blocks of a 16 x 16 product, rows 4 g + r of each, as the N terms of the next product's operand: its eight places
// are the first block's rows 4 g .. 4 g + 3, then the second's.
template <int N>
static __device__ __forceinline__ void dn_operand(iu8_v4f a, iu8_v4f b, iu8_v4u (&t)[N]) {
  unsigned x[4][N];
  dn_split<N>(a[0], a[1], x[0]), dn_split<N>(a[2], a[3], x[1]), dn_split<N>(b[0], b[1], x[2]), dn_split<N>(b[2], b[3], x[3]);
#pragma unroll
  for (int i = 0; i < N; ++i) t[i] = iu8_v4u{x[0][i], x[1][i], x[2][i], x[3][i]};
}
static __device__ __forceinline__ iu8_v4f dn_mfma(iu8_v4u a, iu8_v4u b, iu8_v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(at_bf(a), at_bf(b), c, 0, 0, 0);
}
// A matrix instruction's result, read in the block that makes it (attn_few.h has why).
static __device__ __forceinline__ void dn_settle(iu8_v4f &x) { asm volatile("" : "+v"(x)); }
