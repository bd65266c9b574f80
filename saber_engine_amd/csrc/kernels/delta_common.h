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
static __device__ __forceinline__ dn_rows dn_rows_of(int s, int t0, int end, int place, int tokens, int slots) {
  dn_rows x;
  x.s = s, x.t0 = t0, x.slot = place;
  x.n = min(end, tokens) - t0;
  if (t0 < 0 || (unsigned)place >= (unsigned)slots) x.n = 0;
  return x;
}
static __device__ __forceinline__ dn_rows dn_sequence(const int *__restrict__ cu, const int *__restrict__ slot, int s, int tokens, int slots) {
  return dn_rows_of(s, cu ? cu[s] : s, cu ? cu[s + 1] : s + 1, slot ? slot[s] : s, tokens, slots);
}

// The logarithm of a row's decay, and its beta. (Far below 0 softplus is the exponential, and one exponential of the sum is taken: by themselves the factors may be
// infinite and 0. An infinite sum of a and dt_bias stands for f32's largest number.)
static __device__ __forceinline__ float dn_log_decay(float a, float a_log, float dt_bias) {
  const float x = a + dt_bias, g = -expf(x < -20.f ? a_log + x : a_log) * (x < -20.f ? 1.f : x > 20.f ? (x < INFINITY ? x : 0x1.fffffep127f) : log1pf(expf(x)));
  return g < DN_LEAST ? DN_LEAST : g;
}
static __device__ __forceinline__ float dn_beta(float b) { return 1.f / (1.f + expf(-b)); }

// 1 / sqrt(x) within a unit; v_rsq_f32 takes no subnormal.
static __device__ __forceinline__ float dn_inverse_root(float x) {
  return x < 0x1p-96f ? __builtin_amdgcn_rsqf(x * 0x1p64f) * 0x1p32f : __builtin_amdgcn_rsqf(x);
}

typedef _Float16 dn_v8h __attribute__((ext_vector_type(8)));
typedef _Float16 dn_v2h __attribute__((ext_vector_type(2)));

// f32 as a sum of f16: the first N terms (1 or 2), 11 bits each, of a pair of values (what two terms leave is 2^-22 of a value, and no less than half of f16's last
// step, 2^-25; the matrix instructions keep values below 2^-14). What the first leaves is exact, and rounded once: by the mixed multiply-adds, which take f16 and f32
// as they are and write a half, where conversion, subtraction and conversion are three. (-1 is hidden, so that a multiply-add stays; the first terms as well, so that
// they stay a pair.)
static __device__ __forceinline__ dn_v2h dn_pair(dn_v2h h) {
  unsigned w = __builtin_bit_cast(unsigned, h);
  asm("" : "+v"(w));
  return __builtin_bit_cast(dn_v2h, w);
}
static __device__ __forceinline__ unsigned dn_rounded(float x, float y) { return __builtin_bit_cast(unsigned, dn_v2h{(_Float16)x, (_Float16)y}); }
template <int N>
static __device__ __forceinline__ void dn_split(float x, float y, unsigned (&t)[N]) {
  float less;
  asm("s_mov_b32 %0, -1.0" : "=s"(less));
  const dn_v2h h = dn_pair(__builtin_convertvector(iu8_v2f{x, y}, dn_v2h));
  t[0] = __builtin_bit_cast(unsigned, h);
  if constexpr (N > 1) t[1] = dn_rounded(fmaf((float)h[0], less, x), fmaf((float)h[1], less, y));
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
static __device__ __forceinline__ iu8_v4f dn_mfma_bf(iu8_v4u a, iu8_v4u b, iu8_v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(at_bf(a), at_bf(b), c, 0, 0, 0);
}
static __device__ __forceinline__ iu8_v4f dn_mfma(iu8_v4u a, iu8_v4u b, iu8_v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(dn_v8h, a), __builtin_bit_cast(dn_v8h, b), c, 0, 0, 0);
}
// The power of two at or below |x| (x a number), and its reciprocal; both ordinary numbers.
static __device__ __forceinline__ int dn_exponent(float x) { return min(max((int)(__float_as_uint(x) >> 23 & 255u), 7), 247); }
static __device__ __forceinline__ float dn_power(int e) { return __uint_as_float((unsigned)e << 23); }
static __device__ __forceinline__ float dn_below(int e) { return __uint_as_float((unsigned)(254 - e) << 23); }
// A matrix instruction's result, read in the block that makes it (attn_few.h has why).
static __device__ __forceinline__ void dn_settle(iu8_v4f &x) { asm volatile("" : "+v"(x)); }
