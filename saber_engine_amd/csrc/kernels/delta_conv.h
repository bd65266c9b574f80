// The short causal convolution in front of the delta rule, a channel by itself, and its SiLU:
//   y[t, c] = bias[c] + sum_w weight[c, w] x[t - W + 1 + w, c],   out = y sigmoid(y)
// in f32, rounded once. What lies in front of a sequence's first row is its tail, bf16 [slots][W - 1][channels], the oldest input first;
// the last W - 1 inputs of its first `kept` rows (all, without a table) are the new tail.
//
// Bound by the bytes, rows in and out (6,812 rows of 10,240 channels: 53 us, 5.2 TB/s; stored past the caches a tenth less
// by itself, but then the rule behind it waits for the rows: both together 240 us against 237). A thread takes 8 channels of `run` rows, the inputs that a row shares with the next kept in
// registers, four rows on the way at once. A tail is read and written by one thread alone: rows that see it (a sequence's first W - 1) belong to
// the run of the sequence's first row, also past that run's end.
#pragma once
#include "delta_common.h"

template <int W>
static __device__ __forceinline__ void delta_conv_body(const unsigned short *__restrict__ x, const unsigned short *__restrict__ weight,
                                                       const unsigned short *__restrict__ bias, unsigned short *__restrict__ tail,
                                                       const int *__restrict__ slot, const int *__restrict__ cu, const int *__restrict__ kept,
                                                       unsigned short *__restrict__ out, int x_row, int out_row, int tokens, int seqs, int channels,
                                                       int slots, int run) {
  constexpr int B = W - 1;
  const int groups = channels / 8, per = (groups + 255) / 256;
  const int part = blockIdx.x / per, group = (blockIdx.x - part * per) * 256 + (int)threadIdx.x;
  const int from = part * run, to = min(from + run, tokens);
  int s = from, first = from;  // the sequence that row `from` belongs to (or the next one), its first row
  if (cu) {
    s = at_find(cu, seqs, from);
    if (s >= seqs) return;  // behind the last sequence
    first = cu[s];
  }
  if (group >= groups) return;
  const int c = group * 8;
  float w[W][8], add[8];
  {
    union {
      iu8_v4u v[W];
      unsigned short h[8 * W];
    } raw;
#pragma unroll
    for (int i = 0; i < W; ++i) raw.v[i] = *(const iu8_v4u *)(weight + (size_t)c * W + i * 8);
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) w[i][j] = iu8_bf16_f32(raw.h[j * W + i]);
    iu8_v4u b = {0, 0, 0, 0};
    if (bias) b = *(const iu8_v4u *)(bias + c);
#pragma unroll
    for (int j = 0; j < 8; ++j) add[j] = __uint_as_float(j & 1 ? b[j / 2] & 0xFFFF0000u : b[j / 2] << 16);
  }
  auto input = [&](int t) { return *(const iu8_v4u *)(x + (size_t)t * x_row + c); };
  iu8_v4u back[B];  // the inputs in front of the next row, the oldest first
  auto row = [&](int t, iu8_v4u now) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = add[j];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const iu8_v4u v = i < B ? back[i < B ? i : 0] : now;
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = fmaf(w[i][j], __uint_as_float(j & 1 ? v[j / 2] & 0xFFFF0000u : v[j / 2] << 16), y[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] *= __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(y[j] * -1.44269504088896340736f));
    *(iu8_v4u *)(out + (size_t)t * out_row + c) =
        iu8_v4u{iu8_bf16_pack(y[0], y[1]), iu8_bf16_pack(y[2], y[3]), iu8_bf16_pack(y[4], y[5]), iu8_bf16_pack(y[6], y[7])};
#pragma unroll
    for (int i = 0; i + 1 < B; ++i) back[i] = back[i + 1];
    back[B - 1] = now;
  };

  int t = max(from, first);
  while (t < to) {
    // sequence s, whose row t is the first of this part
    const int end = cu ? min(cu[s + 1], tokens) : t + 1, place = slot ? slot[s] : s;
    const bool here = (unsigned)place < (unsigned)slots && first >= 0;
    unsigned short *mine = tail + (size_t)(here ? place : 0) * B * channels + c;
    if (here && t < end) {
      int stop = min(end, to);
      if (t == first) {
        stop = min(end, max(stop, first + B));
#pragma unroll
        for (int i = 0; i < B; ++i) back[i] = *(const iu8_v4u *)(mine + (size_t)i * channels);
        const int n = end - first, k = kept ? min(max(kept[s], 0), n) : n;
        if (k > 0) {  // the new tail: inputs k - B .. k - 1, those before 0 the old tail's
          iu8_v4u next[B];
#pragma unroll
          for (int i = 0; i < B; ++i) {
            const int at = k - B + i;
            if (at >= 0) {
              next[i] = input(first + at);
            } else {
              next[i] = back[B - 1];
#pragma unroll
              for (int j = 0; j < B; ++j) next[i] = at + B == j ? back[j] : next[i];
            }
          }
#pragma unroll
          for (int i = 0; i < B; ++i) *(iu8_v4u *)(mine + (size_t)i * channels) = next[i];
        }
      } else {
        if (t - first < B) t = min(first + B, stop);  // the run of the sequence's first row has them
        if (t < stop) {
#pragma unroll
          for (int i = 0; i < B; ++i) back[i] = input(t - B + i);
        }
      }
      for (; t + 4 <= stop; t += 4) {
        iu8_v4u v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = input(t + i);
#pragma unroll
        for (int i = 0; i < 4; ++i) row(t + i, v[i]);
      }
      for (; t < stop; ++t) row(t, input(t));
    }
    if (!cu) {
      first = t = ++s;
    } else {
      do ++s;
      while (s < seqs && cu[s + 1] <= cu[s]);
      if (s >= seqs) return;
      first = cu[s], t = max(first, from);
    }
  }
}
