// New tokens into the paged cache: per-head norm (optional) and position rotation of q and k, k and v to their pages.
//
//   y = x * 1/sqrt(mean(x^2) + eps) * (1 + w)          (w given; over the head's D channels)
//   (a, b) -> (a cos - b sin, b cos + a sin), angle = position * inv_freq[i], over the first `rot` channels: channels i and
//   i + rot/2, or 2i and 2i + 1
// all in f32, rounded once: to bf16 (q, k, v) or, k and v divided by their head's scale, to e4m3 (nearest even, saturating at 448).
//
// The angle: turns = position * (inv_freq / 2 pi) in f64, its fraction in f32 (the error of the fraction is 2^-25 of a turn at any
// position), then the hardware's sine and cosine of turns, 1.3e-7 at most from the function over all of [-1/2, 1/2] (measured),
// a 30,000th of what the rounding to bf16 leaves.
//
// Bound by the bytes (rows in, rows and pages out), and with few tokens by the launch. A lane owns 16 channels of one head: two
// pieces of 8 that the rotation pairs, so a pair never crosses lanes. Measured: 6,772 tokens of 40 + 2 x 8 heads of 128 channels, 205 MB
// of rows, 44 us (4.65 TB/s; a device copy reaches 4.9), up to 1,500 of 7 prompts into e4m3 39.8 (4.5); 64 tokens of 24 + 2 x 4 heads of 256 into e4m3
// 4.1 us, one token 3.1.
#pragma once
#include "attn_common.h"

// The quotient from the reciprocal, one of a head, and the remainder's correction (Markstein's: q + (x - q scale) / scale, each an fma), two operations
// more than the product with the reciprocal, which is rounded twice on the way to the quotient and moved 26 of a million stored values of
// bf16 rows at a scale of 0.3 to a neighbour. The remainder is taken the other way round and subtracted, which leaves a zero its sign. `most` is 448 scales,
// within a rounding: x is bounded first, by operations that keep a NaN, so that an infinity leaves none in the remainder.
static __device__ __forceinline__ unsigned at_e4m3x4(const float *x, float scale, float inv, float most) {
#pragma clang fp contract(off)
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float b = __builtin_elementwise_minimum(__builtin_elementwise_maximum(x[i], -most), most), q = b * inv;
    y[i] = fmaf(-fmaf(q, scale, -b), inv, q);
  }
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], r, true);
}

// `form`: bits 0-7 log2 of the page's tokens, bit 8 the interleaved pairing, bits 16.. the rotated channels.
template <int D, bool F8>
static __device__ __forceinline__ void kv_append_body(
    const unsigned short *__restrict__ q, const unsigned short *__restrict__ k, const unsigned short *__restrict__ v,
    unsigned short *__restrict__ q_out, unsigned char *__restrict__ kc, unsigned char *__restrict__ vc, const float *__restrict__ k_scale,
    const float *__restrict__ v_scale, const int *__restrict__ table, const int *__restrict__ kv_len, const int *__restrict__ cu_q,
    const unsigned short *__restrict__ q_norm, const unsigned short *__restrict__ k_norm, const double *__restrict__ inv_freq, int q_row,
    int q_head, int kv_row, int tokens, int seqs, int shape, int form, int pages, int table_stride, float eps) {
  constexpr int TPH = D / 16, HPW = 64 / TPH;  // lanes a head, heads a wave
  const int heads = shape & 0xFFFF, kv_heads = shape >> 16, page_shift = form & 0xFF, rot = form >> 16;
  const bool interleaved = form & 0x100;
  const int rows = heads + 2 * kv_heads, wpt = (rows + HPW - 1) / HPW;
  const int lane = threadIdx.x & 63, u = lane % TPH;
  const int wave = at_uniform(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int t = wave / wpt, hr = (wave - t * wpt) * HPW + lane / TPH;
  if (t >= tokens) return;
  int s = t, pos;
  if (cu_q) {
    s = at_find(cu_q, seqs, t);
    if (s >= seqs || t < cu_q[s]) return;  // behind the last sequence, in front of the first
    pos = at_len(kv_len, s, table_stride, page_shift) - (cu_q[s + 1] - t);
  } else {
    pos = at_len(kv_len, s, table_stride, page_shift) - 1;
  }
  if (pos < 0 || hr >= rows) return;

  // the lane's two pieces of 8 channels: the rotation's partners, behind them neighbours
  int c0 = 2 * u, c1 = 2 * u + 1;
  if (!interleaved && u < rot / 16) c0 = u, c1 = u + rot / 16;
  const bool is_q = hr < heads, is_v = hr >= heads + kv_heads;
  const int h = is_q ? hr : is_v ? hr - heads - kv_heads : hr - heads;
  const unsigned short *src = is_q ? q + (size_t)t * q_row + (size_t)h * q_head : (is_v ? v : k) + (size_t)t * kv_row + (size_t)h * D;
  const iu8_v4u r0 = *(const iu8_v4u *)(src + c0 * 8), r1 = *(const iu8_v4u *)(src + c1 * 8);
  const bool rotates = !is_v && 8 * c0 < rot;
  double f[8];
  if (rotates) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = inv_freq[interleaved ? 8 * u + i : 8 * c0 + i];
  }
  int page = -1;
  const int o = pos & ((1 << page_shift) - 1);
  if (!is_q && (pos >> page_shift) < table_stride) page = table[(size_t)s * table_stride + (pos >> page_shift)];
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[2 * i] = __uint_as_float(r0[i] << 16), a[2 * i + 1] = __uint_as_float(r0[i] & 0xFFFF0000u);
    b[2 * i] = __uint_as_float(r1[i] << 16), b[2 * i + 1] = __uint_as_float(r1[i] & 0xFFFF0000u);
  }
  const unsigned short *w = is_q ? q_norm : is_v ? nullptr : k_norm;
  if (q_norm || k_norm) {  // (a wave may hold heads of both kinds: every lane takes part in the exchange)
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
#pragma unroll
    for (int x = 1; x < TPH; x *= 2) ss += __shfl_xor(ss, x);
    if (w) {
      const float inv = 1.f / sqrtf(ss * (1.f / D) + eps);
      const iu8_v4u w0 = *(const iu8_v4u *)(w + c0 * 8), w1 = *(const iu8_v4u *)(w + c1 * 8);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[2 * i] = a[2 * i] * inv * (1.f + __uint_as_float(w0[i] << 16));
        a[2 * i + 1] = a[2 * i + 1] * inv * (1.f + __uint_as_float(w0[i] & 0xFFFF0000u));
        b[2 * i] = b[2 * i] * inv * (1.f + __uint_as_float(w1[i] << 16));
        b[2 * i + 1] = b[2 * i + 1] * inv * (1.f + __uint_as_float(w1[i] & 0xFFFF0000u));
      }
    }
  }
  if (rotates) {
    float cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double turns = (double)pos * (f[i] * 0.15915494309189533577);
      const float x = (float)(turns - __builtin_rint(turns));
      cs[i] = __builtin_amdgcn_cosf(x), sn[i] = __builtin_amdgcn_sinf(x);
    }
    if (interleaved) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = a[2 * i], y = a[2 * i + 1];
        a[2 * i] = x * cs[i] - y * sn[i], a[2 * i + 1] = y * cs[i] + x * sn[i];
        const float z = b[2 * i], t2 = b[2 * i + 1];
        b[2 * i] = z * cs[4 + i] - t2 * sn[4 + i], b[2 * i + 1] = t2 * cs[4 + i] + z * sn[4 + i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = a[i], y = b[i];
        a[i] = x * cs[i] - y * sn[i], b[i] = y * cs[i] + x * sn[i];
      }
    }
  }
  auto pack = [](const float *x) { return iu8_v4u{iu8_bf16_pack(x[0], x[1]), iu8_bf16_pack(x[2], x[3]), iu8_bf16_pack(x[4], x[5]), iu8_bf16_pack(x[6], x[7])}; };
  if (is_q) {
    unsigned short *dst = q_out + ((size_t)t * heads + h) * D;
    *(iu8_v4u *)(dst + c0 * 8) = pack(a);
    *(iu8_v4u *)(dst + c1 * 8) = pack(b);
    return;
  }
  if ((unsigned)page >= (unsigned)pages) return;  // a hole
  const size_t base = (((size_t)page * kv_heads + h) << page_shift) * D;
  auto at = [&](int c) -> size_t {  // the element that piece c (8 channels) of this token starts at
    if (is_v) return base + (size_t)o * D + c * 8;
    const size_t block = base + (size_t)(o >> 4) * 16 * D;
    return F8 ? block + ((c >> 1) * 16 + (o & 15)) * 16 + (c & 1) * 8 : block + (c * 16 + (o & 15)) * 8;
  };
  unsigned char *dst = is_v ? vc : kc;
  if constexpr (F8) {
    const float by = (is_v ? v_scale : k_scale)[h], inv = 1.f / by, most = 448.f * fabsf(by);
    *(iu8_v2u *)(dst + at(c0)) = iu8_v2u{at_e4m3x4(a, by, inv, most), at_e4m3x4(a + 4, by, inv, most)};
    *(iu8_v2u *)(dst + at(c1)) = iu8_v2u{at_e4m3x4(b, by, inv, most), at_e4m3x4(b + 4, by, inv, most)};
  } else {
    *(iu8_v4u *)(dst + 2 * at(c0)) = pack(a);
    *(iu8_v4u *)(dst + 2 * at(c1)) = pack(b);
  }
}
