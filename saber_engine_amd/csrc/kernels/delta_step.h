// The gated delta rule a row at a time (delta_common.h has the formulas): single tokens, drafted ones, and any call without a workspace.
//
// One workgroup: a value head of a sequence; a wave has 32 columns of the state in registers, lane (dg, cq) the columns 4 cq .. 4 cq + 3 of the
// key's channels 8 j + dg: whole 128-byte lines on the way in and out, and three exchanges a sum over the keys. Both sums of a row are taken of the
// state before it, so that they share the exchanges:
//   past = decay S, u = beta (v - decay S^T k^), o = scale (decay S^T q^ + (k^ . q^) u), S <- past + k^ u^T
// Rows are normed eight at a time, two a wave, into LDS. Bound by the state, read and written once.
//
// kept: the state behind the first kept[s] rows is the one that is stored (no table: behind all; 0: none); the rows behind them are still
// answered. Without `out` only the state is made.
#pragma once
#include "delta_common.h"

static __device__ __forceinline__ float dn_sum8(float v) {  // over the lanes that differ in bits 3 to 5
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, false));  // row_ror:8
  return at_both<32>(at_both<16>(v, at_sum2), at_sum2);
}
static __device__ __forceinline__ float dn_sum64(float v) {
#pragma unroll
  for (int x = 1; x < 64; x *= 2) v += __shfl_xor(v, x);
  return v;
}

static __device__ __forceinline__ void delta_step_body(const unsigned short *__restrict__ q, const unsigned short *__restrict__ k,
                                                       const unsigned short *__restrict__ v, const unsigned short *__restrict__ a,
                                                       const unsigned short *__restrict__ b, const float *__restrict__ a_log,
                                                       const float *__restrict__ dt_bias, float *__restrict__ state, const int *__restrict__ slot,
                                                       const int *__restrict__ cu, const int *__restrict__ kept, unsigned short *__restrict__ out,
                                                       int row, int ab_row, int tokens, int seqs, int shape, int slots, float eps, float scale) {
  constexpr int BATCH = 8, PAD = 20;
  const int heads = shape & 0xFFFF, group = heads / (shape >> 16);
  const int s = blockIdx.x / heads, h = blockIdx.x - s * heads, hk = h / group;
  const int lane = threadIdx.x & 63, wave = at_uniform(threadIdx.x >> 6), dg = lane >> 3, cq = lane & 7;
  dn_rows x = dn_sequence(cu, slot, s, tokens, slots);
  if (x.n <= 0) return;
  const int hold = kept ? min(max(kept[s], 0), x.n) : x.n;
  if (!out) x.n = hold;
  if (x.n <= 0) return;
  __shared__ __attribute__((aligned(16))) float s_k[BATCH][8][PAD], s_q[BATCH][8][PAD];
  __shared__ float s_g[BATCH], s_b[BATCH], s_kq[BATCH];

  float *mine = state + ((size_t)x.slot * heads + h) * (DN * DN) + 32 * wave + 4 * cq;
  iu8_v4f st[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) st[j] = *(const iu8_v4f *)(mine + (8 * j + dg) * DN);
  const float al = a_log[h], dt = dt_bias[h];
  auto store = [&]() {
#pragma unroll
    for (int j = 0; j < 16; ++j) *(iu8_v4f *)(mine + (8 * j + dg) * DN) = st[j];
  };

  for (int base = 0; base < x.n; base += BATCH) {
    const int count = min(BATCH, x.n - base);
    if (base) __syncthreads();
    for (int i = wave; i < count; i += 4) {
      const size_t t = x.t0 + base + i;
      const unsigned kk = *(const unsigned *)(k + t * row + hk * DN + 2 * lane);
      const unsigned qq = out ? *(const unsigned *)(q + t * row + hk * DN + 2 * lane) : 0u;
      const float k0 = __uint_as_float(kk << 16), k1 = __uint_as_float(kk & 0xFFFF0000u), q0 = __uint_as_float(qq << 16), q1 = __uint_as_float(qq & 0xFFFF0000u);
      const float rk = 1.f / sqrtf(dn_sum64(fmaf(k0, k0, k1 * k1)) + eps), rq = scale / sqrtf(dn_sum64(fmaf(q0, q0, q1 * q1)) + eps);
      const float kq = dn_sum64(fmaf(k0, q0, k1 * q1));
      const int c = 2 * lane;  // channel 8 j + dg lies at [dg][j]
      s_k[i][c & 7][c >> 3] = k0 * rk, s_k[i][(c & 7) + 1][c >> 3] = k1 * rk;
      s_q[i][c & 7][c >> 3] = q0 * rq, s_q[i][(c & 7) + 1][c >> 3] = q1 * rq;
      if (lane == 0) {
        s_g[i] = expf(dn_log_decay(iu8_bf16_f32(a[t * ab_row + h]), al, dt));
        s_b[i] = dn_beta(iu8_bf16_f32(b[t * ab_row + h]));
        s_kq[i] = kq * rk * rq;
      }
    }
    __syncthreads();
    iu8_v2u vv = *(const iu8_v2u *)(v + (size_t)(x.t0 + base) * row + h * DN + 32 * wave + 4 * cq);
    for (int i = 0; i < count; ++i) {
      const iu8_v2u now = vv;
      if (i + 1 < count) vv = *(const iu8_v2u *)(v + (size_t)(x.t0 + base + i + 1) * row + h * DN + 32 * wave + 4 * cq);
      float kr[16];
      iu8_v4f sk = {0.f, 0.f, 0.f, 0.f}, sq = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const iu8_v4f y = *(const iu8_v4f *)&s_k[i][dg][j], z = *(const iu8_v4f *)&s_q[i][dg][j];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          kr[j + e] = y[e];
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) sk[cc] = fmaf(st[j + e][cc], y[e], sk[cc]), sq[cc] = fmaf(st[j + e][cc], z[e], sq[cc]);
        }
      }
      const float g = s_g[i], be = s_b[i], kq = s_kq[i];
      const float vf[4] = {__uint_as_float(now[0] << 16), __uint_as_float(now[0] & 0xFFFF0000u), __uint_as_float(now[1] << 16), __uint_as_float(now[1] & 0xFFFF0000u)};
      float u[4], o[4];
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) {
        u[cc] = be * fmaf(-g, dn_sum8(sk[cc]), vf[cc]);
        o[cc] = fmaf(g, dn_sum8(sq[cc]), kq * u[cc]);
      }
      if (out && dg == 0)
        *(iu8_v2u *)(out + ((size_t)(x.t0 + base + i) * heads + h) * DN + 32 * wave + 4 * cq) = iu8_v2u{iu8_bf16_pack(o[0], o[1]), iu8_bf16_pack(o[2], o[3])};
#pragma unroll
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) st[j][cc] = fmaf(kr[j], u[cc], g * st[j][cc]);
      if (base + i + 1 == hold) store();
    }
  }
}
