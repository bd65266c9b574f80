// The gated delta rule a row at a time (delta_common.h has the formulas): single tokens, drafted ones, and any call without a workspace.
//
// One workgroup: a value head of a sequence; a wave has C columns of the state in registers, lane (dg, cq) the columns 4 cq .. 4 cq + 3 of the
// key's channels 256 / C j + dg, so that its loads are rows of 4 C bytes. Both sums of a row are taken of the
// state before it, so that they share the exchanges:
//   past = decay S, u = beta (v - decay S^T k^), o = scale (decay S^T q^ + (k^ . q^) u), S <- past + k^ u^T
// Rows are taken eight at a time, one or two a wave, normed, into LDS, their gates by the last wave; the first eight are asked for before the state. Bound by the state, read and written
// once (64 sequences of a row, 48 heads: 76 us, 5.3 TB/s in and out), and with few sequences by a row's chain, about a microsecond.
//
// kept: the state behind the first kept[s] rows is the one that is stored (no table: behind all; 0: none); the rows behind them are still
// answered. Without `out` only the state is made.
#pragma once
#include "delta_common.h"

template <int X>
static __device__ __forceinline__ float dn_dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), X, 0xF, 0xF, false));
}
// The sum over the lanes that hold the same columns: those that differ from bit log2(CQ) on.
template <int CQ>
static __device__ __forceinline__ float dn_sum_keys(float v) {
  if constexpr (CQ <= 4) v += dn_dpp<0x124>(v);  // row_ror:4
  v += dn_dpp<0x128>(v);                         // row_ror:8
  return at_both<32>(at_both<16>(v, at_sum2), at_sum2);
}
static __device__ __forceinline__ float dn_sum64(float v) {
  v += dn_dpp<0xB1>(v);   // lane ^ 1
  v += dn_dpp<0x4E>(v);   // lane ^ 2
  v += dn_dpp<0x141>(v);  // half rows mirrored
  v += dn_dpp<0x140>(v);  // rows mirrored
  return at_both<32>(at_both<16>(v, at_sum2), at_sum2);
}

template <int C>
static __device__ __forceinline__ void delta_step_body(const unsigned short *__restrict__ q, const unsigned short *__restrict__ k,
                                                       const unsigned short *__restrict__ v, const unsigned short *__restrict__ a,
                                                       const unsigned short *__restrict__ b, const float *__restrict__ a_log,
                                                       const float *__restrict__ dt_bias, float *__restrict__ state, const int *__restrict__ slot,
                                                       const int *__restrict__ cu, const int *__restrict__ kept, unsigned short *__restrict__ out,
                                                       int row, int ab_row, int tokens, int seqs, int shape, int slots, float eps, float scale) {
  constexpr int WAVES = DN / C, BATCH = 8, MINE = BATCH / WAVES, CQ = C / 4, DG = 64 / CQ, J = DN / DG, PAD = J + 4;
  const int heads = shape & 0xFFFF, group = heads / (shape >> 16);
  const int s = blockIdx.x / heads, h = blockIdx.x - s * heads, hk = h / group;
  const int lane = threadIdx.x & 63, wave = at_uniform(threadIdx.x >> 6), dg = lane / CQ, cq = lane % CQ, column = C * wave + 4 * cq;
  dn_rows x = dn_sequence(cu, slot, s, tokens, slots);
  if (x.n <= 0) return;
  const int hold = kept ? min(max(kept[s], 0), x.n) : x.n;
  if (!out) x.n = hold;
  if (x.n <= 0) return;
  __shared__ __attribute__((aligned(16))) float s_k[BATCH][DG][PAD], s_q[BATCH][DG][PAD];
  __shared__ float s_g[BATCH], s_b[BATCH];
  __shared__ __attribute__((aligned(8))) iu8_v2f s_kq[BATCH];  // k^ . q^; what the decays held back may fall to
  __shared__ __attribute__((aligned(16))) unsigned s_v[BATCH][64];

  unsigned kk[MINE], qq[MINE], vv[MINE];
  unsigned short aa = 0, bb = 0;  // the last wave's: a row's gates a lane
  auto fetch = [&](int base) {
#pragma unroll
    for (int y = 0; y < MINE; ++y) {
      const size_t t = x.t0 + min(base + y * WAVES + wave, x.n - 1);
      kk[y] = *(const unsigned *)(k + t * row + hk * DN + 2 * lane);
      qq[y] = out ? *(const unsigned *)(q + t * row + hk * DN + 2 * lane) : 0u;
      vv[y] = *(const unsigned *)(v + t * row + h * DN + 2 * lane);
    }
    if (wave == WAVES - 1) {
      const size_t t = x.t0 + min(base + (lane & (BATCH - 1)), x.n - 1);
      aa = a[t * ab_row + h], bb = b[t * ab_row + h];
    }
  };
  fetch(0);
  const float al = a_log[h], dt = dt_bias[h];
  float *mine = state + ((size_t)x.slot * heads + h) * (DN * DN) + column;
  iu8_v4f st[J];
#pragma unroll
  for (int j = 0; j < J; ++j) st[j] = __builtin_nontemporal_load((const iu8_v4f *)(mine + (DG * j + dg) * DN));

  // The state is `kept_by` times what the registers hold: a row's decay is a factor of one number, not of 128, until that is small, or
  // values come that 2^16 of would bring near f32's range.
  float kept_by = 1.f;
  for (int base = 0; base < x.n; base += BATCH) {
    const int count = min(BATCH, x.n - base);
    if (base) {
      fetch(base);
      __syncthreads();
    }
#pragma unroll
    for (int y = 0; y < MINE; ++y) {
      const int i = y * WAVES + wave;
      if (i >= count) break;
      const float k0 = __uint_as_float(kk[y] << 16), k1 = __uint_as_float(kk[y] & 0xFFFF0000u), q0 = __uint_as_float(qq[y] << 16), q1 = __uint_as_float(qq[y] & 0xFFFF0000u);
      const float rk = dn_inverse_root(dn_sum64(fmaf(k0, k0, k1 * k1)) + eps), rq = scale * dn_inverse_root(dn_sum64(fmaf(q0, q0, q1 * q1)) + eps);
      const float kq = dn_sum64(fmaf(k0, q0, k1 * q1));
      s_v[i][lane] = vv[y];
      const int c = 2 * lane;  // channel DG j + dg lies at [dg][j]
      s_k[i][c % DG][c / DG] = k0 * rk, s_k[i][c % DG + 1][c / DG] = k1 * rk;
      s_q[i][c % DG][c / DG] = q0 * rq, s_q[i][c % DG + 1][c / DG] = q1 * rq;
      const bool large = __any((vv[y] & 0x7F80u) >= 0x7180u || (vv[y] & 0x7F800000u) >= 0x71800000u);  // (from 2^100 on)
      if (lane == 0) s_kq[i] = iu8_v2f{kq * rk * rq, large ? 2.f : 0x1p-16f};
    }
    if (wave == WAVES - 1 && lane < BATCH) s_g[lane] = expf(dn_log_decay(iu8_bf16_f32(aa), al, dt)), s_b[lane] = dn_beta(iu8_bf16_f32(bb));
    __syncthreads();
    for (int i = 0; i < count; ++i) {
      const iu8_v2u now = *(const iu8_v2u *)&s_v[i][column / 2];
      float kr[J];
      iu8_v4f sk = {0.f, 0.f, 0.f, 0.f}, sq = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < J; j += 4) {
        const iu8_v4f y = *(const iu8_v4f *)&s_k[i][dg][j], z = *(const iu8_v4f *)&s_q[i][dg][j];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          kr[j + e] = y[e];
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) sk[cc] = fmaf(st[j + e][cc], y[e], sk[cc]), sq[cc] = fmaf(st[j + e][cc], z[e], sq[cc]);
        }
      }
      const iu8_v2f and_least = s_kq[i];
      const float g = kept_by * s_g[i], be = s_b[i], kq = and_least[0];
      const float vf[4] = {__uint_as_float(now[0] << 16), __uint_as_float(now[0] & 0xFFFF0000u), __uint_as_float(now[1] << 16), __uint_as_float(now[1] & 0xFFFF0000u)};
      float u[4], o[4];
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) {
        u[cc] = be * fmaf(-g, dn_sum_keys<CQ>(sk[cc]), vf[cc]);
        o[cc] = fmaf(g, dn_sum_keys<CQ>(sq[cc]), kq * u[cc]);
      }
      if (out && dg == 0)
        *(iu8_v2u *)(out + ((size_t)(x.t0 + base + i) * heads + h) * DN + column) = iu8_v2u{iu8_bf16_pack(o[0], o[1]), iu8_bf16_pack(o[2], o[3])};
      kept_by = at_uniform_f(g);
      if (__any(!(g > and_least[1])) || base + i + 1 == hold) {
#pragma unroll
        for (int j = 0; j < J; ++j) st[j] *= kept_by;
        kept_by = 1.f;
      }
      const float per = 1.f / kept_by;
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) u[cc] *= per;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) st[j][cc] = fmaf(kr[j], u[cc], st[j][cc]);
      if (base + i + 1 == hold) {
#pragma unroll
        for (int j = 0; j < J; ++j) __builtin_nontemporal_store(st[j], (iu8_v4f *)(mine + (DG * j + dg) * DN));
      }
    }
  }
}
