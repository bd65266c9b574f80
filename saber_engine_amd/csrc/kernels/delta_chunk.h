// The gated delta rule in chunks of 64 rows (delta_common.h has the formulas): prompts.
//
// With G_i the sum of the logarithms of the decays of a chunk's rows 0 .. i, S0 the state in front of it, and
//   A_ij = beta_i exp(G_i - G_j) k^_i . k^_j (j < i),   T = (1 + A)^-1,
// the rows' updates u (the rule's beta (v - ...)) are the solution of a unit triangular system, and everything is matrix products:
//   U  = T diag(beta) (V - diag(exp G) K^ S0)
//   O  = scale (diag(exp G) Q^ S0 + [exp(G_i - G_j) q^_i . k^_j, j <= i] U)
//   S1 = exp(G_63) S0 + K^^T diag(exp(G_63 - G_j)) U
// Two kernels. delta_prep makes, for all chunks at once, T diag(beta) and the inner matrix of O, each already as the other's operand, the rows'
// factors, and K and Q as the walk reads them; delta_scan walks a sequence's chunks in order.
//
// Precision: the state and all that enters it is f32, on the f16 matrix cores. A row of K or Q, bf16 as it comes, is an f16 row times a power
// of two (the one at or below its length, so that no value passes 2); its norm's and decay's factors are moved to the other side of the product; the other side is split
// into two f16 terms, 22 bits (dn_split), in a column's own unit, a power of two that follows the column's largest value. What goes only into the rows' bf16 answers takes
// one term, 11 bits. Units: nothing is kept below 2^-26 of the largest value that a column has in a chunk and the one before.
// (Three bf16 terms, which need no units, are half as many products again and twice the lane arithmetic: the walk of 8,192 rows of 48 heads 304 us in a trace, with f16 221.) G is summed, and its differences taken, in f64: after a strong decay the later rows' differences would be left with the sum's digits.
#pragma once
#include "delta_step.h"

// The workspace: of a chunk and key head K and Q, f16, 16 KiB each, piece p (16 bytes) of row t where dn_turned(p) ^ (t % 4 * 4 + t / 4 % 4) says, as the walk keeps
// them in LDS: the 16 lanes that a wide read serves at once (of a quarter's fours 0 and 3, of the next one's 1 and 2) meet on no bank. Of a chunk and value
// head T diag(beta) in two terms, the inner matrix in one, the factors. Operands are kept as fragments, 64 lanes x 16 bytes: lane (l % 16, g = l / 16) has row l % 16 of 16 and the
// columns 4 g .. 4 g + 3 of the first and of the second 16 of 32, which is how a product's result lies (dn_operand).
// Fragment f of a lower triangle: row blocks 0, 1 of the first 32 columns; row blocks 2, 3 of the first and of the last.
static __host__ __device__ constexpr int dn_turned(int p) { return (p & ~3) | (-p & 3); }
constexpr int DN_KEYS = 32768, DN_FRAGS = 6, DN_FRAG = 1024;
static __host__ __device__ constexpr int dn_frag_block(int f) { return f < 2 ? f : 2 + (f - 2) / 2; }
static __host__ __device__ constexpr int dn_frag_half(int f) { return f < 2 ? 0 : (f - 2) & 1; }
constexpr int DN_T = 0, DN_INNER = 2 * DN_FRAGS * DN_FRAG, DN_FACTORS = DN_INNER + DN_FRAGS * DN_FRAG, DN_PART = DN_FACTORS + 1024;
// the factors, f32: [64] exp(G_i) / |k_i|, [64] exp(G_i) / |q_i|, [64] exp(G_63 - G_i) / |k_i| (of the f16 rows), exp(G_63)

static __device__ __forceinline__ int dn_chunk_id(const dn_rows &x) { return (x.t0 >> 6) + x.s; }  // of its first chunk: no two sequences' meet

// A step of a running sum over the lanes.
template <int X, int ROWS>
static __device__ __forceinline__ void dn_scan_step(double &v) {
  const iu8_v2u w = __builtin_bit_cast(iu8_v2u, v);
  v += __builtin_bit_cast(double, iu8_v2u{(unsigned)__builtin_amdgcn_update_dpp(0, (int)w[0], X, ROWS, 0xF, false), (unsigned)__builtin_amdgcn_update_dpp(0, (int)w[1], X, ROWS, 0xF, false)});
}
// What lane I of each 16 holds.
template <int I>
static __device__ __forceinline__ float dn_shared(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + I, 0xF, 0xF, false));
}
template <int I>
static __device__ __forceinline__ double dn_shared(double v) {
  const iu8_v2f w = __builtin_bit_cast(iu8_v2f, v);
  return __builtin_bit_cast(double, iu8_v2f{dn_shared<I>(w[0]), dn_shared<I>(w[1])});
}
// Column n of the inverse of 1 + F, F strictly below the diagonal, in y, which begins as the identity's: from y_J on, y_i -= F_iJ y_J. (asm: the compiler makes
// three instructions and a wait of it. f comes from LDS, so no lane operation has just written it.)
template <int J, int I = J + 1>
static __device__ __forceinline__ void dn_below_row(const float (&f)[16], float (&y)[16]) {
  if constexpr (I < 16) {
    asm("v_fmac_f32_dpp %0, -%1, %2 row_newbcast:%3 row_mask:0xf bank_mask:0xf" : "+v"(y[I]) : "v"(f[I]), "v"(y[J]), "n"(J));
    dn_below_row<J, I + 1>(f, y);
  } else if constexpr (J < 14) {
    dn_below_row<J + 1>(f, y);
  }
}

// Bound by what it moves and, a workgroup at a time, by the chain behind its loads: 8,192 rows of 16 and 48 heads, 67 MB in and 187 out, 59 us, a round
// of workgroups some 15.
static __device__ __forceinline__ void delta_prep_body(const unsigned short *__restrict__ q, const unsigned short *__restrict__ k,
                                                       const unsigned short *__restrict__ a, const unsigned short *__restrict__ b,
                                                       const float *__restrict__ a_log, const float *__restrict__ dt_bias,
                                                       const int *__restrict__ slot, const int *__restrict__ cu, unsigned char *__restrict__ keys,
                                                       unsigned char *__restrict__ work, int row, int ab_row, int tokens, int seqs, int shape, int slots,
                                                       int places, int many, float eps) {
  constexpr int P = 68;  // floats of a row in LDS
  const int heads = shape & 0xFFFF, key_heads = shape >> 16, group = heads / key_heads;
  // a workgroup: `many` value heads (1 to 4) of a key head; to one XCD those that read the same rows
  const int parts = (group + many - 1) / many, turn = (int)(blockIdx.x >> 3) / parts, item = turn * 8 + (int)(blockIdx.x & 7);
  if (item >= places * key_heads) return;
  const int id = item / key_heads, hk = item - id * key_heads, part = (int)(blockIdx.x >> 3) - turn * parts, h0 = hk * group + part * many;
  const int count = min(many, group - part * many);
  const int lane = threadIdx.x & 63, wave = at_uniform(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  // the sequence of place `id`: the last whose first place is not behind it
  dn_rows x;
  x.n = 0;
  for (int base = 0; base < seqs; base += 64) {
    const int i = min(base + lane, seqs - 1), from = cu[i], end = cu[i + 1], to = slot ? slot[i] : i;
    const int below = __popcll(__ballot(base + lane < seqs && (from >> 6) + i <= id));
    if (!below) break;
    x = dn_rows_of(base + below - 1, __builtin_amdgcn_readlane(from, below - 1), __builtin_amdgcn_readlane(end, below - 1), __builtin_amdgcn_readlane(to, below - 1),
                   tokens, slots);
  }
  if (x.n <= 0) return;
  const int c0 = (id - dn_chunk_id(x)) * DN_CHUNK, m = min(x.n - c0, DN_CHUNK);  // the chunk's first row, its rows
  if (c0 < 0 || m <= 0) return;

  // K and Q, 16 KiB each, then in their place of one head and the next A: blocks on the diagonal become T's, T's others stand in the block across it
  __shared__ __attribute__((aligned(16))) float s_m[2][DN_CHUNK][P];
  __shared__ __attribute__((aligned(16))) double s_sums[4][DN_CHUNK];  // in units of log 2
  __shared__ __attribute__((aligned(16))) float s_betas[4][DN_CHUNK], s_in[4][DN_CHUNK], s_past[4][DN_CHUNK], s_rk[DN_CHUNK], s_rq[DN_CHUNK];
  __shared__ int s_unit[DN_CHUNK];  // K's and Q's rows' units, as exponents
  unsigned char *s_k = (unsigned char *)s_m, *s_q = s_k + DN_KEYS / 2;

  // a row past the end is the last one again, and takes no part
  const size_t t0 = x.t0 + c0;
  iu8_v4u kr[4], qr[4];  // rows 16 wave + 4 i + lane / 16, piece lane % 16
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const size_t at = (t0 + min(16 * wave + 4 * i + g, m - 1)) * row + hk * DN + 8 * n;
    kr[i] = __builtin_nontemporal_load((const iu8_v4u *)(k + at)), qr[i] = __builtin_nontemporal_load((const iu8_v4u *)(q + at));
  }
  if (wave < count) {  // a head's gates a wave
    const int i = lane, h = h0 + wave;
    float lg = 0.f, be = 0.f;
    if (i < m) {
      lg = dn_log_decay(iu8_bf16_f32(a[(t0 + i) * ab_row + h]), a_log[h], dt_bias[h]);
      be = dn_beta(iu8_bf16_f32(b[(t0 + i) * ab_row + h]));
    }
    double sum = lg * 1.4426950408889634074;
    dn_scan_step<0x111, 0xF>(sum), dn_scan_step<0x112, 0xF>(sum), dn_scan_step<0x114, 0xF>(sum), dn_scan_step<0x118, 0xF>(sum);  // row_shr
    dn_scan_step<0x142, 0xA>(sum), dn_scan_step<0x143, 0xC>(sum);                                                            // row_bcast
    s_sums[wave][i] = sum, s_betas[wave][i] = be;
    // decays from the first of its 16 rows to it, from it to the last
    s_in[wave][i] = __builtin_amdgcn_exp2f((float)(sum - dn_shared<0>(sum))), s_past[wave][i] = __builtin_amdgcn_exp2f((float)(dn_shared<15>(sum) - sum));
  }
  const int turned = (dn_turned(n) ^ (g << 2)) << 4;  // piece n of row 16 wave + 4 i + g, ^ 16 i
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = (16 * wave + 4 * i + g) * 256 + (turned ^ (i << 4));
    *(iu8_v4u *)(s_k + at) = kr[i], *(iu8_v4u *)(s_q + at) = qr[i];
  }
  __syncthreads();
  // the products of the rows, row block `wave` with those up to it, and Q's with themselves; row i = 16 wave + n, rows j = 16 jb + 4 g + r in place r
  const int row_piece = n * 256 + ((dn_turned(g) ^ (n >> 2)) << 4);
  auto fragment = [&](const unsigned char *from, int rb, int ks) { return *(const iu8_v4u *)(from + rb * 4096 + row_piece + ((ks ^ (n & 3)) << 6)); };
  iu8_v4f kk[3], qk[3], own = {0.f, 0.f, 0.f, 0.f}, qq = own, across = own;  // own, across: block `wave` itself
  {
    iu8_v4u kf[4], qf[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) kf[ks] = fragment(s_k, wave, ks), qf[ks] = fragment(s_q, wave, ks);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) own = dn_mfma_bf(kf[ks], kf[ks], own), qq = dn_mfma_bf(qf[ks], qf[ks], qq), across = dn_mfma_bf(kf[ks], qf[ks], across);
    dn_settle(own), dn_settle(qq), dn_settle(across);
#pragma unroll
    for (int jb = 0; jb < 3; ++jb) {
      kk[jb] = qk[jb] = iu8_v4f{0.f, 0.f, 0.f, 0.f};
      if (jb < wave) {
        iu8_v4u f[4];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) f[ks] = fragment(s_k, jb, ks);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) kk[jb] = dn_mfma_bf(f[ks], kf[ks], kk[jb]), qk[jb] = dn_mfma_bf(f[ks], qf[ks], qk[jb]);
        dn_settle(kk[jb]), dn_settle(qk[jb]);
      }
    }
  }
  // |k|^2 and |q|^2 stand on the diagonals; a row's unit is the power of two at or below its length (so that no value passes 2; lengths whose squares
  // are no f32 count as 2^-63, below anything beside eps)
  if (g == n >> 2) {
    const float ks = (n & 2) ? ((n & 1) ? own[3] : own[2]) : ((n & 1) ? own[1] : own[0]), qs = (n & 2) ? ((n & 1) ? qq[3] : qq[2]) : ((n & 1) ? qq[1] : qq[0]);
    const bool live = 16 * wave + n < m;
    auto unit_of = [](float ss) { return max((dn_exponent(ss) + 127) >> 1, 64); };  // half the exponent
    s_rk[16 * wave + n] = live ? dn_inverse_root(ks + eps) : 0.f, s_rq[16 * wave + n] = live ? dn_inverse_root(qs + eps) : 0.f;
    s_unit[16 * wave + n] = unit_of(ks) | unit_of(qs) << 16;
  }
  __syncthreads();
  if (part == 0) {
    unsigned char *to = keys + ((size_t)id * key_heads + hk) * DN_KEYS;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 16 * wave + 4 * i + g, at = t * 256 + (turned ^ (i << 4));
      const float bk = dn_below(s_unit[t] & 0xFFFF), bq = dn_below(s_unit[t] >> 16);
      auto as_f16 = [&](iu8_v4u f, float by) {
        iu8_v4u y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const dn_v2h z = __builtin_convertvector(iu8_v2f{__uint_as_float(f[e] << 16) * by, __uint_as_float(f[e] & 0xFFFF0000u) * by}, dn_v2h);
          y[e] = t < m ? __builtin_bit_cast(unsigned, z) : 0u;
        }
        return y;
      };
      *(iu8_v4u *)(to + at) = as_f16(kr[i], bk), *(iu8_v4u *)(to + DN_KEYS / 2 + at) = as_f16(qr[i], bq);
    }
  }
  auto give = [&](iu8_v4f y, iu8_v4f z, int f, unsigned char *to, bool both) {
    iu8_v4u w[2];
    dn_operand<2>(y, z, w);
    *(iu8_v4u *)(to + f * DN_FRAG + lane * 16) = w[0];
    if (both) *(iu8_v4u *)(to + (DN_FRAGS + f) * DN_FRAG + lane * 16) = w[1];
  };
  const iu8_v4f none = {0.f, 0.f, 0.f, 0.f};
  const float rk = s_rk[16 * wave + n], rq = s_rq[16 * wave + n];
  for (int hh = 0; hh < count; ++hh) {
    unsigned char *mine = work + ((size_t)id * heads + h0 + hh) * DN_PART;
    const double *s_sum = s_sums[hh];
    const float *s_beta = s_betas[hh];
    float(*s_a)[P] = s_m[hh & 1];
    // exp(G_i - G_j) / |k_j|: on the diagonal by their difference; under it by three factors of at most 1, so that what is lost of one was lost of all
    iu8_v4f w[3], wd;
    const float *past = s_past[hh];
    const float in = s_in[hh][16 * wave + n], by = s_beta[16 * wave + n] * rk;
    const double si = s_sum[16 * wave + n], top = s_sum[16 * wave];
    const iu8_v4f rd = *(const iu8_v4f *)(s_rk + 16 * wave + 4 * g);
    double sd[4], ends[3];
#pragma unroll
    for (int r = 0; r < 4; ++r) sd[r] = s_sum[16 * wave + 4 * g + r];
#pragma unroll
    for (int jb = 0; jb < 3; ++jb) {
      w[jb] = *(const iu8_v4f *)(past + 16 * jb + 4 * g) * *(const iu8_v4f *)(s_rk + 16 * jb + 4 * g);
      ends[jb] = s_sum[16 * jb + 15];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) wd[r] = 4 * g + r <= n ? __builtin_amdgcn_exp2f((float)(si - sd[r])) * rd[r] : 0.f;
    {
      iu8_v4f y = own * by * wd;
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = 4 * g + r < n ? y[r] : 0.f;
      *(iu8_v4f *)&s_a[16 * wave + n][16 * wave + 4 * g] = y;
    }
#pragma unroll
    for (int jb = 0; jb < 3; ++jb) w[jb] *= in * __builtin_amdgcn_exp2f((float)(top - ends[jb]));
#pragma unroll
    for (int jb = 0; jb < 3; ++jb)
      if (jb < wave) *(iu8_v4f *)&s_a[16 * wave + n][16 * jb + 4 * g] = kk[jb] * by * w[jb];
    // T's blocks on the diagonal by substitution, a column a lane: of row i of F, whose 16 places 16 lanes hold, a place times what stands in y
    {
      float(*at)[P] = (float(*)[P])(&s_a[16 * wave][16 * wave]);
      __builtin_amdgcn_wave_barrier();
      int column = n;  // (not known before this head: the 16 values would be kept)
      asm volatile("" : "+v"(column));
      float f[16], y[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = at[i][n], y[i] = i == column ? 1.f : 0.f;
      dn_below_row<0>(f, y);
#pragma unroll
      for (int i = 0; i < 16; ++i) at[i][n] = y[i];
    }
    __syncthreads();
    // those under it, wave j the column of blocks j: T_ij = -T_ii sum_k A_ik T_kj, on the f32 matrix instruction; a result's rows 4 g + r are the next
    // product's places r of lane group g
    iu8_v4f t[3], f[6], of[3];
#pragma unroll
    for (int r = 0; r < 4; ++r) t[0][r] = s_a[16 * wave + 4 * g + r][16 * wave + n];
#pragma unroll
    for (int d = 1; d < 4; ++d) {
      const int i = min(wave + d, 3);
      of[d - 1] = *(const iu8_v4f *)&s_a[16 * i + n][16 * i + 4 * g];
#pragma unroll
      for (int e = 0; e < d; ++e) f[d * (d - 1) / 2 + e] = *(const iu8_v4f *)&s_a[16 * i + n][16 * min(wave + e, 3) + 4 * g];
    }
#pragma unroll
    for (int d = 1; d < 4; ++d) {
      const int i = wave + d;
      if (i < 4) {
        iu8_v4f y = none, z = none;
#pragma unroll
        for (int e = 0; e < d; ++e)
#pragma unroll
          for (int r = 0; r < 4; ++r) y = __builtin_amdgcn_mfma_f32_16x16x4f32(f[d * (d - 1) / 2 + e][r], t[e][r], y, 0, 0, 0);
        dn_settle(y);
#pragma unroll
        for (int r = 0; r < 4; ++r) z = __builtin_amdgcn_mfma_f32_16x16x4f32(of[d - 1][r], y[r], z, 0, 0, 0);
        dn_settle(z);
        z = -z;
        if (d < 3) t[d < 3 ? d : 0] = z;
#pragma unroll
        for (int r = 0; r < 4; ++r) s_a[16 * wave + 4 * g + r][16 * i + n] = z[r];
      }
    }
    // the inner matrix, row block `wave`
    auto inner = [&](int jb) { return jb < 3 && jb < wave ? qk[jb < 3 ? jb : 0] * rq * w[jb < 3 ? jb : 0] : jb == wave ? across * rq * wd : none; };
    give(inner(0), inner(1), wave < 2 ? wave : 2 * wave - 2, mine + DN_INNER, false);
    if (wave >= 2) give(inner(2), inner(3), 2 * wave - 1, mine + DN_INNER, false);
    if (wave == 3) {
      const int i = lane;
      const double end = s_sum[DN_CHUNK - 1];
      float *f = (float *)(mine + DN_FACTORS);
      const float eg = __builtin_amdgcn_exp2f((float)s_sum[i]);
      const float k1 = s_rk[i] * dn_power(s_unit[i] & 0xFFFF), q1 = s_rq[i] * dn_power(s_unit[i] >> 16);
      f[i] = eg * k1, f[64 + i] = eg * q1, f[128 + i] = __builtin_amdgcn_exp2f((float)(end - s_sum[i])) * k1;
      if (i == 0) f[192] = __builtin_amdgcn_exp2f((float)end);
    }
    __syncthreads();
    for (int f = wave; f < DN_FRAGS; f += 4) {
      const int i = dn_frag_block(f), j = 2 * dn_frag_half(f);
      auto block = [&](int b) { return *(const iu8_v4f *)(i == b ? &s_a[16 * i + n][16 * i + 4 * g] : &s_a[16 * b + n][16 * i + 4 * g]); };
      const iu8_v4f y = block(j) * *(const iu8_v4f *)(s_beta + 16 * j + 4 * g);
      const iu8_v4f z = j < i ? block(j + 1) * *(const iu8_v4f *)(s_beta + 16 * j + 16 + 4 * g) : none;
      give(y, z, f, mine + DN_T, true);
    }
  }
}

// The order of issue of what stands since the last such call: `AHEAD` reads, then M products, each with up to V lane operations and R reads (`READS` of
// them in all) behind it. What is left follows.
template <int M, int V, int R, int AHEAD, int READS>
static __device__ __forceinline__ void dn_step() {
  if constexpr (AHEAD > 0) __builtin_amdgcn_sched_group_barrier(AT_DS_READ, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < M; ++i) {
    __builtin_amdgcn_sched_group_barrier(AT_MFMA, 1, 0);
    if (R > 0 && i * R < READS) __builtin_amdgcn_sched_group_barrier(AT_DS_READ, R, 0);
    if constexpr (V > 0) __builtin_amdgcn_sched_group_barrier(AT_VALU, V, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
}
static __device__ __forceinline__ iu8_v2u dn_transposed(const unsigned char *from) {
  return __builtin_bit_cast(iu8_v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) at_v4s *)from));
}

// The walk over a sequence's chunks. A wave has 16 columns of a head's state, 32 registers a lane, for the whole walk, and no sum passes between
// waves: with the state's columns as the MFMA's columns every product's result is the next one's operand where it lies (rows 4 g + r of two
// blocks of 16 are the eight places of the next, dn_operand). So K's channels are taken 32 ks + 8 g + e by lane group g, as 16 bytes of a row hold
// them, and row 4 p + r of block 2 ks + hb of K^T S's new state is channel 32 ks + 8 p + 4 hb + r, which the LDS's transposing reads give.
//
// The chunks' chain of products bounds a walk (a wave's lane arithmetic does not run under its own matrix instructions here), so its waves come in pairs: one walks
// the chain (K S, V - .., U, the next S), the other does what hangs from it, the rows' answers, with the operands that the first leaves in LDS, and asks for K, Q,
// T, the inner matrix, the factors and V of the next chunk, which come straight from memory into the LDS stage that the chunk before has left. O is
// taken the other way round (the operands exchanged), so that a lane has four neighbouring values of one row to store. Two meetings a chunk: behind U, where the
// stage has been read, and behind the next S. W pairs a workgroup share a stage. A chunk takes 1.7 us with two pairs
// (8,192 rows of 48 heads: 271 us with the preparation's 58; in a trace the walk has 216 to 222), 2.2 with four.
template <int W>
static __device__ __forceinline__ void delta_scan_body(const unsigned short *__restrict__ v, const unsigned char *__restrict__ keys,
                                                       const unsigned char *__restrict__ work, float *__restrict__ state, const int *__restrict__ slot,
                                                       const int *__restrict__ cu, unsigned short *__restrict__ out, int row, int tokens, int seqs, int shape,
                                                       int slots, float scale) {
  constexpr int PARTS = 8 / W, K_AT = 0, Q_AT = DN_KEYS / 2, W_AT = DN_KEYS, V_AT = W_AT + DN_PART, STAGE = V_AT + W * 2048, GIVEN = 8192 + 128;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * STAGE + W * GIVEN];  // stages; of each pair S in one term, U, the columns' units
  const int heads = shape & 0xFFFF, key_heads = shape >> 16, group = heads / key_heads;
  // heads are dealt to the XCDs in turn, a head's workgroups, which read the same bytes, to one
  const int turn = (int)(blockIdx.x >> 3), item = turn / PARTS * 8 + (int)(blockIdx.x & 7), part = turn % PARTS;
  if (item >= seqs * heads) return;
  const int lane = threadIdx.x & 63, wave = at_uniform(threadIdx.x >> 6), pair = wave % W, n = lane & 15, g = lane >> 4;
  int s = item / heads;
  const int h = item - s * heads, hk = h / group;
  // The longest walks first, where a lane a sequence can tell and walks are long enough to pay for it (prompts of 2100, 777, 1859, 903 and 1173 rows, 48
  // heads: 113 us; in the sequences' order, an eighth of the whole to each XCD, 158).
  dn_rows x;
  if (seqs <= 64) {
    const int i = min(lane, seqs - 1), from = cu[i], end = cu[i + 1], to = slot ? slot[i] : i, length = max((end - from + DN_CHUNK - 1) / DN_CHUNK, 0);
    if (__any(length > 4)) {
      const int key = length * 64 + 63 - lane;
      int place = 0;
      for (int i = 0; i < seqs; ++i) place += __builtin_amdgcn_readlane(key, i) > key;
      s = __builtin_ctzll(__ballot(lane < seqs && place == s));
    }
    x = dn_rows_of(s, __builtin_amdgcn_readlane(from, s), __builtin_amdgcn_readlane(end, s), __builtin_amdgcn_readlane(to, s), tokens, slots);
  } else {
    x = dn_sequence(cu, slot, s, tokens, slots);
  }
  if (x.n <= 0) return;
  const int chunks = (x.n + DN_CHUNK - 1) / DN_CHUNK, column = 16 * (W * part + pair);
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char *)smem;
  unsigned char *given = smem + 2 * STAGE + pair * GIVEN;  // 1 KiB each: S's four steps, U's row blocks; the state's unit over U's, U's
  float *units = (float *)(given + 8192);
  const int row_piece = n * 256 + ((dn_turned(g) ^ (n >> 2)) << 4);  // of K's and Q's row n; ^ 4 (ks ^ n % 4) pieces
  auto meet = []() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  if (wave < W) {  // ---- the chain
    float *mine = state + ((size_t)x.slot * heads + h) * (DN * DN) + (8 * g) * DN + column + n;
    auto channel = [](int b, int r) { return 32 * (b >> 1) + 4 * (b & 1) + r; };  // beside 8 g
    iu8_v4f st[8];  // in units of `unit`
    float unit, per_unit, most = 0.f;  // most: the column's largest value, in units
    float none = 0.f;                  // a `top` of no more has nothing to say; -1 where the unit is past 2^16, in which inputs may vanish
    iu8_v4u sw[4][2];
    auto largest = [](float m, iu8_v4f y) { return fmaxf(fmaxf(fmaxf(fmaxf(m, fabsf(y[0])), fabsf(y[1])), fabsf(y[2])), fabsf(y[3])); };
    auto give_state = [&](int ks) {
      dn_operand<2>(st[2 * ks], st[2 * ks + 1], sw[ks]);
      *(iu8_v4u *)(given + ks * 1024 + lane * 16) = sw[ks][0];
    };
#pragma unroll
    for (int b = 0; b < 8; ++b) {
#pragma unroll
      for (int r = 0; r < 4; ++r) st[b][r] = mine[channel(b, r) * DN];
    }
#pragma unroll
    for (int b = 0; b < 8; ++b) most = largest(most, st[b]);
    auto of_column = [](float m) { return at_both<32>(at_both<16>(m, at_max2), at_max2); };
    auto exponent = [](float m) { return (int)(__float_as_uint(m) >> 23); };  // (of a number from 0)
    most = of_column(most);
    {
      const int e = most > 0.f ? min(max(exponent(most) - 4, 7), 247) : 127;
      unit = dn_power(e), per_unit = dn_below(e), none = e > 143 ? -1.f : 0.f, most *= per_unit;
    }
#pragma unroll
    for (int b = 0; b < 8; ++b) st[b] *= per_unit;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) give_state(ks);
    meet();
    for (int c = 0; c < chunks; ++c) {
      const unsigned char *at = smem + (c & 1) * STAGE, *wk = at + W_AT;
      const float *factor = (const float *)(wk + DN_FACTORS);
      iu8_v4u kf[4][4], tf[DN_FRAGS][2], kt[8][2], rt[2][2], ru[2][2];
      iu8_v4f p[4], u[4], er[4], ew[4];
      iu8_v2u vv[4];
      // K S; what the next steps need from LDS is asked for ahead of them
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int rb = 0; rb < 4; ++rb) kf[ks][rb] = *(const iu8_v4u *)(at + K_AT + rb * 4096 + row_piece + ((ks ^ (n & 3)) << 6));
#pragma unroll
      for (int rb = 0; rb < 4; ++rb) {
        p[rb] = u[rb] = iu8_v4f{0.f, 0.f, 0.f, 0.f};
        vv[rb] = dn_transposed(at + V_AT + (16 * rb + 4 * g + (n >> 2)) * (32 * W) + pair * 32 + (n & 3) * 8);
        er[rb] = *(const iu8_v4f *)(factor + 16 * rb + 4 * g);
      }
#pragma unroll
      for (int f = 0; f < DN_FRAGS; ++f)
#pragma unroll
        for (int e = 0; e < 2; ++e) tf[f][e] = *(const iu8_v4u *)(wk + DN_T + (e * DN_FRAGS + f) * DN_FRAG + lane * 16);
      const float whole = factor[192];
      // what the next state needs; where a wave has 512 registers, all the way ahead
      auto ask_turned = [&]() {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int b = 0; b < 8; ++b) {
            const unsigned char *from = at + K_AT + (4 * g + (n >> 2)) * 256 + ((dn_turned(n & 3) ^ g) << 4) + (((b >> 1) ^ (n >> 2)) << 6) + (b & 1) * 8;
            const iu8_v2u lo = dn_transposed(from + 2 * i * 4096), hi = dn_transposed(from + (2 * i + 1) * 4096);
            kt[b][i] = iu8_v4u{lo[0], lo[1], hi[0], hi[1]};
          }
#pragma unroll
        for (int rb = 0; rb < 4; ++rb) ew[rb] = *(const iu8_v4f *)(factor + 128 + 16 * rb + 4 * g);
      };
      if constexpr (W == 2) ask_turned();
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int e = 1; e >= 0; --e)
#pragma unroll
          for (int rb = 0; rb < 4; ++rb) p[rb] = dn_mfma(kf[ks][rb], sw[ks][e], p[rb]);
      dn_step<32, 0, W == 2 ? 2 : 1, 8, W == 2 ? 64 : 29>();
      // V - exp(G) / |k| K S
      float top = most;
#pragma unroll
      for (int rb = 0; rb < 4; ++rb) {
        const float vf[4] = {__uint_as_float(vv[rb][0] << 16), __uint_as_float(vv[rb][0] & 0xFFFF0000u), __uint_as_float(vv[rb][1] << 16),
                             __uint_as_float(vv[rb][1] & 0xFFFF0000u)};
#pragma unroll
        for (int r = 0; r < 4; ++r) p[rb][r] = fmaf(vf[r], per_unit, -er[rb][r] * p[rb][r]);
        top = largest(top, p[rb]);
      }
      top = of_column(top);
      // The unit, in the beginning a 16th of the column's largest value, moves only when that has left 2 .. 256 of it: below, terms of f16 would lack bits; above,
      // they could pass its range (inputs are at most 256 (1 + sqrt(128)), and 64 of them lengthen a column by no more than 8 of them). Where a column held nothing, or
      // nothing beside inputs that pass f32's range in its unit, V alone says where it goes, and is taken again.
      float by = 1.f;
      if (__any(top > 256.f || (top < 2.f && top > none))) {
        auto inputs = [&](int rb) {
          return iu8_v4f{__uint_as_float(vv[rb][0] << 16), __uint_as_float(vv[rb][0] & 0xFFFF0000u), __uint_as_float(vv[rb][1] << 16), __uint_as_float(vv[rb][1] & 0xFFFF0000u)};
        };
        const int was = dn_exponent(unit);
        int to = was + exponent(top) - 131;
        bool anew = false;
        if (__any(!(top > 0x1p-60f && top < 0x1p60f))) {
          float in = 0.f;
#pragma unroll
          for (int rb = 0; rb < 4; ++rb) in = largest(in, inputs(rb));
          in = of_column(in);
          const bool empty = of_column(most) == 0.f;
          anew = empty || !(top < INFINITY);
          if (anew) to = exponent(in) - 4;
          to = (anew ? in : top) > 0.f ? max(to, empty ? 7 : was - 127) : 127;
        }
        to = min(max(to, 7), 247);
        by = dn_power(min(max(was - to + 127, 0), 254));  // (0: what the column held is nothing beside its inputs)
        unit = dn_power(to), per_unit = dn_below(to), none = to > 143 ? -1.f : 0.f;
#pragma unroll
        for (int b = 0; b < 8; ++b) st[b] *= by;
#pragma unroll
        for (int rb = 0; rb < 4; ++rb) p[rb] *= by;
        if (__any(anew)) {
#pragma unroll
          for (int rb = 0; rb < 4; ++rb) {
            const iu8_v4f vf = inputs(rb) * per_unit;
#pragma unroll
            for (int r = 0; r < 4; ++r) p[rb][r] = anew ? vf[r] : p[rb][r];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) dn_operand<2>(p[2 * i], p[2 * i + 1], rt[i]);
      if constexpr (W > 2) ask_turned();
      // U, the smallest products first
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int y = 0; y < 3; ++y)
#pragma unroll
          for (int rb = 2 * i; rb < 4; ++rb) u[rb] = dn_mfma(tf[rb < 2 ? rb : 2 * rb - 2 + i][y == 1], rt[i][y == 0], u[rb]);
#pragma unroll
      for (int b = 0; b < 8; ++b) st[b] *= whole;
#pragma unroll
      for (int rb = 0; rb < 4; ++rb) *(iu8_v4f *)(given + (4 + rb) * 1024 + lane * 16) = u[rb];
      if (g == 0) units[n] = by, units[16 + n] = unit;
      meet();
      // the next state
#pragma unroll
      for (int rb = 0; rb < 4; ++rb) u[rb] *= ew[rb];
#pragma unroll
      for (int i = 0; i < 2; ++i) dn_operand<2>(u[2 * i], u[2 * i + 1], ru[i]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 1; e >= 0; --e)
#pragma unroll
          for (int b = 0; b < 8; ++b) st[b] = dn_mfma(kt[b][i], ru[i][e], st[b]);
      most = 0.f;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        give_state(ks);
        most = largest(largest(most, st[2 * ks]), st[2 * ks + 1]);
      }
      meet();
    }
#pragma unroll
    for (int b = 0; b < 8; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) mine[channel(b, r) * DN] = st[b][r] * unit;
    return;
  }

  // ---- the answers, and what comes from memory
  const size_t id = dn_chunk_id(x);
  const unsigned row_bytes = row * 2;
  auto dma = [&](const unsigned char *from, unsigned off, unsigned to) {  // 64 lanes x 16 bytes, in a row in LDS
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(at_uniform((int)to)), "v"(off), "s"(from) : "memory", "m0");
  };
  constexpr int KEY_LOADS = DN_KEYS / 1024 / W, PART_LOADS = (DN_PART / 1024 + W - 1) / W, LOADS = KEY_LOADS + PART_LOADS + 2;  // a wave's
  auto issue = [&](int c) {
    const int last = x.n - c * DN_CHUNK - 1;  // (a row of V past the end is the last one again, and takes no part)
    const unsigned to = lds0 + (c & 1) * STAGE;
    const unsigned char *kp = keys + ((id + c) * key_heads + hk) * DN_KEYS, *p = work + ((id + c) * heads + h) * DN_PART;
    const unsigned char *vp = (const unsigned char *)v + (size_t)(x.t0 + c * DN_CHUNK) * row_bytes + (h * DN + 16 * W * part) * 2;
#pragma unroll
    for (int i = 0; i < KEY_LOADS; ++i) dma(kp + (W * i + pair) * 1024, lane * 16, to + K_AT + (W * i + pair) * 1024);
    // (as many a wave: the last one again where there are too few)
#pragma unroll
    for (int i = 0; i < PART_LOADS; ++i) {
      const int l = min(W * i + pair, DN_PART / 1024 - 1);
      dma(p + l * 1024, lane * 16, to + W_AT + l * 1024);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int l = W * i + pair;  // 32 / W rows of 32 W bytes
      dma(vp, (unsigned)min(32 / W * l + lane / (2 * W), last) * row_bytes + lane % (2 * W) * 16, to + V_AT + l * 1024);
    }
  };
  auto arrived = [&](bool more) {  // (loads are counted in order: all but the youngest chunk's)
    if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  };
  iu8_v2u y[4];
  unsigned short *to = out + ((size_t)(x.t0 + n) * heads + h) * DN + column + 4 * g;  // of the chunk's row n
  const size_t block = (size_t)16 * heads * DN;
  auto store = [&](int left) {  // (rows from the chunk's first on)
    if (left >= DN_CHUNK) {
#pragma unroll
      for (int rb = 0; rb < 4; ++rb) *(iu8_v2u *)(to + rb * block) = y[rb];
    } else {
#pragma unroll
      for (int rb = 0; rb < 4; ++rb)
        if (16 * rb + n < left) *(iu8_v2u *)(to + rb * block) = y[rb];
    }
    to += 4 * block;
  };
  issue(0);
  if (chunks > 1) issue(1);
  arrived(chunks > 1);
  meet();
  for (int c = 0; c < chunks; ++c) {
    const unsigned char *at = smem + (c & 1) * STAGE, *wk = at + W_AT;
    const float *factor = (const float *)(wk + DN_FACTORS);
    if (c) {
      if (c + 1 < chunks) issue(c + 1);  // (its stage was read in the chunk before)
      store(DN_CHUNK);
    }
    iu8_v4f o[4];
    float eq[4];
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) o[rb] = iu8_v4f{0.f, 0.f, 0.f, 0.f}, eq[rb] = factor[64 + 16 * rb + n];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const iu8_v4u w = *(const iu8_v4u *)(given + ks * 1024 + lane * 16);
#pragma unroll
      for (int rb = 0; rb < 4; ++rb) o[rb] = dn_mfma(w, *(const iu8_v4u *)(at + Q_AT + rb * 4096 + row_piece + ((ks ^ (n & 3)) << 6)), o[rb]);
    }
    iu8_v4u inner[DN_FRAGS];
#pragma unroll
    for (int f = 0; f < DN_FRAGS; ++f) inner[f] = *(const iu8_v4u *)(wk + DN_INNER + f * DN_FRAG + lane * 16);
    meet();  // (the stage has been read)
    const iu8_v4f ratio = *(const iu8_v4f *)(units + 4 * g), un = *(const iu8_v4f *)(units + 16 + 4 * g) * scale;
    iu8_v4u ut[2][1];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      dn_operand<1>(*(const iu8_v4f *)(given + (4 + 2 * i) * 1024 + lane * 16), *(const iu8_v4f *)(given + (5 + 2 * i) * 1024 + lane * 16), ut[i]);
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) o[rb] *= ratio * eq[rb];
#pragma unroll
    for (int f = 0; f < DN_FRAGS; ++f) o[dn_frag_block(f)] = dn_mfma(ut[dn_frag_half(f)][0], inner[f], o[dn_frag_block(f)]);
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      o[rb] *= un;
      y[rb] = iu8_v2u{iu8_bf16_pack(o[rb][0], o[rb][1]), iu8_bf16_pack(o[rb][2], o[rb][3])};
    }
    arrived(false);
    meet();
  }
  store(x.n - (chunks - 1) * DN_CHUNK);
}
