// The gated delta rule in chunks of 64 rows (delta_common.h has the formulas): prompts.
//
// With G_i the sum of the logarithms of the decays of a chunk's rows 0 .. i, S0 the state in front of it, and
//   A_ij = beta_i exp(G_i - G_j) k^_i . k^_j (j < i),   T = (1 + A)^-1,
// the rows' updates u (the rule's beta (v - ...)) are the solution of a unit triangular system, and everything is matrix products:
//   U  = T diag(beta) (V - diag(exp G) K^ S0)
//   O  = scale (diag(exp G) Q^ S0 + [exp(G_i - G_j) q^_i . k^_j, j <= i] U)
//   S1 = exp(G_63) S0 + K^^T diag(exp(G_63 - G_j)) U
// Two kernels. delta_prep makes, for all chunks at once, T diag(beta) and the inner matrix of O, each already as the other's operand, and the rows'
// factors; delta_scan walks a sequence's chunks in order.
//
// Precision: the state and all that enters it is f32, on the bf16 matrix cores: a row of K or Q is bf16 as it comes (its norm's and decay's
// factors are moved to the other side of the product), the other side is split into three bf16 terms, 24 bits (dn_split). What goes only
// into the rows' bf16 answers takes two terms, 16 bits. G is summed, and its differences taken, in f64: after a strong decay the later rows'
// differences would be left with the sum's digits.
#pragma once
#include "delta_step.h"

// A chunk and value head's part of the workspace. Operands are kept as fragments, 64 lanes x 16 bytes: lane (l % 16, g = l / 16) has row l % 16 of 16 and
// the columns 4 g .. 4 g + 3 of the first and of the second 16 of 32, which is how a product's result lies (dn_operand).
// Fragment f of a lower triangle: row block 0, 1 of the first 32 columns; row blocks 2, 3 of the first and of the last.
constexpr int DN_FRAGS = 6, DN_FRAG = 1024;
static __host__ __device__ constexpr int dn_frag_block(int f) { return f < 2 ? f : 2 + (f - 2) / 2; }
static __host__ __device__ constexpr int dn_frag_half(int f) { return f < 2 ? 0 : (f - 2) & 1; }
constexpr int DN_T = 0, DN_INNER = 3 * DN_FRAGS * DN_FRAG, DN_FACTORS = DN_INNER + 2 * DN_FRAGS * DN_FRAG, DN_PART = DN_FACTORS + 1024;
// the factors, f32: [64] exp(G_i) / |k_i|, [64] scale exp(G_i) / |q_i|, [64] exp(G_63 - G_i) / |k_i|, exp(G_63)

static __device__ __forceinline__ int dn_chunk_id(const dn_rows &x) { return (x.t0 >> 6) + x.s; }  // of its first chunk: no two sequences' meet

static __device__ __forceinline__ void delta_prep_body(const unsigned short *__restrict__ q, const unsigned short *__restrict__ k,
                                                       const unsigned short *__restrict__ a, const unsigned short *__restrict__ b,
                                                       const float *__restrict__ a_log, const float *__restrict__ dt_bias,
                                                       const int *__restrict__ slot, const int *__restrict__ cu, unsigned char *__restrict__ work, int row,
                                                       int ab_row, int tokens, int seqs, int shape, int slots, float eps, float scale) {
  constexpr int P = 68;  // floats of a row in LDS
  const int heads = shape & 0xFFFF, group = heads / (shape >> 16);
  const int id = blockIdx.x / heads, h = blockIdx.x - id * heads, hk = h / group;
  const int lane = threadIdx.x & 63, wave = at_uniform(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  int s = -1;
  if (!cu) {
    s = id - id / 65;  // (a sequence a row: (s >> 6) + s)
    while ((s >> 6) + s > id) --s;
  } else {
    for (int base = 0; base < seqs; base += 64) {
      const int i = base + lane;
      s += __popcll(__ballot(i < seqs && (cu[i] >> 6) + i <= id));
    }
  }
  if (s < 0 || s >= seqs) return;
  const dn_rows x = dn_sequence(cu, slot, s, tokens, slots);
  const int c0 = (id - dn_chunk_id(x)) * DN_CHUNK, m = min(x.n - c0, DN_CHUNK);  // the chunk's first row, its rows
  if (c0 < 0 || m <= 0) return;

  __shared__ __attribute__((aligned(16))) float s_a[DN_CHUNK][P], s_i[DN_CHUNK][P], s_t[DN_CHUNK][P];
  __shared__ double s_sum[DN_CHUNK];
  __shared__ float s_beta[DN_CHUNK], s_rk[DN_CHUNK], s_rq[DN_CHUNK];

  // the products of the rows, row block `wave` with those up to it; a row past the end is the last one again, and takes no part
  const size_t t0 = x.t0 + c0;
  auto fragment = [&](const unsigned short *from, int rb, int ks) {
    return *(const iu8_v4u *)(from + (t0 + min(16 * rb + n, m - 1)) * row + hk * DN + 32 * ks + 8 * g);
  };
  iu8_v4u kf[4], qf[4];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) kf[ks] = fragment(k, wave, ks), qf[ks] = fragment(q, wave, ks);
  if (wave == 0) {
    const int i = lane;
    float lg = 0.f, be = 0.f;
    if (i < m) {
      lg = dn_log_decay(iu8_bf16_f32(a[(t0 + i) * ab_row + h]), a_log[h], dt_bias[h]);
      be = dn_beta(iu8_bf16_f32(b[(t0 + i) * ab_row + h]));
    }
    double sum = lg;
#pragma unroll
    for (int y = 1; y < 64; y *= 2) {
      const double z = __shfl_up(sum, y);
      sum += i >= y ? z : 0.0;
    }
    s_sum[i] = sum, s_beta[i] = be;
  }
  {
    auto norm = [&](const iu8_v4u (&f)[4]) {
      float ss = 0.f;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = __uint_as_float(f[ks][e] << 16), z = __uint_as_float(f[ks][e] & 0xFFFF0000u);
          ss = fmaf(y, y, fmaf(z, z, ss));
        }
      ss = at_both<32>(at_both<16>(ss, at_sum2), at_sum2);
      return 1.f / sqrtf(ss + eps);
    };
    const float rk = norm(kf), rq = norm(qf);
    const bool live = 16 * wave + n < m;
    if (g == 0) s_rk[16 * wave + n] = live ? rk : 0.f, s_rq[16 * wave + n] = live ? rq * scale : 0.f;
  }
  iu8_v4f kk[4], qk[4];
#pragma unroll
  for (int jb = 0; jb < 4; ++jb) {
    kk[jb] = qk[jb] = iu8_v4f{0.f, 0.f, 0.f, 0.f};
    if (jb <= wave) {
      iu8_v4u f[4];
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) f[ks] = fragment(k, jb, ks);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) kk[jb] = dn_mfma(kf[ks], f[ks], kk[jb]), qk[jb] = dn_mfma(qf[ks], f[ks], qk[jb]);
      dn_settle(kk[jb]), dn_settle(qk[jb]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int jb = 0; jb < 4; ++jb) {
    const int j = 16 * jb + n;
    if (jb <= wave) {
      const double sj = s_sum[j];
      const float rj = s_rk[j];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * wave + 4 * g + r;
        const float w = i >= j ? expf((float)(s_sum[i] - sj)) * rj : 0.f;
        s_a[i][j] = i > j ? s_beta[i] * s_rk[i] * w * kk[jb][r] : 0.f;
        s_i[i][j] = s_rq[i] * w * qk[jb][r];
      }
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) s_i[16 * wave + 4 * g + r][j] = 0.f, s_t[16 * wave + 4 * g + r][j] = 0.f;
    }
  }
  unsigned char *mine = work + ((size_t)id * heads + h) * DN_PART;
  if (wave == 3) {
    const int i = lane;
    const double end = s_sum[DN_CHUNK - 1];
    float *f = (float *)(mine + DN_FACTORS);
    const float eg = expf((float)s_sum[i]);
    f[i] = eg * s_rk[i], f[64 + i] = eg * s_rq[i], f[128 + i] = expf((float)(end - s_sum[i])) * s_rk[i];
    if (i == 0) f[192] = expf((float)end);
  }
  __syncthreads();
  // T's blocks on the diagonal by substitution, a column a lane
  if (g == 0) {
    float y[16];
    const float(*at)[P] = (const float(*)[P])(&s_a[16 * wave][16 * wave]);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float z = i == n ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) z = fmaf(-at[i][j], y[j], z);
      y[i] = z;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s_t[16 * wave + i][16 * wave + n] = y[i];
  }
  __syncthreads();
  // those under it, wave j the column of blocks j: T_ij = -T_ii sum_k A_ik T_kj, on the f32 matrix instruction; a result's rows 4 g + r are the next
  // product's places r of lane group g
  {
    iu8_v4f t[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) t[0][r] = s_t[16 * wave + 4 * g + r][16 * wave + n];
#pragma unroll
    for (int d = 1; d < 4; ++d) {
      const int i = wave + d;
      if (i < 4) {
        iu8_v4f y = {0.f, 0.f, 0.f, 0.f}, z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < d; ++e) {
          const iu8_v4f f = *(const iu8_v4f *)&s_a[16 * i + n][16 * (wave + e) + 4 * g];
#pragma unroll
          for (int r = 0; r < 4; ++r) y = __builtin_amdgcn_mfma_f32_16x16x4f32(f[r], t[e][r], y, 0, 0, 0);
        }
        dn_settle(y);
        const iu8_v4f f = *(const iu8_v4f *)&s_t[16 * i + n][16 * i + 4 * g];
#pragma unroll
        for (int r = 0; r < 4; ++r) z = __builtin_amdgcn_mfma_f32_16x16x4f32(f[r], y[r], z, 0, 0, 0);
        dn_settle(z);
        t[d] = -z;
#pragma unroll
        for (int r = 0; r < 4; ++r) s_t[16 * i + 4 * g + r][16 * wave + n] = -z[r];
      }
    }
  }
  __syncthreads();
  // both as fragments
  for (int f = wave; f < 2 * DN_FRAGS; f += 4) {
    const bool inner = f >= DN_FRAGS;
    const int ff = inner ? f - DN_FRAGS : f, i = 16 * dn_frag_block(ff) + n, j = 32 * dn_frag_half(ff) + 4 * g;
    const float *from = inner ? s_i[i] : s_t[i];
    iu8_v4f y = *(const iu8_v4f *)(from + j), z = *(const iu8_v4f *)(from + j + 16);
    if (!inner) y = y * *(const iu8_v4f *)(s_beta + j), z = z * *(const iu8_v4f *)(s_beta + j + 16);
    iu8_v4u w[3];
    dn_operand<3>(y, z, w);
    unsigned char *to = mine + (inner ? DN_INNER : DN_T) + ff * DN_FRAG + lane * 16;
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (!inner || e < 2) *(iu8_v4u *)(to + e * DN_FRAGS * DN_FRAG) = w[e];
  }
}

// The walk over a sequence's chunks. A wave has 16 columns of a head's state, 32 registers a lane, for the whole walk, and nothing passes between
// waves: with the state's columns as the MFMA's columns every product's result is the next one's operand where it lies (rows 4 g + r of two
// blocks of 16 are the eight places of the next, dn_operand). So K's channels are taken 32 ks + 8 g + e by lane group g, as 16 bytes of a row hold
// them, and row 4 p + r of block 2 ks + hb of K^T S's new state is channel 32 ks + 8 p + 4 hb + r, which the LDS's transposing reads give. Only O is taken
// the other way round (the same registers, the operands exchanged), so that a lane has four neighbouring values of one row to store.
//
// The waves of a workgroup are W neighbouring column blocks of one head and share what they multiply by: a chunk's K, Q, T, inner matrix and factors and
// each wave's own columns of V come straight from memory into one of two LDS stages, the next chunk's under this one's products; one barrier a
// chunk.
template <int W>
static __device__ __forceinline__ void delta_scan_body(const unsigned short *__restrict__ q, const unsigned short *__restrict__ k,
                                                       const unsigned short *__restrict__ v, const unsigned char *__restrict__ work,
                                                       float *__restrict__ state, const int *__restrict__ slot, const int *__restrict__ cu,
                                                       unsigned short *__restrict__ out, int row, int tokens, int seqs, int shape, int slots) {
  constexpr int PARTS = 8 / W, K_AT = 0, Q_AT = 16384, W_AT = 32768, V_AT = W_AT + DN_PART, STAGE = V_AT + W * 2048;
  constexpr int LOADS = 32 + DN_PART / 1024;  // wave-loads of 1 KiB of what is shared
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * STAGE];
  const int heads = shape & 0xFFFF, group = heads / (shape >> 16);
  // workgroups are dealt to the XCDs in turn: those of neighbouring heads, which read the same keys, to one
  const int all = seqs * heads * PARTS, share = (all + 7) / 8, item = (blockIdx.x & 7) * share + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= share || item >= all) return;
  const int s = item / (heads * PARTS), h = item / PARTS - s * heads, hk = h / group, part = item % PARTS;
  const int lane = threadIdx.x & 63, wave = at_uniform(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const dn_rows x = dn_sequence(cu, slot, s, tokens, slots);
  if (x.n <= 0) return;
  const int chunks = (x.n + DN_CHUNK - 1) / DN_CHUNK, column = 16 * (W * part + wave);
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char *)smem;
  const unsigned char *parts = work + ((size_t)dn_chunk_id(x) * heads + h) * DN_PART;

  auto dma = [&](const unsigned char *from, unsigned to) {  // (a lane's own address; 64 x 16 bytes in a row in LDS)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(at_uniform((int)to)), "v"(from) : "memory", "m0");
  };
  auto issue = [&](int c, int stage) {
    const int t0 = x.t0 + c * DN_CHUNK, last = x.t0 + x.n - 1;
    const unsigned to = lds0 + stage * STAGE;
    const unsigned char *p = parts + (size_t)c * heads * DN_PART;
#pragma unroll
    for (int i = 0; i < (LOADS + W - 1) / W; ++i) {
      const int l = i * W + wave;  // (uniform)
      if (l < 32) {
        const unsigned short *base = l < 16 ? k : q;
        const int rb = (l & 15) >> 2, ks = l & 3;
        dma((const unsigned char *)(base + (size_t)min(t0 + 16 * rb + n, last) * row + hk * DN + 32 * ks + 8 * g), to + l * 1024);
      } else if (l < LOADS) {
        dma(p + (l - 32) * 1024 + lane * 16, to + l * 1024);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      dma((const unsigned char *)(v + (size_t)min(t0 + 32 * i + (lane >> 1), last) * row + h * DN + column + 8 * (lane & 1)), to + V_AT + wave * 2048 + i * 1024);
  };
  auto transposed = [](const unsigned char *from) {
    return __builtin_bit_cast(iu8_v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) at_v4s *)from));
  };

  issue(0, 0);
  float *mine = state + ((size_t)x.slot * heads + h) * (DN * DN) + column + n;
  auto channel = [&](int b, int r) { return 32 * (b >> 1) + 8 * g + 4 * (b & 1) + r; };
  iu8_v4f st[8];
#pragma unroll
  for (int b = 0; b < 8; ++b)
#pragma unroll
    for (int r = 0; r < 4; ++r) st[b][r] = mine[channel(b, r) * DN];

  for (int c = 0; c < chunks; ++c) {
    unsigned char *at = smem + (c & 1) * STAGE;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (c + 1 < chunks) issue(c + 1, (c + 1) & 1);
    const unsigned char *wk = at + W_AT;
    const float *factor = (const float *)(wk + DN_FACTORS);
    auto frag = [&](int from, int f) { return *(const iu8_v4u *)(at + from + f * 1024 + lane * 16); };

    // K S and (Q S)^T
    iu8_v4f p[4], o[4];
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) p[rb] = o[rb] = iu8_v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      iu8_v4u w[3];
      dn_operand<3>(st[2 * ks], st[2 * ks + 1], w);
#pragma unroll
      for (int rb = 0; rb < 4; ++rb) {
        const iu8_v4u kf = frag(K_AT, rb * 4 + ks), qf = frag(Q_AT, rb * 4 + ks);
#pragma unroll
        for (int e = 2; e >= 0; --e) p[rb] = dn_mfma(kf, w[e], p[rb]);
        o[rb] = dn_mfma(w[1], qf, o[rb]);
        o[rb] = dn_mfma(w[0], qf, o[rb]);
      }
    }
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) dn_settle(p[rb]), dn_settle(o[rb]);
    // V - exp(G) / |k| K S
    iu8_v4u rt[2][3];
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      const iu8_v2u vv = transposed(at + V_AT + wave * 2048 + (16 * rb + 4 * g + (n >> 2)) * 32 + (n & 3) * 8);
      const iu8_v4f er = *(const iu8_v4f *)(factor + 16 * rb + 4 * g);
      const float vf[4] = {__uint_as_float(vv[0] << 16), __uint_as_float(vv[0] & 0xFFFF0000u), __uint_as_float(vv[1] << 16), __uint_as_float(vv[1] & 0xFFFF0000u)};
#pragma unroll
      for (int r = 0; r < 4; ++r) p[rb][r] = fmaf(-er[r], p[rb][r], vf[r]);
      o[rb] *= factor[64 + 16 * rb + n];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) dn_operand<3>(p[2 * i], p[2 * i + 1], rt[i]);
    // U
    iu8_v4f u[4];
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) u[rb] = iu8_v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int f = 0; f < DN_FRAGS; ++f) {
      const int rb = dn_frag_block(f), i = dn_frag_half(f);
      iu8_v4u w[3];
#pragma unroll
      for (int e = 0; e < 3; ++e) w[e] = frag(W_AT + DN_T, e * DN_FRAGS + f);
#pragma unroll
      for (int d = 2; d >= 0; --d)  // the smallest products first
#pragma unroll
        for (int e = 0; e <= d; ++e) u[rb] = dn_mfma(w[e], rt[i][d - e], u[rb]);
    }
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) dn_settle(u[rb]);
    // the rows' answers
    iu8_v4u ut[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) dn_operand<2>(u[2 * i], u[2 * i + 1], ut[i]);
#pragma unroll
    for (int f = 0; f < DN_FRAGS; ++f) {
      const int rb = dn_frag_block(f), i = dn_frag_half(f);
      const iu8_v4u w0 = frag(W_AT + DN_INNER, f), w1 = frag(W_AT + DN_INNER, DN_FRAGS + f);
      o[rb] = dn_mfma(ut[i][1], w0, o[rb]);
      o[rb] = dn_mfma(ut[i][0], w1, o[rb]);
      o[rb] = dn_mfma(ut[i][0], w0, o[rb]);
    }
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) dn_settle(o[rb]);
    if (out) {
#pragma unroll
      for (int rb = 0; rb < 4; ++rb) {
        const int t = c * DN_CHUNK + 16 * rb + n;
        if (t < x.n)
          *(iu8_v2u *)(out + ((size_t)(x.t0 + t) * heads + h) * DN + column + 4 * g) =
              iu8_v2u{iu8_bf16_pack(o[rb][0], o[rb][1]), iu8_bf16_pack(o[rb][2], o[rb][3])};
      }
    }
    // the next state
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) u[rb] *= *(const iu8_v4f *)(factor + 128 + 16 * rb + 4 * g);
#pragma unroll
    for (int i = 0; i < 2; ++i) dn_operand<3>(u[2 * i], u[2 * i + 1], rt[i]);
    const float whole = factor[192];
#pragma unroll
    for (int b = 0; b < 8; ++b) st[b] *= whole;
#pragma unroll
    for (int b = 0; b < 8; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const unsigned char *kt = at + K_AT + (b >> 1) * 1024 + ((n & 3) * 16 + 4 * g + (n >> 2)) * 16 + (b & 1) * 8;
        const iu8_v2u lo = transposed(kt + 2 * i * 4096), hi = transposed(kt + (2 * i + 1) * 4096);
        const iu8_v4u kf = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
        for (int e = 2; e >= 0; --e) st[b] = dn_mfma(kf, rt[i][e], st[b]);
      }
#pragma unroll
    for (int b = 0; b < 8; ++b) dn_settle(st[b]);
  }
#pragma unroll
  for (int b = 0; b < 8; ++b)
#pragma unroll
    for (int r = 0; r < 4; ++r) mine[channel(b, r) * DN] = st[b][r];
}
