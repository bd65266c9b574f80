// Attention of few new rows a sequence (decode: one token; verify: a few drafted ones) over the paged cache, split over the
// cache's length and joined.
//
//   s_j = scale * q . k_j over the positions j <= the row's own, m = max s, l = sum exp(s - m), o = sum exp(s - m) v_j / l
// with the running maximum and sum of a streamed softmax; parts (waves, then splits) are joined as
//   M = max m_i, L = sum exp(m_i - M) l_i, o = sum exp(m_i - M) o_i / L.
// A row that sees no key gives zeros.
//
// One workgroup: one kv head of one sequence, a run of `chunk` tokens; its four waves take the run's 32-token tiles in turn and
// every wave streams K and V from memory to registers, no LDS between: the rows of the whole group of query heads (and of all new
// tokens: row r is new token r / G, head r % G) share each byte. Bound by the bytes of the cache. Both products have the
// row as the MFMA's column (S^T = K Q^T, O^T = V^T P^T), so a lane keeps one row: its maximum, sum and rescale are plain lane
// arithmetic but for two exchanges a tile, and P goes from the first product's result to the second's operand where it is (the
// second's token order is whatever the first left: 4 g + r of the two blocks of 16).
//
// Rounding: scores, statistics and sums in f32; P is rounded to bf16 for the second product (each weight off by at most 2^-8 of
// itself, the sum of weights taken of the unrounded ones), the output once to bf16.
#pragma once
#include "attn_common.h"

constexpr float AT_LOG2E = 1.44269504088896340736f;

// The tokens of a part: as the launch law cut them, or equal shares where the sequence is longer than the law was told.
static __device__ __forceinline__ int at_chunk(int len, int chunk, int splits) {
  return (long long)chunk * splits >= len ? chunk : (((len - 1) / splits + 1) + 127) / 128 * 128;
}

// Joins `ns` parts of one item: part i's rows at part + i * R * D, their (m, l) at ml + i * 2 R; rows r < live go out.
template <int D, int R, int T>
static __device__ __forceinline__ void at_join(const float *__restrict__ part, const float *__restrict__ ml, int ns, int live, float vs, int tid,
                                               unsigned short *__restrict__ out, const long long *s_dst, float *s_m, float *s_il) {
  // the rows' joint maximum and sum, a row a thread
  for (int r = tid; r < live; r += T) {
    float m = -__builtin_inff(), l = 0.f;
    for (int i = 0; i < ns; ++i) {
      const iu8_v4f x = at_load_through(ml + ((size_t)i * R + r) * 4);
      const float mn = fmaxf(m, x[0]), base = mn == -__builtin_inff() ? 0.f : mn;
      l = l * __builtin_amdgcn_exp2f(m - base) + x[1] * __builtin_amdgcn_exp2f(x[0] - base);
      m = mn;
    }
    s_m[r] = m == -__builtin_inff() ? 0.f : m;
    s_il[r] = l == 0.f ? 0.f : vs / l;
  }
  __syncthreads();
  for (int e = tid; e < live * (D / 4); e += T) {
    const int r = e / (D / 4), d = (e % (D / 4)) * 4;
    iu8_v4f o = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < ns; ++i) {
      const float m = at_load_through(ml + ((size_t)i * R + r) * 4)[0], f = __builtin_amdgcn_exp2f(m - s_m[r]);
      const iu8_v4f x = at_load_through(part + ((size_t)i * R + r) * D + d);
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] = fmaf(f, x[c], o[c]);
    }
    const float il = s_il[r];
    *(iu8_v2u *)(out + s_dst[r] + d) = iu8_v2u{iu8_bf16_pack(o[0] * il, o[1] * il), iu8_bf16_pack(o[2] * il, o[3] * il)};
  }
}

// The rows' (m, l) in a partial take four floats a row, so that a row's pair is one 16-byte store.
template <int D, bool F8, int RT>
static __device__ __forceinline__ void attn_few_body(
    const unsigned short *__restrict__ q, const unsigned char *__restrict__ kc, const unsigned char *__restrict__ vc,
    const float *__restrict__ k_scale, const float *__restrict__ v_scale, const int *__restrict__ table, const int *__restrict__ kv_len,
    const int *__restrict__ cu_q, unsigned short *__restrict__ out, float *__restrict__ partial, int *__restrict__ counter, int q_row,
    int tokens, int shape, int page_shift, int pages, int table_stride, int chunk, int splits, float scale) {
  constexpr int ES = F8 ? 1 : 2, R = 16 * RT, KS = D / 32, DL = D / 16, W = 4;
  constexpr int NV = DL * ES >= 16 ? DL * ES / 16 : 1;  // 16-byte loads (one shorter load) a token and lane of V
  constexpr int VD = DL * ES >= 16 ? 4 : DL * ES / 4;   // dwords of each
  const int heads = shape & 0xFFFF, kv_heads = shape >> 16, G = heads / kv_heads;
  const int split = blockIdx.x % splits, item = blockIdx.x / splits, h = item % kv_heads, s = item / kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, wave = at_uniform(tid >> 6), n = lane & 15, g = lane >> 4;

  const int t0 = cu_q ? cu_q[s] : s;
  const int nq = min((cu_q ? cu_q[s + 1] : s + 1), tokens) - t0;
  const int len = at_len(kv_len, s, table_stride, page_shift);
  const int live = min(nq * G, R);
  if (live <= 0) return;
  chunk = at_chunk(len, chunk, splits);
  const int ns = len > chunk ? (len + chunk - 1) / chunk : 1;
  if (split >= ns) return;

  __shared__ __attribute__((aligned(16))) float s_o[W][R][D + 4];
  __shared__ float s_ml[2][W][R];
  __shared__ float s_m[R], s_il[R];
  __shared__ long long s_dst[R];
  __shared__ int s_last;

  // query fragments and the last position that each row sees
  iu8_v4u qf[RT][KS];
  int limit[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = rt * 16 + n, i = r / G;
    const bool real = r < live;
    limit[rt] = real ? len - nq + i : len - 1;
    const unsigned short *src = q + (size_t)(t0 + (real ? i : 0)) * q_row + (size_t)(h * G + (real ? r - i * G : 0)) * D;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = F8 ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1) : 32 * ks + 8 * g;
      qf[rt][ks] = real ? *(const iu8_v4u *)(src + d) : iu8_v4u{0, 0, 0, 0};
    }
  }
  if (tid < R) {
    const int i = tid / G;
    s_dst[tid] = tid < live ? ((long long)(t0 + i) * heads + h * G + (tid - i * G)) * D : 0;
  }
  const float ks_ = F8 ? k_scale[h] : 1.f, vs = F8 ? v_scale[h] : 1.f, c = scale * AT_LOG2E * ks_;
  const int free_end = len - nq + 1;  // tokens below it are seen by every row
  const int begin = split * chunk, end = len - begin > chunk ? begin + chunk : len;

  iu8_v4f o[RT][DL];
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -__builtin_inff(), l[rt] = 0.f;
#pragma unroll
    for (int i = 0; i < DL; ++i) o[rt][i] = iu8_v4f{0.f, 0.f, 0.f, 0.f};
  }
  const int *row = table + (size_t)s * table_stride;
  const size_t head_elems = (size_t)D << page_shift;
  const int mask = (1 << page_shift) - 1;

  for (int tile = begin + wave * 32; tile < end; tile += W * 32) {
    // the two blocks of 16 tokens; a block past the end or in a hole is read at page 0 and masked
    size_t at[2];
    bool hole[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int tok = tile + 16 * b, p = tok < end ? at_uniform(row[tok >> page_shift]) : -1;
      hole[b] = (unsigned)p >= (unsigned)pages;
      at[b] = hole[b] ? 0 : (((size_t)p * kv_heads + h) * head_elems + (size_t)(tok & mask) * D) * ES;
    }
    iu8_v4u kf[2][KS * ES / 2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < KS * ES / 2; ++i) kf[b][i] = *(const iu8_v4u *)(kc + at[b] + i * 1024 + lane * 16);
    unsigned vf[8][NV][VD];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const unsigned char *p = vc + at[j >> 2] + (4 * g + (j & 3)) * (D * ES) + i * 256 + n * (VD * 4);
        if constexpr (VD == 4) {
          const iu8_v4u x = *(const iu8_v4u *)p;
#pragma unroll
          for (int w = 0; w < 4; ++w) vf[j][i][w] = x[w];
        } else if constexpr (VD == 2) {
          const iu8_v2u x = *(const iu8_v2u *)p;
          vf[j][i][0] = x[0], vf[j][i][1] = x[1];
        } else {
          vf[j][i][0] = *(const unsigned *)p;
        }
      }
    // scores of the tile's tokens 16 b + 4 g + r, in units of log2
    float sc[RT][8];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        iu8_v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          iu8_v4u a;
          if constexpr (F8) a = ks & 1 ? at_e4m3x8(kf[b][ks >> 1][2], kf[b][ks >> 1][3]) : at_e4m3x8(kf[b][ks >> 1][0], kf[b][ks >> 1][1]);
          else a = kf[b][ks];
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(at_bf(a), at_bf(qf[rt][ks]), acc, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[rt][4 * b + r] = acc[r] * c;
      }
    }
    if (tile + 32 > min(end, free_end) || hole[0] || hole[1]) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int tok = tile + 16 * (j >> 2) + 4 * g + (j & 3);
        const bool gone = hole[j >> 2] || tok >= end;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          if (gone || tok > limit[rt]) sc[rt][j] = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int w = 0; w < VD; ++w) vf[j][i][w] = gone ? 0u : vf[j][i][w];
      }
    }
    unsigned pf[RT][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float top = sc[rt][0];
#pragma unroll
      for (int j = 1; j < 8; ++j) top = fmaxf(top, sc[rt][j]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float mn = fmaxf(m[rt], top), base = mn == -__builtin_inff() ? 0.f : mn;
      if (__any(mn > m[rt])) {
        const float f = __builtin_amdgcn_exp2f(m[rt] - base);
        l[rt] *= f;
#pragma unroll
        for (int i = 0; i < DL; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[rt][i][r] *= f;
        m[rt] = mn;
      }
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(sc[rt][j] - base), l[rt] += p[j];
#pragma unroll
      for (int j = 0; j < 4; ++j) pf[rt][j] = iu8_bf16_pack(p[2 * j], p[2 * j + 1]);
    }
    // V's operand, channel after channel: eight tokens of one channel a lane
#pragma unroll
    for (int i = 0; i < DL; i += 2) {
      unsigned lo[4], hi[4];
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        unsigned x, y;  // channels i, i + 1 of tokens 2 jj and 2 jj + 1
        if constexpr (F8) {
          const unsigned dx = vf[2 * jj][i / 16][i / 4 % 4 % VD], dy = vf[2 * jj + 1][i / 16][i / 4 % 4 % VD];
          x = i & 2 ? at_e4m3_bf16<true>(dx) : at_e4m3_bf16<false>(dx);
          y = i & 2 ? at_e4m3_bf16<true>(dy) : at_e4m3_bf16<false>(dy);
        } else {
          x = vf[2 * jj][i / 8][i / 2 % 4 % VD], y = vf[2 * jj + 1][i / 8][i / 2 % 4 % VD];
        }
        lo[jj] = __builtin_amdgcn_perm(y, x, 0x05040100u);
        hi[jj] = __builtin_amdgcn_perm(y, x, 0x07060302u);
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const at_v8bf p = at_bf(pf[rt][0], pf[rt][1], pf[rt][2], pf[rt][3]);
        o[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(at_bf(lo[0], lo[1], lo[2], lo[3]), p, o[rt][i], 0, 0, 0);
        o[rt][i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(at_bf(hi[0], hi[1], hi[2], hi[3]), p, o[rt][i + 1], 0, 0, 0);
      }
    }
  }

  // the waves' parts: maxima and sums first, then each wave's rows on the joint maximum
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] += __shfl_xor(l[rt], 16);
    l[rt] += __shfl_xor(l[rt], 32);
    if (g == 0) s_ml[0][wave][rt * 16 + n] = m[rt], s_ml[1][wave][rt * 16 + n] = l[rt];
  }
  __syncthreads();
  float top[RT], sum[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = rt * 16 + n;
    top[rt] = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < W; ++w) top[rt] = fmaxf(top[rt], s_ml[0][w][r]);
    const float base = top[rt] == -__builtin_inff() ? 0.f : top[rt];
    sum[rt] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) sum[rt] += s_ml[1][w][r] * __builtin_amdgcn_exp2f(s_ml[0][w][r] - base);
    const float f = __builtin_amdgcn_exp2f(m[rt] - base);
    // lane (n, g) holds row n: channel index 4 g + r of each of the DL products
    constexpr int RUN = F8 ? DL : DL < 8 ? DL : 8;  // channels in a row: DL of an e4m3 row, up to 8 of a bf16 one
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int i = 0; i < DL; i += 4) {
        const int d = (i / RUN) * 16 * RUN + (4 * g + x) * RUN + i % RUN;
        *(iu8_v4f *)&s_o[wave][r][d] = iu8_v4f{o[rt][i][x] * f, o[rt][i + 1][x] * f, o[rt][i + 2][x] * f, o[rt][i + 3][x] * f};
      }
    if (wave == 0 && g == 0) s_m[r] = top[rt], s_il[r] = sum[rt];
  }
  __syncthreads();
  float *part = nullptr, *ml = nullptr;
  if (ns > 1) {
    const size_t per = (size_t)R * (D + 4);
    part = partial + (size_t)item * splits * per;
    ml = part + (size_t)splits * R * D;
  }
  for (int e = tid; e < live * (D / 4); e += 256) {
    const int r = e / (D / 4), d = (e % (D / 4)) * 4;
    iu8_v4f x = *(const iu8_v4f *)&s_o[0][r][d];
#pragma unroll
    for (int w = 1; w < W; ++w) x += *(const iu8_v4f *)&s_o[w][r][d];
    if (ns > 1) {
      at_store_through(part + ((size_t)split * R + r) * D + d, x);
    } else {
      const float il = s_il[r] == 0.f ? 0.f : vs / s_il[r];
      *(iu8_v2u *)(out + s_dst[r] + d) = iu8_v2u{iu8_bf16_pack(x[0] * il, x[1] * il), iu8_bf16_pack(x[2] * il, x[3] * il)};
    }
  }
  if (ns == 1) return;
  if (tid < live) at_store_through(ml + ((size_t)split * R + tid) * 4, iu8_v4f{s_m[tid], s_il[tid], 0.f, 0.f});
  iu8_stores_done();
  __syncthreads();
  if (tid == 0) {
    const int before = iu8_arrive(counter + item);
    s_last = before == ns - 1;
    if (s_last) __hip_atomic_store(counter + item, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s_last) return;
  at_join<D, R, 256>(part, ml, ns, live, vs, tid, out, s_dst, s_m, s_il);
}
