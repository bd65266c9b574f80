// Attention of many new rows a sequence (whole prompts, chunks behind a cached prefix) over the paged cache, causal, with the
// formulas of attn_few.h.
//
// One workgroup: 128 rows of one kv head of one sequence, 32 a wave; row r is new token r / G, head r % G of the group, so every
// head of the group shares the staged keys and a short prompt still fills its rows. K and V come tile by tile (BK tokens, two
// LDS stages): bf16 straight from memory into LDS, e4m3 through registers, widened once for all four waves. Bound by the matrix
// cores and the LDS that feeds them.
//
// Both products have the row as the MFMA's column (attn_few.h has why): S^T = K Q^T leaves lane (row, half) the tokens
// 8 i + 4 half + r, which is the token order that P's operand of O^T = V^T P^T then has, and the LDS's transposing read gives V^T
// in the same order (4 tokens of a channel a read).
//
// LDS order: K as it lies in the cache. V's rows with their 16-byte pieces exchanged in groups of four (piece ^ 4 (row % 8) and so
// on by width): the transposing read takes 64 bytes of 8 rows at a time, which the exchange spreads over all banks.
#pragma once
#include "attn_few.h"

template <int D>
constexpr int at_many_bk() { return D == 256 ? 32 : 64; }

template <int D, bool F8>
static __device__ __forceinline__ void attn_many_body(
    const unsigned short *__restrict__ q, const unsigned char *__restrict__ kc, const unsigned char *__restrict__ vc,
    const float *__restrict__ k_scale, const float *__restrict__ v_scale, const int *__restrict__ table, const int *__restrict__ kv_len,
    const int *__restrict__ cu_q, unsigned short *__restrict__ out, float *__restrict__ partial, int *__restrict__ counter, int q_row,
    int tokens, int shape, int page_shift, int pages, int table_stride, int chunk, int splits, int qtiles, float scale) {
  constexpr int ES = F8 ? 1 : 2, R = 128, BK = at_many_bk<D>(), HB = BK / 32, KS = D / 16, MT = D / 32, ROWB = D * 2, TILE = BK * ROWB;
  const int heads = shape & 0xFFFF, kv_heads = shape >> 16, G = heads / kv_heads;
  const int split = blockIdx.x % splits, item = blockIdx.x / splits;
  const int qt = qtiles - 1 - item % qtiles, h = item / qtiles % kv_heads, s = item / qtiles / kv_heads;  // the longest rows first
  const int tid = threadIdx.x, lane = tid & 63, wave = at_uniform(tid >> 6), n = lane & 31, hf = lane >> 5;

  const int t0 = cu_q ? cu_q[s] : s;
  const int nq = min((cu_q ? cu_q[s + 1] : s + 1), tokens) - t0;
  const int len = at_len(kv_len, s, table_stride, page_shift);
  const long long all = (long long)max(nq, 0) * G;
  if ((long long)qt * R >= all) return;
  const int live = (int)min((long long)R, all - (long long)qt * R);
  const int i_first = qt * R / G, i_last = (qt * R + live - 1) / G;
  const int kv_end = max(min(len, len - nq + i_last + 1), 0), free_end = len - nq + i_first + 1;
  chunk = at_chunk(kv_end, chunk, splits);
  const int ns = kv_end > chunk ? (kv_end + chunk - 1) / chunk : 1;
  if (split >= ns) return;

  __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * TILE];  // K, V of stage 0; K, V of stage 1
  __shared__ float s_m[R], s_il[R];
  __shared__ long long s_dst[R];
  __shared__ int s_last;

  const int r = qt * R + wave * 32 + n, i = r / G;
  const bool real = wave * 32 + n < live;
  const int limit = real ? len - nq + i : len - 1;
  iu8_v4u qf[KS];
  {
    const unsigned short *src = q + (size_t)(t0 + (real ? i : 0)) * q_row + (size_t)(h * G + (real ? r - i * G : 0)) * D;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = real ? *(const iu8_v4u *)(src + 16 * ks + 8 * hf) : iu8_v4u{0, 0, 0, 0};
  }
  const long long dst = ((long long)(t0 + i) * heads + h * G + (r - i * G)) * D;
  if (hf == 0) s_dst[wave * 32 + n] = dst;
  const float ks_ = F8 ? k_scale[h] : 1.f, vs = F8 ? v_scale[h] : 1.f, c = scale * AT_LOG2E * ks_;
  const int begin = split * chunk, end = kv_end - begin > chunk ? begin + chunk : kv_end;

  const int *row = table + (size_t)s * table_stride;
  const size_t head_elems = (size_t)D << page_shift;
  const int mask = (1 << page_shift) - 1;
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char *)smem;

  // where a block of 16 tokens lies (a block past the end or in a hole: page 0, masked later)
  auto block_at = [&](int tok, bool &hole) -> size_t {
    const int p = tok < end ? at_uniform(row[tok >> page_shift]) : -1;
    hole = (unsigned)p >= (unsigned)pages;
    return hole ? 0 : (((size_t)p * kv_heads + h) * head_elems + (size_t)(tok & mask) * D) * ES;
  };
  auto swz = [](int t) { return D == 256 ? t & 7 : D == 128 ? t & 3 : t & 1; };

  constexpr int RAW = F8 ? BK * D / 256 / 16 : 1;  // 16-byte pieces of K (and of V) a thread, e4m3
  iu8_v4u rk[RAW], rv[RAW];
  auto issue = [&](int tile, int stage) {
    if constexpr (F8) {
#pragma unroll
      for (int x = 0; x < RAW; ++x) {
        // a block is D pieces, and 256 threads take whole blocks or a whole number of threads share one: uniform a wave
        const int piece = x * 256 + tid, blk = at_uniform((x * 256 + wave * 64) / D);
        bool hole;
        const size_t at = block_at(tile + 16 * blk, hole);
        rk[x] = *(const iu8_v4u *)(kc + at + (size_t)(piece % D) * 16);
        rv[x] = *(const iu8_v4u *)(vc + at + (size_t)(piece % D) * 16);
      }
    } else {
      constexpr int BLK = 16 * ROWB / 1024, LOADS = BK / 16 * BLK;  // wave-loads of 1 KiB a block, a tile
#pragma unroll
      for (int x = 0; x < LOADS / 4; ++x) {
        const int ld = x * 4 + wave, blk = ld / BLK, part = ld % BLK;
        bool hole;
        const size_t at = block_at(tile + 16 * blk, hole);
        const unsigned lk = lds0 + stage * 2 * TILE + ld * 1024, lv = lk + TILE;
        // V: lane's slot is row t, piece p; it holds piece p ^ 4 swz(t) of the row
        const int t = part * (1024 / ROWB) + lane * 16 / ROWB, p = lane % (ROWB / 16);
        const unsigned ok = part * 1024 + lane * 16, ov = t * ROWB + ((p ^ (4 * swz(t))) * 16);
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lk), "v"(ok), "s"(kc + at) : "memory", "m0");
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lv), "v"(ov), "s"(vc + at) : "memory", "m0");
      }
    }
  };
  auto commit = [&](int stage) {  // e4m3: widen into the stage
    if constexpr (F8) {
      unsigned char *sk = smem + stage * 2 * TILE, *sv = sk + TILE;
#pragma unroll
      for (int x = 0; x < RAW; ++x) {
        const int piece = x * 256 + tid, blk = piece / D, in = piece % D;
        unsigned char *pk = sk + blk * 16 * ROWB + ((in / 16) * 32 + in % 16) * 16;
        *(iu8_v4u *)pk = at_e4m3x8(rk[x][0], rk[x][1]);
        *(iu8_v4u *)(pk + 256) = at_e4m3x8(rk[x][2], rk[x][3]);
        const int t = blk * 16 + in / (D / 16), p = in % (D / 16) * 2;
        unsigned char *pv = sv + t * ROWB + ((p ^ (4 * swz(t))) * 16);
        *(iu8_v4u *)pv = at_e4m3x8(rv[x][0], rv[x][1]);
        *(iu8_v4u *)(pv + 16) = at_e4m3x8(rv[x][2], rv[x][3]);
      }
    }
  };
  auto arrived = [&]() {
    if constexpr (!F8) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };

  at_v16f o[MT];
#pragma unroll
  for (int x = 0; x < MT; ++x) o[x] = at_v16f{};
  float m = -__builtin_inff(), l = 0.f;
  const unsigned k_lane = (n >> 4) * 16 * ROWB + hf * 256 + (n & 15) * 16;
  const int vrow = 4 * hf + ((lane & 15) >> 2);
  const unsigned v_lane = vrow * ROWB + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;

  if (begin < end) {
    issue(begin, 0);
    commit(0);
  }
  arrived();
  int stage = 0;
  for (int tile = begin; tile < end; tile += BK, stage ^= 1) {
    const bool more = tile + BK < end;
    if (more) issue(tile + BK, stage ^ 1);
    unsigned char *sk = smem + stage * 2 * TILE, *sv = sk + TILE;
    unsigned holes = 0;
#pragma unroll
    for (int b = 0; b < BK / 16; ++b) {
      bool hole;
      (void)block_at(tile + 16 * b, hole);
      holes |= (hole ? 1u : 0u) << b;
    }
    const bool special = holes || tile + BK > min(end, free_end);
    if (holes || tile + BK > end) {  // rows of V that take no part: a weight of zero would keep their NaNs
      for (int x = tid; x < BK * (ROWB / 16); x += 256) {
        const int t = x / (ROWB / 16);
        if (tile + t >= end || (holes >> (t >> 4) & 1)) *(iu8_v4u *)(sv + x * 16) = iu8_v4u{0, 0, 0, 0};
      }
      __syncthreads();
    }
    at_v16f sc[HB];
#pragma unroll
    for (int hb = 0; hb < HB; ++hb) {
      sc[hb] = at_v16f{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const iu8_v4u a = *(const iu8_v4u *)(sk + k_lane + hb * 32 * ROWB + ks * 512);
        sc[hb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(at_bf(a), at_bf(qf[ks]), sc[hb], 0, 0, 0);
      }
    }
    // (the products are read here, in the block that makes them: behind a branch this compiler leaves too few wait states between
    // a matrix instruction and the first read of its result, seen as wrong scores)
    float st[HB][16];
#pragma unroll
    for (int hb = 0; hb < HB; ++hb)
#pragma unroll
      for (int x = 0; x < 16; ++x) st[hb][x] = sc[hb][x] * c;
    if (special) {
#pragma unroll
      for (int hb = 0; hb < HB; ++hb)
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const int t = 32 * hb + 8 * (x >> 2) + 4 * hf + (x & 3);
          if (tile + t > limit || tile + t >= end || (holes >> (t >> 4) & 1)) st[hb][x] = -__builtin_inff();
        }
    }
    float top = st[0][0];
#pragma unroll
    for (int hb = 0; hb < HB; ++hb)
#pragma unroll
      for (int x = 0; x < 16; ++x) top = fmaxf(top, st[hb][x]);
    top = fmaxf(top, __shfl_xor(top, 32));
    const float mn = fmaxf(m, top), base = mn == -__builtin_inff() ? 0.f : mn;
    if (__any(mn > m)) {
      const float f = __builtin_amdgcn_exp2f(m - base);
      l *= f;
#pragma unroll
      for (int x = 0; x < MT; ++x) o[x] *= f;
      m = mn;
    }
    unsigned pf[HB][8];
#pragma unroll
    for (int hb = 0; hb < HB; ++hb)
#pragma unroll
      for (int x = 0; x < 16; x += 2) {
        const float p0 = __builtin_amdgcn_exp2f(st[hb][x] - base), p1 = __builtin_amdgcn_exp2f(st[hb][x + 1] - base);
        l += p0 + p1;
        pf[hb][x / 2] = iu8_bf16_pack(p0, p1);
      }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const unsigned char *pv = sv + v_lane + ((mt ^ swz(vrow)) * 64);
#pragma unroll
      for (int hb = 0; hb < HB; ++hb)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const at_v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) at_v4s *)(pv + (32 * hb + 16 * t) * ROWB));
          const at_v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) at_v4s *)(pv + (32 * hb + 16 * t + 8) * ROWB));
          const iu8_v2u a0 = __builtin_bit_cast(iu8_v2u, lo), a1 = __builtin_bit_cast(iu8_v2u, hi);
          o[mt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(at_bf(a0[0], a0[1], a1[0], a1[1]), at_bf(pf[hb][4 * t], pf[hb][4 * t + 1], pf[hb][4 * t + 2], pf[hb][4 * t + 3]),
                                                          o[mt], 0, 0, 0);
        }
    }
    if (more) commit(stage ^ 1);
    arrived();
  }
  l += __shfl_xor(l, 32);
  if (ns == 1) {
    const float il = l == 0.f ? 0.f : vs / l;
    if (real) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int x = 0; x < 16; x += 4)
          *(iu8_v2u *)(out + dst + 32 * mt + 2 * x + 4 * hf) =
              iu8_v2u{iu8_bf16_pack(o[mt][x] * il, o[mt][x + 1] * il), iu8_bf16_pack(o[mt][x + 2] * il, o[mt][x + 3] * il)};
    }
    return;
  }
  const size_t per = (size_t)R * (D + 4);
  float *part = partial + (size_t)item * splits * per, *ml = part + (size_t)splits * R * D;
  if (real) {
    float *p = part + ((size_t)split * R + wave * 32 + n) * D;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int x = 0; x < 16; x += 4)
        at_store_through(p + 32 * mt + 2 * x + 4 * hf, iu8_v4f{o[mt][x], o[mt][x + 1], o[mt][x + 2], o[mt][x + 3]});
    if (hf == 0) at_store_through(ml + ((size_t)split * R + wave * 32 + n) * 4, iu8_v4f{m, l, 0.f, 0.f});
  }
  iu8_stores_done();
  __syncthreads();
  if (tid == 0) {
    const int before = iu8_arrive(counter + item);
    s_last = before == ns - 1;
    if (s_last) __hip_atomic_store(counter + item, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s_last) return;
  at_join<D, R, 256, 4 * TILE / (R * 8), 4, 8>(part, ml, ns, live, vs, tid, out, s_dst, s_m, s_il, (float *)smem);
}
