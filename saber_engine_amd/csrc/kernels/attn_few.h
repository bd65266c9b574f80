// Attention of few new rows a sequence (decode: one token; verify: a few drafted ones) over the paged cache, split over the
// cache's length and joined.
//
//   s_j = scale * q . k_j over the positions j <= the row's own, m = max s, l = sum exp(s - m), o = sum exp(s - m) v_j / l
// with the running maximum and sum of a streamed softmax; parts (waves, then splits) are joined as
//   M = max m_i, L = sum exp(m_i - M) l_i, o = sum exp(m_i - M) o_i / L.
// A row that sees no key gives zeros.
//
// The work is dealt level: an item is one kv head of one sequence and up to R of its rows (row r is new token r / G, head r % G of
// the group: all of them share each byte), its length counted in units of 128 tokens; every workgroup of the grid gets the same
// number of consecutive units over all items, whatever the sequences' lengths (it counts them itself, from kv_len). An item
// that several workgroups have parts of is joined by the last of them to arrive. A unit is four tiles of 32 tokens, one a wave.
//
// Bound by the bytes of the cache, so what matters is bytes in flight: every wave has a tile of K and a tile of V in LDS of its own, filled
// straight from memory, and asks for the next K as soon as its scores are made, for the next V as soon as its product is: up to
// 128 KiB a compute unit on the way, with no register held for it and no barrier between the waves. Measured: one row on 131,072 keys, 4
// kv heads of 256, 537 MB of cache, 91 us (5.9 TB/s; a plain read reaches 6.0 to 6.4); 64 rows on up to 8,192, 8 heads of 128,
// 1.27 GB, 202 us (6.3); 33 on up to 16,001 in e4m3, 586 MB, 102 us (5.7); 9 x 5 new rows of group 6 on up to 6,007, 154 MB, 46 us
// (3.4). One row on 1,800 keys 13 us: the chain of lengths, pages, keys, parts and join, behind 3 of the launch.
//
// Both products have the row as the MFMA's column (S^T = K Q^T, O^T = V^T P^T), so a lane keeps one row: its maximum, sum and
// rescale are plain lane arithmetic but for two exchanges a tile, and P goes from the first product's result to the second's
// operand where it is (the second's token order is whatever the first left: 4 g + r of the two blocks of 16). V's operand has
// eight tokens of one channel a lane: the LDS's transposing reads give it from V's rows, whose 16-byte pieces are exchanged
// within a row on the way into LDS so that a read's rows lie in all banks.
//
// A weight of zero would keep an infinity or a NaN of V (0 * inf), so what a row does not see must not reach its product: V's
// rows behind the end and in holes are zeroed in LDS; a value that is not finite among the new tokens themselves, which some
// rows see and others do not, takes the product's slow form (lane arithmetic, only for the rows that see it).
//
// Rounding: scores, statistics and sums in f32; P is rounded to bf16 for the second product (each weight off by at most 2^-8 of
// itself, the sum of weights taken of the unrounded ones), the output once to bf16.
#pragma once
#include "attn_common.h"
#include "attn_deal.h"

constexpr float AT_LOG2E = 1.44269504088896340736f;

// The tokens of a part of the many-row kernels: as the launch law cut them, or equal shares where the sequence is longer than the
// law was told.
static __device__ __forceinline__ int at_chunk(int len, int chunk, int splits) {
  return (long long)chunk * splits >= len ? chunk : (((len - 1) / splits + 1) + 127) / 128 * 128;
}

// Joins `ns` parts of one item: part i's rows at part + i * step (part 0's at part + first), behind them their (m, l), four floats a
// row (one 16-byte store); rows r < live go out. The parts come from memory (other XCDs wrote them), so as many loads as registers allow are
// in flight, U items x K parts a thread, the first of them beside the (m, l). `s_f`: ns * live floats of LDS; ns at most 128 (R = 128: 32).
template <int D, int R, int T, int U, int K>
static __device__ __forceinline__ void at_join_of(const float *__restrict__ part, size_t first, size_t step, int ns, int live, float vs, int tid,
                                               unsigned short *__restrict__ out, const long long *s_dst, float *s_il, float *s_f) {
  constexpr int D4 = D / 4, NI = (R * D4 + T - 1) / T;
  const int all = live * D4;
  const __amdgpu_buffer_rsrc_t from = at_resource(part);
  const unsigned first4 = (unsigned)first * 4, step4 = (unsigned)step * 4;
  iu8_v4f x[U][K];
  auto load = [&](int it, int i) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int e = min((it + u) * T + tid, all - 1);
        const int ii = min(i + k, ns - 1);
        x[u][k] = at_load_through(from, (ii ? ii * step4 : first4) + e * 16);
      }
  };
  load(0, 0);
  {  // a row's joint maximum, its parts' factors, its sum: LPR lanes a row, up to PL parts a lane
    constexpr int LPR = T / R, PL = 128 / LPR < 16 ? 128 / LPR : 16;
    const int r = tid / LPR, j = tid % LPR;
    float m[PL], l[PL], top = -__builtin_inff(), sum = 0.f;
#pragma unroll
    for (int x = 0; x < PL; ++x) {
      const int i = x * LPR + j;
      iu8_v4f y = {-__builtin_inff(), 0.f, 0.f, 0.f};
      if (i < ns && r < live) y = at_load_through(from, (i ? i * step4 : first4) + R * D * 4 + r * 16);
      m[x] = y[0], l[x] = y[1];
    }
#pragma unroll
    for (int x = 0; x < PL; ++x) top = fmaxf(top, m[x]);
#pragma unroll
    for (int x = 1; x < LPR; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
    const float base = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
    for (int x = 0; x < PL; ++x) {
      const int i = x * LPR + j;
      const float f = __builtin_amdgcn_exp2f(m[x] - base);
      sum = fmaf(f, l[x], sum);
      if (i < ns && r < live) s_f[i * live + r] = f;
    }
#pragma unroll
    for (int x = 1; x < LPR; x *= 2) sum += __shfl_xor(sum, x);
    if (j == 0 && r < live) s_il[r] = sum == 0.f ? 0.f : vs / sum;
  }
  __syncthreads();
  for (int it = 0; it < NI; it += U) {
    if (it * T >= all) break;  // (the same for every thread)
    iu8_v4f o[U];
#pragma unroll
    for (int u = 0; u < U; ++u) o[u] = iu8_v4f{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < ns; i += K) {
      if (it || i) load(it, i);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = min((it + u) * T + tid, all - 1) / D4;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const float f = s_f[min(i + k, ns - 1) * live + r];
#pragma unroll
          for (int c = 0; c < 4; ++c) o[u][c] = i + k < ns ? fmaf(f, x[u][k][c], o[u][c]) : o[u][c];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = (it + u) * T + tid;
      if (it + u < NI && e < all) {
        const int r = e / D4;
        const float il = s_il[r];
        *(iu8_v2u *)(out + s_dst[r] + e % D4 * 4) = iu8_v2u{iu8_bf16_pack(o[u][0] * il, o[u][1] * il), iu8_bf16_pack(o[u][2] * il, o[u][3] * il)};
      }
    }
  }
}

template <int D, int R, int T, int U, int K>
static __device__ __forceinline__ void at_join(const float *__restrict__ part, size_t first, size_t step, int ns, int live, float vs, int tid,
                                               unsigned short *__restrict__ out, const long long *s_dst, float *s_il, float *s_f) {
  if (ns <= 2) at_join_of<D, R, T, U * K / 2, 2>(part, first, step, ns, live, vs, tid, out, s_dst, s_il, s_f);
  else if (ns <= 4) at_join_of<D, R, T, U * K / 4, 4>(part, first, step, ns, live, vs, tid, out, s_dst, s_il, s_f);
  else at_join_of<D, R, T, U, K>(part, first, step, ns, live, vs, tid, out, s_dst, s_il, s_f);
}

template <int D, bool F8>
struct AtFew {
  static constexpr int ES = F8 ? 1 : 2, ROWB = D * ES, TILE = 32 * ROWB, NL = TILE / 1024;  // wave-loads of 1 KiB a tile
  // where V's piece lies in its row: piece ^ swz(token), so that the rows that one transposing read takes together (16 of
  // 32 bytes for bf16, 32 of 16 bytes for e4m3) lie in all banks
  static __device__ __forceinline__ int swz(int t) {
    if constexpr (F8) return D == 256 ? t & 15 : D == 128 ? t & 7 : (t >> 1) & 3;
    else return 2 * (D == 256 ? t & 15 : D == 128 ? t & 7 : t & 3);
  }
};

template <int D, bool F8, int RT>
static __device__ __forceinline__ void attn_few_body(
    const unsigned short *__restrict__ q, const unsigned char *__restrict__ kc, const unsigned char *__restrict__ vc,
    const float *__restrict__ k_scale, const float *__restrict__ v_scale, const int *__restrict__ table, const int *__restrict__ kv_len,
    const int *__restrict__ cu_q, unsigned short *__restrict__ out, float *__restrict__ partial, int *__restrict__ counter, int q_row,
    int tokens, int seqs, int shape, int page_shift, int pages, int table_stride, int unit_shift, int qtiles, float scale) {
  using A = AtFew<D, F8>;
  constexpr int ES = A::ES, ROWB = A::ROWB, TILE = A::TILE, NL = A::NL, R = 16 * RT, KS = D / 32, DT = D / 16, W = 4;
  constexpr int REGION = 2 * TILE > R * (D + 4) * 4 ? 2 * TILE : R * (D + 4) * 4;  // a wave's LDS: its tiles, then its part of the sum
  constexpr size_t SLOT = (size_t)R * (D + 4);                                      // floats of a part
  const int heads = shape & 0xFFFF, kv_heads = shape >> 16, G = heads / kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, wave = at_uniform(tid >> 6), n = lane & 15, g = lane >> 4;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[W * REGION];
  __shared__ float s_ml[2][W][R];
  __shared__ float s_m[R], s_il[R];
  __shared__ long long s_dst[R];
  __shared__ int s_last;
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char *)smem;
  unsigned char *sk = smem + wave * REGION, *sv = sk + TILE;
  const size_t head_elems = (size_t)D << page_shift;
  const int mask = (1 << page_shift) - 1;

  // (Where a workgroup's 32 rows leave few registers: a number made anew, with the addresses that follow from it, which kept across the tiles would be registers
  // that the loop lacks)
  auto anew = [](int x) {
    if constexpr (RT == 2 || (F8 && D == 256)) asm volatile("" : "+v"(x));
    return x;
  };

  // ---- this workgroup's units
  struct Seq {
    int t0, nq, pos, len;
  };
  auto sequence = [&](int i) {  // its new rows (those of `tokens`), the first one's position, its length
    Seq x;
    x.t0 = cu_q ? cu_q[i] : i;
    const int to = cu_q ? cu_q[i + 1] : i + 1;
    x.nq = min(to, tokens) - x.t0;
    x.len = at_len(kv_len, i, table_stride, page_shift);
    x.pos = x.len - (to - x.t0);
    return x;
  };
  auto own_units = [&](const Seq &x) { return (unsigned)((max(x.len, 1) - 1) >> unit_shift) + 1; };
  auto tiles_of = [&](const Seq &x) { return x.nq > 0 ? (unsigned)min(((long long)x.nq * G - 1) / R + 1, (long long)qtiles) : 0u; };
  unsigned mine = 0, before = 0, total, longest = 0;  // (units: the launch law keeps their sum below 2^31)
  const int per_lane = (seqs - 1) / 64 + 1;
  if (seqs == 1) {
    const Seq x = sequence(0);
    total = mine = own_units(x) * tiles_of(x) * kv_heads, longest = own_units(x);
  } else {
    for (int i = lane * per_lane; i < min(lane * per_lane + per_lane, seqs); ++i) {
      const Seq x = sequence(i);
      const unsigned u = own_units(x), t = tiles_of(x);
      mine += u * t * kv_heads, longest = max(longest, t ? u : 0u);
    }
    before = mine;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
      const unsigned y = __shfl_up(before, x);
      before += lane >= x ? y : 0;
      longest = max(longest, __shfl_xor(longest, x));
    }
    total = __builtin_amdgcn_readlane(before, 63), longest = at_uniform(longest);
    before -= mine;
  }
  if (!total) return;
  // (an item's parts are bounded: they lie in one workgroup's LDS when they are joined)
  const unsigned grid = gridDim.x;
  unsigned share = max((total + grid - 1) / grid, (longest + AT_PARTS - 2) / (AT_PARTS - 1));
  // A join costs a workgroup about what four units do: whole items where they are no more than that longer.
  const unsigned over = share % longest, lone = longest - over;
  if (over && lone <= 4) share += lone;
  // Where the items' parts of `share` units fit the grid, each item begins with a workgroup of its own, as if its last part were
  // whole: no workgroup then has the end of one item and the beginning of another. (9 x 5 new rows
  // of group 6 on 4,000 keys 52.6 us -> 47.1; 100 on 1,000 35.0 -> 26.3; the look at the lengths costs 0.5 us.)
  bool apart = share > 1 && (long long)seqs * kv_heads * qtiles <= grid;
  if (apart) {
    unsigned parts = 0, ahead, all;
    if (seqs == 1) {
      all = ahead = parts = ((longest - 1) / share + 1) * (total / longest);
    } else {
      for (int i = lane * per_lane; i < min(lane * per_lane + per_lane, seqs); ++i) {
        const Seq x = sequence(i);
        parts += ((own_units(x) - 1) / share + 1) * tiles_of(x) * kv_heads;
      }
      ahead = parts;
#pragma unroll
      for (int x = 1; x < 64; x *= 2) {
        const unsigned y = __shfl_up(ahead, x);
        ahead += lane >= x ? y : 0;
      }
      all = __builtin_amdgcn_readlane(ahead, 63);
    }
    apart = all <= grid;
    if (apart) mine = parts * share, before = (ahead - parts) * share, total = all * share;
  }
  auto units_of = [&](const Seq &x) {
    const unsigned u = own_units(x);
    return apart ? ((u - 1) / share + 1) * share : u;
  };
  if (blockIdx.x > (total - 1) / share) return;
  unsigned at_unit = blockIdx.x * share;
  const unsigned last_unit = min(at_unit + share, total);
  // the item that the first unit lies in: sequence s, kv head h, row tile qt, `u0` units of it before
  int s = 0;
  unsigned base = 0;
  if (seqs > 1) {
    const int owner = at_uniform(__ffsll((unsigned long long)__ballot(before + mine > at_unit)) - 1);
    s = owner * per_lane, base = __builtin_amdgcn_readlane(before, owner);
  }
  Seq q_;
  s = at_walk([&](int i) { return q_ = sequence(i), units_of(q_) * tiles_of(q_) * kv_heads; }, s, seqs, base, at_unit);
  if (s >= seqs) return;
  unsigned u0, h, qt;
  {
    const unsigned u = units_of(q_), it = (at_unit - base) / u, tiles = tiles_of(q_);
    u0 = at_unit - base - it * u, h = tiles == 1 ? it : it / tiles, qt = it - h * tiles;
  }

  // where a tile's two blocks of 16 tokens lie; a block past the end or in a hole is read at page 0 and masked
  struct Tile {
    size_t at[2];
    unsigned holes;
  };
  auto dma = [&](const unsigned char *src, unsigned off, unsigned lds) {  // (nt: a byte of the cache is used once)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" : : "s"(lds), "v"(off), "s"(src) : "memory", "m0");
  };
  const unsigned lk = lds0 + wave * REGION, lv = lk + TILE;
  auto issue_k = [&](const Tile &t) {
#pragma unroll
    for (int i = 0; i < NL; ++i) dma(kc + t.at[i / (NL / 2)], (i % (NL / 2)) * 1024 + lane * 16, lk + i * 1024);
  };
  auto issue_v = [&](const Tile &t) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const unsigned slot = i * 1024 + lane * 16, tok = slot / ROWB, p = slot % ROWB / 16;
      dma(vc + t.at[i / (NL / 2)], (tok % 16) * ROWB + ((p ^ A::swz(tok)) * 16), lv + i * 1024);
    }
  };

  for (;;) {
    // ---- a segment: units u0 .. of one item
    const unsigned units = units_of(q_), u1 = min(units, u0 + (last_unit - at_unit));
    const int nq = q_.nq, t0 = q_.t0, pos = q_.pos, len = q_.len, begin = u0 << unit_shift, end = u1 == units ? len : (int)(u1 << unit_shift);
    const int live = (int)min((long long)nq * G - (long long)qt * R, (long long)R);
    const int free_end = pos + (int)(qt * R) / G + 1;  // tokens below it are seen by every row
    const int *row = table + (size_t)s * table_stride;
    auto fetch = [&](int tile, int (&p)[2]) {
#pragma unroll
      for (int b = 0; b < 2; ++b) p[b] = row[min((unsigned)(tile + 16 * b) >> page_shift, (unsigned)table_stride - 1u)];
    };
    auto locate = [&](int tile, const int (&p)[2]) {
      Tile t;
      t.holes = 0;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int tok = tile + 16 * b;
        const bool hole = tok >= end || (unsigned)p[b] >= (unsigned)pages;
        t.holes |= hole ? 1u << b : 0u;
        t.at[b] = hole ? 0 : (((size_t)p[b] * kv_heads + h) * head_elems + (size_t)(tok & mask) * D) * ES;
      }
      return t;
    };

    int tile = begin + wave * 32, p_at[2];
    Tile cur;
    if (tile < end) {
      fetch(tile, p_at);
      cur = locate(tile, p_at);
      issue_k(cur);
      issue_v(cur);
    }
    // query fragments and the last position that each row sees; with a negative scale the rows change sign (exact), so that the
    // factor of the scores is positive and their order the weights'
    const float ks_ = F8 ? k_scale[h] : 1.f, vs = F8 ? v_scale[h] : 1.f, cs = scale * AT_LOG2E * ks_;
    const unsigned flip = cs < 0.f ? 0x80008000u : 0u;
    const float c = at_uniform_f(fmaxf(fabsf(cs), 1e-37f));  // (of a zero scale: every weight rounds to one)
    iu8_v4u qf[RT][KS];
    int limit[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = (int)qt * R + rt * 16 + n, i = r / G;
      const bool real = rt * 16 + n < live;
      limit[rt] = real ? pos + i : len - 1;
      const unsigned short *src = q + (size_t)(t0 + (real ? i : 0)) * q_row + (size_t)(h * G + (real ? r - i * G : 0)) * D;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d = F8 ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1) : 32 * ks + 8 * g;
        qf[rt][ks] = *(const iu8_v4u *)(src + d);
      }
    }
    if (tid < R) {
      const int r = (int)qt * R + tid, i = r / G;
      s_dst[tid] = tid < live ? ((long long)(t0 + i) * heads + h * G + (r - i * G)) * D : 0;
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qf[rt][ks] = (qf[rt][ks] ^ flip) & (rt * 16 + n < live ? ~0u : 0u);
        asm volatile("" : "+v"(qf[rt][ks]));  // here, not in the loop, is what waits for them
      }

    iu8_v4f o[RT][DT];
    float m[RT], l[RT];  // m of the scores as they come, in units of 1 / c of log2
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = -__builtin_inff(), l[rt] = 0.f;
#pragma unroll
      for (int i = 0; i < DT; ++i) o[rt][i] = iu8_v4f{0.f, 0.f, 0.f, 0.f};
    }

    for (; tile < end; tile += W * 32) {
      const bool more = tile + W * 32 < end;
      Tile next;
      if (more) fetch(tile + W * 32, p_at);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");  // K is in (its loads are older than V's)
      // scores of the tile's tokens 16 b + 4 g + r
      float sc[RT][8];
      {
        constexpr int KL = KS * ES / 2;  // 16-byte reads a block
        iu8_v4u kf[2][KL];
        iu8_v4f acc[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt][0] = acc[rt][1] = iu8_v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KL; ++i)
#pragma unroll
          for (int b = 0; b < 2; ++b) kf[b][i] = *(const iu8_v4u *)(sk + b * 16 * ROWB + i * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < KL; ++i)
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              const iu8_v4u x = kf[b][i];
              if constexpr (F8) {
                acc[rt][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(at_bf(at_e4m3x8(x[0], x[1])), at_bf(qf[rt][2 * i]), acc[rt][b], 0, 0, 0);
                acc[rt][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(at_bf(at_e4m3x8(x[2], x[3])), at_bf(qf[rt][2 * i + 1]), acc[rt][b], 0, 0, 0);
              } else {
                acc[rt][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(at_bf(x), at_bf(qf[rt][i]), acc[rt][b], 0, 0, 0);
              }
            }
        // the order of issue: reads ahead of the products by a few, not one read, one wait, one product
        constexpr int AHEAD = 2 * KL < 6 ? 2 * KL : 6;
        __builtin_amdgcn_sched_group_barrier(AT_DS_READ, AHEAD, 0);
#pragma unroll
        for (int i = 0; i < 2 * KL - AHEAD; ++i) {
          __builtin_amdgcn_sched_group_barrier(AT_MFMA, RT * (F8 ? 2 : 1), 0);
          __builtin_amdgcn_sched_group_barrier(AT_DS_READ, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(AT_MFMA, AHEAD * RT * (F8 ? 2 : 1), 0);
        // (read in the block that makes them: behind a branch this compiler leaves too few wait states between a matrix
        // instruction and the first read of its result, seen as wrong scores)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float x = acc[rt][j >> 2][j & 3];
            asm volatile("" : "+v"(x));
            sc[rt][j] = x;
          }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) {
        next = locate(tile + W * 32, p_at);
        issue_k(next);
      }
      const bool special = tile + 32 > min(end, free_end) || cur.holes;
      if (special) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int tok = tile + 16 * (j >> 2) + 4 * g + (j & 3);
          const bool gone = (cur.holes >> (j >> 2) & 1) || tok >= end;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            if (gone || tok > limit[rt]) sc[rt][j] = -__builtin_inff();
        }
      }
      float p[RT][8];
      unsigned pf[RT][4];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float top = sc[rt][0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, sc[rt][j]);
        top = at_both<32>(at_both<16>(top, at_max2), at_max2);
        // (the maximum moves only when a score passes it by 2^8: attn_many.h)
        if (__any((top - m[rt]) * c > 8.f)) {
          const float mn = fmaxf(m[rt], top), f = __builtin_amdgcn_exp2f((m[rt] - (mn == -__builtin_inff() ? 0.f : mn)) * c);
          l[rt] *= f;
#pragma unroll
          for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[rt][i][r] *= f;
          m[rt] = mn;
        }
        const float mc = m[rt] == -__builtin_inff() ? 0.f : m[rt] * c;
#pragma unroll
        for (int j = 0; j < 8; ++j) p[rt][j] = __builtin_amdgcn_exp2f(fmaf(sc[rt][j], c, -mc)), l[rt] += p[rt][j];
#pragma unroll
        for (int j = 0; j < 4; ++j) pf[rt][j] = iu8_bf16_pack(p[rt][2 * j], p[rt][2 * j + 1]);
      }
      if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");  // V is in (the next K's loads are younger)
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (special) {
        auto piece = [&](int t, int x) -> unsigned char * { return sv + t * ROWB + ((x ^ A::swz(t)) * 16); };
        const int ln = anew(lane), lane = ln, n = ln & 15, g = ln >> 4;
        constexpr int PR = ROWB / 16;  // pieces a row
        const int stop = min(end - tile, 32);
        // what takes no part: rows behind the end, a hole's block
        for (int x = stop * PR + lane; x < 32 * PR; x += 64) *(iu8_v4u *)(sv + x * 16) = iu8_v4u{0, 0, 0, 0};
        if (cur.holes)
          for (int x = lane; x < 32 * PR; x += 64)
            if (cur.holes >> (x / (16 * PR)) & 1) *(iu8_v4u *)(sv + x * 16) = iu8_v4u{0, 0, 0, 0};
        bool odd = false;  // a value that is not finite among tokens that some rows see and others do not
        for (int x = max(free_end - tile, 0) * PR + lane; x < stop * PR; x += 64) {
          const iu8_v4u v = *(const iu8_v4u *)(sv + x * 16);
#pragma unroll
          for (int w = 0; w < 4; ++w) odd |= F8 ? at_e4m3_nan4(v[w]) : at_nonfinite2(v[w]);
        }
        if (__any(odd)) {
#pragma unroll 1
          for (int t = max(free_end - tile, 0); t < min(end - tile, 32); ++t) {
            if (cur.holes >> (t >> 4) & 1) continue;
            const int j = 4 * (t >> 4) + (t & 3);
            float pj[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              pj[rt] = p[rt][0];
#pragma unroll
              for (int x = 1; x < 8; ++x) pj[rt] = j == x ? p[rt][x] : pj[rt];
              pj[rt] = __shfl(pj[rt], n + 16 * ((t >> 2) & 3));
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
              float v[4];
              at_four<F8>(piece(t, (16 * dt + 4 * g) * ES / 16) + (16 * dt + 4 * g) * ES % 16, v);
#pragma unroll
              for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[rt][dt][r] = tile + t <= limit[rt] ? fmaf(pj[rt], v[r], o[rt][dt][r]) : o[rt][dt][r];
            }
            for (int x = lane; x < ROWB / 16; x += 64) *(iu8_v4u *)(sv + t * ROWB + x * 16) = iu8_v4u{0, 0, 0, 0};
          }
        }
      }
      // V's operand: eight tokens of channel 16 dt + n a lane
      {
        constexpr int RD = F8 ? 1 : 2;  // reads a channel block
        iu8_v2u vf[DT][RD];
        const int ln = anew(lane), n = ln & 15, g = ln >> 4;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          if constexpr (F8) {
            const int e = n >> 1, t = (e & 4) * 4 + 4 * g + (e & 3);
            typedef int v2i __attribute__((ext_vector_type(2)));
            vf[dt][0] = __builtin_bit_cast(iu8_v2u, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i *)(
                                                        sv + t * ROWB + ((dt ^ A::swz(t)) * 16) + (n & 1) * 8)));
          } else {
            const int t = 4 * g + (n >> 2), p16 = 2 * dt + ((n >> 1) & 1);
            const unsigned char *at = sv + t * ROWB + (n & 1) * 8 + (p16 ^ A::swz(t)) * 16;
            vf[dt][0] = __builtin_bit_cast(iu8_v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) at_v4s *)at));
            vf[dt][1] = __builtin_bit_cast(iu8_v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) at_v4s *)(at + 16 * ROWB)));
          }
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const iu8_v4u a = F8 ? at_e4m3x8(vf[dt][0][0], vf[dt][0][1]) : iu8_v4u{vf[dt][0][0], vf[dt][0][1], vf[dt][RD - 1][0], vf[dt][RD - 1][1]};
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(at_bf(a), at_bf(pf[rt][0], pf[rt][1], pf[rt][2], pf[rt][3]), o[rt][dt], 0, 0, 0);
        }
        constexpr int AHEAD = DT < 4 ? DT : 4;
        __builtin_amdgcn_sched_group_barrier(AT_DS_READ, AHEAD * RD, 1);
#pragma unroll
        for (int i = 0; i < DT - AHEAD; ++i) {
          __builtin_amdgcn_sched_group_barrier(AT_MFMA, RT, 1);
          __builtin_amdgcn_sched_group_barrier(AT_DS_READ, RD, 1);
        }
        __builtin_amdgcn_sched_group_barrier(AT_MFMA, AHEAD * RT, 1);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) issue_v(next);
      cur = next;
    }

    // the waves' parts: maxima and sums first, then each wave's rows on the joint maximum
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] *= c;
      l[rt] = at_both<32>(at_both<16>(l[rt], at_sum2), at_sum2);
      if (g == 0) s_ml[0][wave][rt * 16 + n] = m[rt], s_ml[1][wave][rt * 16 + n] = l[rt];
    }
    __syncthreads();
    float *so = (float *)(smem + wave * REGION);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = rt * 16 + n;
      float top = -__builtin_inff(), sum = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, s_ml[0][w][r]);
      const float on = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
      for (int w = 0; w < W; ++w) sum += s_ml[1][w][r] * __builtin_amdgcn_exp2f(s_ml[0][w][r] - on);
      const float f = __builtin_amdgcn_exp2f(m[rt] - on);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *(iu8_v4f *)(so + r * (D + 4) + 16 * dt + 4 * g) = o[rt][dt] * f;
      if (wave == 0 && g == 0) s_m[r] = top, s_il[r] = sum;
    }
    __syncthreads();
    // whole items go out, parts to this workgroup's slots (one for what it begins with, one for what it ends with)
    const bool whole = u0 == 0 && u1 == units;
    const unsigned start = at_unit - u0;  // the item's first unit
    const bool leads = at_unit == blockIdx.x * share;
    float *slot = partial + (size_t)(blockIdx.x * 2 + !leads) * SLOT;
    const int me = anew(tid);
    for (int e = me; e < live * (D / 4); e += 256) {
      const int r = e / (D / 4), d = (e % (D / 4)) * 4;
      const float *x0 = (const float *)smem + r * (D + 4) + d;
      iu8_v4f x = *(const iu8_v4f *)x0;
#pragma unroll
      for (int w = 1; w < W; ++w) x += *(const iu8_v4f *)(x0 + w * (REGION / 4));
      if (!whole) {
        at_store_through(slot + r * D + d, x);
      } else {
        const float il = s_il[r] == 0.f ? 0.f : vs / s_il[r];
        *(iu8_v2u *)(out + s_dst[r] + d) = iu8_v2u{iu8_bf16_pack(x[0] * il, x[1] * il), iu8_bf16_pack(x[2] * il, x[3] * il)};
      }
    }
    if (!whole) {
      if (tid < live) at_store_through(slot + R * D + tid * 4, iu8_v4f{s_m[tid], s_il[tid], 0.f, 0.f});
      iu8_stores_done();
      __syncthreads();
      const int first = start / share, ns = at_parts_of(start, units, share, first, grid);  // the workgroups that have parts
      if (tid == 0) {
        int *count = counter + ((size_t)s * kv_heads + h) * qtiles + qt;
        const int arrived = iu8_arrive(count);
        s_last = arrived == ns - 1;
        if (s_last) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      if (s_last)
        at_join<D, R, 256, 2, RT == 1 ? 16 : 8>(partial + (size_t)first * 2 * SLOT, start == first * share ? 0 : SLOT, 2 * SLOT, ns, live, vs, me, out, s_dst, s_il,
                                  (float *)smem);
    }
    at_unit += u1 - u0;
    if (at_unit == last_unit) return;
    __syncthreads();  // the LDS is the next segment's
    u0 = 0;
    if (++qt == tiles_of(q_)) {
      qt = 0;
      if (++h == (unsigned)kv_heads) {
        h = 0;
        s = at_next([&](int i) { return q_ = sequence(i), tiles_of(q_); }, s, seqs);
        if (s >= seqs) return;
      }
    }
  }
}
