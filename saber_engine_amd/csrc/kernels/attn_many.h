// Attention of many new rows a sequence (whole prompts, chunks behind a cached prefix) over the paged cache, causal, with the
// formulas of attn_few.h.
//
// One workgroup: 128 rows of one kv head of one sequence, 32 a wave; row r is new token r / G, head r % G of the group, so every
// head of the group shares the staged keys and a short prompt still fills its rows. K and V come tile by tile (BK tokens, two
// LDS stages): bf16 straight from memory into LDS, e4m3 through registers, widened once for all four waves. Two workgroups a compute
// unit (256 registers a lane, 64 KiB of LDS), so that one's softmax runs under the other's products; up to 128 channels, where the
// registers allow, also under its own (the scores of the next tile in the block of this one's weights: 8,192 tokens of 40 heads of
// 128 channels 696 us -> 672).
//
// Bound by the matrix cores at the clock that they leave (60 % of their cycles busy at 8,192 tokens of 24 heads of 256: 719 to 745 us,
// 1,107 to 1,147 TF/s, where the library's largest plain product reaches 1,348), and on short prompts by the chain of a workgroup's
// beginning and end, about four tiles' time: five prompts of 883 to 2,100 tokens, 40 heads of 128, 180 to 189 us, 138 GF. LDS: 30 % of
// the cycles, no conflicts (e4m3: 14 % of its accesses).
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
  // the longest rows first; a head's tiles lie a launch's heads apart, so that few XCDs (to which workgroups are dealt in turn)
  // hold its keys
  const int items = gridDim.x / splits, split = blockIdx.x / items, item = blockIdx.x % items;
  const int heads_all = items / qtiles, qt = qtiles - 1 - item / heads_all, h = item % heads_all % kv_heads, s = item % heads_all / kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, wave = at_uniform(tid >> 6), n = lane & 31, hf = lane >> 5;

  const int t0 = cu_q ? cu_q[s] : s;
  const int to = cu_q ? cu_q[s + 1] : s + 1, nq = min(to, tokens) - t0;
  const int len = at_len(kv_len, s, table_stride, page_shift), pos = len - (to - t0);  // of the first new row
  const long long all = (long long)max(nq, 0) * G;
  if ((long long)qt * R >= all) return;
  const int live = (int)min((long long)R, all - (long long)qt * R);
  const int i_first = qt * R / G, i_last = (qt * R + live - 1) / G;
  const int kv_end = max(min(len, pos + i_last + 1), 0), free_end = pos + i_first + 1;
  chunk = at_chunk(kv_end, chunk, splits);
  const int ns = kv_end > chunk ? (kv_end + chunk - 1) / chunk : 1;
  if (split >= ns) return;

  __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * TILE];  // K, V of stage 0; K, V of stage 1
  __shared__ float s_il[R];
  __shared__ int s_limit[R];  // the last position that each row sees
  __shared__ long long s_dst[R];
  __shared__ int s_last;

  const int r = qt * R + wave * 32 + n, i = r / G;
  const bool real = wave * 32 + n < live;
  if (hf == 0) s_limit[wave * 32 + n] = real ? pos + i : len - 1;
  const float ks_ = F8 ? k_scale[h] : 1.f, vs = F8 ? v_scale[h] : 1.f, cs = scale * AT_LOG2E * ks_;
  const unsigned flip = cs < 0.f ? 0x80008000u : 0u;  // attn_few.h
  const float c = at_uniform_f(fmaxf(fabsf(cs), 1e-37f));
  if (hf == 0) s_dst[wave * 32 + n] = ((long long)(t0 + i) * heads + h * G + (r - i * G)) * D;
  const int begin = split * chunk, end = kv_end - begin > chunk ? begin + chunk : kv_end;

  const int *row = table + (size_t)s * table_stride;
  const size_t head_elems = (size_t)D << page_shift;
  const int mask = (1 << page_shift) - 1;
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char *)smem;

  // where a tile's blocks of 16 tokens lie (a block past the end or in a hole: page 0, masked later); the pages are looked up a
  // tile ahead
  constexpr int NB = BK / 16;
  typedef size_t places __attribute__((ext_vector_type(NB)));  // (vectors: an array here ends up in memory)
  typedef int page_numbers __attribute__((ext_vector_type(NB)));
  places at{};
  page_numbers page{};
  auto look_up = [&](int tile) {
#pragma unroll
    for (int b = 0; b < NB; ++b) page[b] = row[min((unsigned)(tile + 16 * b) >> page_shift, (unsigned)table_stride - 1u)];
  };
  auto locate = [&](int tile) {
    unsigned holes = 0;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const bool hole = tile + 16 * b >= end || (unsigned)page[b] >= (unsigned)pages;
      holes |= hole ? 1u << b : 0u;
      at[b] = hole ? 0 : (((size_t)page[b] * kv_heads + h) * head_elems + (size_t)((tile + 16 * b) & mask) * D) * ES;
    }
    return holes;
  };
  auto block = [](places of, int first, int more) {  // (the wave's: `more` is uniform)
    size_t x = of[first];
#pragma unroll
    for (int b = first + 1; b < NB; ++b) x = b == first + more ? of[b] : x;
    return x;
  };
  auto swz = [](int t) { return D == 256 ? t & 7 : D == 128 ? t & 3 : t & 1; };

  const unsigned v_off = lane * 16 / ROWB * ROWB + ((lane % (ROWB / 16)) ^ (4 * swz(lane * 16 / ROWB))) * 16;
  constexpr int RAW = F8 ? BK * D / 256 / 16 : 1;  // 16-byte pieces of K (and of V) a thread, e4m3
  iu8_v4u raw[RAW];
  // (a thread's number, made anew: what hangs on it would otherwise be kept across the loop, in registers that it lacks)
  auto thread = [&]() {
    int t = tid;
    asm volatile("" : "+v"(t));
    return t;
  };
  auto fetch = [&](const unsigned char *src, places of) {  // e4m3: a tile of K or of V into registers
    const int me = thread();
#pragma unroll
    for (int x = 0; x < RAW; ++x)  // (a block is D pieces: a wave's 64 lie in one)
      raw[x] = *(const iu8_v4u *)(src + block(of, x * 256 / D, wave * 64 / D) + (unsigned)((x * 256 + me) % D) * 16);
  };
  constexpr int BLK = 16 * ROWB / 1024, LOADS = BK / 16 * BLK;  // wave-loads of 1 KiB a block, a tile
  auto issue_k = [&](int stage, places of) {  // bf16: a tile straight into a stage
#pragma unroll
    for (int x = 0; x < LOADS / 4; ++x) {
      const int ld = x * 4 + wave, part = ld % BLK;
      const size_t from = block(of, x * 4 / BLK, BLK < 4 ? wave / BLK : 0) + part * 1024;
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                   :
                   : "s"(lds0 + stage * 2 * TILE + ld * 1024), "v"(lane * 16), "s"(kc + from)
                   : "memory", "m0");
    }
  };
  auto issue_v = [&](int stage, places of) {
#pragma unroll
    for (int x = 0; x < LOADS / 4; ++x) {
      const int ld = x * 4 + wave, part = ld % BLK;
      const size_t from = block(of, x * 4 / BLK, BLK < 4 ? wave / BLK : 0) + part * 1024;
      // a lane's slot is row t, piece p; it holds piece p ^ 4 swz(t) of the row (of a whole kilobyte's rows, `part` shows in
      // the piece at D = 256 alone)
      const unsigned ov = D == 256 ? v_off ^ ((part & 3) * 128) : v_off;
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                   :
                   : "s"(lds0 + (stage * 2 + 1) * TILE + ld * 1024), "v"(ov), "s"(vc + from)
                   : "memory", "m0");
    }
  };
  auto widen_k = [&](int stage) {
    const int me = thread();
#pragma unroll
    for (int x = 0; x < RAW; ++x) {
      const int piece = x * 256 + me, blk = piece / D, in = piece % D;
      unsigned char *to = smem + stage * 2 * TILE + blk * 16 * ROWB + ((in / 16) * 32 + in % 16) * 16;
      *(iu8_v4u *)to = at_e4m3x8(raw[x][0], raw[x][1]);
      *(iu8_v4u *)(to + 256) = at_e4m3x8(raw[x][2], raw[x][3]);
    }
  };
  auto widen_v = [&](int stage) {
    const int me = thread();
#pragma unroll
    for (int x = 0; x < RAW; ++x) {
      const int piece = x * 256 + me, t = piece / (D / 16), p = piece % (D / 16) * 2;
      unsigned char *to = smem + (stage * 2 + 1) * TILE + t * ROWB + ((p ^ (4 * swz(t))) * 16);
      *(iu8_v4u *)to = at_e4m3x8(raw[x][0], raw[x][1]);
      *(iu8_v4u *)(to + 16) = at_e4m3x8(raw[x][2], raw[x][3]);
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
  const int vrow = 4 * hf + ((lane & 15) >> 2);
  const unsigned v_lane = vrow * ROWB + swz(vrow) * 64 + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;  // ^ 64 mt: channel block mt
  iu8_v4u qf[KS];

  // ---- the steps of a tile
  // V before its product: zeros in what takes no part (rows behind the end, a hole's block), whose NaNs a weight of zero would
  // keep; whether a value that is not finite lies among tokens that some rows see and others do not
  auto clean = [&](int tile, unsigned holes, unsigned char *sv) -> int {
    constexpr int PR = ROWB / 16;  // pieces a row
    const int stop = min(end - tile, BK), me = thread();
    int odd = 0;
    for (int x = stop * PR + me; x < BK * PR; x += 256) *(iu8_v4u *)(sv + x * 16) = iu8_v4u{0, 0, 0, 0};
    if (holes)
      for (int x = me; x < BK * PR; x += 256)
        if (holes >> (x / (16 * PR)) & 1) *(iu8_v4u *)(sv + x * 16) = iu8_v4u{0, 0, 0, 0};
    for (int x = max(free_end - tile, 0) * PR + me; x < stop * PR; x += 256) {
      const iu8_v4u v = *(const iu8_v4u *)(sv + x * 16);
      if (holes >> (x / (16 * PR)) & 1) continue;
#pragma unroll
      for (int w = 0; w < 4; ++w) odd |= at_nonfinite2(v[w]);
    }
    return __syncthreads_or(odd);
  };
  // S^T = K Q^T of a stage's K
  auto scores = [&](const unsigned char *sk, at_v16f (&sc)[HB]) {
    const int ln = (F8 ? thread() : tid) & 63;
    const unsigned char *ka = sk + ((ln >> 4) & 1) * 16 * ROWB + (ln >> 5) * 256 + (ln & 15) * 16;
    iu8_v4u kf[HB][KS];
#pragma unroll
    for (int hb = 0; hb < HB; ++hb)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kf[hb][ks] = *(const iu8_v4u *)(ka + hb * 32 * ROWB + ks * 512);
#pragma unroll
    for (int hb = 0; hb < HB; ++hb) {
      sc[hb] = at_v16f{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) sc[hb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(at_bf(kf[hb][ks]), at_bf(qf[ks]), sc[hb], 0, 0, 0);
    }
  };
  // (The products are read in the block that makes them: behind a branch this compiler can leave too few wait states between a
  // matrix instruction and the first read of its result, seen as wrong scores.)
  auto settle = [&](const at_v16f (&sc)[HB], float (&st)[HB][16]) {
#pragma unroll
    for (int hb = 0; hb < HB; ++hb)
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        float y = sc[hb][x];
        asm volatile("" : "+v"(y));
        st[hb][x] = y;
      }
  };
  // the order of issue: reads ahead of the products by a few (attn_few.h)
  auto order_scores = [&]() {
    constexpr int AHEAD = D == 256 ? (F8 ? 2 : 3) : 4;
    __builtin_amdgcn_sched_group_barrier(AT_DS_READ, AHEAD, 0);
#pragma unroll
    for (int x = 0; x < HB * KS - AHEAD; ++x) {
      __builtin_amdgcn_sched_group_barrier(AT_MFMA, 1, 0);
      __builtin_amdgcn_sched_group_barrier(AT_DS_READ, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(AT_MFMA, AHEAD, 0);
  };
  auto hide = [&](int tile, unsigned holes, float (&st)[HB][16]) {  // what a row does not see
    int ln = lane;
    asm volatile("" : "+v"(ln));  // (what this rare block needs is made here and not kept across the loop)
    const int last = min(s_limit[wave * 32 + (ln & 31)], end - 1) - tile - 4 * (ln >> 5);
#pragma unroll
    for (int hb = 0; hb < HB; ++hb)
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int t = 32 * hb + 8 * (x >> 2) + (x & 3);  // + 4 half
        if (t > last || (holes >> (t >> 4) & 1)) st[hb][x] = -__builtin_inff();
      }
  };
  // The maximum that the weights are taken against moves only when a score passes it by 2^8 or more (and at the first key): until
  // then weights of up to 256 are as exact, and the sums' rescale is saved. Returns it in units of log2.
  auto maximum = [&](const float (&st)[HB][16]) -> float {
    float top = st[0][0];
#pragma unroll
    for (int hb = 0; hb < HB; ++hb)
#pragma unroll
      for (int x = 0; x < 16; ++x) top = fmaxf(top, st[hb][x]);
    top = at_both<32>(top, at_max2);
    if (__any((top - m) * c > 8.f)) {
      const float mn = fmaxf(m, top), f = __builtin_amdgcn_exp2f((m - (mn == -__builtin_inff() ? 0.f : mn)) * c);
      l *= f;
#pragma unroll
      for (int x = 0; x < MT; ++x) o[x] *= f;
      m = mn;
    }
    return m == -__builtin_inff() ? 0.f : m * c;
  };
  auto weights = [&](const float (&st)[HB][16], float mc, unsigned (&pf)[HB][8]) {
#pragma unroll
    for (int hb = 0; hb < HB; ++hb)
#pragma unroll
      for (int x = 0; x < 16; x += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(st[hb][x], c, -mc)), p1 = __builtin_amdgcn_exp2f(fmaf(st[hb][x + 1], c, -mc));
        l += p0 + p1;
        pf[hb][x / 2] = iu8_bf16_pack(p0, p1);
      }
  };
  // the tokens from free_end on by lane arithmetic, for the rows that see them; the product then finds zeros
  auto by_lanes = [&](int tile, unsigned holes, unsigned char *sv, const unsigned (&pf)[HB][8]) {
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int from = max(free_end - tile, 0), to = min(end - tile, BK), last = s_limit[wave * 32 + (ln & 31)] - tile;
#pragma unroll
    for (int hb = 0; hb < HB; ++hb)
#pragma unroll 1
      for (int t = max(from - 32 * hb, 0); t < min(to - 32 * hb, 32); ++t) {
        unsigned w = pf[hb][0];
        const int j = (t >> 3) * 4 + (t & 3), tt = t + 32 * hb;
#pragma unroll
        for (int x = 1; x < 8; ++x) {
          unsigned p = pf[hb][x];
          asm volatile("" : "+v"(p));  // (or the choice becomes an index, and the weights of every tile go to memory)
          w = j >> 1 == x ? p : w;
        }
        const float pj = __shfl(__uint_as_float(j & 1 ? w & 0xFFFF0000u : w << 16), (ln & 31) + 32 * ((t >> 2) & 1));
        if (tt <= last && !(holes >> (tt >> 4) & 1)) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int x = 0; x < 16; x += 4) {
              float v[4];
              at_four<false>(sv + tt * ROWB + ((4 * (mt ^ swz(tt)) + x / 4) * 16) + 8 * (ln >> 5), v);
#pragma unroll
              for (int r2 = 0; r2 < 4; ++r2) o[mt][x + r2] = fmaf(pj, v[r2], o[mt][x + r2]);
            }
        }
      }
    __syncthreads();
    for (int x = thread(); x < BK * (ROWB / 16); x += 256)
      if (x / (ROWB / 16) >= from) *(iu8_v4u *)(sv + x * 16) = iu8_v4u{0, 0, 0, 0};
    __syncthreads();
  };
  auto product = [&](unsigned char *sv, const unsigned (&pf)[HB][8]) {  // O^T += V^T P^T
    constexpr int NP = MT * HB * 2;                                      // two reads each
    unsigned va = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char *)sv + v_lane;
    asm volatile("" : "+v"(va));  // (the addresses are made from it here: kept across the loop they would be registers that it lacks)
    iu8_v2u vf[NP][2];
#pragma unroll
    for (int x = 0; x < NP; ++x) {
      const int mt = x / (2 * HB), t16 = x % (2 * HB);
      auto *pv = (__attribute__((address_space(3))) unsigned char *)(size_t)(va ^ (mt * 64)) + 16 * t16 * ROWB;
      vf[x][0] = __builtin_bit_cast(iu8_v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) at_v4s *)pv));
      vf[x][1] = __builtin_bit_cast(iu8_v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) at_v4s *)(pv + 8 * ROWB)));
    }
#pragma unroll
    for (int x = 0; x < NP; ++x) {
      const int mt = x / (2 * HB), t16 = x % (2 * HB);
      const unsigned *w = &pf[t16 / 2][t16 % 2 * 4];
      o[mt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(at_bf(vf[x][0][0], vf[x][0][1], vf[x][1][0], vf[x][1][1]), at_bf(w[0], w[1], w[2], w[3]), o[mt], 0, 0, 0);
    }
    constexpr int AHEAD = D == 256 ? 2 : 3;
    __builtin_amdgcn_sched_group_barrier(AT_DS_READ, 2 * AHEAD, 1);
#pragma unroll
    for (int x = 0; x < NP - AHEAD; ++x) {
      __builtin_amdgcn_sched_group_barrier(AT_MFMA, 1, 1);
      __builtin_amdgcn_sched_group_barrier(AT_DS_READ, 2, 1);
    }
    __builtin_amdgcn_sched_group_barrier(AT_MFMA, AHEAD, 1);
  };
  auto queries = [&]() {
    const unsigned short *src = q + (size_t)(t0 + (real ? i : 0)) * q_row + (size_t)(h * G + (real ? r - i * G : 0)) * D + 8 * hf;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *(const iu8_v4u *)(src + 16 * ks);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = (qf[ks] ^ flip) & (real ? ~0u : 0u);
      asm volatile("" : "+v"(qf[ks]));  // here, not in the loop, is what waits for them
    }
  };

  if constexpr (D == 256) {
    // a tile at a time; the next one's K and V are on the way
    unsigned holes_next = 0;
    if (begin < end) {
      look_up(begin);
      holes_next = locate(begin);
      if constexpr (F8) {
        fetch(kc, at);
        widen_k(0);
        fetch(vc, at);
        widen_v(0);
      } else {
        issue_k(0, at);
        issue_v(0, at);
      }
      look_up(begin + BK);
    }
    queries();
    arrived();
    int stage = 0;
    for (int tile = begin; tile < end; tile += BK, stage ^= 1) {
      const bool more = tile + BK < end;
      const unsigned holes = holes_next;
      if (more) {
        holes_next = locate(tile + BK);
        if constexpr (F8) {
          fetch(kc, at);
        } else {
          issue_k(stage ^ 1, at);
          issue_v(stage ^ 1, at);
        }
        look_up(tile + 2 * BK);
      }
      unsigned char *sk = smem + stage * 2 * TILE, *sv = sk + TILE;
      const bool special = holes || tile + BK > min(end, free_end);
      int odd = 0;
      if (special) odd = clean(tile, holes, sv);
      float st[HB][16];
      {
        at_v16f sc[HB];
        scores(sk, sc);
        order_scores();
        settle(sc, st);
      }
      if constexpr (F8) {
        if (more) {
          widen_k(stage ^ 1);
          fetch(vc, at);
        }
      }
      if (special) hide(tile, holes, st);
      const float mc = maximum(st);
      unsigned pf[HB][8];
      weights(st, mc, pf);
      if (odd) by_lanes(tile, holes, sv, pf);
      product(sv, pf);
      if constexpr (F8) {
        if (more) widen_v(stage ^ 1);
      }
      arrived();
    }
  } else {
    // A tile's scores are made while the weights of the one before it are, in one block: matrix instructions and the
    // exponentials' lane arithmetic side by side. K is a tile ahead of V: while tile j is weighed, K of j + 1 and V of j are here, K of
    // j + 2 and V of j + 1 on the way.
    unsigned holes = 0, holes_1 = 0, holes_2 = 0;
    float st[2][HB][16];
    if (begin < end) {
      look_up(begin);
      holes = locate(begin);
      look_up(begin + BK);
      if constexpr (F8) {
        fetch(kc, at);
        widen_k(0);
        fetch(vc, at);
        widen_v(0);
      } else {
        issue_k(0, at);
        issue_v(0, at);
      }
      holes_1 = locate(begin + BK);
      look_up(begin + 2 * BK);
      if constexpr (F8) {
        fetch(kc, at);
        widen_k(1);
      } else {
        issue_k(1, at);
      }
    }
    queries();
    arrived();
    if (begin < end) {
      at_v16f sc[HB];
      scores(smem, sc);
      order_scores();
      settle(sc, st[0]);
    }
    __syncthreads();
    auto step = [&](int tile, int stage, float (&now_st)[HB][16], float (&next_st)[HB][16]) {
      unsigned char *sv = smem + (stage * 2 + 1) * TILE;
      const places at_v = at;  // V's, of the tile before K's
      holes_2 = locate(tile + 2 * BK);
      look_up(tile + 3 * BK);
      const bool more = tile + BK < end, more_2 = tile + 2 * BK < end;
      if constexpr (F8) {
        if (more_2) fetch(kc, at);
      } else {
        if (more_2) issue_k(stage, at);
        if (more) issue_v(stage ^ 1, at_v);
      }
      const bool special = holes || tile + BK > min(end, free_end);
      int odd = 0;
      if (special) {
        odd = clean(tile, holes, sv);
        hide(tile, holes, now_st);
      }
      const float mc = maximum(now_st);
      unsigned pf[HB][8];
      {
        // (behind the last tile the scores are of whatever the stage holds, and not looked at)
        at_v16f sc[HB];
        scores(smem + (stage ^ 1) * 2 * TILE, sc);
        weights(now_st, mc, pf);
        // an exponential pair and what feeds it behind each product (lane arithmetic of any kind, seven at a time: 690 us for 671 at
        // 8,192 tokens of 40 heads of 128, 362 for 348 of 32 of 64)
        constexpr int AHEAD = 4, NM = HB * KS;
        __builtin_amdgcn_sched_group_barrier(AT_DS_READ, AHEAD, 0);
#pragma unroll
        for (int x = 0; x < NM; ++x) {
          __builtin_amdgcn_sched_group_barrier(AT_MFMA, 1, 0);
          if (x + AHEAD < NM) __builtin_amdgcn_sched_group_barrier(AT_DS_READ, 1, 0);
          __builtin_amdgcn_sched_group_barrier(AT_VALU, 4, 0);
          __builtin_amdgcn_sched_group_barrier(AT_TRANS, HB * 16 / NM, 0);
        }
        settle(sc, next_st);
      }
      if constexpr (F8) {
        if (more_2) widen_k(stage);
        if (more) fetch(vc, at_v);
      }
      if (odd) by_lanes(tile, holes, sv, pf);
      product(sv, pf);
      if constexpr (F8) {
        if (more) widen_v(stage ^ 1);
      }
      holes = holes_1, holes_1 = holes_2;
      arrived();
    };
    for (int tile = begin; tile < end; tile += 2 * BK) {
      step(tile, 0, st[0], st[1]);
      if (tile + BK < end) step(tile + BK, 1, st[1], st[0]);
    }
  }
  l = at_both<32>(l, at_sum2);
  const int end_n = thread() & 31, end_hf = (thread() & 63) >> 5;
  const bool end_real = wave * 32 + end_n < live;
  if (ns == 1) {
    const float il = l == 0.f ? 0.f : vs / l;
    const long long dst = s_dst[wave * 32 + end_n];
    if (end_real) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int x = 0; x < 16; x += 4)
          *(iu8_v2u *)(out + dst + 32 * mt + 2 * x + 4 * end_hf) =
              iu8_v2u{iu8_bf16_pack(o[mt][x] * il, o[mt][x + 1] * il), iu8_bf16_pack(o[mt][x + 2] * il, o[mt][x + 3] * il)};
    }
    return;
  }
  constexpr size_t SLOT = (size_t)R * (D + 4);
  float *part = partial + (size_t)item * splits * SLOT, *mine = part + (size_t)split * SLOT;
  if (end_real) {
    float *p = mine + (wave * 32 + end_n) * D;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int x = 0; x < 16; x += 4)
        at_store_through(p + 32 * mt + 2 * x + 4 * end_hf, iu8_v4f{o[mt][x], o[mt][x + 1], o[mt][x + 2], o[mt][x + 3]});
    if (end_hf == 0) at_store_through(mine + R * D + (wave * 32 + end_n) * 4, iu8_v4f{m * c, l, 0.f, 0.f});
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
  at_join<D, R, 256, 2, 8>(part, 0, SLOT, ns, live, vs, thread(), out, s_dst, s_il, (float *)smem);
}
