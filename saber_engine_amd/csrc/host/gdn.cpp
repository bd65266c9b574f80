// A delta-net layer's core (include/saber_iu8.h): the short causal convolution, the gated delta rule, and the copies of pages and states that
// fork a sequence. Checks of arguments, the launch law and the launches. No counterpart among the reference's interfaces for this path.
#include <algorithm>
#include <cmath>
#include <cstddef>

#include "../../../include/saber_iu8.h"
#include "rules.h"
#include "util.h"

using namespace iu8;

namespace {

constexpr uint32_t DIM = 128, CHUNK = 64, I32_MAX = 0x7FFFFFFFu, GRID_MAX = 0xFFFFFFu;  // workgroups of 256 whose threads a launch counts in 32 bits
constexpr uint64_t KEYS = 32768, PART = 19456;  // a chunk and key head's, a chunk and value head's bytes of the workspace (delta_chunk.h)
constexpr uint64_t PIECE = 8192;  // a workgroup's bytes of block_copy, of 512 threads
// Chunks and key heads from which a workgroup of the preparation takes the value heads of a key head, up to four, whose rows' products they share:
// without, the card is not full. Three heads against one a workgroup, microseconds: 272 chunks and key heads 17.0 against 15.5, 400 19.6
// against 21.6, 528 20.5 against 26.0, 2064 59 against 76.
constexpr uint64_t PREP_FULL = 384;
// Sequences and heads up to which the recurrent kernel's waves take 16 columns each (512 threads a workgroup), not 32 (256). 1 / 5 / 8 rows,
// microseconds: 48 items 5.4 / 8.5 / 10.9 on 16 columns, 5.7 / 8.8 / 11.2 on 32; 192 items 6.7 / 10.0 / 12.2 and 6.4 / 10.0 / 12.2; 432 items
// 15.4 / 16.4 / 20.3 and 9.9 / 14.1 / 17.8.
constexpr uint64_t STEP_NARROW = 128;
constexpr uint32_t ROW_MAX = 1u << 24;  // elements of a row: a chunk's bytes are counted in 32 bits
// Rows of a sequence up to which the recurrent kernel runs though a workspace is given: 8 and one more for each 32 of its workgroups (sequences
// and heads), from STEP_FEW to STEP_MANY. Measured, microseconds of a call, recurrent against chunks: 1 sequence of 48 heads, 8 / 12 / 16 rows
// 11.0 / 15.2 / 17.9 against 13.5 / 13.7 / 13.3; 16 of 8 heads 12.7 / 17.0 / 19.6 against 15.5 / 15.4 / 15.7; 4 of 48 heads, 12 / 16 / 24 rows
// 17.1 / 20.9 / 27.2 against 22.1; 64 of 8 heads, 16 / 24 / 32 rows 28 / 37 / 47 against 40 / 41 / 42; 64 of 48 heads 129 / 176 / 224 against 176 / 182 / 190.
// (A line through these, not each of them: 16 sequences of 8 heads stay recurrent up to 12 rows, where chunks are a tenth faster; 4 of 48 heads take chunks from 15, up to 16 a twentieth slower.)
constexpr uint64_t STEP_FEW = 10, STEP_MANY = 24;

// The kernels' arguments as abi.cpp declares them (natural alignment: the order says it all).
struct ConvArgs {
  const void *x, *weight, *bias, *tail, *slot, *cu_q, *kept, *out;
  int32_t x_row, out_row, tokens, seqs, channels, slots, run;
};
struct StepArgs {
  const void *q, *k, *v, *a, *b, *a_log, *dt_bias, *state, *slot, *cu_q, *kept, *out;
  int32_t row, ab_row, tokens, seqs, shape, slots;
  float eps, scale;
};
struct PrepArgs {
  const void *q, *k, *a, *b, *a_log, *dt_bias, *slot, *cu_q, *keys, *work;
  int32_t row, ab_row, tokens, seqs, shape, slots, places, many;
  float eps;
};
struct ScanArgs {
  const void *v, *keys, *work, *state, *slot, *cu_q, *out;
  int32_t row, tokens, seqs, shape, slots;
  float scale;
};
struct CopyArgs {
  const void *a, *b, *src, *dst;
  int64_t a_bytes, b_bytes;
  int32_t blocks;
};
static_assert(offsetof(ConvArgs, run) == 88 && offsetof(StepArgs, scale) == 124 && offsetof(PrepArgs, eps) == 112 && offsetof(ScanArgs, scale) == 76 &&
                  offsetof(CopyArgs, blocks) == 48,
              "as abi.cpp packs them");

int rows_check(const char *op, uint32_t tokens, uint32_t seqs, uint32_t slots, bool packed, bool table) {
  if (!seqs || !tokens || seqs >= I32_MAX || tokens > I32_MAX) return fail(SABER_IU8_E_RULE, fmt("%s: %u rows of %u sequences has nothing to do", op, tokens, seqs));
  if (!packed && tokens != seqs) return fail(SABER_IU8_E_RULE, fmt("%s: %u rows of %u sequences without cu_q (one row a sequence)", op, tokens, seqs));
  if (!slots || slots > I32_MAX) return fail(SABER_IU8_E_RULE, fmt("%s: %u slots; from 1 and below 2^31", op, slots));
  if (!table && slots < seqs) return fail(SABER_IU8_E_RULE, fmt("%s: %u slots for %u sequences, and no table of them", op, slots, seqs));
  return 0;
}

int heads_check(const char *op, uint32_t key_heads, uint32_t heads) {
  if (!heads || !key_heads || heads % key_heads || heads > 0xFFFF || key_heads > 0x7FFF)
    return fail(SABER_IU8_E_RULE, fmt("%s: %u heads over %u key heads: whole groups, at most 65535 and 32767", op, heads, key_heads));
  return 0;
}

int width_check(const char *op, uint32_t channels, uint32_t width) {
  if (width < 2 || width > 4) return fail(SABER_IU8_E_RULE, fmt("%s: a convolution of %u inputs; the kernels hold 2, 3 and 4", op, width));
  if (!channels || channels % 8 || channels > I32_MAX) return fail(SABER_IU8_E_RULE, fmt("%s: %u channels; a multiple of 8", op, channels));
  return 0;
}

int copy(saber_iu8_ctx *ctx, const char *op, void *a, void *b, uint64_t a_bytes, uint64_t b_bytes, uint32_t blocks, const int32_t *src, const int32_t *dst, uint32_t n,
         void *stream) {
  if (!src || !dst) return fail(SABER_IU8_E_ARG, fmt("%s: src and dst must be given", op));
  if (!ctx) return fail(SABER_IU8_E_ARG, fmt("%s: null argument", op));
  if (!n) return 0;
  const uint64_t pieces = (a_bytes + PIECE - 1) / PIECE + (b_bytes + PIECE - 1) / PIECE;
  if ((__int128)pieces * n > GRID_MAX / 2) return fail(SABER_IU8_E_RULE, fmt("%s: %u copies of %llu bytes pass a launch's 32-bit sizes", op, n, (unsigned long long)(a_bytes + b_bytes)));
  CopyArgs x{a, b, src, dst, (int64_t)a_bytes, (int64_t)b_bytes, (int32_t)blocks};
  return launch_image(ctx, "block_copy", (uint32_t)(pieces * n), 512, &x, sizeof x, stream);
}

}  // namespace

extern "C" {

int saber_iu8_gdn_conv(saber_iu8_ctx *ctx, const void *x, uint32_t x_row, const void *weight, const void *bias, void *tail, uint32_t slots, const int32_t *slot,
                       const int32_t *cu_q, const int32_t *kept, void *out, uint32_t out_row, uint32_t tokens, uint32_t seqs, uint32_t channels, uint32_t width,
                       void *stream) {
  if (!x || !weight || !tail || !out) return fail(SABER_IU8_E_ARG, "gdn_conv: x, weight, tail and out must be given");
  if (((uintptr_t)x | (uintptr_t)weight | (uintptr_t)bias | (uintptr_t)tail | (uintptr_t)out) % 16)
    return fail(SABER_IU8_E_ARG, "gdn_conv: rows, weights and tails must lie on 16 bytes");
  if (int rc = rows_check("gdn_conv", tokens, seqs, slots, cu_q, slot)) return rc;
  if (int rc = width_check("gdn_conv", channels, width)) return rc;
  if (x_row % 8 || out_row % 8 || x_row < channels || out_row < channels || x_row > I32_MAX || out_row > I32_MAX)
    return fail(SABER_IU8_E_RULE, fmt("gdn_conv: rows of %u and %u elements: whole 16-byte pieces that cover %u channels", x_row, out_row, channels));
  const uint64_t per = (channels / 8 + 255) / 256;
  // Rows a thread: as many as leave a workgroup a CU. Measured at 10240 channels, microseconds with runs of 1 / 2 / 4 / 8 / 16 rows: 64 sequences
  // of a row 4.4 / 4.8 / 6.5 / 9.6 / 15.9, 200 rows 5.3 / 4.8 / 4.6 / 5.4 / 7.2, 1000 rows 19.6 / 14.4 / 11.1 / 11.3 / 12.2, 6812 rows
  // 111 / 77 / 57 / 53 / 54.
  uint32_t run = 1;
  while (run < 8 && (uint64_t)tokens / (2 * run) * per >= CU_COUNT) run *= 2;
  const uint64_t grid = (tokens + run - 1) / run * per;
  if (grid > GRID_MAX) return fail(SABER_IU8_E_RULE, fmt("gdn_conv: %u rows of %u channels pass a launch's 32-bit sizes", tokens, channels));
  ConvArgs a{x, weight, bias, tail, slot, cu_q, kept, out, (int32_t)x_row, (int32_t)out_row, (int32_t)tokens, (int32_t)seqs, (int32_t)channels, (int32_t)slots, (int32_t)run};
  return launch_image(ctx, width == 2 ? "delta_conv_w2" : width == 3 ? "delta_conv_w3" : "delta_conv_w4", (uint32_t)grid, 256, &a, sizeof a, stream);
}

int saber_iu8_gdn_workspace(uint32_t tokens, uint32_t seqs, uint32_t max_q, uint32_t key_heads, uint32_t heads, uint64_t *bytes) {
  if (int rc = rows_check("gdn_workspace", tokens, seqs, seqs, true, true)) return rc;
  if (int rc = heads_check("gdn_workspace", key_heads, heads)) return rc;
  if (!bytes) return fail(SABER_IU8_E_ARG, "gdn_workspace: null argument");
  *bytes = max_q <= STEP_FEW ? 0 : ((uint64_t)tokens / CHUNK + seqs) * (key_heads * KEYS + heads * PART);
  return 0;
}

int saber_iu8_gdn(saber_iu8_ctx *ctx, const void *q, const void *k, const void *v, uint32_t row, const void *a, const void *b, uint32_t ab_row, const float *a_log,
                  const float *dt_bias, float *state, uint32_t slots, const int32_t *slot, const int32_t *cu_q, const int32_t *kept, void *out, uint32_t tokens,
                  uint32_t seqs, uint32_t max_q, uint32_t key_heads, uint32_t heads, float eps, float scale, void *workspace, void *stream) {
  if (!k || !v || !a || !b || !a_log || !dt_bias || !state || (out && !q)) return fail(SABER_IU8_E_ARG, "gdn: rows, gates, a_log, dt_bias and the state must be given");
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)state | (uintptr_t)out | (uintptr_t)workspace) % 16)
    return fail(SABER_IU8_E_ARG, "gdn: rows, state and workspace must lie on 16 bytes");
  if (((uintptr_t)a | (uintptr_t)b) % 2 || ((uintptr_t)a_log | (uintptr_t)dt_bias) % 4) return fail(SABER_IU8_E_ARG, "gdn: gates, a_log and dt_bias must lie on their elements");
  if (int rc = rows_check("gdn", tokens, seqs, slots, cu_q, slot)) return rc;
  if (int rc = heads_check("gdn", key_heads, heads)) return rc;
  if (!max_q) return fail(SABER_IU8_E_RULE, "gdn: at most 0 new rows a sequence");
  if (row % 8 || row > ROW_MAX || row < (uint64_t)heads * DIM || ab_row > I32_MAX || ab_row < heads)
    return fail(SABER_IU8_E_RULE, fmt("gdn: rows of %u elements (gates %u): whole 16-byte pieces that cover %u heads of 128", row, ab_row, heads));
  if (!(eps >= 0.f && std::isfinite(eps)) || !std::isfinite(scale)) return fail(SABER_IU8_E_RULE, "gdn: eps must be a number from 0, the scale a number");
  const int32_t shape = (int32_t)(heads | key_heads << 16);
  const uint64_t items = (uint64_t)seqs * heads;
  if (!workspace || kept || !out || !cu_q || max_q <= std::min(std::max(8 + items / 32, STEP_FEW), STEP_MANY)) {
    if (items > GRID_MAX) return fail(SABER_IU8_E_RULE, fmt("gdn: %u sequences of %u heads pass a launch's 32-bit sizes", seqs, heads));
    StepArgs x{q, k, v, a, b, a_log, dt_bias, state, slot, cu_q, kept, out, (int32_t)row, (int32_t)ab_row, (int32_t)tokens, (int32_t)seqs, shape, (int32_t)slots, eps, scale};
    const bool narrow = items <= STEP_NARROW;
    return launch_image(ctx, narrow ? "delta_step_c16" : "delta_step_c32", (uint32_t)items, narrow ? 512 : 256, &x, sizeof x, stream);
  }
  const uint64_t places = (uint64_t)tokens / CHUNK + seqs, group = heads / key_heads;
  const uint64_t many = places * key_heads >= PREP_FULL ? std::min<uint64_t>(group, 4) : 1;
  const uint64_t preps = (places * key_heads + 7) / 8 * 8 * ((group + many - 1) / many);
  // Pairs of waves a workgroup of the walk: two, in twice the workgroups, while each has a CU of its own, else four. Microseconds of 4096 rows,
  // two / four: 48 heads 111 / 128, 64 heads 116 / 129, 80 heads 209 / 133, 2 x 48 heads 219 / 149.
  const uint64_t pairs = items * 4 <= CU_COUNT ? 2 : 4, walks = (items + 7) / 8 * 8 * (8 / pairs);
  if (preps > GRID_MAX || walks > GRID_MAX * 2 / pairs)
    return fail(SABER_IU8_E_RULE, fmt("gdn: %u rows of %u sequences and %u heads pass a launch's 32-bit sizes", tokens, seqs, heads));
  unsigned char *const keys = (unsigned char *)workspace, *const parts = keys + places * key_heads * KEYS;
  PrepArgs p{q, k, a, b, a_log, dt_bias, slot, cu_q, keys, parts, (int32_t)row, (int32_t)ab_row, (int32_t)tokens, (int32_t)seqs, shape, (int32_t)slots, (int32_t)places, (int32_t)many, eps};
  if (int rc = launch_image(ctx, "delta_prep", (uint32_t)preps, 256, &p, sizeof p, stream)) return rc;
  ScanArgs x{v, keys, parts, state, slot, cu_q, out, (int32_t)row, (int32_t)tokens, (int32_t)seqs, shape, (int32_t)slots, scale};
  return launch_image(ctx, pairs == 2 ? "delta_scan_w2" : "delta_scan_w4", (uint32_t)walks, 128 * (uint32_t)pairs, &x, sizeof x, stream);
}

int saber_iu8_kv_copy(saber_iu8_ctx *ctx, const saber_iu8_kv_cache *c, const int32_t *src, const int32_t *dst, uint32_t n, void *stream) {
  if (int rc = cache_check("kv_copy", c, c ? c->kv_heads : 0, 1, 1, false)) return rc;
  const uint64_t bytes = saber_iu8_kv_bytes(1, c->kv_heads, c->head_dim, c->page_tokens, c->kind);
  return copy(ctx, "kv_copy", c->k, c->v, bytes, bytes, c->pages, src, dst, n, stream);
}

int saber_iu8_gdn_copy(saber_iu8_ctx *ctx, float *state, void *tail, uint32_t slots, uint32_t heads, uint32_t channels, uint32_t width, const int32_t *src,
                       const int32_t *dst, uint32_t n, void *stream) {
  if (!state || !tail) return fail(SABER_IU8_E_ARG, "gdn_copy: state and tail must be given");
  if (((uintptr_t)state | (uintptr_t)tail) % 16) return fail(SABER_IU8_E_ARG, "gdn_copy: state and tail must lie on 16 bytes");
  if (int rc = heads_check("gdn_copy", 1, heads)) return rc;
  if (int rc = width_check("gdn_copy", channels, width)) return rc;
  if (!slots || slots > I32_MAX) return fail(SABER_IU8_E_RULE, fmt("gdn_copy: %u slots; from 1 and below 2^31", slots));
  return copy(ctx, "gdn_copy", state, tail, (uint64_t)heads * DIM * DIM * 4, (uint64_t)(width - 1) * channels * 2, slots, src, dst, n, stream);
}

}  // extern "C"
