// The paged key/value cache and the attention that reads it (include/saber_iu8.h): checks of arguments, the launch law and the
// launches. No counterpart among the reference's interfaces for this path.
#include <algorithm>
#include <cmath>
#include <cstddef>
#include <string_view>
#include <utility>

#include "../../../include/saber_iu8.h"
#include "rules.h"
#include "util.h"

using namespace iu8;

namespace {

constexpr uint32_t FEW_ROWS = 32;    // rows a kv head and sequence up to which the few-row kernels run (16 or 32 a workgroup)
constexpr uint32_t MANY_ROWS = 128;  // rows a workgroup of the many-row kernels
constexpr int FEW_UNIT_SHIFT = 7, WHOLE_SHIFT = 31;  // log2 of the tokens a unit of the few-row kernels' deal (attn_few.h)
constexpr uint32_t MANY_PARTS = 32;  // parts of an item at most: their maxima and sums lie in one workgroup's LDS when they are joined
// more than 32 rows on the few-row kernels: units a row tile from, units of all up to, and up to for whole prompts
constexpr uint64_t FEW_UNITS_MIN = 8, FEW_UNITS_MAX = 5 * CU_COUNT, FEW_UNITS_MAX_E4M3 = 16 * CU_COUNT, FEW_UNITS_PROMPT = 3 * CU_COUNT, FEW_UNITS_PROMPT_E4M3 = 8 * CU_COUNT;
constexpr uint64_t FEW_BRIEF = 1200;  // units of all below which a part's beginning and end weigh more than its bytes
constexpr uint64_t MANY_TARGET = 2 * CU_COUNT, MANY_LEAST = 320, MANY_LONG = 2048;  // workgroups that the card holds; tokens a part, from; long ones
constexpr uint64_t MANY_UNEVEN = 448, MANY_LONGEST = 8192;  // row tiles that leave an eighth of the places empty, up to; keys that make that worth more parts
constexpr uint32_t I32_MAX = 0x7FFFFFFFu, GRID_MAX = 0xFFFFFFu;  // workgroups of 256 whose threads a launch counts in 32 bits
constexpr uint32_t WHOLE = 0x7FFFFF00u;  // a part that holds any sequence: the positions a table's row may reach

int log2_of(uint32_t x) {
  int s = 0;
  while ((1u << s) < x) ++s;
  return s;
}

struct Plan {
  uint32_t rows;        // a workgroup's: 16 or 32 (few), 128 (many)
  uint64_t qtiles, items, grid;
  int unit_shift;       // few: log2 of the tokens a unit, WHOLE_SHIFT for whole items
  uint32_t chunk, splits;  // many: tokens a part, parts
  uint64_t partial, counter;  // bytes
  bool few() const { return rows <= FEW_ROWS; }
};

// Which kernels, and the grid. Few rows (attn_few.h) up to 32 a kv head and sequence; above, still where a long cache meets so
// few rows that its tiles of 32 make at most a unit a CU (60 new tokens of group 6 on 300 keys, head width 256: 19.7 us against 21.2 of
// the many-row kernel; 60 on 600 24.6 / 31.7; 60 of group 5 on 300, width 128, 13.3 / 16.3) or, on eight units and more, five a CU (200 of group 6 on 1,000 35 / 45; on 1,600, at eight
// a CU, 56 / 44), sixteen a CU in e4m3, which the many-row kernel widens through registers (60 of group 6 on 4,000: 39 / 61; 8 sequences
// of 8 rows each 35 / 44; 32 of them, at 32 a CU, 94 / 93). Of a whole prompt causality hides half, which the few-row kernels walk all the same and
// the many-row kernels do not, so where the new rows are most of the keys the bounds lie lower: three units a CU in bf16 (900 of group 3 on
// themselves, 2.7 units a CU, width 64 / 128 / 256: 14 / 19 / 30 us against 17 / 24 / 39; of group 4, 3.5: 20 / 28 / 45 against 17 / 23 / 39; 900 on 1,200, 4.4: 17 / 24 / 38
// against 18 / 25 / 42), eight in e4m3 (900 of 8 heads on 2, 7.1: 18 / 23 / 34 against 19 / 27 / 44; 1,150, 10: 29 / 40 / 60 against 19 / 27 / 42; 1,400 of 8 on 1, 15: 37 / 48 / 73
// against 25 / 34 / 55), and four units, in e4m3 three, where all make at most one a CU (bf16, 300 of group 4: 11 / 15 / 24 against 11 / 14 / 20, 400: 13 / 17 / 27 against 13 /
// 18 / 29; e4m3, 300: 10 / 13 / 18 against 13 / 17 / 22; of one or two units, 200 on 200, bf16: 21 / 18 at width 256). Their grid, among which the units are dealt level: a workgroup a CU; two where both fit one's LDS and the items
// suffice for nearly all of them to stay whole (256 sequences of 1,000 keys, 8 heads of 128 in e4m3: 256 workgroups 98 us, 512 86; 32 of 2,400 in
// bf16, 256 items: 51 against 55); fewer where few items would be cut into many parts, whose join costs a round of loads for every
// 16 (5,000 keys, 8 heads of 128: 128 workgroups 13.5 us, 256 15.7, 512 20.0; 4 heads of 256 on 131,072: 128 102, 192 92, 256 96).
// Long streams as the others: fewer workgroups gain nothing where tiles are large (64 sequences of up to 8,192, 8 heads of 128, 192 / 256 / 512: 201 / 201 /
// 200; 32 of 20,000 382 / 386 / 388; 128 of 8,192, 4 heads of 256, 192 / 256: 646 / 620) and lose bytes in flight where they are small (64 of up to 8,192, 8 heads of
// 64: 120 / 112 / 105; 32 of 20,000, tiles of 32 rows, 192 / 256: 226 / 206).
// Many rows: parts where the row tiles alone are fewer than the CUs, one workgroup a CU (400 rows of group 6, 76 tiles, on 3,000 keys:
// one part 112 us, three 62, four 68, six 69 to 85), two a CU where the parts are long (512 rows, 96 tiles, on 16,896: two parts
// 395 us, five 248 to 271), three or two each where the row tiles are between one and two a CU and the keys many (1,200 rows of 32 heads on 8
// of 64, 304 tiles, on 20,000: one part 424 us, three 290; 40 on 8 of 128, 376 tiles: 546 and, in two, 525).
// `whole`: no workspaces, every item in one piece; `held`: the tokens that a sequence's row of the page table can hold.
Plan plan(uint32_t seqs, uint32_t max_q, uint32_t max_kv, uint32_t heads, uint32_t kv_heads, uint32_t dim, bool f8, bool whole, uint64_t held) {
  Plan p{};
  const uint64_t rows = (uint64_t)max_q * (heads / kv_heads), units = max_kv ? ((max_kv - 1) >> FEW_UNIT_SHIFT) + 1 : 1;
  const uint64_t all32 = (uint64_t)seqs * kv_heads * ((rows + FEW_ROWS - 1) / FEW_ROWS) * units;
  const bool prompt = (uint64_t)max_q * 8 > (uint64_t)max_kv * 7;  // new rows are most of the keys
  const uint64_t most = prompt ? (f8 ? FEW_UNITS_PROMPT_E4M3 : FEW_UNITS_PROMPT) : f8 ? FEW_UNITS_MAX_E4M3 : FEW_UNITS_MAX;
  const bool sparse = !whole && ((units >= FEW_UNITS_MIN && all32 <= most) || (units >= (prompt && !f8 ? 4 : 3) && all32 <= CU_COUNT));
  p.rows = rows <= 16 ? 16 : rows <= FEW_ROWS || sparse ? FEW_ROWS : MANY_ROWS;
  p.qtiles = (rows + p.rows - 1) / p.rows;
  p.items = (uint64_t)seqs * kv_heads * p.qtiles;
  p.splits = 1, p.chunk = WHOLE, p.unit_shift = WHOLE_SHIFT;
  if (p.few()) {
    const bool two = p.rows == 16 && (f8 || dim < 256) && p.items >= 2 * CU_COUNT, brief = p.items * units < FEW_BRIEF;
    const uint64_t slots = two ? 2 * CU_COUNT
                               : std::clamp<uint64_t>((brief ? 16 : 48) * p.items, brief ? CU_COUNT / 2 : CU_COUNT * 3 / 4, CU_COUNT);
    if (!whole && units > 1) {
      p.unit_shift = FEW_UNIT_SHIFT;
      while (p.unit_shift < WHOLE_SHIFT && p.items * ((held >> p.unit_shift) + 1) > I32_MAX) ++p.unit_shift;  // the kernel counts them in 32 bits
    }
    const bool split = p.unit_shift != WHOLE_SHIFT;
    p.grid = std::min(split ? slots : std::max<uint64_t>(slots, 2 * CU_COUNT), p.items * (split ? units : 1));
    if (split) p.partial = p.grid * 2 * p.rows * (dim + 4) * 4, p.counter = p.items * 4;
    return p;
  }
  uint64_t parts = std::max<uint64_t>(1, CU_COUNT / p.items);
  if (max_kv > MANY_LONG * parts) parts = std::max<uint64_t>(1, MANY_TARGET / p.items);
  if (p.items > CU_COUNT && p.items <= MANY_UNEVEN && max_kv >= MANY_LONGEST) parts = 2 * MANY_TARGET / p.items;
  parts = std::min<uint64_t>({parts, MANY_PARTS, std::max<uint64_t>(1, (max_kv + MANY_LEAST - 1) / MANY_LEAST)});
  if (!whole && parts > 1) {
    p.chunk = (uint32_t)(((max_kv + parts - 1) / parts + 127) / 128 * 128);
    p.splits = (max_kv + p.chunk - 1) / p.chunk;
  }
  p.grid = p.items * p.splits;
  if (p.splits > 1) p.partial = p.grid * p.rows * (dim + 4) * 4, p.counter = p.items * 4;
  return p;
}

// What the plan of any call of up to these sizes takes, caches of either kind: fewer sequences or shorter ones may be cut into more
// parts, and a server allocates once. Few rows: two slots a workgroup, at most 512 of 16 rows or 256 of 32; many: a slot a
// workgroup, at most 512, on long caches 1,024.
void workspace(uint64_t seqs, uint64_t max_q, uint64_t max_kv, uint64_t group, uint64_t kv_heads, uint64_t dim, uint64_t *partial, uint64_t *counter) {
  const uint64_t rows = max_q * group, units = max_kv ? ((max_kv - 1) >> FEW_UNIT_SHIFT) + 1 : 1, row = (dim + 4) * 4;
  auto want = [&](uint64_t items, uint64_t slots, uint64_t a_slot) { *partial = std::max(*partial, slots * a_slot * row), *counter = std::max(*counter, items * 4); };
  if (units < 2) return;
  if (group <= 16) want(seqs * kv_heads, std::min<uint64_t>(2 * CU_COUNT, seqs * kv_heads * units), 2 * 16);
  if (rows > 16) {
    const uint64_t items = std::max(seqs * kv_heads, std::min<uint64_t>(seqs * kv_heads * ((rows + FEW_ROWS - 1) / FEW_ROWS), FEW_UNITS_MAX_E4M3 / FEW_UNITS_MIN));
    want(items, std::min<uint64_t>(CU_COUNT, items * units), 2 * FEW_ROWS);
  }
  const uint64_t items = seqs * kv_heads * ((rows + MANY_ROWS - 1) / MANY_ROWS), parts = std::min<uint64_t>(MANY_PARTS, (max_kv + MANY_LEAST - 1) / MANY_LEAST);
  if (rows > FEW_ROWS && parts > 1) want(std::min(items, MANY_UNEVEN), std::min(items * parts, max_kv < MANY_LONGEST ? MANY_TARGET : 2 * MANY_TARGET), MANY_ROWS);
}

int attn_plan(const char *op, uint32_t seqs, uint32_t max_q, uint32_t max_kv, uint32_t heads, uint32_t kv_heads, uint32_t dim, bool f8, bool whole, uint64_t held, Plan *p) {
  if (!max_q || max_kv > I32_MAX) return fail(SABER_IU8_E_RULE, fmt("%s: at most %u new rows and %u keys a sequence: from 1 and below 2^31", op, max_q, max_kv));
  const uint64_t rows = (uint64_t)max_q * (heads / kv_heads);
  if (rows > I32_MAX || (__int128)seqs * kv_heads * ((rows + MANY_ROWS - 1) / MANY_ROWS) > (int64_t)I32_MAX)
    return fail(SABER_IU8_E_RULE, fmt("%s: %u sequences of up to %u new rows and %u heads pass a launch's 32-bit sizes", op, seqs, max_q, heads));
  *p = plan(seqs, max_q, max_kv, heads, kv_heads, dim, f8, whole, held);
  if (p->grid > GRID_MAX) return fail(SABER_IU8_E_RULE, fmt("%s: %u sequences of up to %u new rows and %u heads pass a launch's 32-bit sizes", op, seqs, max_q, heads));
  return 0;
}

// The kernels' arguments as abi.cpp declares them (natural alignment: the order says it all). An operator of a decode step is a few
// microseconds on the card and called from a serving loop, so its image is laid out here: through a descriptor and its names the
// call took 5.0 us on the host, 2.5 of them the runtime's.
struct Cache {
  const void *k, *v, *k_scale, *v_scale, *table, *kv_len;
};
struct AppendArgs {
  const void *q, *k, *v, *q_out;
  Cache cache;
  const void *cu_q, *q_norm, *k_norm, *inv_freq;
  int32_t q_row, q_head, kv_row, tokens, seqs, shape, form, pages, table_stride;
  float eps;
};
struct AttnArgs {
  const void *q;
  Cache cache;
  const void *cu_q, *out, *partial, *counter;
  int32_t q_row;
  union {
    struct {
      int32_t tokens, seqs, shape, page_shift, pages, table_stride, unit_shift, qtiles;
      float scale;
    } few;
    struct {
      int32_t tokens, shape, page_shift, pages, table_stride, chunk, splits, qtiles;
      float scale;
    } many;
  };
};
static_assert(sizeof(AppendArgs) == 152 && offsetof(AppendArgs, eps) == 148 && sizeof(AttnArgs) == 128 && offsetof(AttnArgs, few.scale) == 124, "as abi.cpp packs them");

Cache cache_of(const saber_iu8_kv_cache *c) {
  const bool f8 = c->kind == SABER_IU8_KV_E4M3;
  return Cache{c->k, c->v, f8 ? c->k_scale : nullptr, f8 ? c->v_scale : nullptr, c->page_table, c->kv_len};
}

// [e4m3][64, 128, 256]
#define NAMES(stem, tail) \
  { {stem "_bf16_d64" tail, stem "_bf16_d128" tail, stem "_bf16_d256" tail}, {stem "_e4m3_d64" tail, stem "_e4m3_d128" tail, stem "_e4m3_d256" tail} }
constexpr const char *APPEND[2][3] = NAMES("kv_append", ""), *FEW16[2][3] = NAMES("attn_few", "_r16"), *FEW32[2][3] = NAMES("attn_few", "_r32"),
                     *MANY[2][3] = NAMES("attn_many", "");
#undef NAMES
int dim_index(uint32_t dim) { return dim == 64 ? 0 : dim == 128 ? 1 : 2; }

const char *kernel_of(const Plan &p, const saber_iu8_kv_cache *c) {
  const auto &names = p.rows == 16 ? FEW16 : p.rows == FEW_ROWS ? FEW32 : MANY;
  return names[c->kind == SABER_IU8_KV_E4M3][dim_index(c->head_dim)];
}

// The scalars of a call on a cache that cache_check has passed, and its plan; `split`: the workspaces are there.
int attn_law(const char *op, const saber_iu8_kv_cache *c, uint32_t q_row, bool packed, uint32_t seqs, uint32_t max_q, uint32_t max_kv, uint32_t heads, float scale,
             bool split, Plan *p) {
  if (q_row % 8 || q_row > I32_MAX || q_row < (uint64_t)heads * c->head_dim)
    return fail(SABER_IU8_E_RULE, fmt("%s: rows of %u elements: whole 16-byte pieces that cover %u heads of %u", op, q_row, heads, c->head_dim));
  if (!std::isfinite(scale)) return fail(SABER_IU8_E_RULE, fmt("%s: the scale must be a number", op));
  return attn_plan(op, seqs, packed ? max_q : 1, max_kv, heads, c->kv_heads, c->head_dim, c->kind == SABER_IU8_KV_E4M3, !split,
                   (uint64_t)c->table_stride * c->page_tokens, p);
}

const saber_iu8_slot *slot(const saber_iu8_desc *d, const char *name) {
  for (uint32_t i = 0; i < d->n_args; ++i)
    if (!strcmp(d->args[i].name, name)) return &d->args[i];
  return nullptr;
}

}  // namespace

int iu8::cache_check(const char *op, const saber_iu8_kv_cache *c, uint32_t heads, uint32_t seqs, uint32_t tokens, bool packed) {
  if (!c) return fail(SABER_IU8_E_ARG, fmt("%s: null cache", op));
  if (!c->k || !c->v || !c->page_table || !c->kv_len) return fail(SABER_IU8_E_ARG, fmt("%s: the cache's k, v, page_table and kv_len must be given", op));
  if (c->kind != SABER_IU8_KV_BF16 && c->kind != SABER_IU8_KV_E4M3) return fail(SABER_IU8_E_ARG, fmt("%s: unknown cache kind %u", op, c->kind));
  if (c->kind == SABER_IU8_KV_E4M3 && (!c->k_scale || !c->v_scale))
    return fail(SABER_IU8_E_ARG, fmt("%s: an e4m3 cache has a k_scale and a v_scale a kv head", op));
  if (((uintptr_t)c->k | (uintptr_t)c->v) % 16) return fail(SABER_IU8_E_ARG, fmt("%s: the cache's k and v must lie on 16 bytes", op));
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(SABER_IU8_E_RULE, fmt("%s: head width %u; the kernels hold 64, 128 and 256", op, c->head_dim));
  if (c->page_tokens < 16 || c->page_tokens > 256 || (c->page_tokens & (c->page_tokens - 1)))
    return fail(SABER_IU8_E_RULE, fmt("%s: pages of %u tokens; a power of two from 16 to 256", op, c->page_tokens));
  if (!heads || !c->kv_heads || heads % c->kv_heads || heads > 0xFFFF || c->kv_heads > 0x7FFF)
    return fail(SABER_IU8_E_RULE, fmt("%s: %u heads over %u kv heads: whole groups, at most 65535 and 32767", op, heads, c->kv_heads));
  if (!c->pages || c->pages > I32_MAX || !c->table_stride || (uint64_t)c->table_stride * c->page_tokens > WHOLE)
    return fail(SABER_IU8_E_RULE, fmt("%s: %u pages, %u of %u tokens a sequence: at least one, positions below 2^31 - 256", op, c->pages, c->table_stride, c->page_tokens));
  if (!seqs || !tokens || seqs >= I32_MAX || tokens > I32_MAX) return fail(SABER_IU8_E_RULE, fmt("%s: %u rows of %u sequences has nothing to do", op, tokens, seqs));
  if (!packed && tokens != seqs) return fail(SABER_IU8_E_RULE, fmt("%s: %u rows of %u sequences without cu_q (one row a sequence)", op, tokens, seqs));
  return 0;
}

// What a hand-edited descriptor could get wrong for these kernels, whose walk over the cache follows their scalars.
int iu8::attn_guard(const saber_iu8_desc *d) {
  auto num = [&](const char *name) -> int64_t {
    const saber_iu8_slot *s = slot(d, name);
    return s && s->kind == SABER_IU8_ARG_I32 ? s->ival : -1;
  };
  const int64_t shape = num("shape"), heads = shape & 0xFFFF, kv_heads = shape >> 16, pages = num("pages"), stride = num("table_stride");
  const bool append = !strncmp(d->kernel, "kv_append_", 10), few = !strncmp(d->kernel, "attn_few_", 9);
  const int64_t form = append ? num("form") : num("page_shift"), shift = form & 0xFF, rot = append ? form >> 16 : 0;
  const char *w = strstr(d->kernel, "_d");
  const int64_t dim = w ? atoi(w + 2) : 0;
  bool ok = shape > 0 && kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && form >= 0 && shift >= 4 && shift <= 8 && pages > 0 && stride > 0 &&
            (stride << shift) <= (int64_t)WHOLE && num("tokens") > 0 && d->grid[1] == 1 && d->grid[2] == 1;
  auto given = [&](const char *name) {
    const saber_iu8_slot *s = slot(d, name);
    return s && s->kind == SABER_IU8_ARG_BUFFER;
  };
  for (const char *name : {"q", "kc", "vc", "table", "kv_len", append ? "q_out" : "out"}) ok = ok && given(name);
  if (strstr(d->kernel, "_e4m3_")) ok = ok && given("k_scale") && given("v_scale");
  if (append) {
    ok = ok && rot % 16 == 0 && rot <= dim && num("seqs") > 0 && given("k") && given("v") && (!rot || given("inv_freq")) &&
         (given("cu_q") || num("tokens") <= num("seqs"));  // without cu_q row t is sequence t's
  } else {
    const bool bound = given("partial") && given("counter");
    ok = ok && form == shift;
    const int64_t qtiles = num("qtiles");
    if (few) {
      const int64_t unit = num("unit_shift"), seqs = num("seqs");
      ok = ok && qtiles > 0 && seqs > 0 && unit >= FEW_UNIT_SHIFT && unit <= WHOLE_SHIFT && (bound || unit == WHOLE_SHIFT) &&
           (__int128)seqs * kv_heads * qtiles * (((stride << shift) >> unit) + 1) <= (int64_t)I32_MAX;
    } else {
      const int64_t chunk = num("chunk"), splits = num("splits");
      ok = ok && qtiles > 0 && splits > 0 && splits <= MANY_PARTS && chunk >= 128 && chunk <= (int64_t)WHOLE && chunk % 128 == 0 && (bound || splits == 1) &&
           d->grid[0] % (uint64_t)(splits * qtiles * kv_heads) == 0;
    }
  }
  return ok ? 0 : fail(SABER_IU8_E_RULE, fmt("%s: scalars that the kernel's walk over the cache does not hold", d->kernel));
}

extern "C" {

uint64_t saber_iu8_kv_bytes(uint32_t pages, uint32_t kv_heads, uint32_t head_dim, uint32_t page_tokens, uint32_t kind) {
  return (uint64_t)pages * kv_heads * head_dim * page_tokens * (kind == SABER_IU8_KV_E4M3 ? 1 : 2);
}

uint64_t saber_iu8_kv_k_offset(uint32_t page, uint32_t kv_head, uint32_t token, uint32_t channel, uint32_t kv_heads, uint32_t head_dim,
                               uint32_t page_tokens, uint32_t kind) {
  const uint64_t size = kind == SABER_IU8_KV_E4M3 ? 1 : 2, e = 16 / size;
  const uint64_t block = ((uint64_t)page * kv_heads + kv_head) * page_tokens * head_dim + (uint64_t)(token / 16) * 16 * head_dim;
  return (block + ((channel / e) * 16 + token % 16) * e + channel % e) * size;
}

uint64_t saber_iu8_kv_v_offset(uint32_t page, uint32_t kv_head, uint32_t token, uint32_t channel, uint32_t kv_heads, uint32_t head_dim,
                               uint32_t page_tokens, uint32_t kind) {
  return ((((uint64_t)page * kv_heads + kv_head) * page_tokens + token) * head_dim + channel) * (kind == SABER_IU8_KV_E4M3 ? 1 : 2);
}

int saber_iu8_kv_append(saber_iu8_ctx *ctx, const void *q, const void *k, const void *v, void *q_out, const saber_iu8_kv_cache *cache,
                        const int32_t *cu_q, uint32_t tokens, uint32_t seqs, uint32_t heads, uint32_t q_row, uint32_t q_head, uint32_t kv_row,
                        const double *inv_freq, uint32_t rot_dim, int interleaved, const void *q_norm, const void *k_norm, float eps, void *stream) {
  if (int rc = cache_check("kv_append", cache, heads, seqs, tokens, cu_q != nullptr)) return rc;
  const uint32_t D = cache->head_dim;
  if (!q || !k || !v || !q_out) return fail(SABER_IU8_E_ARG, "kv_append: null rows");
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)q_norm | (uintptr_t)k_norm) % 16)
    return fail(SABER_IU8_E_ARG, "kv_append: rows and norm weights must lie on 16 bytes");
  if (q_row % 8 || q_head % 8 || kv_row % 8 || q_head < D || q_row > I32_MAX || kv_row > I32_MAX || (uint64_t)(heads - 1) * q_head + D > q_row ||
      (uint64_t)cache->kv_heads * D > kv_row)
    return fail(SABER_IU8_E_RULE, fmt("kv_append: rows of %u (q, heads %u apart) and %u (k, v) elements: whole 16-byte pieces that cover %u and %u heads of %u",
                                      q_row, q_head, kv_row, heads, cache->kv_heads, D));
  if (rot_dim % 16 || rot_dim > D) return fail(SABER_IU8_E_RULE, fmt("kv_append: %u rotated channels; a multiple of 16 up to the head's %u", rot_dim, D));
  if (rot_dim && !inv_freq) return fail(SABER_IU8_E_ARG, "kv_append: a rotation without inv_freq");
  if ((q_norm || k_norm) && !(eps >= 0.f && std::isfinite(eps))) return fail(SABER_IU8_E_RULE, "kv_append: eps must be a number from 0");
  const uint32_t heads_a_wave = 64 / (D / 16), waves = (heads + 2 * cache->kv_heads + heads_a_wave - 1) / heads_a_wave;
  const uint64_t all = (uint64_t)tokens * waves;
  if ((all + 3) / 4 > GRID_MAX) return fail(SABER_IU8_E_RULE, fmt("kv_append: %u rows of %u heads pass a launch's 32-bit sizes", tokens, heads));
  const bool f8 = cache->kind == SABER_IU8_KV_E4M3;
  AppendArgs x{q, k, v, q_out, cache_of(cache), cu_q, q_norm, k_norm, rot_dim ? inv_freq : nullptr, (int32_t)q_row, (int32_t)q_head, (int32_t)kv_row,
               (int32_t)tokens, (int32_t)seqs, (int32_t)(heads | cache->kv_heads << 16),
               (int32_t)(log2_of(cache->page_tokens) | (interleaved ? 0x100 : 0) | rot_dim << 16), (int32_t)cache->pages, (int32_t)cache->table_stride, eps};
  return launch_image(ctx, APPEND[f8][dim_index(D)], (uint32_t)((all + 3) / 4), 256, &x, sizeof x, stream);
}

int saber_iu8_attn_workspace(uint32_t seqs, uint32_t max_q, uint32_t max_kv, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                             uint64_t *partial_bytes, uint64_t *counter_bytes) {
  if (!seqs || !heads || !kv_heads || heads % kv_heads || heads > 0xFFFF || kv_heads > 0x7FFF || (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return fail(SABER_IU8_E_RULE, fmt("attn_workspace: %u sequences of %u heads over %u kv heads of %u", seqs, heads, kv_heads, head_dim));
  Plan p;
  if (int rc = attn_plan("attn_workspace", seqs, max_q, max_kv, heads, kv_heads, head_dim, false, false, max_kv, &p)) return rc;
  uint64_t partial = 0, counter = 0;
  workspace(seqs, max_q, max_kv, heads / kv_heads, kv_heads, head_dim, &partial, &counter);
  if (partial_bytes) *partial_bytes = partial;
  if (counter_bytes) *counter_bytes = counter;
  return 0;
}

int saber_iu8_attn(saber_iu8_ctx *ctx, const void *q, uint32_t q_row, const saber_iu8_kv_cache *cache, const int32_t *cu_q, void *out, uint32_t tokens,
                   uint32_t seqs, uint32_t max_q, uint32_t max_kv, uint32_t heads, float scale, void *partial, void *counter, void *stream) {
  if (int rc = cache_check("attn", cache, heads, seqs, tokens, cu_q != nullptr)) return rc;
  if (!q || !out) return fail(SABER_IU8_E_ARG, "attn: null rows");
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)partial) % 16 || (uintptr_t)counter % 4) return fail(SABER_IU8_E_ARG, "attn: rows and partials must lie on 16 bytes");
  Plan p;
  if (int rc = attn_law("attn", cache, q_row, cu_q != nullptr, seqs, max_q, max_kv, heads, scale, partial && counter, &p)) return rc;
  AttnArgs x{};
  x.q = q, x.cache = cache_of(cache), x.cu_q = cu_q, x.out = out, x.q_row = (int32_t)q_row;
  if (p.partial) x.partial = partial, x.counter = counter;
  const int32_t shape = (int32_t)(heads | cache->kv_heads << 16), page_shift = log2_of(cache->page_tokens), pages = (int32_t)cache->pages,
                stride = (int32_t)cache->table_stride;
  if (p.few()) x.few = {(int32_t)tokens, (int32_t)seqs, shape, page_shift, pages, stride, p.unit_shift, (int32_t)p.qtiles, scale};
  else x.many = {(int32_t)tokens, shape, page_shift, pages, stride, (int32_t)p.chunk, (int32_t)p.splits, (int32_t)p.qtiles, scale};
  return launch_image(ctx, kernel_of(p, cache), (uint32_t)p.grid, 256, &x, sizeof x, stream);
}

int saber_iu8_resolve_attn(const saber_iu8_kv_cache *cache, uint32_t q_row, int packed, uint32_t tokens, uint32_t seqs, uint32_t max_q, uint32_t max_kv,
                           uint32_t heads, float scale, int split, saber_iu8_desc *d) {
  if (!d) return fail(SABER_IU8_E_ARG, "resolve_attn: null descriptor");
  if (int rc = cache_check("resolve_attn", cache, heads, seqs, tokens, packed)) return rc;
  Plan p;
  if (int rc = attn_law("resolve_attn", cache, q_row, packed, seqs, max_q, max_kv, heads, scale, split, &p)) return rc;
  const uint32_t grid[3] = {(uint32_t)p.grid, 1, 1};
  if (int rc = saber_iu8_describe_raw(kernel_of(p, cache), "attn_paged", grid, 256, d)) return rc;
  snprintf(d->op, sizeof d->op, "attn");
  const std::pair<const char *, int64_t> scalars[] = {
      {"q_row", q_row}, {"tokens", tokens}, {"seqs", seqs}, {"shape", heads | (int64_t)cache->kv_heads << 16}, {"page_shift", log2_of(cache->page_tokens)},
      {"pages", cache->pages}, {"table_stride", cache->table_stride}, {"unit_shift", p.unit_shift}, {"chunk", p.chunk}, {"splits", p.splits}, {"qtiles", (int64_t)p.qtiles}};
  for (const auto &[name, value] : scalars)
    if (slot(d, name)) (void)saber_iu8_desc_set_i32(d, name, value);
  for (uint32_t i = 0; i < d->n_args; ++i) {
    saber_iu8_slot &s = d->args[i];
    const std::string_view name = s.name;
    if (name == "scale") s.fval = scale;
    if ((!packed && name == "cu_q") || (cache->kind != SABER_IU8_KV_E4M3 && (name == "k_scale" || name == "v_scale")) ||
        (!p.partial && (name == "partial" || name == "counter")))
      s.kind = SABER_IU8_ARG_NULL_BUFFER;
  }
  if (p.partial) {
    d->n_workspaces = 2;
    snprintf(d->workspaces[0].name, sizeof d->workspaces[0].name, "partial");
    d->workspaces[0].kind = SABER_IU8_WS_SCRATCH, d->workspaces[0].bytes = p.partial;
    snprintf(d->workspaces[1].name, sizeof d->workspaces[1].name, "counter");
    d->workspaces[1].kind = SABER_IU8_WS_PERSISTENT, d->workspaces[1].bytes = p.counter, d->workspaces[1].zero_once = 1;
  }
  return 0;
}

}  // extern "C"
