// Shared device helpers of the paged key/value cache and the attention that reads it.
//
// CACHE ORDER (gfx950 device-final; E = the elements of 16 bytes: 8 bf16 or 16 e4m3). A page holds `page_tokens` tokens (a
// power of two, 16 to 256) of every kv head; page p, head h start at element (p * kv_heads + h) * page_tokens * D in both arrays.
//   K   blocks of 16 tokens, [D / E][16 tokens][E]: 64 lanes x 16 bytes in a row are 16 tokens x 4 pieces, which is the operand
//       of a 16x16x32 MFMA (bf16; two of them for e4m3), and 32 tokens x 2 pieces the one of a 32x32x16 MFMA: both kinds of kernel
//       read whole lines and no lane exchanges anything.
//   V   [token][D]. Its operand wants several tokens of one channel a lane, which the LDS's transposing reads give.
// A block of 16 tokens is the same 16 * D elements in both arrays, contiguous.
//
// A sequence's tokens lie in the pages of its row of the page table. An entry outside 0 .. pages - 1 is a hole: its keys take no
// part and nothing is written through it. Lengths are bounded by the table's row, so no length makes a kernel read past either.
#pragma once
#include "iu8_common.h"

typedef __bf16 at_v8bf __attribute__((ext_vector_type(8)));
typedef float at_v16f __attribute__((ext_vector_type(16)));
typedef short at_v4s __attribute__((ext_vector_type(4)));

// what a scheduling group counts
constexpr int AT_VALU = 0x2, AT_MFMA = 0x8, AT_DS_READ = 0x100, AT_TRANS = 0x400;

// A lane's value beside the one of lane ^ 32 (or ^ 16): what both have, by one exchange between registers.
template <int X, class F>
static __device__ __forceinline__ float at_both(float v, F f) {
  const unsigned u = __float_as_uint(v);
  iu8_v2u r;
  if constexpr (X == 32) r = __builtin_bit_cast(iu8_v2u, __builtin_amdgcn_permlane32_swap(u, u, false, false));
  else r = __builtin_bit_cast(iu8_v2u, __builtin_amdgcn_permlane16_swap(u, u, false, false));
  return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
static __device__ __forceinline__ float at_max2(float a, float b) { return fmaxf(a, b); }
static __device__ __forceinline__ float at_sum2(float a, float b) { return a + b; }

static __device__ __forceinline__ int at_uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

static __device__ __forceinline__ float at_uniform_f(float x) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x))); }

// Tokens of sequence s, bounded by what its row of the page table can hold.
static __device__ __forceinline__ int at_len(const int *kv_len, int s, int table_stride, int page_shift) {
  const long long most = (long long)table_stride << page_shift;
  const int n = kv_len[s];
  return n < 0 ? 0 : (long long)n > most ? (int)most : n;
}

// The sequence that row t belongs to when rows are packed (cu[s] .. cu[s + 1] - 1), by one wave: the number of ends at or before
// t. `seqs` when t lies behind the last sequence.
static __device__ __forceinline__ int at_find(const int *__restrict__ cu, int seqs, int t) {
  int s = 0;
  for (int base = 0; base < seqs; base += 64) {
    const int i = base + (int)(threadIdx.x & 63);
    const bool before = i < seqs && cu[i + 1] <= t;
    s += __popcll(__ballot(before));
  }
  return s;
}

static __device__ __forceinline__ at_v8bf at_bf(iu8_v4u x) { return __builtin_bit_cast(at_v8bf, x); }
static __device__ __forceinline__ at_v8bf at_bf(unsigned a, unsigned b, unsigned c, unsigned d) { return at_bf(iu8_v4u{a, b, c, d}); }

// Two e4m3 values (bytes 0, 1 or 2, 3 of x) as packed bf16: exact, every e4m3 value is a bf16 value.
template <bool HI>
static __device__ __forceinline__ unsigned at_e4m3_bf16(unsigned x) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)x, 1.f, HI));
}
// Eight e4m3 values -> eight bf16.
static __device__ __forceinline__ iu8_v4u at_e4m3x8(unsigned lo, unsigned hi) {
  return iu8_v4u{at_e4m3_bf16<false>(lo), at_e4m3_bf16<true>(lo), at_e4m3_bf16<false>(hi), at_e4m3_bf16<true>(hi)};
}

// A packed pair of bf16 holds an infinity or a NaN.
static __device__ __forceinline__ bool at_nonfinite2(unsigned x) { return (x & 0x7F80u) == 0x7F80u || (x & 0x7F800000u) == 0x7F800000u; }

// A packed quadruple of e4m3 holds a NaN (it has no infinities).
static __device__ __forceinline__ bool at_e4m3_nan4(unsigned x) { return (((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0; }
// Four neighbouring values of an LDS row as f32.
template <bool F8>
static __device__ __forceinline__ void at_four(const unsigned char *p, float (&v)[4]) {
  iu8_v2u x;
  if constexpr (F8) {
    const unsigned y = *(const unsigned *)p;
    x = iu8_v2u{at_e4m3_bf16<false>(y), at_e4m3_bf16<true>(y)};
  } else {
    x = *(const iu8_v2u *)p;
  }
  v[0] = __uint_as_float(x[0] << 16), v[1] = __uint_as_float(x[0] & 0xFFFF0000u);
  v[2] = __uint_as_float(x[1] << 16), v[3] = __uint_as_float(x[1] & 0xFFFF0000u);
}

// f32 partials of a split: 16 bytes a store / load that are coherent across the XCDs' L2s by themselves (iu8_common.h). The loads are
// buffer loads, whose cache policy (both scope bits) the compiler lets one name at 16 bytes and still counts, so many can be in
// flight; `offset` in bytes from the uniform address the resource was made of.
static __device__ __forceinline__ void at_store_through(float *p, iu8_v4f v) { iu8_store_through((int *)p, __builtin_bit_cast(iu8_v4i, v)); }
static __device__ __forceinline__ __amdgpu_buffer_rsrc_t at_resource(const float *p) {
  return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, 0xFFFFFFFFu, 0x00020000);
}
static __device__ __forceinline__ iu8_v4f at_load_through(__amdgpu_buffer_rsrc_t r, unsigned offset) {
  return __builtin_bit_cast(iu8_v4f, __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 1 | 16));
}
