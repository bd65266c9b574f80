// Blocks of two arrays to other blocks of them: block src[i] to block dst[i]. Pages of a key/value cache, states and tails of a delta-net layer.
// A pair with a number outside the pool is passed over. Bound by the bytes: a workgroup takes 8 KiB of one block, 16 bytes a thread of 512, past the caches (700 pages
// of 512 KiB each way 122 us, 6.0 TB/s in and out; four loads a thread of 256 142, two 137).
#pragma once
#include "iu8_common.h"

constexpr int BLOCK_THREADS = 512, BLOCK_PIECE = 16 * BLOCK_THREADS;

static __device__ __forceinline__ void block_copy_body(unsigned char *__restrict__ a, unsigned char *__restrict__ b, const int *__restrict__ src,
                                                       const int *__restrict__ dst, long long a_bytes, long long b_bytes, int blocks) {
  const int a_pieces = (int)((a_bytes + BLOCK_PIECE - 1) / BLOCK_PIECE), b_pieces = (int)((b_bytes + BLOCK_PIECE - 1) / BLOCK_PIECE);
  const int i = blockIdx.x / (unsigned)(a_pieces + b_pieces), piece = blockIdx.x - i * (a_pieces + b_pieces);
  const int from = src[i], to = dst[i];
  if ((unsigned)from >= (unsigned)blocks || (unsigned)to >= (unsigned)blocks || from == to) return;
  unsigned char *base = piece < a_pieces ? a : b;
  const long long bytes = piece < a_pieces ? a_bytes : b_bytes, at = (long long)(piece < a_pieces ? piece : piece - a_pieces) * BLOCK_PIECE;
  const long long o = at + (int)threadIdx.x * 16;
  if (o < bytes) __builtin_nontemporal_store(__builtin_nontemporal_load((const iu8_v4u *)(base + (size_t)from * bytes + o)), (iu8_v4u *)(base + (size_t)to * bytes + o));
}
