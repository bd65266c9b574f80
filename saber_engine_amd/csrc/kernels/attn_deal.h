// The walk over a deal's items (attn_few.h): plain arithmetic on counts that the kernel reads from memory, kept apart so that it can be
// run on the host as well. A launch reads the counts more than once, first to sum them, then along the walk. They must not change
// meanwhile; where they do all the same (a sequence released beside a running launch), what the launch writes is undefined, but no walk
// leaves the arrays and no join the workspace: the bounds here cost a few scalar instructions a segment.
#pragma once

constexpr int AT_PARTS = 128;  // parts of an item at most

// The sequence that unit `at` lies in, from sequence s on, whose units begin at `base` (moved along); `seqs` where there is none.
template <class F>
static __host__ __device__ __forceinline__ int at_walk(F units_of, int s, int seqs, unsigned &base, unsigned at) {
  for (; s < seqs; ++s) {
    const unsigned all = units_of(s);
    if (base + all > at) break;
    base += all;
  }
  return s;
}

// The next sequence behind s that has row tiles; `seqs` where there is none.
template <class F>
static __host__ __device__ __forceinline__ int at_next(F tiles_of, int s, int seqs) {
  do ++s;
  while (s < seqs && tiles_of(s) == 0);
  return s;
}

// How many workgroups have parts of the item of `units` units from `start` on, `share` units each, workgroup `first` the first.
static __host__ __device__ __forceinline__ int at_parts_of(unsigned start, unsigned units, unsigned share, unsigned first, unsigned workgroups) {
  const unsigned last = (start + units - 1) / share, end = last < workgroups ? last : workgroups - 1, n = end - first + 1;
  return (int)(n < (unsigned)AT_PARTS ? n : (unsigned)AT_PARTS);
}
