// Device-side helpers of the kernels that work on a paged cache.
#pragma once
#include "common.h"
#include "args.h"

// The sequence of a work item: the last whose first item is not past it (wave-uniform).
template <class A>
DEVI int paged_seq(const A &a, int item) {
    const int lane = lane_id();
    const int first = lane < a.ns ? a.first[lane] : 0x7fffffff;
    return __builtin_amdgcn_readfirstlane(__popcll(__builtin_amdgcn_ballot_w64(first <= item)) - 1);
}

// Pool row of a sequence's row s, or -1 where its page is none of the pool's.
DEVI int pool_row(const PagePool &p, const int *table, int s) {
    const int page = table[s >> p.shift];
    return (unsigned)page < (unsigned)p.n_pages ? (page << p.shift) + (s & ((1 << p.shift) - 1)) : -1;
}
