// SPDX-License-Identifier: Apache-2.0
// kda_tree.h - what the operators of a drafted token tree share: the lengths and trees that
// sequences bring in device memory, ancestors, and where a paged cache keeps a slot.
//
// None of it is trusted: a length, a count, a parent, an accepted node or a page number outside its
// range is read as the nearest thing that exists (an empty context, a child of the context, no page),
// so that no value in these arrays can make a kernel read or write outside its buffers.
#pragma once

#include "k3kda_common.h"

namespace k3kda {

constexpr int TREE_MAX = 64;   // nodes of a tree: one lane of a wave, one bit of an ancestor mask each

struct TreeSeqs {
    int N;               // node rows of each sequence
    const int *lens;     // [B] committed positions
    const int *counts;   // [B] nodes, nullptr: N
    const int *parents;  // [B][N], nullptr: a chain
};

__device__ __forceinline__ int tree_count(const TreeSeqs &t, int b)
{
    return t.counts ? min(max(t.counts[b], 0), t.N) : t.N;
}

// Node n's parent, -1: the committed context.
__device__ __forceinline__ int tree_parent(const TreeSeqs &t, int b, int n)
{
    if (!t.parents) return n - 1;
    const int p = t.parents[(size_t)b * t.N + n];
    return p >= 0 && p < n ? p : -1;
}

// Lane n of a wave holds node n's parent (-1: none; lanes past the nodes too): the mask of node n and
// its ancestors. Each round takes the ancestors of the node reached so far and doubles the reach, so six
// rounds of two shuffles cover 64 nodes (a walk up the parents takes a dependent load for each).
__device__ __forceinline__ uint64_t tree_ancestors(int parent)
{
    const int lane = threadIdx.x & 63;
    uint64_t m = 1ull << lane;
    int p = parent;
#pragma unroll
    for (int i = 0; i < 6; i++) {
        const int at = p < 0 ? lane : p;
        const uint32_t lo = __shfl((uint32_t)m, at, 64), hi = __shfl((uint32_t)(m >> 32), at, 64);
        const int q = __shfl(p, at, 64);
        if (p >= 0) {
            m |= ((uint64_t)hi << 32) | lo;
            p = q;
        }
    }
    return m;
}

// A paged cache: pages [n_pages][page] rows, table [B][max_pages] page numbers.
struct PagedRows {
    const int *table;
    int n_pages, page, max_pages;
};

// Slots that sequence b's table can hold (the host checks that this fits an int).
__device__ __forceinline__ int paged_cap(const PagedRows &c) { return c.max_pages * c.page; }

__device__ __forceinline__ int paged_len(const PagedRows &c, const int *lens, int b)
{
    return min(max(lens[b], 0), paged_cap(c));
}

// Row of the pool that holds slot `pos` (>= 0) of sequence b, -1: there is none.
__device__ __forceinline__ long paged_row(const PagedRows &c, int b, int pos)
{
    const int i = pos / c.page;
    if (i >= c.max_pages) return -1;
    const int p = c.table[(size_t)b * c.max_pages + i];
    return p >= 0 && p < c.n_pages ? (long)p * c.page + pos % c.page : -1;
}

// Host: what every entry point on a paged cache checks of it, K3HIP_OK or an error that is set.
inline int paged_check(const char *who, int B, int N, int n_pages, int page, int max_pages, const void *pages,
                       const int *table, const int *lens)
{
    if (B < 0 || N < 0) K3_FAIL(K3HIP_EINVAL, "%s: B=%d N=%d", who, B, N);
    if (n_pages <= 0 || page <= 0 || max_pages <= 0)
        K3_FAIL(K3HIP_EINVAL, "%s: n_pages=%d page=%d max_pages=%d", who, n_pages, page, max_pages);
    if ((long)max_pages * page + N > 0x7fffff00L)
        K3_FAIL(K3HIP_EINVAL, "%s: %d pages of %d positions a sequence do not fit an int", who, max_pages, page);
    if (B > 0 && (!pages || !table || !lens)) K3_FAIL(K3HIP_EINVAL, "%s: NULL pages, table or lens", who);
    return K3HIP_OK;
}

}  // namespace k3kda
