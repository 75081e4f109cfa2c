// Trees of drafted tokens: what their kernels share. A request's nodes are its rows row_starts[r] ..
// row_starts[r + 1] - 1, at most 64 of them, one lane of a wave each.
#pragma once
#include <hip/hip_runtime.h>

#include "kernel_args.h"

struct TreeRows {
    uint32_t row0, n;
};
__device__ __forceinline__ TreeRows tree_rows(const uint32_t *row_starts, uint32_t r, uint32_t rows) {
    const uint32_t s = min(row_starts[r], rows), e = min(row_starts[r + 1], rows);
    return {s, e > s ? e - s : 0u};
}

// The request of a row: the last that starts at or before it, found by a whole wave. Only to be called for
// rows in front of row_starts[requests].
__device__ __forceinline__ uint32_t tree_request(const uint32_t *row_starts, uint32_t requests, uint32_t row) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0, hi = requests;
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 63) / 64, at = lo + lane * step;
        const uint32_t n = __popcll(__builtin_amdgcn_ballot_w64(at < hi && row_starts[min(at, hi - 1)] <= row));
        lo += max(n, 1u) * step - step;
        hi = min(lo + step, hi);
    }
    return lo;
}

// This lane's node's parent (a lane), or -1: a parent comes before its children, anything else is none.
__device__ __forceinline__ int tree_parent(const uint32_t *parents, const TreeRows &q, uint32_t lane) {
    const uint32_t p = lane < q.n ? parents[q.row0 + lane] : ~0u;
    return p < lane ? (int)p : -1;
}

// Its ancestors and itself, a bit each: 1, 2, 4 .. 32 generations.
__device__ __forceinline__ uint64_t tree_lineage(int parent, uint32_t lane, bool there) {
    uint64_t mask = there ? 1ull << lane : 0;
    int up = parent;
#pragma unroll
    for (int i = 0; i < 6; i++) {
        const int at = up < 0 ? (int)lane : up;
        const uint64_t m = __shfl(mask, at);
        const int u = __shfl(up, at);
        if (up >= 0) {
            mask |= m;
            up = u;
        }
    }
    return mask;
}
