// The step around trees of drafted tokens: what the target pass needs in front of it and what the accepted
// path leaves of the paged cache, gfx950.
//
//  * ctox_tree_plan_gfx950: every node's ancestors as a 64-bit mask and its position. A wave takes a request, a
//    lane a node; six shuffles of (mask, parent) reach 63 generations.
//  * ctox_paged_commit_gfx950: token path[j] of a request's nodes moves to the place of node j, in the pages of all
//    layers. path rises, so path[j] >= j and no token is overwritten before it was read as long as each
//    byte column goes through the tokens in order: a thread owns a column, no barrier is needed. The
//    request's length and descriptors are cut by one of its workgroups.
//  * ctox_free_mark_gfx950, ctox_free_list_gfx950: slots that no live page of any request holds, ascending. The tables
//    themselves say what is in use, so shared pages need no counts: every live page sets its slot's bit
//    (whole words, their order does not matter), then a workgroup takes 8192 slots and counts the free ones in
//    front of them for itself. ctox_free_small_gfx950 does it in one launch.
//  * ctox_paged_fork_gfx950: a request's table copied to another's place; a last page that is part-filled is copied
//    to a free slot in all layers. Every workgroup counts for itself how many slots the forks before its own take.
// All are bound by launch latency and a few dependent loads: plan 3.0 us (512 trees of 64), commit 6.3 (128 requests, 8
// layers), free slots 7.6 in one launch, 1.7 + 6.6 + 7.2 in three (16 requests of up to 2048 pages), fork 8.0 (32 forks
// of 8 layers).
#include <hip/hip_runtime.h>

#include "kernel_args.h"
#include "lds_barrier.h"
#include "tree.h"

extern "C" __global__ __launch_bounds__(256) void ctox_tree_plan_gfx950(TreePlanArgs a) {
    const uint32_t lane = threadIdx.x & 63, r = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r < a.requests) {
        const TreeRows q = tree_rows(a.row_starts, r, a.rows);
        if (q.n > CTOX_TREE_NODES) {  // not a tree of these kernels
            for (uint32_t i = lane; i < q.n; i += 64) a.masks[q.row0 + i] = 0;
            if (lane == 0) a.depths[r] = ~0u;
        } else {
            const bool there = lane < q.n;
            const uint64_t mask = tree_lineage(tree_parent(a.parents, q, lane), lane, there);
            const uint32_t depth = __popcll(mask), tokens = a.tokens[r];
            if (there) {
                a.masks[q.row0 + lane] = mask;
                a.positions[q.row0 + lane] = (tokens > q.n ? tokens - q.n : 0u) + depth - 1;
            }
            uint32_t deepest = depth;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) deepest = max(deepest, (uint32_t)__shfl_xor((int)deepest, o));
            if (lane == 0) a.depths[r] = deepest;
        }
    }
    const uint32_t total = min(a.row_starts[a.requests], a.rows);
    for (uint32_t i = total + blockIdx.x * 256 + threadIdx.x; i < a.rows; i += gridDim.x * 256) a.masks[i] = 0;
}

// ---------------------------------------------------------------------------
// the accepted path's tokens closed up
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void commit_move(const uint64_t *from, const uint64_t *to, uint32_t moves, uint8_t *base) {
    // Loads of eight tokens are under way at once. A later token is never at an earlier one's new place.
    for (uint32_t j0 = 0; j0 < moves; j0 += 8) {
        T x[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (j0 + i < moves) x[i] = *(const T *)(base + from[j0 + i]);
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (j0 + i < moves) *(T *)(base + to[j0 + i]) = x[i];
    }
}

// grid (columns of all layers / 256, requests)
extern "C" __global__ __launch_bounds__(256) void ctox_paged_commit_gfx950(PagedCommitArgs a) {
    __shared__ uint64_t from[CTOX_TREE_NODES], to[CTOX_TREE_NODES];
    __shared__ uint32_t info[3];
    const uint32_t tid = threadIdx.x, r = blockIdx.y;
    const PagedKvDesc *desc = a.desc + (size_t)r * a.max_pages;
    if (tid < 64) {
        const TreeRows q = tree_rows(a.row_starts, r, a.rows);
        const uint32_t count = a.counts[r], tokens = a.tokens[r], past = tokens - q.n;
        const bool release = count == CTOX_TREE_RELEASE;
        uint32_t code = 0;
        if (!release && (q.n > tokens || count > q.n || count > CTOX_TREE_NODES)) code = 1;
        if (tokens > (uint64_t)a.max_pages * a.page_tokens) code = 1;
        const uint32_t kept = release || code ? 0 : count;
        const bool mine = tid < kept;
        const uint32_t node = mine ? a.path[q.row0 + tid] : 0;
        const uint32_t before = __shfl_up(node, 1);
        bool bad = mine && (node >= q.n || node < tid || (tid && node <= before));
        const bool move = mine && !bad && node != tid;
        if (move) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t pos = past + (i ? tid : node), p = pos / a.page_tokens;
                const PagedKvDesc d = desc[p];
                if (d.precision == 0 || d.physical_slot >= a.q4_slots || d.first_token != p * a.page_tokens) {
                    bad = true;
                } else {
                    const uint64_t at = (uint64_t)d.physical_slot * a.q4_page_bytes +
                                        (uint64_t)(pos - d.first_token) * a.token_bytes;
                    (i ? to : from)[tid] = at;
                }
            }
        }
        const uint64_t moving = __builtin_amdgcn_ballot_w64(move);
        if (!code && __builtin_amdgcn_ballot_w64(bad)) code = 2;
        // (a path that rises moves everything behind the first node that moves)
        if (tid == 0) {
            info[0] = code;
            info[1] = moving ? (uint32_t)__ffsll((unsigned long long)moving) - 1 : kept;
            info[2] = kept;
            if (blockIdx.x == 0) {
                a.status[r] = code;
                a.new_tokens[r] = code ? tokens : release ? 0 : past + kept;
            }
        }
    }
    __syncthreads();
    if (info[0]) return;
    const uint32_t first = info[1], moves = info[2] - min(first, info[2]);
    const uint32_t columns = a.token_bytes / a.unit, c = blockIdx.x * 256 + tid;
    if (moves && c < columns * a.layers) {
        uint8_t *base = a.pools[c / columns] + (size_t)(c % columns) * a.unit;
        if (a.unit == 16) commit_move<uint4>(from + first, to + first, moves, base);
        else commit_move<uint32_t>(from + first, to + first, moves, base);
    }
    if (blockIdx.x == 0) {
        const uint32_t tokens = a.tokens[r];
        const TreeRows q = tree_rows(a.row_starts, r, a.rows);
        const uint32_t now = a.counts[r] == CTOX_TREE_RELEASE ? 0 : tokens - q.n + info[2];
        const uint32_t pages = tokens / a.page_tokens + (tokens % a.page_tokens != 0);
        for (uint32_t p = now / a.page_tokens + tid; p < pages; p += 256) {
            const uint32_t at = p * a.page_tokens;
            a.desc[(size_t)r * a.max_pages + p].tokens = now > at ? min(now - at, a.page_tokens) : 0;
        }
    }
}

// ---------------------------------------------------------------------------
// free slots
// ---------------------------------------------------------------------------
extern "C" __global__ __launch_bounds__(256) void ctox_free_clear_gfx950(FreeSlotsArgs a) {
    const uint32_t words = a.words[0] + a.words[1];
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < words; i += gridDim.x * 256) a.used[i] = 0;
}

// grid (page groups, requests)
extern "C" __global__ __launch_bounds__(256) void ctox_free_mark_gfx950(FreeSlotsArgs a) {
    const uint32_t r = blockIdx.y, tokens = a.tokens[r];
    const uint32_t pages = min(tokens / a.page_tokens + (tokens % a.page_tokens != 0), a.max_pages);
    for (uint32_t p = blockIdx.x * 256 + threadIdx.x; p < pages; p += gridDim.x * 256) {
        const PagedKvDesc d = a.desc[(size_t)r * a.max_pages + p];
        const uint32_t kind = d.precision ? 0 : 1;
        if (d.physical_slot < a.slots[kind])
            atomicOr(&a.used[(kind ? a.words[0] : 0) + d.physical_slot / 32], 1u << (d.physical_slot & 31));
    }
}

// grid (8192 slots, 2 pools): a thread takes a word
extern "C" __global__ __launch_bounds__(256) void ctox_free_list_gfx950(FreeSlotsArgs a) {
    __shared__ uint32_t sums[3][4];
    const uint32_t kind = blockIdx.y, words = a.words[kind], slots = a.slots[kind], tid = threadIdx.x, lane = tid & 63;
    if (blockIdx.x * 256 >= words) {
        if (blockIdx.x == 0 && tid == 0) a.counts[kind] = 0;
        return;
    }
    const uint32_t *used = a.used + (kind ? a.words[0] : 0);
    auto free_of = [&](uint32_t w) {
        const uint32_t left = slots - 32 * w;
        return ~used[w] & (left < 32 ? (1u << left) - 1 : ~0u);
    };
    const uint32_t w0 = blockIdx.x * 256, me = w0 + tid;
    uint32_t before = 0, all = 0;
    for (uint32_t w = tid; w < words; w += 256) {
        const uint32_t n = __popc(free_of(w));
        all += n;
        if (w < w0) before += n;
    }
    const uint32_t mine = me < words ? free_of(me) : 0;
    uint32_t in = __popc(mine);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(in, o);
        if ((int)lane >= o) in += x;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        before += __shfl_xor(before, o);
        all += __shfl_xor(all, o);
    }
    if (lane == 63) {
        sums[0][tid >> 6] = before;
        sums[1][tid >> 6] = all;
        sums[2][tid >> 6] = in;
    }
    __syncthreads();
    uint32_t at = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3] + in - __popc(mine);
    for (uint32_t w = 0; w < tid >> 6; w++) at += sums[2][w];
    const uint32_t total = sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
    uint32_t *list = a.lists[kind];
    for (uint32_t m = mine; m; m &= m - 1) list[at++] = 32 * me + (uint32_t)__ffs((int)m) - 1;
    if (me < words)
        for (uint32_t i = max(32 * me, total); i < min(32 * me + 32, slots); i++) list[i] = CTOX_NO_SLOT;
    if (me == 0) a.counts[kind] = total;
}

// The same by one workgroup of 1024, the bits in LDS: small tables and pools.
extern "C" __global__ __launch_bounds__(1024) void ctox_free_small_gfx950(FreeSlotsArgs a) {
    __shared__ uint32_t used[CTOX_FREE_WORDS], sums[16];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, all = a.requests * a.max_pages;
    for (uint32_t i = tid; i < a.words[0] + a.words[1]; i += 1024) used[i] = 0;
    __syncthreads();
    for (uint32_t i0 = tid; i0 < all; i0 += 4096) {
        PagedKvDesc d[4];
        bool live[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {  // (four entries' loads under way at once, those of dead pages too)
            const uint32_t i = min(i0 + 1024 * k, all - 1), r = i / a.max_pages;
            live[k] = i0 + 1024 * k < all && (uint64_t)(i - r * a.max_pages) * a.page_tokens < a.tokens[r];
            d[k] = a.desc[i];
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t kind = d[k].precision ? 0 : 1, slot = d[k].physical_slot;
            if (live[k] && slot < a.slots[kind]) atomicOr(&used[(kind ? a.words[0] : 0) + slot / 32], 1u << (slot & 31));
        }
    }
    for (uint32_t kind = 0; kind < 2; kind++) {
        const uint32_t words = a.words[kind], slots = a.slots[kind], per = (words + 1023) / 1024;
        const uint32_t *bits = used + (kind ? a.words[0] : 0);
        const uint32_t w0 = min(tid * per, words), w1 = min(w0 + per, words);
        auto free_of = [&](uint32_t w) {
            const uint32_t left = slots - 32 * w;
            return ~bits[w] & (left < 32 ? (1u << left) - 1 : ~0u);
        };
        __syncthreads();
        uint32_t n = 0;
        for (uint32_t w = w0; w < w1; w++) n += __popc(free_of(w));
        uint32_t in = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t x = __shfl_up(in, o);
            if ((int)lane >= o) in += x;
        }
        if (lane == 63) sums[wave] = in;
        __syncthreads();
        uint32_t at = in - n, total = 0;
        for (uint32_t w = 0; w < 16; w++) {
            if (w < wave) at += sums[w];
            total += sums[w];
        }
        uint32_t *list = a.lists[kind];
        for (uint32_t w = w0; w < w1; w++)
            for (uint32_t m = free_of(w); m; m &= m - 1) list[at++] = 32 * w + (uint32_t)__ffs((int)m) - 1;
        for (uint32_t i = total + tid; i < slots; i += 1024) list[i] = CTOX_NO_SLOT;
        if (tid == 0) a.counts[kind] = total;
    }
}

// ---------------------------------------------------------------------------
// forks
// ---------------------------------------------------------------------------
// grid (pieces of a page of all layers, forks). Codes: 1 a source or target is no request, a target is a source or
// another fork's target, or the source is longer than its table; 2 too few free slots, by the count or by the pool; 3 a
// part-filled page is not a Q4 page of its request; 4 a free slot past q4_slots.
extern "C" __global__ __launch_bounds__(256) void ctox_paged_fork_gfx950(PagedForkArgs a) {
    __shared__ uint32_t sources[CTOX_PLAN_REQUESTS / 32], targets[CTOX_PLAN_REQUESTS / 32];
    __shared__ uint32_t bad[5], before, all;
    const uint32_t tid = threadIdx.x, f = blockIdx.y;
    for (uint32_t i = tid; i < CTOX_PLAN_REQUESTS / 32; i += 256) sources[i] = targets[i] = 0;
    if (tid < 5) bad[tid] = 0;
    if (tid == 0) before = all = 0;
    __syncthreads();
    const uint32_t room = *a.free_count;
    uint32_t front = 0, total = 0;
    for (uint32_t i = tid; i < a.forks; i += 256) {
        const uint32_t s = a.sources[i], t = a.targets[i];
        if (s >= a.requests || t >= a.requests) {
            bad[1] = 1;
            continue;
        }
        atomicOr(&sources[s / 32], 1u << (s & 31));
        if (atomicOr(&targets[t / 32], 1u << (t & 31)) >> (t & 31) & 1) bad[1] = 1;
        const uint32_t tokens = a.tokens[s], p = tokens / a.page_tokens;
        if (tokens > (uint64_t)a.max_pages * a.page_tokens) {
            bad[1] = 1;
            continue;
        }
        if (tokens % a.page_tokens) {
            const PagedKvDesc d = a.desc[(size_t)s * a.max_pages + p];
            if (d.precision == 0 || d.physical_slot >= a.q4_slots || d.first_token != p * a.page_tokens) bad[3] = 1;
            total++;
            if (i < f) front++;
        }
    }
    if (front) atomicAdd(&before, front);  // whole numbers: their order does not matter
    if (total) atomicAdd(&all, total);
    __syncthreads();
    for (uint32_t i = tid; i < CTOX_PLAN_REQUESTS / 32; i += 256)
        if (sources[i] & targets[i]) bad[1] = 1;
    // (the list has q4_slots entries, whatever the count says: every slot that is used below is checked here)
    const uint32_t there = min(room, a.q4_slots);
    if (tid == 0 && all > there) bad[2] = 1;
    for (uint32_t i = tid; i < min(all, there); i += 256)
        if (a.free_slots[i] >= a.q4_slots) bad[4] = 1;
    __syncthreads();
    uint32_t code = 0;
#pragma unroll
    for (int k = 4; k > 0; k--)
        if (bad[k]) code = k;
    if (f == 0 && blockIdx.x == 0 && tid == 0) {
        a.status[0] = code;
        a.status[1] = code ? 0 : all;
    }
    if (code || f >= a.forks) return;
    const uint32_t s = a.sources[f], t = a.targets[f], tokens = a.tokens[s];
    const uint32_t last = tokens / a.page_tokens, part = tokens % a.page_tokens;
    const PagedKvDesc *src = a.desc + (size_t)s * a.max_pages;
    PagedKvDesc *dst = a.desc + (size_t)t * a.max_pages;
    const uint32_t fresh = part ? a.free_slots[before] : 0;
    if (part) {
        const uint64_t from = (uint64_t)src[last].physical_slot * a.q4_page_bytes, to = (uint64_t)fresh * a.q4_page_bytes;
        const uint32_t units = part * (a.token_bytes / a.unit);  // of one layer
        const uint64_t most = (uint64_t)units * a.layers;
        for (uint64_t i = (uint64_t)blockIdx.x * 256 + tid; i < most; i += (uint64_t)gridDim.x * 256) {
            const uint32_t layer = (uint32_t)(i / units), u = (uint32_t)(i % units);
            uint8_t *p = a.pools[layer] + (size_t)u * a.unit;
            if (a.unit == 16) *(uint4 *)(p + to) = *(const uint4 *)(p + from);
            else *(uint32_t *)(p + to) = *(const uint32_t *)(p + from);
        }
    }
    if (blockIdx.x == 0) {
        for (uint32_t p = tid; p < last + (part != 0); p += 256) {
            PagedKvDesc d = src[p];
            if (p == last) d.physical_slot = fresh;
            dst[p] = d;
        }
        if (tid == 0) a.tokens[t] = tokens;
    }
}
