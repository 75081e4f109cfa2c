// Which path of a tree of drafted tokens the target's probabilities accept, gfx950.
//
// At a node with target law p = softmax(target / T) its children c_1, c_2 .. are offered in order. If they were
// drawn from the draft law q, child j is tested against what the refusals before it have left of p,
//   r_j = max(p - lambda_j q, 0) / Z_j,   accepted iff u q(c_j) / D_j < r_j(c_j),
//   lambda_{j+1} = lambda_j + Z_j / D_j,  Z_j = sum max(p - lambda_j q, 0),
// lambda_0 = 0, Z_0 = D_0 = 1. D_j is the draft's mass that is still undrawn: 1 - sum of q over the children before
// (siblings drawn without replacement), or 1 (with). Each refusal takes max(r_j - q / D_j, 0), which is the
// same form with a larger lambda, so a single number carries all refusals; a refused token is left with 0.
// Children chosen outright (no draft law) are tested against p without the tokens tried before. Where all are
// refused the next token is drawn from r, at the end of the path from p. One child a node is the chain rule
// of ctox_mtp_decide_gfx950.
//
// The results are whole numbers, and among 150 thousand tokens the borders of the running sum lie 1e-7 apart,
// what 32 bits hold of it: logits are taken apart in 64 bits from the exponential on.
//
//  * ctox_tree_stats_gfx950: maximum and sum of every part of 4096 tokens of a row (target, draft), or its largest
//    logit where the temperature is 0.
//  * ctox_tree_rest_gfx950, round k: sums of r_k (not yet divided by Z_k) by parts, of rows whose first k children
//    are refused; every workgroup repeats its row's tests for itself.
//  * ctox_tree_walk_gfx950: a workgroup a request: every row's tests, the walk down from the root, and the next
//    token: the part where the running sum reaches the request's number, then that part's tokens.
#include <hip/hip_runtime.h>

#include "kernel_args.h"
#include "lds_barrier.h"
#include "tree.h"

#define TV_PART 4096
#define TV_LEAST 0x1p-40  // undrawn mass of the draft below which its rounding errors would be offered

__device__ __forceinline__ double tv_sum64(double x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}
__device__ __forceinline__ float tv_max64(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}

// A law: logits of a row, its maximum and 1 / (sum of exp((x - maximum) / T)).
struct TvLaw {
    const float *row;
    double top, inv;  // inv 0: no law (a logit that is no number or +inf, or no finite one)
    __device__ __forceinline__ double at(float x, double inv_t) const { return exp(((double)x - top) * inv_t) * inv; }
};

// Parts' statistics of one row joined by a wave: TreeStat of `parts` parts.
__device__ __forceinline__ TvLaw tv_law(const float *row, const TreeStat *s, uint32_t parts, double inv_t) {
    const uint32_t lane = threadIdx.x & 63;
    TreeStat x{0.0, -INFINITY, 0};
    if (lane < parts) x = s[lane];
    const float top = tv_max64(x.top);
    const bool bad = __builtin_amdgcn_ballot_w64(x.bad) || !(fabsf(top) < INFINITY);
    const double sum = tv_sum64(x.sum > 0.0 ? x.sum * exp(((double)x.top - (double)top) * inv_t) : 0.0);
    return {row, (double)top, bad ? 0.0 : 1.0 / sum};
}

// What the tests of one row leave, in every lane of the wave that makes them.
struct TvTests {
    double lambda, left;   // of the refusals so far; left = Z
    int chosen;            // the accepted child (its number in the request), or -1
    uint32_t refused;      // how many were
    bool bad, stuck;       // stuck: the next test waits for the sum of round `refused`
};

struct TvRow {
    uint32_t row;        // in the batch
    uint64_t children;   // of the node, by their numbers
};

__device__ __forceinline__ bool tv_point(const TreeVerifyArgs &a) { return a.draft == nullptr; }

__device__ __forceinline__ double tv_draft_at(const TreeVerifyArgs &a, const TvLaw &q, uint32_t token) {
    uint32_t i = token;
    if (a.inverse) i = a.inverse[token];
    return i < a.draft_vocab ? q.at(q.row[i], a.inv_t) : 0.0;
}

// Tests the children of a row as far as the sums of rounds 1 .. rounds go. All lanes of a wave call it.
__device__ __forceinline__ TvTests tv_tests(const TreeVerifyArgs &a, const TreeRows &q, const TvRow &n, const TvLaw &p,
                                            const TvLaw &d, uint32_t rounds) {
    const uint32_t lane = threadIdx.x & 63;
    TvTests t{0.0, 1.0, -1, 0, p.inv == 0.0 || (n.children && !tv_point(a) && d.inv == 0.0), false};
    if (t.bad) return t;
    double undrawn = 1.0;
    uint64_t rest = n.children;
    for (uint32_t k = 0; rest && k < a.width; k++) {
        if (!(undrawn > TV_LEAST)) break;
        if (k) {  // the sum after k refusals
            if (k > rounds) {
                t.stuck = true;
                break;
            }
            const double *z = a.rest + ((size_t)(k - 1) * a.rows + n.row) * a.parts;
            t.left = tv_sum64(lane < a.parts ? z[lane] : 0.0);
        }
        const int child = __ffsll((unsigned long long)rest) - 1;
        rest &= rest - 1;
        const uint32_t token = a.tokens[q.row0 + child];
        double pt = 0.0, qt = tv_point(a) ? 1.0 : 0.0;
        bool tried = false;
        if (token < a.vocab) {
            pt = p.at(p.row[token], a.inv_t);
            if (!tv_point(a)) qt = tv_draft_at(a, d, token);
        }
        if (tv_point(a)) {  // a token that was tried is left with nothing
            uint64_t m = n.children & ((1ull << child) - 1);
            for (; m; m &= m - 1) tried |= a.tokens[q.row0 + __ffsll((unsigned long long)m) - 1] == token;
        }
        const double r = tv_point(a) ? (tried ? 0.0 : pt) : fmax(pt - t.lambda * qt, 0.0);
        if ((double)a.accept[q.row0 + child] * (qt / undrawn) * t.left < r) {
            t.chosen = child;
            break;
        }
        t.refused = k + 1;
        if (!tv_point(a)) {
            t.lambda += t.left / undrawn;
            if (a.without) undrawn -= qt;
        }
    }
    return t;
}

// Children of node `local`: lanes hold the nodes' parents.
__device__ __forceinline__ uint64_t tv_children(int parent, uint32_t local) {
    return __builtin_amdgcn_ballot_w64(parent == (int)local);
}

// ---------------------------------------------------------------------------
// statistics of a part
// ---------------------------------------------------------------------------
// Order of f32 numbers, as f32::total_cmp.
__device__ __forceinline__ int32_t tv_key(float v) {
    const int32_t b = __float_as_int(v);
    return b ^ (int32_t)(((uint32_t)(b >> 31)) >> 1);
}

// grid (parts, rows, 1 or 2: target, draft)
extern "C" __global__ __launch_bounds__(256) void ctox_tree_stats_gfx950(TreeVerifyArgs a) {
    __shared__ float tops[4];
    __shared__ double sums[4];
    __shared__ uint32_t ids[4], bads[4];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.y, part = blockIdx.x;
    if (row >= min(a.row_starts[a.requests], a.rows) || row < a.row_starts[0]) return;
    const bool draft = blockIdx.z != 0;
    const uint32_t len = draft ? a.draft_vocab : a.vocab, parts = draft ? a.draft_parts : a.parts;
    const uint32_t size = draft ? a.draft_part : a.part;
    if (part >= parts) return;
    if (draft) {  // of nodes with children only
        const uint32_t r = tree_request(a.row_starts, a.requests, row);
        const TreeRows q = tree_rows(a.row_starts, r, a.rows);
        if (!tv_children(tree_parent(a.parents, q, lane), row - q.row0)) return;
    }
    const float *x = (draft ? a.draft + (size_t)row * a.draft_stride : a.target + (size_t)row * a.target_stride);
    TreeStat *out = (draft ? a.draft_stats + (size_t)row * a.draft_parts : a.stats + (size_t)row * a.parts) + part;
    const uint32_t b = part * size, e = min(len, b + size);
    float top = -INFINITY;
    uint32_t id = 0;
    bool bad = false;
    for (uint32_t i = b + tid; i < e; i += 256) {
        const float v = x[i];
        bad |= !(v < INFINITY);
        if (tv_key(v) >= tv_key(top)) {  // (a later one wins)
            top = v;
            id = i;
        }
    }
    const float mine = top;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float t = __shfl_xor(top, o);
        const uint32_t j = __shfl_xor(id, o);
        if (tv_key(t) > tv_key(top) || (tv_key(t) == tv_key(top) && j > id)) {
            top = t;
            id = j;
        }
    }
    (void)mine;
    const uint32_t any = __builtin_amdgcn_ballot_w64(bad) != 0;
    if (lane == 0) tops[wave] = top, ids[wave] = id, bads[wave] = any;
    __syncthreads();
    top = tops[0];
    id = ids[0];
    for (int w = 1; w < 4; w++)
        if (tv_key(tops[w]) > tv_key(top) || (tv_key(tops[w]) == tv_key(top) && ids[w] > id)) {
            top = tops[w];
            id = ids[w];
        }
    const bool some_bad = bads[0] | bads[1] | bads[2] | bads[3];
    double sum = 0.0;
    if (a.greedy) {
        if (tid == 0) *out = TreeStat{(double)id, top, some_bad};
        return;
    }
    if (top > -INFINITY && !some_bad)
        for (uint32_t i = b + tid; i < e; i += 256) sum += exp(((double)x[i] - (double)top) * a.inv_t);
    sum = tv_sum64(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (tid == 0) *out = TreeStat{(sums[0] + sums[1]) + (sums[2] + sums[3]), top, some_bad};
}

// ---------------------------------------------------------------------------
// what k refusals leave
// ---------------------------------------------------------------------------
// The weight of token i after `refused` refusals; tried: the tokens of the first `refused` children (point laws).
__device__ __forceinline__ double tv_weight(const TreeVerifyArgs &a, const TvLaw &p, const TvLaw &d, uint32_t i,
                                            double lambda, uint32_t refused, const uint32_t *tried) {
    double w = p.at(p.row[i], a.inv_t);
    if (!refused) return w;
    if (!tv_point(a)) return fmax(w - lambda * tv_draft_at(a, d, i), 0.0);
    for (uint32_t k = 0; k < refused; k++)
        if (tried[k] == i) w = 0.0;
    return w;
}

// grid (parts, rows)
extern "C" __global__ __launch_bounds__(256) void ctox_tree_rest_gfx950(TreeVerifyArgs a) {
    __shared__ double sums[4];
    __shared__ uint32_t tried[CTOX_TREE_NODES];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.y, part = blockIdx.x;
    if (row >= min(a.row_starts[a.requests], a.rows) || row < a.row_starts[0]) return;
    const uint32_t r = tree_request(a.row_starts, a.requests, row);
    const TreeRows q = tree_rows(a.row_starts, r, a.rows);
    const TvRow n{row, tv_children(tree_parent(a.parents, q, lane), row - q.row0)};
    if ((uint32_t)__popcll(n.children) < a.round) return;
    const TvLaw p = tv_law(a.target + (size_t)row * a.target_stride, a.stats + (size_t)row * a.parts, a.parts, a.inv_t);
    TvLaw d{nullptr, 0.0, 0.0};
    if (!tv_point(a))
        d = tv_law(a.draft + (size_t)row * a.draft_stride, a.draft_stats + (size_t)row * a.draft_parts, a.draft_parts, a.inv_t);
    const TvTests t = tv_tests(a, q, n, p, d, a.round - 1);
    if (t.bad || t.chosen >= 0 || t.refused != a.round) return;
    if (tid == 0) {
        uint64_t m = n.children;
        for (uint32_t k = 0; k < t.refused; k++, m &= m - 1) tried[k] = a.tokens[q.row0 + __ffsll((unsigned long long)m) - 1];
    }
    __syncthreads();
    const uint32_t b = part * a.part, e = min(a.vocab, b + a.part);
    double sum = 0.0;
    for (uint32_t i = b + tid; i < e; i += 256) sum += tv_weight(a, p, d, i, t.lambda, t.refused, tried);
    sum = tv_sum64(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (tid == 0) a.rest[((size_t)(a.round - 1) * a.rows + row) * a.parts + part] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// ---------------------------------------------------------------------------
// the path and the next token
// ---------------------------------------------------------------------------
// grid (requests), 1024 threads
extern "C" __global__ __launch_bounds__(1024) void ctox_tree_walk_gfx950(TreeVerifyArgs a) {
    __shared__ int chosen[CTOX_TREE_NODES];
    __shared__ uint32_t refused[CTOX_TREE_NODES], best[CTOX_TREE_NODES], tried[CTOX_TREE_NODES];
    __shared__ double lambda[CTOX_TREE_NODES], sums[16];
    __shared__ uint32_t end, total_nodes, pick, found;
    __shared__ double want;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x;
    const TreeRows all = tree_rows(a.row_starts, r, a.rows);
    const TreeRows q{all.row0, min(all.n, (uint32_t)CTOX_TREE_NODES)};
    for (uint32_t i = tid; i < all.n; i += 1024) a.path[all.row0 + i] = CTOX_NO_SLOT;
    if (q.n == 0) {
        if (tid == 0) {
            a.counts[r] = 0;
            a.next[r] = CTOX_NO_SLOT;
        }
        return;
    }
    const int parent = tree_parent(a.parents, q, lane);
    for (uint32_t i = wave; i < q.n; i += 16) {
        const TvRow n{q.row0 + i, tv_children(parent, i)};
        if (a.greedy) {
            TreeStat x{0.0, -INFINITY, 0};
            if (lane < a.parts) x = a.stats[(size_t)n.row * a.parts + lane];
            float top = x.top;
            uint32_t id = (uint32_t)x.sum;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                const float t = __shfl_xor(top, o);
                const uint32_t j = __shfl_xor(id, o);
                if (tv_key(t) > tv_key(top) || (tv_key(t) == tv_key(top) && j > id)) {
                    top = t;
                    id = j;
                }
            }
            const bool bad = __builtin_amdgcn_ballot_w64(x.bad) || !(fabsf(top) < INFINITY);
            uint64_t m = n.children;
            int c = -1;
            for (uint32_t k = 0; m && k < a.width && c < 0; k++, m &= m - 1) {
                const int child = __ffsll((unsigned long long)m) - 1;
                if (a.tokens[q.row0 + child] == id) c = child;
            }
            if (lane == 0) {
                chosen[i] = bad ? -2 : c;
                best[i] = id;
            }
            continue;
        }
        const TvLaw p = tv_law(a.target + (size_t)n.row * a.target_stride, a.stats + (size_t)n.row * a.parts, a.parts, a.inv_t);
        TvLaw d{nullptr, 0.0, 0.0};
        if (!tv_point(a) && n.children)
            d = tv_law(a.draft + (size_t)n.row * a.draft_stride, a.draft_stats + (size_t)n.row * a.draft_parts,
                       a.draft_parts, a.inv_t);
        const TvTests t = tv_tests(a, q, n, p, d, a.width);
        if (lane == 0) {
            chosen[i] = t.bad ? -2 : t.chosen;
            refused[i] = t.refused;
            lambda[i] = t.lambda;
        }
    }
    __syncthreads();
    if (tid == 0) {
        uint32_t at = 0, count = 1;
        a.path[q.row0] = 0;
        while (chosen[at] >= 0) {  // (children have larger numbers: it ends)
            at = (uint32_t)chosen[at];
            a.path[q.row0 + count++] = at;
        }
        end = at;
        total_nodes = chosen[at] == -2 ? 0 : count;
    }
    __syncthreads();
    if (total_nodes == 0) {  // logits that are no numbers on the path: nothing is accepted
        for (uint32_t i = tid; i < q.n; i += 1024) a.path[q.row0 + i] = CTOX_NO_SLOT;
        if (tid == 0) {
            a.counts[r] = 0;
            a.next[r] = CTOX_TREE_FAILED;
        }
        return;
    }
    if (tid == 0) a.counts[r] = total_nodes;
    if (a.greedy) {
        if (tid == 0) a.next[r] = best[end];
        return;
    }
    const uint32_t node = end, row = q.row0 + node;
    uint32_t gone = refused[node];
    const uint64_t children = tv_children(parent, node);
    const TvLaw p = tv_law(a.target + (size_t)row * a.target_stride, a.stats + (size_t)row * a.parts, a.parts, a.inv_t);
    TvLaw d{nullptr, 0.0, 0.0};
    if (gone && !tv_point(a))
        d = tv_law(a.draft + (size_t)row * a.draft_stride, a.draft_stats + (size_t)row * a.draft_parts, a.draft_parts, a.inv_t);
    if (tid == 0) {
        uint64_t m = children;
        for (uint32_t k = 0; k < gone; k++, m &= m - 1) tried[k] = a.tokens[q.row0 + __ffsll((unsigned long long)m) - 1];
        found = ~0u;
    }
    // The part where the running sum passes the number. Where nothing is left of the target (only rounding could have
    // refused then) the target itself is drawn from.
    double mass = 0.0, in = 0.0;
    for (int again = 0; again < 2; again++) {
        mass = 0.0;
        if (lane < a.parts) {
            if (gone) {
                mass = a.rest[((size_t)(gone - 1) * a.rows + row) * a.parts + lane];
            } else {
                const TreeStat s = a.stats[(size_t)row * a.parts + lane];
                mass = s.sum > 0.0 ? s.sum * exp(((double)s.top - p.top) * a.inv_t) * p.inv : 0.0;
            }
        }
        in = mass;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double x = __shfl_up(in, o);
            if ((int)lane >= o) in += x;
        }
        if (__shfl(in, 63) > 0.0) break;
        gone = 0;
    }
    const double total = __shfl(in, 63), goal = (double)a.sample[r] * total;
    // (the last part with mass where rounding leaves none past the number)
    const uint64_t past = __builtin_amdgcn_ballot_w64(in > goal), massive = __builtin_amdgcn_ballot_w64(mass > 0.0);
    const uint32_t part = past ? (uint32_t)__ffsll((unsigned long long)past) - 1
                               : massive ? 63 - (uint32_t)__clzll((long long)massive) : 0;
    if (tid == part) want = goal - (in - mass);
    if (tid == 0) pick = part;
    __syncthreads();
    // That part's tokens, 4 a thread and round.
    const uint32_t b = pick * a.part, e = min(a.vocab, b + a.part);
    double before = 0.0;
    uint32_t last = b;  // the last token with a weight, of this thread
    bool has = false;
    for (uint32_t i0 = b; i0 < e; i0 += 4096) {
        double w[4], s = 0.0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t i = i0 + 4 * tid + k;
            w[k] = i < e ? tv_weight(a, p, d, i, lambda[node], gone, tried) : 0.0;
            if (w[k] > 0.0) last = i, has = true;
            s += w[k];
        }
        double run = s;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double x = __shfl_up(run, o);
            if ((int)lane >= o) run += x;
        }
        if (lane == 63) sums[wave] = run;
        __syncthreads();
        double at = before + run - s;
        for (uint32_t v = 0; v < 16; v++) {
            if (v < wave) at += sums[v];
            before += sums[v];
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            at += w[k];
            if (w[k] > 0.0 && at > want) {
                atomicMin(&found, i0 + 4 * tid + k);
                break;
            }
        }
        __syncthreads();
        if (found != ~0u) break;
    }
    if (found == ~0u) {  // rounding: the last token with a weight
        __syncthreads();
        if (tid == 0) pick = 0;
        __syncthreads();
        if (has) atomicMax(&pick, last);
        __syncthreads();
        if (tid == 0) a.next[r] = pick;
        return;
    }
    if (tid == 0) a.next[r] = found;
}
