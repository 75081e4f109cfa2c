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
// what 32 bits hold of it: logits are taken apart in 64 bits from the exponential on (tv_exp2).
//
// Rows are cut into parts of 4096 tokens, counted from the 16-byte border in front of the row; the first statistics of
// many rows into parts of a few times that, since a part's reductions cost as much as a third of its exponentials.
//  * ctox_tree_stats_gfx950: maximum and sum of every part (target, draft) of the rows with children and of roots; its
//    largest logit, of all rows, where the temperature is 0.
//  * ctox_tree_first_gfx950, ctox_tree_round_gfx950: round k, the test of a row's k-th child: of every row, then of those
//    that refused it and may still be on the path. Of a row that refuses, the parts' sums of
//    r_k, not yet divided by Z_k; of a leaf that is accepted its own statistics (the others' are never read).
//    Each workgroup repeats its row's test for itself; what it needs of the round before is a TreeRow.
//    ctox_tree_test_gfx950, ctox_tree_rest_gfx950: the first round of many rows, every test made once and the sums only where
//    the tests above still lead.
//  * ctox_tree_walk_gfx950: a workgroup a request: the walk down from the root, and the next token: the part where
//    the running sum passes the request's number, then that part's tokens.
//
// Measured, 151936 tokens, a draft row a node with children: 16 trees of up to 32 nodes (315 rows, 146 with children)
// 130 to 132 us, 48 of it the statistics (177 MB, 3.7 TB/s; 20 operations a logit, the exponential 15: both bound it), the
// first round 6.7 + 21, three more 10-13 each, the walk 11; a chain of five 23 to 24 us in three launches; greedy, 8 trees of
// up to 16 nodes, 17.9 us (47 MB).
#include <hip/hip_runtime.h>

#include "kernel_args.h"
#include "lds_barrier.h"
#include "tree.h"

#define TV_LEAST 0x1p-40  // undrawn mass of the draft below which its rounding errors would be offered

// 2^y for y <= 0 (a hair above 0 at most), within 1.1e-12: 2^f, |f| <= 1/2, by its interpolation in the nine
// Chebyshev points. A running sum is moved by as little, far below the distance of its borders. Whole numbers
// are split off and put into the exponent by additions alone. What is below 2^-1000, -inf too, gives 2^-1000: nothing
// in a sum whose largest term is 1; as a token's weight (TvLaw) it is 0.
__device__ __forceinline__ double tv_exp2(double y) {
    y = fmax(y, -1000.0);
    const double big = 6755399441055744.0, t = y + big, f = y - (t - big);  // 1.5 * 2^52
    double p = 1.3255224887698904e-06;
    p = fma(p, f, 1.5310079402479794e-05);
    p = fma(p, f, 1.5403455852411408e-04);
    p = fma(p, f, 1.3333450567999659e-03);
    p = fma(p, f, 9.6181291594026191e-03);
    p = fma(p, f, 5.5504109412059341e-02);
    p = fma(p, f, 2.4022650695812989e-01);
    p = fma(p, f, 6.9314718054593349e-01);
    p = fma(p, f, 1.0);
    return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
}

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

// A row of logits; `skew` floats lie between the 16-byte border in front of it and its first.
struct TvRow {
    const float *x;
    uint32_t len, skew;
    __device__ __forceinline__ TvRow(const float *x, uint32_t len)
        : x(x), len(len), skew(((uint32_t)(uintptr_t)x >> 2) & 3) {}
    // Four logits from place e (a multiple of 4 counted from the border); places outside the row give -inf.
    __device__ __forceinline__ float4 four(uint32_t e) const {
        if (e >= skew && e - skew + 4 <= len) return *(const float4 *)(x + (e - skew));
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t i = e + k - skew;  // (below 0: large)
            v[k] = i < len ? x[i] : -INFINITY;
        }
        return make_float4(v[0], v[1], v[2], v[3]);
    }
    // The 4096 places from e0: four times four a thread.
    __device__ __forceinline__ void piece(uint32_t e0, float4 (&v)[4]) const {
        if (e0 >= skew && e0 - skew + 4096 <= len) {
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = *(const float4 *)(x + (e0 - skew + 1024 * k + 4 * threadIdx.x));
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = four(e0 + 1024 * k + 4 * threadIdx.x);
        }
    }
};
__device__ __forceinline__ TvRow tv_target(const TreeVerifyArgs &a, uint32_t row) {
    return TvRow(a.target + (size_t)row * a.target_stride, a.vocab);
}
__device__ __forceinline__ TvRow tv_draft(const TreeVerifyArgs &a, uint32_t row) {
    return TvRow(a.draft + (size_t)row * a.draft_stride, a.draft_vocab);
}

// Its law: probability of a logit x is 2^((x - top) c) inv. (The difference is formed first: whatever the logits and the
// temperature, the largest weight is 1.)
struct TvLaw {
    double top, inv;  // inv 0: no law (a logit that is no number or +inf, or none that is finite)
    __device__ __forceinline__ double at(const TreeVerifyArgs &a, float x) const {
        const double y = ((double)x - top) * a.c;
        return y < -1000.0 ? 0.0 : tv_exp2(y) * inv;
    }
};

// Parts' statistics of one row joined by a wave.
__device__ __forceinline__ TvLaw tv_law(const TreeVerifyArgs &a, const TreeStat *s, uint32_t parts) {
    const uint32_t lane = threadIdx.x & 63;
    TreeStat x{0.0, -INFINITY, 0};
    if (lane < parts) x = s[lane];
    const float top = tv_max64(x.top);
    const bool bad = __builtin_amdgcn_ballot_w64(x.bad) || !(fabsf(top) < INFINITY);
    const double sum = tv_sum64(x.sum > 0.0 ? x.sum * tv_exp2(((double)x.top - (double)top) * a.c) : 0.0);
    return {(double)top, bad ? 0.0 : 1.0 / sum};
}

__device__ __forceinline__ bool tv_point(const TreeVerifyArgs &a) { return a.draft == nullptr; }

__device__ __forceinline__ double tv_draft_at(const TreeVerifyArgs &a, const TvLaw &q, const float *x, uint32_t token) {
    const uint32_t i = a.inverse ? a.inverse[token] : token;
    return i < a.draft_vocab ? q.at(a, x[i]) : 0.0;
}

// Children of node `local`: lanes hold the nodes' parents.
__device__ __forceinline__ uint64_t tv_children(int parent, uint32_t local) {
    return __builtin_amdgcn_ballot_w64(parent == (int)local);
}

// Order of f32 numbers, as f32::total_cmp.
__device__ __forceinline__ int32_t tv_key(float v) {
    const int32_t b = __float_as_int(v);
    return b ^ (int32_t)(((uint32_t)(b >> 31)) >> 1);
}
__device__ __forceinline__ void tv_larger(float &top, uint32_t &id, float t, uint32_t i) {  // the later one wins ties
    if (tv_key(t) > tv_key(top) || (tv_key(t) == tv_key(top) && i > id)) {
        top = t;
        id = i;
    }
}

// Marks are written and read in one round: whole 64-bit words.
__device__ __forceinline__ TreeMark tv_mark(const TreeVerifyArgs &a, uint32_t row) {
    return __builtin_bit_cast(TreeMark, __hip_atomic_load(a.marks + row, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
__device__ __forceinline__ void tv_set_mark(const TreeVerifyArgs &a, uint32_t row, TreeMark m) {
    __hip_atomic_store(a.marks + row, __builtin_bit_cast(uint64_t, m), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct TvScratch {
    double sums[4];
    float tops[4];
    uint32_t ids[4], bads[4];
};

// Statistics of parts first .. last - 1 of a row, by a workgroup of 256.
__device__ __forceinline__ void tv_stats(const TreeVerifyArgs &a, const TvRow &row, uint32_t first, uint32_t last,
                                         uint32_t size, TreeStat *out, TvScratch &L) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t end = min(last * size, row.len + row.skew);
    // A row that begins at its border may have no token in its last part.
    for (uint32_t p = first; p < last; p++)
        if (p * size >= end && tid == 0) out[p] = TreeStat{0.0, -INFINITY, 0};
    float top = -INFINITY;  // of the wave; greedy: of the thread
    double sum = 0.0;
    uint32_t id = 0;
    bool bad = false;
    float4 v[4], next[4];
    row.piece(first * size, next);
    for (uint32_t e0 = first * size; e0 < end; e0 += 4096) {
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = next[k];
        if (e0 + 4096 < end) row.piece(e0 + 4096, next);  // (under way during this piece's exponentials)
        const float *x = (const float *)v;
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < 16; k++) {
            bad |= !(x[k] < INFINITY);
            m = fmaxf(m, x[k]);
        }
        if (a.greedy) {
#pragma unroll
            for (int k = 0; k < 16; k++) {
                const uint32_t i = e0 + 1024 * (k >> 2) + 4 * tid + (k & 3) - row.skew;
                if (i < row.len) tv_larger(top, id, x[k], i);
            }
        } else {
            m = tv_max64(m);
            if (m > top) {
                sum = top > -INFINITY ? sum * tv_exp2(((double)top - (double)m) * a.c) : 0.0;
                top = m;
            }
            const double t = top > -INFINITY ? (double)top : 0.0;
            double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
            for (int k = 0; k < 16; k++) s[k & 3] += tv_exp2(((double)x[k] - t) * a.c);
            if (top > -INFINITY) sum += (s[0] + s[1]) + (s[2] + s[3]);
        }
        if ((e0 + 4096) % size && e0 + 4096 < end) continue;
        // ---- the part's end ----
        const uint32_t any = __builtin_amdgcn_ballot_w64(bad) != 0;
        if (a.greedy) {
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) tv_larger(top, id, __shfl_xor(top, o), __shfl_xor(id, o));
        } else {
            sum = tv_sum64(sum);
        }
        if (lane == 0) {
            L.sums[wave] = sum;
            L.tops[wave] = top;
            L.ids[wave] = id;
            L.bads[wave] = any;
        }
        lds_barrier();
        if (tid == 0) {
            if (a.greedy) {
                for (int w = 1; w < 4; w++) tv_larger(top, id, L.tops[w], L.ids[w]);
                sum = (double)id;
            } else {
                const float t = fmaxf(fmaxf(L.tops[0], L.tops[1]), fmaxf(L.tops[2], L.tops[3]));
                sum = 0.0;
                for (int w = 0; w < 4; w++)
                    if (L.sums[w] > 0.0) sum += L.sums[w] * tv_exp2(((double)L.tops[w] - (double)t) * a.c);
                top = t;
            }
            out[e0 / size] = TreeStat{sum, top, L.bads[0] | L.bads[1] | L.bads[2] | L.bads[3]};
        }
        lds_barrier();
        top = -INFINITY, sum = 0.0, id = 0, bad = false;
    }
}

// grid (parts, rows, 1 or 2: target, draft)
extern "C" __global__ __launch_bounds__(256) void ctox_tree_stats_gfx950(TreeVerifyArgs a) {
    __shared__ TvScratch L;
    const uint32_t row = blockIdx.y, part = blockIdx.x;
    if (!a.greedy && blockIdx.x + blockIdx.y + blockIdx.z == 0 && threadIdx.x < CTOX_TREE_NODES) a.waiting[threadIdx.x] = 0;
    if (row >= min(a.row_starts[a.requests], a.rows) || row < a.row_starts[0]) return;
    const bool draft = blockIdx.z != 0;
    if (part >= (draft ? a.draft_parts : a.stat_parts)) return;
    if (!a.greedy) {  // a leaf is read when it is accepted
        const uint32_t r = tree_request(a.row_starts, a.requests, row);
        const TreeRows q = tree_rows(a.row_starts, r, a.rows);
        const bool any = tv_children(tree_parent(a.parents, q, threadIdx.x & 63), row - q.row0) != 0;
        if (!any && (draft || row != q.row0)) return;
    }
    if (draft) tv_stats(a, tv_draft(a, row), part, part + 1, a.draft_part, a.draft_stats + (size_t)row * a.draft_parts, L);
    else tv_stats(a, tv_target(a, row), part, part + 1, a.stat_part, a.stats + (size_t)row * a.parts, L);
}

// ---------------------------------------------------------------------------
// a round of tests
// ---------------------------------------------------------------------------
// Weights of tokens after `refused` refusals; tried: the tokens of the first `refused` children (point laws).
struct TvRest {
    const TreeVerifyArgs &a;
    const TvRow p;
    const float *q;
    const TvLaw pl, ql;
    const double lambda;
    const uint32_t refused;
    const uint32_t *tried;
    // of the four places from e, whose logits are v
    __device__ __forceinline__ void four(uint32_t e, const float4 &v, double (&w)[4]) const {
        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = pl.at(a, x[k]);
        if (!refused) return;
        const uint32_t i0 = e - p.skew;
        if (tv_point(a)) {
            for (uint32_t t = 0; t < refused; t++) {
                const uint32_t k = tried[t] - i0;
                w[0] = k == 0 ? 0.0 : w[0];
                w[1] = k == 1 ? 0.0 : w[1];
                w[2] = k == 2 ? 0.0 : w[2];
                w[3] = k == 3 ? 0.0 : w[3];
            }
            return;
        }
        float y[4];
        if (!a.inverse && i0 + 4 <= p.len && i0 < p.len && ((uintptr_t)(q + i0) & 15) == 0) {
            const float4 u = *(const float4 *)(q + i0);
            y[0] = u.x, y[1] = u.y, y[2] = u.z, y[3] = u.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                uint32_t i = i0 + k;
                if (i < p.len && a.inverse) i = a.inverse[i];
                y[k] = i0 + k < p.len && i < a.draft_vocab ? q[i] : -INFINITY;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = fmax(fma(-lambda, ql.at(a, y[k]), w[k]), 0.0);
    }
};

// What a row's test of its child number k = a.round - 1 leaves.
struct TvTest {
    TreeRow s;
    uint64_t children;
    int leaf;      // row of a child without children that was accepted, else -1
    bool refused;  // else accepted, or nothing to test
};

// By whole waves; the chief's lane 0 keeps the row's records.
__device__ __forceinline__ TvTest tv_test(const TreeVerifyArgs &a, uint32_t row, const TreeRows &q, int parent, bool chief) {
    const uint32_t lane = threadIdx.x & 63, k = a.round - 1;
    TvTest t{{0.0, 1.0, 0.0, 0.0, 0.0, 0.0}, tv_children(parent, row - q.row0), -1, false};
    TreeRow &s = t.s;
    if (k) {
        s = a.states[(size_t)(k & 1) * a.rows + row];
    } else if (!t.children) {
        if (chief) tv_set_mark(a, row, TreeMark{-1, 0});
        return t;
    }
    uint64_t rest = t.children;
    for (uint32_t i = 0; i < k; i++) rest &= rest - 1;
    const int child = __ffsll((unsigned long long)rest) - 1;
    rest &= rest - 1;
    const float *x = tv_point(a) ? nullptr : a.draft + (size_t)row * a.draft_stride;
    const uint32_t token = a.tokens[q.row0 + child];
    const float px = (a.target + (size_t)row * a.target_stride)[min(token, a.vocab - 1)];
    double left = 1.0;
    TvLaw pl, ql{0.0, 0.0};
    if (k) {
        left = tv_sum64(lane < a.parts ? a.rest[((size_t)(k - 1) * a.rows + row) * a.parts + lane] : 0.0);
        pl = {s.p_top, s.p_inv};
        ql = {s.q_top, s.q_inv};
    } else {
        pl = tv_law(a, a.stats + (size_t)row * a.parts, a.stat_parts);
        if (!tv_point(a)) ql = tv_law(a, a.draft_stats + (size_t)row * a.draft_parts, a.draft_parts);
        s.p_top = pl.top, s.p_inv = pl.inv, s.q_top = ql.top, s.q_inv = ql.inv;
        if (pl.inv == 0.0 || (!tv_point(a) && ql.inv == 0.0)) {
            if (chief) tv_set_mark(a, row, TreeMark{-2, 0});
            return t;
        }
    }
    double pt = 0.0, qt = tv_point(a) ? 1.0 : 0.0;
    if (token < a.vocab) {
        pt = pl.at(a, px);
        if (!tv_point(a)) qt = tv_draft_at(a, ql, x, token);
    }
    if (tv_point(a)) {  // a token that was tried is left with nothing
        const uint64_t before = t.children & ((1ull << child) - 1);
        if (__builtin_amdgcn_ballot_w64((before >> lane & 1) && a.tokens[q.row0 + lane] == token)) pt = 0.0;
    } else {
        pt = fmax(pt - s.lambda * qt, 0.0);
    }
    if ((double)a.accept[q.row0 + child] * (qt / s.undrawn) * left < pt) {
        if (chief) tv_set_mark(a, row, TreeMark{child, k});
        if (!tv_children(parent, (uint32_t)child)) t.leaf = (int)(q.row0 + child);
        return t;
    }
    t.refused = true;
    if (!tv_point(a)) {
        s.lambda += left / s.undrawn;
        if (a.without) s.undrawn -= qt;
    }
    if (chief) {
        tv_set_mark(a, row, TreeMark{-1, k + 1});
        a.states[(size_t)(a.round & 1) * a.rows + row] = s;
        // The next round's rows; in which order does not matter.
        if (rest && a.round < a.width && s.undrawn > TV_LEAST) {
            const uint32_t at = atomicAdd(&a.waiting[a.round], 1u);
            a.lists[(size_t)(a.round & 1) * a.rows + at] = row;
        }
    }
    return t;
}

// A row that refused children 0 .. k: sums of what is left in parts first .. last - 1, by a workgroup.
__device__ __forceinline__ void tv_rest(const TreeVerifyArgs &a, uint32_t row, const TreeRows &q, const TvTest &t, uint32_t k,
                                        uint32_t first, uint32_t last, TvScratch &L, uint32_t (&tried)[CTOX_TREE_NODES]) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tv_point(a)) {
        if (wave == 0 && (t.children >> lane & 1)) {
            const uint32_t at = __popcll(t.children & ((1ull << lane) - 1));
            tried[at] = a.tokens[q.row0 + lane];
        }
        lds_barrier();
    }
    const TvRow p = tv_target(a, row);
    const TvRest f{a, p, tv_point(a) ? nullptr : a.draft + (size_t)row * a.draft_stride, {t.s.p_top, t.s.p_inv},
                   {t.s.q_top, t.s.q_inv}, t.s.lambda, k + 1, tried};
    for (uint32_t part = first; part < last; part++) {
        double sum = 0.0;
        for (uint32_t e0 = part * a.part; e0 < (part + 1) * a.part && e0 < p.len + p.skew; e0 += 4096) {
            float4 v[4];
            p.piece(e0, v);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                double w[4];
                f.four(e0 + 1024 * i + 4 * tid, v[i], w);
                sum += (w[0] + w[1]) + (w[2] + w[3]);
            }
        }
        sum = tv_sum64(sum);
        if (lane == 0) L.sums[wave] = sum;
        lds_barrier();
        if (tid == 0)
            a.rest[((size_t)k * a.rows + row) * a.parts + part] = (L.sums[0] + L.sums[1]) + (L.sums[2] + L.sums[3]);
        lds_barrier();
    }
}

// Whether another child was accepted where the row's path branches off, by marks of fewer than `rounds` refusals.
__device__ __forceinline__ bool tv_off(const TreeVerifyArgs &a, const TreeRows &q, int parent, uint32_t row, uint32_t rounds) {
    const uint32_t lane = threadIdx.x & 63;
    TreeMark m{-1, 0};
    if (lane < q.n) m = tv_mark(a, q.row0 + lane);
    const int accepted = m.refused < rounds ? m.chosen : -1;
    const int above = __shfl(accepted, parent < 0 ? (int)lane : parent);
    const uint64_t line = __shfl(tree_lineage(parent, lane, lane < q.n), (int)((row - q.row0) & 63));
    return __builtin_amdgcn_ballot_w64((line >> lane & 1) && parent >= 0 && above != -1 && above != (int)lane) != 0;
}

__device__ __forceinline__ bool tv_has(const TreeVerifyArgs &a, uint32_t row) {
    return row < min(a.row_starts[a.requests], a.rows) && row >= a.row_starts[0];
}

// Round 1 of few rows: grid (parts, rows)
extern "C" __global__ __launch_bounds__(256) void ctox_tree_first_gfx950(TreeVerifyArgs a) {
    __shared__ TvScratch L;
    __shared__ uint32_t tried[CTOX_TREE_NODES];
    const uint32_t row = blockIdx.y, part = blockIdx.x;
    if (!tv_has(a, row)) return;
    const TreeRows q = tree_rows(a.row_starts, tree_request(a.row_starts, a.requests, row), a.rows);
    const int parent = tree_parent(a.parents, q, threadIdx.x & 63);
    const TvTest t = tv_test(a, row, q, parent, part == 0 && threadIdx.x == 0);
    if (t.refused) tv_rest(a, row, q, t, 0, part, part + 1, L, tried);
    else if (t.leaf >= 0)
        tv_stats(a, tv_target(a, t.leaf), part, part + 1, a.part, a.stats + (size_t)t.leaf * a.parts, L);
}

// Round 1 of many: a wave a row tests, ...
#define TV_LEAF 0x80000000u
extern "C" __global__ __launch_bounds__(256) void ctox_tree_test_gfx950(TreeVerifyArgs a) {
    const uint32_t row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (!tv_has(a, row)) return;
    const TreeRows q = tree_rows(a.row_starts, tree_request(a.row_starts, a.requests, row), a.rows);
    const TvTest t = tv_test(a, row, q, tree_parent(a.parents, q, lane), lane == 0);
    if (lane == 0 && (t.refused || t.leaf >= 0))
        a.lists[atomicAdd(&a.waiting[0], 1u)] = t.refused ? row : (uint32_t)t.leaf | TV_LEAF;
}
// ... and what may still be on the path is summed: grid (parts, CTOX_TREE_LANES).
extern "C" __global__ __launch_bounds__(256) void ctox_tree_rest_gfx950(TreeVerifyArgs a) {
    __shared__ TvScratch L;
    __shared__ uint32_t tried[CTOX_TREE_NODES];
    const uint32_t waiting = a.waiting[0], part = blockIdx.x;
    for (uint32_t i = blockIdx.y; i < waiting; i += CTOX_TREE_LANES) {
        const uint32_t entry = a.lists[i], row = entry & ~TV_LEAF;
        const TreeRows q = tree_rows(a.row_starts, tree_request(a.row_starts, a.requests, row), a.rows);
        const int parent = tree_parent(a.parents, q, threadIdx.x & 63);
        if (tv_off(a, q, parent, row, 1)) continue;
        if (entry & TV_LEAF) {
            tv_stats(a, tv_target(a, row), part, part + 1, a.part, a.stats + (size_t)row * a.parts, L);
        } else {
            const TvTest t{a.states[a.rows + row], tv_children(parent, row - q.row0), -1, true};
            tv_rest(a, row, q, t, 0, part, part + 1, L, tried);
        }
        lds_barrier();
    }
}

// The rounds after it: grid (parts, CTOX_TREE_LANES), which take the rows that wait in turn.
extern "C" __global__ __launch_bounds__(256) void ctox_tree_round_gfx950(TreeVerifyArgs a) {
    __shared__ TvScratch L;
    __shared__ uint32_t tried[CTOX_TREE_NODES];
    const uint32_t waiting = a.waiting[a.round - 1], part = blockIdx.x;
    for (uint32_t i = blockIdx.y; i < waiting; i += CTOX_TREE_LANES) {
        const uint32_t row = a.lists[(size_t)((a.round - 1) & 1) * a.rows + i];
        const TreeRows q = tree_rows(a.row_starts, tree_request(a.row_starts, a.requests, row), a.rows);
        const int parent = tree_parent(a.parents, q, threadIdx.x & 63);
        // Marks of this round may be there already or not, so they do not count: every workgroup decides the same.
        if (tv_off(a, q, parent, row, a.round - 1)) continue;
        const TvTest t = tv_test(a, row, q, parent, part == 0 && threadIdx.x == 0);
        if (t.refused) tv_rest(a, row, q, t, a.round - 1, part, part + 1, L, tried);
        else if (t.leaf >= 0)
            tv_stats(a, tv_target(a, t.leaf), part, part + 1, a.part, a.stats + (size_t)t.leaf * a.parts, L);
        lds_barrier();
    }
}

// ---------------------------------------------------------------------------
// the path and the next token
// ---------------------------------------------------------------------------
// grid (requests), 1024 threads
extern "C" __global__ __launch_bounds__(1024) void ctox_tree_walk_gfx950(TreeVerifyArgs a) {
    __shared__ int chosen[CTOX_TREE_NODES];
    __shared__ uint32_t best[CTOX_TREE_NODES], tried[CTOX_TREE_NODES];
    __shared__ double sums[16];
    __shared__ uint32_t found;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x;
    const TreeRows q = tree_rows(a.row_starts, r, a.rows);
    if (q.n == 0 || q.n > CTOX_TREE_NODES) {  // no nodes, or not a tree of these kernels
        for (uint32_t i = tid; i < q.n; i += 1024) a.path[q.row0 + i] = CTOX_NO_SLOT;
        if (tid == 0) {
            a.counts[r] = 0;
            a.next[r] = q.n ? CTOX_TREE_FAILED : CTOX_NO_SLOT;
        }
        return;
    }
    const int parent = tree_parent(a.parents, q, lane);
    if (a.greedy) {
        for (uint32_t i = wave; i < q.n; i += 16) {
            TreeStat x{0.0, -INFINITY, 0};
            if (lane < a.stat_parts) x = a.stats[(size_t)(q.row0 + i) * a.parts + lane];
            float top = x.top;
            uint32_t id = (uint32_t)x.sum;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) tv_larger(top, id, __shfl_xor(top, o), __shfl_xor(id, o));
            const bool bad = __builtin_amdgcn_ballot_w64(x.bad) || !(fabsf(top) < INFINITY);
            const uint64_t children = tv_children(parent, i);
            // the first of the children that are offered
            const bool offered = (children >> lane & 1) && (uint32_t)__popcll(children & ((1ull << lane) - 1)) < a.width;
            const uint64_t same = __builtin_amdgcn_ballot_w64(offered && a.tokens[q.row0 + lane] == id);
            if (lane == 0) {
                chosen[i] = bad ? -2 : __ffsll((unsigned long long)same) - 1;
                best[i] = id;
            }
        }
    } else if (tid < q.n) {
        chosen[tid] = tv_mark(a, q.row0 + tid).chosen;
    }
    if (tid == 0) found = ~0u;
    __syncthreads();
    // Every thread walks for itself (children have larger numbers: it ends).
    uint32_t node = 0, count = 1;
    uint64_t on = 1;
    while (chosen[node] >= 0) {
        node = (uint32_t)chosen[node];
        on |= 1ull << node;
        count++;
    }
    const uint32_t row = q.row0 + node;
    bool failed = chosen[node] == -2;
    TreeRow s{0.0, 1.0, 0.0, 0.0, 0.0, 0.0};
    TvLaw pl{0.0, 0.0}, ql{0.0, 0.0};
    const uint64_t children = tv_children(parent, node);
    // A leaf below the root has the statistics that the round of its test made.
    const bool late = !children && node;
    const uint32_t stats = late ? a.parts : a.stat_parts;
    uint32_t gone = 0;
    if (!a.greedy && !failed) {
        if (children) {
            gone = tv_mark(a, row).refused;  // (one at least: a child was offered, and none accepted)
            s = a.states[(size_t)(gone & 1) * a.rows + row];
            pl = {s.p_top, s.p_inv};
            ql = {s.q_top, s.q_inv};
        } else {
            pl = tv_law(a, a.stats + (size_t)row * a.parts, stats);
            failed = pl.inv == 0.0;
        }
    }
    // (the path rises: a node's place is the number of its nodes in front)
    if (failed) on = 0, count = 0;
    if (tid >= count && tid < q.n) a.path[q.row0 + tid] = CTOX_NO_SLOT;
    if (tid < 64 && (on >> tid & 1)) a.path[q.row0 + __popcll(on & ((1ull << tid) - 1))] = tid;
    if (tid == 0) a.counts[r] = count;
    if (failed || a.greedy) {
        if (tid == 0) a.next[r] = failed ? CTOX_TREE_FAILED : best[node];
        return;
    }
    if (wave == 0 && (children >> lane & 1)) tried[__popcll(children & ((1ull << lane) - 1))] = a.tokens[q.row0 + lane];
    // The part where the running sum passes the number. Where nothing is left of the target (only rounding could have
    // refused then) the target itself is drawn from.
    double mass = 0.0, in = 0.0;
    for (int again = 0; again < 2; again++) {
        mass = 0.0;
        if (lane < (gone ? a.parts : stats)) {
            if (gone) {
                mass = a.rest[((size_t)(gone - 1) * a.rows + row) * a.parts + lane];
            } else {
                // (of a part without a token of weight, by the border of TvLaw: 0)
                const TreeStat x = a.stats[(size_t)row * a.parts + lane];
                const double y = ((double)x.top - pl.top) * a.c;
                mass = x.sum > 0.0 && y >= -1000.0 ? x.sum * tv_exp2(y) * pl.inv : 0.0;
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
    // (of the parts with mass, since a running sum may grow by a rounding where there is none; the last of them where
    // rounding leaves none past the number)
    const uint64_t massive = __builtin_amdgcn_ballot_w64(mass > 0.0), past = __builtin_amdgcn_ballot_w64(in > goal) & massive;
    const uint32_t part = past ? (uint32_t)__ffsll((unsigned long long)past) - 1
                               : massive ? 63 - (uint32_t)__clzll((long long)massive) : 0;
    const double want = goal - __shfl(in - mass, part);
    __syncthreads();
    // That part's tokens, four a thread and round.
    const TvRow p = tv_target(a, row);
    const TvRest f{a, p, tv_point(a) ? nullptr : a.draft + (size_t)row * a.draft_stride, pl, ql, s.lambda, gone, tried};
    const uint32_t size = gone || late ? a.part : a.stat_part;
    double before = 0.0;
    uint32_t last = 0;  // the last token with a weight, of this thread
    bool has = false;
    for (uint32_t e0 = part * size; e0 < (part + 1) * size && e0 < p.len + p.skew; e0 += 4096) {
        double w[4];
        f.four(e0 + 4 * tid, p.four(e0 + 4 * tid), w);
        const uint32_t i0 = e0 + 4 * tid - p.skew;
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (w[k] > 0.0) last = i0 + k, has = true;
        const double sum = (w[0] + w[1]) + (w[2] + w[3]);
        double run = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double x = __shfl_up(run, o);
            if ((int)lane >= o) run += x;
        }
        if (lane == 63) sums[wave] = run;
        __syncthreads();
        double at = before + run - sum;
#pragma unroll
        for (uint32_t v = 0; v < 16; v++) {
            if (v < wave) at += sums[v];
            before += sums[v];
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            at += w[k];
            if (w[k] > 0.0 && at > want) {
                atomicMin(&found, i0 + k);
                break;
            }
        }
        __syncthreads();
        if (found != ~0u) break;
    }
    if (found == ~0u) {  // rounding: the last token with a weight
        __shared__ uint32_t pick;
        if (tid == 0) pick = 0;
        __syncthreads();
        if (has) atomicMax(&pick, last);
        __syncthreads();
        if (tid == 0) a.next[r] = pick;
        return;
    }
    if (tid == 0) a.next[r] = found;
}
