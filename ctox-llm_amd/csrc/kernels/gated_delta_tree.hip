// The GatedDeltaNet token mixer (Q/src/decoder.rs:863-913, recurrence Q/src/reference.rs:230-297) over trees of
// drafted tokens, gfx950.
//
// A node's recurrence starts from its parent's state, so keeping states would cost 3.1 MB a node and layer. With
// S_0 the request's state and L_i the sum of log decays from the root to node i, all that node i needs is
//   delta_i = beta_i (v_i - e^{L_i} k_i.S_0 - sum_{a above i} e^{L_i - L_a} (k_i.k_a) delta_a)
//   o_i     = e^{L_i} q_i.S_0 + sum_{a above or i} e^{L_i - L_a} (q_i.k_a) delta_a
// (q, k normalised, q over sqrt(key_dim)): S_0 is read once and never written. The state behind the accepted path
// is made when the path is known,
//   S = e^{L_n} S_0 + sum_{a on the path} e^{L_n - L_a} k_a delta_a^T,
// from the k, delta and log decays that the first call leaves in the workspace.
//
//  * ctox_gdn_tree{1,2,4}_gfx950: nodes in tiles of 16. A workgroup takes a head and 64 value columns, a
//    wave 16 of them. Conv + SiLU of the head's q and k channels goes to LDS, k S_0 and q S_0 and the products of
//    nodes (shared by the waves) run on fp32 MFMA 16x16x4. The triangular solve goes tile by tile: what lies
//    in tiles before by MFMA, the 16 x 16 on the diagonal by a lane a column.
//    L is kept in 64 bits: differences of it stay exact to 32 bits however strong the decays before were.
//    A node whose values are no numbers must not reach nodes that are not below it, where a
//    product with 0 would carry it: such waves take sums over ancestors alone (GtSolve's second form).
//  * ctox_gdn_tree_commit_gfx950: the state and the conv windows behind the path; bound by reading and writing the state.
#include <hip/hip_runtime.h>

#include "kernel_args.h"
#include "lds_barrier.h"
#include "tree.h"

typedef float gt_v4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ gt_v4 gt_mfma(float a, float b, gt_v4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

#define GT_TAPS 8
#define GT_ROW 136  // floats of a node's q or k in LDS: dims i at (i % 16) * 8 + i / 16, and padding

// Where channel c's input t positions before a node is: >= 0 a row of the batch, else -1 - (place in the window).
__device__ __forceinline__ float gt_input(const GdnTreeArgs &a, const float *window, int32_t at, uint32_t c) {
    return at >= 0 ? a.proj[(size_t)at * a.proj_stride + c] : window[(size_t)c * a.kernel + (uint32_t)(-1 - at)];
}

template <int NT>
struct GtLds {
    float kq[2][16 * NT][GT_ROW];       // [q, k]
    float am[2][16 * NT][16 * NT + 4];  // [delta, output]: coefficients over nodes a
    float d[4][16 * NT][20];            // a wave's deltas [node][column]
    int32_t taps[16 * NT][GT_TAPS];
    float beta[16 * NT], decay[16 * NT];  // decay: e^{L_i}
    double L[16 * NT];
    uint64_t above[16 * NT];            // ancestors and itself
};

template <int NT>
__device__ __forceinline__ void gdn_tree(const GdnTreeArgs &a) {
    constexpr int N = 16 * NT;
    __shared__ __attribute__((aligned(16))) GtLds<NT> s;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, m = lane & 15;
    const uint32_t groups = (a.value_dim + 63) / 64, head = blockIdx.x / groups, group = blockIdx.x % groups, r = blockIdx.y;
    const TreeRows all = tree_rows(a.row_starts, r, a.rows);
    const TreeRows q{all.row0, min(all.n, (uint32_t)CTOX_TREE_NODES)};
    // (a kernel for each number of tiles; the others' requests are left to them)
    if (q.n == 0 || q.n > (uint32_t)N || (NT > 1 && q.n <= (uint32_t)N / 2)) return;
    const uint32_t dk = a.key_dim, dv = a.value_dim, rep = a.heads / a.key_heads, kh = head / rep, kw = a.key_heads * dk;
    const float *window = a.conv_in + (size_t)r * a.conv_stride;
    const float *state = a.state_in + (size_t)r * a.state_stride;
    const uint32_t column = group * 64 + wave * 16 + m;  // of this lane
    const bool live = column < dv;

    // ---- ancestors, taps, gates: a lane a node ----
    if (wave == 0) {
        const int parent = tree_parent(a.parents, q, lane);
        const uint64_t above = tree_lineage(parent, lane, lane < q.n);
        const int depth = __popcll(above) - 1;
        int at = lane < q.n ? (int)lane : -1;
        for (int t = 0; t < (int)a.kernel; t++) {
            if (lane < (uint32_t)N)
                s.taps[lane][t] = at >= 0 ? (int32_t)(q.row0 + at)
                                          : lane < q.n ? -1 - ((int)a.kernel - t + depth) : -1;
            const int up = __shfl(parent, at < 0 ? (int)lane : at);
            if (at >= 0) at = up;
        }
        float be = 0.0f, ld = 0.0f;
        if (lane < q.n) {
            const float *row = a.proj + (size_t)(q.row0 + lane) * a.proj_stride;
            const float x = row[a.a_off + head] + a.dt_bias[head];
            const float sp = x > 20.0f ? x : log1pf(expf(x));
            ld = -expf(a.a_log[head]) * sp;
            be = 1.0f / (1.0f + expf(-row[a.b_off + head]));
            if (group == 0) a.decays[(size_t)(q.row0 + lane) * a.heads + head] = ld;
        }
        // (e^-1e5 is 0; sums of an infinity would be no numbers below it)
        double L = ld < -1e5f ? -1e5 : (double)ld;
        int up = parent;
#pragma unroll
        for (int i = 0; i < 6; i++) {
            const int from = up < 0 ? (int)lane : up;
            const double x = __shfl(L, from);
            const int u = __shfl(up, from);
            if (up >= 0) {
                L += x;
                up = u;
            }
        }
        if (lane < (uint32_t)N) {
            s.beta[lane] = be;
            s.L[lane] = L;
            s.decay[lane] = expf((float)L);
            s.above[lane] = above;
        }
    }
    // ---- S_0 as the products' operand: lane (g, m) holds rows 4 w + g + 16 e of column m ----
    float sb[4][8];
    if (a.blocked) {
        const uint32_t slices = (dv + 15) / 16;
        const float *base = state + ((size_t)head * slices + min(column / 16, slices - 1)) * 2048;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float4 *p = (const float4 *)(base + (size_t)((4 * w + g) * 16 + m) * 8);
            const float4 x = p[0], y = p[1];
            const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 8; e++) sb[w][e] = live ? v[e] : 0.0f;
        }
    } else {
        const float *base = state + (size_t)head * dk * dv + min(column, dv - 1);
#pragma unroll
        for (int w = 0; w < 4; w++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t i = 4 * w + g + 16 * e;
                const float v = base[(size_t)min(i, dk - 1) * dv];
                sb[w][e] = live && i < dk ? v : 0.0f;
            }
    }
    __syncthreads();
    // ---- conv + SiLU of q and k: a thread a channel, 16 nodes at a time ----
    {
        const uint32_t plane = tid >> 7, i = tid & 127, at = (i & 15) * 8 + (i >> 4);
        const bool mine = i < dk;
        const uint32_t c = (plane ? kw : 0) + kh * dk + (mine ? i : 0);
        float w[GT_TAPS];
#pragma unroll
        for (int t = 0; t < GT_TAPS; t++) w[t] = t < (int)a.kernel ? a.conv_w[(size_t)c * a.kernel + (a.kernel - 1 - t)] : 0.0f;
        for (int n0 = 0; n0 < N; n0 += 16) {
            float y[16];
#pragma unroll
            for (int n = 0; n < 16; n++) y[n] = 0.0f;
            for (int t = 0; t < (int)a.kernel; t++) {
                float wt = 0.0f;
#pragma unroll
                for (int u = 0; u < GT_TAPS; u++) wt = u == t ? w[u] : wt;
#pragma unroll
                for (int n = 0; n < 16; n++) y[n] = fmaf(gt_input(a, window, s.taps[n0 + n][t], c), wt, y[n]);
            }
#pragma unroll
            for (int n = 0; n < 16; n++) {
                const float v = y[n] / (1.0f + expf(-y[n]));
                s.kq[plane][n0 + n][at] = mine && n0 + n < (int)q.n ? v : 0.0f;
            }
        }
    }
    __syncthreads();
    // ---- norms: 16 lanes a row ----
    for (uint32_t row = tid / 16; row < 2 * N; row += 16) {
        const uint32_t plane = row / N, n = row % N;
        float4 *p = (float4 *)&s.kq[plane][n][8 * m];
        float4 x = p[0], y = p[1];
        float sum = ((x.x * x.x + x.y * x.y) + (x.z * x.z + x.w * x.w)) + ((y.x * y.x + y.y * y.y) + (y.z * y.z + y.w * y.w));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        const float f = (1.0f / sqrtf(sum + 1e-6f)) * (plane ? 1.0f : 1.0f / sqrtf((float)dk));
        x = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
        y = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
        p[0] = x;
        p[1] = y;
        if (plane && n < q.n && group == 0 && head % rep == 0) {  // k for the commit, in the order of the dims here
            float4 *o = (float4 *)(a.keys + ((size_t)(q.row0 + n) * a.key_heads + kh) * 128 + 8 * m);
            o[0] = x;
            o[1] = y;
        }
    }
    __syncthreads();
    // ---- products of nodes: tiles (i, a <= i), k k and q k, the waves in turn ----
    {
        int turn = 0;
#pragma unroll
        for (int ti = 0; ti < NT; ti++)
#pragma unroll
            for (int ta = 0; ta <= ti; ta++)
#pragma unroll
                for (int plane = 0; plane < 2; plane++, turn++) {
                    if ((turn & 3) != (int)wave) continue;
                    gt_v4 x = {0.0f, 0.0f, 0.0f, 0.0f};
                    const float *pa = &s.kq[plane][16 * ti + m][0], *pb = &s.kq[1][16 * ta + m][0];
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        const float4 *A = (const float4 *)(pa + (4 * w + g) * 8), *B = (const float4 *)(pb + (4 * w + g) * 8);
                        const float4 a0 = A[0], a1 = A[1], b0 = B[0], b1 = B[1];
                        const float av[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
                        const float bv[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
#pragma unroll
                        for (int e = 0; e < 8; e++) x = gt_mfma(av[e], bv[e], x);
                    }
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const int i = 16 * ti + 4 * g + v, at = 16 * ta + m;
                        const bool on = (s.above[i] >> at & 1) && (plane == 0 || at != i);
                        const float f = on ? expf((float)(s.L[i] - s.L[at])) * (plane ? s.beta[i] : 1.0f) : 0.0f;
                        s.am[plane ? 0 : 1][i][at] = on ? x[v] * f : 0.0f;
                    }
                }
    }
    // ---- v, k S_0, q S_0: rows 16 t + 4 g + v of column m ----
    float rhs[NT][4], oq[NT][4];
    {
        const uint32_t c = 2 * kw + head * dv + (live ? column : 0);
        float w[GT_TAPS];
#pragma unroll
        for (int t = 0; t < GT_TAPS; t++) w[t] = t < (int)a.kernel ? a.conv_w[(size_t)c * a.kernel + (a.kernel - 1 - t)] : 0.0f;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            gt_v4 x[2];
#pragma unroll
            for (int plane = 0; plane < 2; plane++) {
                x[plane] = gt_v4{0.0f, 0.0f, 0.0f, 0.0f};
                const float *pa = &s.kq[plane][16 * t + m][0];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float4 *A = (const float4 *)(pa + (4 * k + g) * 8);
                    const float4 a0 = A[0], a1 = A[1];
                    const float av[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
                    for (int e = 0; e < 8; e++) x[plane] = gt_mfma(av[e], sb[k][e], x[plane]);
                }
            }
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const int i = 16 * t + 4 * g + v;
                float y = 0.0f;
#pragma unroll
                for (int u = 0; u < GT_TAPS; u++)
                    if (u < (int)a.kernel) y = fmaf(gt_input(a, window, s.taps[i][u], c), w[u], y);
                y = y / (1.0f + expf(-y));
                const bool there = i < (int)q.n && live;
                rhs[t][v] = there ? s.beta[i] * (y - s.decay[i] * x[1][v]) : 0.0f;
                oq[t][v] = there ? s.decay[i] * x[0][v] : 0.0f;
            }
        }
    }
    __syncthreads();
    // ---- the solve: (I + A) delta = rhs ----
    float(*d)[20] = s.d[wave];
    bool odd = false;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        gt_v4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 4 * t; k++) x = gt_mfma(s.am[0][16 * t + m][4 * k + g], d[4 * k + g][m], x);
#pragma unroll
        for (int v = 0; v < 4; v++) d[16 * t + 4 * g + v][m] = rhs[t][v] - x[v];
        lds_wave_order();
        // A lane a column (the four lanes of a column do the same).
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; i++) y[i] = d[16 * t + i][m];
#pragma unroll
        for (int i = 1; i < 16; i++) {
            const float4 *row = (const float4 *)&s.am[0][16 * t + i][16 * t];
#pragma unroll
            for (int k = 0; k < (i + 3) / 4; k++) {
                const float4 f = row[k];
                const float fv[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (4 * k + e < i) y[i] = fmaf(-fv[e], y[4 * k + e], y[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 16; i++) odd |= !(fabsf(y[i]) < INFINITY);
        lds_wave_order();
#pragma unroll
        for (int i = 0; i < 16; i++)
            if ((i >> 2) == (int)g) d[16 * t + i][m] = y[i];
        lds_wave_order();
    }
    if (__builtin_amdgcn_ballot_w64(odd)) {  // again, over ancestors alone
        for (int i = 0; i < (int)q.n; i++) {
            float x = 0.0f;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int v = 0; v < 4; v++) x = 16 * t + 4 * (int)g + v == i ? rhs[t][v] : x;
            x = __shfl(x, (int)(((i & 15) >> 2) * 16 + m));
            for (uint64_t up = s.above[i] & ~(1ull << i); up; up &= up - 1) {
                const int at = __ffsll((unsigned long long)up) - 1;
                x = fmaf(-s.am[0][i][at], d[at][m], x);
            }
            lds_wave_order();
            if (g == 0) d[i][m] = x;
            lds_wave_order();
        }
    }
    // ---- outputs ----
#pragma unroll
    for (int t = 0; t < NT; t++) {
        gt_v4 x = {0.0f, 0.0f, 0.0f, 0.0f};
        if (__builtin_amdgcn_ballot_w64(odd)) {
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const int i = 16 * t + 4 * g + v;
                for (uint64_t up = s.above[i]; up; up &= up - 1) {
                    const int at = __ffsll((unsigned long long)up) - 1;
                    x[v] = fmaf(s.am[1][i][at], d[at][m], x[v]);
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4 * (t + 1); k++) x = gt_mfma(s.am[1][16 * t + m][4 * k + g], d[4 * k + g][m], x);
        }
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const uint32_t i = 16 * t + 4 * g + v;
            if (i < q.n && live) {
                const size_t at = ((size_t)(q.row0 + i) * a.heads + head) * dv + column;
                a.out[at] = oq[t][v] + x[v];
                a.deltas[at] = d[i][m];
            }
        }
    }
}
extern "C" __global__ __launch_bounds__(256) void ctox_gdn_tree1_gfx950(GdnTreeArgs a) { gdn_tree<1>(a); }
extern "C" __global__ __launch_bounds__(256) void ctox_gdn_tree2_gfx950(GdnTreeArgs a) { gdn_tree<2>(a); }
extern "C" __global__ __launch_bounds__(256) void ctox_gdn_tree4_gfx950(GdnTreeArgs a) { gdn_tree<4>(a); }

// grid (heads * 16-column slices + groups of 256 channels, requests). Thread (i, j) of 16 x 16 holds rows i + 16 e of a
// column.
extern "C" __global__ __launch_bounds__(256) void ctox_gdn_tree_commit_gfx950(GdnTreeArgs a) {
    __shared__ uint32_t rows[CTOX_TREE_NODES];
    __shared__ uint32_t kept;
    const uint32_t tid = threadIdx.x, r = blockIdx.y;
    const uint32_t slices = (a.value_dim + 15) / 16, parts = a.heads * slices;
    const TreeRows all = tree_rows(a.row_starts, r, a.rows);
    const uint32_t n = min(all.n, (uint32_t)CTOX_TREE_NODES);
    if (tid < 64) {  // the path as far as it names nodes
        const uint32_t count = a.counts[r];
        const bool mine = tid < n && count <= n && tid < count;
        const uint32_t node = mine ? a.path[all.row0 + tid] : ~0u;
        const uint64_t ok = __builtin_amdgcn_ballot_w64(mine && node < n);
        const uint32_t len = (uint32_t)__ffsll((unsigned long long)~ok) - 1;  // (a full mask: 64, from ~0 = 0 -> -1)
        if (tid < n) rows[tid] = all.row0 + (node < n ? node : 0);
        if (tid == 0) kept = ok == ~0ull ? 64 : len;
    }
    __syncthreads();
    const uint32_t len = kept;
    if (blockIdx.x >= parts) {  // conv windows
        const uint32_t c = (blockIdx.x - parts) * 256 + tid, C = 2 * a.key_heads * a.key_dim + a.heads * a.value_dim, K = a.kernel;
        if (c >= C) return;
        const float *in = a.conv_in + (size_t)r * a.conv_stride + (size_t)c * K;
        float *out = a.conv_out + (size_t)r * a.conv_stride + (size_t)c * K;
        float w[GT_TAPS];
        for (uint32_t t = 0; t < K; t++) {  // the last K of the old window and the path's inputs
            const uint32_t at = t + len;
            w[t] = at < K ? in[at] : a.proj[(size_t)rows[at - K] * a.proj_stride + c];
        }
        for (uint32_t t = 0; t < K; t++) out[t] = w[t];
        return;
    }
    const uint32_t head = blockIdx.x / slices, slice = blockIdx.x % slices, i0 = tid / 16, column = slice * 16 + tid % 16;
    const uint32_t dk = a.key_dim, dv = a.value_dim, kh = head / (a.heads / a.key_heads);
    const bool live = column < dv;
    const float *in = a.state_in + (size_t)r * a.state_stride;
    float *out = a.state_out + (size_t)r * a.state_stride;
    const size_t run = ((size_t)blockIdx.x * 256 + tid) * 8;
    float x[8];
    if (a.blocked) {
        const float4 u = ((const float4 *)(in + run))[0], v = ((const float4 *)(in + run))[1];
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t i = i0 + 16 * e;
            x[e] = i < dk && live ? in[((size_t)head * dk + i) * dv + column] : 0.0f;
        }
    }
    for (uint32_t t = 0; t < len; t++) {
        const size_t row = rows[t];
        const float f = expf(a.decays[row * a.heads + head]);
        const float dl = live ? a.deltas[(row * a.heads + head) * dv + column] : 0.0f;
        const float4 *k = (const float4 *)(a.keys + (row * a.key_heads + kh) * 128 + 8 * i0);
        const float4 u = k[0], v = k[1];
        const float kv[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = fmaf(kv[e], dl, x[e] * f);
    }
    if (a.blocked) {
        ((float4 *)(out + run))[0] = make_float4(x[0], x[1], x[2], x[3]);
        ((float4 *)(out + run))[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t i = i0 + 16 * e;
            if (i < dk && live) out[((size_t)head * dk + i) * dv + column] = x[e];
        }
    }
}
