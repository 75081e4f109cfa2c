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
//  * ctox_gdn_tree{1,2,4}{n,w}{4,8}_gfx950: trees of up to 16, 32, 64 nodes, in tiles of 16; a convolution of up to 4 or 8
//    inputs. A workgroup takes a head and 64 (n) or 128 (w) value columns, a wave 16 of them. The inputs go to LDS once, where the convolution picks every
//    node's ancestors; k S_0 and q S_0 and the products of nodes (shared by the waves) run on fp32 MFMA 16x16x4. The
//    triangular solve goes tile by tile: what lies in tiles before by MFMA, the 16 x 16 on the diagonal by a
//    lane a column.
//    L is kept in 64 bits: differences of it stay exact to 32 bits however strong the decays before were.
//    A node whose values are no numbers must not reach nodes that are not below it, where a
//    product with 0 would carry it: such waves take sums over ancestors alone (the second form of the solve).
//  * ctox_gdn_tree_commit_gfx950: the state and the conv windows behind the path; bound by reading and writing the state.
//
// Measured, 48 heads over 16, 128 x 128: a tree of 12 nodes 13.4 us and 4.1 for the commit; 16 trees of up to 64 nodes 106 us
// (110 in the first launches on an idle card; 672 workgroups of 8 waves, two a CU: f32 MFMA 21 us, VALU 20, LDS 25 of the
// CUs' time, in phases between barriers) and 23 us (101 MB of states and 5 of windows, read and written: 4.6 TB/s).
#include <hip/hip_runtime.h>

#include "kernel_args.h"
#include "lds_barrier.h"
#include "tree.h"

typedef float gt_v4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ gt_v4 gt_mfma(float a, float b, gt_v4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

#define GT_ROW 132  // floats of a node's q or k in LDS
// Dims i = j + 16 e of it lie at gt_place(j) + e: a lane's operand is 32 bytes. The second half is four floats further
// on, so that 64 dims in turn meet 64 banks.
__device__ __forceinline__ uint32_t gt_place(uint32_t j) { return 8 * j + (j & 8) / 2; }

// Inputs and q, k are dead when the solve begins: its operands take their place, and two workgroups of 128 columns fit
// a CU. Rows 16 NT + j of the inputs are the window's.
// e^x by the exponential instruction: its argument's rounding makes it |x| 2^-24 off, which for x <= 0 is at most 2.2e-8 of
// 1. silu: x / (1 + e^-x) with the reciprocal instruction, within a few 2^-24 (|x| of them where x is negative,
// of a result of |x| e^x). (expf and the division took 25 instructions more a node and channel.)
__device__ __forceinline__ float gt_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float gt_silu(float x) { return x * __builtin_amdgcn_rcpf(1.0f + gt_exp(-x)); }

template <int NT, int W, int TAPS>
struct GtLds {
    union {
        float kq[2][16 * NT + TAPS][GT_ROW];     // [q, k]
        float v[W][16 * NT + TAPS][20];          // a wave's value channels
        struct {
            float am[2][16 * NT][16 * NT + 4];      // [delta, output]: coefficients over nodes a
            float d[W][16 * NT][20];                // a wave's deltas [node][column]
        } solve;
    } u;
    uint64_t taps[16 * NT];               // a byte each: the row with a node's input of t positions before
    float beta[16 * NT], decay[16 * NT];  // decay: e^{L_i}
    double L[16 * NT];
    uint64_t above[16 * NT];              // ancestors and itself
};

template <int NT, int W, int TAPS>
__device__ __forceinline__ void gdn_tree(const GdnTreeArgs &a) {
    constexpr int N = 16 * NT, PARTS = W / 4, PER = N / PARTS, SLOTS = (NT * (NT + 1) + W - 1) / W;
    constexpr int EACH = 16 / PARTS;  // of a tile's nodes, a thread's
    __shared__ __attribute__((aligned(16))) GtLds<NT, W, TAPS> s;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, m = lane & 15;
    const uint32_t groups = (a.value_dim + 16 * W - 1) / (16 * W), head = blockIdx.x / groups, group = blockIdx.x % groups;
    const uint32_t r = blockIdx.y;
    const TreeRows q = tree_rows(a.row_starts, r, a.rows);
    if (q.n == 0) return;
    if (q.n > N) {  // not a tree of this kernel
        for (uint32_t i = wave; i < q.n; i += W)
            for (uint32_t c = group * 16 * W + lane; c < min((group + 1) * 16 * W, a.value_dim); c += 64)
                a.out[((size_t)(q.row0 + i) * a.heads + head) * a.value_dim + c] = 0.0f;
        return;
    }
    const int nt = (int)(q.n + 15) / 16;  // tiles that have nodes
    const uint32_t dk = a.key_dim, dv = a.value_dim, rep = a.heads / a.key_heads, kh = head / rep, kw = a.key_heads * dk;
    const float *window = a.conv_in + (size_t)r * a.conv_stride;
    const float *state = a.state_in + (size_t)r * a.state_stride;
    const uint32_t column = group * 16 * W + wave * 16 + m;  // of this lane
    const bool live = column < dv;
    const uint32_t vc = 2 * kw + head * dv + (live ? column : 0);  // its channel
    // A thread's q or k channel, and of its nodes every PARTS-th.
    const uint32_t plane = tid >> 7 & 1, dim = tid & 127, at = gt_place(dim & 15) + (dim >> 4), part = wave / 4;
    const bool mine = dim < dk;
    const uint32_t kc = (plane ? kw : 0) + kh * dk + (mine ? dim : 0);

    // ---- inputs, under way until they are stored ----
    float xv[NT][4], wv[TAPS / 4], xk[PER], wk[TAPS], cv[TAPS], ck[TAPS];
#pragma unroll
    for (int t = 0; t < NT; t++)
        if (t < nt)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const uint32_t i = 16 * t + 4 * g + v;
                xv[t][v] = a.proj[(size_t)(q.row0 + min(i, q.n - 1)) * a.proj_stride + vc];
            }
#pragma unroll
    for (int j = 0; j < TAPS / 4; j++) wv[j] = window[(size_t)vc * a.kernel + min(4 * j + g, a.kernel - 1)];
#pragma unroll
    for (int t = 0; t < TAPS; t++) cv[t] = a.conv_w[(size_t)vc * a.kernel + (t < (int)a.kernel ? a.kernel - 1 - t : 0)];
#pragma unroll
    for (int t = 0; t < NT; t++)
        if (t < nt)
#pragma unroll
            for (int i = t * EACH; i < (t + 1) * EACH; i++)
                xk[i] = a.proj[(size_t)(q.row0 + min(PARTS * i + part, q.n - 1)) * a.proj_stride + kc];
#pragma unroll
    for (int j = 0; j < TAPS; j++) wk[j] = window[(size_t)kc * a.kernel + min((uint32_t)j, a.kernel - 1)];
#pragma unroll
    for (int t = 0; t < TAPS; t++) ck[t] = a.conv_w[(size_t)kc * a.kernel + (t < (int)a.kernel ? a.kernel - 1 - t : 0)];
#pragma unroll
    for (int t = 0; t < TAPS; t++)
        if (t >= (int)a.kernel) cv[t] = ck[t] = 0.0f;

    // ---- ancestors and taps, gates: a lane a node ----
    if (wave == 0) {
        const int parent = tree_parent(a.parents, q, lane);
        const uint64_t above = tree_lineage(parent, lane, lane < q.n);
        const int depth = __popcll(above) - 1;
        int from = lane < q.n ? (int)lane : -1;
        // Ancestors, then the window from its end; taps that the kernel does not have (their weight is 0) are the node.
        uint64_t taps = 0;
#pragma unroll
        for (int t = 0; t < TAPS; t++) {
            const int old = lane < q.n ? N + (int)a.kernel - t + depth : N;
            taps |= (uint64_t)(t >= (int)a.kernel ? (int)min(lane, N - 1u) : from >= 0 ? from : old) << (8 * t);
            const int up = __shfl(parent, from < 0 ? (int)lane : from);
            if (from >= 0) from = up;
        }
        if (lane < (uint32_t)N) {
            s.taps[lane] = taps;
            s.above[lane] = above;
        }
    } else if (wave == 1) {
        float be = 0.0f, ld = 0.0f;
        const int parent = tree_parent(a.parents, q, lane);
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
            const int p = up < 0 ? (int)lane : up;
            const double x = __shfl(L, p);
            const int u = __shfl(up, p);
            if (up >= 0) {
                L += x;
                up = u;
            }
        }
        if (lane < (uint32_t)N) {
            s.beta[lane] = be;
            s.L[lane] = L;
            s.decay[lane] = expf((float)L);
        }
    }
    __syncthreads();
    // ---- conv + SiLU of v, a wave's own columns: rows 16 t + 4 g + v of column m ----
    float rhs[NT][4];
    {
        float(*x)[20] = s.u.v[wave];
#pragma unroll
        for (int t = 0; t < NT; t++)
            if (t < nt)
#pragma unroll
                for (int v = 0; v < 4; v++) x[16 * t + 4 * g + v][m] = xv[t][v];
#pragma unroll
        for (int j = 0; j < TAPS / 4; j++) x[N + 4 * j + g][m] = wv[j];
        lds_wave_order();
#pragma unroll
        for (int t = 0; t < NT; t++)
            if (t < nt)
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const uint64_t taps = s.taps[16 * t + 4 * g + v];
                    float y = 0.0f;
#pragma unroll
                    for (int u = 0; u < TAPS; u++) y = fmaf(x[taps >> (8 * u) & 255][m], cv[u], y);
                    rhs[t][v] = gt_silu(y);
                }
    }
    __syncthreads();
    // ---- conv + SiLU of q and k: a thread a channel ----
    {
        float(*x)[GT_ROW] = s.u.kq[plane];
#pragma unroll
        for (int t = 0; t < NT; t++)
            if (t < nt)
#pragma unroll
                for (int i = t * EACH; i < (t + 1) * EACH; i++) x[PARTS * i + part][at] = xk[i];
        if (part == 0)
#pragma unroll
            for (int j = 0; j < TAPS; j++) x[N + j][at] = wk[j];
        if (PARTS > 1) lds_barrier();
#pragma unroll
        for (int t = 0; t < NT; t++)
            if (t < nt)
#pragma unroll
                for (int i = t * EACH; i < (t + 1) * EACH; i++) {
                    const uint32_t n = PARTS * i + part;
                    const uint64_t both = s.taps[n];  // (one node a wave)
                    const uint64_t taps = (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(both >> 32)) << 32 |
                                          __builtin_amdgcn_readfirstlane((uint32_t)both);
                    float y = 0.0f;
#pragma unroll
                    for (int u = 0; u < TAPS; u++) y = fmaf(x[taps >> (8 * u) & 255][at], ck[u], y);
                    xk[i] = mine && n < q.n ? gt_silu(y) : 0.0f;
                }
        if (PARTS > 1) lds_barrier();
#pragma unroll
        for (int t = 0; t < NT; t++)
            if (t < nt)
#pragma unroll
                for (int i = t * EACH; i < (t + 1) * EACH; i++) x[PARTS * i + part][at] = xk[i];
    }
    __syncthreads();
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
            for (int e = 0; e < 8; e++) sb[w][e] = v[e];
        }
    } else {
        const float *base = state + (size_t)head * dk * dv + min(column, dv - 1);
#pragma unroll
        for (int w = 0; w < 4; w++)
#pragma unroll
            for (int e = 0; e < 8; e++) sb[w][e] = base[(size_t)min(4 * w + g + 16 * e, dk - 1) * dv];
    }
    // ---- norms: 16 lanes a row ----
    const float qscale = 1.0f / sqrtf((float)dk);
    for (uint32_t row = tid / 16; row < 32u * nt; row += 4 * W) {
        const uint32_t pl = row & 1, n = row >> 1;
        float4 *p = (float4 *)&s.u.kq[pl][n][gt_place(m)];
        float4 x = p[0], y = p[1];
        float sum = ((x.x * x.x + x.y * x.y) + (x.z * x.z + x.w * x.w)) + ((y.x * y.x + y.y * y.y) + (y.z * y.z + y.w * y.w));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        const float f = __builtin_amdgcn_rsqf(sum + 1e-6f) * (pl ? 1.0f : qscale);
        x = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
        y = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
        p[0] = x;
        p[1] = y;
        if (pl && n < q.n && group == 0 && head % rep == 0) {  // k for the commit, in the order of the dims here
            float4 *o = (float4 *)(a.keys + ((size_t)(q.row0 + n) * a.key_heads + kh) * 128 + 8 * m);
            o[0] = x;
            o[1] = y;
        }
    }
    lds_barrier();
    auto operand = [&](int pl, int tile, int w, float (&x)[8]) {  // rows 16 tile + m, dims 4 w + g + 16 e
        const float4 *p = (const float4 *)&s.u.kq[pl][16 * tile + m][gt_place(4 * w + g)];
        const float4 u = p[0], v = p[1];
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    };
    // ---- products of nodes: tiles (i, a <= i), k k and q k, the waves in turn ----
    gt_v4 gram[SLOTS];
    {
        int turn = 0;
#pragma unroll
        for (int ti = 0; ti < NT; ti++)
#pragma unroll
            for (int ta = 0; ta <= ti; ta++)
#pragma unroll
                for (int pl = 0; pl < 2; pl++, turn++) {
                    if (ti >= nt || turn % W != (int)wave) continue;
                    gt_v4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        float av[8], bv[8];
                        operand(pl, ti, w, av);
                        operand(1, ta, w, bv);
#pragma unroll
                        for (int e = 0; e < 8; e++) x = gt_mfma(av[e], bv[e], x);
                    }
                    gram[turn / W] = x;
                }
    }
    // ---- k S_0, q S_0 ----
    if (!live || dk < 128)
#pragma unroll
        for (int w = 0; w < 4; w++)
#pragma unroll
            for (int e = 0; e < 8; e++) sb[w][e] = live && 4 * w + g + 16 * e < dk ? sb[w][e] : 0.0f;
    float oq[NT][4];
#pragma unroll
    for (int t = 0; t < NT; t++)
        if (t < nt) {
            gt_v4 x[2];
#pragma unroll
            for (int pl = 0; pl < 2; pl++) {
                x[pl] = gt_v4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    float av[8];
                    operand(pl, t, k, av);
#pragma unroll
                    for (int e = 0; e < 8; e++) x[pl] = gt_mfma(av[e], sb[k][e], x[pl]);
                }
            }
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const int i = 16 * t + 4 * g + v;
                const bool there = i < (int)q.n && live;
                rhs[t][v] = there ? s.beta[i] * (rhs[t][v] - s.decay[i] * x[1][v]) : 0.0f;
                oq[t][v] = there ? s.decay[i] * x[0][v] : 0.0f;
            }
        }
    lds_barrier();  // q and k are no longer read
    {
        int turn = 0;
#pragma unroll
        for (int ti = 0; ti < NT; ti++)
#pragma unroll
            for (int ta = 0; ta <= ti; ta++)
#pragma unroll
                for (int pl = 0; pl < 2; pl++, turn++) {
                    if (ti >= nt || turn % W != (int)wave) continue;
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const int i = 16 * ti + 4 * g + v, to = 16 * ta + m;
                        const bool on = (s.above[i] >> to & 1) && (pl == 0 || to != i);
                        const float f = on ? gt_exp((float)(s.L[i] - s.L[to])) * (pl ? s.beta[i] : 1.0f) : 0.0f;
                        s.u.solve.am[pl ? 0 : 1][i][to] = on ? gram[turn / W][v] * f : 0.0f;
                    }
                }
    }
    lds_barrier();
    // ---- the solve: (I + A) delta = rhs ----
    float(*d)[20] = s.u.solve.d[wave];
    const float(*am)[16 * NT][16 * NT + 4] = s.u.solve.am;
    bool odd = false;
#pragma unroll
    for (int t = 0; t < NT; t++)
        if (t < nt) {
            gt_v4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < 4 * t; k++) x = gt_mfma(am[0][16 * t + m][4 * k + g], d[4 * k + g][m], x);
#pragma unroll
            for (int v = 0; v < 4; v++) d[16 * t + 4 * g + v][m] = rhs[t][v] - x[v];
            lds_wave_order();
            // A lane a column (the four lanes of a column do the same). (With inverses of these tiles, made once for
            // all columns, and a product here it took as long.)
            float y[16];
#pragma unroll
            for (int i = 0; i < 16; i++) y[i] = d[16 * t + i][m];
#pragma unroll
            for (int i = 1; i < 16; i++) {
                const float4 *row = (const float4 *)&am[0][16 * t + i][16 * t];
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
    const bool some = __builtin_amdgcn_ballot_w64(odd) != 0;
    if (some) {  // again, over ancestors alone
        for (int i = 0; i < (int)q.n; i++) {
            float x = 0.0f;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int v = 0; v < 4; v++) x = 16 * t + 4 * (int)g + v == i ? rhs[t][v] : x;
            x = __shfl(x, (int)(((i & 15) >> 2) * 16 + m));
            for (uint64_t up = s.above[i] & ~(1ull << i); up; up &= up - 1) {
                const int to = __ffsll((unsigned long long)up) - 1;
                x = fmaf(-am[0][i][to], d[to][m], x);
            }
            lds_wave_order();
            if (g == 0) d[i][m] = x;
            lds_wave_order();
        }
    }
    // ---- outputs ----
#pragma unroll
    for (int t = 0; t < NT; t++)
        if (t < nt) {
            gt_v4 x = {0.0f, 0.0f, 0.0f, 0.0f};
            if (some) {
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const int i = 16 * t + 4 * g + v;
                    for (uint64_t up = s.above[i]; up; up &= up - 1) {
                        const int to = __ffsll((unsigned long long)up) - 1;
                        x[v] = fmaf(am[1][i][to], d[to][m], x[v]);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4 * (t + 1); k++) x = gt_mfma(am[1][16 * t + m][4 * k + g], d[4 * k + g][m], x);
            }
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const uint32_t i = 16 * t + 4 * g + v;
                if (i < q.n && live) {
                    const size_t to = ((size_t)(q.row0 + i) * a.heads + head) * dv + column;
                    a.out[to] = oq[t][v] + x[v];
                    a.deltas[to] = d[i][m];
                }
            }
        }
}
#define CTOX_GDN_TREE(nt, n, w, k) \
    extern "C" __global__ __launch_bounds__(64 * w, 4) void ctox_gdn_tree##nt##n##k##_gfx950(GdnTreeArgs a) { gdn_tree<nt, w, k>(a); }
CTOX_GDN_TREE(1, n, 4, 4)
CTOX_GDN_TREE(2, n, 4, 4)
CTOX_GDN_TREE(4, n, 4, 4)
CTOX_GDN_TREE(1, w, 8, 4)
CTOX_GDN_TREE(2, w, 8, 4)
CTOX_GDN_TREE(4, w, 8, 4)
CTOX_GDN_TREE(1, n, 4, 8)
CTOX_GDN_TREE(2, n, 4, 8)
CTOX_GDN_TREE(4, n, 4, 8)
CTOX_GDN_TREE(1, w, 8, 8)
CTOX_GDN_TREE(2, w, 8, 8)
CTOX_GDN_TREE(4, w, 8, 8)

#define GT_TAPS 8
// grid (heads * 16-column slices + groups of 256 channels, requests). Thread (i, j) of 16 x 16 holds rows i + 16 e of a
// column.
extern "C" __global__ __launch_bounds__(256) void ctox_gdn_tree_commit_gfx950(GdnTreeArgs a) {
    __shared__ uint32_t rows[CTOX_TREE_NODES];
    __shared__ uint32_t kept;
    const uint32_t tid = threadIdx.x, r = blockIdx.y;
    const uint32_t slices = (a.value_dim + 15) / 16, parts = a.heads * slices;
    const TreeRows all = tree_rows(a.row_starts, r, a.rows);
    const uint32_t n = all.n > a.nodes ? 0 : all.n;  // (more: the rows' kernel took it for no tree)
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
