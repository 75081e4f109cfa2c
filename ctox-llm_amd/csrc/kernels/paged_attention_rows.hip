// Grouped-query attention of a ragged batch's new rows over the paged mixed Q2/Q4 cache,
// gfx950: Q/src/reference.rs:420-499 over the pages of Q/src/kv_cache.rs:558-605, for every
// request of a batch in one call and any number of rows.
//
// A request's n new rows are its last n cached tokens; row t sees tokens 0 .. tokens - n + t.
// Its queries are the pairs (row, head of the KV group), numbered row * group + head, so
// that all heads that share a KV head share what is read of it. Three kernels:
//
//  * ctox_gqa_rows_gfx950: 64 queries of one KV head a workgroup (below).
//  * ctox_gqa_few_gfx950: requests of at most 16 queries a KV head (decoded tokens), on the
//    split-KV kernel of paged_attention.hip, which is bound by the cache's bytes.
//  * ctox_gqa_join_gfx950: joins the parts of a split token range.
//
// Which workgroup takes what is decided on the device from row_starts and tokens, so the
// host needs no lengths and a captured launch stays right for other lengths. Every
// workgroup adds up the batch's work for itself and finds its own item: a token range of one
// query tile (or, few, of one request) and KV head. Ranges are made so long that the
// items fill the chip about once.
//
// The 64-query kernel. Eight waves walk the tokens 128 at a time.
//  Scores: wave (tw, qw) takes S^T = K Q^T of 32 tokens x 32 queries on f16 MFMA 32x32x16. K
//    enters as the exact whole numbers 2c - 15 (a Q2 code c is the Q4 code 5c), a 64-dim block's
//    sum is then multiplied by its f32 scale. A query is two f16 parts of q 2^-e (22 bits), held in
//    LDS.
//  Softmax: probabilities are 2^(s - m) with m the queries' maxima of earlier tiles; only when a
//    score exceeds m by more than 2^6 is m moved and the tile's probabilities made again, so that
//    no wave waits for the others' maxima. Sums are f32.
//  Values: probabilities pass through LDS. Wave (blk, th) adds O^T += V^T (P s_v)^T for 64 dims, 64
//    queries and 64 of the tokens, s_v the value block's scale: V is exact again, P s_v is two f16
//    parts in units of 2^(E - 9) with 2^E above every scale so far. V's bytes are transposed on
//    their way into LDS (a lane's operand is one byte column of eight tokens).
// Loads of the next tile are under way during this one; page descriptors are read three ahead.
#include <hip/hip_runtime.h>

#include "kernel_args.h"
#include "lds_barrier.h"

typedef float gr_v16 __attribute__((ext_vector_type(16)));

#define GR_QUERIES 64
#define GR_TOKENS 128
#define GR_MOVE 6.0f  // base-2 slack before the running maximum moves

struct __attribute__((packed, aligned(2))) GrBytes16 {
    uint32_t w[4];
};
struct __attribute__((packed, aligned(2))) GrBytes8 {
    uint32_t w[2];
};
struct __attribute__((packed, aligned(2))) GrBytes4 {
    uint32_t w;
};

// ---------------------------------------------------------------------------
// items
// ---------------------------------------------------------------------------
struct GrRequest {
    uint32_t row0, rows, tokens;
};

__device__ __forceinline__ GrRequest gr_request(const GqaRowsArgs &a, uint32_t r) {
    const uint32_t s = min(a.row_starts[r], a.rows), e = min(a.row_starts[r + 1], a.rows);
    GrRequest q{s, e > s ? e - s : 0u, a.tokens[r]};
    q.tokens = min(q.tokens, a.max_tokens);
    return q;
}

__device__ __forceinline__ bool gr_few(const GqaRowsArgs &a, const GrRequest &q) {
    return a.few && q.rows && q.rows * a.group <= 16;
}

// Of one request: query tiles and units of the token axis (16 tokens for few queries, 128 else).
struct GrShape {
    uint32_t qt, units;
};
__device__ __forceinline__ GrShape gr_shape(const GqaRowsArgs &a, const GrRequest &q, bool few) {
    GrShape s{0, 0};
    if (q.rows == 0 || gr_few(a, q) != few) return s;
    s.qt = few ? 1u : (uint32_t)(((uint64_t)q.rows * a.group + GR_QUERIES - 1) / GR_QUERIES);
    s.units = few ? max(1u, (q.tokens + 15) / 16) : max(1u, (q.tokens + GR_TOKENS - 1) / GR_TOKENS);
    return s;
}

struct GrScratch {
    uint64_t sum[8];
    uint32_t scan[8];
    uint32_t found[4];
};

__device__ __forceinline__ uint64_t gr_wave_sum(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// Units a range may hold: few, a multiple of four (one run per wave).
template <int NT>
__device__ __forceinline__ uint32_t gr_range(const GqaRowsArgs &a, bool few, GrScratch &L) {
    if (!few && !a.split) return 0xffffffffu;
    uint64_t work = 0;
    for (uint32_t r = threadIdx.x; r < a.requests; r += NT) {
        const GrShape s = gr_shape(a, gr_request(a, r), few);
        work += (uint64_t)s.qt * s.units;
    }
    work = gr_wave_sum(work);
    if ((threadIdx.x & 63) == 0) L.sum[threadIdx.x >> 6] = work;
    __syncthreads();
    work = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; w++) work += L.sum[w];
    const uint32_t fill = few ? 4 * a.few_fill : a.fill;
    const uint32_t per = (uint32_t)min((work * a.kv_heads + fill - 1) / fill, (uint64_t)0x3fffffff);
    return few ? 4 * max(1u, per) : max(1u, per);
}

struct GrItem {
    uint32_t request, local, base, ranges;  // base: the request's first item; ranges per query tile
    bool ok;
};

// The item `want` (by_item), or the items of request `want`. All threads get the answer.
template <int NT>
__device__ __forceinline__ GrItem gr_find(const GqaRowsArgs &a, bool few, uint32_t range, uint32_t want, bool by_item,
                                          GrScratch &L) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) L.found[0] = 0xffffffffu;
    uint32_t before = 0;
    for (uint32_t r0 = 0; r0 < a.requests; r0 += NT) {
        const uint32_t r = r0 + threadIdx.x;
        uint32_t n = 0, ranges = 0;
        if (r < a.requests) {
            const GrShape s = gr_shape(a, gr_request(a, r), few);
            ranges = (uint32_t)(((uint64_t)s.units + range - 1) / range);
            n = s.qt * ranges * a.kv_heads;
        }
        uint32_t in = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t x = __shfl_up(in, o);
            if ((int)lane >= o) in += x;
        }
        __syncthreads();
        if (lane == 63) L.scan[wave] = in;
        __syncthreads();
        uint32_t at = before + in - n;
#pragma unroll
        for (int w = 0; w < NT / 64; w++) {
            if (w < (int)wave) at += L.scan[w];
            before += L.scan[w];
        }
        if (n && (by_item ? want >= at && want - at < n : want == r)) {
            L.found[0] = r;
            L.found[1] = at;
            L.found[2] = ranges;
        }
        if (by_item && want < before) break;
    }
    __syncthreads();
    GrItem it{L.found[0], want - L.found[1], L.found[1], L.found[2], L.found[0] != 0xffffffffu};
    __syncthreads();
    return it;
}

// ---------------------------------------------------------------------------
// the 64-query kernel
// ---------------------------------------------------------------------------
struct GrLds {
    float4 p[8][4][64];        // [tw + 4 qw][token octet j][lane]: tokens 8 j + 4 (lane / 32) ..
    uint32_t v[2][4][32][33];  // [buffer][block][code byte][token / 4]: that byte of four tokens
    rm_h8 q[2][2][16][64];     // [qw][lo, hi][k step][lane]
    float vs[2][4][GR_TOKENS]; // [buffer][block][token]: value scale
    float ks[8][4][32];        // [wave][block][token]: key scale / 15
    float mx[2][4][GR_QUERIES];
    float vmax[2][8];
    float lsum[4][GR_QUERIES];
    uint64_t tok[4][GR_TOKENS];  // address of the token's K run | kind << 62 (0 absent: the query's, 1 Q2, 2 Q4)
    uint64_t present[4][2];
    uint32_t holes[4][2];      // [tile][half]: a visible token of it is absent
    uint32_t flag[4];
    GrScratch scratch;
};

__device__ __forceinline__ uint32_t gr_kind(uint64_t t) { return (uint32_t)(t >> 62); }
// (in the global address space by type: a table's address would else be read as a flat one)
typedef const __attribute__((address_space(1))) uint8_t *gr_bytes;
__device__ __forceinline__ gr_bytes gr_at(uint64_t t) { return (gr_bytes)(t & 0x3fffffffffffffffull); }
template <typename T>
__device__ __forceinline__ T gr_load(gr_bytes p) {
    return *(const __attribute__((address_space(1))) T *)p;
}

// Eight 2-bit codes (low 16 bits) as eight 4-bit codes of the same value: c -> 5 c.
__device__ __forceinline__ uint32_t gr_widen(uint32_t x) {
    x &= 0xffffu;
    x = (x | (x << 8)) & 0x00FF00FFu;
    x = (x | (x << 4)) & 0x0F0F0F0Fu;
    x = (x | (x << 2)) & 0x33333333u;
    return x | (x << 2);
}

__device__ __forceinline__ rm_h8 gr_k_operand(uint32_t x) {
    const rm_h2 a = rm_pair<4, 15>(x << 4), b = rm_pair<4, 15>(x), c = rm_pair<4, 15>(x >> 4), d = rm_pair<4, 15>(x >> 8);
    return rm_h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Code byte of tokens 0..3 (x) and 4..7 (y) as operands: even dim (low nibble), odd dim; token
// order 0 2 1 3 4 6 5 7.
__device__ __forceinline__ void gr_v_operands(uint32_t x, uint32_t y, rm_h8 (&o)[2]) {
    const rm_h2 a = rm_pair<4, 15>(x << 4), b = rm_pair<4, 15>(x >> 4), c = rm_pair<4, 15>(y << 4), d = rm_pair<4, 15>(y >> 4);
    const rm_h2 e = rm_pair<4, 15>(x), f = rm_pair<4, 15>(x >> 8), g = rm_pair<4, 15>(y), h = rm_pair<4, 15>(y >> 8);
    o[0] = rm_h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    o[1] = rm_h8{e[0], e[1], f[0], f[1], g[0], g[1], h[0], h[1]};
}

// 0 times anything is 0 here: a probability of zero leaves a masked token's scale out, be it
// infinite or no number.
__device__ __forceinline__ float gr_mul(float p, float s) {
    float x;
    asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(x) : "v"(p), "v"(s));
    return x;
}

// Two f16 parts of eight values in the value operand's token order. hi is rounded towards zero, so
// what is left has hi's sign and at most 13 bits.
__device__ __forceinline__ void gr_split(const float (&x)[8], rm_h8 &hi, rm_h8 &lo) {
    constexpr int at[8] = {0, 2, 1, 3, 4, 6, 5, 7};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float u = x[at[i]], v = x[at[i + 1]];
        const rm_h2 h = __builtin_bit_cast(rm_h2, __builtin_amdgcn_cvt_pkrtz(u, v));
        const rm_h2 l = __builtin_bit_cast(
            rm_h2, __builtin_amdgcn_cvt_pkrtz(fmaf((float)h[0], -1.0f, u), fmaf((float)h[1], -1.0f, v)));
        hi[i] = h[0], hi[i + 1] = h[1];
        lo[i] = l[0], lo[i + 1] = l[1];
    }
}

extern "C" __global__ __launch_bounds__(512, 2) void ctox_gqa_rows_gfx950(GqaRowsArgs a) {
    __shared__ GrLds L;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t li = lane & 31, h = lane >> 5;
    const uint32_t tw = wave & 3, qw = wave >> 2;   // scores: token subtile, query half
    const uint32_t blk = wave & 3, th = wave >> 2;  // values: dim block, token half
    const uint32_t range = gr_range<512>(a, false, L.scratch);
    const GrItem it = gr_find<512>(a, false, range, blockIdx.x, true, L.scratch);
    if (!it.ok) return;
    const GrRequest rq = gr_request(a, it.request);
    // Items of a request: query tiles from the last (the longest) to the first, in each the
    // ranges, in each the KV heads (neighbouring workgroups sit on different XCDs: an XCD's L2
    // then sees few of the KV heads).
    const uint32_t nqt = (uint32_t)(((uint64_t)rq.rows * a.group + GR_QUERIES - 1) / GR_QUERIES);
    const uint32_t kvh = it.local % a.kv_heads, rest = it.local / a.kv_heads;
    const uint32_t part = rest % it.ranges, qt = nqt - 1 - rest / it.ranges;
    const uint32_t q0 = qt * GR_QUERIES, nq = rq.rows * a.group;
    const int32_t past = (int32_t)rq.tokens - (int32_t)rq.rows;  // tokens before the first row
    const int32_t lim0 = past + (int32_t)(q0 / a.group);
    const int32_t seen = past + (int32_t)(min(q0 + GR_QUERIES - 1, nq - 1) / a.group) + 1;
    const uint32_t vis = (uint32_t)max(seen, 0);
    const uint32_t vt = (vis + GR_TOKENS - 1) / GR_TOKENS, per = (vt + it.ranges - 1) / it.ranges;
    const uint32_t t0 = min(part * per, vt), t1 = min(t0 + per, vt);

    // This lane's query (the wave's half for the scores, both halves for the values).
    const uint32_t qi = q0 + 32 * qw + li;
    const bool valid = qi < nq;
    const int32_t lim = valid ? past + (int32_t)(qi / a.group) : -1;
    float qs;
    {
        const uint32_t row = valid ? qi / a.group : 0, g = valid ? qi - row * a.group : 0;
        const float *q = a.query + ((size_t)(rq.row0 + row) * a.query_heads + kvh * a.group + g) * 256 + 32 * h;
        const float pre = valid ? a.scale * 1.44269504088896341f : 0.0f;
        // Eight dims of k step s in the key operand's order (read twice rather than kept).
        auto load = [&](int s, float (&x)[8]) {
            const float4 u = *(const float4 *)(q + 64 * (s >> 2) + 8 * (s & 3));
            const float4 v = *(const float4 *)(q + 64 * (s >> 2) + 8 * (s & 3) + 4);
            const float y[8] = {u.x, v.x, u.y, v.y, u.z, v.z, u.w, v.w};
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = y[i] * pre;
        };
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < 16; s++) {
            float x[8];
            load(s, x);
#pragma unroll
            for (int i = 0; i < 8; i++) mx = fmaxf(mx, fabsf(x[i]) < INFINITY ? fabsf(x[i]) : 0.0f);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        int e = 0;
        frexpf(mx, &e);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int s = 0; s < 16; s++) {
            float x[8];
            load(s, x);
            rm_h8 hi, lo;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float v = ldexpf(x[i], 15 - e);
                hi[i] = (_Float16)v;
                lo[i] = fabsf(v) < INFINITY ? (_Float16)(v - (float)hi[i]) : (_Float16)0.0f;
            }
            if ((uint32_t)(s >> 2) == tw) {  // the four waves of a half write a quarter each
                L.q[qw][0][s][lane] = lo;
                L.q[qw][1][s][lane] = hi;
            }
        }
        qs = ldexpf(1.0f, e - 15);
    }

    // Token -> address. A token past what the tile's queries see, or in no page, is absent: its loads
    // go to the query rows (always there, and long enough), its scales count as 0.
    PagedKvDesc dsc{0, 0, 0, 0};
    auto desc_load = [&](uint32_t t) {
        const uint32_t j = t * GR_TOKENS + tid;
        const uint32_t p = (uint32_t)(((uint64_t)j * a.page_magic) >> a.page_shift);
        dsc = a.desc[(size_t)it.request * a.max_pages + (t < t1 && j < vis ? p : 0)];
    };
    auto desc_write = [&](uint32_t t) {
        const uint32_t j = t * GR_TOKENS + tid, tip = j - dsc.first_token;
        const bool want = t < t1 && j < vis;
        const bool in = want && j >= dsc.first_token && tip < min(dsc.tokens, a.page_tokens), q4 = dsc.precision != 0;
        const uint8_t *pool = q4 ? a.q4 : a.q2;
        const uint8_t *run = pool + (size_t)dsc.physical_slot * (q4 ? a.q4_page_bytes : a.q2_page_bytes) +
                             (size_t)tip * (q4 ? a.q4_token_bytes : a.q2_token_bytes) + kvh * (q4 ? 136 : 72);
        L.tok[t & 3][tid] = in ? (uint64_t)(uintptr_t)run | (q4 ? 2ull << 62 : 1ull << 62) : (uint64_t)(uintptr_t)a.query;
        const uint64_t here = __builtin_amdgcn_ballot_w64(in);
        const uint64_t gone = __builtin_amdgcn_ballot_w64(want && !in);
        if (lane == 0) {
            L.present[t & 3][wave] = here;
            L.holes[t & 3][wave] = gone != 0;
        }
    };

    // Keys: this lane's half of four blocks of one token, and two of its scales. A Q2 half is 8 of
    // the 16 bytes read (what lies behind is the token's own).
    uint32_t kw[4][4];
    uint32_t kkind = 0, ksc[2];
    auto issue_k = [&](uint32_t t) {
        const uint64_t at = L.tok[t & 3][32 * tw + li];
        kkind = gr_kind(at);
        const uint32_t step = kkind == 1 ? 18 : 34;
        const gr_bytes p = gr_at(at), c = p + 2 + (kkind == 1 ? 8 * h : 16 * h);
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const GrBytes16 x = gr_load<GrBytes16>(c + b * step);
#pragma unroll
            for (int i = 0; i < 4; i++) kw[b][i] = x.w[i];
        }
        const gr_bytes sc = p + 2 * h * step;
        ksc[0] = gr_load<uint16_t>(sc);
        ksc[1] = gr_load<uint16_t>(sc + step);
    };
    // Values: eight code bytes (Q4) of four tokens of one block; one scale. The four bytes of a Q2 token
    // are one half of an eight-byte piece of its block.
    const uint32_t vq = tid & 31, vb = (tid >> 5) & 3, vo = tid >> 7;  // token quad, block, octet of bytes
    const uint32_t sb = wave >> 1, st = tid & 127;                      // scale: block, token
    const uint32_t vc4 = a.v_off4 + 34 * vb + 2 + 8 * vo, vc2 = a.v_off2 + 18 * vb + 2 + 8 * (vo >> 1);
    const uint32_t vs4 = a.v_off4 + 34 * sb, vs2 = a.v_off2 + 18 * sb;
    uint32_t vw[4][2], vtwo = 0, vsc = 0;  // vtwo: bit i where token i is Q2
    bool vsk = false;
    auto issue_v = [&](uint32_t t) {
        vtwo = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint64_t at = L.tok[t & 3][4 * vq + i];
            const bool two = gr_kind(at) == 1;
            vtwo |= two ? 1u << i : 0u;
            const GrBytes8 x = gr_load<GrBytes8>(gr_at(at) + (two ? vc2 : vc4));
            vw[i][0] = x.w[0], vw[i][1] = x.w[1];
        }
        const uint64_t at = L.tok[t & 3][st];
        vsk = gr_kind(at) != 0;
        vsc = gr_load<uint16_t>(gr_at(at) + (gr_kind(at) == 1 ? vs2 : vs4));
    };
    auto write_v = [&](uint32_t t) {
        const uint32_t buf = t & 1;
        if (__builtin_amdgcn_ballot_w64(vtwo != 0)) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t x = vo & 1 ? vw[i][1] : vw[i][0];
                const bool two = vtwo >> i & 1;
                vw[i][0] = two ? gr_widen(x) : vw[i][0];
                vw[i][1] = two ? gr_widen(x >> 16) : vw[i][1];
            }
        }
#pragma unroll
        for (int w = 0; w < 2; w++) {
            // 4 x 4 bytes across: byte r of the four tokens into one dword.
            const uint32_t ab0 = __builtin_amdgcn_perm(vw[1][w], vw[0][w], 0x05010400u);
            const uint32_t ab1 = __builtin_amdgcn_perm(vw[1][w], vw[0][w], 0x07030602u);
            const uint32_t cd0 = __builtin_amdgcn_perm(vw[3][w], vw[2][w], 0x05010400u);
            const uint32_t cd1 = __builtin_amdgcn_perm(vw[3][w], vw[2][w], 0x07030602u);
            const uint32_t r = 8 * vo + 4 * w;
            L.v[buf][vb][r][vq] = __builtin_amdgcn_perm(cd0, ab0, 0x05040100u);
            L.v[buf][vb][r + 1][vq] = __builtin_amdgcn_perm(cd0, ab0, 0x07060302u);
            L.v[buf][vb][r + 2][vq] = __builtin_amdgcn_perm(cd1, ab1, 0x05040100u);
            L.v[buf][vb][r + 3][vq] = __builtin_amdgcn_perm(cd1, ab1, 0x07060302u);
        }
        const float s = vsk ? (float)__builtin_bit_cast(_Float16, (uint16_t)vsc) : 0.0f;
        L.vs[buf][sb][st] = s;
        float m = fabsf(s) < INFINITY ? fabsf(s) : 0.0f;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        if (lane == 0) L.vmax[buf][wave] = m;
    };

    gr_v16 o[2][2];  // [query half][even, odd dims]
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[i][c][r] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, den = 0.0f;
    int ev = -200;  // 2^ev above every value scale of the wave's block so far

    if (tid < 4) L.flag[tid] = 0;
    __syncthreads();
    if (tid < GR_TOKENS)
        for (uint32_t t = t0; t < t0 + 3; t++) {
            desc_load(t);
            desc_write(t);
        }
    __syncthreads();
    issue_v(t0);
    issue_k(t0);
    write_v(t0);
    for (uint32_t t = t0; t < t1; t++) {
        const uint32_t buf = t & 1;
        issue_v(t + 1);
        if (tid < GR_TOKENS) desc_load(t + 3);
        // ---- scores ----
        if (__builtin_amdgcn_ballot_w64(kkind == 1)) {
            const bool two = kkind == 1;
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const uint32_t x = kw[b][0], y = kw[b][1];
                kw[b][0] = two ? gr_widen(x) : kw[b][0];
                kw[b][1] = two ? gr_widen(x >> 16) : kw[b][1];
                kw[b][2] = two ? gr_widen(y) : kw[b][2];
                kw[b][3] = two ? gr_widen(y >> 16) : kw[b][3];
            }
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
            L.ks[wave][2 * h + i][li] =
                kkind ? (float)__builtin_bit_cast(_Float16, (uint16_t)ksc[i]) * (1.0f / 15.0f) : 0.0f;
        lds_wave_order();
        gr_v16 s;
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = 0.0f;
        // (opaque: the queries do not change from tile to tile, but are not to be kept in registers)
        uint32_t ql = lane;
        asm volatile("" : "+v"(ql));
#pragma unroll
        for (int b = 0; b < 4; b++) {
            gr_v16 x;
#pragma unroll
            for (int r = 0; r < 16; r++) x[r] = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const rm_h8 kf = gr_k_operand(kw[b][k]);
                x = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, L.q[qw][0][4 * b + k][ql], x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, L.q[qw][1][4 * b + k][ql], x, 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float4 f = *(const float4 *)&L.ks[wave][b][8 * j + 4 * h];
                s[4 * j] = fmaf(f.x, x[4 * j], s[4 * j]);
                s[4 * j + 1] = fmaf(f.y, x[4 * j + 1], s[4 * j + 1]);
                s[4 * j + 2] = fmaf(f.z, x[4 * j + 2], s[4 * j + 2]);
                s[4 * j + 3] = fmaf(f.w, x[4 * j + 3], s[4 * j + 3]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        // ---- masks: a tile that ends past the first query's last token, or has absent tokens ----
        if ((int32_t)((t + 1) * GR_TOKENS) - 1 > lim0 || (L.holes[t & 3][0] | L.holes[t & 3][1])) {
            const uint32_t here = (uint32_t)(L.present[t & 3][tw >> 1] >> (32 * (tw & 1))) >> (4 * h);
            const int32_t left = lim - (int32_t)(t * GR_TOKENS + 32 * tw + 4 * h);  // tokens up to this one
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int c = 8 * (r >> 2) + (r & 3);
                if (c > left || !(here >> c & 1)) s[r] = -INFINITY;
            }
        }
        float top = s[0];
#pragma unroll
        for (int r = 1; r < 16; r++) top = fmaxf(top, s[r]);
        top = fmaxf(top, __shfl_xor(top, 32)) * qs;
        if (h == 0) L.mx[buf][tw][32 * qw + li] = top;
        float mq = qw ? m[1] : m[0];
        if (__builtin_amdgcn_ballot_w64(top > mq + GR_MOVE) && lane == 0) L.flag[t & 3] = 1;
        float sum = 0.0f;
        auto probabilities = [&]() {
            const float ms = mq == -INFINITY ? 0.0f : mq;
            sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float4 p;
                p.x = __builtin_amdgcn_exp2f(fmaf(s[4 * j], qs, -ms));
                p.y = __builtin_amdgcn_exp2f(fmaf(s[4 * j + 1], qs, -ms));
                p.z = __builtin_amdgcn_exp2f(fmaf(s[4 * j + 2], qs, -ms));
                p.w = __builtin_amdgcn_exp2f(fmaf(s[4 * j + 3], qs, -ms));
                sum += (p.x + p.y) + (p.z + p.w);
                L.p[wave][j][lane] = p;
            }
        };
        issue_k(t + 1);
        lds_barrier();  // every wave is done with the tile before's probabilities
        probabilities();
        lds_barrier();
        if (L.flag[t & 3]) {  // the maxima move (the same for every wave)
            float al[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float mn = m[i];
#pragma unroll
                for (int w = 0; w < 4; w++) mn = fmaxf(mn, L.mx[buf][w][32 * i + li]);
                al[i] = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[i] - mn);
                m[i] = mn;
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int r = 0; r < 16; r++) o[i][c][r] *= al[i];
            }
            mq = qw ? m[1] : m[0];
            den *= qw ? al[1] : al[0];
            probabilities();
            lds_barrier();
        }
        den += sum;
        if (tid == 0) L.flag[(t + 2) & 3] = 0;
        write_v(t + 1);
        // ---- values ----
        {
            const float vm = fmaxf(L.vmax[buf][2 * blk], L.vmax[buf][2 * blk + 1]);
            int e = 0;
            frexpf(vm, &e);
            e = __builtin_amdgcn_readfirstlane(vm > 0.0f ? e : -200);
            if (e > ev) {
                const int d = max(ev - e, -300);
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int c = 0; c < 2; c++)
#pragma unroll
                        for (int r = 0; r < 16; r++) o[i][c][r] = ldexpf(o[i][c][r], d);
                ev = e;
            }
        }
        const float unit = ldexpf(1.0f, 9 - max(ev, -100));
#pragma unroll
        for (int kk = 0; kk < 4; kk++) {
            const uint32_t w = 2 * th + (kk >> 1), k = kk & 1, tq = 8 * w + 4 * k + h;
            const uint32_t *vr = L.v[buf][blk][li];
            rm_h8 vf[2];
            gr_v_operands(vr[tq], vr[tq + 2], vf);
            const float4 f0 = *(const float4 *)&L.vs[buf][blk][4 * tq], f1 = *(const float4 *)&L.vs[buf][blk][4 * tq + 8];
            const float f[8] = {f0.x * unit, f0.y * unit, f0.z * unit, f0.w * unit,
                                f1.x * unit, f1.y * unit, f1.z * unit, f1.w * unit};
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float4 p0 = L.p[w + 4 * i][2 * k][lane], p1 = L.p[w + 4 * i][2 * k + 1][lane];
                const float p[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
                float x[8];
    #pragma unroll
                for (int r = 0; r < 8; r++) x[r] = gr_mul(p[r], f[r]);
                rm_h8 hi, lo;
                gr_split(x, hi, lo);
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    o[i][c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[c], lo, o[i][c], 0, 0, 0);
                    o[i][c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[c], hi, o[i][c], 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        // The table of tile t + 3 takes the place of tile t - 1's, which no wave reads after this tile's barrier.
        if (tid < GR_TOKENS) desc_write(t + 3);
    }
    // ---- join the two token halves; every wave writes one query half of its dim block ----
    den += __shfl_xor(den, 32);
    if (h == 0) L.lsum[tw][32 * qw + li] = den;
    __syncthreads();
    float4 *xo = (float4 *)L.q;  // (the queries are dead)
    const uint32_t mine = th, other = 1 - th;
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const gr_v16 &x = other ? o[1][c] : o[0][c];
            xo[((wave * 2 + c) * 4 + j) * 64 + lane] = make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
        }
    __syncthreads();
    const uint32_t src = blk + 4 * other, qo = q0 + 32 * mine + li;
    const float total = (L.lsum[0][32 * mine + li] + L.lsum[1][32 * mine + li]) +
                        (L.lsum[2][32 * mine + li] + L.lsum[3][32 * mine + li]);
    float f = ldexpf(1.0f / 15.0f, max(ev, -100) - 9);
    float *dst;
    if (a.split) {
        float *slot = a.part + (size_t)blockIdx.x * (GR_QUERIES * 258);
        dst = slot + (size_t)(32 * mine + li) * 256;
        if (blk == 0 && h == 0) {
            const float mo = mine ? m[1] : m[0];
            // (scores that are no numbers move no maximum; the part is not an empty one)
            slot[GR_QUERIES * 256 + 2 * (32 * mine + li)] = total != total && mo == -INFINITY ? 0.0f : mo;
            slot[GR_QUERIES * 256 + 2 * (32 * mine + li) + 1] = total;
        }
    } else {
        const uint32_t row = qo / a.group, g = qo - row * a.group;
        if (qo >= nq) return;
        dst = a.out + ((size_t)(rq.row0 + row) * a.query_heads + kvh * a.group + g) * 256;
        f = total != 0.0f ? f / total : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float4 x[2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const float4 y = xo[((src * 2 + c) * 4 + j) * 64 + lane];
            const gr_v16 &z = mine ? o[1][c] : o[0][c];
            x[c] = make_float4((z[4 * j] + y.x) * f, (z[4 * j + 1] + y.y) * f, (z[4 * j + 2] + y.z) * f,
                               (z[4 * j + 3] + y.w) * f);
        }
        float4 *d = (float4 *)(dst + 64 * blk + 16 * j + 8 * h);
        d[0] = make_float4(x[0].x, x[1].x, x[0].y, x[1].y);
        d[1] = make_float4(x[0].z, x[1].z, x[0].w, x[1].w);
    }
}

// ---------------------------------------------------------------------------
// few queries: the split-KV kernel of one sequence, a workgroup for each item
// ---------------------------------------------------------------------------
template <bool ALIGNED>
__device__ __forceinline__ void gqa_few(const GqaRowsArgs &a) {
    __shared__ GrScratch L;
    const uint32_t range = gr_range<256>(a, true, L);
    const GrItem it = gr_find<256>(a, true, range, blockIdx.x, true, L);
    if (!it.ok) return;
    const GrRequest rq = gr_request(a, it.request);
    GqaArgs g{};
    g.query = a.query + (size_t)rq.row0 * a.query_heads * 256;
    g.q2 = a.q2;
    g.q4 = a.q4;
    g.desc = a.desc + (size_t)it.request * a.max_pages;
    g.part_out = a.few_part + (size_t)blockIdx.x * (16 * 258);
    g.part_stats = g.part_out + 16 * 256;
    g.q2_page_bytes = a.q2_page_bytes;
    g.q4_page_bytes = a.q4_page_bytes;
    g.query_heads = a.query_heads;
    g.group = a.group;
    g.tokens = rq.tokens;
    g.rows = rq.rows;
    g.queries = rq.rows * a.group;
    g.page_tokens = a.page_tokens;
    g.page_count = a.max_pages;
    g.component_values = a.kv_heads * 256;
    g.q2_token_bytes = a.q2_token_bytes;
    g.q4_token_bytes = a.q4_token_bytes;
    g.tiles = (rq.tokens + 15) / 16;
    g.tiles_per_wave = range / 4;
    g.scale = a.scale;
    g.tile_pages = ALIGNED;
    const uint32_t kvh = it.local % a.kv_heads, part = it.local / a.kv_heads;
    if constexpr (ALIGNED) paged_gqa_partial16<1, true>(g, kvh, part, 0);
    else paged_gqa_partial<1>(g, kvh, part, 0);
}
extern "C" __global__ __launch_bounds__(256, 2) void ctox_gqa_few_aligned_gfx950(GqaRowsArgs a) { gqa_few<true>(a); }
extern "C" __global__ __launch_bounds__(256, 2) void ctox_gqa_few_gfx950(GqaRowsArgs a) { gqa_few<false>(a); }

// ---------------------------------------------------------------------------
// join: grid (rows, query heads), four waves take every fourth part, 64 lanes x 4 dims
// ---------------------------------------------------------------------------
extern "C" __global__ __launch_bounds__(256) void ctox_gqa_join_gfx950(GqaRowsArgs a) {
    __shared__ GrScratch L;
    __shared__ float4 acc4[4][64];
    __shared__ float st[4][2];
    const uint32_t row = blockIdx.x, head = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (row >= min(a.row_starts[a.requests], a.rows)) return;
    uint32_t lo = 0, hi = a.requests;  // the request of this row: the last that starts at or before it
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (a.row_starts[mid] <= row) lo = mid;
        else hi = mid;
    }
    const GrRequest rq = gr_request(a, lo);
    const bool few = gr_few(a, rq);
    if ((!few && !a.split) || row < rq.row0 || row - rq.row0 >= rq.rows) return;
    const uint32_t range = gr_range<256>(a, few, L);
    const GrItem it = gr_find<256>(a, few, range, lo, false, L);
    if (!it.ok) return;
    const uint32_t kvh = head / a.group, q = (row - rq.row0) * a.group + head % a.group;
    const uint32_t nqt = (uint32_t)(((uint64_t)rq.rows * a.group + GR_QUERIES - 1) / GR_QUERIES);
    const uint32_t tile = few ? 0 : nqt - 1 - q / GR_QUERIES, size = few ? 16 : GR_QUERIES;
    const uint32_t slot0 = it.base + tile * it.ranges * a.kv_heads + kvh;
    const float *base = few ? a.few_part : a.part;
    const uint32_t in = few ? q : q % GR_QUERIES;
    const float unit = few ? 1.44269504088896341f : 1.0f;  // few: maxima in natural units
    float m = -INFINITY, den = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t s0 = wave; s0 < it.ranges; s0 += 16) {
        float4 v[4];
        float ms[4], ds[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t s = min(s0 + 4 * k, it.ranges - 1);
            const float *p = base + (size_t)(slot0 + s * a.kv_heads) * (size * 258);
            v[k] = ((const float4 *)(p + (size_t)in * 256))[lane];
            ms[k] = s0 + 4 * k < it.ranges ? p[size * 256 + 2 * in] * unit : -INFINITY;
            ds[k] = p[size * 256 + 2 * in + 1];
        }
        float mn = m;
#pragma unroll
        for (int k = 0; k < 4; k++) mn = fmaxf(mn, ms[k]);
        if (mn == -INFINITY) continue;
        const float al = __builtin_amdgcn_exp2f(m - mn);
        acc = make_float4(acc.x * al, acc.y * al, acc.z * al, acc.w * al);
        den *= al;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (ms[k] == -INFINITY) continue;  // an empty part: its row is not read into the sum
            const float f = __builtin_amdgcn_exp2f(ms[k] - mn);
            acc = make_float4(fmaf(v[k].x, f, acc.x), fmaf(v[k].y, f, acc.y), fmaf(v[k].z, f, acc.z), fmaf(v[k].w, f, acc.w));
            den = fmaf(ds[k], f, den);
        }
        m = mn;
    }
    acc4[wave][lane] = acc;
    if (lane == 0) {
        st[wave][0] = m;
        st[wave][1] = den;
    }
    __syncthreads();
    if (wave) return;
    float mn = fmaxf(fmaxf(st[0][0], st[1][0]), fmaxf(st[2][0], st[3][0]));
    float4 out = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        if (st[w][0] == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(st[w][0] - mn);
        const float4 x = acc4[w][lane];
        out = make_float4(fmaf(x.x, f, out.x), fmaf(x.y, f, out.y), fmaf(x.z, f, out.z), fmaf(x.w, f, out.w));
        total = fmaf(st[w][1], f, total);
    }
    float inv = total != 0.0f ? 1.0f / total : 0.0f;
    if (few) {  // the few-query kernel's fixed point has no infinities: such a query's scores are no numbers
        const float4 x = ((const float4 *)(a.query + ((size_t)row * a.query_heads + head) * 256))[lane];
        const float big = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
        const bool bad = !(big < INFINITY) || x.x != x.x || x.y != x.y || x.z != x.z || x.w != x.w;
        if (__builtin_amdgcn_ballot_w64(bad) && total != 0.0f) inv = __builtin_nanf("");
    }
    ((float4 *)(a.out + ((size_t)row * a.query_heads + head) * 256))[lane] =
        make_float4(out.x * inv, out.y * inv, out.z * inv, out.w * inv);
}
