// Grouped-query attention of a ragged batch's new rows over the paged mixed Q2/Q4 cache,
// gfx950: Q/src/reference.rs:420-499 over the pages of Q/src/kv_cache.rs:558-605, for every
// request of a batch in one call and any number of rows.
//
// A request's n new rows are its last n cached tokens; row t sees tokens 0 .. tokens - n + t.
// Its queries are the pairs (row, head of the KV group), numbered row * group + head, so
// that all heads that share a KV head share what is read of it.
//
//  * ctox_gqa_rows_gfx950: 128 queries of one KV head a workgroup.
//  * ctox_gqa_few_gfx950: the same for requests of at most 32 queries a KV head (verified drafts),
//    32 queries a workgroup.
//  * ctox_gqa_few16_gfx950: the same for batches in which no request has more than 16 (decoded tokens).
//  * ctox_gqa_join_gfx950: joins the parts of a split token range.
//
// Which workgroup takes what is decided on the device from row_starts and tokens, so the
// host needs no lengths and a captured launch stays right for other lengths: every workgroup
// works out for itself how the batch is cut (gr_range) and finds its own item, a token range
// of one query tile and KV head. What is in one range is written at once, the rest is joined, from
// the cuts that a request's first item leaves in the workspace.
//
// A wave takes 32 queries and walks tiles of 32 tokens; the waves of a workgroup are four (or
// one) query subtiles times two (or four) shares of the tiles. The four subtiles of a share load and
// store a quarter of each tile for all four; the shares meet at the end.
//  Scores: S^T = K Q^T on f16 MFMA 32x32x16. K enters as the exact whole numbers 2c - 15 (a Q2
//    code c is the Q4 code 5c), a 64-dim block's sum is then multiplied by its f32 scale. A query
//    is two f16 parts of q 2^-e (22 bits), held in LDS.
//  Softmax: a lane's sixteen scores belong to one query. Probabilities are 2^(s - m) with m the
//    query's maximum at some earlier tile; only when a score exceeds m by more than GR_MOVE is m moved
//    and the sums rescaled.
//  Values: O^T += V^T (P s_v)^T. The scores' output layout is the probabilities' operand layout if the
//    tokens are counted as gr_v_operands does, so they stay in registers. s_v is the value block's
//    scale: V is exact again, P s_v is two f16 parts in units of 2^(E - 9) with 2^E above every scale
//    of the dim block so far; where those scales differ by more than 2^5 every query has its own unit (GrUnit). V's bytes
//    are transposed on their way into LDS, a lane's operand being one byte column of eight tokens.
// Loads of the next tile are under way during this one, its page descriptors one tile before that.
//
// Measured, 24 query heads over 4 KV heads, pages of 16 tokens, old ones of 2-bit codes: a prompt of 4096 tokens
// 584 us (206 G score and value operations, each twice for the two parts: 706 TFLOP/s of products, where a large
// f16 matrix product of the card reaches 1108), 512 rows behind 32768 tokens 1038 us, 32 decoded tokens over up to 8192
// cached ones 70 us (1.23 TB/s). Bound by vector operations (about 840 a tile and wave, 56 % of all issue,
// beside 30 % of the matrix units' time): 352 of them turn codes into f16 operands, 192 split P s_v. All 256 registers
// are taken; the 7 (128 queries) and 8 (32) spilled ones are read outside the tile loop and in its rare branches.
// With four subtiles K is stored while V is in use and V while K is, so that one buffer each is
// enough beside the 128 KiB of queries, and LDS operands are read one step ahead of the products.
#include <hip/hip_runtime.h>

#include "kernel_args.h"
#include "lds_barrier.h"

typedef float gr_v16 __attribute__((ext_vector_type(16)));

#define GR_MOVE 6.0f  // base-2 slack before the running maximum moves

struct __attribute__((packed, aligned(2))) GrBytes16 {
    uint32_t w[4];
};

// ---------------------------------------------------------------------------
// items
// ---------------------------------------------------------------------------
struct GrRequest {
    uint32_t row0, rows, tokens;
};

__device__ __forceinline__ GrRequest gr_request(const GqaRowsArgs &a, uint32_t r) {
    const uint32_t s = min(a.row_starts[r], a.rows), e = min(a.row_starts[r + 1], a.rows);
    return {s, e > s ? e - s : 0u, min(a.tokens[r], a.max_tokens)};
}

__device__ __forceinline__ bool gr_few(const GqaRowsArgs &a, const GrRequest &q) {
    return q.rows * a.group <= a.few;
}

// Of one request: query tiles, and units of the token axis (as many as a workgroup's waves take at once).
struct GrShape {
    uint32_t qt, units;
};
__device__ __forceinline__ GrShape gr_shape(const GqaRowsArgs &a, const GrRequest &q, bool few) {
    GrShape s{0, 0};
    if (q.rows == 0 || gr_few(a, q) != few) return s;
    s.qt = few ? 1u : (q.rows * a.group + 127) / 128;
    s.units = max(1u, few ? (q.tokens + 127) / 128 : (q.tokens + 63) / 64);
    return s;
}

#define GR_UNCUT 0x3fffffffu  // a range that holds any request
struct GrScratch {
    GrShape shape[CTOX_GQA_CUT_REQUESTS];
    uint32_t count[32], longest, range;
    uint32_t scan[8];
    uint32_t found[4];
};

// A unit is the tokens that a workgroup's waves take at once: 64 with 128 queries, else 128.
// Units of one item. Candidates: the longest request in n = 1 .. 16 and on to 256 ranges. A candidate
// takes as many rounds of the chip as its items fill it, each as long as a range and the
// GR_START units that a workgroup spends on starting and joining; the cheapest one is taken. n = 1
// is always allowed, the others up to the items that the workspace holds.
#define GR_START 3
template <int NT>
__device__ __forceinline__ uint32_t gr_range(const GqaRowsArgs &a, bool few, GrScratch &L) {
    const uint32_t slots = few ? a.few_slots : a.slots, most = few ? a.few_items : a.items;
    if ((!few && !a.split) || a.requests > CTOX_GQA_CUT_REQUESTS) return GR_UNCUT;
    const uint32_t tid = threadIdx.x, c = tid & 31;
    if (tid < 32) L.count[tid] = 0;
    if (tid == 0) L.longest = 1;
    __syncthreads();
    for (uint32_t r = tid; r < a.requests; r += NT) {
        const GrShape s = gr_shape(a, gr_request(a, r), few);
        L.shape[r] = s;
        if (s.qt) atomicMax(&L.longest, s.units);
    }
    __syncthreads();
    const uint32_t n = c < 16 ? c + 1 : (uint32_t)(16.0f * __builtin_amdgcn_exp2f((float)(c - 15) * 0.25f));
    const uint32_t range = (L.longest + n - 1) / n;
    uint32_t items = 0;
    for (uint32_t r = tid >> 5; r < a.requests; r += NT / 32) {
        const GrShape s = L.shape[r];
        items += s.qt * ((s.units + range - 1) / range);
    }
    atomicAdd(&L.count[c], items);  // whole numbers: their order does not matter
    __syncthreads();
    if (tid < 32) {
        const uint32_t k = L.count[c] * a.kv_heads;
        uint64_t cost = min((uint64_t)((k + slots - 1) / slots) * (range + GR_START), (uint64_t)0xfffffffe);
        if (c && k > most) cost = 0xffffffff;
        cost = cost << 32 | range;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t x = __shfl_xor(cost, o);
            cost = x < cost ? x : cost;
        }
        if (tid == 0) L.range = (uint32_t)cost;
    }
    __syncthreads();
    return L.range;
}

struct GrItem {
    uint32_t request, local, base, ranges;  // base: the request's first item; ranges per query tile
    bool ok;
};

// The request of item `want`. All threads get the answer.
template <int NT>
__device__ __forceinline__ GrItem gr_find(const GqaRowsArgs &a, bool few, uint32_t range, uint32_t want,
                                          GrScratch &L) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) L.found[0] = 0xffffffffu;
    uint32_t before = 0;
    for (uint32_t r0 = 0; r0 < a.requests; r0 += NT) {
        const uint32_t r = r0 + threadIdx.x;
        uint32_t n = 0, ranges = 0;
        if (r < a.requests) {
            const GrShape s = range == GR_UNCUT ? gr_shape(a, gr_request(a, r), few) : L.shape[r];
            ranges = (s.units + range - 1) / range;
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
        if (n && want >= at && want - at < n) {
            L.found[0] = r;
            L.found[1] = at;
            L.found[2] = ranges;
        }
        if (want < before) break;
    }
    __syncthreads();
    GrItem it{L.found[0], want - L.found[1], L.found[1], L.found[2], L.found[0] != 0xffffffffu};
    __syncthreads();
    return it;
}

// ---------------------------------------------------------------------------
// operands
// ---------------------------------------------------------------------------
typedef const __attribute__((address_space(1))) uint8_t *gr_bytes;
template <typename T>
__device__ __forceinline__ T gr_load(gr_bytes p) {
    return *(const __attribute__((address_space(1))) T *)p;
}

// Eight 2-bit codes (16 bits of x: the upper ones if `upper`) as eight 4-bit codes of the same value: c -> 5 c.
__device__ __forceinline__ uint32_t gr_widen(uint32_t x, bool upper) {
    x = __builtin_amdgcn_perm(0u, x, upper ? 0x0C030C02u : 0x0C010C00u);  // (0x0C: a byte of zeros)
    x = (x | (x << 4)) & 0x0F0F0F0Fu;
    x = (x | (x << 2)) & 0x33333333u;
    return x | (x << 2);
}

__device__ __forceinline__ rm_h8 gr_k_operand(uint32_t x, const RmMagic &g) {
    const uint32_t w[4] = {x, x, x, x};
    return rm_unpack<true>(w, 0, g);
}

// Code byte of tokens 0..3 (x) and 4..7 (y) as operands: even dim (low nibble), odd dim; token
// order 0 2 1 3 4 6 5 7.
__device__ __forceinline__ void gr_v_operands(uint32_t x, uint32_t y, const RmMagic &g, rm_h8 (&o)[2]) {
    auto two = [&](uint32_t v) { return rm_pair<4, 15>(v, g.m[0], g.magic); };
    const rm_h2 a = two(x << 4), b = two(x >> 4), c = two(y << 4), d = two(y >> 4);
    const rm_h2 e = two(x), f = two(x >> 8), p = two(y), q = two(y >> 8);
    o[0] = rm_h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    o[1] = rm_h8{e[0], e[1], f[0], f[1], p[0], p[1], q[0], q[1]};
}

// Four lanes' dwords across: lane i of four gets byte i of each.
__device__ __forceinline__ uint32_t gr_across(uint32_t x, uint32_t lane) {
    // selectors out of (own, other): halves with lane ^ 2, then bytes with lane ^ 1
    const uint32_t two = lane & 2 ? 0x07060302u : 0x01000504u, one = lane & 1 ? 0x07030501u : 0x02060004u;
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, true);  // of lane ^ 2
    const uint32_t a = __builtin_amdgcn_perm(x, y, two);
    const uint32_t b = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0xB1, 0xF, 0xF, true);  // of lane ^ 1
    return __builtin_amdgcn_perm(a, b, one);
}

// A loading lane's token (of 32) and block (of a pair), and the tokens' bits out of a ballot of the first block's.
__device__ __forceinline__ uint32_t gr_token(uint32_t lane) { return (lane & 3) | (lane >> 3) << 2; }
__device__ __forceinline__ uint32_t gr_tokens(uint64_t x) {
    x &= 0x0F0F0F0F0F0F0F0Full;
    x = (x | x >> 4) & 0x00FF00FF00FF00FFull;
    x = (x | x >> 8) & 0x0000FFFF0000FFFFull;
    return (uint32_t)(x | x >> 16);
}

// Exponent of a query whose largest |q * scale * log2 e| is mx: mx < 2^e. Not below -64, so that the scores' unit
// 2^(e - 15) stays a normal number (0 times a masked score's -inf would be no number). What a smaller
// query loses there, 2^-24 units of each value, moves a score by less than 2^(-24 - 79 + 16 + 8).
__device__ __forceinline__ int gr_query_exponent(float mx) {
    int e = 0;
    frexpf(mx, &e);
    return max(e, -64);
}

// Two f16 parts of eight values in the value operand's token order. hi is rounded towards zero, so
// what is left has hi's sign and at most 13 bits.
// (x - hi is one mixed-precision multiply-add by an opaque -1; a plain difference would convert first.)
__device__ __forceinline__ void gr_split(const float (&x)[8], float minus_one, rm_h8 &hi, rm_h8 &lo) {
    constexpr int at[8] = {0, 2, 1, 3, 4, 6, 5, 7};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float u = x[at[i]], v = x[at[i + 1]];
        const rm_h2 h = __builtin_bit_cast(rm_h2, __builtin_amdgcn_cvt_pkrtz(u, v));
        const rm_h2 l = __builtin_bit_cast(rm_h2, __builtin_amdgcn_cvt_pkrtz(fmaf((float)h[0], minus_one, u), fmaf((float)h[1], minus_one, v)));
        hi[i] = h[0], hi[i + 1] = h[1];
        lo[i] = l[0], lo[i + 1] = l[1];
    }
}

// Value scales of a wide range. P s_v in units of 2^(E - 9) ends at f16's last bit, 2^-24 of them. That is far below
// any result as long as all scales so far lie within 2^-6 .. 1 of 2^E: a query's largest probability is 1 or
// more, so its sum of p |v| is at least 2^(E - 6) / 15, and T tokens lose at most T 2^(E - 33), less than the
// roundings of a sum of T in 32 bits. Otherwise (a token that the query does not see, or hardly counts, may have set E; a
// scale may be 0) every query takes a unit of its own for the tile: its largest |P s_v| goes to 2^14 .. 2^15, the sums
// with it and back, by powers of two. (Measured where every third page has a token of scales 64 times smaller: 32 decoded
// tokens 82 us instead of 73, 512 rows behind 32768 1350 us instead of 1038. The choice costs all others 2 %.)
struct GrUnit {
    float up, down;
    // (60 at most: sums of 2^30 tokens stay below 2^(30 + 19 + 60))
    __device__ __forceinline__ explicit GrUnit(float z) {
        int e = 0;
        frexpf(z, &e);
        const int d = z > 0.0f ? max(0, min(15 - e, 60)) : 0;
        up = ldexpf(1.0f, d);
        down = ldexpf(1.0f, -d);
    }
};

// ---------------------------------------------------------------------------
// tiles from the pages
// ---------------------------------------------------------------------------
// A tile of 32 tokens comes in four pieces, two of K and two of V, of two dim blocks each. A lane loads one block of one
// token: 32 code bytes (Q2: 16, both loads the same) and a scale. A token past what the item's queries see, or
// in no page, is absent: its loads go to the query rows (always there), its scales count as 0. R: pieces
// of one wave, from `piece` on.
template <int R>
struct GrLoad {
    const GqaRowsArgs &a;
    const uint32_t request, kvh, vis, t1, token, pb, piece;
    PagedKvDesc dsc{0, 0, 0, 0};
    uint32_t raw[R][8], rsc[R], rkind = 0;  // rkind: 0 absent, 1 Q2, 2 Q4
    uint32_t here = 0, next = 0;            // tokens that are there: of the tile before, and of the one in `raw`
    int ve[R];                              // 2^ve above every value scale of the lane's block so far

    __device__ __forceinline__ GrLoad(const GqaRowsArgs &a, uint32_t request, uint32_t kvh, uint32_t vis, uint32_t t1,
                                      uint32_t lane, uint32_t piece)
        : a(a), request(request), kvh(kvh), vis(vis), t1(t1), token(gr_token(lane)), pb(lane >> 2 & 1), piece(piece) {
#pragma unroll
        for (int i = 0; i < R; i++) ve[i] = -100;
    }
    __device__ __forceinline__ uint32_t block(int i) const { return 2 * ((piece + i) & 1) + pb; }
    __device__ __forceinline__ void desc_load(uint32_t t) {
        const uint32_t j = t * 32 + token;
        const uint32_t p = (uint32_t)(((uint64_t)j * a.page_magic) >> a.page_shift);
        dsc = a.desc[(size_t)request * a.max_pages + (t < t1 && j < vis ? p : 0)];
    }
    // The loads of tile t, after those of tile `after`'s descriptors, which are waited for first.
    __device__ __forceinline__ void issue(uint32_t t, uint32_t after) {
        const uint32_t j = t * 32 + token, tip = j - dsc.first_token;
        const bool want = t < t1 && j < vis;
        const bool in = want && j >= dsc.first_token && tip < min(dsc.tokens, a.page_tokens), q4 = dsc.precision != 0;
        const uint8_t *pool = q4 ? a.q4 : a.q2;
        const uint32_t bytes = q4 ? 34 : 18;
        const uint8_t *run = pool + (size_t)dsc.physical_slot * (q4 ? a.q4_page_bytes : a.q2_page_bytes) +
                             (size_t)tip * (q4 ? a.q4_token_bytes : a.q2_token_bytes) + (4 * kvh + pb) * bytes;
        rkind = in ? (q4 ? 2u : 1u) : 0u;
        here = next;
        next = gr_tokens(__builtin_amdgcn_ballot_w64(in));
        desc_load(after);
        const gr_bytes p = in ? (gr_bytes)(uintptr_t)run : (gr_bytes)(uintptr_t)a.query;
        const uint32_t second = rkind == 1 ? 2 : 18, pair = in ? 2 * bytes : 0, v = in ? (q4 ? a.v_off4 : a.v_off2) : 0;
#pragma unroll
        for (int i = 0; i < R; i++) {
            const uint32_t n = piece + i;
            const gr_bytes c = p + (n & 1 ? pair : 0) + (n >> 1 ? v : 0);
            const GrBytes16 x = gr_load<GrBytes16>(c + 2), y = gr_load<GrBytes16>(c + second);
#pragma unroll
            for (int w = 0; w < 4; w++) raw[i][w] = x.w[w], raw[i][4 + w] = y.w[w];
            rsc[i] = gr_load<uint16_t>(c);
        }
    }
    __device__ __forceinline__ void widen(int i) {
        if (__builtin_amdgcn_ballot_w64(rkind == 1)) {
            const uint32_t two = rkind == 1 ? ~0u : 0u;  // (a mask: a choice would become a branch for every word)
            const uint32_t y[4] = {raw[i][0], raw[i][1], raw[i][2], raw[i][3]};
#pragma unroll
            for (int w = 0; w < 8; w++) raw[i][w] = (gr_widen(y[w >> 1], w & 1) & two) | (raw[i][w] & ~two);
        }
    }
    __device__ __forceinline__ float scale(int i) const {
        return rkind ? (float)__builtin_bit_cast(_Float16, (uint16_t)rsc[i]) : 0.0f;
    }
    __device__ __forceinline__ float key_scale(int i) const { return scale(i) * (1.0f / 15.0f); }
    // Piece i, of V: code bytes across, scales in units of 2^(9 - E), E, the tokens without a finite scale, and marks:
    // 1 there are such tokens, 2 there are scales below 2^(E - 5).
    __device__ __forceinline__ void store_v(int i, uint32_t lane, uint32_t (&v)[32][9], float (&vs)[32], int &ev,
                                            uint32_t &bads, uint32_t &marks) {
        // (opaque with one piece: what follows from the lane alone is not to be kept in registers from tile to tile)
        if (R == 1) asm volatile("" : "+v"(lane));
        widen(i);
        float sv = scale(i), u = ldexpf(sv, 9 - ve[i]);
        uint32_t bad = 0, mark = 0;
        if (__builtin_amdgcn_ballot_w64(rkind && !(fabsf(u) >= 16.0f && fabsf(u) < 512.0f))) {
            const bool odd = !(fabsf(sv) < INFINITY);
            bad = gr_tokens(__builtin_amdgcn_ballot_w64(odd) >> (4 * pb));
            if (odd) sv = 0.0f;
            float z = fabsf(sv);
#pragma unroll
            for (int d = 1; d < 64; d <<= 1)
                if (d != 4) z = fmaxf(z, __shfl_xor(z, d));
            int e = 0;
            frexpf(z, &e);
            if (z != 0.0f) ve[i] = max(ve[i], e);
            u = ldexpf(sv, 9 - ve[i]);
            mark = (bad ? 1u : 0u) | (__builtin_amdgcn_ballot_w64(rkind && fabsf(u) < 16.0f) ? 2u : 0u);
        }
        vs[R == 1 ? gr_token(lane) : token] = u;
        if ((lane & 59) == 0) {
            ev = ve[i];
            bads = bad;
            marks = mark;
        }
#pragma unroll
        for (int w = 0; w < 8; w++) v[4 * w + (lane & 3)][lane >> 3] = gr_across(raw[i][w], lane);
    }
};

// ---------------------------------------------------------------------------
// attention of one item
// ---------------------------------------------------------------------------
// LDS of a workgroup of QS query subtiles x TS token shares: queries and the shares' tiles (while
// tiles run; the joined sums afterwards).
template <int QS, int TS>
struct GrLds {
    union {
        struct {
            rm_h8 q[QS][2][16][64];     // [subtile][lo, hi][k step][lane]
            uint4 k[TS][4][2][34];      // [share][block][half][token]: that half's code bytes
            uint32_t v[TS][4][32][9];   // [share][block][code byte][token / 4]: that byte of four tokens
            float ks[TS][4][32];        // [share][block][token]: key scale / 15
            float vs[TS][4][32];        // value scale in units of 2^(9 - E)
            int ev[TS][4];              // E of a block
            uint32_t bad[TS][4];        // its tokens without a finite value scale
            uint32_t marks[TS][4];      // as store_v leaves them
        } t;
        float4 sum[QS * TS / 2][32][64];  // [publishing wave][dim block, parity, register quad][lane]
        GrScratch scratch;
    } u;
    float stat[QS * TS][2][32];  // (maximum, denominator) of a publishing wave
};

template <int QS, int TS>
__device__ __forceinline__ void gqa_rows(const GqaRowsArgs &a) {
    constexpr int NT = 64 * QS * TS;
    constexpr bool FEW = QS == 1;
    constexpr uint32_t kQueries = 32 * QS;
    __shared__ GrLds<QS, TS> L;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t li = lane & 31, h = lane >> 5, qsub = wave % QS, ts = wave / QS;
    const uint32_t range = gr_range<NT>(a, FEW, L.u.scratch);
    const GrItem it = gr_find<NT>(a, FEW, range, blockIdx.x, L.u.scratch);
    if (!it.ok) return;
    if (it.local == 0 && threadIdx.x == 0) {
        a.cuts[2 * it.request] = it.base;
        a.cuts[2 * it.request + 1] = it.ranges;
    }
    const GrRequest rq = gr_request(a, it.request);
    // Items of a request: query tiles from the last (the longest) to the first, in each the
    // ranges, in each the KV heads (neighbouring workgroups sit on different XCDs: an XCD's L2
    // then sees few of the KV heads).
    const uint32_t nq = rq.rows * a.group, nqt = (nq + kQueries - 1) / kQueries;
    const uint32_t kvh = it.local % a.kv_heads, rest = it.local / a.kv_heads;
    const uint32_t part = rest % it.ranges, q0 = (nqt - 1 - rest / it.ranges) * kQueries;
    const int32_t past = (int32_t)rq.tokens - (int32_t)rq.rows;  // tokens before the first row
    const int32_t seen = past + (int32_t)(min(q0 + kQueries - 1, nq - 1) / a.group) + 1;
    const uint32_t vis = (uint32_t)max(seen, 0);
    const uint32_t units = (vis + 32 * TS - 1) / (32 * TS), per = (units + it.ranges - 1) / it.ranges;
    // Tiles of 32 tokens: this wave's are t0, t0 + TS, ... below t1 (a last one may have no tokens).
    const uint32_t t0 = min(part * per, units) * TS + ts, t1 = min(part * per + per, units) * TS;

    const uint32_t qi = q0 + 32 * qsub + li;  // this lane's query
    const bool valid = qi < nq;
    const int32_t lim = valid ? past + (int32_t)(qi / a.group) : -1;
    const int32_t lim0 = past + (int32_t)(min(q0 + 32 * qsub, nq - 1) / a.group);  // the subtile's first query's
    const uint32_t qrow = valid ? qi / a.group : 0, qg = valid ? qi - qrow * a.group : 0;
    const size_t qat = ((size_t)(rq.row0 + qrow) * a.query_heads + kvh * a.group + qg) * 256;

    // With four subtiles each wave loads one piece of its share's tile for all four, else the one wave all of them.
    // (A SIMD has one wave of each share: one of them stores K, the other V, so that SIMDs stay level.)
    constexpr int R = QS == 4 ? 1 : 4;
    constexpr int AHEAD = QS == 4 ? 1 : 0;  // steps that LDS operands are read ahead (no registers for it in the other)
    GrLoad<R> ld{a, it.request, kvh, vis, t1, lane, QS == 4 ? qsub ^ (2 * ts) : 0};
    auto store_k = [&](int i) {
        const uint32_t b = ld.block(i);
        ld.widen(i);
        L.u.t.ks[ts][b][ld.token] = ld.key_scale(i);
        const uint32_t(&x)[8] = ld.raw[i];
        L.u.t.k[ts][b][0][ld.token] = make_uint4(x[0], x[1], x[2], x[3]);
        L.u.t.k[ts][b][1][ld.token] = make_uint4(x[4], x[5], x[6], x[7]);
    };
    auto store_v = [&](int i) {
        const uint32_t b = ld.block(i);
        ld.store_v(i, lane, L.u.t.v[ts][b], L.u.t.vs[ts][b], L.u.t.ev[ts][b], L.u.t.bad[ts][b], L.u.t.marks[ts][b]);
    };

    const RmMagic magic = rm_magic<true>();
    float minus_one = -1.0f;
    asm("" : "+v"(minus_one));
    ld.desc_load(t0);
    float qs;
    {
        const float *q = a.query + qat + 32 * h;
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
        const int e = gr_query_exponent(mx);
        qs = ldexpf(1.0f, e - 15);
        // The waves of a subtile write a share of it each.
#pragma unroll
        for (int k = 0; k < 16 / TS; k++) {
            const int s = ts * (16 / TS) + k;
            float x[8];
            load(s, x);
            rm_h8 hi, lo;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float v = ldexpf(x[i], 15 - e);
                hi[i] = (_Float16)v;
                lo[i] = fabsf(v) < INFINITY ? (_Float16)(v - (float)hi[i]) : (_Float16)0.0f;
            }
            L.u.t.q[qsub][0][s][lane] = lo;
            L.u.t.q[qsub][1][s][lane] = hi;
        }
    }
    if (QS == 1) __syncthreads();

    gr_v16 o[4][2];  // [dim block][even, odd dims]
#pragma unroll
    for (int b = 0; b < 4; b++)
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[b][c][r] = 0.0f;
    float m = -INFINITY, den = 0.0f;
    int ev[4] = {-100, -100, -100, -100};  // E of the blocks' sums
    int first[4] = {0, 0, 0, 0};           // the first of them
    bool wide = false;                     // value scales that GrUnit is for have been seen

    ld.issue(t0, t0 + TS);
    if (QS == 4 && ld.piece < 2) {
        store_k(0);
        ld.issue(t0 + TS, t0 + 2 * TS);
    }
    // (nothing under way on entry: the loop's waits are then counted by the order of its own loads alone)
    __builtin_amdgcn_s_waitcnt(0x0F70);
    for (uint32_t t = t0; t < t1; t += TS) {
        // ---- this tile's bytes and scales into LDS; the next tile's loads ----
        // With four subtiles K is written during the values before it, V during the scores before it:
        // `raw` holds K of the next tile, or V of this one.
        if (QS == 4) {
            lds_barrier();  // K is written, the last tile's V is no longer read
            if (ld.piece >= 2) store_v(0);
        } else {
            store_k(0);
            store_k(1);
            store_v(2);
            store_v(3);
            lds_wave_order();
        }
        if (QS != 4 || ld.piece >= 2) {
            ld.issue(t + TS, t + 2 * TS);
        }
        // ---- scores ----
        gr_v16 s;
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = 0.0f;
        // (opaque: the queries do not change from tile to tile, but are not to be kept in registers)
        uint32_t ql = lane;
        asm volatile("" : "+v"(ql));
        // Operands are read a step (two products) ahead; without the fences the reads would sink to their uses.
        rm_h8 qf[2][2];
        float4 kf4[4];
        uint4 kq, kn;
        if (AHEAD) kq = L.u.t.k[ts][0][h][li];
        if (AHEAD) qf[0][0] = L.u.t.q[qsub][0][0][ql], qf[0][1] = L.u.t.q[qsub][1][0][ql];
        gr_v16 x;
#pragma unroll
        for (int n = 0; n < 16; n++) {
            const int b = n >> 2, k = n & 3;
            if (n + AHEAD < 16) {
                qf[(n + AHEAD) & 1][0] = L.u.t.q[qsub][0][n + AHEAD][ql];
                qf[(n + AHEAD) & 1][1] = L.u.t.q[qsub][1][n + AHEAD][ql];
            }
            if (AHEAD && k == 3)
#pragma unroll
                for (int j = 0; j < 4; j++) kf4[j] = *(const float4 *)&L.u.t.ks[ts][b][8 * j + 4 * h];
            if (AHEAD && k == 2) kn = L.u.t.k[ts][min(b + 1, 3)][h][li];
            if (k == 0) {
                if (!AHEAD) kq = L.u.t.k[ts][b][h][li];
#pragma unroll
                for (int r = 0; r < 16; r++) x[r] = 0.0f;
            }
            if (AHEAD) __builtin_amdgcn_sched_barrier(0x76);
            const rm_h8 kf = gr_k_operand(k == 0 ? kq.x : k == 1 ? kq.y : k == 2 ? kq.z : kq.w, magic);
            x = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[n & 1][0], x, 0, 0, 0);
            x = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[n & 1][1], x, 0, 0, 0);
            if (AHEAD) __builtin_amdgcn_sched_barrier(0x76);
            if (k == 3) {
                if (AHEAD) kq = kn;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float4 f = AHEAD ? kf4[j] : *(const float4 *)&L.u.t.ks[ts][b][8 * j + 4 * h];
                    s[4 * j] = fmaf(f.x, x[4 * j], s[4 * j]);
                    s[4 * j + 1] = fmaf(f.y, x[4 * j + 1], s[4 * j + 1]);
                    s[4 * j + 2] = fmaf(f.z, x[4 * j + 2], s[4 * j + 2]);
                    s[4 * j + 3] = fmaf(f.w, x[4 * j + 3], s[4 * j + 3]);
                }
            }
        }
        // ---- masks: a tile that ends past the first query's last token, or has absent tokens ----
        if ((int32_t)((t + 1) * 32) - 1 > lim0 || ld.here != ~0u) {
            const uint32_t on = ld.here >> (4 * h);
            const int32_t left = lim - (int32_t)(t * 32 + 4 * h);  // tokens up to this one
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int c = 8 * (r >> 2) + (r & 3);
                if (c > left || !(on >> c & 1)) s[r] = -INFINITY;
            }
        }
        // ---- softmax ----
        float top = s[0];
#pragma unroll
        for (int r = 1; r < 16; r++) top = fmaxf(top, s[r]);
        top = fmaxf(top, __shfl_xor(top, 32)) * qs;
        if (__builtin_amdgcn_ballot_w64(top > m + GR_MOVE)) {
            const float mn = fmaxf(m, top), al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
            for (int b = 0; b < 4; b++)
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int r = 0; r < 16; r++) o[b][c][r] *= al;
            den *= al;
            m = mn;
        }
        {
            const float ms = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], qs, -ms));
            float d = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; r += 4) d += (s[r] + s[r + 1]) + (s[r + 2] + s[r + 3]);
            den += d;
        }
        // ---- values ----
        if (QS == 4) {
            lds_barrier();  // V is written, K is no longer read
            if (ld.piece < 2) {
                store_k(0);
                ld.issue(t + 2 * TS, t + 3 * TS);
            }
        }
        const int4 e4 = *(const int4 *)L.u.t.ev[ts];
        const uint4 marks = *(const uint4 *)L.u.t.marks[ts];
        const int e[4] = {e4.x, e4.y, e4.z, e4.w};
        if (__builtin_amdgcn_ballot_w64(e[0] != ev[0] || e[1] != ev[1] || e[2] != ev[2] || e[3] != ev[3])) {
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const int d = max(ev[b] - e[b], -200);
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int r = 0; r < 16; r++) o[b][c][r] = ldexpf(o[b][c][r], d);
                const int now = __builtin_amdgcn_readfirstlane(e[b]);
                if (ev[b] == -100) first[b] = now;
                if (now > first[b] + 1) wide = true;
                ev[b] = now;
            }
        }
        // A value block without a finite scale makes its dims no numbers for every query that sees the token, however
        // small its probability, and does not count for the others (its scale is 0).
        const uint32_t mark = __builtin_amdgcn_readfirstlane(marks.x | marks.y | marks.z | marks.w);
        wide |= mark >> 1;
        if (mark & 1) {
            const uint4 bad4 = *(const uint4 *)L.u.t.bad[ts];
            const uint32_t bads[4] = {bad4.x, bad4.y, bad4.z, bad4.w};
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const uint32_t bad = bads[b] >> (4 * h);
                bool any = false;
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int c = 8 * (r >> 2) + (r & 3);
                    any |= (bad >> c & 1) && c <= lim - (int32_t)(t * 32 + 4 * h);
                }
                any |= __shfl_xor((int)any, 32) != 0;
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int r = 0; r < 16; r++) o[b][c][r] = any ? __builtin_nanf("") : o[b][c][r];
            }
        }
        // Into the block's units of a wide range and back: probabilities and sums.
        float down;
        auto into = [&](int b) {
            float z = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float4 f = *(const float4 *)&L.u.t.vs[ts][b][8 * j + 4 * h];
                z = fmaxf(fmaxf(z, fabsf(s[4 * j] * f.x)), fabsf(s[4 * j + 1] * f.y));
                z = fmaxf(fmaxf(z, fabsf(s[4 * j + 2] * f.z)), fabsf(s[4 * j + 3] * f.w));
            }
            const GrUnit u(fmaxf(z, __shfl_xor(z, 32)));
            down = u.down;
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] *= u.up, o[b][0][r] *= u.up, o[b][1][r] *= u.up;
        };
        auto back = [&](int b) {
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] *= down, o[b][0][r] *= down, o[b][1][r] *= down;
        };
        uint32_t vx[2][2];
        float4 fx[2][2];
        auto read_v = [&](int n) {
            const uint32_t b = n >> 1, tq = 4 * (n & 1) + h;
            vx[n & 1][0] = L.u.t.v[ts][b][li][tq], vx[n & 1][1] = L.u.t.v[ts][b][li][tq + 2];
            fx[n & 1][0] = *(const float4 *)&L.u.t.vs[ts][b][4 * tq];
            fx[n & 1][1] = *(const float4 *)&L.u.t.vs[ts][b][4 * tq + 8];
        };
        if (AHEAD) read_v(0);
#pragma unroll
        for (int n = 0; n < 8; n++) {
            const int b = n >> 1, k = n & 1;
            if (k == 0 && wide) {
                if (b) back(b - 1);
                into(b);
            }
            if (n + AHEAD < 8) read_v(n + AHEAD);
            if (AHEAD) __builtin_amdgcn_sched_barrier(0x76);
            rm_h8 vf[2];
            gr_v_operands(vx[k][0], vx[k][1], magic, vf);
            const float4 f0 = fx[k][0], f1 = fx[k][1];
            const float x[8] = {s[8 * k] * f0.x,     s[8 * k + 1] * f0.y, s[8 * k + 2] * f0.z, s[8 * k + 3] * f0.w,
                                s[8 * k + 4] * f1.x, s[8 * k + 5] * f1.y, s[8 * k + 6] * f1.z, s[8 * k + 7] * f1.w};
            rm_h8 hi, lo;
            gr_split(x, minus_one, hi, lo);
#pragma unroll
            for (int c = 0; c < 2; c++) o[b][c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[c], lo, o[b][c], 0, 0, 0);
#pragma unroll
            for (int c = 0; c < 2; c++) o[b][c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[c], hi, o[b][c], 0, 0, 0);
            if (AHEAD) __builtin_amdgcn_sched_barrier(0x76);
        }
        if (wide) back(3);
        lds_wave_order();
    }
    // ---- join the token shares, half of the waves publishing to the other half, and write ----
    den += __shfl_xor(den, 32);
#pragma unroll
    for (int b = 0; b < 4; b++) {
        const float f = ldexpf(1.0f / 15.0f, ev[b] - 9);
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[b][c][r] *= f;
    }
#pragma unroll
    for (int n = TS / 2; n > 0; n >>= 1) {
        __syncthreads();  // the queries (and the last round's sums) are dead
        if ((int)ts >= n && (int)ts < 2 * n) {
            const uint32_t slot = (ts - n) * QS + qsub;
            if (h == 0) {
                L.stat[slot][0][li] = m;
                L.stat[slot][1][li] = den;
            }
#pragma unroll
            for (int b = 0; b < 4; b++)
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        L.u.sum[slot][(b * 2 + c) * 4 + j][lane] =
                            make_float4(o[b][c][4 * j], o[b][c][4 * j + 1], o[b][c][4 * j + 2], o[b][c][4 * j + 3]);
        }
        __syncthreads();
        if ((int)ts < n) {
            const uint32_t slot = ts * QS + qsub;
            const float m2 = L.stat[slot][0][li], mn = fmaxf(m, m2);
            const float f1 = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            const float f2 = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m2 - mn);
            den = den * f1 + L.stat[slot][1][li] * f2;
            m = mn;
#pragma unroll
            for (int b = 0; b < 4; b++)
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float4 x = L.u.sum[slot][(b * 2 + c) * 4 + j][lane];
                        o[b][c][4 * j] = fmaf(x.x, f2, o[b][c][4 * j] * f1);
                        o[b][c][4 * j + 1] = fmaf(x.y, f2, o[b][c][4 * j + 1] * f1);
                        o[b][c][4 * j + 2] = fmaf(x.z, f2, o[b][c][4 * j + 2] * f1);
                        o[b][c][4 * j + 3] = fmaf(x.w, f2, o[b][c][4 * j + 3] * f1);
                    }
        }
    }
    if (ts || !valid) return;
    float *dst, f = 1.0f;
    if (it.ranges > 1) {
        float *slot = (FEW ? a.few_part : a.part) + (size_t)blockIdx.x * (kQueries * 258);
        const uint32_t in = 32 * qsub + li;
        dst = slot + (size_t)in * 256;
        if (h == 0) {
            // (scores that are no numbers move no maximum; the part is not an empty one)
            slot[kQueries * 256 + 2 * in] = den != den && m == -INFINITY ? 0.0f : m;
            slot[kQueries * 256 + 2 * in + 1] = den;
        }
    } else {
        dst = a.out + qat;
        f = den != 0.0f ? 1.0f / den : 0.0f;
    }
#pragma unroll
    for (int b = 0; b < 4; b++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float4 *d = (float4 *)(dst + 64 * b + 16 * j + 8 * h);
            const gr_v16 &x = o[b][0], &y = o[b][1];
            d[0] = make_float4(x[4 * j] * f, y[4 * j] * f, x[4 * j + 1] * f, y[4 * j + 1] * f);
            d[1] = make_float4(x[4 * j + 2] * f, y[4 * j + 2] * f, x[4 * j + 3] * f, y[4 * j + 3] * f);
        }
}
extern "C" __global__ __launch_bounds__(512, 2) void ctox_gqa_rows_gfx950(GqaRowsArgs a) { gqa_rows<4, 2>(a); }
extern "C" __global__ __launch_bounds__(256, 2) void ctox_gqa_few_gfx950(GqaRowsArgs a) { gqa_rows<1, 4>(a); }

// ---------------------------------------------------------------------------
// at most 16 queries a KV head
// ---------------------------------------------------------------------------
// Four waves, each with all queries and every fourth tile, on f16 MFMA 16x16x32: half the products, softmax and splits
// of the 32-query kernel, and sums in 64 registers, so that the queries stay in registers too.
typedef float gr_v4 __attribute__((ext_vector_type(4)));
struct GrLds16 {
    union {
        struct {
            uint2 k[4][4][4][36];   // [wave][block][quarter][token]: that quarter's code bytes
            uint32_t v[4][4][32][9];  // [wave][block][code byte][token / 4]: that byte of four tokens
            float ks[4][4][32];
            float vs[4][4][32];
            int ev[4][4];
            uint32_t bad[4][4], marks[4][4];
        } t;
        float4 sum[2][16][64];  // [publishing wave][dim block, half, parity][lane]
        GrScratch scratch;
    } u;
    float stat[2][2][16];
};

extern "C" __global__ __launch_bounds__(256, 2) void ctox_gqa_few16_gfx950(GqaRowsArgs a) {
    __shared__ GrLds16 L;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t li = lane & 15, g = lane >> 4;
    const uint32_t range = gr_range<256>(a, true, L.u.scratch);
    const GrItem it = gr_find<256>(a, true, range, blockIdx.x, L.u.scratch);
    if (!it.ok) return;
    if (it.local == 0 && threadIdx.x == 0) {
        a.cuts[2 * it.request] = it.base;
        a.cuts[2 * it.request + 1] = it.ranges;
    }
    const GrRequest rq = gr_request(a, it.request);
    const uint32_t nq = rq.rows * a.group, kvh = it.local % a.kv_heads, part = it.local / a.kv_heads;
    const int32_t past = (int32_t)rq.tokens - (int32_t)rq.rows;  // tokens before the first row
    const uint32_t vis = rq.tokens;
    const uint32_t units = (vis + 127) / 128, per = (units + it.ranges - 1) / it.ranges;
    const uint32_t t0 = min(part * per, units) * 4 + wave, t1 = min(part * per + per, units) * 4;
    const bool valid = li < nq;
    const int32_t lim = valid ? past + (int32_t)(li / a.group) : -1;
    const uint32_t qrow = valid ? li / a.group : 0, qg = valid ? li - qrow * a.group : 0;
    const size_t qat = ((size_t)(rq.row0 + qrow) * a.query_heads + kvh * a.group + qg) * 256;

    GrLoad<4> ld{a, it.request, kvh, vis, t1, lane, 0};
    ld.desc_load(t0);
    rm_h8 qf[2][8];  // [lo, hi][k step]: 8 dims of each quarter of a block
    float qs;
    {
        const float *q = a.query + qat + 16 * g;
        const float pre = valid ? a.scale * 1.44269504088896341f : 0.0f;
        auto load = [&](int s, float (&x)[8]) {
            const float4 u = *(const float4 *)(q + 64 * (s >> 1) + 8 * (s & 1));
            const float4 v = *(const float4 *)(q + 64 * (s >> 1) + 8 * (s & 1) + 4);
            const float y[8] = {u.x, v.x, u.y, v.y, u.z, v.z, u.w, v.w};
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = y[i] * pre;
        };
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < 8; s++) {
            float x[8];
            load(s, x);
#pragma unroll
            for (int i = 0; i < 8; i++) mx = fmaxf(mx, fabsf(x[i]) < INFINITY ? fabsf(x[i]) : 0.0f);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const int e = gr_query_exponent(mx);
        qs = ldexpf(1.0f, e - 15);
#pragma unroll
        for (int s = 0; s < 8; s++) {
            float x[8];
            load(s, x);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float v = ldexpf(x[i], 15 - e);
                qf[1][s][i] = (_Float16)v;
                qf[0][s][i] = fabsf(v) < INFINITY ? (_Float16)(v - (float)qf[1][s][i]) : (_Float16)0.0f;
            }
        }
    }
    const RmMagic magic = rm_magic<true>();
    float minus_one = -1.0f;
    asm("" : "+v"(minus_one));
    gr_v4 o[4][2][2];  // [dim block][half of its code bytes][even, odd dims]
#pragma unroll
    for (int b = 0; b < 4; b++)
#pragma unroll
        for (int c = 0; c < 4; c++) o[b][c >> 1][c & 1] = gr_v4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, den = 0.0f;
    int ev[4] = {-100, -100, -100, -100};  // E of the blocks' sums
    int first[4] = {0, 0, 0, 0};           // the first of them
    bool wide = false;                     // value scales that GrUnit is for have been seen

    ld.issue(t0, t0 + 4);
    __builtin_amdgcn_s_waitcnt(0x0F70);
    for (uint32_t t = t0; t < t1; t += 4) {
        // ---- this tile's bytes and scales into LDS; the next tile's loads ----
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t b = ld.block(i);
            ld.widen(i);
            L.u.t.ks[wave][b][ld.token] = ld.key_scale(i);
#pragma unroll
            for (int w = 0; w < 4; w++) L.u.t.k[wave][b][w][ld.token] = make_uint2(ld.raw[i][2 * w], ld.raw[i][2 * w + 1]);
        }
#pragma unroll
        for (int i = 2; i < 4; i++) {
            const uint32_t b = ld.block(i);
            ld.store_v(i, lane, L.u.t.v[wave][b], L.u.t.vs[wave][b], L.u.t.ev[wave][b], L.u.t.bad[wave][b],
                       L.u.t.marks[wave][b]);
        }
        lds_wave_order();
        ld.issue(t + 4, t + 8);
        // ---- scores: tokens 16 n + 4 g + r ----
        gr_v4 s[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int b = 0; b < 4; b++) {
            uint2 kw[2];
            gr_v4 x[2];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                kw[n] = L.u.t.k[wave][b][g][16 * n + li];
                x[n] = gr_v4{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const rm_h8 kf = gr_k_operand(k ? kw[n].y : kw[n].x, magic);
                    x[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[0][2 * b + k], x[n], 0, 0, 0);
                    x[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[1][2 * b + k], x[n], 0, 0, 0);
                }
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const float4 f = *(const float4 *)&L.u.t.ks[wave][b][16 * n + 4 * g];
                s[n][0] = fmaf(f.x, x[n][0], s[n][0]);
                s[n][1] = fmaf(f.y, x[n][1], s[n][1]);
                s[n][2] = fmaf(f.z, x[n][2], s[n][2]);
                s[n][3] = fmaf(f.w, x[n][3], s[n][3]);
            }
        }
        // ---- masks ----
        if ((int32_t)((t + 1) * 32) - 1 > past || ld.here != ~0u) {
            const uint32_t on = ld.here >> (4 * g);
            const int32_t left = lim - (int32_t)(t * 32 + 4 * g);  // tokens up to this one
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int c = 16 * n + r;
                    if (c > left || !(on >> c & 1)) s[n][r] = -INFINITY;
                }
        }
        // ---- softmax ----
        float top = s[0][0];
#pragma unroll
        for (int r = 1; r < 8; r++) top = fmaxf(top, s[r >> 2][r & 3]);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32)) * qs;
        if (__builtin_amdgcn_ballot_w64(top > m + GR_MOVE)) {
            const float mn = fmaxf(m, top), al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
            for (int b = 0; b < 4; b++)
#pragma unroll
                for (int c = 0; c < 4; c++) o[b][c >> 1][c & 1] *= al;
            den *= al;
            m = mn;
        }
        float p[8];
        {
            const float ms = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int r = 0; r < 8; r++) p[r] = __builtin_amdgcn_exp2f(fmaf(s[r >> 2][r & 3], qs, -ms));
            den += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        }
        // ---- values ----
        const int4 e4 = *(const int4 *)L.u.t.ev[wave];
        const uint4 marks = *(const uint4 *)L.u.t.marks[wave];
        const int e[4] = {e4.x, e4.y, e4.z, e4.w};
        if (__builtin_amdgcn_ballot_w64(e[0] != ev[0] || e[1] != ev[1] || e[2] != ev[2] || e[3] != ev[3])) {
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const int d = max(ev[b] - e[b], -200);
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int r = 0; r < 4; r++) o[b][c >> 1][c & 1][r] = ldexpf(o[b][c >> 1][c & 1][r], d);
                const int now = __builtin_amdgcn_readfirstlane(e[b]);
                if (ev[b] == -100) first[b] = now;
                if (now > first[b] + 1) wide = true;
                ev[b] = now;
            }
        }
        // (as above: no numbers for every query that sees the token, nothing for the others)
        const uint32_t mark = __builtin_amdgcn_readfirstlane(marks.x | marks.y | marks.z | marks.w);
        wide |= mark >> 1;
        if (mark & 1) {
            const uint4 bad4 = *(const uint4 *)L.u.t.bad[wave];
            const uint32_t bads[4] = {bad4.x, bad4.y, bad4.z, bad4.w};
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const uint32_t bad = bads[b] >> (4 * g);
                bool any = false;
#pragma unroll
                for (int r = 0; r < 8; r++) {
                    const int c = 16 * (r >> 2) + (r & 3);
                    any |= (bad >> c & 1) && c <= lim - (int32_t)(t * 32 + 4 * g);
                }
                any |= __shfl_xor((int)any, 16) != 0;
                any |= __shfl_xor((int)any, 32) != 0;
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int r = 0; r < 4; r++) o[b][c >> 1][c & 1][r] = any ? __builtin_nanf("") : o[b][c >> 1][c & 1][r];
            }
        }
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const float4 f0 = *(const float4 *)&L.u.t.vs[wave][b][4 * g];
            const float4 f1 = *(const float4 *)&L.u.t.vs[wave][b][16 + 4 * g];
            float x[8] = {p[0] * f0.x, p[1] * f0.y, p[2] * f0.z, p[3] * f0.w,
                          p[4] * f1.x, p[5] * f1.y, p[6] * f1.z, p[7] * f1.w};
            float down = 1.0f;
            if (wide) {
                float z = 0.0f;
#pragma unroll
                for (int r = 0; r < 8; r++) z = fmaxf(z, fabsf(x[r]));
                z = fmaxf(z, __shfl_xor(z, 16));
                const GrUnit u(fmaxf(z, __shfl_xor(z, 32)));
#pragma unroll
                for (int r = 0; r < 8; r++) x[r] *= u.up;
#pragma unroll
                for (int c = 0; c < 4; c++) o[b][c >> 1][c & 1] *= u.up;
                down = u.down;
            }
            rm_h8 hi, lo;
            gr_split(x, minus_one, hi, lo);
#pragma unroll
            for (int c = 0; c < 2; c++) {
                rm_h8 vf[2];
                gr_v_operands(L.u.t.v[wave][b][16 * c + li][g], L.u.t.v[wave][b][16 * c + li][4 + g], magic, vf);
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    o[b][c][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[n], lo, o[b][c][n], 0, 0, 0);
                    o[b][c][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[n], hi, o[b][c][n], 0, 0, 0);
                }
            }
            if (wide)
#pragma unroll
                for (int c = 0; c < 4; c++) o[b][c >> 1][c & 1] *= down;
        }
        lds_wave_order();
    }
    // ---- join the waves, half of them publishing to the other half, and write ----
    den += __shfl_xor(den, 16);
    den += __shfl_xor(den, 32);
#pragma unroll
    for (int b = 0; b < 4; b++) {
        const float f = ldexpf(1.0f / 15.0f, ev[b] - 9);
#pragma unroll
        for (int c = 0; c < 4; c++) o[b][c >> 1][c & 1] *= f;
    }
#pragma unroll
    for (uint32_t n = 2; n > 0; n >>= 1) {
        __syncthreads();  // the tiles (and the last round's sums) are dead
        if (wave >= n && wave < 2 * n) {
            const uint32_t slot = wave - n;
            if (g == 0) {
                L.stat[slot][0][li] = m;
                L.stat[slot][1][li] = den;
            }
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const gr_v4 x = o[i >> 2][i >> 1 & 1][i & 1];
                L.u.sum[slot][i][lane] = make_float4(x[0], x[1], x[2], x[3]);
            }
        }
        __syncthreads();
        if (wave < n) {
            const float m2 = L.stat[wave][0][li], mn = fmaxf(m, m2);
            const float f1 = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            const float f2 = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m2 - mn);
            den = den * f1 + L.stat[wave][1][li] * f2;
            m = mn;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                gr_v4 &y = o[i >> 2][i >> 1 & 1][i & 1];
                const float4 x = L.u.sum[wave][i][lane];
                y = gr_v4{fmaf(x.x, f2, y[0] * f1), fmaf(x.y, f2, y[1] * f1), fmaf(x.z, f2, y[2] * f1),
                          fmaf(x.w, f2, y[3] * f1)};
            }
        }
    }
    if (wave || !valid) return;
    float *dst, f = 1.0f;
    if (it.ranges > 1) {
        float *slot = a.few_part + (size_t)blockIdx.x * (16 * 258);
        dst = slot + (size_t)li * 256;
        if (g == 0) {
            slot[16 * 256 + 2 * li] = den != den && m == -INFINITY ? 0.0f : m;
            slot[16 * 256 + 2 * li + 1] = den;
        }
    } else {
        dst = a.out + qat;
        f = den != 0.0f ? 1.0f / den : 0.0f;
    }
#pragma unroll
    for (int b = 0; b < 4; b++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
            float4 *d = (float4 *)(dst + 64 * b + 32 * c + 8 * g);
            const gr_v4 &x = o[b][c][0], &y = o[b][c][1];
            d[0] = make_float4(x[0] * f, y[0] * f, x[1] * f, y[1] * f);
            d[1] = make_float4(x[2] * f, y[2] * f, x[3] * f, y[3] * f);
        }
}

// ---------------------------------------------------------------------------
// join: grid (rows, quarters of the query heads), 64 lanes x 4 dims
// ---------------------------------------------------------------------------
// A wave takes a head of its own, or, where there are more than GR_ALONE parts, every fourth part of one head after the
// other. (A mixed batch of 36 thousand row heads: 19 us, 38 us with four waves a head throughout.)
#define GR_ALONE 8
extern "C" __global__ __launch_bounds__(256) void ctox_gqa_join_gfx950(GqaRowsArgs a) {
    __shared__ float4 acc4[4][64];
    __shared__ float st[4][2];
    const uint32_t row = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= min(a.row_starts[a.requests], a.rows)) return;
    uint32_t lo = 0, hi = a.requests;  // the request of this row: the last that starts at or before it
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 63) / 64, at = lo + lane * step;
        const uint32_t n = __popcll(__builtin_amdgcn_ballot_w64(at < hi && a.row_starts[min(at, hi - 1)] <= row));
        lo += max(n, 1u) * step - step;
        hi = min(lo + step, hi);
    }
    const GrRequest rq = gr_request(a, lo);
    if (row < rq.row0 || row - rq.row0 >= rq.rows) return;
    const bool few = gr_few(a, rq);
    const uint32_t first = a.cuts[2 * lo], ranges = a.cuts[2 * lo + 1];
    const uint32_t size = few ? a.few : 128, nqt = (rq.rows * a.group + size - 1) / size;
    // (Lengths that break the contract can leave a request without items, and its cut unwritten.)
    if (ranges < 2 || first + (uint64_t)nqt * ranges * a.kv_heads > (few ? a.few_items : a.items)) return;
    const float *base = few ? a.few_part : a.part;
    const bool alone = ranges <= GR_ALONE;
    float m, den;
    float4 acc;
    // Parts s0, s0 + step, ... of a head into (m, den, acc).
    auto sum = [&](uint32_t head, uint32_t s0, uint32_t step) {
        const uint32_t kvh = head / a.group, q = (row - rq.row0) * a.group + head % a.group, in = q % size;
        const uint32_t slot0 = first + (nqt - 1 - q / size) * ranges * a.kv_heads + kvh;
        m = -INFINITY, den = 0.0f;
        acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (; s0 < ranges; s0 += 4 * step) {
            float4 v[4];
            float ms[4], ds[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t s = min(s0 + k * step, ranges - 1);
                const float *p = base + (size_t)(slot0 + s * a.kv_heads) * (size * 258);
                v[k] = ((const float4 *)(p + (size_t)in * 256))[lane];
                ms[k] = s0 + k * step < ranges ? p[size * 256 + 2 * in] : -INFINITY;
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
                acc = make_float4(fmaf(v[k].x, f, acc.x), fmaf(v[k].y, f, acc.y), fmaf(v[k].z, f, acc.z),
                                  fmaf(v[k].w, f, acc.w));
                den = fmaf(ds[k], f, den);
            }
            m = mn;
        }
    };
    auto write = [&](uint32_t head, const float4 &x, float total) {
        const float inv = total != 0.0f ? 1.0f / total : 0.0f;
        ((float4 *)(a.out + ((size_t)row * a.query_heads + head) * 256))[lane] =
            make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
    };
    if (alone) {
        const uint32_t head = 4 * blockIdx.y + wave;
        if (head >= a.query_heads) return;
        sum(head, 0, 1);
        write(head, acc, den);
        return;
    }
    for (uint32_t head = 4 * blockIdx.y; head < min(4 * blockIdx.y + 4, a.query_heads); head++) {
        sum(head, wave, 4);
        acc4[wave][lane] = acc;
        if (lane == 0) {
            st[wave][0] = m;
            st[wave][1] = den;
        }
        __syncthreads();
        if (wave == 0) {
            const float mn = fmaxf(fmaxf(st[0][0], st[1][0]), fmaxf(st[2][0], st[3][0]));
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
            write(head, out, total);
        }
        __syncthreads();
    }
}
