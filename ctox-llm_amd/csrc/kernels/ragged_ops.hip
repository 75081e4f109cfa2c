// A ragged batch's new tokens in front of its attention, gfx950.
//
//  * ctox_rope_axes_gfx950 / _any: y = rope(norm(x)) per (row, head). norm is the (1 + w)
//    RMS norm of Q/src/reference.rs:38-62 (optional); pair i of (x[i], x[i + rd/2]) turns by
//    positions[t][axis[i]] * theta^(-2i/rd) (Q/src/reference.rs:115-155 is the one-axis case).
//    Bound by HBM bytes. The angle is formed in turns in 64 bits (position * frequency, less
//    its nearest integer), where 32 would leave an error of position * 2^-24 turns; only the
//    remainder, at most half a turn, goes to the 32-bit sine and cosine. A workgroup makes one
//    row's table once and its four waves take the heads in turn, one head a wave. 4096 rows of
//    28 heads of 256, three axes: 69 us, 3.4 TB/s (51 us where the same rows come from the Infinity
//    Cache); 16 rows: 7 us, the launch.
//  * ctox_paged_plan_gfx950: page descriptors, slot map and row offsets of a batch from the
//    requests' cached and added lengths (PagedKvCache::push's page bookkeeping,
//    Q/src/kv_cache.rs:394-429, for many requests at once). One launch: every workgroup makes
//    both prefix sums (rows, pages) in LDS for itself, then writes its share of the rows and
//    pages; nothing passes between workgroups. 8 requests 6.8 us, 512 requests 8.6 us.
//  * ctox_kv_append_q4_gfx950: token rows of K and V into the Q4 slots of the slot map,
//    bit-exact with Q4Block64::quantize (Q/src/quant.rs:144-168). Eight lanes hold a 64-value
//    block; a token's bytes are assembled in LDS and leave as whole dwords. 32 rows of 2 x 1024
//    values 4.9 us, 4096 rows 12 us (3.1 TB/s read and written).
#include <hip/hip_runtime.h>

#include "kernel_args.h"
#include "lds_barrier.h"

// ---------------------------------------------------------------------------
// rotary positions on several axes
// ---------------------------------------------------------------------------
struct RoHead {
    const float *x;
    float *y;
    const float *w;
};

__device__ __forceinline__ RoHead ro_head(const RopeAxesArgs &a, uint32_t t, uint32_t head) {
    const uint32_t s = head < a.heads[0] ? 0u : 1u, h = head - (s ? a.heads[0] : 0u);
    return {a.in[s] + (size_t)t * a.in_row[s] + (size_t)h * a.in_head[s],
            a.out[s] + (size_t)t * a.out_row[s] + (size_t)h * a.out_head[s], a.norm[s]};
}

// cos and sin of the row's pairs into LDS.
__device__ __forceinline__ void ro_table(const RopeAxesArgs &a, uint32_t t, float *cs, float *sn) {
    for (uint32_t i = threadIdx.x; i < a.rd / 2; i += 256) {
        const double turn = (double)a.positions[(size_t)t * a.axes + a.axis[i]] * a.turns[i];
        float s, c;
        sincospif(2.0f * (float)(turn - rint(turn)), &s, &c);
        cs[i] = c;
        sn[i] = s;
    }
    lds_barrier();
}

__device__ __forceinline__ float ro_wave_sum(float s) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    return s;
}

// grid (rows, head groups). head_dim <= 256 in 16-byte units, the half rotation in whole
// units: a lane holds four values, its pairs' partners are rd/8 lanes away.
extern "C" __global__ __launch_bounds__(256) void ctox_rope_axes_gfx950(RopeAxesArgs a) {
    __shared__ __attribute__((aligned(16))) float cs[128], sn[128];
    const uint32_t t = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (a.row_count && t >= *a.row_count) return;
    const uint32_t h0 = blockIdx.y * a.heads_per_wg, h1 = min(h0 + a.heads_per_wg, a.heads[0] + a.heads[1]);
    const uint32_t c = 4 * lane, half = a.rd / 2;
    const bool mine = c < a.hd;
    ro_table(a, t, cs, sn);
    const bool first = c < half, second = !first && c < a.rd;
    const uint32_t at = first ? c : second ? c - half : 0;
    const float4 cv = *(const float4 *)&cs[at], sv = *(const float4 *)&sn[at];
    const int partner = (int)(first ? lane + half / 4 : second ? lane - half / 4 : lane);
    for (uint32_t head = h0 + wave; head < h1; head += 4) {
        const RoHead r = ro_head(a, t, head);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (mine) v = *(const float4 *)(r.x + c);
        if (r.w) {
            const float sum = ro_wave_sum((v.x * v.x + v.y * v.y) + (v.z * v.z + v.w * v.w));
            const float inv = 1.0f / sqrtf(sum / (float)a.hd + a.eps);
            if (mine) {
                const float4 w = *(const float4 *)(r.w + c);
                v = make_float4(v.x * inv * (1.0f + w.x), v.y * inv * (1.0f + w.y), v.z * inv * (1.0f + w.z),
                                v.w * inv * (1.0f + w.w));
            }
        }
        const float4 o = make_float4(__shfl(v.x, partner), __shfl(v.y, partner), __shfl(v.z, partner),
                                     __shfl(v.w, partner));
        if (first || second) {
            const float g = first ? -1.0f : 1.0f;
            v = make_float4(v.x * cv.x + g * o.x * sv.x, v.y * cv.y + g * o.y * sv.y, v.z * cv.z + g * o.z * sv.z,
                            v.w * cv.w + g * o.w * sv.w);
        }
        if (mine) *(float4 *)(r.y + c) = v;
    }
}

// The same for any head_dim <= 1024, alignment and even rotary dimension: a wave keeps its
// head in LDS. A head is read whole before any of it is written, so it may be in place.
extern "C" __global__ __launch_bounds__(256) void ctox_rope_axes_any_gfx950(RopeAxesArgs a) {
    __shared__ float cs[CTOX_ROPE_MAX_PAIRS], sn[CTOX_ROPE_MAX_PAIRS], buf[4][1024];
    const uint32_t t = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (a.row_count && t >= *a.row_count) return;
    const uint32_t h0 = blockIdx.y * a.heads_per_wg, h1 = min(h0 + a.heads_per_wg, a.heads[0] + a.heads[1]);
    const uint32_t half = a.rd / 2;
    float *x = buf[wave];
    ro_table(a, t, cs, sn);
    for (uint32_t head = h0 + wave; head < h1; head += 4) {
        const RoHead r = ro_head(a, t, head);
        float sum = 0.0f;
        for (uint32_t d = lane; d < a.hd; d += 64) {
            const float v = r.x[d];
            x[d] = v;
            sum += v * v;
        }
        float inv = 1.0f;
        if (r.w) inv = 1.0f / sqrtf(ro_wave_sum(sum) / (float)a.hd + a.eps);
        lds_wave_order();
        auto value = [&](uint32_t d) { return r.w ? x[d] * inv * (1.0f + r.w[d]) : x[d]; };
        for (uint32_t d = lane; d < a.hd; d += 64) {
            float y;
            if (d < half)
                y = value(d) * cs[d] - value(d + half) * sn[d];
            else if (d < a.rd)
                y = value(d) * cs[d - half] + value(d - half) * sn[d - half];
            else
                y = value(d);
            r.y[d] = y;
        }
        lds_wave_order();
    }
}

// ---------------------------------------------------------------------------
// page descriptors and the slot map
// ---------------------------------------------------------------------------
struct PlSum {
    uint64_t rows, pages;
};

// Largest r with prefix[r] <= i, over prefix[0 .. n) (prefix[0] = 0, not falling).
__device__ __forceinline__ uint32_t pl_find(const uint32_t *prefix, uint32_t n, uint32_t i) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (prefix[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

// status: {code, Q4 slots taken, rows, pages of all requests}. Codes: 0 done; 1 a request
// exceeds max_pages; 2 more rows than max_rows; 3 too few free slots; 4 a page to be filled
// up is not a Q4 page of its request; 5 a free slot past q4_slots.
extern "C" __global__ __launch_bounds__(CTOX_PLAN_THREADS) void ctox_paged_plan_gfx950(PagedPlanArgs a) {
    __shared__ uint32_t row_at[CTOX_PLAN_REQUESTS + 1], page_at[CTOX_PLAN_REQUESTS + 1];
    __shared__ uint64_t wave_rows[CTOX_PLAN_THREADS / 64], wave_pages[CTOX_PLAN_THREADS / 64];
    __shared__ uint32_t bad[6], all_pages;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t per = (a.requests + CTOX_PLAN_THREADS - 1) / CTOX_PLAN_THREADS;
    const uint32_t r0 = min(tid * per, a.requests), r1 = min(r0 + per, a.requests);
    const uint64_t room = (uint64_t)a.max_pages * a.page_tokens;
    if (tid < 6) bad[tid] = 0;
    if (tid == 0) all_pages = 0;
    __syncthreads();
    // Prefix sums in 64 bits: a thread's own requests, the wave's, the workgroup's.
    PlSum sum{0, 0};
    uint32_t held_all = 0;
    for (uint32_t r = r0; r < r1; r++) {
        const uint64_t cached = a.cached[r], total = cached + a.added[r];
        if (total > room) {
            bad[1] = 1;
            continue;
        }
        const uint32_t held = (uint32_t)((cached + a.page_tokens - 1) / a.page_tokens);
        const uint32_t pages = (uint32_t)((total + a.page_tokens - 1) / a.page_tokens);
        sum.rows += total - cached;
        sum.pages += pages - held;
        held_all += pages;
        if (total > cached && cached % a.page_tokens) {  // its last page is filled up
            const PagedKvDesc d = a.desc[(size_t)r * a.max_pages + held - 1];
            if (d.precision == 0 || d.first_token != (held - 1) * a.page_tokens || d.physical_slot >= a.q4_slots)
                bad[4] = 1;
        }
    }
    atomicAdd(&all_pages, held_all);  // whole numbers: their order does not matter
    PlSum in = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t x = __shfl_up(in.rows, o), y = __shfl_up(in.pages, o);
        if ((int)lane >= o) {
            in.rows += x;
            in.pages += y;
        }
    }
    if (lane == 63) {
        wave_rows[wave] = in.rows;
        wave_pages[wave] = in.pages;
    }
    __syncthreads();
    uint64_t rows = 0, taken = 0;  // the batch's
    PlSum at{in.rows - sum.rows, in.pages - sum.pages};
    for (uint32_t w = 0; w < CTOX_PLAN_THREADS / 64; w++) {
        if (w == wave) {
            at.rows += rows;
            at.pages += taken;
        }
        rows += wave_rows[w];
        taken += wave_pages[w];
    }
    if (tid == 0) {
        if (rows > a.max_rows) bad[2] = 1;
        if (taken > a.free_count) bad[3] = 1;
    }
    for (uint64_t i = tid; i < min(taken, (uint64_t)a.free_count); i += CTOX_PLAN_THREADS)
        if (a.free_slots[i] >= a.q4_slots) bad[5] = 1;
    // (sums past 32 bits only where the batch is refused)
    for (uint32_t r = r0; r < r1; r++) {
        row_at[r] = (uint32_t)at.rows;
        page_at[r] = (uint32_t)at.pages;
        const uint64_t cached = a.cached[r], total = cached + a.added[r];
        if (total > room) continue;
        at.rows += total - cached;
        at.pages += (total + a.page_tokens - 1) / a.page_tokens - (cached + a.page_tokens - 1) / a.page_tokens;
    }
    __syncthreads();
    uint32_t code = 0;
#pragma unroll
    for (int k = 5; k > 0; k--)
        if (bad[k]) code = k;
    const uint32_t step = gridDim.x * CTOX_PLAN_THREADS, me = blockIdx.x * CTOX_PLAN_THREADS + tid;
    const uint32_t n = code ? 0 : (uint32_t)rows, pages = code ? 0 : (uint32_t)taken;
    for (uint32_t r = me; r < a.requests; r += step) {
        const uint32_t cached = a.cached[r], added = code ? 0 : a.added[r], total = cached + added;
        a.row_starts[r] = code ? 0 : row_at[r];
        a.tokens[r] = total;
        a.page_counts[r] = total / a.page_tokens + (total % a.page_tokens != 0);
        if (added && cached % a.page_tokens) {
            const uint32_t p = cached / a.page_tokens;
            a.desc[(size_t)r * a.max_pages + p].tokens = min(a.page_tokens, total - p * a.page_tokens);
        }
    }
    if (me == 0) {
        a.row_starts[a.requests] = n;
        a.status[0] = code;
        a.status[1] = pages;
        a.status[2] = n;
        a.status[3] = code ? 0 : all_pages;
    }
    for (uint32_t i = me; i < pages; i += step) {
        const uint32_t r = pl_find(page_at, a.requests, i), cached = a.cached[r], total = cached + a.added[r];
        const uint32_t p = cached / a.page_tokens + (cached % a.page_tokens != 0) + (i - page_at[r]);
        const uint32_t first = p * a.page_tokens;
        const PagedKvDesc d{1, a.free_slots[i], min(a.page_tokens, total - first), first};
        a.desc[(size_t)r * a.max_pages + p] = d;
    }
    for (uint32_t i = me; i < a.max_rows; i += step) {
        if (i >= n) {
            a.slots[i] = CTOX_NO_SLOT;
            continue;
        }
        const uint32_t r = pl_find(row_at, a.requests, i), cached = a.cached[r], pos = cached + (i - row_at[r]);
        const uint32_t held = cached / a.page_tokens + (cached % a.page_tokens != 0);
        const uint32_t p = pos / a.page_tokens;
        // A page that was there keeps its slot (no workgroup writes that word), a new one has
        // the free slot that its descriptor gets.
        const uint32_t slot = p < held ? a.desc[(size_t)r * a.max_pages + p].physical_slot
                                       : a.free_slots[page_at[r] + (p - held)];
        a.positions[i] = pos;
        a.slots[i] = slot * a.page_tokens + pos % a.page_tokens;
    }
}

// ---------------------------------------------------------------------------
// append through the slot map
// ---------------------------------------------------------------------------
#pragma clang fp contract(off)
// Code of one value of a block with maximum m > 0 (two roundings, as the crate's f32 steps).
__device__ __forceinline__ uint32_t ap_code(float v, float m) {
    float n = v / m;
    n = fminf(1.0f, fmaxf(-1.0f, n));
    const float sel = n * 7.5f + 7.5f;
    return (uint32_t)fminf(15.0f, fmaxf(0.0f, roundf(sel)));
}
#pragma clang fp contract(fast)

// A workgroup takes rows_per_wg rows, or one row in pieces of 2048 values; a thread holds
// eight values. 2048 values are 32 blocks of 34 bytes.
extern "C" __global__ __launch_bounds__(256) void ctox_kv_append_q4_gfx950(KvAppendArgs a) {
    __shared__ uint32_t bytes[272];
    const uint32_t tid = threadIdx.x, cv = a.component_values, octets = cv / 4;  // eights in a row's K and V
    const uint32_t row_dwords = cv / 64 * 17;
    uint8_t *lds = (uint8_t *)bytes;
    for (uint32_t o0 = 0; o0 < octets; o0 += 256) {
        const uint32_t local = a.rows_per_wg > 1 ? tid / octets : 0;
        const uint32_t o = a.rows_per_wg > 1 ? tid - local * octets : o0 + tid;
        const uint32_t t = blockIdx.x * a.rows_per_wg + local;
        const bool live = local < a.rows_per_wg && o < octets && t < a.rows;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = 0.0f;
        if (live) {
            const uint32_t e = 8 * o;
            const float *src = e < cv ? a.keys + (size_t)t * a.key_stride + e : a.values + (size_t)t * a.value_stride + (e - cv);
            if (a.vec) {
                const float4 x = ((const float4 *)src)[0], y = ((const float4 *)src)[1];
                v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = src[k];
            }
        }
        float m = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) m = fmaxf(m, fabsf(v[k]));
#pragma unroll
        for (int s = 4; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor(m, s));
        uint32_t codes = 0;
        if (m != 0.0f) {
#pragma unroll
            for (int k = 0; k < 8; k++) codes |= ap_code(v[k], m) << (4 * k);
        }
        // Block b of the piece at 34 b: two scale bytes, then eight dwords of codes.
        if (local < a.rows_per_wg) {
            const uint32_t blk = tid >> 3, j = tid & 7;
            uint16_t *dst = (uint16_t *)(lds + 34 * blk + 2 + 4 * j);
            dst[0] = (uint16_t)codes;
            dst[1] = (uint16_t)(codes >> 16);
            if (j == 0) *(uint16_t *)(lds + 34 * blk) = __builtin_bit_cast(uint16_t, (_Float16)m);
        }
        lds_barrier();
        for (uint32_t w = tid; w < 272; w += 256) {
            const uint32_t l = a.rows_per_wg > 1 ? w / row_dwords : 0;
            const uint32_t rest = a.rows_per_wg > 1 ? w - l * row_dwords : o0 / 256 * 272 + w;
            const uint32_t row = blockIdx.x * a.rows_per_wg + l;
            if (l >= a.rows_per_wg || rest >= row_dwords || row >= a.rows) continue;
            const uint32_t slot = a.slots[row];
            if (slot >= a.slot_limit) continue;
            uint8_t *tok = a.q4_pages + (size_t)(slot / a.page_tokens) * a.q4_page_bytes +
                           (size_t)(slot % a.page_tokens) * (4 * (size_t)row_dwords);
            ((uint32_t *)tok)[rest] = bytes[w];
        }
        lds_barrier();
    }
}
