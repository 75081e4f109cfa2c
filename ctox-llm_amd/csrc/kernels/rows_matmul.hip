// Packed Q2 / Q4 matrix products for any number of activation rows, gfx950:
// y = act((x * s_in . W^T + bias) * s_out) + residual, the fused matvec of
// Q/src/backend/mod.rs:115-128 for a prompt's rows.
//
// Mathematics. A weight is s (2c - L) / L with the block's f16 scale s and a
// code c (L = 15 or 3). 2c - L is an odd whole number of magnitude <= 15: exact
// in f16, so the product of one 64-column block runs on f16 MFMA 32x32x16 and
// only its f32 sum is scaled: acc += s * (x . (2c - L)), one f32 multiply-add
// per output and block. An f32 activation enters as two f16 parts hi + lo of
// x 2^-e (e from its row's largest magnitude; 22 bits kept for every value
// within 2^-17 of the row's largest, an absolute 2^-40 of it below that), an
// f16 activation without s_in as itself. Sums are f32 throughout.
//
//  * ctox_rows_max_*: a row's exponent e.
//  * ctox_rows_stage_*: x into MFMA operand order, [32-row tile][block]
//    [part][k step][lane][8 f16]: a fragment is 1 KiB that one wave reads at once.
//  * ctox_rows_q{2,4}_*: the product. A workgroup's four waves share TT 32-row
//    tiles of x in LDS (two buffers, loaded straight from memory while the other is
//    in use) and take RT 32-row weight tiles each; weights come from the
//    tiled copy (kernel_args.h) into registers, one block ahead, and are unpacked
//    there once for all TT tiles.
//    Measured, from card to card: 4096 rows, 5120 x 17408 Q2, f32 (two parts) 1.55-1.64 ms with 0.2 ms of it staging:
//    890-944 TFLOP/s of f16 products, against 1108 of the card's large product; 777 rows, 17408 x 5120 Q4 321-327 us;
//    2048 rows, 5120 x 6144 Q4, f16 194-201 us (641-664 TFLOP/s); 16 rows, 14336 x 5120 Q4 24-25 us (1.6 TB/s).
//  * ctox_rows_reduce_gfx950: adds the partial sums of a split K in order and
//    applies the epilogue.
#include <hip/hip_runtime.h>

#include "kernel_args.h"
#include "lds_barrier.h"

typedef float rm_v16 __attribute__((ext_vector_type(16)));
typedef _Float16 rm_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 rm_h2 __attribute__((ext_vector_type(2)));
typedef uint32_t rm_u4 __attribute__((ext_vector_type(4)));

// Eight values of row t from column k on (four and four `gap` columns apart), times s_in. VEC: rows,
// strides and s_in allow 16-byte (f16: 8-byte) loads.
template <bool VEC>
__device__ __forceinline__ void rm_eight(const RowsStageArgs &a, uint32_t t, uint32_t k, uint32_t gap, float (&v)[8]) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    const size_t at = (size_t)t * a.x_stride + k;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const size_t p = at + i * gap;
        if constexpr (VEC) {
            if (a.x_half) {
                const h4 x = *(const h4 *)((const _Float16 *)a.x + p);
#pragma unroll
                for (int j = 0; j < 4; j++) v[4 * i + j] = (float)x[j];
            } else {
                const float4 x = *(const float4 *)((const float *)a.x + p);
                v[4 * i] = x.x, v[4 * i + 1] = x.y, v[4 * i + 2] = x.z, v[4 * i + 3] = x.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                v[4 * i + j] = a.x_half ? (float)((const _Float16 *)a.x)[p + j] : ((const float *)a.x)[p + j];
        }
        const uint32_t c = k + i * gap;
        if (a.s_in_kind == CTOX_KSCALE_F16) {
            const h4 s = *(const h4 *)((const _Float16 *)a.s_in + c);
#pragma unroll
            for (int j = 0; j < 4; j++) v[4 * i + j] *= (float)s[j];
        } else if (a.s_in_kind == CTOX_KSCALE_F32) {
            const float4 s = *(const float4 *)((const float *)a.s_in + c);
            v[4 * i] *= s.x, v[4 * i + 1] *= s.y, v[4 * i + 2] *= s.z, v[4 * i + 3] *= s.w;
        }
    }
}

// Exponent e with |x s_in| < 2^e over row t's finite values (0 for a row of zeros), to all threads.
template <bool VEC, int NT>
__device__ __forceinline__ int rm_exponent(const RowsStageArgs &a, uint32_t t, float *red) {
    float m = 0.0f;
#pragma unroll 4
    for (uint32_t k = 8 * threadIdx.x; k < a.columns; k += 8 * NT) {
        float v[8];
        rm_eight<VEC>(a, t, k, 4, v);
#pragma unroll
        for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(v[i]) < INFINITY ? fabsf(v[i]) : 0.0f);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    lds_barrier();
    m = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; w++) m = fmaxf(m, red[w]);
    int e = 0;
    frexpf(m, &e);
    return e;
}

// First column and gap of the eight values of fragment (k step s, lane half h), in the order in which the
// codes of a lane's words unpack (rm_unpack): value i is column first + i / 2 + gap * (i % 2).
__device__ __forceinline__ uint32_t rm_first(bool q4, uint32_t h, uint32_t s) {
    return q4 ? 32 * h + 8 * s : 32 * h + 16 * (s >> 1) + 4 * (s & 1);
}

// The fragment piece (block b, k step s, lane half h) of row t, its parts 4 KiB apart.
template <bool VEC>
__device__ __forceinline__ void rm_piece(const RowsStageArgs &a, uint32_t t, uint32_t b, uint32_t s, uint32_t h, int e) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = 0.0f;
    if (t < a.rows) rm_eight<VEC>(a, t, 64 * b + rm_first(a.q4, h, s), a.q4 ? 4 : 8, v);
    rm_h8 hi, lo;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float x = v[(i >> 1) + 4 * (i & 1)];
        if (a.parts == 2) x = ldexpf(x, 15 - e);
        hi[i] = (_Float16)x;
        lo[i] = fabsf(x) < INFINITY ? (_Float16)(x - (float)hi[i]) : (_Float16)0.0f;
    }
    rm_h8 *dst = (rm_h8 *)a.staged + ((size_t)(t >> 5) * a.blocks + b) * a.parts * 256 + 64 * s + 32 * h + (t & 31);
    dst[0] = hi;
    if (a.parts == 2) dst[256] = lo;
}

// grid (rows): the rows' exponents.
template <bool VEC>
__device__ __forceinline__ void rows_max(const RowsStageArgs &a) {
    __shared__ float red[4];
    const int e = rm_exponent<VEC, 256>(a, blockIdx.x, red);
    if (threadIdx.x == 0) a.exps[blockIdx.x] = e;
}
extern "C" __global__ __launch_bounds__(256) void ctox_rows_max_vec_gfx950(RowsStageArgs a) { rows_max<true>(a); }
extern "C" __global__ __launch_bounds__(256) void ctox_rows_max_gfx950(RowsStageArgs a) { rows_max<false>(a); }

// grid (blocks, 32-row tiles), one wave per k step: fragments leave as whole KiB.
template <bool VEC>
__device__ __forceinline__ void rows_stage(const RowsStageArgs &a) {
    const uint32_t lane = threadIdx.x & 63, t = blockIdx.y * 32 + (lane & 31);
    rm_piece<VEC>(a, t, blockIdx.x, threadIdx.x >> 6, lane >> 5, a.parts == 2 && t < a.rows ? a.exps[t] : 0);
}
extern "C" __global__ __launch_bounds__(256) void ctox_rows_stage_vec_gfx950(RowsStageArgs a) { rows_stage<true>(a); }
extern "C" __global__ __launch_bounds__(256) void ctox_rows_stage_gfx950(RowsStageArgs a) { rows_stage<false>(a); }

// grid (rows of whole tiles): exponent and pieces of one row in one launch, for few rows (its 16-byte
// pieces of many rows would reach memory as parts of lines).
template <bool VEC>
__device__ __forceinline__ void rows_stage_few(const RowsStageArgs &a) {
    __shared__ float red[8];
    const uint32_t t = blockIdx.x;
    int e = 0;
    if (a.parts == 2 && t < a.rows) {
        e = rm_exponent<VEC, 512>(a, t, red);
        if (threadIdx.x == 0) a.exps[t] = e;
    }
    for (uint32_t p = threadIdx.x; p < 8 * a.blocks; p += 512) rm_piece<VEC>(a, t, p >> 3, (p >> 1) & 3, p & 1, e);
}
extern "C" __global__ __launch_bounds__(512) void ctox_rows_stage_few_vec_gfx950(RowsStageArgs a) { rows_stage_few<true>(a); }
extern "C" __global__ __launch_bounds__(512) void ctox_rows_stage_few_gfx950(RowsStageArgs a) { rows_stage_few<false>(a); }

// ---------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------
__device__ __forceinline__ rm_h2 rm_h(uint32_t x) { return __builtin_bit_cast(rm_h2, x); }

// Eight codes of a lane (k step s) as odd whole numbers. An f16 with the bits 0x6400 | c << p is
// 1024 + c 2^p; one packed multiply-add makes it 2c - L exactly where 2^(11-p) + L is an f16, so
// p is never 0. The constants are opaque so that they stay in registers and mask and magic go into
// one v_and_or_b32.
struct RmMagic {
    uint32_t magic, m[3];
    __device__ __forceinline__ explicit RmMagic(uint32_t m0, uint32_t m1 = 0, uint32_t m2 = 0)
        : magic(0x64006400u), m{m0, m1, m2} {
        asm("" : "+v"(magic));
        asm("" : "+s"(m[0]));
        asm("" : "+s"(m[1]));
        asm("" : "+s"(m[2]));
    }
};
template <int P, int L>
__device__ __forceinline__ rm_h2 rm_pair(uint32_t x, uint32_t mask, uint32_t magic) {
    constexpr _Float16 f = (_Float16)(2.0f / (1 << P)), g = (_Float16)-(2048.0f / (1 << P) + L);
    return __builtin_elementwise_fma(rm_h((x & mask) | magic), rm_h2{f, f}, rm_h2{g, g});
}

template <bool Q4>
__device__ __forceinline__ RmMagic rm_magic() {
    return Q4 ? RmMagic(0x00F000F0u) : RmMagic(0x000C000Cu, 0x00300030u, 0x00C000C0u);
}

template <bool Q4>
__device__ __forceinline__ rm_h8 rm_unpack(const uint32_t (&w)[4], int s, const RmMagic &g) {
    rm_h2 o[4];
    if constexpr (Q4) {
        const uint32_t x = w[s];
        o[0] = rm_pair<4, 15>(x << 4, g.m[0], g.magic);
        o[1] = rm_pair<4, 15>(x, g.m[0], g.magic);
        o[2] = rm_pair<4, 15>(x >> 4, g.m[0], g.magic);
        o[3] = rm_pair<4, 15>(x >> 8, g.m[0], g.magic);
    } else {
        const uint32_t x = s & 1 ? w[s >> 1] >> 8 : w[s >> 1];
        o[0] = rm_pair<2, 3>(s & 1 ? w[s >> 1] >> 6 : w[s >> 1] << 2, g.m[0], g.magic);
        o[1] = rm_pair<2, 3>(x, g.m[0], g.magic);
        o[2] = rm_pair<4, 3>(x, g.m[1], g.magic);
        o[3] = rm_pair<6, 3>(x, g.m[2], g.magic);
    }
    return rm_h8{o[0][0], o[0][1], o[1][0], o[1][1], o[2][0], o[2][1], o[3][0], o[3][1]};
}

typedef __attribute__((address_space(3))) void *rm_lds;
typedef const __attribute__((address_space(1))) void *rm_global;

// bias and s_out of one weight row.
struct RmColumn {
    float bias, scale;
};
__device__ __forceinline__ RmColumn rm_column_scales(const RowsMulArgs &a, uint32_t n) {
    RmColumn c{0.0f, 1.0f};
    if (a.bias) c.bias = a.bias[n];
    if (a.s_out_kind == CTOX_KSCALE_F32) c.scale = ((const float *)a.s_out)[n];
    else if (a.s_out_kind == CTOX_KSCALE_F16) c.scale = (float)((const _Float16 *)a.s_out)[n];
    return c;
}

// v carries the row's exponent and 1 / L already.
__device__ __forceinline__ float rm_finish(const RowsMulArgs &a, float v, const RmColumn &c, uint32_t t, uint32_t n) {
    v = (v + c.bias) * c.scale;
    if (a.activation) v = v / (1.0f + expf(-v));
    if (a.residual) {
        const size_t at = (size_t)t * a.residual_stride + n;
        v += a.y_half ? (float)((const _Float16 *)a.residual)[at] : ((const float *)a.residual)[at];
    }
    return v;
}

__device__ __forceinline__ void rm_store(const RowsMulArgs &a, float v, uint32_t t, uint32_t n) {
    const size_t at = (size_t)t * a.y_stride + n;
    if (a.y_half) ((_Float16 *)a.y)[at] = (_Float16)v;
    else ((float *)a.y)[at] = v;
}

// Every wave's loads into LDS have landed, and every wave is done with the other buffer. A
// barrier does not wait for loads that go straight to LDS, so the wave waits for its own first
// (vmcnt 0, the other counters at their most).
__device__ __forceinline__ void rm_arrive() {
    __builtin_amdgcn_s_waitcnt(0x0F70);
    lds_barrier();
}

template <bool Q4, int PARTS, int TT, int RT>
__device__ __forceinline__ void rows_product(const RowsMulArgs &a) {
    constexpr uint32_t kFrag = 1024, kTile = PARTS * 4 * kFrag;  // bytes of a fragment, of a tile's block
    __shared__ __attribute__((aligned(16))) uint8_t xs[2][TT * kTile];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wg = blockIdx.x, col = wg % a.col_groups, rowg = wg / a.col_groups;
    const uint32_t split = blockIdx.y;
    const uint32_t b0 = split * a.blocks_per_split, b1 = min(b0 + a.blocks_per_split, a.blocks);
    const uint32_t tile0 = rowg * TT;                     // first 32-row tile of x
    const uint32_t n0 = (col * 4 + wave) * RT * 32;       // first weight row of the wave
    const uint32_t h = lane >> 5, j = lane & 15;
    constexpr uint32_t kUnit = Q4 ? 8704 : 4608, kCodes = Q4 ? 8192 : 4096;
    const RmMagic magic = rm_magic<Q4>();

    // This lane's weight tile (16 rows) of each RT tile; tiles past the matrix read the last one.
    const uint8_t *wp[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) {
        const uint32_t t16 = min((n0 + 32 * r) / 16 + ((lane >> 4) & 1), a.tiles - 1);
        wp[r] = a.weights + (size_t)t16 * kUnit;
    }
    uint32_t code[2][RT][4], scale[2][RT];
    auto load_w = [&](uint32_t b, uint32_t (&c)[RT][4], uint32_t (&s)[RT]) {
        const uint32_t chunk = b >> 4, G = (b >> 2) & 3, g = b & 3;
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const uint8_t *u = wp[r] + (size_t)chunk * a.tiles * kUnit;
            const uint32_t l = 16 * g + j;
            if constexpr (Q4) {
                const rm_u4 v = *(const rm_u4 *)(u + G * 2048 + h * 1024 + l * 16);
                c[r][0] = v[0], c[r][1] = v[1], c[r][2] = v[2], c[r][3] = v[3];
            } else {
                const uint2 v = *(const uint2 *)(u + G * 1024 + l * 16 + h * 8);
                c[r][0] = v.x, c[r][1] = v.y;
            }
            s[r] = *(const uint16_t *)(u + kCodes + l * 8 + 2 * G);
        }
    };
    // The workgroup's x tiles of block b: TT * PARTS * 4 fragments, a quarter to each wave.
    auto load_x = [&](uint32_t b, uint32_t buf) {
#pragma unroll
        for (uint32_t i = 0; i < TT * PARTS; i++) {
            const uint32_t f = wave * TT * PARTS + i, tt = f / (PARTS * 4), in = f % (PARTS * 4);
            const uint32_t tile = min(tile0 + tt, a.x_tiles - 1);
            const uint8_t *src = a.staged + ((size_t)tile * a.blocks + b) * kTile + in * kFrag + lane * 16;
            __builtin_amdgcn_global_load_lds((rm_global)src, (rm_lds)&xs[buf][f * kFrag], 16, 0, 0);
        }
    };
    rm_v16 acc[TT][RT];
#pragma unroll
    for (int t = 0; t < TT; t++)
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[t][r][i] = 0.0f;

    auto block = [&](const uint32_t (&c)[RT][4], const uint32_t (&s)[RT], uint32_t buf) {
        rm_h8 w[RT][4];
        float sc[RT];
#pragma unroll
        for (int r = 0; r < RT; r++) {
            sc[r] = (float)__builtin_bit_cast(_Float16, (uint16_t)s[r]);
#pragma unroll
            for (int k = 0; k < 4; k++) w[r][k] = rm_unpack<Q4>(c[r], k, magic);
        }
#pragma unroll
        for (int t = 0; t < TT; t++) {
            rm_v16 p[RT];
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int i = 0; i < 16; i++) p[r][i] = 0.0f;
#pragma unroll
            for (int q = PARTS - 1; q >= 0; q--)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const rm_h8 x = *(const rm_h8 *)&xs[buf][t * kTile + (q * 4 + k) * kFrag + lane * 16];
#pragma unroll
                    for (int r = 0; r < RT; r++) p[r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, w[r][k], p[r], 0, 0, 0);
                }
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int i = 0; i < 16; i++) acc[t][r][i] = fmaf(sc[r], p[r][i], acc[t][r][i]);
        }
    };
    if (b0 < b1) {
        load_x(b0, 0);
        load_w(b0, code[0], scale[0]);
        for (uint32_t b = b0; b < b1; b += 2) {
            rm_arrive();  // this block's x is there, the other buffer is free
            if (b + 1 < b1) {
                load_x(b + 1, 1);
                load_w(b + 1, code[1], scale[1]);
            }
            block(code[0], scale[0], 0);
            if (b + 1 >= b1) break;
            rm_arrive();
            if (b + 2 < b1) {
                load_x(b + 2, 0);
                load_w(b + 2, code[0], scale[0]);
            }
            block(code[1], scale[1], 1);
        }
    }
    // Output i of a tile: row 8 (i / 4) + 4 h + i % 4 of x, weight row lane % 32.
    const float unit = Q4 ? 1.0f / 15.0f : 1.0f / 3.0f;
#pragma unroll
    for (int r = 0; r < RT; r++) {
        const uint32_t n = n0 + 32 * r + (lane & 31);
        if (n >= a.n) continue;
        const RmColumn c = rm_column_scales(a, n);
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const uint32_t row = (tile0 + t) * 32 + 8 * (i >> 2) + 4 * h + (i & 3);
                if (row >= a.rows) continue;
                float v = acc[t][r][i] * unit;
                if (PARTS == 2) v = ldexpf(v, a.exps[row] - 15);
                if (a.partial) a.partial[((size_t)split * a.rows + row) * a.n + n] = v;
                else rm_store(a, rm_finish(a, v, c, row, n), row, n);
            }
    }
}

#define RM_KERNEL(q4, parts, tt, rt, occ)                                                                      \
    extern "C" __global__ __launch_bounds__(256, occ) void ctox_rows_q##q4##_p##parts##_##tt##x##rt##_gfx950(RowsMulArgs a) { \
        rows_product<q4 == 4, parts, tt, rt>(a);                                                               \
    }
#define RM_KERNELS(q4, parts)      \
    RM_KERNEL(q4, parts, 1, 1, 2)  \
    RM_KERNEL(q4, parts, 2, 1, 2)  \
    RM_KERNEL(q4, parts, 4, 1, 2)  \
    RM_KERNEL(q4, parts, 4, 2, 2)
RM_KERNELS(4, 2)
RM_KERNELS(4, 1)
RM_KERNELS(2, 2)
RM_KERNELS(2, 1)

// grid (rows, ceil(n / 256)): the partial sums of a split K in order, then the epilogue.
extern "C" __global__ __launch_bounds__(256) void ctox_rows_reduce_gfx950(RowsMulArgs a) {
    const uint32_t n = blockIdx.y * 256 + threadIdx.x, t = blockIdx.x;
    if (n >= a.n) return;
    float v = 0.0f;
    for (uint32_t s = 0; s < a.splits; s++) v += a.partial[((size_t)s * a.rows + t) * a.n + n];
    rm_store(a, rm_finish(a, v, rm_column_scales(a, n), t, n), t, n);
}
