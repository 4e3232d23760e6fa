// The experts of a mixture: out[r] = sum_j weight[r][j] * down_e(q(act(gate_e(q x)) *
// up_e(q x))), e = ids[r][j], over block-scaled 8-bit weights, q the rows'
// quantization (fp8_core.cuh).
//
// Few rows: a workgroup takes an expert that some row chose and 16 hidden columns
// (experts_up; then 16 output columns, experts_down), finds its rows among the ids, and
// streams its weights once, 16 rows a pass, as fp8_gemv does. The hidden values stay f32
// until they are quantized, by a pass of their own (hidden_rows), which the second
// product's many workgroups would otherwise each repeat. One row (experts_up_token,
// experts_down_token): a workgroup for each of its experts, and the second product adds up
// the experts itself: two launches.
// Many rows: a plan puts each expert's rows together (expert_plan), one pass quantizes
// them into fragments in that order, and two grouped products (fp8_gemm.hip) follow,
// the first quantizing the hidden values in its store.
// A last pass adds up each row's experts in the order of its ids: no atomics, the same
// bits on every call. (The order within an expert's rows, which the plan's counters
// decide, changes no row's result.)
// What bounds it: few rows, reading the weights of the experts that are used; many
// rows, the products. Measured (weights from memory): one row, 6 of 64 experts, 2048 to 1280
// 14.5 us (47 MB); 37 rows, 8 of 64, 4096 to 1792 270 us (1.39 GB, 5.1 TB/s); 3001 rows, 8 of
// 128, 2048 to 1000 527 us (f16); 2048 rows, 2 of 8, 4096 to 14336 854 us (bf16; 1.7 PFLOP/s).
#include <algorithm>

#include "experts.h"
#include "fp8_core.cuh"
#include "tile_store.cuh"

namespace smg {

namespace {

constexpr int EG_NT = 512, EG_W = EG_NT / 64;  // threads, waves
constexpr uint32_t EG_MAX = 384;               // assignments the few-row form takes

struct EgArgs {
    Fp8Mat a, b;             // gate and up, or down
    const uint16_t *x;       // [rows][d]
    float *h;                // [assignments][hld] f32
    uint8_t *hq, *he;        // their codes [assignments][hld] and exponents [assignments][hld / 128]
    float *part;             // [assignments][n] f32 (down)
    const int32_t *ids;
    const float *weights;
    uint16_t *out;
    float *y;
    uint32_t top_k, assignments, experts, d, xld, hld, act;  // xld: x's rows
};

// The expert of slot y and the assignments that chose it: with no more assignments
// than experts a slot is an assignment, taken by the first that names its expert; else
// a slot is an expert. False (for the whole workgroup) if there is none.
__device__ __forceinline__ bool expert_of(const EgArgs &g, uint32_t slot, uint32_t &expert) {
    int e = (int)slot;
    if (g.assignments <= g.experts) {
        e = g.ids[slot];
        if (e < 0 || e >= (int)g.experts) return false;
        bool dup = false;
        const int lane = threadIdx.x % 64;
        for (uint32_t i = lane; i < slot; i += 64) dup |= g.ids[i] == e;
        if (__builtin_amdgcn_ballot_w64(dup)) return false;
    }
    expert = (uint32_t)__builtin_amdgcn_readfirstlane(e);
    return true;
}
// By each wave for itself: no barrier, and weight loads issued before stay in flight.
__device__ __forceinline__ uint32_t rows_of(const EgArgs &g, uint32_t expert, uint16_t *list) {
    const int lane = threadIdx.x % 64;
    uint32_t n = 0;
    for (uint32_t i0 = 0; i0 < g.assignments; i0 += 64) {
        const uint32_t i = i0 + lane;
        const bool mine = i < g.assignments && g.ids[i] == (int)expert;
        const uint64_t m = __builtin_amdgcn_ballot_w64(mine);
        if (mine) list[n + __builtin_popcountll(m & ((1ull << lane) - 1))] = (uint16_t)i;
        n += __builtin_popcountll(m);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)n);
}

// 32 f32 depths of a row to codes; as fp8_quant32.
__device__ __forceinline__ uint32_t fp8_quant32_f32(float (&x)[32], int8x_t &q) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    if (__builtin_amdgcn_ballot_w64(m >= 0x7F800000u)) {
        m = 0;
#pragma unroll
        for (int i = 0; i < 32; i++) {
            const uint32_t b = __float_as_uint(x[i]) & 0x7FFFFFFFu;
            if (b >= 0x7F800000u) x[i] = __builtin_nanf("");
            else m = max(m, b);
        }
    }
    m = max(m, (uint32_t)__shfl_xor((int)m, 16));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32));
    const uint32_t e = fp8_exp_byte(m);
    const float scale = __uint_as_float(e << 23);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        s16x2_t r = {0, 0};
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, x[4 * i], x[4 * i + 1], scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, x[4 * i + 2], x[4 * i + 3], scale, true);
        q[i] = __builtin_bit_cast(int, r);
    }
    return e;
}

// 32 f32 values of row `row` at depth d (zeros where row is -1), 16-byte aligned.
__device__ __forceinline__ void load_hidden32(const float *h, uint32_t ld, int row, uint32_t d, float (&x)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i++) x[i] = 0.0f;
    if (row < 0) return;
    const float4 *p = (const float4 *)(h + (size_t)row * ld + d);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float4 v = p[i];
        x[4 * i] = v.x;
        x[4 * i + 1] = v.y;
        x[4 * i + 2] = v.z;
        x[4 * i + 3] = v.w;
    }
}

__device__ __forceinline__ float glu_value(uint32_t act, float g, float u) {
    bool past;
    const float h = glu_near(act == EP_ACT_GELU, g, u, past);
    return past ? glu_far(act == EP_ACT_GELU, g, u) : h;
}

// The 32 values d .. of a row of d_max (16 dwords; zeros past it and where there is no
// row), 16-byte aligned and readable to a multiple of 8.
__device__ __forceinline__ void load_x32(const uint16_t *xp, bool live, uint32_t d0, uint32_t d_max, uint32_t (&a)[16]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t d = d0 + 8 * i;
        const uint4 v = live && d < d_max ? *(const uint4 *)(xp + d) : make_uint4(0, 0, 0, 0);
        a[4 * i] = v.x;
        a[4 * i + 1] = v.y;
        a[4 * i + 2] = v.z;
        a[4 * i + 3] = v.w;
    }
}

// Rows that cannot be read 8 values at a time, padded with zeros to where they can (read
// value by value by each workgroup instead, 37 rows of 4095, 8 of 64 experts, took 489 us
// for 277).
__global__ void __launch_bounds__(256) pad_rows(const uint16_t *x, uint32_t rows, uint32_t d, uint32_t ld, uint16_t *out) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, per = ld / 8;
    const size_t r = i / per;
    if (r >= rows) return;
    const uint32_t c = (uint32_t)(i - r * per) * 8;
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < 8; q++)
        if (c + q < d) v[q / 2] |= (uint32_t)x[r * d + c + q] << (16 * (q % 2));
    *(uint4 *)(out + r * ld + c) = make_uint4(v[0], v[1], v[2], v[3]);
}

// Hidden values of 16 columns (blockIdx.x) for slot blockIdx.y's rows.
template <bool BF16>
__global__ void __launch_bounds__(EG_NT, 4) experts_up(EgArgs g) {
    constexpr int U = 2;  // blocks of K a wave holds in flight
    __shared__ float4_t part[2][EG_W][64];
    __shared__ uint16_t lists[EG_W][EG_MAX];
    const int t = threadIdx.x, lane = t % 64, lr = lane % 16, lg = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(t / 64);
    uint32_t expert;
    if (!expert_of(g, blockIdx.y, expert)) return;
    const uint32_t tile = blockIdx.x, nkb = g.a.nkb, bytes = nkb * FP8_FRAG;
    const size_t frag = ((size_t)expert * g.a.n16 + tile) * bytes, sc = ((size_t)expert * (g.a.n16 / 8) + tile / 8) * nkb;
    const rsrc_t rg = make_rsrc(g.a.codes + frag, bytes), ru = make_rsrc(g.b.codes + frag, bytes);
    const rsrc_t sg = make_rsrc(g.a.scales + sc, nkb * 4), su = make_rsrc(g.b.scales + sc, nkb * 4);
    uint4 w[U][4];
    float s[U][2];
    auto load_w = [&](uint32_t kb0) __attribute__((always_inline)) {  // (zeros past the last block)
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t off = (kb0 + u * EG_W) * FP8_FRAG + lane * 16;
            w[u][0] = bload16_nt(rg, off);
            w[u][1] = bload16_nt(rg, off + 1024);
            w[u][2] = bload16_nt(ru, off);
            w[u][3] = bload16_nt(ru, off + 1024);
            s[u][0] = __uint_as_float(bload4(sg, (kb0 + u * EG_W) * 4));
            s[u][1] = __uint_as_float(bload4(su, (kb0 + u * EG_W) * 4));
        }
    };
    load_w(wave);
    const uint16_t *list = lists[wave];
    const uint32_t n = rows_of(g, expert, lists[wave]);
    for (uint32_t r0 = 0; r0 < n; r0 += 16) {
        const int as = r0 + lr < n ? list[r0 + lr] : -1;
        const uint16_t *xp = g.x + (size_t)(as < 0 ? 0 : (uint32_t)as / g.top_k) * g.xld;
        float4_t ag = {0.f, 0.f, 0.f, 0.f}, au = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t kb0 = wave; kb0 < nkb; kb0 += EG_W * U) {
            if (r0 != 0 || kb0 != (uint32_t)wave) load_w(kb0);
            uint32_t a[U][16];
#pragma unroll
            for (int u = 0; u < U; u++) load_x32(xp, as >= 0, (kb0 + u * EG_W) * FP8_BLOCK + 32 * lg, g.d, a[u]);
            int8x_t qs[U];
            float rss[U];
#pragma unroll
            for (int u = 0; u < U; u++) rss[u] = __uint_as_float(fp8_quant32<BF16>(a[u], qs[u]) << 23);  // the row's scale
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int8x_t &q = qs[u];
                const float rs = rss[u];
                const half8_t q16[4] = {fp8_to_f16(q[0], q[1]), fp8_to_f16(q[2], q[3]), fp8_to_f16(q[4], q[5]),
                                        fp8_to_f16(q[6], q[7])};
                fp8_fold(ag, fp8_mfma_f16(fp8_join(w[u][0], w[u][1]), q16), s[u][0] * rs);
                __builtin_amdgcn_sched_barrier(0);  // (one matrix's f16 values at a time: registers)
                fp8_fold(au, fp8_mfma_f16(fp8_join(w[u][2], w[u][3]), q16), s[u][1] * rs);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        part[0][wave][lane] = ag;
        part[1][wave][lane] = au;
        __syncthreads();
        if (t < 256 && r0 + t / 16 < n) {  // column t % 16 of row t / 16
            const uint32_t r = t / 16, c = t % 16;
            const float *p = (const float *)&part[0][0][(c / 4) * 16 + r] + c % 4;
            float xg = 0.0f, xu = 0.0f;
#pragma unroll
            for (int v = 0; v < EG_W; v++) {
                xg += p[v * 256];
                xu += p[(EG_W + v) * 256];
            }
            g.h[(size_t)list[r0 + r] * g.hld + tile * 16 + c] = glu_value(g.act, xg, xu);
        }
        __syncthreads();
    }
}

// The hidden rows' codes and exponents, row by row: a wave per (16 assignments, block of
// depths). Assignments of no expert hold what was there; nothing reads their codes.
__global__ void __launch_bounds__(256) hidden_rows(EgArgs g) {
    const uint32_t kbs = g.hld / FP8_BLOCK, w = blockIdx.x * 4 + threadIdx.x / 64;
    if (w >= (g.assignments + 15) / 16 * kbs) return;  // whole waves, no barrier follows
    const int lane = threadIdx.x % 64, lr = lane % 16, lg = lane / 16;
    const uint32_t as = w / kbs * 16 + lr, kb = w % kbs;
    float x[32];
    load_hidden32(g.h, g.hld, as < g.assignments ? (int)as : -1, kb * FP8_BLOCK + 32 * lg, x);
    int8x_t q;
    const uint32_t e = fp8_quant32_f32(x, q);
    if (as >= g.assignments) return;
    uint8_t *dst = g.hq + (size_t)as * g.hld + kb * FP8_BLOCK + 32 * lg;
    *(uint4 *)dst = make_uint4(q[0], q[1], q[2], q[3]);
    *(uint4 *)(dst + 16) = make_uint4(q[4], q[5], q[6], q[7]);
    if (lg == 0) g.he[(size_t)as * kbs + kb] = (uint8_t)e;
}

// Output columns of slot blockIdx.y's rows: each assignment's own sums.
__global__ void __launch_bounds__(EG_NT, 4) experts_down(EgArgs g) {
    constexpr int U = 2;
    __shared__ float4_t part[EG_W][64];
    __shared__ uint16_t lists[EG_W][EG_MAX];
    const int t = threadIdx.x, lane = t % 64, lr = lane % 16, lg = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(t / 64);
    uint32_t expert;
    if (!expert_of(g, blockIdx.y, expert)) return;
    const uint32_t tile = blockIdx.x, nkb = g.a.nkb, bytes = nkb * FP8_FRAG;
    const rsrc_t rw = make_rsrc(g.a.codes + ((size_t)expert * g.a.n16 + tile) * bytes, bytes);
    const rsrc_t rs = make_rsrc(g.a.scales + ((size_t)expert * (g.a.n16 / 8) + tile / 8) * nkb, nkb * 4);
    uint4 w[U][2];
    float s[U];
    auto load_w = [&](uint32_t kb0) __attribute__((always_inline)) {  // (zeros past the last block)
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t off = (kb0 + u * EG_W) * FP8_FRAG + lane * 16;
            w[u][0] = bload16_nt(rw, off);
            w[u][1] = bload16_nt(rw, off + 1024);
            s[u] = __uint_as_float(bload4(rs, (kb0 + u * EG_W) * 4));
        }
    };
    load_w(wave);
    const uint16_t *list = lists[wave];
    const uint32_t n = rows_of(g, expert, lists[wave]);
    for (uint32_t r0 = 0; r0 < n; r0 += 16) {
        const int as = r0 + lr < n ? list[r0 + lr] : -1;
        const size_t row = as < 0 ? 0 : as;
        float4_t acc = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t kb0 = wave; kb0 < nkb; kb0 += EG_W * U) {
            if (r0 != 0 || kb0 != (uint32_t)wave) load_w(kb0);
            uint4 q[U][2];
            uint32_t e[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t kb = kb0 + u * EG_W;
                q[u][0] = q[u][1] = make_uint4(0, 0, 0, 0);
                e[u] = 1;
                if (as >= 0 && kb < nkb) {
                    const uint8_t *p = g.hq + row * g.hld + kb * FP8_BLOCK + 32 * lg;
                    q[u][0] = *(const uint4 *)p;
                    q[u][1] = *(const uint4 *)(p + 16);
                    e[u] = g.he[row * nkb + kb];
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++)
                fp8_fold(acc, fp8_mfma<0>(fp8_join(w[u][0], w[u][1]), fp8_join(q[u][0], q[u][1]), e[u]), s[u]);
        }
        part[wave][lane] = acc;
        __syncthreads();
        if (t < 256 && r0 + t / 16 < n) {
            const uint32_t r = t / 16, c = t % 16, col = tile * 16 + c;
            const float *p = (const float *)&part[0][(c / 4) * 16 + r] + c % 4;
            float v = 0.0f;
#pragma unroll
            for (int x = 0; x < EG_W; x++) v += p[x * 256];
            if (col < g.a.n) g.part[(size_t)list[r0 + r] * g.a.n + col] = v;
        }
        __syncthreads();
    }
}

// One row. A wave quantizes the blocks it multiplies itself, two values a lane, and reads
// them back from its own LDS as every column of the second operand (of which the first
// counts), so that the weights, all issued before, wait for a few instructions.

// The wave's largest value, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, false));
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, false));
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xF, 0xF, false));
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x140, 0xF, 0xF, false));
    const uint32_t a = __builtin_amdgcn_readlane((int)x, 0), b = __builtin_amdgcn_readlane((int)x, 16);
    const uint32_t c = __builtin_amdgcn_readlane((int)x, 32), d = __builtin_amdgcn_readlane((int)x, 48);
    return max(max(a, b), max(c, d));
}
// Two values a lane of a block to their codes (the low 16 bits); the block's exponent.
__device__ __forceinline__ uint32_t quant_pair(float x, float y, uint32_t &e) {
    uint32_t bx = __float_as_uint(x) & 0x7FFFFFFFu, by = __float_as_uint(y) & 0x7FFFFFFFu;
    if (bx >= 0x7F800000u) {  // infinities and NaN: NaN codes, not counted
        x = __builtin_nanf("");
        bx = 0;
    }
    if (by >= 0x7F800000u) {
        y = __builtin_nanf("");
        by = 0;
    }
    e = fp8_exp_byte(wave_max(max(bx, by)));
    s16x2_t r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, x, y, __uint_as_float(e << 23), false);
    return (uint16_t)r[0];
}
// The 32 bytes a lane multiplies of a block of 128 codes in LDS.
__device__ __forceinline__ int8x_t lds_codes(const uint8_t *block, int lg) {
    const uint4 *p = (const uint4 *)(block + 32 * lg);
    return fp8_join(p[0], p[1]);
}

// Hidden values of 16 columns (blockIdx.x) of the row's expert blockIdx.y.
template <bool BF16>
__global__ void __launch_bounds__(EG_NT, 4) experts_up_token(EgArgs g) {
    constexpr int U = 3;
    __shared__ float4_t part[2][EG_W][64];
    __shared__ __align__(16) uint8_t codes[EG_W][U][FP8_BLOCK];
    const int t = threadIdx.x, lane = t % 64, lg = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(t / 64);
    const int expert = g.ids[blockIdx.y];
    if (expert < 0 || expert >= (int)g.experts) return;
    const uint32_t tile = blockIdx.x, nkb = g.a.nkb, bytes = nkb * FP8_FRAG;
    const size_t frag = ((size_t)expert * g.a.n16 + tile) * bytes, sc = ((size_t)expert * (g.a.n16 / 8) + tile / 8) * nkb;
    const rsrc_t rg = make_rsrc(g.a.codes + frag, bytes), ru = make_rsrc(g.b.codes + frag, bytes);
    const rsrc_t sg = make_rsrc(g.a.scales + sc, nkb * 4), su = make_rsrc(g.b.scales + sc, nkb * 4);
    const rsrc_t rx = make_rsrc(g.x, g.d * 2u);
    float4_t ag = {0.f, 0.f, 0.f, 0.f}, au = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t kb0 = wave; kb0 < nkb; kb0 += EG_W * U) {  // (past the last block all read zeros)
        uint16_t x[U][2];
        uint4 w[U][4];
        float s[U][2];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t d = (kb0 + u * EG_W) * FP8_BLOCK + 2 * lane;
            x[u][0] = bload2(rx, d * 2);
            x[u][1] = bload2(rx, d * 2 + 2);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t off = (kb0 + u * EG_W) * FP8_FRAG + lane * 16;
            w[u][0] = bload16_nt(rg, off);
            w[u][1] = bload16_nt(rg, off + 1024);
            w[u][2] = bload16_nt(ru, off);
            w[u][3] = bload16_nt(ru, off + 1024);
            s[u][0] = __uint_as_float(bload4(sg, (kb0 + u * EG_W) * 4));
            s[u][1] = __uint_as_float(bload4(su, (kb0 + u * EG_W) * 4));
        }
        uint32_t e[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            *(uint16_t *)(codes[wave][u] + 2 * lane) = (uint16_t)quant_pair(to_f32<BF16>(x[u][0]), to_f32<BF16>(x[u][1]), e[u]);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int8x_t q = lds_codes(codes[wave][u], lg);
            const float rs = __uint_as_float(e[u] << 23);
            const half8_t q16[4] = {fp8_to_f16(q[0], q[1]), fp8_to_f16(q[2], q[3]), fp8_to_f16(q[4], q[5]), fp8_to_f16(q[6], q[7])};
            fp8_fold(ag, fp8_mfma_f16(fp8_join(w[u][0], w[u][1]), q16), s[u][0] * rs);
            fp8_fold(au, fp8_mfma_f16(fp8_join(w[u][2], w[u][3]), q16), s[u][1] * rs);
        }
    }
    part[0][wave][lane] = ag;
    part[1][wave][lane] = au;
    __syncthreads();
    if (t >= 16) return;
    const float *p = (const float *)&part[0][0][(t / 4) * 16] + t % 4;
    float xg = 0.0f, xu = 0.0f;
#pragma unroll
    for (int v = 0; v < EG_W; v++) {
        xg += p[v * 256];
        xu += p[(EG_W + v) * 256];
    }
    g.h[(size_t)blockIdx.y * g.hld + tile * 16 + t] = glu_value(g.act, xg, xu);
}

// 16 output columns: the (expert, block of depths) pairs of all the row's experts over the
// waves, the experts' weights folded with the blocks' scales.
template <bool BF16>
__global__ void __launch_bounds__(EG_NT, 4) experts_down_token(EgArgs g) {
    constexpr int U = 8;
    __shared__ float4_t part[EG_W][64];
    __shared__ __align__(16) uint8_t codes[EG_W][U][FP8_BLOCK];
    const int t = threadIdx.x, lane = t % 64, lg = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(t / 64);
    const uint32_t tile = blockIdx.x, nkb = g.a.nkb, pairs = g.top_k * nkb;
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t p0 = wave; p0 < pairs; p0 += EG_W * U) {
        float2 h[U];
        uint4 w[U][2];
        float s[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t p = p0 + u * EG_W, j = p / nkb, kb = p - j * nkb;
            const int e = p < pairs ? g.ids[j] : -1;
            const bool live = e >= 0 && e < (int)g.experts;  // (else nothing is added: zeros by a scale of zero)
            h[u] = make_float2(0.0f, 0.0f);
            w[u][0] = w[u][1] = make_uint4(0, 0, 0, 0);
            s[u] = 0.0f;
            if (live) {
                h[u] = *(const float2 *)(g.h + (size_t)j * g.hld + kb * FP8_BLOCK + 2 * lane);
                const uint8_t *c = g.a.codes + (((size_t)e * g.a.n16 + tile) * nkb + kb) * FP8_FRAG + lane * 16;
                w[u][0] = *(const uint4 *)c;
                w[u][1] = *(const uint4 *)(c + 1024);
                s[u] = g.a.scales[((size_t)e * (g.a.n16 / 8) + tile / 8) * nkb + kb] * g.weights[j];
            }
        }
        uint32_t e[U];
#pragma unroll
        for (int u = 0; u < U; u++) *(uint16_t *)(codes[wave][u] + 2 * lane) = (uint16_t)quant_pair(h[u].x, h[u].y, e[u]);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int u = 0; u < U; u++)
            fp8_fold(acc, fp8_mfma<0>(fp8_join(w[u][0], w[u][1]), lds_codes(codes[wave][u], lg), e[u]), s[u]);
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (t >= 16) return;
    const uint32_t col = tile * 16 + t;
    if (col >= g.a.n) return;
    const float *p = (const float *)&part[0][(t / 4) * 16] + t % 4;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < EG_W; w++) v += p[w * 256];
    if (g.y) g.y[col] += v;
    else g.out[col] = from_f32<BF16>(v);
}

// out[r] (or y[r] +=) the weighted sum of the row's experts' parts, in the order of its
// ids; a part's row is the assignment's, or place[assignment]. Parts are f32: one may lie past
// an f16's range, or below its steps, where the sum and y do not (f16 parts took 369 us for
// 3001 rows, 8 of 128 experts, 407 with f32). A workgroup takes 2048 columns of a row, a
// thread 8, four experts' parts in flight. VEC: whole groups of 8.
template <bool BF16, bool VEC>
__global__ void __launch_bounds__(256) experts_sum(const float *part, const int32_t *place, const int32_t *ids,
                                                   const float *weights, uint32_t top_k, uint32_t experts, uint32_t d,
                                                   uint32_t parts, uint16_t *out, float *y) {
    const uint32_t r = blockIdx.x / parts, col = (blockIdx.x % parts * 256 + threadIdx.x) * 8;
    if (col >= d) return;
    const uint32_t ne = min(d - col, 8u);
    constexpr int U = 4;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (uint32_t j0 = 0; j0 < top_k; j0 += U) {
        float w[U];
        float x[U][8];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t as = (size_t)r * top_k + j0 + u;
            const int e = j0 + u < top_k ? ids[as] : -1;
            w[u] = 0.0f;
#pragma unroll
            for (int c = 0; c < 8; c++) x[u][c] = 0.0f;
            if (e < 0 || e >= (int)experts) continue;
            w[u] = weights[as];
            const float *p = part + (place ? (size_t)place[as] : as) * d + col;
            if (VEC) {
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const float4 v = ((const float4 *)p)[c];
                    x[u][4 * c] = v.x;
                    x[u][4 * c + 1] = v.y;
                    x[u][4 * c + 2] = v.z;
                    x[u][4 * c + 3] = v.w;
                }
            } else {
                for (uint32_t c = 0; c < ne; c++) x[u][c] = p[c];
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int e = j0 + u < top_k ? ids[(size_t)r * top_k + j0 + u] : -1;
            if (e < 0 || e >= (int)experts) continue;
#pragma unroll
            for (int c = 0; c < 8; c++) s[c] = __builtin_fmaf(w[u], x[u][c], s[c]);
        }
    }
    const size_t o = (size_t)r * d + col;
    if (y) {
        for (uint32_t c = 0; c < ne; c++) y[o + c] += s[c];
        return;
    }
    if (ne == 8 && ((uintptr_t)(out + o) & 15) == 0) {
        uint32_t h[4];
#pragma unroll
        for (int c = 0; c < 4; c++)
            h[c] = (uint32_t)from_f32<BF16>(s[2 * c]) | (uint32_t)from_f32<BF16>(s[2 * c + 1]) << 16;
        *(uint4 *)(out + o) = make_uint4(h[0], h[1], h[2], h[3]);
        return;
    }
    for (uint32_t c = 0; c < ne; c++) out[o + c] = from_f32<BF16>(s[c]);
}
// Threads of a launch over rows (launchable).
constexpr size_t MOST_THREADS = (size_t)1 << 31;
template <bool BF16>
hipError_t launch_sum(const ExpertCall &c, const float *part, const int32_t *place, uint32_t experts, uint32_t d,
                      hipStream_t s) {
    const uint32_t parts = (d + 2047) / 2048, piece = (uint32_t)(MOST_THREADS / 256 / parts);
    for (uint32_t r0 = 0; r0 < c.rows; r0 += piece) {
        const size_t as = (size_t)r0 * c.top_k, o = (size_t)r0 * d;
        const dim3 grid(std::min(piece, c.rows - r0) * parts);
        hipLaunchKernelGGL((d % 8 == 0 ? experts_sum<BF16, true> : experts_sum<BF16, false>), grid, dim3(256), 0, s,
                           place ? part : part + as * d, place ? place + as : nullptr, c.ids + as, c.weights + as, c.top_k,
                           experts, d, parts, c.out ? c.out + o : nullptr, c.y ? c.y + o : nullptr);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// The plan, by one workgroup: the experts' counts, their rows' starts, the tiles, and
// every assignment's place.
constexpr int PL_NT = 1024;
__global__ void __launch_bounds__(PL_NT) expert_plan(const int32_t *ids, ExpertPlan p) {
    constexpr uint32_t SRC = 32768;  // of the plan's rows at a time: scattered 4-byte stores would cost 10 us more
    __shared__ uint32_t count[ROUTE_MAX_EXPERTS], start[ROUTE_MAX_EXPERTS], scan[3][PL_NT];
    __shared__ __align__(16) int32_t source[SRC];
    const uint32_t t = threadIdx.x;
    static_assert(ROUTE_MAX_EXPERTS <= PL_NT, "a thread an expert");
    constexpr int U = 8;  // assignments a thread has in flight
    count[t] = 0;
    __syncthreads();
    for (uint32_t i0 = t; i0 < p.assignments; i0 += PL_NT * U) {
        int e[U];
#pragma unroll
        for (int u = 0; u < U; u++) e[u] = i0 + u * PL_NT < p.assignments ? ids[i0 + u * PL_NT] : -1;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const bool live = e[u] >= 0 && e[u] < (int)p.experts;
            const int rank = live ? (int)atomicAdd(&count[live ? e[u] : 0], 1u) : -1;
            if (i0 + u * PL_NT < p.assignments) p.rank[i0 + u * PL_NT] = rank;
        }
    }
    __syncthreads();
    const uint32_t n = t < p.experts ? count[t] : 0, padded = (n + 63) / 64 * 64;
    const bool half = n % 256 != 0 && n % 256 <= 128;  // the last tile
    uint32_t x[3] = {padded, n / 256 + (n % 256 > 128), half};  // rows, tiles of 256, of 128; then inclusive sums
    const uint32_t full = x[1];
#pragma unroll
    for (int i = 0; i < 3; i++) scan[i][t] = x[i];
    __syncthreads();
    for (uint32_t d = 1; d < PL_NT; d <<= 1) {
        uint32_t y[3];
#pragma unroll
        for (int i = 0; i < 3; i++) y[i] = t >= d ? scan[i][t - d] : 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 3; i++) scan[i][t] = x[i] += y[i];
        __syncthreads();
    }
    const uint32_t total = scan[0][PL_NT - 1];
    if (t == 0) {
        p.head[EXPERT_TILES] = scan[1][PL_NT - 1] + scan[2][PL_NT - 1];
        p.head[EXPERT_ROWS] = total;
    }
    const uint32_t first = x[0] - padded;
    start[t] = first;
    const uint32_t mine = full + half, tile0 = x[1] + x[2] - mine;
    for (uint32_t i = 0; i < mine; i++) p.tiles[tile0 + i] = {t, half, tile0, mine, first / 16, (first + padded) / 16};
    // The places of a few chunks of rows go out through LDS, those of more directly (for
    // which the LDS passes would read every assignment once a chunk).
    const bool direct = total > 4 * SRC;
    if (direct)
        for (uint32_t i = n; i < padded; i++) p.source[first + i] = -1;
    __syncthreads();
    for (uint32_t s0 = 0; s0 < total; s0 += SRC) {
        if (!direct) {
            for (uint32_t i = t; i < SRC / 4; i += PL_NT) ((int4 *)source)[i] = make_int4(-1, -1, -1, -1);
            __syncthreads();
        }
        for (uint32_t i0 = t; i0 < p.assignments; i0 += PL_NT * U) {
            int e[U], rank[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t i = i0 + u * PL_NT;
                e[u] = i < p.assignments ? ids[i] : -1;
                rank[u] = i < p.assignments ? p.rank[i] : -1;
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t i = i0 + u * PL_NT;
                const uint32_t at = rank[u] >= 0 ? start[e[u]] + (uint32_t)rank[u] : 0;
                if (rank[u] >= 0) {
                    if (direct) p.source[at] = (int32_t)i;
                    else if (at - s0 < SRC) source[at - s0] = (int32_t)i;
                }
                if (s0 == 0 && i < p.assignments) p.place[i] = rank[u] >= 0 ? (int32_t)at : -1;
            }
        }
        if (direct) return;
        __syncthreads();
        for (uint32_t i = t; i < SRC / 4 && s0 + i * 4 < total; i += PL_NT) ((int4 *)p.source)[s0 / 4 + i] = ((int4 *)source)[i];
        __syncthreads();
    }
    if (total == 0)
        for (uint32_t i = t; i < p.assignments; i += PL_NT) p.place[i] = -1;
}

// The plan's rows quantized into fragments: a wave per (16 rows, block of depths). (A row
// is read and quantized once for each of its experts; quantized once and written to all
// their places instead, the pieces of 16 bytes cost more than that: 48 us against 25 at
// 3001 rows of 2048, 8 experts each.)
template <bool BF16>
__global__ void __launch_bounds__(256) expert_rows(const uint16_t *x, uint32_t xld, ExpertPlan p, uint32_t d, uint32_t nkb,
                                                   Fp8Rows o) {
    const size_t w = (size_t)blockIdx.x * 4 + threadIdx.x / 64;
    const uint32_t mt = (uint32_t)(w / nkb), kb = (uint32_t)(w % nkb);
    if (mt * 16 >= p.head[EXPERT_ROWS]) return;  // whole waves, no barrier follows
    const int lane = threadIdx.x % 64, lr = lane % 16, lg = lane / 16;
    const int as = p.source[mt * 16 + lr];
    const uint16_t *xp = x + (size_t)(as < 0 ? 0 : (uint32_t)as / p.top_k) * xld;
    uint32_t a[16];
    load_x32(xp, as >= 0, kb * FP8_BLOCK + 32 * lg, d, a);
    int8x_t q;
    const uint32_t eb = fp8_quant32<BF16>(a, q);
    uint8_t *dst = o.q + ((size_t)mt * nkb + kb) * FP8_FRAG + lane * 16;
    *(uint4 *)dst = make_uint4(q[0], q[1], q[2], q[3]);
    *(uint4 *)(dst + 1024) = make_uint4(q[4], q[5], q[6], q[7]);
    if (lg == 0) o.e[(((size_t)mt / 4 * nkb + kb) * 16 + lr) * 4 + mt % 4] = (uint8_t)eb;
}

// Calls the few-row form takes. It streams an expert's weights once for each 16 of its
// rows, the tiles once, more slowly and after a plan. Measured (us, few rows / tiles; rows,
// experts a row of so many, width, hidden width): 37, 8 of 64, 4096, 1792 284 / 316; 48 308
// / 317; 56 348 / 321; 64 369 / 323; 64, 8 of 128, 2048, 1000 222 / 197; 16, 2 of 8, 4096,
// 14336 245 / 334; 32 286 / 334; 64 466 / 336; 16, 8 of 16, 2048, 1408 45 / 58; 32 68 / 58.
bool few_rows(size_t rows, size_t top_k, size_t experts) {
    const size_t as = rows * top_k;
    return as <= EG_MAX && as <= 8 * experts;
}

// Whether the call's rows are copied to where they can be read 8 values at a time (one
// row's kernels read two).
bool may_pad(const ExpertSet &e, size_t rows, size_t top_k) { return !(rows == 1 && few_rows(rows, top_k, e.gate.mats)); }
bool pads(const ExpertSet &e, const ExpertCall &c) {
    return (e.gate.k % 8 != 0 || ((uintptr_t)c.x & 15) != 0) && may_pad(e, c.rows, c.top_k);
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// The scratch of a call: few rows: hidden f32 rows and (past one row) f32 parts; many:
// the plan, the rows and the hidden values in fragments, the parts.
struct Layout {
    ExpertPlan p;
    Fp8Rows x, h;
    float *hidden, *part;
    uint8_t *hq, *he;
    uint16_t *padded;
    size_t bytes;
};
Layout layout(const ExpertSet &e, size_t rows, size_t top_k, bool pads, void *scratch) {
    Layout l = {};
    uint8_t *at = (uint8_t *)scratch;
    auto take = [&](size_t bytes) {
        uint8_t *p = at;
        at += up256(bytes);
        return p;
    };
    const size_t as = rows * top_k, experts = e.gate.mats;
    if (pads) l.padded = (uint16_t *)take(rows * ((e.gate.k + 7) / 8 * 8) * 2);
    if (few_rows(rows, top_k, experts)) {
        l.hidden = (float *)take(as * e.down.nkb * FP8_BLOCK * 4);
        if (rows > 1) {
            l.part = (float *)take(as * e.down.n * 4);
            l.hq = take(as * e.down.nkb * FP8_BLOCK);
            l.he = take(as * e.down.nkb);
        }
    } else {
        const size_t used = std::min(experts, as);
        l.p.assignments = (uint32_t)as;
        l.p.top_k = (uint32_t)top_k;
        l.p.experts = (uint32_t)experts;
        l.p.max_rows = (uint32_t)((as + used * 63) / 64 * 64);
        l.p.max_tiles = (uint32_t)(as / 256 + used);
        l.p.head = (uint32_t *)take(256);
        l.p.tiles = (ExpertTile *)take(l.p.max_tiles * sizeof(ExpertTile));
        l.p.place = (int32_t *)take(as * 4);
        l.p.rank = (int32_t *)take(as * 4);
        l.p.source = (int32_t *)take((size_t)l.p.max_rows * 4);
        l.x = Fp8Rows::at(take(Fp8Rows::bytes(l.p.max_rows, e.gate.nkb)), l.p.max_rows, e.gate.nkb);
        l.h = Fp8Rows::at(take(Fp8Rows::bytes(l.p.max_rows, e.down.nkb)), l.p.max_rows, e.down.nkb);
        l.part = (float *)take((size_t)l.p.max_rows * e.down.n * 4);
    }
    l.bytes = (size_t)(at - (uint8_t *)scratch);
    return l;
}

}  // namespace

size_t experts_scratch_bytes(const ExpertSet &e, const ExpertCall &c) {
    return layout(e, c.rows, c.top_k, pads(e, c), nullptr).bytes;
}
size_t experts_scratch_bytes(const ExpertSet &e, size_t rows, size_t top_k) {
    return layout(e, rows, top_k, may_pad(e, rows, top_k), nullptr).bytes;
}

hipError_t launch_experts(const ExpertSet &e, const ExpertCall &c, void *scratch, hipStream_t s) {
    const Layout l = layout(e, c.rows, c.top_k, pads(e, c), scratch);
    const uint32_t d = e.gate.k, as = c.rows * c.top_k, experts = e.gate.mats, xld = l.padded ? (d + 7) / 8 * 8 : d;
    const uint16_t *x = l.padded ? l.padded : c.x;
    hipError_t err;
    if (l.padded) {
        const uint32_t piece = (uint32_t)(MOST_THREADS / (xld / 8));
        for (uint32_t r0 = 0; r0 < c.rows; r0 += piece) {
            const uint32_t n = std::min(piece, c.rows - r0);
            const size_t blocks = ((size_t)n * (xld / 8) + 255) / 256;
            hipLaunchKernelGGL(pad_rows, dim3((uint32_t)blocks), dim3(256), 0, s, c.x + (size_t)r0 * d, n, d, xld,
                               l.padded + (size_t)r0 * xld);
            if ((err = hipGetLastError()) != hipSuccess) return err;
        }
    }
    if (l.hidden) {
        EgArgs g = {};
        g.a = e.gate;
        g.b = e.up;
        g.x = x;
        g.h = l.hidden;
        g.hq = l.hq;
        g.he = l.he;
        g.part = l.part;
        g.ids = c.ids;
        g.weights = c.weights;
        g.out = c.out;
        g.y = c.y;
        g.top_k = c.top_k;
        g.assignments = as;
        g.experts = experts;
        g.d = d;
        g.xld = xld;
        g.hld = e.down.nkb * FP8_BLOCK;
        g.act = e.act;
        const uint32_t slots = std::min(as, experts);
        const dim3 up(e.gate.n16, slots);  // (whole blocks of 128: the padding's hidden values are zeros)
        if (c.rows == 1 && c.bf16) hipLaunchKernelGGL((experts_up_token<true>), dim3(e.gate.n16, as), dim3(EG_NT), 0, s, g);
        else if (c.rows == 1) hipLaunchKernelGGL((experts_up_token<false>), dim3(e.gate.n16, as), dim3(EG_NT), 0, s, g);
        else if (c.bf16) hipLaunchKernelGGL((experts_up<true>), up, dim3(EG_NT), 0, s, g);
        else hipLaunchKernelGGL((experts_up<false>), up, dim3(EG_NT), 0, s, g);
        if ((err = hipGetLastError()) != hipSuccess) return err;
        g.a = e.down;
        const dim3 down((d + 15) / 16, slots);
        if (c.rows == 1) {
            if (c.bf16) hipLaunchKernelGGL((experts_down_token<true>), dim3(down.x), dim3(EG_NT), 0, s, g);
            else hipLaunchKernelGGL((experts_down_token<false>), dim3(down.x), dim3(EG_NT), 0, s, g);
            return hipGetLastError();
        }
        hipLaunchKernelGGL(hidden_rows, dim3(((as + 15) / 16 * e.down.nkb + 3) / 4), dim3(256), 0, s, g);
        if ((err = hipGetLastError()) != hipSuccess) return err;
        hipLaunchKernelGGL(experts_down, down, dim3(EG_NT), 0, s, g);
        if ((err = hipGetLastError()) != hipSuccess) return err;
        return c.bf16 ? launch_sum<true>(c, l.part, nullptr, experts, d, s) : launch_sum<false>(c, l.part, nullptr, experts, d, s);
    }
    hipLaunchKernelGGL(expert_plan, dim3(1), dim3(PL_NT), 0, s, c.ids, l.p);
    if ((err = hipGetLastError()) != hipSuccess) return err;
    const uint32_t nkb = e.gate.nkb;
    const size_t waves = (size_t)l.p.max_rows / 16 * nkb;
    if (!launchable(waves, 64)) return hipErrorInvalidConfiguration;
    const dim3 rows((uint32_t)((waves + 3) / 4));
    if (c.bf16) hipLaunchKernelGGL((expert_rows<true>), rows, dim3(256), 0, s, x, xld, l.p, d, nkb, l.x);
    else hipLaunchKernelGGL((expert_rows<false>), rows, dim3(256), 0, s, x, xld, l.p, d, nkb, l.x);
    if ((err = hipGetLastError()) != hipSuccess) return err;
    // The 8-bit instructions' dropped bits (fp8_mfma) move a hidden value next to the border of
    // two codes to the other one, 0.0011 of the result's 2-norm where f32 sums move 0.0002. An
    // f16 result and f32 rows would show that; bf16's own rounding is 0.0017 (3001 rows, 8 of
    // 128 experts, 2048 to 1000: 407 us with 8-bit products, 532 with f16 ones; 2048 rows, 2 of
    // 8, 4096 to 14336: 892 and 1322).
    const bool exact = c.y != nullptr || !c.bf16;
    if ((err = launch_fp8_grouped(e.gate, &e.up, e.act, l.p, l.x, l.h, nullptr, exact, s)) != hipSuccess) return err;
    if ((err = launch_fp8_grouped(e.down, nullptr, 0, l.p, l.h, l.h, l.part, false, s)) != hipSuccess) return err;
    return c.bf16 ? launch_sum<true>(c, l.part, l.p.place, experts, d, s) : launch_sum<false>(c, l.part, l.p.place, experts, d, s);
}

}  // namespace smg
