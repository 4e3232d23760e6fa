// 8-bit floating-point products of many rows: C = ep(to16(sum_b scale_b (q w_b)))
// over rows quantized into fragments (fp8_quant) and weights packed into them
// (fp8_pack). Products are v_mfma_scale_f32_16x16x128_f8f6f4, one for each block of
// 128 depths, whose scale operand takes the rows' exponents; a block's sums start
// from zero and join the f32 totals by one fma with the weight block's scale, which
// a wave holds in a scalar register.
//
// fp8_big: 256 x 256 (or 128 x 256) tiles. fp8_tile: smaller tiles of four waves for
// smaller products. A fragment is 1 KB a wave read, in order, so nothing is swizzled.
// Grouped (a mixture's experts): the rows are the experts' assignments one expert
// after another, each expert's padded to 64 (ExpertPlan), and a tile's weights are its
// expert's. GLU: a wave's column halves are 32 gate and the same 32 up columns, so that
// a lane holds both factors of a hidden value; the tile's 128 hidden columns are one
// block of the next product's depths, which the store quantizes into its fragments.
// GLU16: tiles of 128 rows over v_mfma_f32_16x16x32_f16 of the codes, widened in registers,
// for results that would show the 8-bit instructions' dropped bits (launch_experts).
#include <algorithm>
#include <type_traits>

#include "dense_tile.cuh"
#include "experts.h"
#include "fp8_core.cuh"

namespace smg {

namespace {

struct F8Args {
    DArgs d;                    // store, m, n and the compiled store's operands
    const uint8_t *q, *e;       // the rows (Fp8Rows)
    const uint8_t *w;           // the weights' codes and scales
    const float *sw;
    uint32_t mt16, n16, nkb;
    uint32_t full;              // dense: tiles of 256 rows; the workgroups past them take 128 rows each
    // grouped: the plan, GLU's up weights, activation and output
    const uint32_t *head;
    const ExpertTile *tiles;
    const uint8_t *w2;
    const float *sw2;
    uint32_t act;
    uint8_t *hq, *he;
    uint32_t hkb;               // blocks of the hidden width
};

enum F8Mode : int { F8_DENSE = 0, F8_GROUPED = 1, F8_GLU = 2, F8_GLU16 = 3 };
constexpr bool f8_glu(int mode) { return mode >= F8_GLU; }

// A weight block's scales for 64 consecutive blocks of K, one a lane, read back by
// v_readlane: a scalar operand for the fold without a memory wait in the loop.
__device__ __forceinline__ float scale_lane(const float *s, uint32_t kb, uint32_t nkb, int lane) {
    float x = s[min(kb + lane, nkb - 1)];
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0), here and not where it is used
    asm volatile("" : "+v"(x));
    return x;
}
__device__ __forceinline__ float scale_at(float lanes, uint32_t kb) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lanes), kb % 64));
}

// A wave-uniform address in scalar registers.
__device__ __forceinline__ const uint8_t *scalar_ptr(const uint8_t *p) {
    const uint64_t b = (uint64_t)p;
    return (const uint8_t *)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32) |
                             (uint32_t)__builtin_amdgcn_readfirstlane((int)b));
}

// Hidden values act(gate) * up of a wave's piece (lane: row lr of row tile i, hidden
// columns 16 j + 4 lg .. of its wave's 32; column tiles 0, 1 the gate's, 2, 3 the up
// weights') quantized into the next product's fragments. mx: the rows' largest
// magnitudes, [BM rows][4 waves].
template <int RT, int NJ>
__device__ __forceinline__ void glu_store(const F8Args &f, const float4_t (&c)[RT][NJ], uint32_t *mx, uint32_t rt0,
                                          uint32_t rt_end, uint32_t kb, int wr, int wc, int lane) {
    static_assert(NJ == 4, "four waves of 32 hidden columns");
    const int lr = lane % 16, lg = lane / 16;
    float4_t h[RT][2];
    uint32_t m[RT];
    bool bad = false, far = false;
    const bool gelu = f.act == EP_ACT_GELU;
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                bool past;
                h[i][j][v] = glu_near(gelu, c[i][j][v], c[i][2 + j][v], past);
                far |= past;
            }
    if (__builtin_amdgcn_ballot_w64(far)) {
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    bool past;
                    const float x = glu_near(gelu, c[i][j][v], c[i][2 + j][v], past);
                    h[i][j][v] = past ? glu_far(gelu, c[i][j][v], c[i][2 + j][v]) : x;
                }
    }
#pragma unroll
    for (int i = 0; i < RT; i++) {
        m[i] = 0;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const uint32_t b = __float_as_uint(h[i][j][v]) & 0x7FFFFFFFu;
                bad |= b >= 0x7F800000u;
                m[i] = max(m[i], b);
            }
    }
    if (__builtin_amdgcn_ballot_w64(bad)) {  // infinities and NaN: NaN codes, not counted
#pragma unroll
        for (int i = 0; i < RT; i++) {
            m[i] = 0;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const uint32_t b = __float_as_uint(h[i][j][v]) & 0x7FFFFFFFu;
                    if (b >= 0x7F800000u) h[i][j][v] = __builtin_nanf("");
                    else m[i] = max(m[i], b);
                }
        }
    }
#pragma unroll
    for (int i = 0; i < RT; i++) {
        m[i] = max(m[i], (uint32_t)__shfl_xor((int)m[i], 16));
        m[i] = max(m[i], (uint32_t)__shfl_xor((int)m[i], 32));
        if (lg == 0) mx[((wr * RT + i) * 16 + lr) * 4 + wc] = m[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RT; i++) {
        const uint4 q4 = *(const uint4 *)(mx + ((wr * RT + i) * 16 + lr) * 4);
        const uint32_t e = fp8_exp_byte(max(max(q4.x, q4.y), max(q4.z, q4.w)));
        const uint32_t rt = rt0 + wr * RT + i;
        if (rt >= rt_end) continue;
        const float scale = __uint_as_float(e << 23);
        uint8_t *dst = f.hq + ((size_t)rt * f.hkb + kb) * FP8_FRAG + (wc * 16 + lr) * 16 + 4 * lg;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            s16x2_t r = {0, 0};
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, h[i][j][0], h[i][j][1], scale, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, h[i][j][2], h[i][j][3], scale, true);
            *(uint32_t *)(dst + j * 1024) = __builtin_bit_cast(uint32_t, r);
        }
        if (wc == 0 && lg == 0) f.he[(((size_t)rt / 4 * f.hkb + kb) * 16 + lr) * 4 + rt % 4] = (uint8_t)e;
    }
}

// A workgroup's tile: its first row tile (and the end of those it may store), whether it
// has 128 rows (else 256; fp8_big), its column number, its weights.
struct F8Place {
    uint32_t rt0, rt_end, tn;
    bool half;
    const uint8_t *codes, *codes2;
    const float *scales, *scales2;
};
template <int BM, int BN, int MODE>
__device__ __forceinline__ bool f8_place(const F8Args &f, DArgs &g, F8Place &p) {
    constexpr int CN = f8_glu(MODE) ? BN / 2 : BN;  // columns a tile stands for
    p.codes = f.w;
    p.codes2 = f.w2;
    p.scales = f.sw;
    p.scales2 = f.sw2;
    p.rt_end = f.mt16;
    p.half = false;
    uint32_t tm;
    const uint32_t nt = (g.n + CN - 1) / CN;
    if constexpr (MODE == F8_DENSE && BM < 256) {
        dense_tile<8>(blockIdx.x, gridDim.x, (g.m + BM - 1) / BM, nt, tm, p.tn);
        p.rt0 = tm * (BM / 16);
    } else if constexpr (MODE == F8_DENSE) {
        const uint32_t b = blockIdx.x, mt = (g.m + 255) / 256;
        p.half = b >= f.full;
        if (f.full == 0) {
            dense_tile<8>(b, gridDim.x, (g.m + 127) / 128, nt, tm, p.tn);
            p.rt0 = tm * 8;
        } else {
            dense_tile<8>(p.half ? f.full + (b - f.full) / 2 : b, mt * nt, mt, nt, tm, p.tn);
            p.rt0 = tm * 16 + (p.half && (b - f.full) % 2 ? 8 : 0);
            if (p.rt0 >= f.mt16) return false;
        }
    } else {
        const uint32_t count = f.head[EXPERT_TILES];
        constexpr uint32_t SPLIT = 256 / BM;  // tiles of 128 rows: two of each of the plan's
        if (blockIdx.x >= count * nt * SPLIT) return false;  // (the grid is what any plan may need)
        // An XCD's workgroups take a contiguous run of an expert's rows tiles x columns, rows
        // first, so that the expert's weights stay in its L2 from one row tile to the next
        // (bands of 2, 4, 8 and 16 row tiles of any expert took 326, 335, 341 and 341 us for
        // both products of 24008 rows over 128 experts and 896, 870, 900 and 880 for 4096
        // over 8; this 315 and 865).
        const uint32_t l = xcd_tile(blockIdx.x, count * nt * SPLIT);
        const ExpertTile s = f.tiles[l / (nt * SPLIT)];
        const uint32_t first = __builtin_amdgcn_readfirstlane((int)s.first);
        const uint32_t own = __builtin_amdgcn_readfirstlane((int)s.count) * SPLIT;
        const uint32_t in = l - first * nt * SPLIT;
        tm = in % own;
        p.tn = in / own;
        p.rt0 = __builtin_amdgcn_readfirstlane((int)s.rt) + tm * (BM / 16);
        p.rt_end = __builtin_amdgcn_readfirstlane((int)s.rt_end);
        p.half = tm + 1 == own && __builtin_amdgcn_readfirstlane((int)s.half) != 0;
        if (SPLIT > 1 && p.rt0 >= p.rt_end) return false;
        g.st.m = p.rt_end * 16;
        const size_t x = (uint32_t)__builtin_amdgcn_readfirstlane((int)s.expert);
        p.codes += x * f.n16 * f.nkb * FP8_FRAG;
        p.scales += x * (f.n16 / 8) * f.nkb;
        if constexpr (f8_glu(MODE)) {
            p.codes2 += x * f.n16 * f.nkb * FP8_FRAG;
            p.scales2 += x * (f.n16 / 8) * f.nkb;
        }
    }
    return true;
}
// The fragments of column slot c of a tile (NJ slots a wave; GLU: the first half of
// them the gate's, the rest the up weights' same columns); a tile past the last
// repeats it (never stored).
template <int BN, int NJ, int MODE>
__device__ __forceinline__ const uint8_t *f8_columns(const F8Args &f, const F8Place &p, uint32_t c) {
    const uint8_t *base = p.codes;
    uint32_t tile;
    if constexpr (f8_glu(MODE)) {
        if (c % NJ >= NJ / 2) base = p.codes2;
        tile = p.tn * (BN / 32) + c / NJ * (NJ / 2) + c % (NJ / 2);
    } else {
        tile = min(p.tn * (BN / 16) + c, f.n16 - 1);
    }
    return scalar_ptr(base + (size_t)tile * f.nkb * FP8_FRAG);
}
// The block of 128 columns that wave column wc's slots lie in.
template <int BN, int NJ, int MODE>
__device__ __forceinline__ uint32_t f8_block(const F8Args &f, const F8Place &p, uint32_t wc) {
    if constexpr (f8_glu(MODE)) return (p.tn * (BN / 32) + wc * (NJ / 2)) / 8;
    else return min((p.tn * BN + wc * NJ * 16) / 128, f.n16 / 8 - 1);
}

// BM x BN, four waves in 2 x 2, a ring of NSTG stages of 128 depths, the DMA of step k +
// NSTG - 1 issued once every wave has read step k - 1's stage. A stage ends in each wave's
// exponents (256 bytes). Bound by K steps in series of few workgroups (29 x 11003 x 4096
// 11.8 us, 3.9 TB/s; rings of 6, 8 or 10 stages took up to a fifth longer).
template <int BM, int BN, int NSTG>
struct F8Tile {
    static constexpr int MI = BM / 32, NJ = BN / 32;  // 16 x 16 tiles of a wave's piece
    static constexpr int A = BM * 128, W = BN * 128, STAGE = A + W + 4 * 256, CS = BN + 8;
    static constexpr int NP = (BM + BN) / 32;  // pieces of 1 KB a wave moves
    static constexpr int PS = NP + 1;          // DMA instructions a wave
    static constexpr int STORE = BM * CS * 2;
    static constexpr int LDS(int epv) {
        const int st = STORE + (epv == 0 ? EP_FUSED * (BM + BN) * 4 : 0);
        return st > NSTG * STAGE ? st : NSTG * STAGE;
    }
    static_assert(MI <= 4, "a wave's rows share a dword of exponents");
};

template <int BM, int BN, int NSTG, bool BF16, int EPV>
__global__ void __launch_bounds__(256, 2) fp8_tile(F8Args f, EpArgs ep) {
    using T = F8Tile<BM, BN, NSTG>;
    constexpr int MI = T::MI, NJ = T::NJ;
    DArgs g = f.d;
    __shared__ __align__(1024) uint8_t ring[T::LDS(EPV)];
    const int t = threadIdx.x, lane = t % 64, lr = lane % 16, lg = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(t / 64);
    const int wr = wave / 2, wc = wave % 2;
    F8Place pl;
    f8_place<BM, BN, F8_DENSE>(f, g, pl);
    const uint32_t rt0 = pl.rt0, row0 = rt0 * 16, col0 = pl.tn * BN;
    const uint32_t lds0 = lds_addr(ring);
    const uint32_t ksteps = f.nkb, last = ksteps - 1;

    // DMA sources: pieces of 1 KB, the rows' first, then the columns'; tiles past the
    // last repeat it (never stored)
    const uint8_t *src[T::NP];
#pragma unroll
    for (int q = 0; q < T::NP; q++) {
        const uint32_t p = q * 4 + wave, slot = p / 2;
        if (q < MI) src[q] = scalar_ptr(f.q + (size_t)min(rt0 + slot, f.mt16 - 1) * f.nkb * FP8_FRAG + p % 2 * 1024);
        else src[q] = f8_columns<BN, NJ, F8_DENSE>(f, pl, slot - BM / 16) + p % 2 * 1024;
    }
    const uint32_t rtw = rt0 + wr * MI, shift = rtw % 4 * 8;  // the wave's first row tile
    const uint8_t *exps = scalar_ptr(f.e + (size_t)min(rtw / 4, (f.mt16 - 1) / 4) * f.nkb * 64);
    const uint32_t v16 = lane * 16, v4 = lr * 4;
    auto dma = [&](uint32_t step, uint32_t stage) __attribute__((always_inline)) {
        const uint32_t ks = min(step, last), dst = lds0 + stage * T::STAGE;
#pragma unroll
        for (int q = 0; q < T::NP; q++) dma16(src[q] + ks * FP8_FRAG, v16, dst + (q * 4 + wave) * 1024);
        dma4(exps + ks * 64, v4, dst + T::A + T::W + wave * 256);
    };

    float4_t acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++) acc[i][j] = (float4_t){0.f, 0.f, 0.f, 0.f};
    // (a wave's columns share a block of 128)
    const float *scales = pl.scales + (size_t)f8_block<BN, NJ, F8_DENSE>(f, pl, wc) * f.nkb;
    float sl = 0.0f, sw = 0.0f;
    // A row tile's products stay in `part` while the next one's are issued, the last
    // one's into the next step, whose fragment reads they then hide.
    float4_t part[2][NJ];
    auto fold = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NJ; j++) fp8_fold(acc[i][j], part[i & 1][j], sw);
    };
#pragma unroll
    for (int j = 0; j < NJ; j++) part[(MI - 1) & 1][j] = (float4_t){0.f, 0.f, 0.f, 0.f};

    if (ksteps != 0) {
#pragma unroll
        for (int j = 0; j < NSTG - 1; j++) dma(j, j);
    }
    uint32_t stage = 0;
    for (uint32_t ks = 0; ks < ksteps; ks++) {
        if (ks % 64 == 0) sl = scale_lane(scales, ks, f.nkb, lane);
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): this wave has read step ks - 1
        wait_vm<(NSTG - 2) * T::PS>();       // step ks landed
        barrier_lds();
        const uint32_t sb = lds0 + stage * T::STAGE;
        uint32_t ba = sb + wr * MI * FP8_FRAG + lane * 16, bb = sb + T::A + wc * NJ * FP8_FRAG + lane * 16;
        asm volatile("" : "+v"(ba), "+v"(bb));  // constant offsets from here
        int8x_t w[NJ], a[2];
        auto read_a = [&](int i) __attribute__((always_inline)) {
            a[i & 1] = fp8_join(lds_load<u32x4_t>(ba + i * FP8_FRAG), lds_load<u32x4_t>(ba + i * FP8_FRAG + 1024));
        };
#pragma unroll
        for (int j = 0; j < NJ; j++)
            w[j] = fp8_join(lds_load<u32x4_t>(bb + j * FP8_FRAG), lds_load<u32x4_t>(bb + j * FP8_FRAG + 1024));
        read_a(0);
        const uint32_t e = lds_load<uint32_t>(sb + T::A + T::W + wave * 256 + lr * 4) >> shift;
        dma(ks + NSTG - 1, stage == 0 ? NSTG - 1 : stage - 1);
        fold(MI - 1);  // (the step before's)
        sw = scale_at(sl, ks);
#pragma unroll
        for (int i = 0; i < MI; i++) {
            if (i + 1 < MI) read_a(i + 1);
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                switch (i) {  // (an immediate)
                case 0: part[i & 1][j] = fp8_mfma<0>(w[j], a[i & 1], e); break;
                case 1: part[i & 1][j] = fp8_mfma<1>(w[j], a[i & 1], e); break;
                case 2: part[i & 1][j] = fp8_mfma<2>(w[j], a[i & 1], e); break;
                default: part[i & 1][j] = fp8_mfma<3>(w[j], a[i & 1], e); break;
                }
            }
            if (i > 0) fold(i - 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        stage = stage + 1 == NSTG ? 0 : stage + 1;
    }
    fold(MI - 1);
    wait_vm<0>();  // the steps issued past the last
    __syncthreads();

    uint16_t *stg = (uint16_t *)ring;
    float *colv = (float *)(ring + T::STORE), *rowv = colv + EP_FUSED * BN;
    constexpr int CG = BN / 8, RS = 256 / CG, R = BM / RS;
    const int cl = (t % CG) * 8, rl = t / CG;
    EpCols cv;
    if constexpr (EPV == 0) ep_load_vectors<BF16, BM, BN, 256>(g.st, ep, colv, rowv, row0, col0);
    if constexpr (EPV >= 2) ep_cols_load<EPV>(g.col_a, g.col_b, col0 + cl, g.n, cv);
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++)
            dense_stage4<BF16>(g, acc[i][j], stg + (wr * (BM / 2) + i * 16 + lr) * T::CS + wc * (BN / 2) + j * 16 + 4 * lg);
    __syncthreads();
    dense_store<BF16, EPV, BM, BN, R>(g, ep, cv, colv, rowv, stg, T::CS, rl, RS, cl, row0, col0);
}

// BM x 256, eight waves in 2 x 4, two per SIMD, a BM / 2 x 64 piece each. A step of 128
// depths is BM / 128 phases of 64 rows a wave; a phase is a memory slot (its fragment
// reads, its share of a later step's DMA, the folds left over) and a product slot (16
// products, each followed by an earlier one's fold, which issues while the matrix core
// works), each ended by a workgroup barrier. Waves 4-7 run one slot behind waves 0-3, so
// on every SIMD one wave multiplies while the other reads.
// A wave waits for its reads within the memory slot, so after the next one both groups
// have read a part of a stage and it is refilled. BM = 256: two stages, refilled a step and
// a half before the next reading, the columns and the first phase's rows apart from the
// second's; BM = 128: three, refilled two steps before. The DMA is never drained inside
// the loop. What bounds it: LDS, whose reads (192 KB a step of 256 rows, 128 of 128) and
// DMA writes (64, 48) do not overlap, so that a product slot waits for the other group's
// memory slot: 4096 x 14336 x 4096 keeps the matrix cores 54 % busy, at the 1.9 GHz that a
// whole chip's power leaves (2.15 PFLOP/s of a library's 2.6; a tile alone takes 1.3 us a
// step, among others 1.95); 128-row tiles take as long a step (1 us) without the products.
// Columns loaded to registers around LDS, whose wait drains the DMA once a step, took 268
// us for 231.
template <int BM>
struct F8Big {
    static constexpr int BN = 256, NT = 512;
    static constexpr int PH = BM / 128, RT = 4;       // phases, row tiles of a wave's phase
    static constexpr int NS = PH == 2 ? 2 : 3;        // stages
    static constexpr int W = BN * 128, AH = 128 * 128, STAGE = W + PH * AH;  // columns, the phases' rows
    static constexpr int EXP = NS * STAGE;            // the waves' exponents: [stage][phase][wave][256]
    static constexpr int QA = 2, QW = 4;              // pieces of 1 KB a wave moves
    static constexpr int Q0 = QW + QA + 1, Q1 = QA + 1;  // DMA instructions: columns and first rows; second rows
    static constexpr int CS = BN + 8, STG = 128 * CS * 2;  // staged rows of the output tile
    static constexpr int LDS = EXP + NS * PH * 8 * 256;
    static_assert(STG + EP_FUSED * (BM + BN) * 4 <= LDS, "the store exceeds the ring");
};

template <int BM, bool BF16, int EPV, int MODE>
__device__ __forceinline__ void f8_big(const F8Args &f, const EpArgs &ep, const DArgs &g, const F8Place &pl, uint8_t *ring) {
    using T = F8Big<BM>;
    constexpr int PH = T::PH, RT = T::RT, BN = T::BN;
    const int t = threadIdx.x, lane = t % 64, lr = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(t / 64);
    const int wr = wave / 4, wc = wave % 4;
    const uint32_t rt0 = pl.rt0, tn = pl.tn, row0 = rt0 * 16, col0 = tn * BN;
    const uint32_t lds0 = lds_addr(ring);
    const uint32_t ksteps = f.nkb, last = ksteps - 1;

    // (phase h of wave row wr: row tiles rt0 + (wr PH + h) RT ..)
    const uint8_t *pa[PH][T::QA], *pw[T::QW], *pe[PH];
#pragma unroll
    for (int h = 0; h < PH; h++) {
#pragma unroll
        for (int q = 0; q < T::QA; q++) {
            const uint32_t p = q * 8 + wave, slot = p / 2;
            const uint32_t tile = min(rt0 + (slot / RT * PH + h) * RT + slot % RT, f.mt16 - 1);
            pa[h][q] = scalar_ptr(f.q + (size_t)tile * f.nkb * FP8_FRAG + p % 2 * 1024);
        }
        pe[h] = scalar_ptr(f.e + (size_t)min(rt0 / 4 + wr * PH + h, (f.mt16 - 1) / 4) * f.nkb * 64);
    }
#pragma unroll
    for (int q = 0; q < T::QW; q++) {
        const uint32_t p = q * 8 + wave;
        pw[q] = f8_columns<BN, 4, MODE>(f, pl, p / 2) + p % 2 * 1024;
    }
    const uint32_t v16 = lane * 16, v4 = lr * 4;
    auto dma_rows = [&](uint32_t step, int h) __attribute__((always_inline)) {
        const uint32_t ks = min(step, last), st = step % T::NS, dst = lds0 + st * T::STAGE + T::W + h * T::AH + wave * 1024;
#pragma unroll
        for (int q = 0; q < T::QA; q++) dma16(pa[h][q] + ks * FP8_FRAG, v16, dst + q * 8192);
        dma4(pe[h] + ks * 64, v4, lds0 + T::EXP + ((st * PH + h) * 8 + wave) * 256);
    };
    auto dma_first = [&](uint32_t step) __attribute__((always_inline)) {
        const uint32_t ks = min(step, last), dst = lds0 + step % T::NS * T::STAGE + wave * 1024;
#pragma unroll
        for (int q = 0; q < T::QW; q++) dma16(pw[q] + ks * FP8_FRAG, v16, dst + q * 8192);
        dma_rows(step, 0);
    };

    constexpr bool EXACT = MODE == F8_GLU16;
    static_assert(!EXACT || PH == 1, "the f16 fragments' registers");
    float4_t acc[PH * RT][4], part[4];
#pragma unroll
    for (int i = 0; i < PH * RT; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; j++) part[j] = (float4_t){0.f, 0.f, 0.f, 0.f};
    int8x_t a[RT], w[4];
    uint32_t e = 0;
    const float *scales = pl.scales + (size_t)f8_block<BN, 4, MODE>(f, pl, wc) * f.nkb;
    const float *scales2 = f8_glu(MODE) ? pl.scales2 + (size_t)f8_block<BN, 4, MODE>(f, pl, wc) * f.nkb : nullptr;
    float sl = 0.0f, sl2 = 0.0f, sw = 0.0f, sw2 = 0.0f;
    const uint32_t fa = lds0 + T::W + wr * RT * FP8_FRAG + lane * 16, fw = lds0 + wc * 4 * FP8_FRAG + lane * 16;

    // product p of a phase: row tile p / 4, column tile p % 4; folded LAG products later
    constexpr int N = 4 * RT, LAG = 3;
    auto fold = [&](int h, int p) __attribute__((always_inline)) {
        fp8_fold(acc[h * RT + p / 4][p % 4], part[p % 4], f8_glu(MODE) && p % 4 >= 2 ? sw2 : sw);
    };
    auto read_rows = [&](uint32_t step, int h) __attribute__((always_inline)) {
        const uint32_t st = step % T::NS;
        uint32_t b = fa + st * T::STAGE + h * T::AH;
        asm volatile("" : "+v"(b));
#pragma unroll
        for (int i = 0; i < RT; i++)
            a[i] = fp8_join(lds_load<u32x4_t>(b + i * FP8_FRAG), lds_load<u32x4_t>(b + i * FP8_FRAG + 1024));
        e = lds_load<uint32_t>(lds0 + T::EXP + ((st * PH + h) * 8 + wave) * 256 + lane * 4);
    };
    auto read_columns = [&](uint32_t step) __attribute__((always_inline)) {
        uint32_t b = fw + step % T::NS * T::STAGE;
        asm volatile("" : "+v"(b));
#pragma unroll
        for (int j = 0; j < 4; j++)
            w[j] = fp8_join(lds_load<u32x4_t>(b + j * FP8_FRAG), lds_load<u32x4_t>(b + j * FP8_FRAG + 1024));
    };
    auto mem_end = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0xC07F);            // lgkmcnt(0): this wave's reads are done
        wait_vm<PH == 2 ? T::Q0 + T::Q1 : T::Q0>();    // what the next memory slot reads has landed
        barrier_lds();
        __builtin_amdgcn_sched_barrier(0);
    };
    auto mul = [&](auto h_c) __attribute__((always_inline)) {
        constexpr int H = decltype(h_c)::value;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int p = 0; p < N; p++) {
            switch (p / 4) {  // (an immediate)
            case 0: part[p % 4] = fp8_mfma<0>(w[p % 4], a[0], e); break;
            case 1: part[p % 4] = fp8_mfma<1>(w[p % 4], a[1], e); break;
            case 2: part[p % 4] = fp8_mfma<2>(w[p % 4], a[2], e); break;
            default: part[p % 4] = fp8_mfma<3>(w[p % 4], a[3], e); break;
            }
            if (p >= LAG) fold(H, p - LAG);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        barrier_lds();
        __builtin_amdgcn_sched_barrier(0);
    };
    // F8_GLU16: the same products of the codes' f16 values, which drop nothing: four
    // instructions for a block's depths, four column tiles side by side, each followed by its
    // share of the next row tile's widening and of the last one's folds, which issue while the
    // matrix core works.
    half8_t a16[2][4], w16[EXACT ? 4 : 1][4];
    float4_t p16[2][4];
    float s16[2][2];  // the row's scale times the gate's and the up weights', by p16's row tile
    if constexpr (EXACT) {
#pragma unroll
        for (int j = 0; j < 4; j++) p16[(RT - 1) & 1][j] = (float4_t){0.f, 0.f, 0.f, 0.f};
        s16[(RT - 1) & 1][0] = s16[(RT - 1) & 1][1] = 0.0f;
    }
    auto fold16 = [&](int i, int j, int v) __attribute__((always_inline)) {
        acc[i][j][v] = __builtin_fmaf(p16[i & 1][j][v], s16[i & 1][j / 2], acc[i][j][v]);
    };
    auto mul_exact = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < RT; i++) {
#pragma unroll
            for (int c = 0; c < 4; c++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float4_t z = {0.f, 0.f, 0.f, 0.f};
                    if (i == 0) {
                        if (j == 0) a16[0][c] = fp8_to_f16(a[0][2 * c], a[0][2 * c + 1]);
                        w16[j][c] = fp8_to_f16(w[j][2 * c], w[j][2 * c + 1]);
                    }
                    p16[i & 1][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w16[j][c], a16[i & 1][c], c == 0 ? z : p16[i & 1][j], 0, 0, 0);
                    if (i + 1 < RT) {
                        const half2_t x = fp8_pair_f16(a[i + 1][2 * c + j / 2], j % 2);
                        a16[(i + 1) & 1][c][2 * j] = x[0];
                        a16[(i + 1) & 1][c][2 * j + 1] = x[1];
                    }
                    if (i > 0) fold16(i - 1, c, j);
                    __builtin_amdgcn_sched_barrier(0);
                }
            const float rs = __uint_as_float((e >> (8 * i) & 0xFF) << 23);
            s16[i & 1][0] = sw * rs;
            s16[i & 1][1] = sw2 * rs;
        }
        __builtin_amdgcn_s_setprio(0);
        barrier_lds();
        __builtin_amdgcn_sched_barrier(0);
    };
    auto rest = [&](int h) __attribute__((always_inline)) {
        if constexpr (EXACT) {
#pragma unroll
            for (int p = 0; p < 16; p++) fold16(RT - 1, p / 4, p % 4);
        } else {
#pragma unroll
            for (int p = N - LAG; p < N; p++) fold(h, p);
        }
    };
    constexpr std::integral_constant<int, 0> h0;
    constexpr std::integral_constant<int, PH - 1> h1;

    if (ksteps != 0) {
        dma_first(0);
        if constexpr (PH == 2) dma_rows(0, 1);
        dma_first(1);
        wait_vm<PH == 2 ? T::Q0 + T::Q1 : T::Q0>();  // step 0's columns and first rows landed
        barrier_lds();
        if (wr == 1) barrier_lds();  // waves 4-7 run one slot behind
        for (uint32_t ks = 0; ks < ksteps; ks++) {
            read_columns(ks);
            read_rows(ks, 0);
            if constexpr (PH == 2) dma_rows(ks + 1, 1);
            else dma_first(ks + 2);
            rest(PH - 1);  // (the step before's)
            if (ks % 64 == 0) {
                sl = scale_lane(scales, ks, f.nkb, lane);
                if constexpr (f8_glu(MODE)) sl2 = scale_lane(scales2, ks, f.nkb, lane);
            }
            sw = scale_at(sl, ks);
            if constexpr (f8_glu(MODE)) sw2 = scale_at(sl2, ks);
            mem_end();
            if constexpr (EXACT) mul_exact();
            else mul(h0);
            if constexpr (PH == 2) {
                read_rows(ks, 1);
                dma_first(ks + 2);
                rest(0);
                mem_end();
                mul(h1);
            }
        }
        if (wr == 0) barrier_lds();
        rest(PH - 1);
        wait_vm<0>();  // the steps issued past the last
    }
    __syncthreads();

    // (the thread's place, opaque: the loop then keeps none of what derives from
    // it for the store)
    int to = t;
    asm volatile("" : "+v"(to));
    const int lro = to % 16, lgo = to % 64 / 16;
    if constexpr (f8_glu(MODE)) {
        glu_store<PH * RT, 4>(f, acc, (uint32_t *)ring, rt0, pl.rt_end, tn, wr, wc, to % 64);
        return;
    }
    if constexpr (MODE == F8_GROUPED) {  // f32 parts, as they are
        float *dst = (float *)g.st.dst;
#pragma unroll
        for (int i = 0; i < PH * RT; i++) {
            const uint32_t row = row0 + (wr * PH * RT + i) * 16 + lro;
            if (row >= g.st.m) continue;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t col = col0 + wc * 64 + j * 16 + 4 * lgo;
                float *p = dst + (size_t)row * g.n + col;
                if (g.n % 4 == 0 && col < g.n) {
                    *(float4_t *)p = acc[i][j];
                } else {
#pragma unroll
                    for (int v = 0; v < 4; v++)
                        if (col + v < g.n) p[v] = acc[i][j][v];
                }
            }
        }
        return;
    }
    constexpr int RH = 16 * RT;  // rows of a wave's phase
    uint16_t *stg = (uint16_t *)ring;
    float *colv = (float *)(ring + T::STG), *rowv = colv + EP_FUSED * BN;
    const int cl = (to % 32) * 8, rl = to / 32;
    EpCols cv;
    if constexpr (EPV == 0) ep_load_vectors<BF16, BM, BN, T::NT>(g.st, ep, colv, rowv, row0, col0);
    if constexpr (EPV >= 2) ep_cols_load<EPV>(g.col_a, g.col_b, col0 + cl, g.n, cv);
    auto store_phase = [&](int h) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                dense_stage4<BF16>(g, acc[h * RT + i][j], stg + (wr * RH + i * 16 + lro) * T::CS + wc * 64 + j * 16 + 4 * lgo);
        __syncthreads();
#pragma unroll 1
        for (int v = 0; v < 2; v++) {
            const uint32_t r = (v * PH + h) * RH;
            dense_store<BF16, EPV, BM, BN, RT>(g, ep, cv, colv, rowv + r, stg + v * RH * T::CS, T::CS, rl, 16, cl, row0 + r,
                                               col0);
        }
    };
    // (two calls, not a loop: a loop left rolled would index the accumulators at run
    // time, and keep them in memory)
    store_phase(0);
    if constexpr (PH == 2) {
        __syncthreads();
        store_phase(1);
    }
}

template <bool BF16, int EPV, int MODE>
__global__ void __launch_bounds__(512, 2) fp8_big(F8Args f, EpArgs ep) {
    __shared__ __align__(1024) uint8_t ring[F8Big<256>::LDS > F8Big<128>::LDS ? F8Big<256>::LDS : F8Big<128>::LDS];
    DArgs g = f.d;
    F8Place pl;
    if (!f8_place<MODE == F8_GLU16 ? 128 : 256, 256, MODE>(f, g, pl)) return;
    if constexpr (MODE == F8_GLU16) {
        f8_big<128, BF16, EPV, MODE>(f, ep, g, pl, ring);
    } else {
        if (pl.half) f8_big<128, BF16, EPV, MODE>(f, ep, g, pl, ring);
        else f8_big<256, BF16, EPV, MODE>(f, ep, g, pl, ring);
    }
}

// Where the last round of 256-row tiles would leave half of the compute units or more
// without one, its tiles are split into halves of 128 rows, two workgroups each.
uint32_t f8_full_tiles(size_t m, size_t n) {
    const size_t tiles = ((m + 255) / 256) * ((n + 255) / 256), cus = (size_t)device_cus();
    return (uint32_t)(tiles % cus * 2 <= cus ? tiles / cus * cus : tiles);
}
template <bool BF16>
hipError_t launch_f8_big(F8Args f, bool halves, const EpArgs &ep, int epv, hipStream_t s) {
    const size_t nt = (f.d.n + 255) / 256, tiles = (f.d.m + (size_t)255) / 256 * nt;
    if (!launchable(2 * tiles, 512)) return hipErrorInvalidConfiguration;
    f.full = halves ? 0 : f8_full_tiles(f.d.m, f.d.n);
    const dim3 grid((uint32_t)(f.full == 0 ? (f.d.m + 127) / 128 * nt : f.full + 2 * (tiles - f.full))), block(512);
    switch (epv) {
    case 1: hipLaunchKernelGGL((fp8_big<BF16, 1, F8_DENSE>), grid, block, 0, s, f, ep); break;
    case 2: hipLaunchKernelGGL((fp8_big<BF16, 2, F8_DENSE>), grid, block, 0, s, f, ep); break;
    case 3: hipLaunchKernelGGL((fp8_big<BF16, 3, F8_DENSE>), grid, block, 0, s, f, ep); break;
    default: hipLaunchKernelGGL((fp8_big<BF16, 0, F8_DENSE>), grid, block, 0, s, f, ep); break;
    }
    return hipGetLastError();
}

template <int BM, int BN, int NSTG, bool BF16>
hipError_t launch_f8_tile(const F8Args &f, const EpArgs &ep, int epv, hipStream_t s) {
    const size_t tiles = (size_t)((f.d.m + BM - 1) / BM) * ((f.d.n + BN - 1) / BN);
    if (!launchable(tiles, 256)) return hipErrorInvalidConfiguration;
    const dim3 grid((uint32_t)tiles), block(256);
    switch (epv) {
    case 1: hipLaunchKernelGGL((fp8_tile<BM, BN, NSTG, BF16, 1>), grid, block, 0, s, f, ep); break;
    case 2: hipLaunchKernelGGL((fp8_tile<BM, BN, NSTG, BF16, 2>), grid, block, 0, s, f, ep); break;
    case 3: hipLaunchKernelGGL((fp8_tile<BM, BN, NSTG, BF16, 3>), grid, block, 0, s, f, ep); break;
    default: hipLaunchKernelGGL((fp8_tile<BM, BN, NSTG, BF16, 0>), grid, block, 0, s, f, ep); break;
    }
    return hipGetLastError();
}

// The tile for an m x n x k product: the least of a cost in us, steps of 128 depths x
// (full rounds of the compute units x occupancy, each at `full`, and a last round that
// grows from `one` to `full`) + `fixed`, the constants measured on 256 compute units
// (large grids draw the clock down, so `full` is also what the power allows). Measured
// (us with the rows' quantization, bf16, weights from memory, tiles of 256 rows ended by
// halves / 128x256 / 64x128 / 64x64): 4096 x 14336 x 4096 241 / 279 / 361 / 431; 2048 x
// 14336 x 4096 131 / 159 / 190 / 222; 512 x 14336 x 4096 45 / 44 / 60 / 68; 1000 x 5000 x
// 3000 34 / 34 / 38 / 40; 512 x 4096 x 14336 107 / 107 / 64 / 68; 2048^3 28 / 28 / 23 / 27;
// 128 x 14336 x 4096 35 / 34 / 22 / 22; 300 x 1536 x 7168 50 / 50 / 31 / 23 (32x64: 21).
struct F8Cost {
    uint32_t bm, bn, occ;
    float one, full, fixed;
};
constexpr F8Cost F8_TILES[] = {{256, 256, 1, 1.32f, 1.95f, 8.0f},
                               {128, 256, 1, 0.90f, 1.25f, 6.0f},
                               {64, 128, 2, 0.49f, 0.735f, 4.5f},
                               {64, 64, 2, 0.37f, 0.465f, 4.0f},
                               {32, 64, 3, 0.27f, 0.56f, 4.0f}};
int f8_pick(size_t m, size_t n, size_t steps) {
    const size_t cus = (size_t)device_cus();
    int best = 0;
    float least = 0.0f;
    for (int i = 0; i < 5; i++) {
        const F8Cost &c = F8_TILES[i];
        const size_t tiles = ((m + c.bm - 1) / c.bm) * ((n + c.bn - 1) / c.bn), cap = cus * c.occ;
        const size_t rounds = tiles / cap, rest = tiles % cap, one = c.occ > 1 ? cus : 0;
        float t = (float)rounds * c.full;
        if (i == 0 && rest * 2 <= cap) t += rest != 0 ? F8_TILES[1].one : 0.0f;  // (halves: f8_full_tiles)
        else if (rest != 0) t += c.one + (rest > one ? (c.full - c.one) * (float)(rest - one) / (float)(cap - one) : 0.0f);
        t = t * (float)steps + c.fixed;
        if (i == 0 || t < least) {
            best = i;
            least = t;
        }
    }
    return best;
}
template <bool BF16>
hipError_t launch_f8_shape(const F8Args &f, const EpArgs &ep, int epv, hipStream_t s) {
    switch (f8_pick(f.d.m, f.d.n, f.nkb)) {
    case 0: return launch_f8_big<BF16>(f, false, ep, epv, s);
    case 1: return launch_f8_big<BF16>(f, true, ep, epv, s);
    case 2: return launch_f8_tile<64, 128, 3, BF16>(f, ep, epv, s);
    case 3: return launch_f8_tile<64, 64, 4, BF16>(f, ep, epv, s);
    default: return launch_f8_tile<32, 64, 4, BF16>(f, ep, epv, s);
    }
}

}  // namespace

TileDims fp8_gemm_tile(size_t m, size_t n, size_t k) {
    const F8Cost &c = F8_TILES[f8_pick(m, n, (k + 127) / 128)];
    return {c.bm, c.bn};
}

hipError_t launch_fp8_gemm(const Fp8Mat &w, size_t m, uint16_t *dst, Fp8Rows a, const EpArgs &ep, bool bf16,
                           hipStream_t s) {
    F8Args f = {};
    DArgs &g = f.d;
    const EpPick pk = pick_ep(ep);
    g.st = {dst, (long)w.n, 1, (uint32_t)m, w.n, 0.0f, 0};
    g.beta = 1.0f;
    g.m = (uint32_t)m;
    g.n = w.n;
    g.col_a = pk.a;
    g.col_b = pk.b;
    g.act = pk.act;
    g.act_alpha = pk.alpha;
    f.q = a.q;
    f.e = a.e;
    f.w = w.codes;
    f.sw = w.scales;
    f.mt16 = (uint32_t)((m + 15) / 16);
    f.n16 = w.n16;
    f.nkb = w.nkb;
    return bf16 ? launch_f8_shape<true>(f, ep, pk.v, s) : launch_f8_shape<false>(f, ep, pk.v, s);
}

hipError_t launch_fp8_grouped(const Fp8Mat &w, const Fp8Mat *up, uint32_t act, const ExpertPlan &p, Fp8Rows a, Fp8Rows h,
                              float *dst, bool exact, hipStream_t s) {
    F8Args f = {};
    DArgs &g = f.d;
    g.st.dst = (uint16_t *)dst;
    g.n = w.n;
    f.q = a.q;
    f.e = a.e;
    f.w = w.codes;
    f.sw = w.scales;
    f.mt16 = p.max_rows / 16;
    f.n16 = w.n16;
    f.nkb = w.nkb;
    f.head = p.head;
    f.tiles = p.tiles;
    const uint32_t cols = up ? 128 : 256;
    const size_t tiles = (size_t)p.max_tiles * (up && exact ? 2 : 1) * ((w.n + cols - 1) / cols);
    if (!launchable(tiles, 512)) return hipErrorInvalidConfiguration;
    const dim3 grid((uint32_t)tiles), block(512);
    if (tiles == 0) return hipSuccess;
    if (up) {
        f.w2 = up->codes;
        f.sw2 = up->scales;
        f.act = act;
        f.hq = h.q;
        f.he = h.e;
        f.hkb = w.n16 / 8;
    }
    if (up && exact) hipLaunchKernelGGL((fp8_big<false, 1, F8_GLU16>), grid, block, 0, s, f, EpArgs{});
    else if (up) hipLaunchKernelGGL((fp8_big<false, 1, F8_GLU>), grid, block, 0, s, f, EpArgs{});
    else hipLaunchKernelGGL((fp8_big<false, 1, F8_GROUPED>), grid, block, 0, s, f, EpArgs{});
    return hipGetLastError();
}

}  // namespace smg
