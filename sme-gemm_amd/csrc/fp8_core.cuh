// What the 8-bit floating-point kernels share: the rows' quantization and the
// product of two fragments.
//
// A row's block of 128 depths is scaled by 2^e, the least power of two (2^-126 at
// least) that takes its largest finite magnitude to 448, e4m3's largest, or less,
// and rounded to e4m3, ties to even: with a power of two the scaling is exact, so
// the rounding is the only one, and as a floating-point format loses nothing to a
// coarser scale but the smallest of its subnormals, the rounding error is what an
// f32 scale's would be. The exponent byte e + 127 is what the matrix instructions'
// scale operand takes, so the rows' scales cost no instruction.
#pragma once

#include "fp8.h"
#include "lds_dma.cuh"

namespace smg {

namespace {

typedef int int8x_t __attribute__((ext_vector_type(8)));  // a fragment: 32 bytes a lane
typedef short s16x2_t __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// The exponent byte for a block whose largest finite magnitude has the f32 bits
// `amax`: floor(log2(amax)) - 8, one more past 448 / 256 = 1.75, at least 1 - 127.
__device__ __forceinline__ uint32_t fp8_exp_byte(uint32_t amax) {
    const uint32_t e = (amax + 0x1FFFFFu) >> 23;
    return e < 9 ? 1u : e - 8;
}

// Largest of two packed magnitudes' bits.
__device__ __forceinline__ uint32_t max_mag2(uint32_t m, uint32_t x) {
    const u16x2_t a = __builtin_bit_cast(u16x2_t, m), b = __builtin_bit_cast(u16x2_t, x & 0x7FFF7FFFu);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(a, b));
}

// 32 consecutive depths of a row (16 dwords of two 16-bit values) to 32 codes.
// The block's other three quarters are in the lanes 16, 32 and 48 on; every lane
// gets the block's exponent byte. Infinities become NaN and, as NaN, do not count
// for the scale.
template <bool BF16>
__device__ __forceinline__ uint32_t fp8_quant32(uint32_t (&w)[16], int8x_t &q) {
    constexpr uint32_t INF = BF16 ? 0x7F80u : 0x7C00u;
    uint32_t m2 = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) m2 = max_mag2(m2, w[i]);
    uint32_t m = max(m2 & 0xFFFFu, m2 >> 16);
    if (__builtin_amdgcn_ballot_w64(m >= INF)) {  // a value that is not finite
        m = 0;
#pragma unroll
        for (int i = 0; i < 16; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t b = (w[i] >> (16 * h)) & 0x7FFFu;
                if (b >= INF) w[i] |= 0x7FFFu << (16 * h);  // NaN
                else m = max(m, b);
            }
    }
    m = max(m, (uint32_t)__shfl_xor((int)m, 16));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32));
    const uint32_t e = fp8_exp_byte(__float_as_uint(to_f32<BF16>((uint16_t)m)));
    const float scale = __uint_as_float(e << 23);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        s16x2_t r = {0, 0};
        if constexpr (BF16) {
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, w[2 * i]), scale, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, w[2 * i + 1]), scale, true);
        } else {
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(half2_t, w[2 * i]), scale, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(half2_t, w[2 * i + 1]), scale, true);
        }
        q[i] = __builtin_bit_cast(int, r);
    }
    return e;
}

// 16 weight columns x 16 rows over 128 depths. The instruction adds up groups of 8
// consecutive depths aligned at the product of the largest exponent, dropping what of
// the others lies 2^-13 below it, and the groups in f32: a group loses less than 7 x
// 2^-13 of its largest product, where f16 products of the same codes would lose
// nothing at half the rate. On normally distributed data that is 2^-16 of a sum (its
// 2-norm), under the f16 store's 2^-12. Lane l gets columns 4 (l / 16) ..
// + 3 of row l % 16, the codes' sums times the rows' scales (byte SEL of `e` in
// row l % 16's lanes), from zero.
template <int SEL>
__device__ __forceinline__ float4_t fp8_mfma(const int8x_t &w, const int8x_t &a, uint32_t e) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, (float4_t){0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0x7F7F7F7F, SEL,
                                                            (int)e);
}

// Two codes (a dword's low or high half) as f16 values, exact; eight (two dwords).
__device__ __forceinline__ half2_t fp8_pair_f16(uint32_t a, bool high) {
    return high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
}
__device__ __forceinline__ half8_t fp8_to_f16(uint32_t a, uint32_t b) {
    const half2_t x = fp8_pair_f16(a, false), y = fp8_pair_f16(a, true), z = fp8_pair_f16(b, false), w = fp8_pair_f16(b, true);
    return (half8_t){x[0], x[1], y[0], y[1], z[0], z[1], w[0], w[1]};
}
// The codes' sums of a fragment by f16 products, which drop nothing of them (2^-27 of a sum's
// 2-norm on the same data), at half the rate and after widening: for kernels that wait for
// memory and whose results are rounded to codes again (where a sum a little off may cross
// the border of two).
__device__ __forceinline__ float4_t fp8_mfma_f16(const int8x_t &w, const half8_t (&a)[4]) {
    float4_t c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp8_to_f16(w[2 * i], w[2 * i + 1]), a[i], c, 0, 0, 0);
    return c;
}

// A hidden value act(g) u, act silu or the tanh form of gelu: g / (1 + e^-y) by the
// hardware's 2^x and reciprocal (2^-23 each). past: e^-y is beyond 2^100 or so, and the
// value is glu_far's: g e^y u, a half of the power with either factor, as g e^y alone may
// be too small for an f32 where u is large. (An f64 branch for each of a lane's values instead cost the products of few
// rows a sixth of their time, in registers: 296 assignments of 4096 to 1792, 324 us
// against 277.)
__device__ __forceinline__ float glu_power(bool gelu, float g) {  // -log2 of e^y
    return (gelu ? -2.0f * 0.7978845608028654f * 1.4426950408889634f * (g + 0.044715f * g * g * g) : -1.4426950408889634f * g);
}
__device__ __forceinline__ float glu_near(bool gelu, float g, float u, bool &past) {
    const float e = __builtin_amdgcn_exp2f(glu_power(gelu, g));
    past = e >= 0x1p100f;
    return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}
__device__ __forceinline__ float glu_far(bool gelu, float g, float u) {
    const float h = __builtin_amdgcn_exp2f(-0.5f * glu_power(gelu, g));
    return (g * h) * (h * u);
}

// acc += part * sw, the weight block's scale: one f32 rounding an element.
__device__ __forceinline__ void fp8_fold(float4_t &acc, const float4_t &part, float sw) {
#pragma unroll
    for (int v = 0; v < 4; v++) acc[v] = __builtin_fmaf(part[v], sw, acc[v]);
}

__device__ __forceinline__ int8x_t fp8_join(const u32x4_t &lo, const u32x4_t &hi) {
    return __builtin_bit_cast(int8x_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
__device__ __forceinline__ int8x_t fp8_join(const uint4 &lo, const uint4 &hi) {
    return (int8x_t){(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}

}  // namespace

}  // namespace smg
