// Launch interface of the 8-bit floating-point products (fp8_gemv.hip,
// fp8_gemm.hip). Internal to the library.
//
// Launches whose threads would pass 2^32 - 1 (which run their number modulo 2^32, without
// an error) are refused with hipErrorInvalidConfiguration, or split.
//
// Weights are e4m3 codes with an f32 scale for each 128 x 128 block of a matrix
// of n columns and k depths (a checkpoint's [n][k] codes and [n/128][k/128]
// scales). On the device the codes are in the order the matrix instructions read
// them: 16 columns x 128 depths make a fragment of 2 KB, 32 bytes a lane (column
// lane % 16, depths 32 (lane / 16) ..), its two 16-byte halves 1 KB apart, so that
// a wave's load is contiguous and a tile's DMA linear:
//   code (j, d) of a matrix: ((j / 16) * nkb + d / 128) * 2048
//                            + (d % 32 / 16) * 1024 + ((d % 128 / 32) * 16 + j % 16) * 16 + d % 16
// Columns are padded to a multiple of 128 and depths to a multiple of 128 with
// zeros. Activations are quantized into the same fragments, 16 rows each, with an
// exponent byte for each row and block of 128 depths (fp8_core.cuh).
#pragma once

#include "kernels.h"

namespace smg {

constexpr uint32_t FP8_BLOCK = 128;      // depths (and columns) of a scale
constexpr uint32_t FP8_FRAG = 2048;      // bytes of 16 columns (rows) x 128 depths
inline bool launchable(size_t blocks, size_t threads) { return blocks * threads < (size_t)1 << 32; }

// One or several matrices of one shape (a mixture's experts), one after another.
struct Fp8Mat {
    const uint8_t *codes;  // [mats][n16][nkb][FP8_FRAG]
    const float *scales;   // [mats][n16 / 8][nkb]
    uint32_t n, k;
    uint32_t n16;          // column tiles, a multiple of 8
    uint32_t nkb;          // blocks of 128 depths
    uint32_t mats;
    size_t code_bytes() const { return (size_t)n16 * nkb * FP8_FRAG; }       // of one matrix
    size_t scale_count() const { return (size_t)(n16 / 8) * nkb; }
};
inline Fp8Mat fp8_shape(uint32_t n, uint32_t k, uint32_t mats) {
    return {nullptr, nullptr, n, k, (n + 127) / 128 * 8, (k + 127) / 128, mats};
}

// Codes and scales as a checkpoint holds them (device memory: [mats][n][k] and
// [mats][ceil(n/128)][nkb]) into the device order above.
hipError_t launch_fp8_pack(const Fp8Mat &w, const uint8_t *src, uint8_t *codes, hipStream_t s);

// Rows of activations quantized into fragments: q [ceil(rows/16)][nkb][FP8_FRAG],
// then the exponent bytes [ceil(rows/64)][nkb][16 rows][4 row tiles].
struct Fp8Rows {
    uint8_t *q, *e;
    static size_t q_bytes(size_t rows, size_t nkb) { return (rows + 15) / 16 * nkb * FP8_FRAG; }
    static size_t bytes(size_t rows, size_t nkb) { return q_bytes(rows, nkb) + (rows + 63) / 64 * nkb * 64; }
    static Fp8Rows at(void *p, size_t rows, size_t nkb) {
        return {(uint8_t *)p, (uint8_t *)p + q_bytes(rows, nkb)};
    }
};
hipError_t launch_fp8_quant(const uint16_t *x, size_t rows, size_t k, bool bf16, Fp8Rows out, hipStream_t s);

// C [m][n] = ep(to16(A W)): the rows' quantization and the product. scratch:
// fp8_scratch_bytes(w, m) bytes (0 where the product quantizes its rows itself).
size_t fp8_scratch_bytes(const Fp8Mat &w, size_t m);
hipError_t launch_fp8_matmul(const Fp8Mat &w, size_t m, uint16_t *dst, const uint16_t *lhs, const EpArgs &ep, bool bf16,
                             void *scratch, hipStream_t s);

// The product of quantized rows (fp8_gemm.hip), and its output tile.
TileDims fp8_gemm_tile(size_t m, size_t n, size_t k);
hipError_t launch_fp8_gemm(const Fp8Mat &w, size_t m, uint16_t *dst, Fp8Rows a, const EpArgs &ep, bool bf16,
                           hipStream_t s);

}  // namespace smg
