// 8-bit floating-point products of few rows, the rows' quantization and the
// weights' packing.
//
// fp8_gemv: C = ep(to16(sum_b scale_b (q w_b))) for few rows in one launch. A workgroup
// of eight waves owns 16 (or 32) columns, wave w blocks w, w + 8, .. of K; each
// loads its weight fragments (1 KB a wave load, streamed past the caches), and
// quantizes the same blocks of the rows in registers while they are in flight (a
// lane 32 depths of a row, the block's largest magnitude by two lane exchanges),
// so that neither a pass over the activations nor a barrier comes first. The waves'
// partial sums meet in LDS in fixed order. Up to 64 rows of few columns are quantized by a
// pass first and multiplied in the same way (fp8_gemv_rows).
// What bounds it: reading the weights once (one row, weights from HBM: 16.8 MB of a 4096 x
// 4096 layer in 5.1 us, 58.7 MB of 14336 x 4096 in 11.4, 5.1 TB/s).
#include <algorithm>

#include "fp8_core.cuh"

namespace smg {

namespace {

constexpr int GV_NT = 512, GV_W = GV_NT / 64;  // threads, waves

struct GvArgs {
    const uint8_t *codes;
    const float *scales;
    const uint16_t *lhs;
    uint16_t *dst;
    uint32_t m, n, k, nkb, n16;
};

// The 32 depths d .. of row `row` (zeros outside m x k).
template <bool VEC>
__device__ __forceinline__ void load_row32(rsrc_t r, uint32_t row, uint32_t m, uint32_t k, uint32_t d, uint32_t (&w)[16]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint4 x = load_row8(r, row, m, k, d + 8 * i, VEC);
        w[4 * i] = x.x;
        w[4 * i + 1] = x.y;
        w[4 * i + 2] = x.z;
        w[4 * i + 3] = x.w;
    }
}

// The waves' shares added up in order, and the store.
template <int RT, int CT, bool BF16>
__device__ __forceinline__ void gv_join(const GvArgs &g, const EpArgs &ep, uint32_t tile0, int t, int wave, int lane,
                                        const float4_t (&acc)[RT][CT], float4_t (*part)[GV_W][64]) {
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int c = 0; c < CT; c++) part[i * CT + c][wave][lane] = acc[i][c];
    __syncthreads();
    // thread: column t % 16 of row t / 16 of a tile
#pragma unroll
    for (int p = t / 256; p < RT * CT; p += GV_NT / 256) {
        const uint32_t rl = t % 256 / 16, cl = t % 16, row = p / CT * 16 + rl, col = (tile0 + p % CT) * 16 + cl;
        if (row >= g.m || col >= g.n) continue;
        const float *q = (const float *)&part[p][0][(cl / 4) * 16 + rl] + cl % 4;
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < GV_W; w++) x += q[w * 256];
        g.dst[(size_t)row * g.n + col] = finish<BF16>(ep, x, row, col, g.n);
    }
}

// RT tiles of 16 rows, CT of 16 columns, U blocks of K a wave holds in flight.
template <int RT, int CT, int U, bool BF16, bool VEC>
__global__ void __launch_bounds__(GV_NT, 4) fp8_gemv(GvArgs g, EpArgs ep) {
    __shared__ float4_t part[RT * CT][GV_W][64];
    const int t = threadIdx.x, lane = t % 64, lr = lane % 16, lg = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(t / 64);
    const uint32_t tile0 = xcd_tile(blockIdx.x, gridDim.x) * CT;
    const rsrc_t rw = make_rsrc(g.codes + (size_t)tile0 * g.nkb * FP8_FRAG, CT * g.nkb * FP8_FRAG);
    const rsrc_t ra = make_rsrc(g.lhs, g.m * g.k * 2u);
    const rsrc_t rs = make_rsrc(g.scales + (size_t)(tile0 / 8) * g.nkb, g.nkb * 4u);  // (CT tiles share a block)
    float4_t acc[RT][CT];
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int c = 0; c < CT; c++) acc[i][c] = (float4_t){0.f, 0.f, 0.f, 0.f};
    for (uint32_t kb0 = wave; kb0 < g.nkb; kb0 += GV_W * U) {
        uint32_t a[U][RT][16];
        uint4 w[U][CT][2];
        float sw[U];
        // (blocks past the last read zeros)
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < RT; i++)
                load_row32<VEC>(ra, i * 16 + lr, g.m, g.k, (kb0 + u * GV_W) * FP8_BLOCK + 32 * lg, a[u][i]);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t kb = kb0 + u * GV_W;
#pragma unroll
            for (int c = 0; c < CT; c++) {
                const uint32_t off = kb < g.nkb ? (c * g.nkb + kb) * FP8_FRAG + lane * 16 : OOB;
                w[u][c][0] = bload16_nt(rw, off);
                w[u][c][1] = bload16_nt(rw, off + 1024);
            }
            sw[u] = __uint_as_float(bload4(rs, kb * 4));
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < RT; i++) {
                int8x_t q;
                const uint32_t e = fp8_quant32<BF16>(a[u][i], q);
#pragma unroll
                for (int c = 0; c < CT; c++)
                    fp8_fold(acc[i][c], fp8_mfma<0>(fp8_join(w[u][c][0], w[u][c][1]), q, e), sw[u]);
            }
    }
    gv_join<RT, CT, BF16>(g, ep, tile0, t, wave, lane, acc, part);
}

// Up to 64 rows that are quantized already (r, their fragments): 16 columns, the same split,
// the rows' fragments from the caches. A dword of exponents serves the four row tiles.
template <int RT, bool BF16>
__global__ void __launch_bounds__(GV_NT, 4) fp8_gemv_rows(GvArgs g, Fp8Rows r, EpArgs ep) {
    constexpr int U = 2;  // blocks of K a wave holds in flight
    __shared__ float4_t part[RT][GV_W][64];
    const int t = threadIdx.x, lane = t % 64, lr = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(t / 64);
    const uint32_t tile = xcd_tile(blockIdx.x, gridDim.x), mt16 = (g.m + 15) / 16;
    const rsrc_t rw = make_rsrc(g.codes + (size_t)tile * g.nkb * FP8_FRAG, g.nkb * FP8_FRAG);
    const rsrc_t rq = make_rsrc(r.q, mt16 * g.nkb * FP8_FRAG), re = make_rsrc(r.e, g.nkb * 64u);
    const rsrc_t rs = make_rsrc(g.scales + (size_t)(tile / 8) * g.nkb, g.nkb * 4u);
    float4_t acc[RT][1];
#pragma unroll
    for (int i = 0; i < RT; i++) acc[i][0] = (float4_t){0.f, 0.f, 0.f, 0.f};
    for (uint32_t kb0 = wave; kb0 < g.nkb; kb0 += GV_W * U) {
        uint4 q[U][RT][2], w[U][2];
        uint32_t e[U];
        float sw[U];
        // (blocks past the last, and row tiles past it, read zeros)
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t kb = kb0 + u * GV_W, off = kb * FP8_FRAG + lane * 16;
            w[u][0] = bload16_nt(rw, off);
            w[u][1] = bload16_nt(rw, off + 1024);
            sw[u] = __uint_as_float(bload4(rs, kb * 4));
            e[u] = bload4(re, kb * 64 + lr * 4);
#pragma unroll
            for (int i = 0; i < RT; i++) {
                const uint32_t at = kb < g.nkb ? i * g.nkb * FP8_FRAG + off : OOB;
                q[u][i][0] = bload16(rq, at);
                q[u][i][1] = bload16(rq, at + 1024);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int8x_t x = fp8_join(w[u][0], w[u][1]);
#pragma unroll
            for (int i = 0; i < RT; i++) {
                const int8x_t y = fp8_join(q[u][i][0], q[u][i][1]);
                float4_t p;
                switch (i) {  // (an immediate)
                case 0: p = fp8_mfma<0>(x, y, e[u]); break;
                case 1: p = fp8_mfma<1>(x, y, e[u]); break;
                case 2: p = fp8_mfma<2>(x, y, e[u]); break;
                default: p = fp8_mfma<3>(x, y, e[u]); break;
                }
                fp8_fold(acc[i][0], p, sw[u]);
            }
        }
    }
    gv_join<RT, 1, BF16>(g, ep, tile, t, wave, lane, acc, part);
}

// A wave per (16 rows, block of 128 depths). Bound by the rows' bytes: 4096 x 4096 bf16 (34
// MB read, 17 written) in 12 us.
template <bool BF16, bool VEC>
__global__ void __launch_bounds__(256) fp8_quant(const uint16_t *x, uint32_t rows, uint32_t k, uint32_t nkb, uint8_t *q,
                                                 uint8_t *e) {
    const uint32_t w = blockIdx.x * 4 + threadIdx.x / 64, mt16 = (rows + 15) / 16;
    if (w >= mt16 * nkb) return;  // whole waves, no barrier follows
    const uint32_t mt = w / nkb, kb = w % nkb;
    const int lane = threadIdx.x % 64, lr = lane % 16, lg = lane / 16;
    // the row tile's own resource: offsets stay small for any number of rows
    const rsrc_t r = make_rsrc(x + (size_t)mt * 16 * k, min(rows - mt * 16, 16u) * k * 2u);
    uint32_t a[16];
    load_row32<VEC>(r, lr, rows - mt * 16, k, kb * FP8_BLOCK + 32 * lg, a);
    int8x_t c;
    const uint32_t eb = fp8_quant32<BF16>(a, c);
    uint8_t *dst = q + (size_t)w * FP8_FRAG + lane * 16;
    *(uint4 *)dst = make_uint4(c[0], c[1], c[2], c[3]);
    *(uint4 *)(dst + 1024) = make_uint4(c[4], c[5], c[6], c[7]);
    if (lg == 0) e[(((size_t)mt / 4 * nkb + kb) * 16 + lr) * 4 + mt % 4] = (uint8_t)eb;
}

// A thread 16 bytes of the fragment order, from number `first` on.
__global__ void __launch_bounds__(256) fp8_pack(const uint8_t *src, uint8_t *dst, uint32_t n, uint32_t k, uint32_t n16,
                                                uint32_t nkb, size_t first, size_t chunks) {
    const size_t i = first + (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= chunks) return;
    const uint32_t lane = i % 64, half = i / 64 % 2;
    const size_t frag = i / 128;
    const uint32_t kb = frag % nkb;
    const size_t tile = frag / nkb;
    const uint32_t j = (uint32_t)(tile % n16) * 16 + lane % 16, d = kb * FP8_BLOCK + lane / 16 * 32 + half * 16;
    const size_t mat = tile / n16;
    uint32_t w[4] = {0, 0, 0, 0};
    if (j < n) {
        const uint8_t *p = src + (mat * n + j) * k + d;
        if (d + 16 <= k && ((uintptr_t)p & 15) == 0) {
            const uint4 x = *(const uint4 *)p;
            w[0] = x.x;
            w[1] = x.y;
            w[2] = x.z;
            w[3] = x.w;
        } else {
            for (uint32_t b = 0; b < 16 && d + b < k; b++) w[b / 4] |= (uint32_t)p[b] << (8 * (b % 4));
        }
    }
    *(uint4 *)(dst + i * 16) = make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace

hipError_t launch_fp8_pack(const Fp8Mat &w, const uint8_t *src, uint8_t *codes, hipStream_t s) {
    const size_t chunks = w.code_bytes() * w.mats / 16;
    constexpr size_t PIECE = (size_t)1 << 31;
    for (size_t first = 0; first < chunks; first += PIECE) {
        const size_t blocks = (std::min(chunks - first, PIECE) + 255) / 256;
        hipLaunchKernelGGL(fp8_pack, dim3((uint32_t)blocks), dim3(256), 0, s, src, codes, w.n, w.k, w.n16, w.nkb, first, chunks);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

static bool rows_vec(const uint16_t *x, size_t k) { return k % 8 == 0 && ((uintptr_t)x & 15) == 0; }

hipError_t launch_fp8_quant(const uint16_t *x, size_t rows, size_t k, bool bf16, Fp8Rows out, hipStream_t s) {
    const uint32_t nkb = (uint32_t)((k + 127) / 128), waves = (uint32_t)((rows + 15) / 16) * nkb;
    if (waves == 0) return hipSuccess;
    const dim3 grid((waves + 3) / 4);
    if (!launchable(grid.x, 256)) return hipErrorInvalidConfiguration;
#define SMG_FP8_Q(B, V) hipLaunchKernelGGL((fp8_quant<B, V>), grid, dim3(256), 0, s, x, (uint32_t)rows, (uint32_t)k, nkb, out.q, out.e)
    if (rows_vec(x, k)) {
        if (bf16) SMG_FP8_Q(true, true);
        else SMG_FP8_Q(false, true);
    } else {
        if (bf16) SMG_FP8_Q(true, false);
        else SMG_FP8_Q(false, false);
    }
#undef SMG_FP8_Q
    return hipGetLastError();
}

// Calls the GEMV takes: up to 16 rows (of few depths, where it has to read them value by
// value: with a pass first 16 x 11008 x 4099 takes 17 us for 48, 2 x 14336 x 4099 19 for 26, 8 x
// 4096 x 1283 7.7 for 7.4), and up to 64 while a wave quantizes at most four
// fragments and the workgroups fit the compute units once; past that quantizing the rows
// in every workgroup costs more than a pass over them and the tiles' longer start (us
// with the weights in HBM, GEMV and tiles: 24 x 1536 x 384 3.3 / 5.6, 32 x 1536 x 2048
// 7.1 / 8.9, 64 x 512 x 512 4.7 / 6.0; the other side 32 x 4096 x 4096 12.8 / 12.0, 64 x
// 4096 x 4096 20.9 / 12.2).
static bool gemv_serves(const Fp8Mat &w, size_t m) {
    if (m <= 16) return w.k % 8 == 0 || w.nkb <= 12;
    const size_t rt = m <= 32 ? 2 : 4;
    return m <= 64 && rt * ((w.nkb + GV_W - 1) / GV_W) <= 4 && w.n16 <= 256;
}

size_t fp8_scratch_bytes(const Fp8Mat &w, size_t m) {
    return gemv_serves(w, m) || w.nkb == 0 ? 0 : Fp8Rows::bytes(m, w.nkb);
}

// Quantized rows that fp8_gemv_rows takes from the tiles, whose workgroups are few and add
// up K in series: columns enough to fill the compute units twice (once past 32 rows), where
// the tiles catch up (us, GEMV and tiles: 32 x 4096 x 4096 8.6 / 12.0, 32 x 4096 x 14336 21
// / 35, 32 x 8192 x 8192 22 / 26, 32 x 6144 x 4096 12.4 / 12.1, 29 x 11003 x 4096 17.1 /
// 16.6; 64 x 4096 x 14336 28 / 35, 64 x 4096 x 4096 11.8 / 12.2, 64 x 6144 x 4096 16 / 13).
// (K: the fragments of 64 rows lie within a resource of 2 GiB.)
static bool rows_serve(const Fp8Mat &w, size_t m) {
    return m <= 16 ? w.nkb < 1u << 18 : m <= 64 && w.n16 <= (m <= 32 ? 512u : 256u) && w.nkb < 1u << 18;
}

template <int RT>
static hipError_t launch_gemv_rows(const GvArgs &g, Fp8Rows r, const EpArgs &ep, bool bf16, hipStream_t s) {
    const dim3 grid((g.n + 15) / 16);
    if (bf16) hipLaunchKernelGGL((fp8_gemv_rows<RT, true>), grid, dim3(GV_NT), 0, s, g, r, ep);
    else hipLaunchKernelGGL((fp8_gemv_rows<RT, false>), grid, dim3(GV_NT), 0, s, g, r, ep);
    return hipGetLastError();
}

template <int RT, int CT, int U, bool VEC>
static hipError_t launch_gemv(const GvArgs &g, const EpArgs &ep, bool bf16, hipStream_t s) {
    const dim3 grid((g.n + 16 * CT - 1) / (16 * CT));
    if (bf16) hipLaunchKernelGGL((fp8_gemv<RT, CT, U, true, VEC>), grid, dim3(GV_NT), 0, s, g, ep);
    else hipLaunchKernelGGL((fp8_gemv<RT, CT, U, false, VEC>), grid, dim3(GV_NT), 0, s, g, ep);
    return hipGetLastError();
}

// Two column tiles a workgroup where one each would be more than two rounds of the
// compute units (1 x 14336 x 4096 13.3 us with one, 11.4 with two; 1 x 4096 x 4096 5.1 and
// 5.8); two blocks in flight a wave where it has them (1 x 1536 x 384 2.6 us, with one
// 2.3). Rows read value by value are read once for two tiles (3 x 5000 x 1001 9.1 us with
// one tile, 5.7 with two).
hipError_t launch_fp8_matmul(const Fp8Mat &w, size_t m, uint16_t *dst, const uint16_t *lhs, const EpArgs &ep, bool bf16,
                             void *scratch, hipStream_t s) {
    const GvArgs g = {w.codes, w.scales, lhs, dst, (uint32_t)m, w.n, w.k, w.nkb, w.n16};
    if (!gemv_serves(w, m)) {
        const Fp8Rows a = Fp8Rows::at(scratch, m, w.nkb);
        const hipError_t e = launch_fp8_quant(lhs, m, w.k, bf16, a, s);
        if (e != hipSuccess) return e;
        if (!rows_serve(w, m)) return launch_fp8_gemm(w, m, dst, a, ep, bf16, s);
        if (m <= 16) return launch_gemv_rows<1>(g, a, ep, bf16, s);
        return m <= 32 ? launch_gemv_rows<2>(g, a, ep, bf16, s) : launch_gemv_rows<4>(g, a, ep, bf16, s);
    }
    const bool vec = rows_vec(lhs, w.k);
    if (m > 32) return vec ? launch_gemv<4, 1, 1, true>(g, ep, bf16, s) : launch_gemv<4, 1, 1, false>(g, ep, bf16, s);
    if (m > 16) return vec ? launch_gemv<2, 1, 1, true>(g, ep, bf16, s) : launch_gemv<2, 1, 1, false>(g, ep, bf16, s);
    if (!vec) return launch_gemv<1, 2, 1, false>(g, ep, bf16, s);
    if (w.nkb <= (uint32_t)GV_W) return launch_gemv<1, 1, 1, true>(g, ep, bf16, s);
    return w.n16 > 512 ? launch_gemv<1, 2, 2, true>(g, ep, bf16, s) : launch_gemv<1, 1, 2, true>(g, ep, bf16, s);
}

}  // namespace smg
