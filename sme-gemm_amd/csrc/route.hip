// Routing to experts: for each row of logits the scores (softmax or sigmoid), the
// choice (score + bias), the groups whose two largest choices add up to most, the
// top_k experts of those, lowest index first among equals, and their weights.
//
// A row is taken by 16 lanes (four rows a wave) up to 256 experts and 15 taken, by a wave
// past that; lane l of them holds experts l, l + LPR, ... The answer is defined by scores
// in 64 bits: sigmoids a few f32 ulps apart would pick other experts from one
// implementation to the next. Without bias and groups the logits themselves order the
// experts (both scores grow with them), short of the range in which the scores saturate:
// those rows, and all with bias or groups, are scored in f64, which costs as little as f32
// here (scalar f64 instructions issue at f32's rate). The choices stay in LDS and their f32
// values, which order them but for those that round alike, in registers; where two of those
// meet among the taken or at their end, the f64 ones decide.
// What bounds it: one token, the launch; many rows, the latency of one wave's work and of
// fetching its code, which is why the scores are a rolled loop of four experts a lane (8192
// rows, 8 of 256 experts, 4 of 8 groups: 16 us; f32 scores unrolled, with an f64 repeat of
// the few rows in which they could not tell: 23).
#include "experts.h"

namespace smg {

namespace {

constexpr int RT_NT = 256, RT_W = RT_NT / 64;  // threads, waves a workgroup

// Orders LDS written by a wave before its own reads.
__device__ __forceinline__ void wave_lds() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Over a row's lanes (LPR: 16 or 64), the result in each of them.
template <int CTRL>
__device__ __forceinline__ uint32_t lane_of(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xF, 0xF, false);
}
template <int CTRL>
__device__ __forceinline__ double lane_of(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    return __longlong_as_double((long long)((uint64_t)lane_of<CTRL>((uint32_t)(u >> 32)) << 32 | lane_of<CTRL>((uint32_t)u)));
}
template <int LPR, class T, class F>
__device__ __forceinline__ T row_reduce(T x, F f) {
    x = f(x, lane_of<0xB1>(x));   // lane ^ 1
    x = f(x, lane_of<0x4E>(x));   // lane ^ 2
    x = f(x, lane_of<0x141>(x));  // 7 - lane of 8
    x = f(x, lane_of<0x140>(x));  // 15 - lane of 16
    if constexpr (LPR == 64) {
        x = f(x, __shfl_xor(x, 16));
        x = f(x, __shfl_xor(x, 32));
    }
    return x;
}
template <int LPR>
__device__ __forceinline__ float row_max(float x) {
    return __uint_as_float(row_reduce<LPR>(__float_as_uint(x), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
template <int LPR>
__device__ __forceinline__ uint32_t row_min(uint32_t x) {
    return row_reduce<LPR>(x, [](uint32_t a, uint32_t b) { return min(a, b); });
}
template <int LPR>
__device__ __forceinline__ double row_max(double x) {
    return row_reduce<LPR>(x, [](double a, double b) { return fmax(a, b); });
}
template <int LPR>
__device__ __forceinline__ double row_sum(double x) {
    return row_reduce<LPR>(x, [](double a, double b) { return a + b; });
}

// e^x to 2^-52 or so: 2^k e^r, |r| <= ln 2 / 2, e^r by its Taylor series to r^13 (the rest
// is below 2^-57). 0 and infinity past the range; x is not NaN.
__device__ __forceinline__ double exp64(double x) {
    x = fmin(fmax(x, -800.0), 800.0);
    const double k = rint(x * 1.4426950408889634);
    // ln 2 in two parts, the first of 32 bits: its product with k is exact
    const double r = __builtin_fma(k, -1.9082149292705877e-10, __builtin_fma(k, -0.6931471803691238, x));
    double p = 1.0 / 6227020800.0;
    p = __builtin_fma(p, r, 1.0 / 479001600.0);
    p = __builtin_fma(p, r, 1.0 / 39916800.0);
    p = __builtin_fma(p, r, 1.0 / 3628800.0);
    p = __builtin_fma(p, r, 1.0 / 362880.0);
    p = __builtin_fma(p, r, 1.0 / 40320.0);
    p = __builtin_fma(p, r, 1.0 / 5040.0);
    p = __builtin_fma(p, r, 1.0 / 720.0);
    p = __builtin_fma(p, r, 1.0 / 120.0);
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_amdgcn_ldexp(p, (int)k);
}

// NE experts a lane, LPR lanes a row.
template <int TYPE, int NE, int LPR>
__global__ void __launch_bounds__(RT_NT) route(RouteArgs a) {
    constexpr int RPW = 64 / LPR;  // rows a wave
    static_assert(NE % 4 == 0, "four experts a step");
    // a row's choices [groups][per + 1], the next row's in other banks; its logits
    constexpr int CS = NE * LPR + ROUTE_MAX_GROUPS + (RPW > 1 ? 9 : 0);
    __shared__ double choices[RT_W][RPW * CS];
    __shared__ float logits[RT_W][RPW][NE * LPR];
    __shared__ double totals[RT_W][RPW][ROUTE_MAX_GROUPS];
    const int lane = threadIdx.x % 64, sub = lane % LPR, rw = lane / LPR;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t row0 = (blockIdx.x * RT_W + wave) * RPW;
    if (row0 >= a.rows) return;  // whole waves, no barrier follows
    const uint32_t rows = min((uint32_t)RPW, a.rows - row0), own = min((uint32_t)rw, rows - 1), row = row0 + own;
    constexpr uint32_t ES = TYPE == LOGIT_F32 ? 4 : 2;
    const rsrc_t lr = make_rsrc((const uint8_t *)a.logits + (size_t)row0 * a.experts * ES, rows * a.experts * ES);
    const rsrc_t br = make_rsrc(a.bias, a.bias ? a.experts * 4 : 0);  // (zeros without one, and past the end)
    float l[NE];
#pragma unroll
    for (int i = 0; i < NE; i++) {
        const uint32_t off = (own * a.experts + i * LPR + sub) * ES;
        if constexpr (TYPE == LOGIT_F32) l[i] = __uint_as_float(bload4(lr, off));
        else l[i] = to_f32<TYPE == LOGIT_BF16>(bload2(lr, off));
    }
    float m = -INFINITY;  // the row's largest logit
#pragma unroll
    for (int i = 0; i < NE; i++) {  // (NaN is masked, as -inf is)
        l[i] = (uint32_t)(i * LPR + sub) < a.experts && l[i] > -INFINITY ? l[i] : -INFINITY;
        m = fmaxf(m, l[i]);
    }
    m = row_max<LPR>(m);
    float *lg = logits[wave][rw];
    double *ch = choices[wave] + rw * CS, *tot = totals[wave][rw];
    const uint32_t per = a.experts / a.groups;
    const float per_inv = 1.0f / (float)per;
    // (e + 0.5) / per is never within a half's distance of rounding to the next group
    auto place_of = [&](uint32_t e) __attribute__((always_inline)) {
        return e + (uint32_t)(((float)e + 0.5f) * per_inv);
    };
    // e^(l - max) or e^-l; the score from it
    auto power = [&](float x) __attribute__((always_inline)) {
        return exp64(a.sigmoid ? -(double)x : x == m ? 0.0 : (double)x - (double)m);
    };
    double sum = 1.0;  // a softmax's
    auto score_of = [&](double p) __attribute__((always_inline)) { return (a.sigmoid ? 1.0 : p) / (a.sigmoid ? 1.0 + p : sum); };

    bool by_logit = !a.bias && a.groups == 1 && a.top_k < LPR;  // (a lane for the first left out, below)
    int id;
    double score;
    for (;;) {
        float key[NE];  // -inf: masked, or taken
        if (by_logit) {
#pragma unroll
            for (int i = 0; i < NE; i++) key[i] = l[i];
        } else {
#pragma unroll
            for (int i = 0; i < NE; i++) lg[i * LPR + sub] = l[i];
            wave_lds();
        }
        if (!a.sigmoid) {
            // (where only the logits decide, f32 powers do for the weights: 2^-19 of them)
            if (by_logit) {
                float t = 0.0f;
#pragma unroll
                for (int i = 0; i < NE; i++)
                    t += l[i] == m ? 1.0f : __builtin_amdgcn_exp2f((l[i] - m) * 1.4426950408889634f);
                sum = row_sum<LPR>((double)t);
            } else {
                double t = 0.0;
#pragma unroll 1
                for (int i0 = 0; i0 < NE; i0 += 4)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float x = lg[(i0 + i) * LPR + sub];
                        t += x > -INFINITY ? power(x) : 0.0;
                    }
                sum = row_sum<LPR>(t);
            }
        }
        if (!by_logit) {
            float b[4];
#pragma unroll
            for (int i = 0; i < 4; i++) b[i] = __uint_as_float(bload4(br, (i * LPR + sub) * 4));
#pragma unroll 1
            for (uint32_t i0 = 0; i0 < NE; i0 += 4) {
                float x[4], bn[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[i] = lg[(i0 + i) * LPR + sub];
                    bn[i] = __uint_as_float(bload4(br, ((i0 + 4 + i) * LPR + sub) * 4));
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t e = (i0 + i) * LPR + sub;
                    const double c = score_of(power(x[i])) + (double)b[i];
                    if (e < a.experts) ch[place_of(e)] = x[i] > -INFINITY && c > -INFINITY ? c : -INFINITY;
                    b[i] = bn[i];
                }
            }
            wave_lds();
            if (a.groups > 1) {
                // 1, 2 or 4 lanes a group, each its share of the group's choices, then merged
                const uint32_t split = a.groups * 4 <= LPR ? 2 : a.groups * 2 <= LPR ? 1 : 0, part = sub & ((1u << split) - 1);
                for (uint32_t g = sub >> split; g < a.groups; g += LPR >> split) {
                    double t1 = -INFINITY, t2 = -INFINITY;
                    const double *c = ch + g * (per + 1);
                    for (uint32_t x0 = part; x0 < per; x0 += 8u << split) {
                        double v[8];
#pragma unroll
                        for (int x = 0; x < 8; x++) {
                            const uint32_t at = x0 + (x << split);
                            v[x] = c[min(at, per - 1)];
                            v[x] = at < per ? v[x] : -INFINITY;
                        }
#pragma unroll
                        for (int x = 0; x < 8; x++) {
                            t2 = fmax(t2, fmin(t1, v[x]));
                            t1 = fmax(t1, v[x]);
                        }
                    }
                    auto merge = [&](double o1, double o2) __attribute__((always_inline)) {
                        t2 = fmax(fmax(t2, o2), fmin(t1, o1));
                        t1 = fmax(t1, o1);
                    };
                    if (split > 0) merge(lane_of<0xB1>(t1), lane_of<0xB1>(t2));
                    if (split > 1) merge(lane_of<0x4E>(t1), lane_of<0x4E>(t2));
                    tot[g] = t2 > -INFINITY ? t1 + t2 : t1;  // (-inf: nothing left in the group)
                }
                wave_lds();
                for (uint32_t g = sub >> split; g < a.groups; g += LPR >> split) {
                    const double t = tot[g];
                    uint32_t rank = 0;
                    for (uint32_t o0 = 0; o0 < a.groups; o0 += 4)
#pragma unroll
                        for (uint32_t o = o0; o < o0 + 4; o++) {
                            const double x = o < a.groups ? tot[min(o, a.groups - 1)] : -INFINITY;
                            rank += x > t || (x == t && o < g);
                        }
                    if (rank >= a.top_groups)
                        for (uint32_t x = part; x < per; x += 1u << split) ch[g * (per + 1) + x] = -INFINITY;
                }
                wave_lds();
            }
#pragma unroll
            for (int i = 0; i < NE; i++) {
                const uint32_t e = i * LPR + sub;
                key[i] = e < a.experts ? (float)ch[place_of(min(e, a.experts - 1))] : -INFINITY;
            }
        }
        // lane j of the row gets its j-th expert and that one's key; one more than asked
        // for, so that the last taken and the first left out are compared too
        id = -1;
        float mine = -INFINITY;
        for (uint32_t j = 0; j <= a.top_k; j++) {
            float best = -INFINITY;
            uint32_t at = 0;
#pragma unroll
            for (int i = 0; i < NE; i++) best = fmaxf(best, key[i]);
            const float top = row_max<LPR>(best);
            const bool some = top > -INFINITY;
#pragma unroll
            for (int i = NE - 1; i >= 0; i--) at = key[i] == top ? i : at;
            if (__builtin_amdgcn_ballot_w64(some) == 0) break;
            // the lowest index that has it
            const uint32_t e = row_min<LPR>(some && best == top ? at * LPR + sub : 0xFFFFFFFFu);
#pragma unroll
            for (int i = 0; i < NE; i++) key[i] = (uint32_t)(i * LPR + sub) == e ? -INFINITY : key[i];
            if (sub == (int)j && some) {
                id = (int)e;
                mine = top;
            }
        }
        const float before = __shfl_up(mine, 1);
        const bool pair = id >= 0 && sub > 0;
        if (by_logit) {
            // logits whose f64 scores could be equal: too near, or scores near 1 or 0
            float gap = before - mine;
            if (a.sigmoid && before > 0.0f) gap *= __builtin_amdgcn_exp2f(before * -1.4426950408889634f);
            const bool flat = !(gap >= 0x1p-48f) || (a.sigmoid ? before : fminf(before, mine) - m) < -700.0f;
            if (__builtin_amdgcn_ballot_w64(pair && mine != before && flat)) {
                by_logit = false;
                continue;
            }
        } else if (__builtin_amdgcn_ballot_w64((pair && mine == before) || a.top_k >= LPR)) {
            // f64 choices that round alike: select by those themselves
            id = -1;
#pragma unroll 1
            for (uint32_t j = 0; j < a.top_k; j++) {
                double best = -INFINITY;
                uint32_t at = 0;
#pragma unroll 1
                for (uint32_t e = sub; e < a.experts; e += LPR) {
                    const double x = ch[place_of(e)];
                    at = x > best ? e : at;
                    best = fmax(best, x);
                }
                const double top = row_max<LPR>(best);
                const bool some = top > -INFINITY;
                if (__builtin_amdgcn_ballot_w64(some) == 0) break;
                const uint32_t e = row_min<LPR>(some && best == top ? at : 0xFFFFFFFFu);
                if (some && e % LPR == (uint32_t)sub) ch[place_of(e)] = -INFINITY;
                wave_lds();
                if (sub == (int)j && some) id = (int)e;
            }
        }
        if (sub >= (int)a.top_k) id = -1;
        score = id < 0 ? 0.0 : score_of(power(by_logit ? mine : lg[max(id, 0)]));
        break;
    }
    if (a.renormalize) {
        const double of = row_sum<LPR>(score);
        score = of > 0.0 ? score / of : 0.0;
    }
    if (sub < (int)a.top_k && (uint32_t)rw < rows) {
        a.ids[(size_t)row * a.top_k + sub] = id;
        a.weights[(size_t)row * a.top_k + sub] = (float)(score * (double)a.scale);
    }
}

template <int TYPE>
hipError_t launch_rows(const RouteArgs &a, hipStream_t s) {
    const bool quarter = a.experts <= 256 && a.top_k < 16;  // 16 lanes a row
    const uint32_t per = RT_W * (quarter ? 4 : 1);
    const dim3 grid((a.rows + per - 1) / per), block(RT_NT);
    if (quarter) {
        if (a.experts <= 64) hipLaunchKernelGGL((route<TYPE, 4, 16>), grid, block, 0, s, a);
        else if (a.experts <= 128) hipLaunchKernelGGL((route<TYPE, 8, 16>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((route<TYPE, 16, 16>), grid, block, 0, s, a);
    } else {
        if (a.experts <= 256) hipLaunchKernelGGL((route<TYPE, 4, 64>), grid, block, 0, s, a);
        else if (a.experts <= 512) hipLaunchKernelGGL((route<TYPE, 8, 64>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((route<TYPE, 16, 64>), grid, block, 0, s, a);
    }
    return hipGetLastError();
}
// (as launchable asks)
template <int TYPE>
hipError_t launch_type(RouteArgs a, hipStream_t s) {
    constexpr uint32_t PIECE = 1u << 24;  // rows
    for (uint32_t left = a.rows; left != 0; left -= a.rows) {
        a.rows = left < PIECE ? left : PIECE;
        const hipError_t e = launch_rows<TYPE>(a, s);
        if (e != hipSuccess) return e;
        a.logits = (const uint8_t *)a.logits + (size_t)a.rows * a.experts * (TYPE == LOGIT_F32 ? 4 : 2);
        a.ids += (size_t)a.rows * a.top_k;
        a.weights += (size_t)a.rows * a.top_k;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_route(const RouteArgs &a, int logit_type, hipStream_t s) {
    switch (logit_type) {
    case LOGIT_F32: return launch_type<LOGIT_F32>(a, s);
    case LOGIT_F16: return launch_type<LOGIT_F16>(a, s);
    default: return launch_type<LOGIT_BF16>(a, s);
    }
}

}  // namespace smg
