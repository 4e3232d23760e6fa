// The C ABI of the 8-bit floating-point weights and products, of routing and of the
// experts (include/smegemm_gpu.h).
#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <new>

#include "call_scratch.h"
#include "experts.h"

using namespace smg;

namespace {

// Bounds within which a matrix's and a call's offsets stay in the kernels' types: a
// column tile's fragments within 2^31 bytes (nkb <= 2^18), a launch's threads below 2^32 (the
// products of few rows: 512 for 16 columns).
constexpr size_t FP8_MAX_K = (size_t)1 << 25, FP8_MAX_N = (size_t)1 << 27;

// No exception leaves a C entry.
template <class F>
int guarded(F f) {
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return report(SMG_ENOMEM, "out of host memory");
    } catch (...) {
        return report(SMG_EHIP, "unexpected failure");
    }
}

// e4m3, ties to even, of |x| <= 448 (larger saturates); NaN stays NaN.
uint8_t e4m3_rne(float x) {
    uint32_t u;
    std::memcpy(&u, &x, 4);
    const uint8_t sign = (uint8_t)(u >> 24 & 0x80);
    if (x != x) return (uint8_t)(sign | 0x7F);
    const float a = std::fabs(x);
    if (a >= 464.0f) return (uint8_t)(sign | 0x7E);
    if (a < 0.015625f) return (uint8_t)(sign | (uint8_t)std::nearbyint(a * 512.0f));  // subnormals, steps of 2^-9; 8 is 2^-6
    u &= 0x7FFFFFFFu;
    u += 0x7FFFFu + (u >> 20 & 1);  // to 3 mantissa bits
    return (uint8_t)(sign | ((u >> 20) - ((127 - 7) << 3)));
}

// `mats` matrices of n columns and k depths, one after another.
int fp8_create(const uint8_t *codes, const float *scales, size_t n, size_t k, size_t mats, bool dev, void *stream,
               smg_weights **out) {
    if (!out || (n && k && (!codes || !scales))) return report(SMG_EINVAL, "null argument");
    if (k >= FP8_MAX_K || n >= FP8_MAX_N) return report(SMG_EINVAL, "fp8 weights: too many columns or depths");
    if (!smg_available()) return report(SMG_ENODEV, "no gfx950 device");
    smg_weights *w = handle_new(W_FP8, n, k, FP8_BLOCK);
    Fp8Mat &f = w->f8;
    f = fp8_shape((uint32_t)n, (uint32_t)k, (uint32_t)mats);
    int rc = SMG_OK;
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (dev) {
        rc = check_device_pointers(w->device, EpPlan{}, {n && k ? codes : nullptr, n && k ? scales : nullptr});
        if (!rc && (hipStreamIsCapturing((hipStream_t)stream, &st) != hipSuccess || st != hipStreamCaptureStatusNone)) {
            (void)hipGetLastError();
            rc = report(SMG_EINVAL, "weights are not created while the stream is captured");
        }
    }
    void *pc = nullptr, *ps = nullptr, *raw = nullptr;
    const size_t raw_bytes = n * k * mats, scale_bytes = f.scale_count() * mats * 4;
    if (!rc) rc = handle_alloc(w, f.code_bytes() * mats, &pc);
    if (!rc) rc = handle_alloc(w, scale_bytes, &ps);
    f.codes = (const uint8_t *)pc;
    f.scales = (const float *)ps;
    if (!rc && n && k) {
        hipStream_t s = (hipStream_t)stream;
        hipError_t e = hipSuccess;
        if (!dev) {
            if (device_malloc(&raw, raw_bytes) != hipSuccess) rc = report(SMG_ENOMEM, "weights hipMalloc");
            else e = hipMemcpyAsync(raw, codes, raw_bytes, hipMemcpyHostToDevice, s);
        }
        if (!rc && e == hipSuccess)
            e = hipMemcpyAsync(ps, scales, scale_bytes, dev ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice, s);
        if (!rc && e == hipSuccess) e = launch_fp8_pack(f, dev ? codes : (const uint8_t *)raw, (uint8_t *)pc, s);
        const hipError_t done = rc ? hipSuccess : hipStreamSynchronize(s);
        if (e == hipSuccess) e = done;
        if (raw) (void)hipFree(raw);
        if (!rc && e != hipSuccess) rc = report_hip(SMG_EHIP, "fp8 weights", e);
    }
    if (rc) {
        handle_destroy(w);
        return rc;
    }
    *out = w;
    return SMG_OK;
}

int check_fp8(const smg_weights *w) {
    if (!w) return report(SMG_EINVAL, "null weights");
    return w->d.kind == W_FP8 ? SMG_OK : report(SMG_EKIND, "weight handle of another kind");
}

int check_rows(const smg_weights *w, size_t m) {
    const size_t big = (size_t)1 << 31;
    if (m >= big || (m + 15) / 16 * w->f8.nkb >= big || (m + 15) / 16 * w->f8.n16 >= big)
        return report(SMG_EINVAL, "too many rows a call");
    return SMG_OK;
}

int fp8_host(size_t m, const smg_weights *w, uint16_t *dst, const uint16_t *lhs, const ep_desc16 *ep, bool bf16) {
    int rc = check_fp8(w);
    if (rc) return rc;
    const size_t n = w->d.n, k = w->d.k;
    if (m == 0 || n == 0) return SMG_OK;
    if (!dst || (k && !lhs)) return report(SMG_EINVAL, "null array");
    if ((rc = check_rows(w, m))) return rc;
    const Fp8Mat f = w->f8;
    return host_product(bf16 ? "gemm_gpu_b16_fp8" : "gemm_gpu_f16_fp8", w->device, m, n, k, dst, lhs, ep,
                        fp8_scratch_bytes(f, m),
                        [&](uint16_t *dd, const uint16_t *dl, const EpPlan &p, void *sc, hipStream_t s) {
                            const hipError_t e = launch_fp8_matmul(f, m, dd, dl, p.fused, bf16, sc, s);
                            return e == hipSuccess ? run_graph_tail(p, dd, m, n, bf16, s) : e;
                        });
}

}  // namespace

struct smg_experts {
    smg_weights *gate = nullptr, *up = nullptr, *down = nullptr;
    uint32_t act = 0;
    int device = 0;
    ExpertSet set() const { return {gate->f8, up->f8, down->f8, act}; }
};

namespace {

void experts_destroy(smg_experts *e) {
    if (!e) return;
    for (smg_weights *w : {e->gate, e->up, e->down})
        if (w) handle_destroy(w);
    delete e;
}

struct ExpertArrays {
    const uint8_t *gate, *up, *down;
    const float *gate_s, *up_s, *down_s;
};
int experts_create(const ExpertArrays &a, size_t experts, size_t d, size_t ffn, uint32_t act, bool dev, void *stream,
                   smg_experts **out) {
    if (!out || !a.gate || !a.up || !a.down || !a.gate_s || !a.up_s || !a.down_s) return report(SMG_EINVAL, "null argument");
    if (experts == 0 || experts > ROUTE_MAX_EXPERTS) return report(SMG_EINVAL, "from 1 to 1024 experts");
    if (d == 0 || ffn == 0) return report(SMG_EINVAL, "an expert has a width and a hidden width");
    if (d >= FP8_MAX_K || ffn >= FP8_MAX_K) return report(SMG_EINVAL, "fp8 weights: too many columns or depths");
    if (act != EP_ACT_SILU && act != EP_ACT_GELU) return report(SMG_EINVAL, "an expert's gate is silu or gelu");
    if (!smg_available()) return report(SMG_ENODEV, "no gfx950 device");
    std::unique_ptr<smg_experts, void (*)(smg_experts *)> own(new smg_experts(), experts_destroy);
    smg_experts *e = own.get();
    e->act = act;
    int rc = fp8_create(a.gate, a.gate_s, ffn, d, experts, dev, stream, &e->gate);
    if (!rc) rc = fp8_create(a.up, a.up_s, ffn, d, experts, dev, stream, &e->up);
    if (!rc) rc = fp8_create(a.down, a.down_s, d, ffn, experts, dev, stream, &e->down);
    if (rc) return rc;
    e->device = e->gate->device;
    *out = own.release();
    return SMG_OK;
}

int experts_limits(const smg_experts *e, size_t rows, size_t top_k) {
    if (!e) return report(SMG_EINVAL, "null experts");
    if (top_k == 0) return report(SMG_EINVAL, "a row has at least one expert");
    const size_t big = (size_t)1 << 31;
    // (the kernels' grids: a wave per 16 padded rows and block of depths, a workgroup
    // per tile of 128 rows x 128 columns, one per 2048 columns of a row)
    if (rows >= big || top_k >= big || rows * top_k >= big - 63 * ROUTE_MAX_EXPERTS)
        return report(SMG_EINVAL, "too many rows a call");
    const size_t padded = rows * top_k + 63 * ROUTE_MAX_EXPERTS, blocks = std::max(e->gate->f8.nkb, e->down->f8.nkb);
    if (padded / 16 * blocks >= big || rows * ((e->gate->d.k + 2047) / 2048) >= big)
        return report(SMG_EINVAL, "too many rows a call");
    return SMG_OK;
}

int experts_check(const smg_experts *e, const void *x, const int32_t *ids, const float *weights, const void *out, size_t rows,
                  size_t top_k) {
    const int rc = experts_limits(e, rows, top_k);
    if (rc) return rc;
    return x && ids && weights && out ? SMG_OK : report(SMG_EINVAL, "null array");
}

int experts_dev(const smg_experts *e, const uint16_t *x, int bf16, const int32_t *ids, const float *weights, size_t rows,
                size_t top_k, uint16_t *out, float *y, void *stream, const OwnScratch *own = nullptr) {
    if (e && rows == 0) return SMG_OK;
    int rc = experts_check(e, x, ids, weights, out ? (const void *)out : y, rows, top_k);
    if (rc) return rc;
    if ((rc = check_device_pointers(e->device, EpPlan{}, {x, ids, weights, out, y, own ? own->buf : nullptr}))) return rc;
    DeviceScope on(e->device);
    if (on.error() != hipSuccess) return report_hip(SMG_EHIP, "hipSetDevice", on.error());
    const ExpertSet set = e->set();
    const ExpertCall c = {x, ids, weights, out, y, (uint32_t)rows, (uint32_t)top_k, bf16 != 0};
    CallScratch sc(e->device, stream, experts_scratch_bytes(set, c), own);
    if ((rc = sc.check("experts"))) return rc;
    const hipError_t err = launch_experts(set, c, sc.buf(), (hipStream_t)stream);
    if (err == hipErrorInvalidConfiguration) return report(SMG_EINVAL, "too many rows a call");
    return err == hipSuccess ? SMG_OK : report_hip(SMG_EHIP, "experts", err);
}

// The host form: the device form over staged arrays.
int experts_host(const smg_experts *e, const uint16_t *x, int bf16, const int32_t *ids, const float *weights, size_t rows,
                 size_t top_k, uint16_t *out, float *y) {
    if (e && rows == 0) return SMG_OK;
    const int rc = experts_check(e, x, ids, weights, out ? (const void *)out : y, rows, top_k);
    if (rc) return rc;
    const size_t n = rows * e->gate->d.k;
    const Slice s[] = {{(void *)x, n * 2, true, false},
                       {(void *)ids, rows * top_k * 4, true, false},
                       {(void *)weights, rows * top_k * 4, true, false},
                       {out, out ? n * 2 : 0, false, true},
                       {y, y ? n * 4 : 0, true, true}};
    return host_slices(e->device, s, 5, [&](void **d, void *st) {
        return experts_dev(e, (const uint16_t *)d[0], bf16, (const int32_t *)d[1], (const float *)d[2], rows, top_k,
                           (uint16_t *)d[3], (float *)d[4], st);
    });
}

int fp8_dev(size_t m, const smg_weights *w, uint16_t *dst, const uint16_t *lhs, const ep_desc16 *ep, int bf16, void *stream,
            const OwnScratch *own) {
    int rc = check_fp8(w);
    if (rc) return rc;
    const size_t n = w->d.n, k = w->d.k;
    if (m == 0 || n == 0) return SMG_OK;
    if (!dst || (k && !lhs)) return report(SMG_EINVAL, "null array");
    if ((rc = check_rows(w, m))) return rc;
    EpPlan p;
    if ((rc = plan_graph(ep, &p, n))) return rc;
    if ((rc = check_device_pointers(w->device, p, {dst, k ? lhs : nullptr, own ? own->buf : nullptr}))) return rc;
    DeviceScope on(w->device);
    if (on.error() != hipSuccess) return report_hip(SMG_EHIP, "hipSetDevice", on.error());
    CallScratch sc(w->device, stream, fp8_scratch_bytes(w->f8, m), own);
    if ((rc = sc.check("smg_fp8_matmul_dev"))) return rc;
    hipStream_t s = (hipStream_t)stream;
    hipError_t e = launch_fp8_matmul(w->f8, m, dst, lhs, p.fused, bf16 != 0, sc.buf(), s);
    if (e == hipErrorInvalidConfiguration) return report(SMG_EINVAL, "too many rows a call");
    if (e == hipSuccess) e = run_graph_tail(p, dst, m, n, bf16 != 0, s);
    return e == hipSuccess ? SMG_OK : report_hip(SMG_EHIP, "smg_fp8_matmul_dev", e);
}

int route_check(const smg_router *r, size_t rows, const void *logits, int type, const int32_t *ids, const float *weights) {
    if (!r) return report(SMG_EINVAL, "null router");
    if (r->experts == 0 || r->experts > ROUTE_MAX_EXPERTS) return report(SMG_EINVAL, "from 1 to 1024 experts");
    if (r->score > 1) return report(SMG_EINVAL, "score is 0 (softmax) or 1 (sigmoid)");
    if (r->groups == 0 || r->groups > ROUTE_MAX_GROUPS || r->experts % r->groups)
        return report(SMG_EINVAL, "from 1 to 64 groups, of equally many experts");
    if (r->top_groups == 0 || r->top_groups > r->groups) return report(SMG_EINVAL, "from 1 to all of the groups are kept");
    if (r->top_k == 0 || r->top_k > ROUTE_MAX_TOP || r->top_k > r->experts / r->groups * r->top_groups)
        return report(SMG_EINVAL, "from 1 to 64 experts a row, no more than the kept groups have");
    if (type < LOGIT_F32 || type > LOGIT_BF16) return report(SMG_EINVAL, "logits are f32 (0), f16 (1) or bf16 (2)");
    if (rows >= (size_t)1 << 31) return report(SMG_EINVAL, "too many rows a call");
    if (rows && (!logits || !ids || !weights)) return report(SMG_EINVAL, "null array");
    return SMG_OK;
}

}  // namespace

extern "C" {

int smg_route_dev(const smg_router *r, size_t rows, const void *logits, int type, const float *bias, int32_t *ids,
                  float *weights, void *stream) {
    return guarded([&]() -> int {
        int rc = route_check(r, rows, logits, type, ids, weights);
        if (rc || rows == 0) return rc;
        int device = 0;
        const hipError_t ed = hipGetDevice(&device);
        if (ed != hipSuccess) return report_hip(SMG_ENODEV, "hipGetDevice", ed);
        if ((rc = check_device_pointers(device, EpPlan{}, {logits, bias, ids, weights}))) return rc;
        const RouteArgs a = {logits, bias, ids, weights, (uint32_t)rows, r->experts, r->top_k, r->score, r->groups,
                             r->top_groups, r->renormalize, r->scale};
        const hipError_t e = launch_route(a, type, (hipStream_t)stream);
        return e == hipSuccess ? SMG_OK : report_hip(SMG_EHIP, "smg_route_dev", e);
    });
}

int smg_route(const smg_router *r, size_t rows, const void *logits, int type, const float *bias, int32_t *ids,
              float *weights) {
    return guarded([&]() -> int {
        int rc = route_check(r, rows, logits, type, ids, weights);
        if (rc || rows == 0) return rc;
        int device = 0;
        const hipError_t ed = hipGetDevice(&device);
        if (ed != hipSuccess) return report_hip(SMG_ENODEV, "hipGetDevice", ed);
        const Slice s[] = {{(void *)logits, rows * r->experts * (type == LOGIT_F32 ? 4 : 2), true, false},
                           {(void *)bias, bias ? r->experts * 4u : 0u, true, false},
                           {ids, rows * r->top_k * 4, false, true},
                           {weights, rows * r->top_k * 4, false, true}};
        return host_slices(device, s, 4, [&](void **d, void *st) {
            return smg_route_dev(r, rows, d[0], type, (const float *)d[1], (int32_t *)d[2], (float *)d[3], st);
        });
    });
}

int smg_experts_create(const uint8_t *gate, const float *gate_scales, const uint8_t *up, const float *up_scales,
                       const uint8_t *down, const float *down_scales, size_t experts, size_t d, size_t ffn, uint32_t act,
                       smg_experts **out) {
    return guarded([&] {
        return experts_create({gate, up, down, gate_scales, up_scales, down_scales}, experts, d, ffn, act, false, nullptr, out);
    });
}

int smg_experts_create_dev(const uint8_t *gate, const float *gate_scales, const uint8_t *up, const float *up_scales,
                           const uint8_t *down, const float *down_scales, size_t experts, size_t d, size_t ffn, uint32_t act,
                           void *stream, smg_experts **out) {
    return guarded([&] {
        return experts_create({gate, up, down, gate_scales, up_scales, down_scales}, experts, d, ffn, act, true, stream, out);
    });
}

void smg_experts_destroy(smg_experts *e) { experts_destroy(e); }

int smg_experts_forward_dev(const smg_experts *e, const uint16_t *x, int bf16, const int32_t *ids, const float *weights,
                            size_t rows, size_t top_k, uint16_t *out, void *stream) {
    return guarded([&] { return experts_dev(e, x, bf16, ids, weights, rows, top_k, out, nullptr, stream); });
}

int smg_experts_accumulate_dev(const smg_experts *e, const uint16_t *x, int bf16, const int32_t *ids, const float *weights,
                               size_t rows, size_t top_k, float *y, void *stream) {
    return guarded([&] { return experts_dev(e, x, bf16, ids, weights, rows, top_k, nullptr, y, stream); });
}

int smg_experts_scratch_bytes(const smg_experts *e, size_t rows, size_t top_k, size_t *bytes) {
    if (!bytes) return report(SMG_EINVAL, "null argument");
    const int rc = experts_limits(e, rows, top_k);
    if (rc) return rc;
    *bytes = rows ? experts_scratch_bytes(e->set(), rows, top_k) : 0;
    return SMG_OK;
}

int smg_experts_forward_ws_dev(const smg_experts *e, const uint16_t *x, int bf16, const int32_t *ids, const float *weights,
                               size_t rows, size_t top_k, uint16_t *out, void *scratch, size_t bytes, void *stream) {
    const OwnScratch own = {scratch, bytes};
    return guarded([&] { return experts_dev(e, x, bf16, ids, weights, rows, top_k, out, nullptr, stream, &own); });
}

int smg_experts_accumulate_ws_dev(const smg_experts *e, const uint16_t *x, int bf16, const int32_t *ids, const float *weights,
                                  size_t rows, size_t top_k, float *y, void *scratch, size_t bytes, void *stream) {
    const OwnScratch own = {scratch, bytes};
    return guarded([&] { return experts_dev(e, x, bf16, ids, weights, rows, top_k, nullptr, y, stream, &own); });
}

int smg_experts_forward(const smg_experts *e, const uint16_t *x, int bf16, const int32_t *ids, const float *weights, size_t rows,
                        size_t top_k, uint16_t *out) {
    return guarded([&] { return experts_host(e, x, bf16, ids, weights, rows, top_k, out, nullptr); });
}

int smg_experts_accumulate(const smg_experts *e, const uint16_t *x, int bf16, const int32_t *ids, const float *weights,
                           size_t rows, size_t top_k, float *y) {
    return guarded([&] { return experts_host(e, x, bf16, ids, weights, rows, top_k, nullptr, y); });
}

int smg_fp8_quantize(const float *w, int layout, size_t n, size_t k, uint8_t *codes, float *scales) {
    if (n && k && (!w || !codes || !scales)) return report(SMG_EINVAL, "null array");
    if (layout != 0 && layout != 1) return report(SMG_EINVAL, "layout is 0 (OutIn) or 1 (InOut)");
    auto at = [&](size_t j, size_t d) { return layout == 0 ? w[j * k + d] : w[d * n + j]; };
    const size_t nkb = (k + FP8_BLOCK - 1) / FP8_BLOCK;
    for (size_t j0 = 0; j0 < n; j0 += FP8_BLOCK)
        for (size_t d0 = 0; d0 < k; d0 += FP8_BLOCK) {
            const size_t j1 = std::min<size_t>(j0 + FP8_BLOCK, n), d1 = std::min<size_t>(d0 + FP8_BLOCK, k);
            float amax = 0.0f;
            for (size_t j = j0; j < j1; j++)
                for (size_t d = d0; d < d1; d++) {
                    const float a = std::fabs(at(j, d));
                    if (std::isfinite(a) && a > amax) amax = a;
                }
            // (a scale that rounds to zero or a subnormal would lose the codes)
            float s = amax / 448.0f;
            if (s < 1.17549435e-38f) s = amax > 0.0f ? 1.17549435e-38f : 1.0f;
            scales[j0 / FP8_BLOCK * nkb + d0 / FP8_BLOCK] = s;
            for (size_t j = j0; j < j1; j++)
                for (size_t d = d0; d < d1; d++) {
                    const float x = at(j, d);
                    codes[j * k + d] = std::isinf(x) ? e4m3_rne(NAN) : e4m3_rne(x / s);
                }
        }
    return SMG_OK;
}

int smg_fp8_create(const uint8_t *codes, const float *scales, size_t n, size_t k, smg_weights **out) {
    return guarded([&] { return fp8_create(codes, scales, n, k, 1, false, nullptr, out); });
}

int smg_fp8_create_dev(const uint8_t *codes, const float *scales, size_t n, size_t k, void *stream, smg_weights **out) {
    return guarded([&] { return fp8_create(codes, scales, n, k, 1, true, stream, out); });
}

int gemm_gpu_f16_fp8(size_t m, const smg_weights *w, uint16_t *dst, const uint16_t *lhs, const ep_desc16 *ep) {
    return guarded([&] { return fp8_host(m, w, dst, lhs, ep, false); });
}

int gemm_gpu_b16_fp8(size_t m, const smg_weights *w, uint16_t *dst, const uint16_t *lhs, const ep_desc16 *ep) {
    return guarded([&] { return fp8_host(m, w, dst, lhs, ep, true); });
}

int smg_fp8_matmul_dev(size_t m, const smg_weights *w, uint16_t *dst, const uint16_t *lhs, const ep_desc16 *ep, int bf16,
                       void *stream) {
    return guarded([&] { return fp8_dev(m, w, dst, lhs, ep, bf16, stream, nullptr); });
}

int smg_fp8_scratch_bytes(const smg_weights *w, size_t m, size_t *bytes) {
    int rc = check_fp8(w);
    if (rc) return rc;
    if (!bytes) return report(SMG_EINVAL, "null argument");
    if ((rc = check_rows(w, m))) return rc;
    *bytes = m && w->d.n ? fp8_scratch_bytes(w->f8, m) : 0;
    return SMG_OK;
}

int smg_fp8_matmul_ws_dev(size_t m, const smg_weights *w, uint16_t *dst, const uint16_t *lhs, const ep_desc16 *ep, int bf16,
                          void *scratch, size_t bytes, void *stream) {
    const OwnScratch own = {scratch, bytes};
    return guarded([&] { return fp8_dev(m, w, dst, lhs, ep, bf16, stream, &own); });
}

}  // extern "C"
