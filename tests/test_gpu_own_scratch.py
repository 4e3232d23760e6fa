"""Calls of the 8-bit products and the experts in the caller's scratch: the same bits, a
captured call's memory given back with its graph, refusals."""
import gc

import numpy as np
import pytest

import fp8_ref as ref
from test_gpu_experts import build, random_experts
from test_gpu_fp8 import bits, dev16, host16, run

pytestmark = pytest.mark.gpu


def bytes_of(n):
    import torch
    return torch.empty(n, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("m", [1, 20, 70, 300])
@pytest.mark.parametrize("k", [257, 1536, 2200])
def test_products_in_own_scratch(smg, m, k):
    import torch
    rng = np.random.default_rng(m + k)
    n = 300
    w = smg.Fp8Weights(*ref.random_weights(rng, n, k), n, k)
    for bf16 in (False, True):
        a = dev16(bits(rng.standard_normal((m, k)), bf16), bf16)
        bias = dev16(bits(rng.standard_normal(n), bf16), bf16)
        ep = smg.Epilogue(bf16).add_col(bias)
        want, plain = run(smg, a, w, m, bf16, ep), run(smg, a, w, m, bf16)
        need = w.scratch_bytes(m)
        s = torch.full((need + 64,), 0x5A, dtype=torch.uint8, device="cuda")
        c = torch.empty(m, n, dtype=a.dtype, device="cuda")
        (smg.matmul_fp8_bf16_ep if bf16 else smg.matmul_fp8_ep)(a, w, c, m, ep, scratch=s)
        assert np.array_equal(host16(c), want)
        (smg.matmul_fp8_bf16 if bf16 else smg.matmul_fp8)(a, w, c, m, scratch=s[:need])
        assert np.array_equal(host16(c), plain)
        assert bool((s[need:] == 0x5A).all())


@pytest.mark.parametrize("rows", [0, 1, 5, 40, 700])
@pytest.mark.parametrize("d", [131, 136])
def test_experts_in_own_scratch(smg, rows, d):
    """Rows at a multiple of 16 bytes and not (those are copied into the scratch first)."""
    import torch
    rng = np.random.default_rng(rows + d)
    experts, ffn, k = 6, 77, 3
    e = build(smg, random_experts(rng, experts, d, ffn), experts, d, ffn)
    x = dev16(bits(rng.standard_normal((rows, d)), False), False)
    off = torch.empty(rows * d + 1, dtype=torch.float16, device="cuda")[1:].view(rows, d)
    off.copy_(x)
    ids = torch.from_numpy(rng.integers(-1, experts, (rows, k)).astype(np.int32)).cuda()
    w = torch.from_numpy(rng.uniform(0.1, 1, (rows, k)).astype(np.float32)).cuda()
    want = torch.empty_like(x)
    e.forward(x, ids, w, want, rows)
    need = e.scratch_bytes(rows, k)
    for xi in (x, off):
        s = torch.full((need + 64,), 0x5A, dtype=torch.uint8, device="cuda")
        out, y = torch.full_like(x, 7), torch.zeros(rows, d, device="cuda")
        e.forward(xi, ids, w, out, rows, scratch=s)
        assert torch.equal(out, want)
        e.accumulate(xi, ids, w, y, rows, scratch=s[:need])
        assert torch.equal(y.half(), want)
        assert bool((s[need:] == 0x5A).all())


def test_memory_goes_with_the_graph(smg):
    """Twelve captures of a call with scratch of its own, from the graph's own memory:
    replayed beside eager calls, each ended before the next, and nothing is left of them."""
    import torch
    rng = np.random.default_rng(1)
    experts, d, ffn, k, rows = 8, 512, 512, 4, 6000
    e = build(smg, random_experts(rng, experts, d, ffn), experts, d, ffn)
    x = dev16(bits(rng.standard_normal((rows, d)), True), True)
    ids = torch.from_numpy(rng.integers(0, experts, (rows, k)).astype(np.int32)).cuda()
    w = torch.ones(rows, k, device="cuda")
    want, need = torch.empty_like(x), e.scratch_bytes(rows, k)
    e.forward(x, ids, w, want, rows)
    assert need > 60 << 20
    out = torch.empty_like(x)
    cap = torch.cuda.Stream()

    def left():
        gc.collect()
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        return torch.cuda.mem_get_info()[0]

    free = None
    for i in range(12):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=cap):
            e.forward(x, ids, w, out, rows, scratch=bytes_of(need))
        for _ in range(3):
            out.zero_()
            g.replay()
            e.forward(x, ids, w, out.clone(), rows)
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        del g
        free = left() if free is None else free
    assert left() > free - need, (left(), free)


def test_refusals(smg):
    import torch
    rng = np.random.default_rng(1)
    experts, d, ffn, k, m = 4, 64, 64, 2, 500
    e = build(smg, random_experts(rng, experts, d, ffn), experts, d, ffn)
    w = smg.Fp8Weights(*ref.random_weights(rng, 96, d), 96, d)
    x, c = torch.zeros(m, d, device="cuda").half(), torch.full((m, 96), 7.0, device="cuda").half()
    ids, wt = torch.zeros(m, k, dtype=torch.int32, device="cuda"), torch.zeros(m, k, device="cuda")
    out = torch.full((m, d), 7.0, device="cuda").half()
    for need, f in ((w.scratch_bytes(m), lambda s: smg.matmul_fp8(x, w, c, m, scratch=s)),
                    (e.scratch_bytes(m, k), lambda s: e.forward(x, ids, wt, out, m, scratch=s))):
        s = bytes_of(need + 512)
        assert need > 0 and s.data_ptr() % 256 == 0
        for bad in (s[:need // 2], s[1:], s[:0], s.cpu(), s.cpu().numpy(), s[::2], s.data_ptr()):
            with pytest.raises((ValueError, TypeError, smg.SmeGemmError)):
                f(bad)
    with pytest.raises(TypeError):
        smg.matmul_fp8(x.cpu().numpy(), w, np.zeros((m, 96), np.float16), m, scratch=s)
    torch.cuda.synchronize()
    assert bool((c == 7).all()) and bool((out == 7).all())
    L = smg.lib()
    host = np.zeros(1 << 22, np.uint8)
    stream = torch.cuda.current_stream().cuda_stream
    assert L.smg_fp8_matmul_ws_dev(m, w._h, c.data_ptr(), x.data_ptr(), None, 0, host.ctypes.data, host.size, stream) == -1
    assert L.smg_fp8_scratch_bytes(w._h, m, None) == -1 and L.smg_experts_scratch_bytes(e._h, m, k, None) == -1
    assert L.smg_fp8_matmul_ws_dev(1, w._h, c.data_ptr(), x.data_ptr(), None, 0, None, 0, stream) == 0  # (none needed)
    with pytest.raises(smg.SmeGemmError):
        e.scratch_bytes(m, 0)
    torch.cuda.synchronize()
