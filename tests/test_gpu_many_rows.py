"""Calls of so many rows that a launch of a thread, or a few, for each would pass 2^32 threads
(such a launch runs their number modulo 2^32, without an error)."""
import numpy as np
import pytest

from test_gpu_experts import build, random_experts, run_experts
from test_gpu_fp8 import bits, dev16

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_back():
    """What these tests took does not stay in torch's cache."""
    yield
    import gc

    import torch
    gc.collect()
    torch.cuda.empty_cache()


def room(n):
    import torch
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < n:
        pytest.skip("not enough memory free")


# 16 lanes a row, and a wave a row
@pytest.mark.parametrize("rows,experts,top_k", [(2 ** 28 + 5, 2, 1), (2 ** 26 + 3, 17, 16)])
def test_routing(smg, rows, experts, top_k):
    import torch
    room(20 << 30)
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.empty(rows, experts, dtype=torch.float16, device="cuda").normal_(generator=g)
    ids = torch.full((rows, top_k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((rows, top_k), -7.0, device="cuda")
    smg.Router(experts, top_k).route(logits, None, ids, w, rows)
    assert int(ids.min()) >= 0 and float(w.min()) >= 0
    for at in (0, rows // 2, rows - 1000):
        l = logits[at:at + 1000].float()
        want = torch.sort(l, dim=1, descending=True, stable=True)
        assert torch.equal(ids[at:at + 1000], want.indices[:, :top_k].int())
        assert torch.allclose(w[at:at + 1000], torch.softmax(want.values[:, :top_k], 1), rtol=1e-5, atol=0)


@pytest.mark.parametrize("d", [16, 15])
def test_experts(smg, d):
    """Rows of a few kinds: equal rows give equal bits, to the last."""
    import torch
    room(40 << 30)
    rng = np.random.default_rng(d)
    rows, experts, ffn, kinds = 2 ** 24 + 3, 2, 16, 7
    e = build(smg, random_experts(rng, experts, d, ffn), experts, d, ffn)
    few = bits(rng.standard_normal((kinds, d)), True)
    ids, w = rng.integers(0, experts, (kinds, 1)).astype(np.int32), rng.uniform(0.1, 1, (kinds, 1)).astype(np.float32)
    many = 200  # (the tiles' form, as the long call's)
    at = np.arange(kinds * many) // many
    want = run_experts(e, few[at], ids[at], w[at], True)[::many]
    kind = torch.arange(rows, device="cuda") % kinds
    x = dev16(few, True)[kind]
    out = torch.full((rows, d), float("nan"), dtype=torch.bfloat16, device="cuda")
    e.forward(x, torch.from_numpy(ids).cuda()[kind], torch.from_numpy(w).cuda()[kind], out, rows)
    assert torch.equal(out, dev16(want, True)[kind])


def test_products_of_too_many_tiles_are_refused(smg):
    """2^30 rows of one column: 2^26 waves quantize them, 2^24 workgroups of 256 threads multiply."""
    import torch
    room(180 << 30)
    m = 2 ** 30
    w = smg.Fp8Weights(np.uint8([[0x38]]), np.float32([[1]]), 1, 1)
    a, c = torch.ones(m, 1, device="cuda", dtype=torch.float16), torch.full((m, 1), 7.0, device="cuda", dtype=torch.float16)
    scratch = torch.empty(w.scratch_bytes(m), dtype=torch.uint8, device="cuda")
    with pytest.raises(smg.SmeGemmError, match="too many rows"):
        smg.matmul_fp8(a, w, c, m, scratch=scratch)
    torch.cuda.synchronize()
    assert bool((c == 7).all())
    smg.matmul_fp8(a[:m // 2], w, c[:m // 2], m // 2, scratch=scratch)
    assert bool((c[:m // 2] == 1).all()) and bool((c[m // 2:] == 7).all())
