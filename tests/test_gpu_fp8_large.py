"""8-bit weights past 64 GiB: more 16-byte pieces than one launch has threads."""
import numpy as np
import pytest

import fp8_ref as ref
from test_gpu_fp8 import check, host16, values

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_back():
    """What these tests took does not stay in torch's cache."""
    yield
    import gc

    import torch
    gc.collect()
    torch.cuda.empty_cache()


def test_weights_past_64_gib(smg):
    import torch
    n, k = 65664, 1 << 20
    assert n * k > 2 ** 36
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 2.2 * n * k:
        pytest.skip("no room for two copies")
    g = torch.Generator(device="cuda").manual_seed(1)
    codes = torch.zeros(n, k, dtype=torch.uint8, device="cuda")
    at = [0, 129, n // 2, 2 ** 36 // k - 1, 2 ** 36 // k, n - 1]
    for c in at:
        codes[c] = torch.randint(0, 126, (k,), dtype=torch.uint8, device="cuda", generator=g)
    sub = codes[at].cpu().numpy()
    scales = (torch.rand(n // 128, k // 128, device="cuda", generator=g) + 0.5) / (180 * k ** 0.5)
    sc = scales[[c // 128 for c in at]].cpu().numpy().astype(np.float64)
    w = smg.Fp8Weights(codes, scales, n, k)
    del codes
    x = torch.randn(2, k, device="cuda", generator=g).bfloat16()
    c = torch.full((2, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    smg.matmul_fp8_bf16(x, w, c, 2)
    want, off = ref.matmul(values(host16(x), True), ref.VALUES[sub] * np.repeat(sc, 128, 1))
    got = values(host16(c), True)
    check(got[:, at], want, off, True, "the columns that are not zero")
    got[:, at] = 0
    assert not got.any()
