"""The router's weights to f32's own rounding."""
import numpy as np
import pytest

import fp8_ref as ref
from test_gpu_experts import ROUTES, route

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("spread", [0.1, 2.0, 30.0])
def test_weights_of_64_bit_scores(smg, spread, renormalize, biased, sigmoid):
    """Scores and their quotients are of 64 bits, then rounded once: 2^-24, with as much again
    for what 64 bits lose. But for a softmax's sum where the logits alone decide: of f32
    powers e^x, x = l - max, whose difference, product with log2 e and 2^x round by 2^-24 (1 +
    2 |x|) or less, and of at most 16 additions a lane; the sum of |x| e^x over the sum of
    e^x is below ln 1024 = 7, so 2^-24 (2 + 14 + 16) = 2^-19, and it divides only weights that are not
    renormalized."""
    import torch
    rng = np.random.default_rng(int(spread * 10))
    for rows, experts, top_k, groups, top_groups in ROUTES:
        logits = (rng.standard_normal((rows, experts)) * spread).astype(np.float32)
        bias = (0.05 * rng.standard_normal(experts)).astype(np.float32) if biased else None
        r = smg.Router(experts, top_k, smg.Score.Sigmoid if sigmoid else smg.Score.Softmax, groups=groups, top_groups=top_groups,
                       renormalize=renormalize, scale=1.5)
        ids, w = route(smg, r, torch.from_numpy(logits).cuda(), bias)
        want_ids, want = ref.route(logits, bias, top_k, sigmoid, groups, top_groups, renormalize, 1.5)
        assert np.array_equal(ids, want_ids)
        f32_sum = not (sigmoid or renormalize or biased or groups > 1)
        off = np.abs(w - want)
        assert (off <= (2.0 ** -18 if f32_sum else 2.0 ** -23) * want + 2.0 ** -149).all(), (rows, experts, (off / want).max())
