"""The experts' products element by element, over hidden values that have no rounding of
their own (experts_exact.py): parts of any size."""
import numpy as np
import pytest

import experts_exact as exact
from test_gpu_experts import build, run_experts
from test_gpu_fp8 import bits, check, dev16, host16, values

pytestmark = pytest.mark.gpu


def choose(rng, rows, experts, top_k):
    """Experts named by several rows, twice by a row, by none, and none at all."""
    ids = np.stack([rng.permutation(experts)[:top_k] for _ in range(rows)]).astype(np.int32)
    ids[rng.random((rows, top_k)) < 0.1] = -1
    if top_k > 1:
        ids[rows // 2, 1] = ids[rows // 2, 0]
    if rows > 1:
        ids[-1] = ids[0][::-1]
        ids[rows // 3, 0] = experts
    return ids


def accumulate(e, x, ids, w, y0, bf16):
    import torch
    y = torch.from_numpy(y0).cuda()
    e.accumulate(dev16(x, bf16), torch.from_numpy(ids).cuda(), torch.from_numpy(w).cuda(), y, len(x))
    return y.cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("scale", [2.0 ** 8, 2.0 ** -36])
@pytest.mark.parametrize("rows", [1, 48, 49, 300])
def test_parts_of_any_size(smg, rows, scale, bf16):
    """Parts past f16's largest, and below its steps: f32 rows get them whole, whatever
    the number of rows beside them."""
    rng = np.random.default_rng(rows)
    experts, d, ffn, k = 64, 72, 40, 8
    parts = exact.make(rng, experts, d, ffn, scale)
    e = build(smg, parts, experts, d, ffn)
    xv, ids = exact.rows_of(rng, rows, d), choose(rng, rows, experts, k)
    w = rng.uniform(0.1, 1, (rows, k)).astype(np.float32)
    want, off, size = exact.experts(xv, parts, ids, w)
    assert size.max() > 1e7 if scale > 1 else size.max() < 1e-5
    got = accumulate(e, bits(xv, bf16), ids, w, np.zeros((rows, d), np.float32), bf16)
    bad = ~(np.abs(got - want) <= off + 2.0 ** -24 * np.abs(want))
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[0], got[bad][0], want[bad][0])


@pytest.mark.parametrize("rows", [1, 48, 49, 300])
def test_parts_that_cancel(smg, rows):
    """Two experts of opposite output weights: parts past f16's largest whose sum is not."""
    rng = np.random.default_rng(rows)
    experts, d, ffn, k = 64, 72, 40, 8
    half = exact.make(rng, 1, d, ffn, 2.0 ** 3)
    other = (half[2][0] ^ 0x80, half[2][1], -half[2][2])
    parts = [tuple(np.concatenate([a] * experts) for a in p) for p in half[:2]]
    parts.append(tuple(np.concatenate([a, b] * (experts // 2)) for a, b in zip(half[2], other)))
    e = build(smg, parts, experts, d, ffn)
    ids = np.stack([rng.permutation(experts // 2)[:k // 2] for _ in range(rows)])
    ids = np.concatenate([2 * ids, 2 * ids + 1], 1).astype(np.int32)
    w = rng.uniform(0.1, 1, (rows, k // 2)).astype(np.float32)
    w = np.concatenate([w, w * np.float32(1 - 2.0 ** -14)], 1)
    xv = exact.rows_of(rng, rows, d)
    want, off, size = exact.experts(xv, parts, ids, w)
    assert size.max() > 1e6 and np.abs(want).max() < 1e4
    check(values(run_experts(e, bits(xv, False), ids, w, False), False), want, off, False, f"{rows} rows")
