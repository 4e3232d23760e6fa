"""The experts' products element by element, over hidden values that have no rounding of
their own (experts_exact.py): every form's loops, decode calls of many experts, parts of
any size, weights past 4 GB."""
import numpy as np
import pytest

import experts_exact as exact
import fp8_ref as ref
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


def check_both(smg, e, parts, xv, ids, w, bf16, what, y0=None):
    """forward and accumulate."""
    want, off, size = exact.experts(xv, parts, ids, w)
    x = bits(xv, bf16)
    check(values(run_experts(e, x, ids, w, bf16), bf16), want, off, bf16, what)
    y0 = np.zeros(want.shape, np.float32) if y0 is None else y0
    got = accumulate(e, x, ids, w, y0, bf16)
    tol = off + 2.0 ** -24 * (np.abs(want) + 2 * np.abs(y0)) + 2.0 ** -149
    bad = ~(np.abs(got - y0 - want) <= tol)
    assert not bad.any(), f"{what}, accumulate: {bad.sum()} of {bad.size}, first {np.argwhere(bad)[0]}: " \
                          f"{(got - y0)[bad][0]} for {want[bad][0]} (tol {tol[bad][0]})"


# (rows, d, ffn, experts, top_k): one row, and past the blocks its waves hold at once (24 of
# d, 64 of its experts' ffn); few rows, with no more assignments than experts and more, past
# 16 blocks of either width; tiles of few and of many experts, past 64 blocks of either
# width; the last call of the few rows' form and the first of the tiles'
SHAPES = [(1, 64, 64, 4, 2), (1, 513, 130, 8, 6), (1, 3300, 200, 3, 2), (1, 130, 2200, 5, 4), (2, 200, 130, 64, 6),
          (5, 136, 200, 64, 6), (8, 129, 96, 70, 8), (17, 200, 96, 6, 2), (60, 128, 384, 4, 2), (5, 2300, 140, 3, 2),
          (20, 140, 2300, 3, 2), (300, 256, 128, 8, 2), (513, 130, 200, 3, 1), (400, 130, 96, 128, 2), (500, 40, 24, 1024, 2),
          (200, 8400, 64, 2, 2), (200, 70, 8400, 2, 2), (48, 100, 72, 64, 8), (49, 100, 72, 64, 8), (700, 300, 260, 2, 2)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,d,ffn,experts,top_k", SHAPES)
def test_every_element(smg, rows, d, ffn, experts, top_k, bf16):
    rng = np.random.default_rng(rows * 41 + d + experts)
    parts = exact.make(rng, experts, d, ffn)
    e = build(smg, parts, experts, d, ffn)
    w = rng.uniform(0.1, 1, (rows, top_k)).astype(np.float32)
    y0 = rng.standard_normal((rows, d)).astype(np.float32)
    check_both(smg, e, parts, exact.rows_of(rng, rows, d), choose(rng, rows, experts, top_k), w, bf16,
               f"{rows} rows, {top_k} of {experts}, {d} to {ffn}", y0)


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


def test_a_lost_element_is_seen():
    """Planted in the oracle's own result: an element set to zero, or to its neighbour's,
    fails the bound nearly everywhere (its values are not all far from zero)."""
    rng = np.random.default_rng(0)
    for rows, d, ffn, experts, top_k in ((60, 128, 384, 4, 2), (20, 140, 2300, 3, 2)):
        parts = exact.make(rng, experts, d, ffn)
        want, off, _ = exact.experts(exact.rows_of(rng, rows, d), parts, choose(rng, rows, experts, top_k),
                                     rng.uniform(0.1, 1, (rows, top_k)))
        live = np.abs(want).sum(1) > 0
        for other in (np.zeros_like(want), np.roll(want, 1, 1)):
            tol = ref.half_step(True) * (np.abs(want) + off) + off
            assert (np.abs(other - want) <= tol)[live].mean() < 0.04


@pytest.mark.parametrize("rows", [1, 7, 500])
def test_experts_past_4_gb(smg, rows):
    """Offsets of more than 32 bits within a matrix: the first experts, the last and those
    around 2^32 bytes."""
    import torch
    rng = np.random.default_rng(rows)
    experts, d, ffn, k = 1024, 2048, 2100, 3
    assert experts * d * ffn > 2 ** 32
    g = torch.Generator(device="cuda").manual_seed(rows)
    small = torch.from_numpy(exact.SMALL).cuda()
    plus, minus = (int(exact.code_of(v)) for v in (448.0, -448.0))

    def codes(n, kk):
        return torch.cat([small[torch.randint(0, 5, (64, n, kk), device="cuda", generator=g)] for _ in range(experts // 64)])

    gate, up, down = codes(ffn, d), codes(ffn, d), codes(d, ffn)
    gate[:, :, 0] = torch.where(torch.rand(experts, ffn, device="cuda", generator=g) < 0.1, minus, plus).to(torch.uint8)
    up[:, :, 0] = 0
    ones = torch.ones(experts, -(-ffn // 128), -(-d // 128), device="cuda")
    low = torch.full((experts, -(-d // 128), -(-ffn // 128)), 2.0 ** -22, device="cuda")
    at = 2 ** 32 // (d * ffn)
    used = [0, 1, at - 1, at, at + 1, experts - 1]
    parts = [(None, None, np.stack([ref.VALUES[m[i].cpu().numpy()] * s for i in used]))
             for m, s in ((gate, 1.0), (up, 1.0), (down, 2.0 ** -22))]
    e = smg.Experts(gate, ones, up, ones, down, low, experts, d, ffn)
    del gate, up, down
    few = choose(rng, rows, len(used), k)
    ids = np.where((few >= 0) & (few < len(used)), np.int32(used)[np.clip(few, 0, len(used) - 1)], -1).astype(np.int32)
    few = np.where(ids < 0, -1, few)
    w = rng.uniform(0.1, 1, (rows, k)).astype(np.float32)
    xv = exact.rows_of(rng, rows, d)
    want, off, _ = exact.experts(xv, parts, few, w)
    check(values(run_experts(e, bits(xv, True), ids, w, True), True), want, off, True, f"{rows} rows")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_hidden_values_keep_their_codes(smg, rows, bf16):
    """Random weights: the error of the whole by its 2-norm. f32 sums of a few thousand
    products are off by less than 2^-21 of their 2-norm, and the hidden values by twice that;
    codes lie 2^-4 of a value apart or more, so one in 2^-20 2^5 takes its neighbour, a step of
    2^-3 of it at most: sqrt(2^-15) 2^-3 = 2^-10.5 of the whole. The second product's dropped
    bits (2^-16) and an f16 result's rounding (2^-11 / sqrt(3)) add up to less than 2^-11.5.
    In f32 rows the same without the rounding; bf16 results are not held to it."""
    rng = np.random.default_rng(rows)
    experts, d, ffn, k = 4, 2048, 768, 2
    parts = []
    for n, kk in ((ffn, d), (ffn, d), (d, ffn)):
        v = ref.e4m3_round(np.clip(rng.standard_normal((experts, n, kk)) * 112, -448, 448))
        s = (rng.uniform(0.7, 1.3, (experts, -(-n // 128), -(-kk // 128))) / (112 * np.sqrt(kk))).astype(np.float32)
        c = exact.code_of(v)
        parts.append((c, s, np.stack([ref.weights(ci, si, n, kk) for ci, si in zip(c, s)])))
    e = build(smg, parts, experts, d, ffn)
    x = bits(rng.standard_normal((rows, d)), bf16)
    ids = np.stack([rng.permutation(experts)[:k] for _ in range(rows)]).astype(np.int32)
    w = rng.uniform(0.1, 1, (rows, k)).astype(np.float32)
    a, want = ref.quantize_rows(values(x, bf16)), np.zeros((rows, d))
    for i in range(experts):
        r, j = np.nonzero(ids == i)
        h = ref.act(a[r] @ parts[0][2][i].T, False) * (a[r] @ parts[1][2][i].T)
        np.add.at(want, r, w[r, j][:, None].astype(np.float64) * (ref.quantize_rows(h) @ parts[2][2][i].T))
    got = [accumulate(e, x, ids, w, np.zeros((rows, d), np.float32), bf16)]
    if not bf16:
        got.append(values(run_experts(e, x, ids, w, False), False))
    for g in got:
        err = np.linalg.norm(g - want) / np.linalg.norm(want)
        assert err < 2.0 ** -10, err


@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("rows", [1, 3, 60, 500])
def test_gates_whose_power_is_no_f32(smg, rows, gelu):
    """Gates of -72 .. -120 (gelu: -8 .. -12), where g / (1 + e^-y) lies below f32's normal
    range, times up values that bring it back: the second product is the identity, so the
    outputs are the hidden values' codes, those within 2^-10 of a border aside (the hardware's
    2^x of arguments up to 2^8 is off by 2^-15)."""
    rng = np.random.default_rng(rows)
    n, gates = 128, -np.float64(np.arange(8, 13) if gelu else np.arange(72, 121, 8))
    experts = len(gates)
    y = 2 * 0.7978845608028654 * (gates + 0.044715 * gates ** 3) if gelu else gates
    up = rng.choice(ref.VALUES[0x38:0x58], (experts, n, n))  # 1 .. 15
    h = (gates * np.exp(y) / (1 + np.exp(y)))[:, None, None] * up * 2.0 ** 100
    back = 2.0 ** -np.round(np.log2(np.abs(h).max((1, 2)) / 64))
    ones = np.ones((experts, 1, 1))
    gate = np.broadcast_to(exact.code_of(gates)[:, None, None], (experts, n, n))
    e = smg.Experts(gate, np.float32(ones), exact.code_of(up), np.float32(ones * 2.0 ** 100),
                    np.broadcast_to(np.where(np.eye(n, dtype=bool), 0x38, 0).astype(np.uint8), (experts, n, n)),
                    np.float32(ones * back[:, None, None]), experts, n, n, smg.Gate.Gelu if gelu else smg.Gate.Silu)
    at, ids = rng.integers(0, n, rows), rng.integers(0, experts, (rows, 1)).astype(np.int32)
    x = np.zeros((rows, n))
    x[np.arange(rows), at] = 1
    hr = h[ids[:, 0], :, at]
    want = ref.quantize_rows(hr)
    clear = (ref.quantize_rows(hr * (1 + 2.0 ** -10)) == want) & (ref.quantize_rows(hr * (1 - 2.0 ** -10)) == want)
    # (a whole row's exponent changes with its largest value)
    clear &= clear[np.arange(rows), np.abs(hr).argmax(1)][:, None]
    assert clear.mean() > 0.8
    want *= back[ids]
    for bf16 in (False, True):
        b, w = bits(x, bf16), np.ones((rows, 1), np.float32)
        got = values(run_experts(e, b, ids, w, bf16), bf16)
        acc = accumulate(e, b, ids, w, np.zeros((rows, n), np.float32), bf16)
        for g in (got, acc):
            assert np.array_equal(g[clear], want[clear]), (np.argwhere(clear & (g != want))[0], (clear & (g != want)).sum())


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows", [1, 5, 40, 400])
def test_nan_codes_and_rows(smg, rows, bf16):
    """A NaN code of a gate or up matrix makes the rows of its expert NaN, one of a down matrix
    that column of them; a NaN or infinite activation its row. Nothing else changes."""
    rng = np.random.default_rng(rows)
    experts, d, ffn, k = 6, 140, 136, 2
    parts = exact.make(rng, experts, d, ffn)
    xv, w = exact.rows_of(rng, rows, d), rng.uniform(0.1, 1, (rows, k)).astype(np.float32)
    ids = np.stack([rng.permutation(experts)[:k] for _ in range(rows)]).astype(np.int32)
    plain = build(smg, parts, experts, d, ffn)
    want = [values(run_experts(plain, bits(xv, bf16), ids, w, bf16), bf16),
            accumulate(plain, bits(xv, bf16), ids, w, np.zeros((rows, d), np.float32), bf16)]
    for which, at in ((0, (1, 77, 3)), (1, (2, 135, 139)), (2, (3, 99, 130))):
        bad = [tuple(np.copy(a) for a in p) for p in parts]
        bad[which][0][at] = 0x7F if which else 0xFF
        e = build(smg, bad, experts, d, ffn)
        hit = np.zeros((rows, d), bool)
        hit[(ids == at[0]).any(1), at[1] if which == 2 else slice(None)] = True
        got = [values(run_experts(e, bits(xv, bf16), ids, w, bf16), bf16),
               accumulate(e, bits(xv, bf16), ids, w, np.zeros((rows, d), np.float32), bf16)]
        for g, x in zip(got, want):
            assert np.array_equal(np.isnan(g), hit) and np.array_equal(g[~hit], x[~hit]), which
    for v in (np.nan, np.inf, -np.inf):
        x = xv.copy()
        x[rows // 2, 133] = v
        got = [values(run_experts(plain, bits(x, bf16), ids, w, bf16), bf16),
               accumulate(plain, bits(x, bf16), ids, w, np.zeros((rows, d), np.float32), bf16)]
        for g, y in zip(got, want):
            hit = np.arange(rows) == rows // 2
            assert np.isnan(g[hit]).all() and np.array_equal(g[~hit], y[~hit])
