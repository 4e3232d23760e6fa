"""Experts whose hidden values have no rounding before their codes, so that every element
of the output can be held to the second product's own rounding.

Rows and gate and up weights are small integers (times powers of two): their codes are
exact, and so is every sum, in f32 and in the matrix cores (a product of 1 lies within
2^-13 of a group's largest, 3584). Depth 0 adds +-3584 to the gate, where silu(g) is g or
vanishes. A hidden value is then a multiple of 1/4 below 2^22, exact in f32, and its code
the nearest, ties to even, on the device as here."""
import numpy as np

import fp8_ref as ref


def code_of(values):
    """The codes of e4m3 values."""
    order = np.argsort(np.where(np.isnan(ref.VALUES), np.inf, ref.VALUES), kind="stable")
    at = np.searchsorted(ref.VALUES[order], np.asarray(values, np.float64))
    return order[np.minimum(at, 255)].astype(np.uint8)


SMALL = code_of([-2, -1, 0, 1, 2])


def make(rng, experts, d, ffn, down_scale=2.0 ** -16):
    """[(codes, scales, values)] of gate, up and down."""
    out = []
    for which in ("gate", "up"):
        codes = SMALL[rng.integers(0, 5, (experts, ffn, d))]
        shape = (experts, -(-ffn // 128), -(-d // 128))
        scales = (rng.choice([0.5, 1.0], shape) if d < 4000 else np.ones(shape)).astype(np.float32)
        if which == "gate":
            scales[:, :, 0] = 1
            codes[:, :, 0] = code_of(rng.choice([-448.0, 448.0], (experts, ffn), p=(0.1, 0.9)))
        else:
            codes[:, :, 0] = 0
        out.append((codes, scales))
    downs = [ref.random_weights(rng, d, ffn) for _ in range(experts)]
    out.append((np.stack([c for c, _ in downs]), np.stack([s for _, s in downs]) * np.float32(down_scale)))
    return [(c, s, np.stack([ref.weights(ci, si, *ci.shape) for ci, si in zip(c, s)])) for c, s in out]


def rows_of(rng, rows, d):
    x = rng.integers(-2, 3, (rows, d)).astype(np.float64)
    x[:, 0] = 8
    return x


def experts(x, parts, ids, w):
    """(the weighted sums, how far f32 sums of 8-bit products may be off, the sums of the
    parts' magnitudes): as fp8_ref.matmul's bound for each part; the weight joins by a
    rounding or two and the parts add up, 2^-24 each of the sum of magnitudes."""
    gate, up, down = (p[2] for p in parts)
    out, off, size = (np.zeros((len(x), down.shape[1])) for _ in range(3))
    assert np.array_equal(ref.quantize_rows(x), x)
    w = np.asarray(w, np.float64)
    for e in range(len(gate)):
        r, j = np.nonzero(ids == e)
        if not len(r):
            continue
        g, u = x[r] @ gate[e].T, x[r] @ up[e].T
        assert np.abs(g).min() > 1000
        h = np.where(g > 0, g * u, 0.0)
        assert np.abs(h).max() < 2.0 ** 22 and np.array_equal(h * 4, np.rint(h * 4))
        hq = ref.quantize_rows(h)
        p, o = ref.matmul(hq, down[e], quantized=True)
        mag = np.abs(hq) @ np.abs(down[e]).T
        wj = w[r, j][:, None]
        np.add.at(out, r, wj * p)
        np.add.at(off, r, np.abs(wj) * (o + (ids.shape[1] + 4) * 2.0 ** -24 * mag))
        np.add.at(size, r, np.abs(wj * p))
    return out, off, size
