"""Performance cases of the 8-bit floating-point products and the mixture of
experts: the block-scaled product (``matmul_fp8``), routing (``Router.route``)
and the experts' products (``Experts.forward``), from one token to a long
prompt. ``own`` false computes them from elementary torch operations, true
through ``smegemm`` on device tensors, on torch's current stream.

A case is a dict: ``op``, its sizes and its options. ``listed()`` names the fixed
ones, ``draw()`` gives others of the same ranges, ``prepare`` makes a program's
state, ``run`` is one pass, ``exact`` the same result in 64 bits.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
BLK = 128  # depths, and columns, that share a scale


def _smg():
    p = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sme-gemm_amd")
    if p not in sys.path:
        sys.path.insert(0, p)
    import smegemm
    return smegemm


def listed():
    return [
        # A small model's projection, one token: the smallest call, all latency.
        dict(name="fp8_decode_small", op="fp8", m=1, n=1536, k=384, bf16=False, ep="none"),
        # A 4096-wide model's square projection, one token.
        dict(name="fp8_decode", op="fp8", m=1, n=4096, k=4096, bf16=True, ep="none"),
        # A batch of sequences decoding together: ragged rows and columns, bias
        # and activation.
        dict(name="fp8_batch", op="fp8", m=29, n=11003, k=4096, bf16=True, ep="bias_silu"),
        # A prompt's up projection: column scale, bias, activation.
        dict(name="fp8_prefill", op="fp8", m=512, n=14336, k=4096, bf16=False, ep="scale_bias_silu"),
        # Long prompts of a batch through the same projection.
        dict(name="fp8_gemm", op="fp8", m=4096, n=14336, k=4096, bf16=True, ep="none"),
        # One generated token's choice of experts.
        dict(name="route_token", op="route", rows=1, experts=64, top_k=6, score="softmax", bias=False, groups=1,
             top_groups=1, renorm=True, logits="f16", masked=False),
        # A ragged prompt, a number of experts that is no power of two, some
        # of them masked.
        dict(name="route_odd", op="route", rows=777, experts=60, top_k=4, score="softmax", bias=False, groups=1,
             top_groups=1, renorm=False, logits="bf16", masked=True),
        # Long prompts: sigmoid scores, a balancing bias, 4 of 8 groups.
        dict(name="route_prompt", op="route", rows=8192, experts=256, top_k=8, score="sigmoid", bias=True, groups=8,
             top_groups=4, renorm=True, logits="f32", masked=False),
        # One generated token through its 6 of 64 experts.
        dict(name="experts_token", op="experts", rows=1, d=2048, ffn=1280, experts=64, top_k=6, bf16=True, drop=0.0),
        # A batch of sequences decoding together, some of its rows padding.
        dict(name="experts_batch", op="experts", rows=37, d=4096, ffn=1792, experts=64, top_k=8, bf16=True, drop=0.1),
        # A prompt through many small experts, of an odd width.
        dict(name="experts_many", op="experts", rows=3001, d=2048, ffn=1000, experts=128, top_k=8, bf16=False, drop=0.0),
        # A long prompt through few large experts.
        dict(name="experts_prefill", op="experts", rows=2048, d=4096, ffn=14336, experts=8, top_k=2, bf16=True, drop=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, odd):
    """A layer width: a multiple of 128 as models have, or (odd) any size."""
    x = _log(rng, lo, hi)
    return x if odd else max(128, x // 128 * 128)


# The most a drawn case costs (operations): under the largest listed ones.
_MOST = {"fp8": 4.5e11, "experts": 1.4e12}


def draw(rng):
    op = rng.choice(["fp8", "fp8", "fp8", "route", "route", "experts", "experts", "experts"])
    while True:
        odd = rng.random() < 0.35
        if op == "fp8":
            c = dict(op=op, m=rng.choice([1, _log(rng, 2, 32), _log(rng, 33, 4096), _log(rng, 33, 4096)]),
                     n=_width(rng, 384, 16384, odd), k=_width(rng, 256, 14336, odd), bf16=rng.random() < 0.5,
                     ep=rng.choice(["none", "bias_silu", "scale_bias_silu"]))
        elif op == "route":
            experts = rng.choice([8, 16, 60, 64, 96, 128, 160, 256, 384])
            groups = rng.choice([1, 1, 2, 4])
            top_groups = rng.randint(1, groups)
            top_k = rng.randint(1, min(10, experts // groups * top_groups))
            return dict(op=op, rows=rng.choice([1, _log(rng, 2, 64), _log(rng, 65, 8192), _log(rng, 65, 8192)]),
                        experts=experts, top_k=top_k, score=rng.choice(["softmax", "sigmoid"]),
                        bias=rng.random() < 0.5, groups=groups, top_groups=top_groups, renorm=rng.random() < 0.6,
                        logits=rng.choice(["f32", "f16", "bf16"]), masked=rng.random() < 0.3)
        else:
            d, ffn, experts, top_k = rng.choice([(2048, 1280, 64, 6), (4096, 1792, 64, 8), (2048, 1024, 128, 8),
                                                 (4096, 14336, 8, 2), (1024, 512, 32, 4), (1024, 2816, 16, 2)])
            if odd:
                d, ffn = _log(rng, 512, 4096), _log(rng, 256, 2048)
            c = dict(op=op, rows=rng.choice([1, _log(rng, 2, 32), _log(rng, 33, 4096), _log(rng, 33, 4096)]), d=d,
                     ffn=ffn, experts=experts, top_k=top_k, bf16=rng.random() < 0.5, drop=rng.choice([0.0, 0.0, 0.15]))
        if work(c)["flops"] <= _MOST[op]:
            return c


# ---- inputs -------------------------------------------------------------------

_FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class _Rng:
    """Seeded inputs, made on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device=DEV)

    def uniform(self, lo, hi, *shape):
        return torch.rand(shape, generator=self.g, device=DEV) * (hi - lo) + lo


def _nb(x):
    return -(-x // BLK)


def _weights(r, n, k):
    """A checkpoint's weights: e4m3 codes [n][k] (as uint8 bits) and an f32
    scale for each 128 x 128 block, so that a column's values have a standard
    deviation of about 1 / sqrt(k)."""
    codes = r.normal(n, k).mul_(112.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, r.uniform(0.7, 1.3, _nb(n), _nb(k)) / (112.0 * math.sqrt(k))


def _inputs(case, seed):
    """Everything `case` is computed from: the same for prepare and exact."""
    r, op, i = _Rng(seed), case["op"], {}
    if op == "fp8":
        t = torch.bfloat16 if case["bf16"] else torch.float16
        i["codes"], i["scales"] = _weights(r, case["n"], case["k"])
        # some columns of the activations are far larger than the rest
        a = r.normal(case["m"], case["k"]) * torch.where(r.uniform(0, 1, case["k"]) < 0.01, 20.0, 1.0)
        i["a"] = a.to(t)
        i["cs"] = r.uniform(0.5, 1.5, case["n"]).to(t) if "scale" in case["ep"] else None
        i["cb"] = (0.1 * r.normal(case["n"])).to(t) if "bias" in case["ep"] else None
    elif op == "route":
        lo = r.normal(case["rows"], case["experts"])
        if case["masked"]:
            lo = torch.where(r.uniform(0, 1, case["rows"], case["experts"]) < 0.2, -math.inf, lo)
            lo[case["rows"] // 2:case["rows"] // 2 + 1] = -math.inf  # a row of padding
        i["logits"] = lo.to(_FLOAT[case["logits"]])
        i["bias"] = 0.05 * r.normal(case["experts"]) if case["bias"] else None
    else:
        rows, d, ffn, experts, k = (case[x] for x in ("rows", "d", "ffn", "experts", "top_k"))
        t = torch.bfloat16 if case["bf16"] else torch.float16
        for name, n, kk in (("gate", ffn, d), ("up", ffn, d), ("down", d, ffn)):
            i[name] = torch.empty(experts, n, kk, dtype=torch.uint8, device=DEV)
            i[name + "_s"] = torch.empty(experts, _nb(n), _nb(kk), device=DEV)
            for e in range(experts):
                i[name][e], i[name + "_s"][e] = _weights(r, n, kk)
        i["x"] = r.normal(rows, d).to(t)
        # experts are not equally popular
        lo = r.normal(rows, experts) + 0.5 * r.normal(experts)
        top = torch.topk(lo, k, dim=1)
        i["ids"] = top.indices.to(torch.int32)
        i["w"] = torch.softmax(top.values, 1)
        if case["drop"]:
            i["ids"] = torch.where(r.uniform(0, 1, rows, 1) < case["drop"], -1, i["ids"])
    return i


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    op = case["op"]
    if not own:
        return s
    smg = _smg()
    if op == "fp8":
        s["weights"] = smg.Fp8Weights(s.pop("codes"), s.pop("scales"), case["n"], case["k"])
        s["c"] = torch.empty(case["m"], case["n"], dtype=s["a"].dtype, device=DEV)
        ep = smg.Epilogue(case["bf16"])
        if s["cs"] is not None:
            ep = ep.mul_col(s["cs"])
        if s["cb"] is not None:
            ep = ep.add_col(s["cb"]).silu()
        s["ep"] = ep
    elif op == "route":
        score = smg.Score.Softmax if case["score"] == "softmax" else smg.Score.Sigmoid
        s["router"] = smg.Router(case["experts"], case["top_k"], score, groups=case["groups"],
                                 top_groups=case["top_groups"], renormalize=case["renorm"], scale=1.0)
        s["ids"] = torch.empty(case["rows"], case["top_k"], dtype=torch.int32, device=DEV)
        s["w"] = torch.empty(case["rows"], case["top_k"], device=DEV)
    else:
        parts = [s.pop(x) for x in ("gate", "gate_s", "up", "up_s", "down", "down_s")]
        s["experts"] = smg.Experts(*parts, case["experts"], case["d"], case["ffn"], smg.Gate.Silu)
        s["out"] = torch.empty_like(s["x"])
    return s


# ---- one pass -----------------------------------------------------------------

def _dequant(codes, scales):
    """Weights (..., n, k) in 32 bits: each code times its block's scale."""
    n, k = codes.shape[-2:]
    s = scales.repeat_interleave(BLK, -2)[..., :n, :].repeat_interleave(BLK, -1)[..., :k]
    return codes.view(torch.float8_e4m3fn).float() * s


def _quantized(x):
    """x (rows, k) in 32 bits, each row's block of 128 rounded to e4m3 times the
    least power of two (2^-126 at least) that takes its largest finite
    magnitude to 448 or less; the values the codes stand for."""
    rows, k = x.shape
    b = torch.nn.functional.pad(x, (0, -k % BLK)).reshape(rows, -1, BLK)
    amax = torch.where(torch.isfinite(b), b.abs(), 0.0).amax(2, keepdim=True)
    # exponent and 1.75 = 448 / 256 compared on the bits
    e = (((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp_(min=1)
    up, down = ((254 - e) << 23).view(torch.float32), (e << 23).view(torch.float32)
    q = (b * up).to(torch.float8_e4m3fn).float() * down
    return q.reshape(rows, -1)[:, :k]


def _plain_fp8(s):
    t = s["a"].dtype
    c = (_quantized(s["a"].float()) @ _dequant(s["codes"], s["scales"]).t()).to(t)
    if s["cb"] is None:
        return c
    x = c.float() * s["cs"].float() if s["cs"] is not None else c.float()
    x = x + s["cb"].float()
    return (x / (1.0 + torch.exp(-x))).to(t)


def _plain_route(s):
    case = s["case"]
    rows, experts, k, groups = case["rows"], case["experts"], case["top_k"], case["groups"]
    lo = s["logits"].double()
    off = lo == -math.inf
    if case["score"] == "softmax":
        e = torch.where(off, 0.0, torch.exp(lo - lo.amax(1, keepdim=True)))
        score = e / e.sum(1, keepdim=True).clamp_min(1e-300)
    else:
        score = 1.0 / (1.0 + torch.exp(-lo))
    choice = score if s["bias"] is None else score + s["bias"].double()
    choice = torch.where(off, -math.inf, choice)
    if groups > 1:
        two = choice.reshape(rows, groups, -1).sort(dim=2, descending=True).values[:, :, :2]
        total = torch.where(two == -math.inf, 0.0, two).sum(2)
        total = torch.where(two[:, :, 0] == -math.inf, -math.inf, total)
        first = total.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = torch.zeros(rows, groups, dtype=torch.bool, device=DEV).scatter_(1, first, True)
        choice = torch.where(kept.repeat_interleave(experts // groups, 1), choice, -math.inf)
    best = choice.sort(dim=1, descending=True, stable=True)
    ids, none = best.indices[:, :k], best.values[:, :k] == -math.inf
    w = torch.where(none, 0.0, score.gather(1, ids))
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
    return torch.where(none, -1, ids).to(torch.int32), w.float()


def _plain_experts(s):
    case = s["case"]
    rows, k, d = case["rows"], case["top_k"], case["d"]
    flat = s["ids"].reshape(-1).long()
    live = (flat >= 0).nonzero().reshape(-1)
    x = _quantized(s["x"].float())
    used, which, counts = flat[live].unique(return_inverse=True, return_counts=True)
    if not used.numel():
        return torch.zeros_like(s["x"])
    # each used expert's rows side by side, padded to the most that one has
    order = which.sort(stable=True).indices
    place = torch.arange(order.numel(), device=DEV) - (counts.cumsum(0) - counts)[which[order]]
    most, slot, live = int(counts.max()), which[order], live[order]
    xs = torch.zeros(used.numel(), most, d, device=DEV)
    xs[slot, place] = x[live // k]
    weights = [_dequant(s[n][used], s[n + "_s"][used]) for n in ("gate", "up", "down")]
    g, u = xs @ weights[0].transpose(1, 2), xs @ weights[1].transpose(1, 2)
    h = g / (1.0 + torch.exp(-g)) * u
    h = _quantized(h.reshape(-1, case["ffn"])).reshape(h.shape)
    y = torch.zeros(rows * k, d, device=DEV)
    y[live] = (h @ weights[2].transpose(1, 2))[slot, place] * s["w"].reshape(-1)[live].unsqueeze(1)
    return y.reshape(rows, k, d).sum(1).to(s["x"].dtype)


def run(s):
    op, case = s["case"]["op"], s["case"]
    if not own:
        return {"fp8": _plain_fp8, "route": _plain_route, "experts": _plain_experts}[op](s)
    smg = _smg()
    if op == "fp8":
        f = smg.matmul_fp8_bf16_ep if case["bf16"] else smg.matmul_fp8_ep
        return f(s["a"], s["weights"], s["c"], case["m"], s["ep"])
    if op == "route":
        return s["router"].route(s["logits"], s["bias"], s["ids"], s["w"], case["rows"])
    return s["experts"].forward(s["x"], s["ids"], s["w"], s["out"], case["rows"])


# ---- what a pass cannot do without --------------------------------------------

def _bytes(n, k):
    return n * k + 4 * _nb(n) * _nb(k)


def work(case):
    op = case["op"]
    if op == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        vec = 2 * n * (("scale" in case["ep"]) + ("bias" in case["ep"]))
        return {"bytes": _bytes(n, k) + 2 * m * k + 2 * m * n + vec, "flops": 2 * m * n * k}
    if op == "route":
        rows, experts = case["rows"], case["experts"]
        size = 4 if case["logits"] == "f32" else 2
        return {"bytes": rows * (experts * size + case["top_k"] * 8) + 4 * experts * case["bias"],
                "flops": rows * experts * 2}
    rows, d, ffn, experts, k = (case[x] for x in ("rows", "d", "ffn", "experts", "top_k"))
    live = rows * k * (1.0 - case["drop"])
    used = experts * (1.0 - (1.0 - k / experts) ** (rows * (1.0 - case["drop"])))  # experts that a row uses
    return {"bytes": used * (2 * _bytes(ffn, d) + _bytes(d, ffn)) + 4 * rows * d + 8 * rows * k,
            "flops": 6 * live * d * ffn}


# ---- the same in 64 bits -------------------------------------------------------

def _block_rounded64(x):
    """The codes' values of x (rows, k) in 64 bits."""
    out = torch.empty_like(x)
    for b in range(0, x.shape[1], BLK):
        v = x[:, b:b + BLK]
        m, e = torch.frexp(v.abs().amax(1, keepdim=True))  # amax = m 2^e, m in [0.5, 1)
        p = torch.pow(2.0, (e - 9 + (m > 0.875)).clamp_min(-126).double())
        out[:, b:b + BLK] = (v / p).float().to(torch.float8_e4m3fn).double() * p
    return out


def _weights64(codes, scales):
    w = codes.view(torch.float8_e4m3fn).double()
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            w[i * BLK:(i + 1) * BLK, j * BLK:(j + 1) * BLK] *= scales[i, j].double()
    return w


def _exact_route(case, i):
    lo = i["logits"].double().cpu()
    bias = torch.zeros(case["experts"], dtype=torch.float64) if i["bias"] is None else i["bias"].double().cpu()
    score = torch.softmax(lo, 1) if case["score"] == "softmax" else torch.sigmoid(lo)
    per = case["experts"] // case["groups"]
    ids, weights = [], []
    for row, sc in zip(lo.tolist(), score.tolist()):
        left = {e: sc[e] + b for e, b in enumerate(bias.tolist()) if row[e] > -math.inf}
        if case["groups"] > 1:
            total = {}
            for e in sorted(left, key=lambda e: -left[e]):
                total.setdefault(e // per, []).append(left[e])
            best = sorted(total, key=lambda g: (-sum(total[g][:2]), g))[:case["top_groups"]]
            left = {e: c for e, c in left.items() if e // per in best}
        chosen = sorted(left, key=lambda e: (-left[e], e))[:case["top_k"]]
        w = [sc[e] for e in chosen]
        if case["renorm"] and sum(w) > 0:
            w = [x / sum(w) for x in w]
        rest = case["top_k"] - len(chosen)
        ids.append(chosen + [-1] * rest)
        weights.append(w + [0.0] * rest)
    return torch.tensor(ids, dtype=torch.int32), torch.tensor(weights, dtype=torch.float64)


def exact(case, seed):
    i, op = _inputs(case, seed), case["op"]
    if op == "route":
        return _exact_route(case, i)
    if op == "fp8":
        x = _block_rounded64(i["a"].double()) @ _weights64(i["codes"], i["scales"]).t().contiguous()
        if i["cs"] is not None:
            x = x * i["cs"].double()
        if i["cb"] is not None:
            x = x + i["cb"].double()
            x = x * torch.sigmoid(x)
        return x
    x, out = _block_rounded64(i["x"].double()), torch.zeros(case["rows"], case["d"], dtype=torch.float64, device=DEV)
    for e in range(case["experts"]):
        row, j = (i["ids"] == e).nonzero(as_tuple=True)
        if row.numel():
            g = x[row] @ _weights64(i["gate"][e], i["gate_s"][e]).t().contiguous()
            h = g * torch.sigmoid(g) * (x[row] @ _weights64(i["up"][e], i["up_s"][e]).t().contiguous())
            p = _block_rounded64(h) @ _weights64(i["down"][e], i["down_s"][e]).t().contiguous()
            out.index_add_(0, row, p * i["w"][row, j].double().unsqueeze(1))
    return out
