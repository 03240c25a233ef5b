"""The operators of an expert layer: their cases, and their plain forms.

A layer of experts over the slot arrays of ``uccl_amd.ep.Buffer`` is: route the
tokens, dispatch them, multiply each expert's rows by its weights, gate, multiply
again, combine.  The operators here are the ones between the communication calls:

    route     router logits -> (expert indices, weights), and its gradient
    matmul    slot rows x expert weights, in 8 bits with a scale for each block
              of 128, or in 16 bits; the weights may lie transposed (the
              gradient of the rows)
    wgrad     gradient of the expert weights over the valid slot rows
    swiglu    gated activation between the two products, to 8 bits with scales
              or in 16 bits, and its gradient

Slot arrays are [experts, sources * length, columns]; source r of expert e has
counts[e, r] valid rows from row r * length on.  Rows behind them are neither read
nor written.
"""

import math

import numpy as np
import torch

own = False

F8 = torch.float8_e4m3fn
F8_MAX = 448.0
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one token of a decoding step: nothing but latency
        dict(name="route, one token", op="route", tokens=1, experts=256, topk=8, type="f32",
             scoring="sigmoid", bias=True, groups=8, topk_groups=4, train=False),
        # the tokens of one rank's dispatch, 256 experts top-8, limited to groups
        dict(name="route, 4096 tokens", op="route", tokens=4096, experts=256, topk=8, type="f32",
             scoring="sigmoid", bias=True, groups=8, topk_groups=4, train=False),
        # a training step's router, forward and backward, logits as a 16-bit gate gives them
        dict(name="route, training step", op="route", tokens=16384, experts=64, topk=6, type="bf16",
             scoring="softmax", bias=False, groups=1, topk_groups=1, train=True),
        # one row through one matrix: the smallest product a decoding step makes
        dict(name="matmul 8 bit, one row", op="matmul", experts=1, sources=1, length=1, rows=1,
             k=2048, n=7168, type="f8", transposed=False),
        # a rank's experts in a decoding step: few rows for each, all weights are read
        dict(name="matmul 8 bit, decode", op="matmul", experts=32, sources=8, length=16, rows=1024,
             k=7168, n=4096, type="f8", transposed=False),
        # a rank of 8 with 8 of 64 experts, 4096 tokens a rank, top-8: gate and up product
        dict(name="matmul 8 bit, prefill", op="matmul", experts=8, sources=8, length=768, rows=32768,
             k=7168, n=4096, type="f8", transposed=False),
        # the sizes of the two-rank example: 1024 tokens, top-2 of 8 experts, 1024 columns
        dict(name="matmul 16 bit, small", op="matmul", experts=8, sources=2, length=512, rows=2048,
             k=1024, n=1024, type="bf16", transposed=False),
        # gradient of the rows in training: the weights as they lie, read transposed
        dict(name="matmul 16 bit, row gradient", op="matmul", experts=8, sources=2, length=2048, rows=16384,
             k=4096, n=7168, type="bf16", transposed=True),
        # gradient of the same weights over the same rows
        dict(name="wgrad, large", op="wgrad", experts=8, sources=2, length=2048, rows=16384,
             n=4096, k=7168, type="bf16", out="bf16"),
        # ragged rows, sums kept in 32 bits for accumulation over steps
        dict(name="wgrad, small", op="wgrad", experts=8, sources=2, length=512, rows=1111,
             n=1000, k=1024, type="bf16", out="f32"),
        # between the two products of the prefill case, to 8 bits
        dict(name="swiglu to 8 bit", op="swiglu", experts=8, sources=8, length=768, rows=32768,
             cols=2048, type="bf16", quantize=True, train=False),
        # training: forward and gradient in 16 bits
        dict(name="swiglu, training step", op="swiglu", experts=8, sources=2, length=2048, rows=16384,
             cols=2048, type="bf16", quantize=False, train=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "matmul", "matmul", "wgrad", "swiglu"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        size = _log(rng, 4, 512 // groups)
        topk_groups = rng.randint(1, groups)
        return dict(op=op, tokens=_log(rng, 1, 16384), experts=groups * size,
                    topk=rng.randint(2, min(8, topk_groups * size)), type=rng.choice(["f32", "bf16", "f16"]),
                    scoring=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5,
                    groups=groups, topk_groups=topk_groups, train=rng.random() < 0.5)
    experts, sources = _log(rng, 1, 32), rng.choice([1, 2, 4, 8])
    length = _log(rng, 1, 8192)
    if op == "matmul":
        kind = rng.choice(["f8", "f8", "bf16", "f16"])
        k = 128 * _log(rng, 1, 56) if kind == "f8" else 8 * _log(rng, 1, 896)
        n = _log(rng, 1, 8192)
        length = max(1, min(length, int(6e11 / (experts * sources * k * n))))
        case = dict(op=op, experts=experts, sources=sources, length=length, k=k, type=kind)
        turned = kind != "f8" and rng.random() < 0.5
        case |= dict(n=8 * max(1, n // 8) if turned else n, transposed=turned)
    elif op == "wgrad":
        n, k = 8 * _log(rng, 1, 512), 8 * _log(rng, 1, 896)
        length = max(1, min(length, int(4e11 / (experts * sources * k * n))))
        case = dict(op=op, experts=experts, sources=sources, length=length, n=n, k=k,
                    type=rng.choice(["bf16", "f16"]), out=rng.choice(["bf16", "f16", "f32"]))
    else:
        quantize = rng.random() < 0.5
        cols = 128 * _log(rng, 1, 32) if quantize else 8 * _log(rng, 1, 512)
        length = max(1, min(length, int(4e7 / (experts * sources * cols))))
        case = dict(op=op, experts=experts, sources=sources, length=length, cols=cols,
                    type=rng.choice(["bf16", "f16"]), quantize=quantize, train=not quantize)
    slots = experts * sources * case["length"]
    case["rows"] = max(1, int(slots * rng.uniform(0.3, 1.0)))
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _counts(case, seed):
    """[experts, sources] counts with the case's sum of rows, experts of unlike popularity."""
    rng = np.random.RandomState(seed % (1 << 31))
    cells, room = case["experts"] * case["sources"], case["length"]
    like = np.repeat(rng.gamma(4.0, size=case["experts"]), case["sources"]) * rng.gamma(8.0, size=cells)
    counts, left = np.zeros(cells, dtype=np.int64), case["rows"]
    while left:
        open_ = like * (counts < room)
        counts += rng.multinomial(left, open_ / open_.sum())
        over = np.maximum(counts - room, 0)
        counts -= over
        left = int(over.sum())
    return torch.from_numpy(counts.reshape(case["experts"], case["sources"]).astype(np.int32)).cuda()


def _rows_to_8bit(x):
    """[..., K] -> values in 8 bits and a scale for each 128 of a row, as dispatch sends them."""
    g = x.float().reshape(*x.shape[:-1], -1, 128)
    amax = g.abs().amax(-1, keepdim=True)
    s = torch.where(amax > 0, amax / F8_MAX, torch.ones_like(amax))
    return (g / s).to(F8).reshape(x.shape), s.squeeze(-1).contiguous()


def _weights_to_8bit(w):
    """[N, K] -> values in 8 bits and a scale for each block of 128 by 128."""
    n, k = w.shape
    full = torch.zeros(-(-n // 128) * 128, k, device=w.device)
    full[:n] = w
    b = full.view(-1, 128, k // 128, 128)
    amax = b.abs().amax((1, 3), keepdim=True)
    s = torch.where(amax > 0, amax / F8_MAX, torch.ones_like(amax))
    return (b / s).to(F8).view(-1, k)[:n], s.view(-1, k // 128)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, times=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * times

    s = {"case": case}
    if case["op"] == "route":
        t, e = case["tokens"], case["experts"]
        logits = randn(t, e, times=2.0)
        if t > 16:  # padded tokens, and experts that are closed to some tokens
            logits[torch.rand(t, 1, device="cuda", generator=gen).expand(t, e) < 0.01] = -math.inf
            logits[torch.rand(t, e, device="cuda", generator=gen) < 0.02] = -math.inf
        s["logits"] = logits.to(TYPES[case["type"]])
        s["bias"] = randn(e, times=0.05) if case["bias"] else None
        s["grad"] = randn(t, case["topk"]) if case["train"] else None
        return s
    e, slots = case["experts"], case["sources"] * case["length"]
    s["counts"] = _counts(case, seed)
    if case["op"] == "matmul":
        k, n = case["k"], case["n"]
        if case["type"] == "f8":
            s["x"], s["x_scales"] = _rows_to_8bit(randn(e, slots, k))
            s["w"] = torch.empty(e, n, k, dtype=F8, device="cuda")
            s["w_scales"] = torch.empty(e, -(-n // 128), k // 128, device="cuda")
            for i in range(e):
                s["w"][i], s["w_scales"][i] = _weights_to_8bit(randn(n, k, times=0.02))
            s["out"] = torch.zeros(e, slots, n, dtype=torch.bfloat16, device="cuda")
        else:
            kind = TYPES[case["type"]]
            s["x"] = randn(e, slots, k).to(kind)
            s["w"] = torch.empty(e, k, n, dtype=kind, device="cuda").transpose(1, 2) if case["transposed"] \
                else torch.empty(e, n, k, dtype=kind, device="cuda")
            for i in range(e):
                s["w"][i] = randn(n, k, times=0.02)
            s["x_scales"] = s["w_scales"] = None
            s["out"] = torch.zeros(e, slots, n, dtype=kind, device="cuda")
    elif case["op"] == "wgrad":
        kind = TYPES[case["type"]]
        s["grad"] = randn(e, slots, case["n"], times=0.05).to(kind)
        s["x"] = randn(e, slots, case["k"]).to(kind)
        s["out"] = torch.zeros(e, case["n"], case["k"], dtype=TYPES[case["out"]], device="cuda")
    else:
        kind, cols = TYPES[case["type"]], case["cols"]
        s["h"] = randn(e, slots, 2 * cols, times=1.5).to(kind)
        if case["quantize"]:
            s["out"] = torch.zeros(e, slots, cols, device="cuda").to(F8)
            s["out_scales"] = torch.zeros(e, slots, cols // 128, device="cuda")
        else:
            s["out"] = torch.zeros(e, slots, cols, dtype=kind, device="cuda")
        if case["train"]:
            s["grad"] = randn(e, slots, cols, times=0.05).to(kind)
            s["grad_h"] = torch.zeros(e, slots, 2 * cols, dtype=kind, device="cuda")
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    case = s["case"]
    return (_run_own if own else _run_plain)(case, s)


def _run_own(case, s):
    import uccl_amd.ep as ep

    if case["op"] == "route":
        how = dict(scoring=case["scoring"], renormalize=True, scale=2.5)
        idx, weights = ep.route(s["logits"], case["topk"], bias=s["bias"], num_groups=case["groups"],
                                topk_groups=case["topk_groups"], **how)
        if not case["train"]:
            return {"idx": idx, "weights": weights}
        return {"idx": idx, "weights": weights, "grad": ep.route_grad(s["grad"], s["logits"], idx, **how)}
    if case["op"] == "matmul":
        expected = -(-case["rows"] // case["experts"])
        return ep.expert_matmul(s["x"], s["w"], s["counts"], x_scales=s["x_scales"], w_scales=s["w_scales"],
                                out=s["out"], expected_rows=expected)
    if case["op"] == "wgrad":
        return ep.expert_weight_grad(s["grad"], s["x"], s["counts"], out=s["out"])
    if case["quantize"]:
        q, scales = ep.expert_swiglu(s["h"], s["counts"], quantize=True, out=s["out"], out_scales=s["out_scales"])
        return {"values": q, "scales": scales}
    out = ep.expert_swiglu(s["h"], s["counts"], out=s["out"])
    return {"out": out, "grad": ep.expert_swiglu_grad(s["grad"], s["h"], s["counts"], out=s["grad_h"])}


def _run_plain(case, s):
    if case["op"] == "route":
        return _plain_route(case, s)
    if case["op"] == "matmul":
        return _plain_matmul(s)
    if case["op"] == "wgrad":
        return _plain_wgrad(s)
    return _plain_swiglu(case, s)


def _valid(counts, slots):
    """[experts, slots, 1]: which slot rows hold a token."""
    e, sources = counts.shape
    at = torch.arange(slots // sources, device=counts.device)
    return (at < counts[:, :, None]).view(e, slots, 1)


def _scores(x, scoring):
    """Scores in 64 bits; an expert whose logit is -inf has none."""
    closed = x == -math.inf
    if scoring == "sigmoid":
        return torch.sigmoid(x).masked_fill(closed, 0.0), closed
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top.masked_fill(top == -math.inf, 0.0)).masked_fill(closed, 0.0)
    total = p.sum(-1, keepdim=True)
    return p / total.masked_fill(total == 0, 1.0), closed


def _plain_route(case, s):
    # in 64 bits: which expert comes first is decided between values that may lie close together
    x, topk = s["logits"].double(), case["topk"]
    score, closed = _scores(x, case["scoring"])
    ranked = score + s["bias"].double() if case["bias"] else score
    key = (ranked if case["bias"] else x).masked_fill(closed, -math.inf)
    if case["groups"] > 1:
        size = case["experts"] // case["groups"]
        grouped = ranked.masked_fill(closed, -math.inf).view(-1, case["groups"], size)
        best = grouped.sort(-1, descending=True).values[..., :2]
        total = best.masked_fill(best == -math.inf, 0.0).sum(-1).masked_fill(best[..., 0] == -math.inf, -math.inf)
        order = total.sort(dim=-1, descending=True, stable=True).indices[:, : case["topk_groups"]]
        inside = torch.zeros_like(total, dtype=torch.bool).scatter_(1, order, True)
        key = key.masked_fill(~inside.repeat_interleave(size, 1), -math.inf)
    by = key.sort(dim=-1, descending=True, stable=True)
    idx = by.indices[:, :topk]
    none = by.values[:, :topk] == -math.inf
    picked = score.gather(1, idx).masked_fill(none, 0.0)
    total = picked.sum(-1, keepdim=True)
    total = total.masked_fill(total == 0, 1.0)
    out = {"idx": idx.masked_fill(none, -1), "weights": (2.5 * picked / total).float()}
    if not case["train"]:
        return out
    share, g = picked / total, s["grad"].double().masked_fill(none, 0.0)
    inner = 2.5 * (g - (g * share).sum(-1, keepdim=True))
    slope = share * (1 - picked) if case["scoring"] == "sigmoid" else share
    grad = torch.zeros_like(x).scatter_add_(1, idx, (inner * slope).masked_fill(none, 0.0))
    return {**out, "grad": grad.to(s["logits"].dtype)}


def _plain_matmul(s):
    x, w, out = s["x"].float(), s["w"].float(), s["out"]
    if s["x_scales"] is not None:
        x = x * s["x_scales"].repeat_interleave(128, -1)
        n = w.shape[1]
        w = w * s["w_scales"].repeat_interleave(128, 1)[:, :n].repeat_interleave(128, 2)
    y = torch.matmul(x, w.transpose(1, 2))
    return torch.where(_valid(s["counts"], x.shape[1]), y.to(out.dtype), out)


def _plain_wgrad(s):
    valid = _valid(s["counts"], s["x"].shape[1])
    g = s["grad"].float().masked_fill(~valid, 0.0)
    x = s["x"].float().masked_fill(~valid, 0.0)
    return torch.matmul(g.transpose(1, 2), x).to(s["out"].dtype)


def _nearest_8bit(y):
    """64-bit values to the nearest of the 8-bit type, ties to even, no rounding between."""
    _, exponent = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (exponent - 4).clamp(min=-9))
    return (torch.round(y / step) * step).clamp(-F8_MAX, F8_MAX).float().to(F8)


def _plain_swiglu(case, s):
    valid = _valid(s["counts"], s["h"].shape[1])
    if case["quantize"]:
        # in 64 bits: values next to a border between two 8-bit values
        gate, up = s["h"].double().chunk(2, -1)
        v = gate * torch.sigmoid(gate) * up
        groups = v.view(*v.shape[:-1], -1, 128)
        amax = groups.abs().amax(-1, keepdim=True)
        scales = torch.where(amax > 0, amax / F8_MAX, torch.ones_like(amax)).float()
        q = _nearest_8bit(groups / scales.double()).view(v.shape)
        values = torch.where(valid, q.float(), s["out"].float()).to(F8)
        return {"values": values, "scales": torch.where(valid, scales.squeeze(-1), s["out_scales"])}
    gate, up = s["h"].float().chunk(2, -1)
    sig = torch.sigmoid(gate)
    out = torch.where(valid, (gate * sig * up).to(s["out"].dtype), s["out"])
    g = s["grad"].float()
    grad = torch.cat([g * up * sig * (1 + gate * (1 - sig)), g * gate * sig], -1)
    return {"out": out, "grad": torch.where(valid, grad.to(out.dtype), s["grad_h"])}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] == "route":
        size = 4 if case["type"] == "f32" else 2
        read = case["tokens"] * case["experts"] * size
        picked = case["tokens"] * case["topk"]
        train = (read + picked * 4) if case["train"] else 0  # the gradient written, its input read
        return {"bytes": read + picked * 12 + train, "flops": case["tokens"] * case["experts"] * 8}
    e, rows = case["experts"], case["rows"]
    used = min(e, rows)
    if case["op"] == "matmul":
        k, n = case["k"], case["n"]
        if case["type"] == "f8":
            data = rows * (k + k // 32 + 2 * n) + used * (n * k + -(-n // 128) * (k // 128) * 4)
        else:
            data = 2 * (rows * (k + n) + used * n * k)
        return {"bytes": data, "flops": 2 * rows * n * k}
    if case["op"] == "wgrad":
        n, k = case["n"], case["k"]
        return {"bytes": 2 * rows * (n + k) + e * n * k * (4 if case["out"] == "f32" else 2),
                "flops": 2 * rows * n * k}
    cols = case["cols"]
    if case["quantize"]:
        return {"bytes": rows * (4 * cols + cols + cols // 32), "flops": rows * cols * 10}
    return {"bytes": rows * cols * (4 + 2 + 2 + 4), "flops": rows * cols * 20}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, written apart from the plain forms
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(case, s)
    counts = s["counts"].cpu().tolist()
    length = case["length"]

    def rows_of(e):
        at = [torch.arange(r * length, r * length + c) for r, c in enumerate(counts[e])]
        return torch.cat(at).cuda()

    if case["op"] == "matmul":
        out = s["out"].double()
        for e in range(case["experts"]):
            at = rows_of(e)
            x, w = s["x"][e][at].double(), s["w"][e].double()
            if case["type"] == "f8":
                x = (x.view(len(at), -1, 128) * s["x_scales"][e][at].double()[..., None]).view(len(at), -1)
                col = torch.arange(case["k"], device="cuda") // 128
                row = torch.arange(case["n"], device="cuda") // 128
                w = w * s["w_scales"][e].double()[row][:, col]
            out[e, at] = x @ w.t().contiguous()
        return out
    if case["op"] == "wgrad":
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            at = rows_of(e)
            out[e] = s["grad"][e][at].double().t().contiguous() @ s["x"][e][at].double()
        return out
    out = s["out"].double()
    cols = case["cols"]
    scales = s["out_scales"].double() if case["quantize"] else None
    grad = s["grad_h"].double() if case["train"] else None
    for e in range(case["experts"]):
        at = rows_of(e)
        h = s["h"][e][at].double()
        a, b = h[:, :cols], h[:, cols:]
        gate = a / (1 + torch.exp(-a))
        if case["quantize"]:
            v = (gate * b).view(len(at), -1, 128)
            most = v.abs().max(-1).values
            unit = (most / F8_MAX).float().double()
            unit[most == 0] = 1.0
            y = v / unit[..., None]
            # 4 significant bits, and no finer than 2^-9
            fine = torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            out[e, at] = (torch.round(y / fine) * fine).view(len(at), cols)
            scales[e, at] = unit
        else:
            out[e, at] = gate * b
            g = s["grad"][e][at].double()
            slope = (1 + torch.exp(-a) + a * torch.exp(-a)) / (1 + torch.exp(-a)) ** 2
            grad[e, at] = torch.cat([g * b * slope, g * gate], 1)
    return {"values": out, "scales": scales} if case["quantize"] else {"out": out, "grad": grad}


def _exact_route(case, s):
    x = s["logits"].double().cpu().numpy()
    t, e = x.shape
    k, groups = case["topk"], case["groups"]
    with np.errstate(all="ignore"):
        if case["scoring"] == "sigmoid":
            score = 1.0 / (1.0 + np.exp(-x))
        else:
            shifted = np.exp(x - np.where(np.isneginf(x.max(1)), 0.0, x.max(1))[:, None])
            score = shifted / np.maximum(shifted.sum(1), 1e-300)[:, None]
    key = score + s["bias"].double().cpu().numpy() if case["bias"] else score
    key = np.where(np.isneginf(x), -np.inf, key)
    if groups > 1:
        best = -np.sort(-key.reshape(t, groups, -1), -1)[..., :2]
        value = np.where(np.isneginf(best[..., 0]), -np.inf, np.where(np.isneginf(best), 0.0, best).sum(-1))
        place = np.argsort(np.argsort(-value, 1, kind="stable"), 1)
        shut = np.repeat(place >= case["topk_groups"], e // groups, 1)
    else:
        shut = np.zeros((t, e), bool)
    order = np.argsort(-np.where(shut, -np.inf, key if case["bias"] else x), 1, kind="stable")[:, :k]
    take = np.arange(t)[:, None]
    open_ = ~(np.isneginf(key) | shut)[take, order]
    p = np.where(open_, score[take, order], 0.0)
    total = p.sum(1, keepdims=True)
    share = np.divide(p, total, out=np.zeros_like(p), where=total > 0)
    out = {"idx": np.where(open_, order, -1), "weights": 2.5 * share}
    if case["train"]:
        g = np.where(open_, s["grad"].double().cpu().numpy(), 0.0)
        d = 2.5 * share * (g - (g * share).sum(1, keepdims=True))
        if case["scoring"] == "sigmoid":
            d = d * (1.0 - p)
        grad = np.zeros((t, e))
        np.add.at(grad, (np.broadcast_to(take, order.shape), order), d)
        out["grad"] = grad
    return out
