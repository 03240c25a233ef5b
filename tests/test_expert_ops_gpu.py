"""Expert-layer operators against plain implementations in 64 bits.

Tolerances count roundings: u(t) = finfo(t).eps / 2 is the half step of a
result type, 2^-23 bounds one 32-bit operation (the matrix unit may truncate),
and a sum of n terms is off by at most n * 2^-23 * sum |terms|. The 8-bit matrix
unit aligns the products of an instruction before it adds them; on bytes of
all magnitudes that was measured to cost up to 8.4e-5 = 2^-13.5 of
sum |products|, and 2^-13 is allowed for it.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("requires GPU", allow_module_level=True)

import uccl_amd.ep as ep  # noqa: E402

F8, BF, HF, F32 = (torch.float8_e4m3fn, torch.bfloat16, torch.float16,
                   torch.float32)
STEP32 = 2.0 ** -23


def half_step(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def close(got, want, tol, what=""):
    """|got - want| <= tol everywhere, and the same NaN."""
    got, want = got.double(), want.double()
    off = (got - want).abs()
    bad = ~(off <= tol) & ~((got != got) & (want != want))
    if bad.any():
        at = int(bad.flatten().nonzero()[0])
        pytest.fail(f"{what}: {int(bad.sum())} of {bad.numel()} off; first at "
                    f"{at}: {got.flatten()[at]} for {want.flatten()[at]}, "
                    f"allowed {tol.expand_as(off).flatten()[at]}")


def mask_of(counts, slots):
    e, r = counts.shape
    at = torch.arange(slots // r, device=counts.device)
    return (at < counts[:, :, None]).view(e, slots)


def some_counts(g, e, r, length, kind="random"):
    if kind == "random":
        c = torch.randint(0, length + 1, (e, r), device="cuda", generator=g)
    elif kind == "none":
        c = torch.zeros(e, r, device="cuda")
    elif kind == "full":
        c = torch.full((e, r), length, device="cuda")
    else:  # one row somewhere
        c = torch.zeros(e, r, device="cuda")
        c[e // 2, r - 1] = 1
    return c.int()


# ---------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------

def route_oracle(logits, topk, scoring="softmax", bias=None, num_groups=1,
                 topk_groups=1, group_best=2, renormalize=True, scale=1.0):
    """One token after the other, by the definition, on the CPU."""
    x = logits.double().cpu()
    T, E = x.shape
    idx = torch.full((T, topk), -1, dtype=torch.int64)
    w = torch.zeros(T, topk, dtype=torch.float64)
    for t in range(T):
        row = x[t]
        open_ = [e for e in range(E) if row[e] > -math.inf]
        nan = bool(torch.isnan(row).any())
        if scoring == "sigmoid":
            s = torch.sigmoid(row)
        elif open_:
            s = torch.softmax(torch.where(torch.isnan(row), -math.inf, row), 0)
            nan = nan or bool(torch.isnan(s).any())
        else:
            s = torch.zeros(E, dtype=torch.float64)
        rank = s if bias is None else s + bias.double().cpu()
        key = row if bias is None else rank
        open_ = [e for e in open_ if key[e] > -math.inf]
        if num_groups > 1:
            size = E // num_groups
            value = []
            for g in range(num_groups):
                best = sorted((float(rank[e]) for e in open_
                               if e // size == g and rank[e] > -math.inf),
                              reverse=True)
                value.append(sum(best[:group_best]) if best else -math.inf)
            keep = sorted(range(num_groups), key=lambda g: (-value[g], g))
            open_ = [e for e in open_ if e // size in keep[:topk_groups]]
        order = sorted(open_, key=lambda e: (-float(key[e]), e))[:topk]
        idx[t, :len(order)] = torch.tensor(order, dtype=torch.int64)
        p = s[order]
        if renormalize:
            p = p / p.sum() if p.sum() > 0 else torch.zeros_like(p)
        w[t, :len(order)] = p * scale
        if nan:
            w[t] = math.nan
    return idx, w


ROUTES = [
    # tokens, experts, topk, keywords
    (1, 1, 1, {}),
    (1, 8, 2, {}),
    (7, 64, 6, dict(renormalize=False)),
    (5, 65, 8, dict(scoring="sigmoid")),
    (13, 256, 8, dict(scoring="sigmoid", num_groups=8, topk_groups=4, bias=1,
                      scale=2.5)),
    (9, 160, 6, dict(num_groups=8, topk_groups=3, group_best=1,
                     renormalize=False, scale=16.0)),
    (6, 96, 5, dict(bias=1)),
    (3, 1024, 64, dict(bias=1, scoring="sigmoid", renormalize=False)),
    (4, 513, 9, dict()),
    (3, 192, 7, dict(num_groups=64, topk_groups=9, scoring="sigmoid")),
    (3, 24, 24, dict(num_groups=3, topk_groups=3, bias=1)),
]


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("tokens, experts, topk, kw", ROUTES)
def test_route(tokens, experts, topk, kw, dtype):
    g = gen(experts + topk)
    logits = (randn(g, tokens, experts) * 2).to(dtype)
    kw = dict(kw)
    if kw.pop("bias", 0):
        kw["bias"] = randn(g, experts) * 0.1
    idx, w = ep.route(logits, topk, **kw)
    want_idx, want_w = route_oracle(logits, topk, **kw)
    assert torch.equal(idx.cpu(), want_idx)
    close(w.cpu(), want_w, want_w.abs() * 2 ** -24 * (1 + 1e-6) + 1e-45)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_odd_rows(scoring, bias, groups):
    """Ties, closed experts, rows without an open one, huge and NaN logits."""
    x = torch.zeros(12, 32, device="cuda")
    x[1] = -math.inf
    x[2, 1:] = -math.inf
    x[3, 4:] = -math.inf
    x[4] = 3e38
    x[5] = torch.finfo(F32).min
    x[6, ::2] = 1.0
    x[7, 9] = math.nan
    x[8, 5] = math.inf
    x[9] = math.nan
    x[10] = torch.arange(32, device="cuda") * 1e-30
    x[11, :31] = -math.inf
    x[11, 31] = -900.0
    kw = dict(scoring=scoring, num_groups=groups, topk_groups=max(1, groups - 1))
    if bias:
        kw["bias"] = torch.zeros(32, device="cuda")
        kw["bias"][3] = -math.inf
    idx, w = ep.route(x, 6, **kw)
    want_idx, want_w = route_oracle(x, 6, **kw)
    assert torch.equal(idx.cpu(), want_idx)
    close(w.cpu(), want_w, want_w.abs() * 2 ** -23 + 1e-45)


def test_route_strided_and_empty():
    g = gen(3)
    wide = randn(g, 6, 40)
    idx, w = ep.route(wide[:, 3:35], 4)
    want = ep.route(wide[:, 3:35].contiguous(), 4)
    assert torch.equal(idx, want[0]) and torch.equal(w, want[1])
    idx, w = ep.route(wide[:0], 4)
    assert idx.shape == (0, 4) and w.shape == (0, 4)
    same = wide[0].expand(5, 40)
    idx, w = ep.route(same, 4)
    assert torch.equal(idx, idx[:1].expand(5, 4))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("tokens, experts, topk, kw", [
    (4097, 8, 2, {}),
    (5000, 64, 6, {}),
    (4999, 40, 16, dict(scoring="sigmoid", num_groups=5, topk_groups=3)),
    (4500, 200, 8, dict(bias=1)),
    (4200, 256, 8, dict(scoring="sigmoid", bias=1, num_groups=8,
                        topk_groups=4)),
    (4100, 256, 17, {}),
    (4100, 300, 5, dict(renormalize=False)),
    (32771, 256, 8, dict(scoring="sigmoid", bias=1, num_groups=8,
                         topk_groups=4)),
    (32770, 200, 8, dict(bias=1)),
])
def test_route_many_tokens(tokens, experts, topk, kw, dtype):
    """A token's picks, weights and gradient do not hang on how many others
    there are (few tokens have more lanes each), nor on where it stands."""
    g = gen(tokens)
    x = (randn(g, tokens, experts) * 2).to(dtype)
    x[torch.rand(tokens, experts, device="cuda", generator=g) < 0.1] = -math.inf
    x[7] = -math.inf
    x[11, 3] = math.nan
    kw = dict(kw)
    if kw.pop("bias", 0):
        kw["bias"] = randn(g, experts) * 0.1
    gw = randn(g, tokens, topk)
    how = {k: v for k, v in kw.items() if k in ("scoring", "renormalize")}
    idx, w = ep.route(x, topk, **kw)
    grad = ep.route_grad(gw, x, idx, **how)
    for at in range(0, tokens, 1500):
        part = slice(at, min(at + 1500, tokens))
        idx_p, w_p = ep.route(x[part], topk, **kw)
        assert torch.equal(idx[part], idx_p)
        close(w[part], w_p, w_p.abs() * 2 ** -23)
        grad_p = ep.route_grad(gw[part], x[part], idx_p, **how)
        close(grad[part], grad_p, grad_p.abs() * half_step(dtype) * 2 + 1e-13)
    some = torch.randint(0, tokens, (20,), device="cuda", generator=g)
    some[:2] = torch.tensor([7, 11], device="cuda")
    want_idx, want_w = route_oracle(x[some], topk, **kw)
    assert torch.equal(idx[some].cpu(), want_idx)
    close(w[some].cpu(), want_w, want_w.abs() * 2 ** -23 + 1e-45)


def weights_of(x, idx, scoring, renormalize, scale):
    """The weights as a function of 64-bit logits, the picks held fixed."""
    s = torch.sigmoid(x) if scoring == "sigmoid" else torch.softmax(x, -1)
    w = s.gather(1, idx.clamp(min=0)) * (idx >= 0)
    if renormalize:
        w = w / w.sum(-1, keepdim=True)
    return w * scale


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens, experts, topk",
                         [(1, 8, 2), (5, 64, 6), (3, 100, 1), (4, 300, 8),
                          (2, 1024, 64)])
def test_route_grad(tokens, experts, topk, scoring, renormalize):
    g = gen(experts)
    logits = randn(g, tokens, experts)
    how = dict(scoring=scoring, renormalize=renormalize, scale=2.5)
    idx, _ = ep.route(logits, topk, **how)
    if topk > 2:
        idx[0, 1] = -1
        idx[-1, 2] = idx[-1, 0]  # the same expert twice
    gw = randn(g, tokens, topk)
    got = ep.route_grad(gw, logits, idx, **how)

    x = logits.double().requires_grad_()
    (weights_of(x, idx, **how) * gw.double()).sum().backward()
    # rounded once from 64 bits; the sums inside cancel to 2^-50 of |g|
    close(got, x.grad, x.grad.abs() * 2 ** -24 * (1 + 1e-6) + 1e-13, "formula")

    # and against differences of the weights: h^2 of the third derivative
    x, h = logits.double(), 1e-5
    for e in {0, experts - 1, int(idx[0, 0])}:
        d = torch.zeros_like(x)
        d[:, e] = h
        slope = (weights_of(x + d, idx, **how)
                 - weights_of(x - d, idx, **how)) / (2 * h)
        want = (slope * gw.double()).sum(-1)
        close(got[:, e], want,
              want.abs() * 2 ** -24 + gw.double().abs().sum(-1) * 1e-8,
              f"difference at {e}")


def test_route_grad_edges():
    x = torch.randn(4, 16, device="cuda")
    x[1] = -math.inf
    gw = torch.randn(4, 3, device="cuda")
    for how in (dict(), dict(scoring="sigmoid"), dict(renormalize=False),
                dict(scoring="sigmoid", renormalize=False)):
        idx, _ = ep.route(x, 3, **how)
        idx[2] = torch.tensor([99, -5, 1 << 40], device="cuda")
        got = ep.route_grad(gw, x, idx, **how)
        assert torch.isfinite(got).all()
        assert (got[1] == 0).all() and (got[2] == 0).all(), how
        assert (got[0] != 0).any()
    # a single renormalised pick has no gradient at all
    idx, _ = ep.route(x, 1)
    assert (ep.route_grad(gw[:, :1].contiguous(), x, idx) == 0).all()


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------

def rows_to_8bit(x):
    g = x.float().reshape(*x.shape[:-1], -1, 128)
    amax = g.abs().amax(-1, keepdim=True)
    s = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
    return (g / s).to(F8).reshape(x.shape), s.squeeze(-1).contiguous()


def weights_to_8bit(w):
    e, n, k = w.shape
    nb = -(-n // 128)
    full = torch.zeros(e, nb * 128, k, device=w.device)
    full[:, :n] = w
    b = full.view(e, nb, 128, k // 128, 128)
    amax = b.abs().amax((2, 4), keepdim=True)
    s = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
    q = (b / s).to(F8).view(e, nb * 128, k)[:, :n].contiguous()
    return q, s.view(e, nb, k // 128)


def values_of(q, scales, rows):
    """8-bit values and scales (of `rows` rows each) as 64-bit values."""
    v = q.double()
    s = scales.double().repeat_interleave(128, -1)
    if rows > 1:
        s = s.repeat_interleave(rows, 1)[:, :v.shape[1]]
    return v * s


def product(x, w):
    """64-bit product, and the same of the magnitudes."""
    wt = w.transpose(1, 2).contiguous()
    return torch.matmul(x, wt), torch.matmul(x.abs(), wt.abs())


def check_product(got, x, w, mask, eight=False, before=None):
    want, size = product(x, w)
    k = x.shape[-1]
    tol = want.abs() * half_step(got.dtype) + size * k * STEP32
    tol = tol + torch.finfo(got.dtype).smallest_normal * half_step(got.dtype)
    if eight:
        tol = tol + size * 2.0 ** -13
    close(got[mask], want[mask], tol[mask], "product")
    if before is not None:
        assert torch.equal(got[~mask], before[~mask]), "rows behind changed"


SIZES = [
    # experts, sources, length, n, k, expected rows
    (1, 1, 1, 8, 128, None),
    (1, 1, 1, 1, 256, None),
    (3, 2, 5, 37, 128, None),
    (2, 4, 40, 130, 384, None),
    (2, 4, 40, 130, 384, 3),
    (5, 1, 129, 257, 256, None),
    (1, 3, 300, 512, 640, None),
    (40, 2, 9, 64, 128, 4),
    (2, 2, 700, 515, 256, 1024),
    (9, 1, 300, 1030, 128, 300),
]


@pytest.mark.parametrize("out", [BF, HF])
@pytest.mark.parametrize("kind", ["random", "none", "full", "one"])
@pytest.mark.parametrize("e, r, length, n, k, expected", SIZES)
def test_matmul_8bit(e, r, length, n, k, expected, kind, out):
    g = gen(n + k)
    counts = some_counts(g, e, r, length, kind)
    mask = mask_of(counts, r * length)
    x, xs = rows_to_8bit(randn(g, e, r * length, k))
    w, ws = weights_to_8bit(randn(g, e, n, k) * 0.05)
    # nothing behind the valid rows is read: fill it with NaN
    x.view(torch.uint8)[~mask] = 0x7F
    xs[~mask] = math.nan
    y = torch.full((e, r * length, n), 7.0, dtype=out, device="cuda")
    before = y.clone()
    got = ep.expert_matmul(x, w, counts, x_scales=xs, w_scales=ws, out=y,
                           expected_rows=expected)
    assert got is y
    x0 = torch.where(mask[..., None], values_of(x, xs, 1), 0.0)
    check_product(got, x0, values_of(w, ws, 128), mask, True, before)


@pytest.mark.parametrize("dtype, out", [(BF, None), (HF, None), (BF, F32),
                                        (HF, BF)])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("kind", ["random", "full", "one"])
@pytest.mark.parametrize("e, r, length, n, k, expected",
                         [(1, 1, 1, 8, 8, None), (3, 2, 5, 40, 24, None),
                          (2, 4, 40, 136, 200, None), (2, 4, 40, 136, 200, 5),
                          (5, 1, 129, 264, 72, 128), (1, 3, 300, 512, 520, 900),
                          (2, 2, 700, 520, 264, 1400),
                          (9, 1, 300, 1032, 136, 300)])
def test_matmul_16bit(e, r, length, n, k, expected, kind, turned, dtype, out):
    g = gen(n + k)
    counts = some_counts(g, e, r, length, kind)
    mask = mask_of(counts, r * length)
    x = randn(g, e, r * length, k).to(dtype)
    x[~mask] = math.nan
    w = (randn(g, e, n, k) * 0.05).to(dtype)
    if turned:
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    got = ep.expert_matmul(x, w, counts, out_dtype=out, expected_rows=expected)
    assert got.dtype == (out or dtype)
    x0 = torch.where(mask[..., None], x.double(), 0.0)
    check_product(got, x0, w.double(), mask)


@pytest.mark.parametrize("expected", [1, 16, 17, 40, 64, 65, 128, 200])
@pytest.mark.parametrize("dtype", [F8, BF, HF])
def test_matmul_expected_rows(dtype, expected):
    """The hint changes how the product is computed, never what."""
    e, r, length, n, k = 40, 3, 23, 1032, 384
    g = gen(expected)
    counts = some_counts(g, e, r, length, "random")
    mask = mask_of(counts, r * length)
    y = torch.full((e, r * length, n), 7.0, dtype=BF, device="cuda")
    before = y.clone()
    if dtype == F8:
        x, xs = rows_to_8bit(randn(g, e, r * length, k))
        w, ws = weights_to_8bit(randn(g, e, n, k) * 0.05)
        x.view(torch.uint8)[~mask] = 0x7F
        xs[~mask] = math.nan
        ep.expert_matmul(x, w, counts, x_scales=xs, w_scales=ws, out=y,
                         expected_rows=expected)
        x0, w0 = values_of(x, xs, 1), values_of(w, ws, 128)
    else:
        k = 376
        x = randn(g, e, r * length, k).to(dtype)
        w = (randn(g, e, n, k) * 0.05).to(dtype)
        x[~mask] = math.nan
        ep.expert_matmul(x, w, counts, out=y, expected_rows=expected)
        x0, w0 = x.double(), w.double()
    x0 = torch.where(mask[..., None], x0, 0.0)
    check_product(y, x0, w0, mask, dtype == F8, before)


@pytest.mark.parametrize("k", [64, 136, 1024])
@pytest.mark.parametrize("length, n", [(300, 1032), (65, 3), (1000, 17)])
@pytest.mark.parametrize("kind", ["random", "full", "one", "none"])
def test_matmul_of_middling_sizes(kind, length, n, k):
    g = gen(k + n)
    counts = some_counts(g, 4, 1, length, kind)
    mask = mask_of(counts, length)
    y = torch.full((4, length, n), 7.0, dtype=BF, device="cuda")
    for eight in (False, True):
        if eight and k % 128:
            continue
        y.fill_(7.0)
        before = y.clone()
        if eight:
            x, xs = rows_to_8bit(randn(g, 4, length, k))
            w, ws = weights_to_8bit(randn(g, 4, n, k) * 0.05)
            x.view(torch.uint8)[~mask] = 0x7F
            ep.expert_matmul(x, w, counts, x_scales=xs, w_scales=ws, out=y)
            x0, w0 = values_of(x, xs, 1), values_of(w, ws, 128)
        else:
            x = randn(g, 4, length, k).to(BF)
            w = (randn(g, 4, n, k) * 0.05).to(BF)
            x[~mask] = math.nan
            ep.expert_matmul(x, w, counts, out=y)
            x0, w0 = x.double(), w.double()
        x0 = torch.where(mask[..., None], x0, 0.0)
        check_product(y, x0, w0, mask, eight, before)


@pytest.mark.parametrize("kind, out", [("product", BF), ("product", F32),
                                       ("turned", BF), ("turned", F32),
                                       ("8 bit", BF), ("8 bit", HF)])
def test_matmul_more_tiles_than_compute_units(kind, out):
    """Several tiles for each block, the last of them half empty."""
    e, r, length, n, k = 20, 3, 210, 1304, 328
    g = gen(len(kind))
    counts = some_counts(g, e, r, length, "random")
    counts[3:9] = length
    mask = mask_of(counts, r * length)
    y = torch.full((e, r * length, n), 7.0, dtype=out, device="cuda")
    before = y.clone()
    if kind == "8 bit":
        k = 384
        x, xs = rows_to_8bit(randn(g, e, r * length, k))
        w, ws = weights_to_8bit(randn(g, e, n, k) * 0.05)
        ep.expert_matmul(x, w, counts, x_scales=xs, w_scales=ws, out=y)
        x0, w0 = values_of(x, xs, 1), values_of(w, ws, 128)
    else:
        x = randn(g, e, r * length, k).to(BF)
        w = (randn(g, e, n, k) * 0.05).to(BF)
        if kind == "turned":
            w = w.transpose(1, 2).contiguous().transpose(1, 2)
        x[~mask] = math.nan
        ep.expert_matmul(x, w, counts, out=y)
        x0, w0 = x.double(), w.double()
    x0 = torch.where(mask[..., None], x0, 0.0)
    check_product(y, x0, w0, mask, kind == "8 bit", before)


@pytest.mark.parametrize("kind", ["product", "turned", "8 bit", "wgrad",
                                  "wider wgrad"])
def test_rows_of_an_expert_span_more_than_4_gib(kind):
    slots, n, k = 4200, 520, 264
    if kind == "wider wgrad":
        kind, n, k = "wgrad", 2056, 1032
    pitch = 1 << 19
    g = gen(len(kind))
    counts = torch.tensor([slots - 3], dtype=torch.int32, device="cuda")
    mask = mask_of(counts[None], slots)[0]

    def far(rows):  # [1, slots, cols], the rows `pitch` elements apart
        wide = torch.empty(slots, pitch * (2 if rows.dtype == F8 else 1),
                           dtype=rows.dtype, device="cuda")
        wide[:, :rows.shape[1]] = rows
        return wide[None, :, :rows.shape[1]]

    if kind == "8 bit":
        k = 256
        x, xs = rows_to_8bit(randn(g, 1, slots, k))
        w, ws = weights_to_8bit(randn(g, 1, n, k) * 0.05)
        got = ep.expert_matmul(far(x[0]), w, counts, x_scales=xs, w_scales=ws)
        check_product(got, values_of(x, xs, 1), values_of(w, ws, 128),
                      mask[None], True)
        return
    x = randn(g, slots, k).to(BF)
    if kind == "wgrad":
        grad = (randn(g, slots, n) * 0.05).to(BF)
        got = ep.expert_weight_grad(far(grad), far(x), counts)
        gt = grad.double()[mask].t().contiguous()[None]
        check_product(got, gt, x.double()[mask].t().contiguous()[None],
                      torch.ones(1, n, dtype=torch.bool, device="cuda"))
        return
    w = (randn(g, 1, n, k) * 0.05).to(BF)
    if kind == "turned":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    got = ep.expert_matmul(far(x), w, counts)
    check_product(got, x.double()[None], w.double(), mask[None])


def test_matmul_weights_far_apart():
    """Rows of weights so far apart that a tile's span more than 4 GiB."""
    n, k, pitch = 300, 72, 1 << 23
    g = gen(3)
    wide = torch.empty(n, pitch, dtype=BF, device="cuda")
    wide[:, :k] = randn(g, n, k) * 0.05
    w = wide[None, :, :k]
    x = randn(g, 1, 200, k).to(BF)
    every = torch.ones(1, 200, dtype=torch.bool, device="cuda")
    for rows in (1, 200):
        check_product(ep.expert_matmul(x, w, expected_rows=rows), x.double(),
                      w.double(), every)


def test_matmul_odd_n_16bit():
    g = gen(5)
    for n in (1, 3, 17, 255, 259):
        x = randn(g, 2, 33, 48).to(BF)
        w = randn(g, 2, n, 48).to(BF)
        check_product(ep.expert_matmul(x, w), x.double(), w.double(),
                      torch.ones(2, 33, dtype=torch.bool, device="cuda"))


def test_matmul_counts_are_clamped():
    g = gen(6)
    x, w = randn(g, 3, 20, 64).to(BF), randn(g, 3, 48, 64).to(BF)
    counts = torch.tensor([[-4, 99], [1 << 30, -(1 << 31)], [3, 0]],
                          dtype=torch.int32, device="cuda")
    y = torch.full((3, 20, 48), 7.0, dtype=BF, device="cuda")
    before = y.clone()
    ep.expert_matmul(x, w, counts, out=y)
    mask = mask_of(counts.clamp(0, 10), 20)
    check_product(y, x.double(), w.double(), mask, before=before)


def test_matmul_two_dimensions_and_counts_of_one_source():
    g = gen(7)
    x, w = randn(g, 30, 64).to(BF), randn(g, 48, 64).to(BF)
    full = ep.expert_matmul(x, w)
    every = torch.ones(1, 30, dtype=torch.bool, device="cuda")
    check_product(full[None], x[None].double(), w[None].double(), every)
    counts = torch.tensor([4, 9, 0], dtype=torch.int32, device="cuda")
    part = ep.expert_matmul(x, w, counts)
    mask = mask_of(counts[None], 30)[0]
    assert torch.equal(part[mask], full[mask])
    x3, w3 = x.view(3, 10, 64), randn(g, 3, 48, 64).to(BF)
    a = ep.expert_matmul(x3, w3, counts)
    b = ep.expert_matmul(x3, w3, counts[:, None])
    m = mask_of(counts[:, None], 10)
    assert torch.equal(a[m], b[m])


def test_matmul_strides():
    """Padded rows, weights shared by all experts, results inside a larger
    tensor, experts and slots swapped in memory."""
    g = gen(8)
    pad = randn(g, 2, 50, 96).to(BF)
    x = pad[:, 5:45, 16:80]
    w = randn(g, 24, 64).to(BF).expand(2, 24, 64)
    room = torch.full((40, 2, 33), 7.0, dtype=BF, device="cuda")
    y = room.transpose(0, 1)[..., 5:29]
    ep.expert_matmul(x, w, out=y)
    every = torch.ones(2, 40, dtype=torch.bool, device="cuda")
    check_product(y, x.double(), w.double(), every)
    assert (room[..., :5] == 7).all() and (room[..., 29:] == 7).all()
    q, s = rows_to_8bit(randn(g, 2, 40, 256))
    qw, sw = weights_to_8bit(randn(g, 2, 24, 256))
    wide = torch.zeros(2, 40, 5, device="cuda")
    wide[..., 1:3] = s
    got = ep.expert_matmul(q, qw, x_scales=wide[..., 1:3], w_scales=sw)
    want = ep.expert_matmul(q, qw, x_scales=s, w_scales=sw)
    assert torch.equal(got, want)


def test_matmul_8bit_extremes():
    """Values at the ends of the type, zero and tiny scales, a NaN value and
    an infinite scale, which reach only their own row."""
    x = torch.full((1, 4, 256), 448.0, device="cuda").to(F8)
    w = torch.full((1, 16, 256), -448.0, device="cuda").to(F8)
    xs = torch.ones(1, 4, 2, device="cuda") / 448
    ws = torch.ones(1, 1, 2, device="cuda") / 448
    xs[0, 1] = 0.0
    xs[0, 2, 0] = math.inf
    x.view(torch.uint8)[0, 3, 7] = 0x7F
    y = ep.expert_matmul(x, w, x_scales=xs, w_scales=ws).float()
    close(y[0, 0], torch.full((16,), -256.0, device="cuda"),
          torch.tensor(256 * (2 ** -9 + 2 ** -13), device="cuda"))
    assert (y[0, 1] == 0).all()
    assert (y[0, 2] == -math.inf).all()
    assert torch.isnan(y[0, 3]).all()


def test_matmul_behind_32_bits():
    """Rows whose byte offsets pass 32 bits, in x, its scales and the result."""
    length, k, n = 700_000, 7168, 4096
    x = torch.empty(1, 2 * length, k, dtype=F8, device="cuda")
    xs = torch.empty(1, 2 * length, k // 128, device="cuda")
    y = torch.empty(1, 2 * length, n, dtype=BF, device="cuda")
    g = gen(9)
    some, scales = rows_to_8bit(randn(g, 1, 5, k))
    x[:, length:length + 5], xs[:, length:length + 5] = some, scales
    x[:, length - 3:length], xs[:, length - 3:length] = some[:, :3], scales[:, :3]
    w, ws = weights_to_8bit(randn(g, 1, n, k) * 0.02)
    counts = torch.tensor([[0, 5]], dtype=torch.int32, device="cuda")
    want = ep.expert_matmul(some, w, x_scales=scales, w_scales=ws,
                            expected_rows=5)
    ep.expert_matmul(x, w, counts, x_scales=xs, w_scales=ws, out=y,
                     expected_rows=5)
    assert torch.equal(y[:, length:length + 5], want)
    mask = torch.ones(1, 5, dtype=torch.bool, device="cuda")
    check_product(want, values_of(some, scales, 1), values_of(w, ws, 128),
                  mask, True)


@pytest.mark.parametrize("dtype, out", [(BF, None), (HF, None), (BF, F32),
                                        (HF, BF)])
@pytest.mark.parametrize("kind", ["random", "none", "full", "one"])
@pytest.mark.parametrize("e, r, length, n, k",
                         [(1, 1, 1, 8, 8), (3, 2, 5, 40, 24),
                          (2, 4, 40, 136, 200), (1, 3, 300, 512, 520),
                          (2, 2, 70, 2064, 2056), (17, 1, 65, 16, 264)])
def test_weight_grad(e, r, length, n, k, kind, dtype, out):
    g = gen(n + k)
    counts = some_counts(g, e, r, length, kind)
    mask = mask_of(counts, r * length)[..., None]
    d = (randn(g, e, r * length, n) * 0.1).to(dtype)
    x = randn(g, e, r * length, k).to(dtype)
    d[~mask[..., 0]], x[~mask[..., 0]] = math.nan, math.nan
    got = ep.expert_weight_grad(d, x, counts, out_dtype=out)
    assert got.dtype == (out or dtype)
    d0 = torch.where(mask, d.double(), 0.0).transpose(1, 2).contiguous()
    x0 = torch.where(mask, x.double(), 0.0)
    want, size = torch.matmul(d0, x0), torch.matmul(d0.abs(), x0.abs())
    tol = (want.abs() * half_step(got.dtype) + size * r * length * STEP32
           + torch.finfo(got.dtype).smallest_normal * half_step(got.dtype))
    close(got, want, tol, "weight gradient")
    # the same again, bit for bit
    assert torch.equal(got, ep.expert_weight_grad(d, x, counts, out_dtype=out))


@pytest.mark.parametrize("kind", ["random", "full", "one", "none"])
@pytest.mark.parametrize("e, r, length, n, k", [
    (1, 3, 700, 8, 8),        # few tiles, many rows
    (3, 2, 1100, 88, 3544),
    (2, 1, 1, 72, 64),
    (9, 1, 130, 520, 1032),   # tiles for half of the card
    (20, 3, 30, 1304, 1032),  # and for more than all of it
])
def test_weight_grad_of_all_sizes(e, r, length, n, k, kind):
    g = gen(n)
    counts = some_counts(g, e, r, length, kind)
    mask = mask_of(counts, r * length)[..., None]
    d = (randn(g, e, r * length, n) * 0.05).to(BF)
    x = randn(g, e, r * length, k).to(BF)
    d[~mask[..., 0]], x[~mask[..., 0]] = math.nan, math.nan
    room = torch.full((e, n + 1, k + 8), 7.0, device="cuda")
    got = ep.expert_weight_grad(d, x, counts, out=room[:, :n, :k])
    d0 = torch.where(mask, d.double(), 0.0).transpose(1, 2).contiguous()
    x0 = torch.where(mask, x.double(), 0.0)
    want, size = torch.matmul(d0, x0), torch.matmul(d0.abs(), x0.abs())
    close(got, want, want.abs() * STEP32 + size * r * length * STEP32,
          "weight gradient")
    assert (room[:, n:] == 7).all() and (room[:, :, k:] == 7).all()


@pytest.mark.parametrize("kind", ["random", "full", "one", "none"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("e, r, length, n, k, expected", [
    (1, 2, 100, 8, 1000, None),    # few tiles, a long contraction
    (2, 3, 60, 200, 72, 7),
    (3, 1, 1, 64, 8, None),
    (4, 1, 300, 1032, 136, None),  # tiles for half of the card
    (40, 2, 40, 1032, 200, 20),    # few rows of many experts
    (40, 2, 40, 1032, 200, 40),
    (40, 2, 40, 1032, 200, 80),
])
def test_row_gradient_of_all_sizes(e, r, length, n, k, expected, dtype, kind):
    g = gen(n + k)
    counts = some_counts(g, e, r, length, kind)
    mask = mask_of(counts, r * length)
    x = randn(g, e, r * length, k).to(dtype)
    x[~mask] = math.nan
    w = (randn(g, e, k, n) * 0.05).to(dtype).transpose(1, 2)
    y = torch.full((e, r * length, n), 7.0, dtype=dtype, device="cuda")
    before = y.clone()
    ep.expert_matmul(x, w, counts, out=y, expected_rows=expected)
    x0 = torch.where(mask[..., None], x.double(), 0.0)
    check_product(y, x0, w.double(), mask, before=before)


def test_weight_grad_strides_and_two_dimensions():
    g = gen(11)
    d = randn(g, 20, 2, 48).to(BF).transpose(0, 1)[..., 8:32]
    x = randn(g, 2, 20, 64).to(BF)[:, :, 16:56]
    room = torch.full((2, 24, 50), 7.0, device="cuda")
    got = ep.expert_weight_grad(d, x, out=room[..., 3:43])
    want = ep.expert_weight_grad(d.contiguous(), x.contiguous(),
                                 out_dtype=F32)
    assert torch.equal(got, want)
    assert (room[..., :3] == 7).all() and (room[..., 43:] == 7).all()
    one = ep.expert_weight_grad(d[0], x[0], out_dtype=F32)
    assert torch.equal(one, want[0])
    empty = ep.expert_weight_grad(d[:, :0], x[:, :0])
    assert empty.shape == (2, 24, 40) and (empty == 0).all()


def test_products_are_each_others_gradient():
    """<y, dy> moves by <dx, x> and <dw, w> under small changes: the product,
    its row gradient and its weight gradient agree as differences."""
    g = gen(12)
    counts = some_counts(g, 3, 2, 30)
    mask = mask_of(counts, 60)[..., None]
    x, w = randn(g, 3, 60, 64).to(BF), randn(g, 3, 40, 64).to(BF)
    dy = randn(g, 3, 60, 40).to(BF)

    def loss(x, w):
        y = torch.matmul(x, w.transpose(1, 2).contiguous())
        return torch.where(mask, y * dy.double(), 0.0).sum()

    dx = ep.expert_matmul(dy, w.transpose(1, 2), counts, out_dtype=F32)
    dw = ep.expert_weight_grad(dy, x, counts, out_dtype=F32)
    dx = torch.where(mask, dx, 0.0)
    h = 1e-3
    for a, b in ((randn(g, *x.shape).double(), 0), (0, randn(g, *w.shape).double())):
        up = loss(x.double() + h * a, w.double() + h * b)
        down = loss(x.double() - h * a, w.double() - h * b)
        # the loss is linear in each, so the difference is exact but for 64-bit
        # rounding; the gradients carry k (or rows) * 2^-23 of their terms
        terms = (dx.double() * a).abs().sum() + (dw.double() * b).abs().sum()
        got = (dx.double() * a).sum() + (dw.double() * b).sum()
        size = torch.matmul(dy.double().abs(), w.double().abs()).abs().sum()
        assert abs(float(got - (up - down) / (2 * h))) <= \
            float(terms + size * 4) * 64 * STEP32


# ---------------------------------------------------------------------------
# activation
# ---------------------------------------------------------------------------

def swiglu_oracle(h):
    a, b = h.double().chunk(2, -1)
    return a / (1 + torch.exp(-a)) * b


def nearest_8bit(y):
    """The nearest of the type's 127 magnitudes, ties to the even code."""
    value = torch.arange(127, dtype=torch.uint8, device=y.device).view(F8).double()
    middle = (value[1:] + value[:-1]) / 2
    a = y.abs().contiguous()
    code = torch.searchsorted(middle, a)  # middles below a
    tie = (middle[code.clamp(max=125)] == a) & (code < 126)
    code = code + (tie & (code % 2 == 1))
    return torch.copysign(value[code], y)


SHAPES = [(1, 1, 1, 128), (3, 2, 5, 256), (2, 4, 33, 640), (5, 1, 300, 128),
          (1, 8, 130, 2048), (300, 4, 3, 128)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kind", ["random", "none", "full", "one"])
@pytest.mark.parametrize("e, r, length, cols", SHAPES)
def test_swiglu_8bit(e, r, length, cols, kind, dtype):
    g = gen(cols + length)
    counts = some_counts(g, e, r, length, kind)
    mask = mask_of(counts, r * length)
    h = (randn(g, e, r * length, 2 * cols) * 2).to(dtype)
    h[:, 0, :128] = 0
    h[:, -1] *= 1e-3
    h[~mask] = math.nan
    q = torch.full((e, r * length, cols), 7.0, device="cuda").to(F8)
    s = torch.full((e, r * length, cols // 128), 7.0, device="cuda")
    got = ep.expert_swiglu(h, counts, quantize=True, out=q, out_scales=s)
    assert got[0] is q and got[1] is s
    v = swiglu_oracle(h).view(e, r * length, -1, 128)
    amax = v.abs().amax(-1)
    want_s = torch.where(amax > 0, amax / 448, 1.0).float()
    want_q = nearest_8bit(v / want_s.double()[..., None]).view(q.shape)
    assert torch.equal(s[mask], want_s[mask])
    assert torch.equal(q.double()[mask], want_q[mask])
    assert (s[~mask] == 7).all() and (q.float()[~mask] == 7).all()


def test_swiglu_8bit_borders():
    """Values on and next to the middle between two 8-bit values, found by
    aiming: with the gate at 40, sigmoid is 1 to 2^-57, so v is a * b."""
    b = torch.zeros(1, 64, 128, device="cuda")
    code = torch.arange(128, device="cuda") % 126
    value = code.to(torch.uint8).view(F8).float()
    upper = (code + 1).to(torch.uint8).view(F8).float()
    mid = (value + upper) / 2
    for row in range(64):
        b[0, row] = mid * (1 + (row - 32) * 2.0 ** -9)
    b[0, :, 127] = 448.0
    h = torch.cat([torch.full_like(b, 32.0), b], -1).to(BF)
    q, s = ep.expert_swiglu(h, quantize=True)
    v = swiglu_oracle(h)
    want_s = (v.abs().amax(-1) / 448).float()
    assert torch.equal(s[..., 0], want_s)
    assert torch.equal(q.double(), nearest_8bit(v / want_s[..., None].double()))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kind", ["random", "full", "one"])
@pytest.mark.parametrize("e, r, length, cols",
                         SHAPES + [(1, 1, 1, 8), (3, 2, 7, 24), (2, 1, 9, 1000)])
def test_swiglu_and_gradient(e, r, length, cols, kind, dtype):
    g = gen(cols + length)
    counts = some_counts(g, e, r, length, kind)
    mask = mask_of(counts, r * length)
    h = (randn(g, e, r * length, 2 * cols) * 2).to(dtype)
    h[:, 0, :8] = torch.tensor([0.0, -1.278, 20, -20, 60, -60, 1e-3, -100.0])
    d = randn(g, e, r * length, cols).to(dtype)
    h[~mask], d[~mask] = math.nan, math.nan
    out = torch.full((e, r * length, cols), 7.0, dtype=dtype, device="cuda")
    grad = torch.full((e, r * length, 2 * cols), 7.0, dtype=dtype,
                      device="cuda")
    ep.expert_swiglu(h, counts, out=out)
    ep.expert_swiglu_grad(d, h, counts, out=grad)
    assert (out[~mask] == 7).all() and (grad[~mask] == 7).all()

    u = half_step(dtype)
    tiny = torch.finfo(dtype).smallest_normal * u * 2
    hd = h[mask].double().requires_grad_()
    want = swiglu_oracle(hd)
    (want * d[mask].double()).sum().backward()
    # an exponential good to 2 units, and six more operations in 32 bits
    close(out[mask], want.detach(), want.detach().abs() * (u + 8 * STEP32) + tiny)
    a, b = hd.detach().chunk(2, -1)
    sig = torch.sigmoid(a)
    gd = d[mask].double()
    # 1 + a (1 - sig) cancels near a = -1.28: its terms count, not its value
    terms = torch.cat([(gd * b).abs() * sig * (1 + a.abs()),
                       (gd * a).abs() * sig], -1)
    close(grad[mask], hd.grad, hd.grad.abs() * u + terms * 12 * STEP32 + tiny)


def test_swiglu_gradient_against_differences():
    g = gen(13)
    h = randn(g, 1, 6, 32).to(BF)
    d = randn(g, 1, 6, 16).to(BF)
    got = ep.expert_swiglu_grad(d, h).double()
    for c in (0, 5, 15, 16, 31):
        e = torch.zeros(1, 6, 32, dtype=torch.float64, device="cuda")
        e[..., c] = 1e-4
        slope = (swiglu_oracle(h.double() + e) - swiglu_oracle(h.double() - e)) / 2e-4
        want = (slope * d.double()).sum(-1)
        size = (1 + h.double().abs()).amax(-1) ** 2 * d.double().abs().amax(-1)
        close(got[..., c], want, want.abs() * half_step(BF) + size * 1e-7)


def test_swiglu_strides_and_two_dimensions():
    g = gen(14)
    h = randn(g, 2, 20, 320).to(BF)[..., 32:288]
    every = ep.expert_swiglu(h.contiguous())
    room = torch.full((2, 20, 144), 7.0, dtype=BF, device="cuda")
    got = ep.expert_swiglu(h, out=room[..., 8:136])
    assert torch.equal(got, every)
    assert (room[..., :8] == 7).all() and (room[..., 136:] == 7).all()
    assert torch.equal(ep.expert_swiglu(h[0]), every[0])
    q, s = ep.expert_swiglu(h, quantize=True)
    q0, s0 = ep.expert_swiglu(h[0], quantize=True)
    assert torch.equal(q[0].view(torch.uint8), q0.view(torch.uint8))
    assert torch.equal(s[0], s0)
    assert ep.expert_swiglu(h[:, :0]).shape == (2, 0, 128)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

def layer_inputs(seed, tokens, hidden, inner, experts):
    g = gen(seed)
    x = randn(g, tokens, hidden).to(BF)
    gate = randn(g, experts, hidden) * hidden ** -0.5
    w13 = (randn(g, experts, 2 * inner, hidden) * hidden ** -0.5).to(BF)
    w2 = (randn(g, experts, hidden, inner) * inner ** -0.5).to(BF)
    return x, gate, w13, w2


def test_layer_in_8_bits():
    """route, dispatch in 8 bits, product, activation to 8 bits, product,
    combine: against the same steps in 64 bits, from the 8-bit values that
    dispatch made and with the activation rounded to 8 bits."""
    T, H, I, E, K = 100, 512, 256, 8, 2
    x, gate, w13, w2 = layer_inputs(20, T, H, I, E)
    q13, s13 = weights_to_8bit(w13.float())
    q2, s2 = weights_to_8bit(w2.float())
    buf = ep.Buffer(num_experts=E, topk=K, hidden=H, max_tokens=128,
                    dtype=BF, use_fp8=True)
    logits = x.float() @ gate.t()
    logits[17] = -math.inf  # a padded token
    idx, weights = ep.route(logits, K, scoring="sigmoid")
    recv, counts, scales = buf.dispatch(x, idx)
    h = ep.expert_matmul(recv, q13, counts, x_scales=scales, w_scales=s13)
    a, a_scales = ep.expert_swiglu(h, counts, quantize=True)
    y = ep.expert_matmul(a, q2, counts, x_scales=a_scales, w_scales=s2)
    out = buf.combine(y, idx, weights)
    torch.cuda.synchronize()

    assert (idx[17] == -1).all() and (out[17] == 0).all()
    mask = mask_of(counts, recv.shape[1])
    assert int(mask.sum()) == (T - 1) * K
    rx = torch.where(mask[..., None], values_of(recv, scales, 1), 0.0)
    check_product(h, rx, values_of(q13, s13, 128), mask, True)
    ra = torch.where(mask[..., None], values_of(a, a_scales, 1), 0.0)
    check_product(y, ra, values_of(q2, s2, 128), mask, True)
    # rows of an expert lie in token order
    want = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    for e in range(E):
        t, k = (idx == e).nonzero(as_tuple=True)
        rows = y[e, :len(t)].double() * weights[t, k].double()[:, None]
        want.index_add_(0, t, rows)
        size.index_add_(0, t, rows.abs())
    close(out, want, want.abs() * half_step(BF) + size * 4 * STEP32, "combine")


def test_training_step():
    """Forward and backward of a layer in 16 bits, each gradient against
    autograd in 64 bits through the same rounded activations."""
    T, H, I, E, K = 90, 256, 128, 4, 2
    x, gate, w13, w2 = layer_inputs(21, T, H, I, E)
    buf = ep.Buffer(num_experts=E, topk=K, hidden=H, max_tokens=96, dtype=BF)
    logits = x.float() @ gate.t()
    idx, weights = ep.route(logits, K)
    view, counts = buf.dispatch(x, idx)
    recv = view.clone()
    h = ep.expert_matmul(recv, w13, counts)
    a = ep.expert_swiglu(h, counts)
    y = ep.expert_matmul(a, w2, counts)
    out = buf.combine(y, idx, weights)
    torch.cuda.synchronize()

    # the gradient arrives at the experts the way the tokens did
    dout = randn(gen(22), T, H).to(BF)
    rows = torch.zeros_like(y)
    dweights = torch.zeros(T, K, device="cuda")
    for e in range(E):
        t, k = (idx == e).nonzero(as_tuple=True)
        rows[e, :len(t)] = (dout[t].float() * weights[t, k][:, None]).to(BF)
        dweights[t, k] = (dout[t].float() * y[e, :len(t)].float()).sum(-1)
    da = ep.expert_matmul(rows, w2.transpose(1, 2), counts)
    dw2 = ep.expert_weight_grad(rows, a, counts)
    dh = ep.expert_swiglu_grad(da, h, counts)
    dw13 = ep.expert_weight_grad(dh, recv, counts)
    drecv = ep.expert_matmul(dh, w13.transpose(1, 2), counts)
    dlogits = ep.route_grad(dweights, logits, idx)

    # 64 bits, without any rounding between
    xd = x.double().requires_grad_()
    l64 = logits.double().requires_grad_()
    p13, p2 = w13.double().requires_grad_(), w2.double().requires_grad_()
    w64 = weights_of(l64, idx, "softmax", True, 1.0)
    o64 = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for e in range(E):
        t, k = (idx == e).nonzero(as_tuple=True)
        ye = swiglu_oracle(xd[t] @ p13[e].t()) @ p2[e].t()
        o64 = o64.index_add(0, t, ye * w64[t, k][:, None])
    (o64 * dout.double()).sum().backward()
    dx = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for e in range(E):
        t, _ = (idx == e).nonzero(as_tuple=True)
        dx.index_add_(0, t, drecv[e, :len(t)].double())

    # each value passes at most 6 roundings to bfloat16 on its way; in the
    # 2-norm they add up to at most their sum
    for name, got, want in (("out", out, o64), ("x", dx, xd.grad),
                            ("w13", dw13, p13.grad), ("w2", dw2, p2.grad),
                            ("logits", dlogits, l64.grad)):
        off = (got.double() - want).norm() / want.norm()
        assert off <= 6 * half_step(BF), (name, float(off))


def test_captured_and_replayed():
    """The layer's own operators in a graph: every replay is checked against
    the eager result on that replay's inputs."""
    E, R, L, H, I = 4, 2, 32, 256, 128
    g = gen(30)
    logits = randn(g, 64, 8)
    x, xs = rows_to_8bit(randn(g, E, R * L, H))
    w13, s13 = weights_to_8bit(randn(g, E, 2 * I, H) * 0.06)
    w2, s2 = weights_to_8bit(randn(g, E, H, I) * 0.06)
    counts = some_counts(g, E, R, L)
    d = randn(g, E, R * L, I).to(BF)

    def step():
        idx, weights = ep.route(logits, 2, scoring="sigmoid")
        gl = ep.route_grad(weights, logits, idx, scoring="sigmoid")
        h = ep.expert_matmul(x, w13, counts, x_scales=xs, w_scales=s13,
                             out=bufs[0])
        a, sa = ep.expert_swiglu(h, counts, quantize=True, out=bufs[1],
                                 out_scales=bufs[2])
        y = ep.expert_matmul(a, w2, counts, x_scales=sa, w_scales=s2,
                             out=bufs[3])
        dh = ep.expert_swiglu_grad(d, h, counts, out=bufs[4])
        dw = ep.expert_weight_grad(dh, d, counts)
        return [idx, weights, gl, h, y, dh, dw]

    def fresh():
        return [torch.zeros(E, R * L, 2 * I, dtype=BF, device="cuda"),
                torch.zeros(E, R * L, I, device="cuda").to(F8),
                torch.zeros(E, R * L, I // 128, device="cuda"),
                torch.zeros(E, R * L, H, dtype=BF, device="cuda"),
                torch.zeros(E, R * L, 2 * I, dtype=BF, device="cuda")]

    bufs = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    captured = bufs = fresh()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(3):
        logits.copy_(randn(g, 64, 8))
        counts.copy_(some_counts(g, E, R, L))
        x.copy_(rows_to_8bit(randn(g, E, R * L, H))[0])
        for b in captured:
            b.zero_()
        graph.replay()
        torch.cuda.synchronize()
        bufs = fresh()
        want = step()
        torch.cuda.synchronize()
        for i, (p, q) in enumerate(zip(got, want)):
            assert torch.equal(p, q), (turn, i)


def test_on_another_stream():
    g = gen(31)
    x, w = randn(g, 2, 64, 128).to(BF), randn(g, 2, 64, 128).to(BF)
    want = ep.expert_matmul(x, w)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for s in (one, two):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(ep.expert_matmul(x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
