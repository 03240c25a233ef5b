"""The gated activation where its values leave the ordinary range: closed
gates, scales below the smallest float, infinities and NaN, against the
formulas in 64 bits on the CPU.

Tolerances in 16 bits as for ordinary values: the half step of the type, an
exponential good to 2 units and six more operations in 32 bits.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("requires GPU", allow_module_level=True)

import uccl_amd.ep as ep  # noqa: E402

F8, BF, HF = torch.float8_e4m3fn, torch.bfloat16, torch.float16
STEP32 = 2.0 ** -23


def swiglu(a, b):
    a, b = a.double(), b.double()
    return a / (1 + torch.exp(-a)) * b


def nearest_8bit(y):
    """The nearest of the type's 127 magnitudes, ties to the even code; above
    the largest, the largest; NaN stays."""
    value = torch.arange(127, dtype=torch.uint8).view(F8).double()
    middle = (value[1:] + value[:-1]) / 2
    a = y.abs().nan_to_num(nan=0.0, posinf=1e300).contiguous()
    code = torch.searchsorted(middle, a)
    tie = (middle[code.clamp(max=125)] == a) & (code < 126)
    code = code + (tie & (code % 2 == 1))
    return torch.where(y.isnan(), y, torch.copysign(value[code], y))


def quantized(a, b):
    """Values and scale of one group of 128: a NaN does not count for the
    scale, which is 1 where max |v| / 448 is 0 as a float."""
    v = swiglu(a, b)
    amax = v.abs().nan_to_num(nan=0.0, posinf=math.inf).max()
    scale = (amax / 448).float()
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    return nearest_8bit(v / scale.double()), scale


def check_quantized(a, b, dtype):
    """Rows a, b [rows, 128] through the operator and through the formula."""
    a, b = a.to(dtype), b.to(dtype)
    h = torch.cat([a, b], -1)[None]
    q, s = ep.expert_swiglu(h.cuda(), quantize=True)
    q, s = q.cpu()[0].double(), s.cpu()[0, :, 0]
    for row in range(len(a)):
        want_q, want_s = quantized(a[row], b[row])
        assert s[row] == want_s, (row, float(s[row]), float(want_s))
        same = (q[row] == want_q) | (q[row].isnan() & want_q.isnan())
        assert same.all(), (row, q[row][~same], want_q[~same])


@pytest.mark.parametrize("dtype", [BF, HF])
def test_swiglu_8bit_of_closed_gates(dtype):
    """Groups whose largest value, or its 448th part, is below the smallest
    float or below the smallest normal one, with exact zeros among them."""
    gates = torch.tensor([-86., -90, -95, -98, -100, -102, -104, -105, -106,
                          -108, -110, -120, -200, -700, -744, -750, -1000])
    a = gates[:, None].expand(-1, 128).clone()
    up = torch.tensor([1.0, 0.0, -2.0, 0.25, -0.0, 1.5, 3.0, -1e-3])
    check_quantized(a, up.repeat(16).expand(len(a), 128), dtype)


def test_swiglu_8bit_of_far_groups():
    """Groups whose largest value lies outside 1e-20 .. 1e30, up to beyond
    the largest float, and one whose scale is beyond it."""
    g = torch.Generator().manual_seed(1)
    a = torch.randn(8, 128, generator=g).abs() + 0.1
    b = torch.randn(8, 128, generator=g)
    size = torch.tensor([1e-38, 1e-30, 1e-22, 1e-18, 1e28, 1e32, 1e37, 1e38])
    check_quantized(a, b * size[:, None], BF)
    check_quantized(a * torch.tensor([1e2, 1e3, 1e19, 1e36])[:, None]
                    .repeat(2, 1), b * 1e37, BF)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_swiglu_8bit_of_infinities_and_nan(dtype):
    inf, nan = math.inf, math.nan
    g = torch.Generator().manual_seed(2)
    a, b = torch.randn(9, 128, generator=g), torch.randn(9, 128, generator=g)
    for row, (x, y) in enumerate([(inf, 1.0), (inf, -2.0), (inf, 0.0),
                                  (-inf, 1.0), (nan, 1.0), (1.0, nan),
                                  (1.0, inf), (1.0, -inf)]):
        a[row, 37], b[row, 37] = x, y
    a[8] = nan
    check_quantized(a, b, dtype)


def same_kind(got, want, tol):
    """The same NaN and infinities, other values within tol."""
    assert torch.equal(got.isnan(), want.isnan()), (got, want)
    far = want.isinf()
    assert torch.equal(got[far], want[far]), (got[far], want[far])
    fine = want.isfinite()
    assert ((got - want).abs() <= tol)[fine].all(), (got[fine], want[fine])


@pytest.mark.parametrize("dtype", [BF, HF])
def test_swiglu_and_gradient_of_infinities_and_nan(dtype):
    """At a gate of +inf the result and the second half's gradient are
    infinite. The formulas leave 0 * inf, NaN, for the first half's gradient
    there, and for all three at -inf."""
    inf, nan = math.inf, math.nan
    special = [inf, -inf, nan, 1.0, -3.0, 50.0, -20.0, 0.0]
    a, b = torch.meshgrid(torch.tensor(special),
                          torch.tensor([inf, -inf, nan, 2.0, -0.5, 1.0, -1.0,
                                        0.0]), indexing="ij")
    a, b = a.reshape(1, -1).to(dtype), b.reshape(1, -1).to(dtype)
    d = torch.linspace(-2, 3, 64).to(dtype)[None]
    h = torch.cat([a, b], -1)
    out = ep.expert_swiglu(h.cuda()).cpu().double()
    grad = ep.expert_swiglu_grad(d.cuda(), h.cuda()).cpu().double()

    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * u * 2
    want = swiglu(a, b)
    same_kind(out, want, want.abs() * (u + 8 * STEP32) + tiny)
    x, y, g = a.double(), b.double(), d.double()
    sig = torch.sigmoid(x)
    da = g * y * sig * (1 + x * (1 - sig))
    db = g * x * sig
    terms = torch.cat([(g * y).abs() * sig * (1 + x.abs()), db.abs()], -1)
    want = torch.cat([da, db], -1)
    same_kind(grad, want, want.abs() * u + terms * 12 * STEP32 + tiny)


def test_swiglu_of_gates_at_the_ends_of_the_type():
    """Finite gates whose exponential underflows or is 1: no NaN arises."""
    big = torch.finfo(BF).max
    a = torch.tensor([[big, -big, 1e30, -1e30, 300.0, -300.0, 1000.0, -1000.0]])
    b = torch.tensor([[1e-30, 2.0, -1e-10, -2.0, 1.0, 1.0, 0.0, 0.0]])
    a, b = a.to(BF), b.to(BF)
    h = torch.cat([a, b], -1)
    out = ep.expert_swiglu(h.cuda()).cpu().double()
    want = swiglu(a, b)
    same_kind(out, want, want.abs() * (2.0 ** -8 + 8 * STEP32) + 1e-38)
    d = torch.ones(1, 8, dtype=BF)
    grad = ep.expert_swiglu_grad(d.cuda(), h.cuda()).cpu().double()
    sig = torch.sigmoid(a.double())
    da = b.double() * sig * (1 + a.double() * (1 - sig))
    want = torch.cat([da, a.double() * sig], -1)
    same_kind(grad, want, want.abs() * (2.0 ** -8 + 12 * STEP32) + 1e-38)
