"""Products on both sides of every limit by which a kernel is chosen: the
expected rows and the number of tiles change the kernel, never the result.

Tolerances as for all products: one rounding to the result type, n terms in 32
bits, and 2^-13 of the terms' magnitudes for the 8-bit matrix unit.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("requires GPU", allow_module_level=True)

import uccl_amd.ep as ep  # noqa: E402

F8, BF = torch.float8_e4m3fn, torch.bfloat16


@pytest.mark.parametrize("expected", [2, 3, 8, 9, 16, 17, 24, 25, 192, 193])
@pytest.mark.parametrize("kind", ["8 bit", "16 bit", "turned"])
@pytest.mark.parametrize("e, n", [(40, 1032),   # 200 tiles of 256 x 64
                                  (60, 1288)])  # 360, more than the card has
def test_limits_of_expected_rows(e, n, kind, expected):
    g = torch.Generator(device="cuda").manual_seed(expected)
    slots, k = 200, 256
    x = torch.randn(e, slots, k, device="cuda", generator=g)
    w = torch.randn(e, n, k, device="cuda", generator=g) * 0.05
    counts = torch.randint(0, min(2 * expected, slots) + 1, (e, 1),
                           device="cuda", generator=g, dtype=torch.int32)
    mask = torch.arange(slots, device="cuda") < counts
    y = torch.full((e, slots, n), 7.0, dtype=BF, device="cuda")
    if kind == "8 bit":
        x, w = (x * 50).to(F8), (w * 1000).to(F8)
        xs = torch.full((e, slots, 2), 0.02, device="cuda")
        ws = torch.full((e, -(-n // 128), 2), 1e-3, device="cuda")
        ep.expert_matmul(x, w, counts, x_scales=xs, w_scales=ws, out=y,
                         expected_rows=expected)
        scale = xs[0, 0, 0].double() * ws[0, 0, 0].double()
    else:
        x, w = x.to(BF), w.to(BF)
        if kind == "turned":
            w = w.transpose(1, 2).contiguous().transpose(1, 2)
        ep.expert_matmul(x, w, counts, out=y, expected_rows=expected)
        scale = 1.0
    x, wt = x.double(), w.double().transpose(1, 2).contiguous()
    want = torch.matmul(x, wt) * scale
    size = torch.matmul(x.abs(), wt.abs()) * scale
    off = (k + 3) * 2.0 ** -23 + (2.0 ** -13 if kind == "8 bit" else 0.0)
    bad = (y.double() - want).abs() > want.abs() * 2.0 ** -8 + size * off
    assert not bad[mask].any()
    assert (y[~mask] == 7).all()


@pytest.mark.parametrize("expected", [2, 3, 16, 17, 32, 33])
@pytest.mark.parametrize("precise", [False, True])
def test_limits_where_8_bit_rows_lie_far_apart(precise, expected):
    """Rows that a tile's 32-bit offsets do not reach, shared by all experts."""
    g = torch.Generator(device="cuda").manual_seed(expected)
    e, slots, n, k = 40, 300, 1032, 256
    room = torch.empty(slots << 24, dtype=torch.uint8, device="cuda").view(F8)
    x = room.view(1, slots, 1 << 24)[..., :k]
    x.copy_((torch.randn(1, slots, k, device="cuda", generator=g) * 50).to(F8))
    x = x.expand(e, slots, k)
    w = (torch.randn(e, n, k, device="cuda", generator=g) * 50).to(F8)
    xs = torch.full((e, slots, 2), 0.0625, device="cuda")
    ws = torch.full((e, 9, 2), 0.125, device="cuda")
    counts = torch.randint(0, 2 * expected + 1, (e, 1), device="cuda",
                           generator=g, dtype=torch.int32)
    mask = torch.arange(slots, device="cuda") < counts
    y = torch.full((e, slots, n), 7.0, dtype=BF, device="cuda")
    ep.expert_matmul(x, w, counts, x_scales=xs, w_scales=ws, out=y,
                     expected_rows=expected, precise=precise)
    x, wt = x.double(), w.double().transpose(1, 2).contiguous()
    want = torch.matmul(x.contiguous(), wt) * 2.0 ** -7
    size = torch.matmul(x.abs().contiguous(), wt.abs()) * 2.0 ** -7
    off = (k + 3) * 2.0 ** -23 + (0.0 if precise else 2.0 ** -13)
    bad = (y.double() - want).abs() > want.abs() * 2.0 ** -8 + size * off
    assert not bad[mask].any()
    assert (y[~mask] == 7).all()
