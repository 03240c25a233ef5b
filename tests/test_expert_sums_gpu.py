"""expert_matmul of 8-bit operands with precise=True: sums in 32 bits.

The operands are whole numbers whose products' magnitudes add up to less than
2^24, with scales that are powers of two. A sum in 32 bits is then exact in
any order, and a result is the exact one, rounded once. Among the products are
pairs of +-448 * 448 that cancel: a sum that is aligned to its largest term
loses the small ones beside them.
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


def operands(e, slots, n, k, seed=0):
    """x, w and their scales, and the exact products in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def whole(*shape):
        return torch.randint(-4, 5, shape, device="cuda", generator=g).float()

    x, w = whole(e, slots, k), whole(e, n, k)
    for b in range(k // 128):  # one pair of columns in every block
        at = torch.randperm(128, device="cuda", generator=g)[:2] + b * 128
        x[..., at] = 448.0
        w[..., at[0]] = 448.0
        w[..., at[1]] = -448.0
    xs = torch.full((e, slots, k // 128), 0.5, device="cuda")
    ws = torch.full((e, -(-n // 128), k // 128), 2.0, device="cuda")
    # 128 products of at most 16, and two of 2^17.7, in each of the blocks
    assert k // 128 * (126 * 16 + 2 * 448 * 448) < 1 << 24
    want = torch.matmul(x.double(), w.double().transpose(1, 2).contiguous())
    return x.to(F8), w.to(F8), xs, ws, want


def check(want, got, mask):
    assert torch.equal(got[mask], want.to(got.dtype)[mask])


def mask_of(counts, slots):
    e, r = counts.shape
    at = torch.arange(slots // r, device="cuda")
    return (at < counts[:, :, None]).view(e, slots)


@pytest.mark.parametrize("out", [BF, HF, F32])
@pytest.mark.parametrize("e, r, length, n, k, expected", [
    (1, 1, 1, 8, 128, None),        # one row
    (1, 1, 1, 1, 256, None),
    (1, 1, 70, 512, 2048, None),    # few rows, several turns of a block
    (40, 2, 9, 64, 128, 4),
    (2, 4, 40, 130, 384, 3),
    (40, 3, 23, 1032, 384, 17),     # narrow tiles
    (60, 3, 23, 1032, 384, 3),
    (40, 3, 23, 1032, 384, 33),     # wide ones
    (40, 3, 23, 1032, 384, 65),
    (9, 1, 300, 1030, 128, None),
    (33, 1, 300, 515, 640, None),
])
def test_precise_products_are_exact(e, r, length, n, k, expected, out):
    x, w, xs, ws, want = operands(e, r * length, n, k)
    g = torch.Generator(device="cuda").manual_seed(1)
    counts = torch.randint(0, length + 1, (e, r), device="cuda", generator=g,
                           dtype=torch.int32)
    counts[0, 0] = length
    mask = mask_of(counts, r * length)
    x.view(torch.uint8)[~mask] = 0x7F  # NaN
    xs[~mask] = math.nan
    y = torch.full((e, r * length, n), 7.0, dtype=out, device="cuda")
    got = ep.expert_matmul(x, w, counts, x_scales=xs, w_scales=ws, out=y,
                           expected_rows=expected, precise=True)
    assert got is y
    check(want, y, mask)
    assert (y[~mask] == 7).all(), "rows behind changed"


@pytest.mark.parametrize("expected", [1, 32, 600])
def test_precise_products_of_ordinary_data(expected):
    """Against 64 bits: a sum of n terms in 32 bits is off by at most
    n * 2^-23 * sum |terms|, its scaling by two more steps."""
    g = torch.Generator(device="cuda").manual_seed(3)
    e, slots, n, k = 20, 90, 1032, 384

    def randn(*shape):
        v = torch.randn(*shape, device="cuda", generator=g)
        return (v * 100).clamp(-448, 448).to(F8)

    x, w = randn(e, slots, k), randn(e, n, k)
    xs = torch.rand(e, slots, 3, device="cuda", generator=g) + 0.01
    ws = torch.rand(e, 9, 3, device="cuda", generator=g) + 0.01
    x64 = x.double() * xs.double().repeat_interleave(128, -1)
    w64 = w.double() * ws.double().repeat_interleave(128, -1) \
        .repeat_interleave(128, 1)[:, :n]
    wt = w64.transpose(1, 2).contiguous()
    want = torch.matmul(x64, wt)
    size = torch.matmul(x64.abs(), wt.abs())
    got = ep.expert_matmul(x, w, x_scales=xs, w_scales=ws, out_dtype=F32,
                           expected_rows=expected, precise=True)
    assert ((got - want).abs() <= size * (k + 3) * 2.0 ** -23).all()


def test_precise_products_of_extremes():
    """Every byte of the type is widened to its value; a NaN value, zero and
    infinite scales reach only their own row."""
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    w = torch.zeros(1, 256, 128, device="cuda").to(F8)
    w[0, :, 5] = codes.view(F8)
    x = torch.zeros(1, 4, 128, device="cuda").to(F8)
    x[0, :, 5] = 1.0
    x.view(torch.uint8)[0, 3, 7] = 0x7F
    xs = torch.tensor([1.0, 0.0, math.inf, 1.0], device="cuda").view(1, 4, 1)
    ws = torch.ones(1, 2, 1, device="cuda")
    for expected in (1, 40, 200):
        y = ep.expert_matmul(x, w, x_scales=xs, w_scales=ws, out_dtype=F32,
                             expected_rows=expected, precise=True)[0].double()
        for row, scale in ((0, 1.0), (1, 0.0), (2, math.inf)):
            want = codes.view(F8).double() * scale
            assert ((y[row] == want) | (y[row].isnan() & want.isnan())).all()
        assert y[3].isnan().all()


@pytest.mark.parametrize("kind", ["rows", "weights"])
def test_precise_products_of_far_rows(kind):
    """Rows that lie further apart than 32 bits reach."""
    e, k = 1, 256
    slots, n = (300, 4200) if kind == "rows" else (2000, 300)
    x, w, xs, ws, want = operands(e, slots, n, k, 5)
    # 300 rows of x 16 MiB apart, or rows of weights just less than that, the
    # most there may be: a tile's then span more than 32 bits
    if kind == "rows":
        room = torch.empty(slots * (1 << 24), dtype=torch.uint8,
                           device="cuda").view(F8)
        far = room.view(1, slots, 1 << 24)[..., :k]
        far.copy_(x)
        x = far
    else:
        pitch = (1 << 24) - 16
        room = torch.empty(n * pitch, dtype=torch.uint8, device="cuda").view(F8)
        far = room.view(1, n, pitch)[..., :k]
        far.copy_(w)
        w = far
    got = ep.expert_matmul(x, w, x_scales=xs, w_scales=ws, out_dtype=F32,
                           precise=True)
    check(want, got, torch.ones(e, slots, dtype=torch.bool, device="cuda"))


def test_precise_products_captured_and_replayed():
    x, w, xs, ws, want = operands(2, 200, 1000, 256, 7)
    y = torch.zeros(2, 200, 1000, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ep.expert_matmul(x, w, x_scales=xs, w_scales=ws, out=y, precise=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ep.expert_matmul(x, w, x_scales=xs, w_scales=ws, out=y, precise=True)
    every = torch.ones(2, 200, dtype=torch.bool, device="cuda")
    for turn in range(3):
        x2, w2, _, _, want = operands(2, 200, 1000, 256, 7 + turn)
        x.copy_(x2)
        w.copy_(w2)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check(want, y, every)
