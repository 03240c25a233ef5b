"""Results that lie between the columns of operands in one tensor."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("requires GPU", allow_module_level=True)

import uccl_amd.ep as ep  # noqa: E402

BF = torch.bfloat16


@pytest.mark.parametrize("slots, expected", [(6, None), (300, None), (300, 20)])
def test_results_between_the_columns_of_operands(slots, expected):
    """The same bits as into tensors of their own, and nothing beside them
    changes."""
    g = torch.Generator(device="cuda").manual_seed(slots)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(BF)

    e, i, n = 40, 64, 520
    room = randn(e, slots, 2 * i + i + 8 + n)
    before = room.clone()
    h, a = room[..., :2 * i], room[..., 2 * i:3 * i]
    y = room[..., -n:]
    w = randn(e, n, i)
    counts = torch.randint(0, slots + 1, (e, 1), device="cuda", generator=g,
                           dtype=torch.int32)
    valid = torch.arange(slots, device="cuda") < counts
    ep.expert_swiglu(h, counts, out=a)
    ep.expert_matmul(a, w, counts, out=y, expected_rows=expected)
    want = before.clone()
    want_a = ep.expert_swiglu(before[..., :2 * i].contiguous())
    want[..., 2 * i:3 * i][valid] = want_a[valid]
    want_y = ep.expert_matmul(want_a, w, counts, expected_rows=expected)
    want[..., -n:][valid] = want_y[valid]
    assert torch.equal(room, want)

    # gradients into the columns of the rows that they belong to
    d = randn(e, slots, i)
    pair = torch.cat([before[..., :2 * i], randn(e, slots, 2 * i)], -1)
    ep.expert_swiglu_grad(d, pair[..., :2 * i], counts, out=pair[..., 2 * i:])
    want = ep.expert_swiglu_grad(d, before[..., :2 * i].contiguous(), counts)
    assert torch.equal(pair[..., 2 * i:][valid], want[valid])
    assert torch.equal(pair[..., :2 * i], before[..., :2 * i])
    both = randn(e, slots, 2 * i)
    x, grad = both[..., :i], both[..., i:]
    full = torch.zeros(e, i, 2 * i, dtype=BF, device="cuda")
    ep.expert_weight_grad(grad, x, counts, out=full[..., :i])
    want = ep.expert_weight_grad(grad.contiguous(), x.contiguous(), counts)
    assert torch.equal(full[..., :i], want)
    assert (full[..., i:] == 0).all()
