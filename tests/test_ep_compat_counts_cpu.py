"""The counts of each rank that a low-latency dispatch's handle keeps: rows of
rank r lie at [e, r * max_tokens], so the sums over ranks do not find them."""

import pytest
import torch

from uccl_amd.ep import deep_ep_compat

COUNTS = torch.tensor([[3, 0], [1, 4]], dtype=torch.int32)


class TwoRanks:
    """The native buffer of a rank with 2 of 4 experts, without a GPU."""

    rank, world, local_experts = 0, 2, 2

    def __init__(self, hidden, max_tokens, topk, dtype, **_):
        self.hidden, self.topk, self.dtype = hidden, topk, dtype
        self.recv = torch.zeros(2, 2 * max_tokens, hidden, dtype=dtype)

    def dispatch_send(self, x, topk_idx, reuse_plan=False):
        pass

    def dispatch_recv(self, counts):
        counts.copy_(COUNTS)

    def recv_x_view(self):
        return self.recv

    def recv_scale_view(self):
        return self.recv[..., :1]


@pytest.mark.parametrize("use_fp8", [False, True])
@pytest.mark.parametrize("later", [False, True])
def test_handle_keeps_the_counts_of_each_rank(monkeypatch, later, use_fp8):
    monkeypatch.setattr(deep_ep_compat, "_NativeBuffer", TwoRanks)
    monkeypatch.setattr(deep_ep_compat, "_event", lambda: None)
    buf = deep_ep_compat.Buffer()
    packed, summed, handle, _, hook = buf.low_latency_dispatch(
        torch.zeros(4, 128), torch.zeros(4, 2, dtype=torch.int64), 8, 4,
        use_fp8=use_fp8, return_recv_hook=later)
    if later:
        hook()
    assert torch.equal(handle.recv_counts, COUNTS)
    assert summed.tolist() == [3, 5]
