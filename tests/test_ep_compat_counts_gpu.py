"""The expert operators over what deep_ep_compat's low-latency dispatch gives."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("requires GPU", allow_module_level=True)

import uccl_amd.ep as ep  # noqa: E402
from uccl_amd.ep import deep_ep_compat  # noqa: E402


def test_product_over_a_low_latency_dispatch():
    g = torch.Generator(device="cuda").manual_seed(0)
    T, H, E, K, N = 50, 256, 4, 2, 64
    x = torch.randn(T, H, device="cuda", generator=g).bfloat16()
    w = torch.randn(E, N, H, device="cuda", generator=g).bfloat16()
    idx, _ = ep.route(torch.randn(T, E, device="cuda", generator=g), K)
    buf = deep_ep_compat.Buffer()
    packed, summed, handle, _, _ = buf.low_latency_dispatch(x, idx, 64, E)
    assert handle.recv_counts.shape == (E, 1)
    y = ep.expert_matmul(packed, w, handle.recv_counts)
    torch.cuda.synchronize()
    for e in range(E):
        tokens = (idx == e).any(-1).nonzero()[:, 0]
        n = int(handle.recv_counts[e, 0])
        assert n == len(tokens) == int(summed[e])
        # rows of a rank lie in token order
        want = x[tokens].double() @ w[e].double().t()
        size = x[tokens].double().abs() @ w[e].double().abs().t()
        # one rounding to bfloat16, and H terms in 32 bits
        tol = want.abs() * 2.0 ** -8 + size * H * 2.0 ** -23
        assert ((y[e, :n].double() - want).abs() <= tol).all()
