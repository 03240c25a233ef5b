"""Further refusals of the expert-layer operators, and calls that pass every
check: without a GPU those end with the refusal of operands that are not on
one."""

import pytest
import torch
from torch.autograd import forward_ad

import uccl_amd
import uccl_amd.ep as ep

if not uccl_amd.native_available():
    pytest.skip("native extension not built", allow_module_level=True)

F8, BF = torch.float8_e4m3fn, torch.bfloat16


def refused(message, call, *args, **kw):
    with pytest.raises(RuntimeError, match=message):
        call(*args, **kw)


def passes(call, *args, **kw):
    refused("must be on GPU", call, *args, **kw)


# --- sums of 8-bit products ------------------------------------------------

def test_precise_belongs_to_8_bit_operands():
    x, w = torch.zeros(2, 6, 256).to(F8), torch.zeros(2, 130, 256).to(F8)
    scales = dict(x_scales=torch.zeros(2, 6, 2), w_scales=torch.zeros(2, 2, 2))
    for out_dtype in (None, BF, torch.float16, torch.float32):
        passes(ep.expert_matmul, x, w, out_dtype=out_dtype, precise=True,
               **scales)
    refused("does not keep", ep.expert_matmul, x, w, out_dtype=torch.float32,
            precise=False, **scales)
    refused("out has unsupported", ep.expert_matmul, x, w, out_dtype=F8,
            precise=True, **scales)
    refused("precise belongs", ep.expert_matmul, x.to(BF), w.to(BF),
            precise=True)


# --- derivatives -----------------------------------------------------------

def with_every_operator(x):
    """(operand's name, call) of each operator with `x` [2, 8, 16] in every
    place that takes values."""
    plain = torch.zeros_like(x)
    row = x[0].float()
    idx = torch.zeros(8, 2, dtype=torch.int64)
    return [
        ("logits", lambda: ep.route(row, 2)),
        ("bias", lambda: ep.route(torch.zeros(8, 16), 2, bias=row[0])),
        ("grad_weights", lambda: ep.route_grad(row[:, :2].contiguous(),
                                               torch.zeros(8, 16), idx)),
        ("logits", lambda: ep.route_grad(torch.zeros(8, 2), row, idx)),
        ("x", lambda: ep.expert_matmul(x, plain)),
        ("w", lambda: ep.expert_matmul(plain, x)),
        ("grad_out", lambda: ep.expert_weight_grad(x, plain)),
        ("x", lambda: ep.expert_weight_grad(plain, x)),
        ("h", lambda: ep.expert_swiglu(x)),
        ("grad_out", lambda: ep.expert_swiglu_grad(
            x[..., :8].contiguous(), plain)),
        ("h", lambda: ep.expert_swiglu_grad(plain[..., :8].contiguous(), x)),
    ]


@pytest.mark.parametrize("grad_mode", [True, False])
def test_no_forward_mode_derivative_is_lost(grad_mode):
    plain = torch.zeros(2, 8, 16, dtype=BF)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = forward_ad.make_dual(plain, torch.ones_like(plain))
        for name, call in with_every_operator(dual):
            refused(f"{name} carries a forward-mode derivative", call)
        primal = forward_ad.unpack_dual(dual).primal
        for _, call in with_every_operator(primal):
            passes(call)
    for _, call in with_every_operator(plain):
        passes(call)


def test_an_autograd_function_may_call_them_in_forward_mode():
    """A Function with a jvp of its own: its forward sees the operands'
    values, whatever they carry."""

    class Gate(torch.autograd.Function):
        @staticmethod
        def forward(ctx, h):
            return ep.expert_swiglu(h)

        @staticmethod
        def jvp(ctx, t):
            return t[..., :8]

    plain = torch.zeros(2, 8, 16, dtype=BF)
    with forward_ad.dual_level():
        passes(Gate.apply, forward_ad.make_dual(plain, torch.ones_like(plain)))
