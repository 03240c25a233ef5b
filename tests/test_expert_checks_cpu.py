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


# --- results inside a larger tensor ----------------------------------------

def test_results_may_lie_between_the_columns_of_operands():
    room = torch.zeros(2, 6, 96, dtype=BF)
    h, out, grad = room[..., :32], room[..., 32:48], room[..., 48:80]
    w = torch.zeros(2, 16, 32, dtype=BF)
    passes(ep.expert_swiglu, h, out=out)
    passes(ep.expert_swiglu_grad, out, h, out=grad)
    passes(ep.expert_swiglu_grad, room[..., 80:], grad, out=h)
    passes(ep.expert_matmul, h, w, out=out)
    passes(ep.expert_matmul, grad, w, out=out)
    passes(ep.expert_matmul, h[:, :1], w, out=out[:, :1])
    # weights read turned, between the columns of their gradient
    both = torch.zeros(2, 16, 64, dtype=BF)
    passes(ep.expert_weight_grad, room[..., 32:48], h, out=both[..., :32])
    passes(ep.expert_matmul, out.contiguous(), both[..., :32].transpose(1, 2),
           out=torch.zeros(2, 6, 32, dtype=BF))
    # one row of 6, next to each other
    flat = torch.zeros(6 * 48, dtype=BF)
    passes(ep.expert_swiglu, flat[:192].view(1, 6, 32),
           out=flat[192:].view(1, 6, 16))


def test_results_that_share_an_element_with_an_operand_are_refused():
    room = torch.zeros(2, 6, 96, dtype=BF)
    h = room[..., :32]
    w = torch.zeros(2, 16, 32, dtype=BF)
    for first in (0, 8, 16, 24):
        refused("overlaps", ep.expert_swiglu, h, out=room[..., first:first + 16])
        refused("overlaps", ep.expert_matmul, h, w,
                out=room[..., first:first + 16])
    refused("overlaps", ep.expert_matmul, h, w, out=room[..., 31:47])
    passes(ep.expert_matmul, h, w, out=room[..., 32:48])
    # columns that a row's end wraps into
    line = torch.zeros(2 * 6 * 48 + 48, dtype=BF)
    x = line[40:].as_strided((2, 6, 32), (6 * 48, 48, 1))
    refused("overlaps", ep.expert_matmul, x, w,
            out=line.as_strided((2, 6, 16), (6 * 48, 48, 1), 16))
    passes(ep.expert_matmul, x, w,
           out=line.as_strided((2, 6, 16), (6 * 48, 48, 1), 24))
    # another pitch, so that some rows meet
    refused("overlaps", ep.expert_matmul, h, w,
            out=room.view(-1).as_strided((2, 6, 16), (6 * 80, 80, 1), 32))
    # rows shared by all experts
    one = torch.zeros(6, 48, dtype=BF)
    refused("overlaps", ep.expert_matmul, one[:, :32].expand(1, 6, 32), w[:1],
            out=one[:, 31:47].unsqueeze(0))
    # 8-bit values and their scales in one place
    h8, q = torch.zeros(1, 6, 256, dtype=BF), torch.zeros(1, 6, 128).to(F8)
    refused("out_scales overlaps", ep.expert_swiglu, h8, quantize=True, out=q,
            out_scales=q.view(-1)[:24].view(torch.float32).view(1, 6, 1))


def test_results_over_the_counts_are_refused():
    """Blocks read the counts while others already write results."""
    out = torch.zeros(2, 6, 16, dtype=BF)
    counts = out.view(torch.int32).view(-1)[8:12].view(2, 2)
    x, w = torch.zeros(2, 6, 32, dtype=BF), torch.zeros(2, 16, 32, dtype=BF)
    refused("out overlaps", ep.expert_matmul, x, w, counts, out=out)
    refused("out overlaps", ep.expert_swiglu, x, counts, out=out)
    refused("out overlaps", ep.expert_swiglu_grad, torch.zeros_like(out[..., :8])
            .contiguous(), x[..., :16].contiguous(), counts, out=out)
    dw = torch.zeros(2, 8, 32, dtype=BF)
    refused("out overlaps", ep.expert_weight_grad, x[..., :8].contiguous(), x,
            dw.view(torch.int32).view(-1)[:4].view(2, 2), out=dw)
    scales = torch.zeros(2, 6, 1)
    refused("out_scales overlaps", ep.expert_swiglu,
            torch.zeros(2, 6, 256, dtype=BF),
            scales.view(torch.int32).view(-1)[:4].view(2, 2), quantize=True,
            out_scales=scales)
