"""Refusals of the expert-layer operators. Every argument is checked before
the operands' device is, so the checks run here, without a GPU; the last
refusal of a good call is that its operands are not on one."""

import pytest
import torch

import uccl_amd
import uccl_amd.ep as ep

if not uccl_amd.native_available():
    pytest.skip("native extension not built", allow_module_level=True)

F8 = torch.float8_e4m3fn
BF = torch.bfloat16


def f8(*shape):
    return torch.zeros(*shape).to(F8)


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def refused(message, call, *args, **kw):
    with pytest.raises(RuntimeError, match=message):
        call(*args, **kw)


# --- routing ---------------------------------------------------------------

LOGITS = torch.zeros(4, 16)


@pytest.mark.parametrize("message, args, kw", [
    ("must be on GPU", (LOGITS, 2), {}),
    ("logits must be", (LOGITS[0], 2), {}),
    ("unsupported dtype", (LOGITS.double(), 2), {}),
    ("unsupported dtype", (LOGITS.to(F8), 2), {}),
    ("scoring is", (LOGITS, 2), dict(scoring="tanh")),
    ("topk is 1 to 16", (LOGITS, 0), {}),
    ("topk is 1 to 16", (LOGITS, 17), {}),
    ("topk is 1 to 64", (torch.zeros(1, 128), 65), {}),
    ("1 to 1024 experts", (torch.zeros(1, 1025), 2), {}),
    ("contiguous", (torch.zeros(16, 4).t(), 2), {}),
    ("num_groups", (LOGITS, 2), dict(num_groups=3)),
    ("num_groups", (LOGITS, 2), dict(num_groups=0)),
    ("num_groups", (torch.zeros(1, 128), 2), dict(num_groups=128)),
    ("topk_groups", (LOGITS, 2), dict(num_groups=4, topk_groups=5)),
    ("topk_groups", (LOGITS, 2), dict(num_groups=4, topk_groups=0)),
    ("exceeds the experts", (LOGITS, 5), dict(num_groups=4, topk_groups=1)),
    ("group_best", (LOGITS, 2), dict(num_groups=4, topk_groups=2, group_best=3)),
    ("bias must be float32", (LOGITS, 2), dict(bias=torch.zeros(16, dtype=BF))),
    ("bias has shape", (LOGITS, 2), dict(bias=torch.zeros(15))),
    ("bias must be contiguous", (LOGITS, 2), dict(bias=torch.zeros(32)[::2])),
])
def test_route_refuses(message, args, kw):
    refused(message, ep.route, *args, **kw)


@pytest.mark.parametrize("message, change", [
    ("must be on GPU", {}),
    ("grad_weights must be float32", dict(g=torch.zeros(4, 2, dtype=BF))),
    ("grad_weights has shape", dict(g=torch.zeros(4, 3))),
    ("topk_idx must be int64", dict(idx=i32(4, 2))),
    ("topk_idx must be", dict(idx=torch.zeros(8, dtype=torch.int64))),
    ("topk_idx has shape", dict(idx=torch.zeros(3, 2, dtype=torch.int64))),
    ("topk is 1 to", dict(idx=torch.zeros(4, 0, dtype=torch.int64))),
    ("out must have the dtype", dict(out=torch.zeros(4, 16, dtype=BF))),
    ("out must be contiguous", dict(out=torch.zeros(16, 4).t())),
    ("overlaps", dict(out=LOGITS)),
])
def test_route_grad_refuses(message, change):
    a = dict(g=torch.zeros(4, 2), idx=torch.zeros(4, 2, dtype=torch.int64),
             out=None) | change
    refused(message, ep.route_grad, a["g"], LOGITS, a["idx"], out=a["out"])


# --- products --------------------------------------------------------------

def matmul16(**change):
    a = dict(x=torch.zeros(2, 6, 32, dtype=BF),
             w=torch.zeros(2, 24, 32, dtype=BF), counts=i32(2, 3), kw={})
    a |= change
    return ep.expert_matmul(a["x"], a["w"], a["counts"], **a["kw"])


SHARED = torch.zeros(2 * 6 * 32 + 2 * 6 * 24, dtype=BF)


@pytest.mark.parametrize("message, change", [
    ("must be on GPU", {}),
    ("must be on GPU", dict(counts=None)),
    ("must be on GPU", dict(counts=i32(2))),
    ("must be on GPU", dict(x=torch.zeros(6, 32, dtype=BF),
                            w=torch.zeros(24, 32, dtype=BF), counts=i32(3))),
    ("must be \\[experts", dict(x=torch.zeros(2, 1, 6, 32, dtype=BF))),
    ("w has shape", dict(w=torch.zeros(3, 24, 32, dtype=BF))),
    ("w has shape", dict(w=torch.zeros(2, 24, 40, dtype=BF))),
    ("w has shape", dict(w=torch.zeros(24, 32, dtype=BF))),
    ("x is", dict(w=torch.zeros(2, 24, 32, dtype=torch.float16))),
    ("x has unsupported", dict(x=torch.zeros(2, 6, 32),
                               w=torch.zeros(2, 24, 32))),
    ("k % 8", dict(x=torch.zeros(2, 6, 36, dtype=BF),
                   w=torch.zeros(2, 24, 36, dtype=BF))),
    ("no rows or no columns", dict(w=torch.zeros(2, 0, 32, dtype=BF))),
    ("1 to 1024 experts", dict(x=torch.zeros(1025, 1, 8, dtype=BF),
                               w=torch.zeros(1025, 8, 8, dtype=BF),
                               counts=None)),
    ("counts must be int32", dict(counts=i32(2, 3).long())),
    ("counts has shape", dict(counts=i32(3, 2))),
    ("counts has shape", dict(counts=i32(2, 0))),
    ("counts must be contiguous", dict(counts=i32(3, 2).t())),
    ("do not divide", dict(counts=i32(2, 4))),
    ("rows of x must start", dict(x=torch.zeros(2, 6, 33, dtype=BF)[..., :32])),
    ("rows of x must start", dict(
        x=torch.zeros(2 * 6 * 32 + 1, dtype=BF)[1:].view(2, 6, 32))),
    ("columns of x", dict(x=torch.zeros(2, 6, 64, dtype=BF)[..., ::2])),
    ("columns of w", dict(w=torch.zeros(2, 24, 64, dtype=BF)[..., ::2])),
    ("n % 8", dict(w=torch.zeros(2, 32, 20, dtype=BF).transpose(1, 2))),
    ("scales belong", dict(kw=dict(x_scales=torch.zeros(2, 6, 1)))),
    ("out has shape", dict(kw=dict(out=torch.zeros(2, 6, 23, dtype=BF)))),
    ("out_dtype", dict(kw=dict(out=torch.zeros(2, 6, 24, dtype=BF),
                               out_dtype=torch.float32))),
    ("out has unsupported", dict(kw=dict(out=f8(2, 6, 24)))),
    ("columns of out", dict(
        kw=dict(out=torch.zeros(2, 24, 6, dtype=BF).transpose(1, 2)))),
    ("share memory", dict(
        kw=dict(out=torch.zeros(1, 6, 24, dtype=BF).expand(2, 6, 24)))),
    ("overlaps", dict(
        x=SHARED[:384].view(2, 6, 32),
        kw=dict(out=SHARED[376:376 + 288].view(2, 6, 24)))),
    ("expected_rows", dict(kw=dict(expected_rows=-1))),
])
def test_matmul_refuses(message, change):
    refused(message, matmul16, **change)


def matmul8(**change):
    a = dict(x=f8(2, 6, 256), w=f8(2, 130, 256),
             x_scales=torch.zeros(2, 6, 2), w_scales=torch.zeros(2, 2, 2),
             kw={}) | change
    return ep.expert_matmul(a["x"], a["w"], None, x_scales=a["x_scales"],
                            w_scales=a["w_scales"], **a["kw"])


@pytest.mark.parametrize("message, change", [
    ("must be on GPU", {}),
    ("need x_scales and w_scales", dict(x_scales=None)),
    ("need x_scales and w_scales", dict(w_scales=None)),
    ("x_scales has shape", dict(x_scales=torch.zeros(2, 6, 3))),
    ("w_scales has shape", dict(w_scales=torch.zeros(2, 1, 2))),
    ("x_scales must be float32", dict(x_scales=torch.zeros(2, 6, 2, dtype=BF))),
    ("k % 128", dict(x=f8(2, 6, 192), w=f8(2, 130, 192))),
    ("contiguous along k", dict(w=f8(2, 256, 130).transpose(1, 2))),
    ("does not keep", dict(kw=dict(out_dtype=torch.float32))),
    ("x is", dict(w=torch.zeros(2, 130, 256, dtype=BF))),
])
def test_matmul_8bit_refuses(message, change):
    refused(message, matmul8, **change)


@pytest.mark.parametrize("message, change", [
    ("must be on GPU", {}),
    ("grad_out has shape", dict(g=torch.zeros(2, 5, 24, dtype=BF))),
    ("multiples of 8", dict(g=torch.zeros(2, 6, 20, dtype=BF))),
    ("multiples of 8", dict(x=torch.zeros(2, 6, 20, dtype=BF))),
    ("grad_out is", dict(g=torch.zeros(2, 6, 24, dtype=torch.float16))),
    ("must be bfloat16", dict(g=f8(2, 6, 24), x=f8(2, 6, 32))),
    ("out has shape", dict(out=torch.zeros(2, 32, 24, dtype=BF))),
    ("out has unsupported", dict(out=f8(2, 24, 32))),
    ("counts has shape", dict(counts=i32(1, 2))),
])
def test_weight_grad_refuses(message, change):
    a = dict(g=torch.zeros(2, 6, 24, dtype=BF),
             x=torch.zeros(2, 6, 32, dtype=BF), counts=i32(2, 2),
             out=None) | change
    refused(message, ep.expert_weight_grad, a["g"], a["x"], a["counts"],
            out=a["out"])


# --- activation ------------------------------------------------------------

@pytest.mark.parametrize("message, h, kw", [
    ("must be on GPU", torch.zeros(2, 6, 32, dtype=BF), {}),
    ("must be on GPU", torch.zeros(2, 6, 256, dtype=BF), dict(quantize=True)),
    ("must be bfloat16", torch.zeros(2, 6, 32), {}),
    ("multiple of 8 columns", torch.zeros(2, 6, 24, dtype=BF), {}),
    ("multiple of 128", torch.zeros(2, 6, 128, dtype=BF), dict(quantize=True)),
    ("out must have the dtype", torch.zeros(2, 6, 32, dtype=BF),
     dict(out=torch.zeros(2, 6, 16))),
    ("out must be float8", torch.zeros(2, 6, 256, dtype=BF),
     dict(quantize=True, out=torch.zeros(2, 6, 128, dtype=BF))),
    ("out_scales has shape", torch.zeros(2, 6, 256, dtype=BF),
     dict(quantize=True, out_scales=torch.zeros(2, 6, 2))),
    ("out_scales belongs", torch.zeros(2, 6, 256, dtype=BF),
     dict(out_scales=torch.zeros(2, 6, 1))),
])
def test_swiglu_refuses(message, h, kw):
    refused(message, ep.expert_swiglu, h, i32(2, 3), **kw)


def test_swiglu_grad_refuses():
    h, g = torch.zeros(2, 6, 32, dtype=BF), torch.zeros(2, 6, 16, dtype=BF)
    refused("must be on GPU", ep.expert_swiglu_grad, g, h)
    refused("grad_out has shape", ep.expert_swiglu_grad, g[:, :5], h)
    refused("dtype of h", ep.expert_swiglu_grad, g.float(), h)
    refused("overlaps", ep.expert_swiglu_grad, g, h, out=h)


def test_no_gradient_is_lost():
    """These operators record no autograd graph, so an operand that would want
    one is refused, unless grad mode is off."""
    x = torch.zeros(2, 6, 32, dtype=BF, requires_grad=True)
    w = torch.zeros(2, 24, 32, dtype=BF)
    refused("x requires grad", ep.expert_matmul, x, w)
    refused("logits requires grad", ep.route, LOGITS.clone().requires_grad_(), 2)
    refused("h requires grad", ep.expert_swiglu, x)
    with torch.no_grad():
        refused("must be on GPU", ep.expert_matmul, x, w)


def test_results_that_require_grad_are_refused():
    x, w = torch.zeros(2, 6, 32, dtype=BF), torch.zeros(2, 24, 32, dtype=BF)

    def leaf(*shape):
        return torch.zeros(*shape, dtype=BF, requires_grad=True)

    refused("out requires grad", ep.expert_matmul, x, w, out=leaf(2, 6, 24))
    refused("out requires grad", ep.expert_weight_grad, x, x,
            out=leaf(2, 32, 32))
    refused("out requires grad", ep.expert_swiglu, x, out=leaf(2, 6, 16))
    refused("out requires grad", ep.expert_swiglu_grad, x[..., :16], x,
            out=leaf(2, 6, 32))


def test_sizes_that_32_bits_do_not_count_are_refused():
    def wide(*shape):  # one element, repeated
        return torch.zeros(1, dtype=BF).expand(*shape)

    long = 1 << 28
    refused("too large", ep.expert_matmul, wide(1, 1, long), wide(1, 8, long),
            out=torch.zeros(1, 1, 8, dtype=BF))
    refused("too large", ep.expert_matmul, wide(1, 1, 8), wide(1, long, 8),
            out=wide(1, 1, long))
    refused("too large|too many slots", ep.expert_matmul, wide(1, 4 * long, 8),
            wide(1, 8, 8), out=wide(1, 4 * long, 8))
    refused("too large", ep.expert_weight_grad, wide(1, 1, 8),
            wide(1, 1, long), out=wide(1, 8, long))
    refused("too many slots", ep.expert_swiglu, wide(1, 4 * long, 16),
            out=wide(1, 4 * long, 8))
    row = torch.zeros(1, 8).expand(1 << 25, 8)
    idx = torch.zeros(1, 2, dtype=torch.int64).expand(1 << 25, 2)
    refused("too many tokens", ep.route_grad, row[:, :2], row, idx,
            out=row)
