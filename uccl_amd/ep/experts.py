"""Operators of an expert layer over the slot arrays of ``uccl_amd.ep.Buffer``.

Between the router's logits and ``combine``, on one rank:

    idx, weights = ep.route(logits, topk)
    recv_x, counts, recv_scales = buf.dispatch(x, idx)          # use_fp8=True
    rows = -(-len(x) * buf.world * topk // buf.num_experts)     # on average
    h = ep.expert_matmul(recv_x, w13, counts, x_scales=recv_scales,
                         w_scales=w13_scales, expected_rows=rows)
    a, a_scales = ep.expert_swiglu(h, counts, quantize=True)
    y = ep.expert_matmul(a, w2, counts, x_scales=a_scales,
                         w_scales=w2_scales, expected_rows=rows)
    out = buf.combine(y, idx, weights)

A slot array is [experts, slots, columns]; with counts [experts, sources]
(int32, as ``dispatch`` returns it) source r of expert e has counts[e, r] valid
rows from row r * slots / sources on. Counts stay on the GPU; one below zero or
above slots / sources counts as the nearest of the two. Rows behind the valid
ones are neither read nor written: in a result that was passed as ``out`` they
keep their values, in a fresh one they are undefined. ``counts=None``: all rows
are valid; counts [experts] stands for one source. ``deep_ep_compat`` returns
sums over the ranks, which fit only where there is one rank: its handle's
``recv_counts`` are the counts to pass. Two-dimensional operands are those of a
single expert. At most 1024 experts and 2048 counts. A result shares no memory
with an operand or the counts; it may lie between an operand's columns in a
larger tensor.

Every call is enqueued on the current stream of its operands' device and may be
captured into a graph. Operands lie on one device; rows start at 16-byte
boundaries, which sets the multiples of columns that the functions name.
Nothing here records an autograd graph: each operator with a gradient has its
own function for it, and an operand that requires grad is refused while grad
mode is on, so that a gradient is not lost silently (call it under
``torch.no_grad()``, from an ``autograd.Function``, or with ``.detach()``). One
that carries a forward-mode derivative is refused as well.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad


def _native(**operands):
    from uccl_amd import _load_native

    if torch.is_grad_enabled():
        for name, t in operands.items():
            if t is not None and t.requires_grad:
                raise RuntimeError(
                    f"uccl_amd: {name} requires grad, and this operator "
                    "records no autograd graph; call it under torch.no_grad() "
                    "and take the gradient from its *_grad function")
    # inside a dual_level(), and whatever grad mode says; a Function's forward
    # has them off
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for name, t in operands.items():
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(
                    f"uccl_amd: {name} carries a forward-mode derivative, "
                    "which this operator would drop; take the primal with "
                    "torch.autograd.forward_ad.unpack_dual")
    return _load_native(required=True)


def _slots(t: Optional[torch.Tensor]):
    return t.unsqueeze(0) if t is not None and t.dim() == 2 else t


def _counts(counts: Optional[torch.Tensor], x: torch.Tensor):
    """[experts, sources] counts from what the caller has."""
    if counts is None or counts.dim() != 1:
        return counts
    return counts.unsqueeze(0 if x.dim() == 2 else 1)


def route(logits: torch.Tensor, topk: int, *, scoring: str = "softmax",
          bias: Optional[torch.Tensor] = None, num_groups: int = 1,
          topk_groups: int = 1, group_best: int = 2,
          renormalize: bool = True, scale: float = 1.0):
    """Pick each token's experts: returns (topk_idx [T, topk] int64,
    topk_weights [T, topk] float32), as dispatch and combine take them.

    logits [T, E] (float32, bfloat16 or float16, E <= 1024, topk <= 64) become
    scores by ``scoring`` ("softmax" over the row, or "sigmoid"). An expert is
    ranked by its score plus ``bias`` [E] (float32; the weights leave it out).
    With ``num_groups`` > 1 (at most 64, a divisor of E) a group's value is the
    sum of its ``group_best`` (1 or 2) largest ranks, and only experts of the
    ``topk_groups`` best groups are picked. Picks are in falling order, ties go
    to the lowest index; ranks are formed and compared in 64 bits. The weights
    are the picks' scores, divided by their sum if ``renormalize``, times
    ``scale``.

    An expert whose logit (or logit plus bias) is -inf is closed: it is never
    picked. A row with fewer than topk open experts is filled with index -1 and
    weight 0, which dispatch and combine skip. A logit that is NaN is never
    picked and makes all weights of its row NaN, as +inf does under softmax.
    """
    C = _native(logits=logits, bias=bias)
    tokens = logits.shape[0] if logits.dim() == 2 else 0
    idx = torch.empty(tokens, topk, dtype=torch.int64, device=logits.device)
    weights = torch.empty(tokens, topk, dtype=torch.float32,
                          device=logits.device)
    C.ep_route(logits, bias, scoring, num_groups, topk_groups, group_best,
               renormalize, scale, idx, weights)
    return idx, weights


def route_grad(grad_weights: torch.Tensor, logits: torch.Tensor,
               topk_idx: torch.Tensor, *, scoring: str = "softmax",
               renormalize: bool = True, scale: float = 1.0,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of route()'s logits, [T, E] in their dtype, from the gradient
    of its weights (float32) and the picks it returned. An index outside
    [0, E) adds nothing; one that occurs twice in a row adds twice. The picks
    themselves, and so the bias, have no gradient."""
    C = _native(grad_weights=grad_weights, logits=logits, out=out)
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype,
                          device=logits.device)
    C.ep_route_grad(grad_weights, logits, topk_idx, scoring, renormalize,
                    scale, out)
    return out


def expert_matmul(x: torch.Tensor, w: torch.Tensor,
                  counts: Optional[torch.Tensor] = None, *,
                  x_scales: Optional[torch.Tensor] = None,
                  w_scales: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None,
                  out_dtype: Optional[torch.dtype] = None,
                  expected_rows: Optional[int] = None,
                  precise: bool = False) -> torch.Tensor:
    """out[e, m] = x[e, m] @ w[e].T for the valid rows m of each expert e.

    x [E, slots, K], w [E, N, K], out [E, slots, N].

    8 bits: x and w float8_e4m3fn, K a multiple of 128, with x_scales
    [E, slots, K/128] (what dispatch and expert_swiglu give) and w_scales
    [E, ceil(N/128), K/128], both float32: a value of x stands for value *
    scale of its 128 columns, one of w for value * scale of its block of 128
    by 128. out is bfloat16 (default) or float16. Each block of 128 columns is
    summed by the 8-bit matrix unit, which drops what lies far below the
    block's largest product: a sum is off by up to 2^-13 of its terms'
    magnitudes (about 2^-16 on normal data). The blocks' sums are scaled and
    added in 32 bits. With ``precise`` all sums are held in 32 bits, and out
    may be float32, too; the product then takes 1.1 (one row) to 1.9 times
    (large ones) as long.

    16 bits: x and w bfloat16 or float16, K a multiple of 8; out has their
    dtype, or ``out_dtype`` (bfloat16, float16, float32); sums are held in 32
    bits. The gradient of the rows is this product with the weights transposed:
    ``expert_matmul(grad_out, w.transpose(1, 2), counts)``. The view is read
    as it lies (its N, the weights' K, a multiple of 8).

    ``expected_rows``: how many rows an expert is expected to have, by which
    the kernel is chosen. It changes the speed and the order of the sums, never
    which rows are computed. Without it all slots are expected, which suits
    full ones: 32 rows of 32 experts each, 4096 x 7168, take 238 us instead of
    175 in 8 bits, 420 instead of 322 in 16.
    """
    C = _native(x=x, w=w, x_scales=x_scales, w_scales=w_scales, out=out)
    if out is None:
        if out_dtype is None:
            out_dtype = x.dtype if x.element_size() == 2 else torch.bfloat16
        out = torch.empty(*x.shape[:-1], w.shape[-2], dtype=out_dtype,
                          device=x.device)
    elif out_dtype not in (None, out.dtype):
        raise RuntimeError(
            f"uccl_amd: out is {out.dtype}, out_dtype is {out_dtype}")
    C.ep_expert_matmul(_slots(x), _slots(w), _counts(counts, x),
                       _slots(x_scales), _slots(w_scales), _slots(out),
                       expected_rows or 0, precise)
    return out


def expert_weight_grad(grad_out: torch.Tensor, x: torch.Tensor,
                       counts: Optional[torch.Tensor] = None, *,
                       out: Optional[torch.Tensor] = None,
                       out_dtype: Optional[torch.dtype] = None
                       ) -> torch.Tensor:
    """out[e] = sum over the valid rows m of grad_out[e, m].T x[e, m]: the
    gradient of expert_matmul's weights, [E, N, K]. grad_out [E, slots, N] and
    x [E, slots, K] are bfloat16 or float16 with N and K multiples of 8; out
    has their dtype, or ``out_dtype`` (bfloat16, float16, float32). Sums are
    held in 32 bits and taken in a fixed order. An expert without
    valid rows gets zeros."""
    C = _native(grad_out=grad_out, x=x, out=out)
    if out is None:
        out = torch.empty(*x.shape[:-2], grad_out.shape[-1], x.shape[-1],
                          dtype=out_dtype or x.dtype, device=x.device)
    elif out_dtype not in (None, out.dtype):
        raise RuntimeError(
            f"uccl_amd: out is {out.dtype}, out_dtype is {out_dtype}")
    C.ep_expert_weight_grad(_slots(grad_out), _slots(x), _counts(counts, x),
                            _slots(out))
    return out


def expert_swiglu(h: torch.Tensor, counts: Optional[torch.Tensor] = None, *,
                  quantize: bool = False,
                  out: Optional[torch.Tensor] = None,
                  out_scales: Optional[torch.Tensor] = None):
    """silu(a) * b for the valid rows of h [E, slots, 2 * I] (bfloat16 or
    float16), a the first I columns and b the others; I a multiple of 8. A gate
    a of +inf gives +-inf, one of -inf NaN, as a * sigmoid(a) * b does.

    Returns [E, slots, I] in h's dtype. With ``quantize`` (I a multiple of
    128) returns (values float8_e4m3fn, scales float32 [E, slots, I/128]) for
    an 8-bit expert_matmul: scale = max |v| / 448 over each 128 columns, or 1
    where that is 0 as a float32; values the nearest to v / scale, ties to
    even, decided as if v were exact. A NaN stays NaN and does not count for
    its scale; an infinite v makes its scale infinite and itself NaN."""
    C = _native(h=h, out=out, out_scales=out_scales)
    cols = h.shape[-1] // 2
    if out is None:
        out = torch.empty(*h.shape[:-1], cols, device=h.device,
                          dtype=torch.float8_e4m3fn if quantize else h.dtype)
    if not quantize:
        if out_scales is not None:
            raise RuntimeError("uccl_amd: out_scales belongs to quantize=True")
        C.ep_expert_swiglu(_slots(h), _counts(counts, h), _slots(out), None)
        return out
    if out_scales is None:
        out_scales = torch.empty(*h.shape[:-1], cols // 128,
                                 dtype=torch.float32, device=h.device)
    C.ep_expert_swiglu(_slots(h), _counts(counts, h), _slots(out),
                       _slots(out_scales))
    return out, out_scales


def expert_swiglu_grad(grad_out: torch.Tensor, h: torch.Tensor,
                       counts: Optional[torch.Tensor] = None, *,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of expert_swiglu's h, [E, slots, 2 * I] in its dtype, from
    grad_out [E, slots, I] of the same dtype. At an infinite gate the first
    half's is NaN, as sigmoid(a) * (1 + a * (1 - sigmoid(a))) is."""
    C = _native(grad_out=grad_out, h=h, out=out)
    if out is None:
        out = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    C.ep_expert_swiglu_grad(_slots(grad_out), _slots(h), _counts(counts, h),
                            _slots(out))
    return out
