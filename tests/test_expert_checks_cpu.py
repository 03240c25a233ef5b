"""Further refusals of the expert-layer operators, and calls that pass every
check: without a GPU those end with the refusal of operands that are not on
one."""

import pytest
import torch

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
