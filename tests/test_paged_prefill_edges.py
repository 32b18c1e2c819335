"""Attention of packed new tokens over a paged INT8 cache: inputs at which single steps of the kernels can go wrong.

Inputs, oracle and tolerances are those of test_paged_prefill.py; where a test needs another bound it derives it."""
import ctypes

import numpy as np
import pytest

import kvdecode as kvd
from test_paged_prefill import DEV, TYPES, close, make_case, oracle, prefill, prefill_desc


def tokens(s, b=0):
    """(blocks, offsets) of request b's tokens, in their order."""
    import torch

    t = torch.arange(int(s["len"][b]), device=DEV)
    return s["table"][b].long()[t // s["bs"]], t % s["bs"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n,every", [("float32", 128, 1024), ("float16", 256, 8192), ("bfloat16", 256, 8192)])
@pytest.mark.parametrize("what", ["scores", "values"])
@pytest.mark.parametrize("times", [1, 2])
def test_references_that_move_where_sums_are_put_aside(dtype, n, every, what, times):
    # Sums in parts: a warpgroup puts its sums aside after some of its tiles, and starts again from zero. Here the
    # scores rise by 10 in base 2, or value scales by 2^10, at just those tiles (every so many tokens), so that sums are
    # put aside and scaled in the same step. What was put aside is 0.25 to 20 percent of what comes after it, and all
    # values are above zero: a sum that counts twice, or not at all, is off by more than the tolerance.
    import torch

    H = torch.cuda.get_device_properties(0).multi_processor_count  # a unit of work a CTA: rows are not split
    ln = times * every + 400
    s = make_case(1, [n], [ln], H, 1, 64, 64, dtype, seed=31)
    s["V"] = s["V"].abs()
    s["K"][..., 0] = 0
    blk, off = tokens(s)
    level = torch.arange(ln, device=DEV) // every
    if what == "scores":
        s["q"] *= 0.02
        s["q"][:, :, 0] = 8.0
        s["ks"].fill_(10 * np.log(2) / 60)  # 8 x 60 level ks / sqrt(64) = 10 ln 2 level
        s["K"][blk, :, off, 0] = (60 * level).to(torch.int8).unsqueeze(-1)
    else:
        s["vs"][blk, :, off] *= (2.0 ** (10 * level.float())).unsqueeze(-1)
    close(prefill(s, causal=False), s, oracle(s, causal=False))
    assert kvd.device_status() == 0
