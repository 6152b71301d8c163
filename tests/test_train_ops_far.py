"""The training-step operators where their kernels go further than a small case
takes them: members without work, loops past their first pass, in-place
gradients, many rows to a lane, values at the ends of their range. The oracle
and the arrays are test_train_ops.py's; every bound is counted from the
operations that a value goes through (u = 2^-24 for each in fp32)."""
import numpy as np
import pytest

import xucg_amd
from oracle import train_ref as R
from test_train_ops import DTS, U, Arr, gpu, ptr
from xucg_amd import group as G


# ---- members without work ------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("cols", [0, 5, 16385, 20000, 1 << 20, (1 << 31) - 1])
def test_policy_of_a_member_without_rows(dev_ctx, dt, cols):
    """No rows of any length: zeros, also where a row would be many parts; in a
    group, the member adds its zeros and takes part in the allreduce."""
    s, c = Arr(dev_ctx, np.ones(2, np.float32)), Arr(dev_ctx, np.ones(3, np.int64))
    loss, ws = Arr(dev_ctx, np.ones(3, np.float32)), dev_ctx.alloc(dev_ctx.policy_workspace(0, cols))
    for per_row in (False, True):
        for ref in (None, 1 << 20):           # never looked at
            dev_ctx.policy(dt, None, None, None, 0, cols, s.ptr, c.ptr, ref=ref, adv_per_row=per_row,
                           per_sequence=per_row, loss=loss.ptr, workspace=ws)
            dev_ctx.policy_grad(dt, None, None, None, None, 0, cols, c.ptr, ref=ref, adv_per_row=per_row)
            dev_ctx.sync()
            assert not s.get().any() and not c.get().any() and not loss.get().any()
            for a in (s, c, loss):
                a.buf.upload(a.whole)         # ones again
    other = {"float32": Arr(dev_ctx, np.array([6, 3], np.float32)), "int64": Arr(dev_ctx, np.array([4, 2, 1], np.int64))}
    joined = []

    def allreduce(buf, t, n):
        """the other member's share is added"""
        joined.append(t)
        assert dev_ctx.reduce("sum", t, buf, other[t].ptr, n) == 0
    G.group_policy(dev_ctx, allreduce, dt, None, None, None, 0, cols, s.ptr, c.ptr, loss.ptr, kl_coef=0.5,
                   workspace=ws)
    dev_ctx.sync()
    assert sorted(joined) == ["float32", "int64"]
    assert c.get().tolist() == [4, 2, 1] and loss.get().tolist() == [1.875, 1.5, 0.75]
