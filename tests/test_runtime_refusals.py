"""What the library says where the machine's runtime refuses something."""
import pytest

import conftest
from _launch import launch


def test_needs_name_tests_that_exist():
    """A test that is renamed takes its entry along: one without a test would
    skip nothing, silently."""
    import os
    src = "".join(open(os.path.join(conftest.ROOT, "tests", f)).read()
                  for f in ("test_group.py", "test_host_combine.py"))
    for name, need in conftest.RUNTIME_NEEDS.items():
        assert f"def {name}(" in src
        got = {need({"shareable": s, "kind": k}) for s in (0, 1) for k in ("plain", "torch")}
        assert got - {None} and all(g in conftest.REFUSED for g in got - {None})


@pytest.mark.gpu
def test_refused_peer_import_names_its_cause():
    """Where the runtime does not import a peer's descriptor, the refusal says
    what tells the causes apart: whether the descriptor arrived, the size of
    what is behind it, and how this process hands descriptors over."""
    if not conftest.runtime_answers().get("peer_import"):
        pytest.skip("the runtime here imports them")
    codes, outs = launch("_worker_ipc.py", 2, timeout=100, env_extra={"XUCG_IPC_SHAREABLE": "1"})
    assert codes == [1, 1]
    for out in outs:
        assert "import of the peer's descriptor (open, 2097152 bytes; descriptors are taken by " in out


@pytest.mark.gpu
def test_a_refused_call_is_reported_once(dev_ctx):
    """A HIP call that fails is the error of the call that made it, and not of
    the launches after it, which ask the runtime for the last error."""
    import numpy as np
    from xucg_amd import _lib
    host = np.zeros(1 << 16, np.uint8)               # was never registered
    x = dev_ctx.alloc(4096)
    x.upload(np.ones(1024, np.float32))
    counts, sums, loss = dev_ctx.alloc(72), dev_ctx.alloc(36), dev_ctx.alloc(12)
    for launch in (lambda: dev_ctx.reduce_checked("sum", "float32", x.ptr, x.ptr, 1024),
                   lambda: dev_ctx.balance("float32", x, x, 0, 8, 1, counts, sums),
                   lambda: dev_ctx.sum_dropout("float32", x, [x], 1, 1024, 0.0, 1),
                   lambda: dev_ctx.balance_loss(counts, sums, 8, 1, loss)):
        assert _lib.dev().ucg_builtin_dev_host_unregister(dev_ctx.handle, host.ctypes.data) != 0
        launch()
    dev_ctx.sync()
    assert (x.download(np.float32, 1024) == 2).all()
