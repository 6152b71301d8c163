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
