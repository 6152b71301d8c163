import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
# a timed-out engine wait prints the op's state and the stash (builtin_ops.c,
# timeout_dump) into the worker's output, which a failing test shows
os.environ.setdefault("UCX_BUILTIN_TIMEOUT_DUMP", "y")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs via gpurun)")
    config.addinivalue_line("markers", "slow: longer CPU test")


@pytest.fixture(scope="session")
def dev_ctx():
    """One device context for the whole GPU session (device 0)."""
    import xucg_amd
    ctx = xucg_amd.DevContext(device=0)
    yield ctx
    ctx.close()


@pytest.fixture
def in_child(request):
    """For GPU tests that initialise torch's device context: in the pytest
    process, run this test in a child pytest and return True (the caller then
    returns at once); in that child return False (run the body). torch's
    context held by the pytest process for the rest of the session slowed the
    multi-process device tests that follow it (stalls)."""
    import subprocess

    def run():
        if os.environ.get("XUCG_IN_CHILD") == request.node.nodeid:
            return False
        env = dict(os.environ, XUCG_IN_CHILD=request.node.nodeid)
        p = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider",
                            "-m", "gpu", request.node.nodeid], cwd=ROOT, env=env,
                           capture_output=True, text=True, timeout=300)
        assert p.returncode == 0 and " passed" in p.stdout, p.stdout[-3000:] + p.stderr[-2000:]
        return True
    return run


# ---- what a machine's runtime refuses ------------------------------------------------
# A GPU test that rests on something the runtime of some machines does not do
# at all is skipped there, with the runtime's answer as its reason, and runs
# everywhere else. The question is put to the runtime itself, past this
# library (_probe_runtime.py), so a fault of the library's never skips a test.
RUNTIME_NEEDS = {
    "test_oneshot_reduce_scatter_over_ipc": lambda p: "peer_import" if p["shareable"] else None,
    "test_ipc_keys_survive_free_and_reallocation": lambda p: "peer_import" if p["kind"] != "plain" else None,
    "test_stage_bench_c_harness_bit_exact": lambda p: "host_register",
}
REFUSED = {
    "peer_import": "the runtime here does not import a shareable allocation of another process "
                   "(hipMemImportFromShareableHandle: status %d)",
    "host_register": "the runtime here does not register host memory that already exists "
                     "(hipHostRegister: status %d)",
}
_answers = None


def runtime_answers():
    """{name: hip status} of _probe_runtime.py, asked once a session; {} where
    it could not be asked (the tests then run)"""
    global _answers
    if _answers is None:
        import json
        import subprocess
        p = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "_probe_runtime.py")],
                           capture_output=True, text=True, timeout=200)
        lines = [line for line in p.stdout.splitlines() if line.startswith("{")]
        _answers = json.loads(lines[-1]) if p.returncode == 0 and lines else {}
    return _answers


def pytest_runtest_setup(item):
    name = getattr(item, "originalname", item.name)
    if name in RUNTIME_NEEDS and item.get_closest_marker("gpu"):
        need = RUNTIME_NEEDS[name](item.callspec.params if hasattr(item, "callspec") else {})
        status = runtime_answers().get(need, 0) if need else 0
        if status:
            pytest.skip(REFUSED[need] % status)
