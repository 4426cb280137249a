import os
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run on the B200 box)")


def _has_gpu() -> bool:
    try:
        import torch
        return torch.cuda.is_available()
    except Exception:
        return False


# Tests that hold a wrong value, and the proof: they run on, and are expected to fail.
_LOST_LOG = ("the oracle forms row - (top + log(sum)): beside a row of the lowest r32 or r64 value the sum's logarithm is lost, so that each of 500 equal "
             "tokens gets probability 1 (score -30) instead of 1/500 (-30 - ln 500 = -36.2); test_select_masked_and_impossible_rows has the right ones")
WRONG_VALUES = {f"test_state_ops_gpu.py::test_select_masked_and_impossible[{sfx}]": _LOST_LOG for sfx in ("r32", "r64")}


def pytest_collection_modifyitems(config, items):
    for item in items:
        reason = next((why for name, why in WRONG_VALUES.items() if item.nodeid.endswith(name)), None)
        if reason is not None:
            item.add_marker(pytest.mark.xfail(reason=reason, strict=True))
    if _has_gpu():
        return
    skip = pytest.mark.skip(reason="no CUDA device in this container")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(scope="module", autouse=True)
def refused_calls_see_no_device(request):
    """Tests of refusals call launchers with made-up addresses in processes of their own.  A refusal that went missing must end there, not on a GPU."""
    if not request.module.__name__.endswith("refusals"):
        yield
        return
    before = os.environ.get("CUDA_VISIBLE_DEVICES")
    os.environ["CUDA_VISIBLE_DEVICES"] = ""
    yield
    if before is None:
        del os.environ["CUDA_VISIBLE_DEVICES"]
    else:
        os.environ["CUDA_VISIBLE_DEVICES"] = before


@pytest.fixture(scope="session")
def mp():
    import metaphor_b200
    metaphor_b200.lib()  # raises if the CUDA library is not built: no fallback
    return metaphor_b200


@pytest.fixture(scope="session")
def stream(mp):
    import torch
    torch.cuda.init()
    torch.zeros(1, device="cuda")  # make the primary context current
    s = mp.Stream()
    yield s
    s.close()


@pytest.fixture(scope="session")
def orc():
    from oracle import pyoracle
    pyoracle.lib()
    return pyoracle
