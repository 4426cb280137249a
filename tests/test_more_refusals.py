"""Refusals of the operators that go on from a kept state, continued (test_state_refusals.py; no GPU needed)."""
import subprocess
import sys


def test_no_device_is_seen():
    """The processes in which calls are refused have no GPU to fault on, should a refusal go missing."""
    code = "import os\nprint(repr(os.environ.get('CUDA_VISIBLE_DEVICES')))\nimport torch\nprint(torch.cuda.device_count())"
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert res.stdout.split() == ["''", "0"], res.stdout + res.stderr
