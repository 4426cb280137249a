"""Refusals of the operators that go on from a kept state, continued (test_state_refusals.py; no GPU needed)."""
import json
import subprocess
import sys

import pytest

from test_state_refusals import CHILD, ROOT, conv, reorder, scan, select


def test_no_device_is_seen():
    """The processes in which calls are refused have no GPU to fault on, should a refusal go missing."""
    code = "import os\nprint(repr(os.environ.get('CUDA_VISIBLE_DEVICES')))\nimport torch\nprint(torch.cuda.device_count())"
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert res.stdout.split() == ["''", "0"], res.stdout + res.stderr


# Sizes of 64 bits whose products wrap round to small ones, and rows p that fit 31 bits but not once they are rounded up to whole tiles.
WIDE = 1 << 33
CASES = [(conv(form, channels=1 << 62, xp=1 << 62, yp=1 << 62), "31 bits") for form in ("prompt", "token")]
for form in ("prompt", "token"):
    CASES += [(scan(form, heads=1 << 40, headdim=1 << 24, dstate=1, rp=1 << 40), "31 bits"),
              (scan(form, heads=1 << 40, headdim=1 << 24, dstate=1, groups=1 << 40, rp=1 << 40, bcp=1 << 40), "31 bits"),
              (scan(form, heads=WIDE, groups=WIDE, headdim=1 << 31, dstate=128, rp=WIDE, bcp=1 << 40), "31 bits"),
              (scan(form, heads=1, headdim=(1 << 31) - 8, dstate=1, xp=1 << 31, yp=1 << 31), "31 bits"),
              (scan(form, heads=1, headdim=(1 << 30) + 8, dstate=1, xp=1 << 31, yp=1 << 31, dtype="r32"), "31 bits")]
CASES += [(select(batch=1 << 63, beams=2), "too many"), (select(batch=1 << 62, beams=4), "too many"), (reorder(row=1 << 63), "too long"), (reorder(row=(1 << 63) + 8), "too long")]


@pytest.fixture(scope="module")
def answers():
    res = subprocess.run([sys.executable, "-c", CHILD], input=json.dumps([c for c, _ in CASES]), capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert res.returncode == 0, res.stderr
    return json.loads(res.stdout.rsplit("RESULT", 1)[1])


@pytest.mark.parametrize("k", range(len(CASES)), ids=[f"{k}-{c[0]}-{what}" for k, (c, what) in enumerate(CASES)])
def test_refused(answers, k):
    (call, what), (code, text) = CASES[k], answers[k]
    assert code == 1 and what in text and "went through" not in text, (call, code, text)
