"""Calls of the operators that go on from a kept state which the host refuses before anything is launched (no GPU needed): each in a forked
process of one that has the library loaded, with addresses that are only looked at."""
import json
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
P = 1 << 20


def conv(form, channels=64, width=4, xp=64, yp=64, rows=10):
    if form == "prompt":     # x, pitch, w, bias, states, slots, resume, starts, y, pitch, nseq, rows, nslots, channels, width
        return "causal_conv1d_silu_prompt", "r16", (P, xp, P, P, P, P, P, P, P, yp, 2, rows, 3, channels, width)
    return "causal_conv1d_silu_token", "r16", (P, xp, P, P, P, P, P, yp, rows, 3, channels, width)


def scan(form, heads=4, headdim=64, dstate=128, groups=1, xp=256, rp=4, bcp=128, yp=256, rows=10, scratch=P, dtype="r16"):
    ins = (P, xp, P, rp, P, P, P, P, bcp, P, P)
    if form == "prompt":
        return "ssd_scan_prompt", dtype, (*ins, P, P, P, yp, scratch, 2, rows, 3, heads, headdim, dstate, groups)
    return "ssd_scan_token", dtype, (*ins, P, yp, rows, 3, heads, headdim, dstate, groups)


def select(batch=2, beams=4, vocab=100, picks=4, pitch=None, scratch=P):
    return "beam_select", "r16", (P, vocab if pitch is None else pitch, P, 0, 200, P, P, P, 0, scratch, batch, beams, vocab, picks)


def reorder(beams=4, batch=1, row=8):
    return "reorder_states", "r16", (P, 0, P, 2, batch, beams, batch * beams, row)


CASES = []
for form in ("prompt", "token"):
    CASES += [(conv(form, **a), what) for a, what in (
        (dict(width=1), "width 1"), (dict(width=5), "width 5"), (dict(xp=63), "pitch"), (dict(yp=63), "pitch"), (dict(rows=1 << 31), "31 bits"))]
    CASES += [(scan(form, **a), what) for a, what in (
        (dict(groups=3), "divisible"), (dict(groups=0), "divisible"), (dict(xp=255), "pitch"), (dict(rp=3), "pitch"), (dict(bcp=127), "pitch"), (dict(yp=255), "pitch"),
        (dict(rows=1 << 31), "31 bits"), (dict(dstate=0), "state"))]
for dtype in ("r16", "r32"):
    CASES += [(scan("prompt", dstate=257, bcp=257, dtype=dtype), "state size 257"), (scan("prompt", scratch=P + 8, dtype=dtype), "16-byte aligned")]
CASES += [(scan("token", heads=1, headdim=1, dstate=(1 << 30) + 1, bcp=(1 << 30) + 1), "31 bits")]
CASES += [(select(**a), what) for a, what in (
    (dict(beams=0), "0 beams"), (dict(beams=65), "65 beams"), (dict(picks=0), "0 picks"), (dict(picks=33), "33 picks"), (dict(vocab=5, picks=6), "6 picks"),
    (dict(pitch=99), "pitch 99"), (dict(scratch=0), "must not be NULL"), (dict(scratch=P + 4), "8-byte"), (dict(vocab=1 << 31), "vocabulary"), (dict(batch=1 << 31), "too many"))]
CASES += [(reorder(**a), what) for a, what in ((dict(beams=65), "65 beams"), (dict(batch=65536), "16 bits"), (dict(row=1 << 40), "too long"))]

CHILD = """
import json, os, sys, torch, metaphor_b200 as mp
mp.lib()
types = dict(r16=torch.float16, r32=torch.float32)
out = []
for name, dtype, args in json.loads(sys.stdin.read()):
    r, w = os.pipe()
    pid = os.fork()
    if pid == 0:
        os.dup2(w, 1); os.dup2(w, 2); os.close(r)
        mp.launch(name, types[dtype], *args, mp.StreamContext())
        os.write(1, b"went through")
        os._exit(0)
    os.close(w)
    text = b""
    while piece := os.read(r, 4096):
        text += piece
    os.close(r)
    out.append((os.waitstatus_to_exitcode(os.waitpid(pid, 0)[1]), text.decode()))
print("RESULT" + json.dumps(out))
"""


@pytest.fixture(scope="module")
def answers():
    res = subprocess.run([sys.executable, "-c", CHILD], input=json.dumps([c for c, _ in CASES]), capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert res.returncode == 0, res.stderr
    return json.loads(res.stdout.rsplit("RESULT", 1)[1])


@pytest.mark.parametrize("k", range(len(CASES)), ids=[f"{c[0]}-{what}" for c, what in CASES])
def test_refused(answers, k):
    (call, what), (code, text) = CASES[k], answers[k]
    assert code == 1 and what in text and "went through" not in text, (call, code, text)
