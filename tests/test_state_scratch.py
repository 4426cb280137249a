"""The scratch of a call suffices for every smaller one (no GPU needed): what the launchers lay out in it, restated here, against the sizes that the
library names for the largest call."""
import random

import pytest

SMS = 148
LANES = ((32, 8, 8), (64, 8, 16), (128, 8, 32), (256, 16, 32))      # state columns up to, least and most lanes of a row


def recurrence_need(key, nseq, rows, heads, headdim, dstate):
    held, size = (2, 8) if key == 2 else (4, 4)
    least, most = next((a, b) for n, a, b in LANES if dstate <= n)
    lanes = least
    while lanes < most and 2 * headdim <= held * (128 // lanes):
        lanes *= 2
    units = heads * -(-headdim // (held * (128 // lanes)))
    if nseq * units >= 8 * SMS or min(2 * rows // nseq, rows) <= 320:
        return 0
    want = 8 * SMS // units + 1
    steps = max(32, ((rows + want - 1) // want + 15) // 16 * 16)
    if steps >= rows:
        return 0
    return (rows // steps + nseq) * heads * (headdim * dstate + 1) * size


def chunks_need(nseq, rows, heads, headdim, dstate):
    units = heads * -(-headdim // 64)
    if dstate > 128 or nseq * units >= SMS:
        return 0
    want = 2 * SMS // units
    steps = max(256, ((rows + want - 1) // want + 127) // 128 * 128)
    if steps >= rows:
        return 0
    return (rows // steps + nseq) * units * (64 * 128 + 1) * 4


def select_need(key, rows, vocab):
    size, entry = ((2, 8), (4, 8), (8, 16))[key]
    most = -(-vocab * size // 4096)
    pieces = max(1, min(8 * SMS // rows, most))
    return rows * pieces * (16 + 32 * entry)


def between(r, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** r.random())))


@pytest.mark.parametrize("key", [0, 1, 2])
def test_prompt_scan(mp_cpu, key):
    r = random.Random(key)
    for _ in range(300):
        heads, headdim, dstate = between(r, 1, 64), between(r, 1, 256), between(r, 1, 256)
        nseq, rows = between(r, 1, 2000), between(r, 1, 100000)
        have = mp_cpu.mpSsdScanPromptScratchBytes(key, nseq, rows, heads, headdim, dstate, 1)
        for _ in range(40):
            n, m = between(r, 1, nseq), between(r, 1, rows)
            need = recurrence_need(key, n, m, heads, headdim, dstate)
            if key == 0:
                need = max(need, chunks_need(n, m, heads, headdim, dstate))
            assert need <= have, (nseq, rows, heads, headdim, dstate, n, m)
            assert mp_cpu.mpSsdScanPromptScratchBytes(key, n, m, heads, headdim, dstate, 1) <= have


def test_many_short_prompts_then_a_long_one(mp_cpu):
    """Sixty prompts of 300 steps need nothing; the same rows as one prompt are cut into ranges."""
    for key, need in ((0, chunks_need(1, 18000, 24, 64, 128)), (1, recurrence_need(1, 1, 18000, 24, 64, 128))):
        assert 0 < need <= mp_cpu.mpSsdScanPromptScratchBytes(key, 60, 18000, 24, 64, 128, 1)


@pytest.mark.parametrize("key", [0, 1, 2])
def test_selection(mp_cpu, key):
    r = random.Random(10 + key)
    assert select_need(key, 592, 50280) <= mp_cpu.mpBeamSelectScratchBytes(key, 150, 4, 50280, 4)
    for _ in range(300):
        batch, beams, vocab = between(r, 1, 2000), between(r, 1, 64), between(r, 1, 300000)
        have = mp_cpu.mpBeamSelectScratchBytes(key, batch, beams, vocab, 1)
        for _ in range(40):
            b, k, v = between(r, 1, batch), between(r, 1, beams), between(r, 1, vocab)
            assert select_need(key, b * k, v) <= have, (batch, beams, vocab, b, k, v)
            assert mp_cpu.mpBeamSelectScratchBytes(key, b, k, v, 1) <= have


@pytest.fixture(scope="module")
def mp_cpu():
    import metaphor_b200
    return metaphor_b200.lib()
