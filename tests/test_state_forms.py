"""The forms that the launchers take for large calls of the operators that go on from a kept state: several rounds of loads, several turns, ranges
behind ranges.  `test_forms` restates the rules (no GPU needed): the sizes below reach them, on 148 SMs."""
import numpy as np
import pytest

import state_ref as ref
from test_state_ops_gpu import Scan, chunked, check_select, select, within
from util import dev, host, run, torch_dtype

SMS, TYPES = 148, ("r16", "r32", "r64")
SIZE = {"r16": 2, "r32": 4, "r64": 8}

# rows, channels, width, offset (elements)
CONV = [(8000, 1792, 4, 0), (5000, 515, 3, 1), (17_000_000, 1, 2, 0)]
# rows, heads, headdim, dstate
TOKENS = [(110, 24, 64, 128), (90, 24, 80, 77)]
# layers, batch, beams, row (16-byte words and some more elements)
REORDER = [(3, 2, 4, 140_001 * 16), (2, 2, 5, 1_600_003 * 16)]
# batch, beams, vocab, picks
SELECT = [(75, 4, 50280, 9), (150, 2, 20011, 32)]
# lens, heads, headdim, dstate
RECURRENCE = [([1500, 3], 12, 64, 128), ([1400], 12, 64, 50), ([120] * 13, 24, 64, 128)]
# lens, heads
RANGES = [([5000], 2), ([40, 2600], 1)]


def conv_run(sfx, rows, channels, aligned):
    v = min(4, 16 // SIZE[sfx]) if aligned else 1
    cols = -(-channels // (32 * v))
    run_ = min(64, max(4, -(-rows * cols // (28 * SMS))))
    while -(-rows // (run_ * 4)) > 65535:
        run_ *= 2
    return run_


def token_batches(sfx, rows, heads, headdim, dstate):
    size = 8 if sfx == "r64" else 4
    v = 16 // size if dstate % (16 // size) == 0 else 1
    width = 1
    while width < 32 and width * v < dstate:
        width *= 2
    at_once = 8 * (32 // width)
    turns = -(-headdim // at_once)
    return 2 if turns > 1 and rows * heads * ((turns + 1) // 2) >= 16 * SMS else 1


def reorder_turns(layers, batch, beams, row_bytes):
    words, threads = row_bytes // 16, 128
    while threads > 16 and 2 * threads * beams * 16 > 46 * 1024:
        threads //= 2
    return min(8, max(1, words * layers * batch // (threads * 20 * SMS))), words % threads


def packs_of_a_thread(sfx, rows, vocab):
    pieces = max(1, min(8 * SMS // rows, -(-vocab * SIZE[sfx] // 4096)))
    return vocab * SIZE[sfx] // 16 / pieces / 128


def recurrence_lanes(sfx, nseq, rows, heads, headdim, least, most):
    held, lanes, ids = 2 if sfx == "r64" else 4, least, nseq
    splits = lambda: -(-headdim // (held * (128 // lanes)))
    while lanes < most and 2 * headdim <= held * (128 // lanes):
        lanes *= 2
    units = heads * splits()
    if nseq * units < 8 * SMS and min(2 * rows // nseq, rows) > 320:
        want = 8 * SMS // units + 1
        steps = max(32, (-(-rows // want) + 15) // 16 * 16)
        if steps < rows:
            ids = rows // steps + nseq
    while lanes < most and ids * heads * splits() < 2 * SMS:
        lanes *= 2
    return lanes, ids


def test_forms():
    for sfx in TYPES:
        assert conv_run(sfx, *CONV[0][:2], True) > 2 * 8 and conv_run(sfx, *CONV[1][:2], False) > 8, "runs of several rounds of eight rows"
        assert conv_run(sfx, *CONV[2][:2], False) > 64, "runs that the grid's second dimension makes longer"
        assert all(token_batches(sfx, *c) == 2 for c in TOKENS), "two batches of rows a warp"
        for c in SELECT:
            assert packs_of_a_thread(sfx, c[0] * c[1], c[2]) > (8 if sfx != "r16" or c[2] > 40000 else 4), "more packs than are loaded at once"
        for lens, heads, headdim, dstate in RECURRENCE:
            lanes, ids = recurrence_lanes(sfx, len(lens), sum(lens) + 3, heads, headdim, 8, 32 if dstate > 64 else 16)
            assert lanes == 8 and (len(lens) > 12 or ids > 4 * 4), "eight lanes of a row; more ranges than are carried at once"
    for c, turns in zip(REORDER, (2, 8)):
        got, rest = reorder_turns(*c[:3], c[3])
        assert got == turns and rest != 0, "several turns, the last one not whole"
    for lens, heads in RANGES:
        want = 2 * SMS // heads
        steps = max(256, (-(-(sum(lens) + 3) // want) + 127) // 128 * 128)
        assert max(lens) // steps > 8, "more ranges than are carried at once"


@pytest.mark.gpu
@pytest.mark.parametrize("sfx", TYPES)
@pytest.mark.parametrize("rows,channels,width,off", CONV)
def test_conv_prompt(mp, stream, sfx, rows, channels, width, off):
    r = np.random.default_rng(rows)
    if channels == 1:
        lens = [rows - 500, 0, 497]
    else:
        lens = [int(n) for n in r.multinomial(rows - 3, r.dirichlet(np.ones(9)))] + [0, 2]
    rows = sum(lens) + 3
    starts, slots, resume, rows = ref.packed(r, lens, len(lens) + 1)
    x, y0 = ref.storage(r, (rows, channels + off), sfx, 2.0), ref.storage(r, (rows, channels), sfx)
    w, b = ref.storage(r, (channels, width), sfx, 0.6), ref.storage(r, (channels,), sfx, 0.3)
    states = ref.storage(r, (len(lens) + 1, width - 1, channels), sfx)
    want, size, kept = ref.conv(x[:, off:], w, b, states, starts, slots, resume, y0)
    dx, dst, dy = dev(x), dev(states), dev(y0)
    run(mp, stream, "causal_conv1d_silu_prompt", sfx, dx.data_ptr() + off * dx.element_size(), channels + off, dev(w), dev(b), dst, dev(slots), dev(resume), dev(starts),
        dy, channels, len(lens), rows, len(lens) + 1, channels, width)
    got, last = host(dy), starts[-1]
    within(got[:last], want[:last], ref.conv_tolerance(sfx, want, size, width)[:last], "y")
    assert np.array_equal(got[last:], y0[last:]) and np.array_equal(host(dst), kept)


@pytest.mark.gpu
@pytest.mark.parametrize("sfx", TYPES)
@pytest.mark.parametrize("n,heads,headdim,dstate", TOKENS)
def test_scan_token(mp, stream, sfx, n, heads, headdim, dstate):
    r = np.random.default_rng(n)
    slots = r.permutation(n + 2)[:n].astype(np.int32)
    slots[7] = -1
    s = Scan(r, sfx, n, n + 2, heads, headdim, dstate, 2)
    s.check(s.go(mp, stream, slots), np.arange(n + 1), slots, np.ones(n))


@pytest.mark.gpu
@pytest.mark.parametrize("layers,batch,beams,row", REORDER)
def test_reorder(mp, stream, layers, batch, beams, row):
    """Whole numbers under a floating point type: every bit is compared."""
    import torch
    r = np.random.default_rng(beams)
    n = batch * beams
    states = torch.randint(-2 ** 31, 2 ** 31 - 1, (layers, n, row // 4), dtype=torch.int32, device="cuda", generator=torch.Generator("cuda").manual_seed(beams))
    slots, parents = torch.from_numpy(r.permutation(n).astype(np.int32)).cuda(), torch.from_numpy(r.integers(0, beams, (batch, beams)).astype(np.int32)).cuda()
    parents[0] = torch.arange(beams, device="cuda").roll(1)
    at = slots.long().reshape(batch, beams)
    want = states.clone()
    want[:, at.reshape(-1)] = states[:, at.gather(1, parents.long()).reshape(-1)]
    run(mp, stream, "reorder_states", "r32", states, slots, parents, layers, batch, beams, n, row // 4)
    assert torch.equal(states, want)


@pytest.mark.gpu
@pytest.mark.parametrize("sfx", TYPES)
@pytest.mark.parametrize("batch,beams,vocab,picks", SELECT)
@pytest.mark.parametrize("what", ["plain", "one thread", "few values"])
def test_select(mp, stream, sfx, batch, beams, vocab, picks, what):
    """`one thread`: the best tokens of a row lie where one thread looks, more of them than it remembers packs; `few values`: more equal ones than the
    list holds."""
    r = np.random.default_rng(vocab)
    shape = (batch, beams, vocab)
    logits = ref.storage(r, shape, sfx, 2.0)
    pack = 16 // SIZE[sfx]
    if what == "one thread":
        at = np.arange(vocab) // pack % 128 == 5
        logits[..., at] = (logits[..., at] + np.float64(9)).astype(logits.dtype)
    elif what == "few values":
        logits = r.integers(0, 3, shape).astype(logits.dtype)
    scores = r.uniform(-20, 0, (batch, beams)).astype(ref.ACC[sfx])
    finished = (r.random((batch, beams)) < 0.75).astype(np.int32)
    args = (logits, scores, finished, vocab // 2, picks)
    check_select(select(mp, stream, sfx, *args), *args, sfx)


@pytest.mark.gpu
@pytest.mark.parametrize("sfx", TYPES)
@pytest.mark.parametrize("lens,heads,headdim,dstate", RECURRENCE)
def test_recurrence(mp, stream, sfx, lens, heads, headdim, dstate):
    """(r16: rows off the 16-byte boundary, which the chunks do not take)"""
    r = np.random.default_rng(sum(lens))
    starts, slots, resume, rows = ref.packed(r, lens, len(lens))
    resume[0] = 1
    s = Scan(r, sfx, rows, len(lens), heads, headdim, dstate, 1, off=1 if sfx == "r16" else 0)
    s.check(s.go(mp, stream, slots, resume, starts), starts, slots, resume)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,heads", RANGES)
def test_chunks_in_many_ranges(mp, stream, lens, heads):
    r = np.random.default_rng(sum(lens))
    s, starts, slots, resume = chunked(r, lens, (heads, 64, 128, 1))
    resume[:] = 1
    s.check(s.go(mp, stream, slots, resume, starts), starts, slots, resume)
