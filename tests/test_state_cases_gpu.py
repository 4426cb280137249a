"""Sequences that go on from a kept state, continued (test_state_ops_gpu.py): values of one call that lie far apart."""
import numpy as np
import pytest

import state_ref as ref
from test_state_ops_gpu import chunked, select, within

pytestmark = pytest.mark.gpu
TYPES = ("r16", "r32", "r64")


# ---------------------------------------------------------------------------------------------------- selection
def log_probabilities(logits):
    """log softmax in 64 bits, the maximum taken off before the sum's logarithm: log(sum) beside a maximum of 1e38 would be lost."""
    z = logits.astype(np.float64) - logits.astype(np.float64).max(-1, keepdims=True)
    return z - np.log(np.exp(z).sum(-1, keepdims=True))


@pytest.mark.parametrize("sfx", TYPES)
@pytest.mark.parametrize("vocab", [40, 500, 4999])
def test_select_rows_of_the_lowest_value(mp, stream, sfx, vocab):
    """A beam whose tokens are all masked with the type's lowest value, or lie around any other large one, pays -log(vocab) for each."""
    r = np.random.default_rng(vocab)
    logits = ref.storage(r, (2, 4, vocab), sfx)
    info = np.finfo(logits.dtype)
    logits[0, 1], logits[0, 2] = info.min, info.max
    logits[1, 0], logits[1, 1] = info.min / 2, info.min
    logits[1, 2, 5:] = info.min
    scores = np.zeros((2, 4), ref.ACC[sfx])
    scores[0, 2], scores[1, 1] = -1, 0.5
    picks = 32
    got = select(mp, stream, sfx, logits, scores, None, vocab, picks)
    total = scores.astype(np.float64)[..., None] + log_probabilities(logits)
    for b in range(2):
        # within a beam by the logit, the lower token first; between beams by the score, the lower beam first
        ranked = [(-total[b, i, v], i, k, v) for i in range(4) for k, v in enumerate(np.lexsort((np.arange(vocab), -logits[b, i].astype(np.float64)))[:picks])]
        best = sorted(ranked)[:picks]
        want = -np.array([c[0] for c in best])
        assert [c[1] for c in best] == got[1][b].tolist() and [c[3] for c in best] == got[2][b].tolist()
        u = ref.U_ACC[sfx]      # the sum of exponentials as in check_select (test_state_ops_gpu.py), the result rounded
        assert np.all(np.abs(got[0][b] - want) <= 4 * u * (1 + np.log(vocab)) + u * (vocab / 32 + 8) + u * np.abs(want))


def plain_select(logits, scores, finished, eos, picks):
    """(next_scores, parents, tokens, next_finished) by sorting every candidate, the scores from `log_probabilities`."""
    batch, beams, vocab = logits.shape
    res = []
    for b in range(batch):
        cand = []
        for i in range(beams):
            had, order, sc = np.float64(scores[b, i]), np.arange(vocab), np.full(vocab, -np.inf)
            done = finished is not None and finished[b, i] != 0
            if had > -np.inf and done:
                order, sc[0] = np.array([eos] + [v for v in range(vocab) if v != eos]), had
            elif had > -np.inf:
                with np.errstate(all="ignore"):
                    logp = log_probabilities(logits[b, i])
                if not np.isnan(logp).any():      # a NaN or plus infinity, or nothing above minus infinity
                    order = np.lexsort((np.arange(vocab), -logits[b, i].astype(np.float64)))
                    sc = had + logp[order]
            cand += [(-sc[k], i, k, int(order[k])) for k in range(picks)]
        cand.sort(key=lambda c: c[:3])
        res.append([(-c[0], c[1], c[3], int((finished is not None and finished[b, c[1]] != 0) or c[3] == eos)) for c in cand[:picks]])
    return [np.array([[c[k] for c in r] for r in res]) for k in range(4)]


@pytest.mark.parametrize("sfx", TYPES)
def test_select_masked_and_impossible_rows(mp, stream, sfx):
    """The calls of test_select_masked_and_impossible (test_state_ops_gpu.py) against log probabilities that keep the sum's logarithm."""
    r = np.random.default_rng(4)
    vocab, picks = 500, 9
    logits = ref.storage(r, (1, 8, vocab), sfx)
    low = np.finfo(logits.dtype).min
    logits[0, 0, 3:] = -np.inf
    logits[0, 1, 7], logits[0, 2, 9], logits[0, 3] = np.nan, np.inf, -np.inf
    logits[0, 4, 2:], logits[0, 5] = low, low
    scores = np.array([[-1, 0, 0, 0, -2, -30, 0, 0]], ref.ACC[sfx])
    scores[0, 6], scores[0, 7] = np.nan, -np.inf
    dead, lowest = scores.copy(), np.full((1, 8), np.finfo(ref.ACC[sfx]).min, ref.ACC[sfx])
    dead[0, :6] = -np.inf
    for had, finished, eos in ((scores, None, vocab), (dead, None, vocab), (scores, np.ones((1, 8), np.int32), 11), (lowest, None, vocab)):
        if had is lowest and sfx == "r16":
            continue      # (its logits do not vanish beside scores in r32)
        got, want = select(mp, stream, sfx, logits, had, finished, eos, picks), plain_select(logits, had, finished, eos, picks)
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2]), (got[1:3], want[1:3])
        assert finished is None or np.array_equal(got[3], want[3])
        u = ref.U_ACC[sfx]
        with np.errstate(invalid="ignore"):
            off = np.abs(got[0].astype(np.float64) - want[0]) <= 4 * u * (1 + np.log(vocab)) + u * (vocab / 32 + 8) + u * np.abs(want[0])
        assert (off | (got[0] == want[0])).all(), (got[0], want[0])


# ---------------------------------------------------------------------------------------------------- scan
def check_finite_part(s, got, starts, slots, resume):
    """Scan.check for results beyond r16's largest value too: that value stands for what lies beyond it, infinities included, on both sides (a
    difference does not grow when both sides are cut off at the same place)."""
    H, P, N, G = s.dims
    most = float(np.finfo(np.float16).max)
    (y, states), (wy, ysize, ws, ssize, ysteps, ssteps) = got, s.want(starts, slots, resume)
    y = y[:, :s.inner].reshape(-1, H, P)[starts[0]:starts[-1]].astype(np.float64)
    assert not np.isnan(y).any()
    tol = ref.scan_tolerance("r16", wy, ysize, ysteps, N, True)[starts[0]:starts[-1]]
    within(np.clip(y, -most, most), np.clip(wy[starts[0]:starts[-1]], -most, most), tol, "y")
    within(states[slots], ws[slots], ref.scan_tolerance("r16", ws, ssize, ssteps, N, False)[slots], "states")


@pytest.mark.parametrize("lens", [[2], [200, 90], [900, 5]])
@pytest.mark.parametrize("shape", [(2, 64, 128, 1), (1, 80, 64, 1)])
@pytest.mark.parametrize("what", ["x", "states", "C", "sizes", "late", "huge"])
def test_chunks_of_values_far_apart(mp, stream, lens, shape, what):
    """Values of one tile that lie up to 2^40 apart: each row p of a head, and each step's y, has the accuracy that it would have alone."""
    r = np.random.default_rng(sum(lens) + sum(shape))
    s, starts, slots, resume = chunked(r, lens, shape)
    resume[:] = 1
    H, P, N, G = shape
    falling = 2.0 ** -np.round(np.linspace(0, 36, P))            # over the rows p of a head
    rows = s.xbc.shape[0]
    if what == "x":
        x = s.xbc[:, :s.inner].astype(np.float64).reshape(rows, H, P) * falling * 2.0 ** 13
        s.xbc[:, :s.inner] = x.reshape(rows, -1).astype(np.float16)
        s.states *= (falling * 2.0 ** 13)[None, None, :, None].astype(np.float32)
    elif what == "states":
        s.states *= (falling * 2.0 ** 40)[None, None, :, None].astype(np.float32)
    elif what == "C":
        c = s.xbc[:, s.inner + s.bc:].astype(np.float64) * 2.0 ** (10 - np.arange(rows)[:, None] % 24)
        s.xbc[:, s.inner + s.bc:] = c.astype(np.float16)
    elif what == "sizes":
        s.zx[:, 3:] = r.uniform(-14, 8, s.zx[:, 3:].shape).astype(np.float16)
    elif what == "huge":      # one row of the state beside scores of next to nothing
        s.xbc[:, s.inner:] = (s.xbc[:, s.inner:].astype(np.float64) * 2.0 ** -12).astype(np.float16)
        s.states[:, :, 1:] = 0
        s.states *= np.float32(2.0 ** 110)
    else:      # nothing new in a sequence's last thirty steps, of which each leaves a fifth
        s.zx[:, 3:], s.dt_bias[:], s.A_log[:] = 0, np.log(np.expm1(0.1)), np.log(16)
        for lo, hi in zip(starts[:-1], starts[1:]):
            s.xbc[max(lo, hi - 30):hi, :s.inner] = 0
    check_finite_part(s, s.go(mp, stream, slots, resume, starts), starts, slots, resume)
