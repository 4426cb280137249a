"""Plain 64-bit forms of the operators that go on from a kept state, sequence by sequence and step by step, and how far a result may be from them.

Tolerances: u is half a step of the accumulator (2^-24, r64: 2^-53), U half a step of the storage type.  Beside a value stands the sum of the
absolute values of its terms; a sum of n terms is off by at most n u times that."""
import numpy as np

from util import NP_OF

ACC = {"r16": np.float32, "r32": np.float32, "r64": np.float64}
U_ACC = {"r16": 2.0 ** -24, "r32": 2.0 ** -24, "r64": 2.0 ** -53}
U_OUT = {"r16": 2.0 ** -11, "r32": 2.0 ** -24, "r64": 2.0 ** -53}
TINY = {"r16": 2.0 ** -25, "r32": 2.0 ** -126, "r64": 0.0}      # half a step among the subnormal values, or what is flushed


def packed(r, lens, nslots, first=0, behind=3):
    """starts, slots, resume of sequences with these lengths, and the number of rows."""
    starts = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32) + np.int32(first)
    slots = r.permutation(nslots)[:len(lens)].astype(np.int32)
    resume = r.integers(0, 2, len(lens)).astype(np.int32)
    return starts, slots, resume, int(starts[-1]) + behind


def sequences(starts, slots, resume, nslots):
    for i in range(len(slots)):
        if 0 <= slots[i] < nslots:
            yield int(starts[i]), int(starts[i + 1]), int(slots[i]), bool(resume[i])


def conv(x, w, bias, states, starts, slots, resume, y):
    """(y, its tolerance without the output's rounding, states): y holds what rows of no sequence keep."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    b = np.zeros(w.shape[0]) if bias is None else bias.astype(np.float64)
    y, size, states = y.astype(np.float64).copy(), np.zeros(y.shape), states.copy()
    K = w.shape[1]
    for lo, hi, slot, go in sequences(starts, slots, resume, states.shape[0]):
        kept = states[slot] if go else np.zeros_like(states[slot])
        line = np.concatenate([kept.astype(np.float64), x[lo:hi]])
        pre, mag = np.tile(b, (hi - lo, 1)), np.tile(np.abs(b), (hi - lo, 1))
        for k in range(K):
            pre += w[:, k] * line[k:k + hi - lo]
            mag += np.abs(w[:, k] * line[k:k + hi - lo])
        y[lo:hi] = pre / (1 + np.exp(-pre))
        size[lo:hi] = mag
        states[slot] = line[hi - lo:].astype(states.dtype)
    return y, size, states


def conv_tolerance(sfx, y, size, K):
    # the sum of K + 1 terms in K + 1 roundings, through a derivative of at most 1.1; the sigmoid to 2^-21 (r16: exponential and reciprocal of the
    # special-function unit, the exponent's own rounding times |pre| e^-|pre| < 1) or to 8 u; the product and the output rounded
    u = U_ACC[sfx]
    sig = 2.0 ** -21 if sfx == "r16" else 8 * u
    return 1.1 * (K + 1) * u * size + (sig + u) * np.abs(y) + U_OUT[sfx] * np.abs(y) * 1.001 + TINY[sfx]


def scan(x, raw, dt_bias, A_log, B, C, states, starts, slots, resume, y, groups):
    """(y, the size of its terms, states, the size of theirs, the number of steps behind each); x: [rows, H, P], B, C: [rows, G, N]."""
    f = np.float64
    H = x.shape[1]
    heads_of = np.repeat(np.arange(groups), H // groups)
    dt = np.logaddexp(0, raw.astype(f) + dt_bias.astype(f))
    rate = np.exp(A_log.astype(f))
    out, states = y.astype(f).copy(), states.astype(f).copy()
    ysize, ssize = np.zeros(y.shape), np.zeros(states.shape)
    ysteps, ssteps = np.zeros(y.shape[0]), np.zeros(states.shape[0])
    for lo, hi, slot, go in sequences(starts, slots, resume, states.shape[0]):
        S = states[slot] if go else np.zeros_like(states[slot])
        M = np.abs(S)
        for t in range(lo, hi):
            a = np.exp(-dt[t] * rate)[:, None, None]
            new = dt[t][:, None, None] * x[t].astype(f)[:, :, None] * B[t].astype(f)[heads_of][:, None, :]
            S, M = a * S + new, a * M + np.abs(new)
            c = C[t].astype(f)[heads_of][:, None, :]
            out[t], ysize[t] = (S * c).sum(2), (M * np.abs(c)).sum(2)
            ysteps[t] = t - lo + 1
        states[slot], ssize[slot], ssteps[slot] = S, M, hi - lo
    return out, ysize, states, ssize, ysteps, ssteps


def scan_tolerance(sfx, ref, size, steps, N, out):
    """What a term has gone through: its step size to 8 u (exponential and logarithm to 2 steps each), its product with x and B to 2 u; per step a
    decay to 2 u and the product and sum with it, and the exponent's own 10 u times the exponent (e^-v v < 1 over all steps together: 10 u); chunks
    instead of steps, or two terms of 11 bits (2^-22 = 4 u) instead of a value, are no worse; then the sum over the N columns."""
    u = U_ACC[sfx]
    steps = steps.reshape(steps.shape + (1,) * (ref.ndim - steps.ndim))
    tol = (24 + 4 * steps + (N if out else 0)) * u * size
    return tol + (U_OUT[sfx] * 1.001 * np.abs(ref) + TINY[sfx] if out else TINY[sfx] if sfx != "r16" else 2.0 ** -126)


def select(logits, scores, finished, eos, picks):
    """(next_scores, parents, tokens, next_finished) of [batch, beams, vocab] logits, by sorting every candidate."""
    f = np.float64
    batch, beams, vocab = logits.shape
    res = []
    for b in range(batch):
        cand = []
        for i in range(beams):
            had, row = f(scores[b, i]), logits[b, i].astype(f)
            done = finished is not None and finished[b, i] != 0 and eos < vocab
            if np.isnan(had) or had == -np.inf:
                order, sc = np.arange(vocab), np.full(vocab, -np.inf)
            elif done:
                order = np.array([eos] + [v for v in range(vocab) if v != eos])
                sc = np.where(order == eos, had, -np.inf)
            else:
                with np.errstate(all="ignore"):
                    top = row.max()
                    lse = top + np.log(np.exp(row - top).sum())
                if np.isfinite(lse):
                    order = np.lexsort((np.arange(vocab), -row))
                    sc = had + (row[order] - lse)
                else:
                    order, sc = np.arange(vocab), np.full(vocab, -np.inf)
            for rank in range(min(picks, vocab)):
                cand.append((-sc[rank], i, rank, int(order[rank]), done))
        cand.sort(key=lambda c: c[:3])
        res.append([(-c[0], c[1], c[3], int((finished is not None and finished[b, c[1]] != 0) or c[3] == eos)) for c in cand[:picks]])
    pick = lambda k, t: np.array([[c[k] for c in r] for r in res], dtype=t)
    return pick(0, f), pick(1, np.int32), pick(2, np.int32), pick(3, np.int32)


def storage(r, shape, sfx, scale=1.0):
    return (r.standard_normal(shape) * scale).astype(NP_OF[sfx])
