"""Sequences that go on from a kept state: convolution and scan over packed prompts and single tokens, selection of a beam search, states that
follow the beams.  Every result against the plain forms in 64 bits (state_ref.py), element by element."""
import ctypes as C

import numpy as np
import pytest

import state_ref as ref
from util import NP_OF, dev, host, run, torch_dtype

pytestmark = pytest.mark.gpu
TYPES = ("r16", "r32", "r64")


def within(got, want, tol, what):
    g = np.asarray(got, dtype=np.float64)
    assert g.shape == want.shape, (what, g.shape, want.shape)
    bad = ~(np.abs(g - want) <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} outside, worst {np.max((np.abs(g - want) / np.maximum(tol, 1e-300))[bad]):.3g} times the tolerance"


# ---------------------------------------------------------------------------------------------------- convolution
LENGTHS = {"one": [1], "short": [2, 0, 3, 1], "mixed": [37, 0, 1, 2, 3, 4, 65, 16, 0, 129, 5], "many": [3] * 40 + [0] * 5 + [1, 17] * 15}


@pytest.mark.parametrize("sfx", TYPES)
@pytest.mark.parametrize("lens", list(LENGTHS))
@pytest.mark.parametrize("channels,width,pad,off", [(64, 4, 0, 0), (40, 3, 8, 0), (33, 2, 5, 0), (64, 4, 7, 1)])
def test_conv_prompt(mp, stream, sfx, lens, channels, width, pad, off):
    r = np.random.default_rng(len(lens) * channels + width)
    lens = LENGTHS[lens]
    nslots = len(lens) + 3
    starts, slots, resume, rows = ref.packed(r, lens, nslots, first=2)
    if len(lens) > 3:
        slots[1], slots[3] = -1, nslots        # nobody's
    x = ref.storage(r, (rows, channels + pad), sfx, 2.0)
    w, b = ref.storage(r, (channels, width), sfx, 0.6), ref.storage(r, (channels,), sfx, 0.3)
    bias = None if width == 3 else b
    states, y0 = ref.storage(r, (nslots, width - 1, channels), sfx), ref.storage(r, (rows, channels), sfx)
    want, size, kept = ref.conv(x[:, off:off + channels], w, bias, states, starts, slots, resume, y0)
    dx, dst, dy = dev(x), dev(states), dev(y0)
    run(mp, stream, "causal_conv1d_silu_prompt", sfx, dx.data_ptr() + off * dx.element_size(), channels + pad, dev(w), None if bias is None else dev(bias), dst,
        dev(slots), dev(resume), dev(starts), dy, channels, len(lens), rows, nslots, channels, width)
    tol = ref.conv_tolerance(sfx, want, size, width)
    mine = np.zeros(rows, bool)
    for lo, hi, _, _ in ref.sequences(starts, slots, resume, nslots):
        mine[lo:hi] = True
    assert np.array_equal(host(dy)[~mine], y0[~mine])
    within(host(dy)[mine], want[mine], tol[mine], "y")
    assert np.array_equal(host(dst), kept)


@pytest.mark.parametrize("sfx", TYPES)
@pytest.mark.parametrize("n,channels,width,pad,off", [(1, 64, 4, 0, 0), (70, 256, 4, 8, 0), (5, 33, 2, 0, 0), (9, 48, 3, 3, 1)])
def test_conv_token(mp, stream, sfx, n, channels, width, pad, off):
    r = np.random.default_rng(n + channels)
    nslots = n + 2
    slots = r.permutation(nslots)[:n].astype(np.int32)
    if n > 4:
        slots[2], slots[4] = -7, nslots
    x = ref.storage(r, (n, channels + pad), sfx, 2.0)
    w, b, states = ref.storage(r, (channels, width), sfx, 0.6), ref.storage(r, (channels,), sfx, 0.3), ref.storage(r, (nslots, width - 1, channels), sfx)
    xin = x[:, off:off + channels]
    want, size, kept = ref.conv(xin, w, b, states, np.arange(n + 1), slots, np.ones(n), xin)
    dx, dst = dev(x), dev(states)
    at = dx.data_ptr() + off * dx.element_size()
    run(mp, stream, "causal_conv1d_silu_token", sfx, at, channels + pad, dev(w), dev(b), dst, dev(slots), at, channels + pad, n, nslots, channels, width)   # in place
    got = host(dx)
    live = (slots >= 0) & (slots < nslots)
    within(got[live, off:off + channels], want[live], ref.conv_tolerance(sfx, want, size, width)[live], "y")
    assert np.array_equal(got[~live], x[~live]) and np.array_equal(got[:, :off], x[:, :off]) and np.array_equal(got[:, off + channels:], x[:, off + channels:])
    assert np.array_equal(host(dst), kept)


# ---------------------------------------------------------------------------------------------------- scan
class Scan:
    """One call's operands: x | B | C in the rows of one buffer, raw step sizes in those of another, columns in front of each."""

    def __init__(self, r, sfx, rows, nslots, heads, headdim, dstate, groups, off=0, strong=False, behind=1):
        self.sfx, self.dims, self.off, self.nslots = sfx, (heads, headdim, dstate, groups), off, nslots
        inner, bc = heads * headdim, groups * dstate
        self.inner, self.bc = inner, bc
        self.xbc = ref.storage(r, (rows, off + inner + 2 * bc), sfx)
        self.zx = ref.storage(r, (rows, 3 + heads), sfx)
        step = np.exp(r.uniform(np.log(1e-3), np.log(1e-1), heads)) if not strong else r.uniform(0.5, 40.0, heads)
        self.dt_bias = np.log(np.expm1(step)).astype(ref.ACC[sfx])
        self.A_log = np.log(r.uniform(1, 16, heads)).astype(ref.ACC[sfx])
        self.states = r.standard_normal((nslots, heads, headdim, dstate)).astype(ref.ACC[sfx])
        self.y0 = ref.storage(r, (rows, inner + behind), sfx)

    def want(self, starts, slots, resume):
        H, P, N, G = self.dims
        o, i, b = self.off, self.inner, self.bc
        rows = self.xbc.shape[0]
        return ref.scan(self.xbc[:, o:o + i].reshape(rows, H, P), self.zx[:, 3:], self.dt_bias, self.A_log, self.xbc[:, o + i:o + i + b].reshape(rows, G, N),
                        self.xbc[:, o + i + b:].reshape(rows, G, N), self.states, starts, slots, resume, self.y0[:, :i].reshape(rows, H, P), G)

    def go(self, mp, stream, slots, resume=None, starts=None, scratch=True):
        import torch
        H, P, N, G = self.dims
        self.d = {k: dev(getattr(self, k)) for k in ("xbc", "zx", "dt_bias", "A_log", "states", "y0")}
        d, size = self.d, np.dtype(NP_OF[self.sfx]).itemsize
        x = d["xbc"].data_ptr() + self.off * size
        ins = (x, self.xbc.shape[1], d["zx"].data_ptr() + 3 * size, self.zx.shape[1], d["dt_bias"], d["A_log"], x + self.inner * size,
               x + (self.inner + self.bc) * size, self.xbc.shape[1], d["states"], dev(slots) if slots is not None else None)
        rows = self.xbc.shape[0]
        if starts is None:
            run(mp, stream, "ssd_scan_token", self.sfx, *ins, d["y0"], self.y0.shape[1], rows, self.nslots, *self.dims)
        else:
            n = len(starts) - 1
            nbytes = mp.lib().mpSsdScanPromptScratchBytes(TYPES.index(self.sfx), n, rows, *self.dims)
            self.scratch = torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda")      # NaN wherever something is read before it is written
            run(mp, stream, "ssd_scan_prompt", self.sfx, *ins, dev(resume) if resume is not None else None, dev(starts), d["y0"], self.y0.shape[1],
                self.scratch if scratch else None, n, rows, self.nslots, *self.dims)
        return host(d["y0"]), host(d["states"])

    def check(self, got, starts, slots, resume):
        H, P, N, G = self.dims
        (y, states), (wy, ysize, ws, ssize, ysteps, ssteps) = got, self.want(starts, slots, resume)
        rows = y.shape[0]
        mine, used = np.zeros(rows, bool), np.zeros(self.nslots, bool)
        for lo, hi, slot, _ in ref.sequences(starts, slots, resume, self.nslots):
            mine[lo:hi], used[slot] = True, True
        assert np.array_equal(y[~mine], self.y0[~mine]) and np.array_equal(y[:, self.inner:], self.y0[:, self.inner:]), "rows of no sequence, or columns behind"
        assert np.array_equal(states[~used], self.states[~used]), "states of no sequence"
        y = y[:, :self.inner].reshape(rows, H, P)
        within(y[mine], wy[mine], ref.scan_tolerance(self.sfx, wy, ysize, ysteps, N, True)[mine], "y")
        within(states[used], ws[used], ref.scan_tolerance(self.sfx, ws, ssize, ssteps, N, False)[used], "states")


SCAN_SHAPES = [(2, 64, 128, 1), (4, 64, 128, 2), (3, 33, 77, 1), (2, 16, 16, 2), (1, 80, 64, 1), (2, 128, 256, 1), (1, 1, 1, 1), (6, 32, 96, 3)]


@pytest.mark.parametrize("sfx", TYPES)
@pytest.mark.parametrize("lens", ["one", "short", "mixed"])
@pytest.mark.parametrize("shape", SCAN_SHAPES)
def test_scan_prompt(mp, stream, sfx, lens, shape):
    r = np.random.default_rng(sum(shape) + len(lens))
    lens = LENGTHS[lens]
    nslots = len(lens) + 2
    starts, slots, resume, rows = ref.packed(r, lens, nslots, first=1)
    if len(lens) > 3:
        slots[2] = nslots + 5
    s = Scan(r, sfx, rows, nslots, *shape, off=0 if shape[1] % 16 == 0 else 1)
    s.check(s.go(mp, stream, slots, resume, starts), starts, slots, resume)


@pytest.mark.parametrize("sfx", TYPES)
@pytest.mark.parametrize("lens", [[700], [64, 128, 63, 65, 191], [1] * 33 + [200]])
def test_scan_prompt_lengths(mp, stream, sfx, lens):
    r = np.random.default_rng(len(lens))
    starts, slots, resume, rows = ref.packed(r, lens, len(lens))
    s = Scan(r, sfx, rows, len(lens), 2, 64, 128, 1)
    s.check(s.go(mp, stream, slots, resume, starts), starts, slots, resume)


@pytest.mark.parametrize("sfx", TYPES)
def test_scan_prompt_strong_decay(mp, stream, sfx):
    """Steps of which next to nothing is left at the following one, down to decays that are zero."""
    r = np.random.default_rng(5)
    lens = [90, 7, 200]
    starts, slots, resume, rows = ref.packed(r, lens, 3)
    s = Scan(r, sfx, rows, 3, 4, 64, 128, 1, strong=True)
    s.check(s.go(mp, stream, slots, resume, starts), starts, slots, resume)


@pytest.mark.parametrize("sfx", TYPES)
def test_scan_prompt_every_default(mp, stream, sfx):
    """No slots (sequence i uses state i), no resume (all begin with zeros, whatever the states hold)."""
    r = np.random.default_rng(6)
    lens = [70, 3, 0]
    starts, _, _, rows = ref.packed(r, lens, 3)
    s = Scan(r, sfx, rows, 3, 2, 64, 128, 1)
    s.states[:] = np.nan
    got = s.go(mp, stream, None, None, starts)
    s.states[:] = 0
    s.check(got, starts, np.arange(3), np.zeros(3))


@pytest.mark.parametrize("sfx", TYPES)
@pytest.mark.parametrize("n", [1, 2, 40])
@pytest.mark.parametrize("shape", SCAN_SHAPES)
def test_scan_token(mp, stream, sfx, n, shape):
    r = np.random.default_rng(sum(shape) + n)
    nslots = n + 2
    slots = r.permutation(nslots)[:n].astype(np.int32)
    if n > 5:
        slots[3], slots[4] = -1, nslots
    s = Scan(r, sfx, n, nslots, *shape, off=0 if shape[1] % 16 == 0 else 1)
    s.check(s.go(mp, stream, slots), np.arange(n + 1), slots, np.ones(n))


@pytest.mark.parametrize("sfx", TYPES)
def test_nan_stays_with_its_sequence(mp, stream, sfx):
    """A NaN in one prompt, and an infinity in another's state, do not reach their neighbours in the packed rows."""
    r = np.random.default_rng(8)
    lens = [40, 50, 60]
    starts, slots, _, rows = ref.packed(r, lens, 3)
    resume = np.array([1, 1, 1], np.int32)
    s = Scan(r, sfx, rows, 3, 2, 64, 128, 1)
    clean = s.go(mp, stream, slots, resume, starts)
    s.xbc[starts[1] + 20, 5] = np.nan
    s.states[slots[2]] = np.inf
    y, states = s.go(mp, stream, slots, resume, starts)
    assert np.array_equal(y[:40], clean[0][:40]) and np.array_equal(states[slots[0]], clean[1][slots[0]])
    within(y[40:60].astype(np.float64), clean[0][40:60].astype(np.float64), np.abs(clean[0][40:60].astype(np.float64)) * 2 * ref.U_OUT[sfx] + 1e-5, "before the NaN")
    assert np.isnan(y[60:90, 5].astype(np.float64)).all() and not np.isfinite(states[slots[2]].astype(np.float64)).any()


# Prompts in r16 whose rows are aligned: chunks on the tensor cores.
def chunked(r, lens, shape, nslots=None, first=0, **more):
    nslots = nslots or len(lens) + 1
    starts, slots, resume, rows = ref.packed(r, lens, nslots, first=first)
    return Scan(r, "r16", rows, nslots, *shape, behind=8, **more), starts, slots, resume


@pytest.mark.parametrize("lens", [[1], [128], [2, 0, 3, 1], [127, 129, 128, 1, 0, 255, 256, 257], [3] * 60 + [0] * 3 + [140]])
@pytest.mark.parametrize("shape", [(2, 64, 128, 1), (4, 64, 128, 2), (3, 8, 8, 3), (2, 16, 16, 2), (1, 80, 64, 1), (1, 128, 128, 1), (6, 32, 96, 3), (1, 200, 24, 1)])
def test_chunks(mp, stream, lens, shape):
    r = np.random.default_rng(sum(shape) + sum(lens))
    s, starts, slots, resume = chunked(r, lens, shape, first=3)
    if len(lens) > 3:
        slots[2] = -1
    s.check(s.go(mp, stream, slots, resume, starts), starts, slots, resume)


@pytest.mark.parametrize("lens", [[700], [1000, 5, 0, 600], [256] * 3, [257, 511, 513], [0, 0, 1290]])
@pytest.mark.parametrize("scratch", [True, False])
def test_chunks_in_ranges(mp, stream, lens, scratch):
    """Few sequences: cut into ranges where there is scratch, whole otherwise."""
    r = np.random.default_rng(sum(lens))
    s, starts, slots, resume = chunked(r, lens, (3, 64, 128, 1), first=1)
    s.check(s.go(mp, stream, slots, resume, starts, scratch), starts, slots, resume)


def test_chunks_in_ranges_of_partial_tiles(mp, stream):
    r = np.random.default_rng(77)
    s, starts, slots, resume = chunked(r, [900, 333], (2, 80, 40, 2))
    s.check(s.go(mp, stream, slots, resume, starts), starts, slots, resume)


@pytest.mark.parametrize("lens", [[150], [90, 7, 200], [900]])
def test_chunks_strong_decay(mp, stream, lens):
    r = np.random.default_rng(sum(lens))
    s, starts, slots, resume = chunked(r, lens, (4, 64, 128, 1), strong=True)
    s.check(s.go(mp, stream, slots, resume, starts), starts, slots, resume)


@pytest.mark.parametrize("xs,bs,ss", [(1e-3, 1.0, 1.0), (30.0, 1.0, 1e2), (1.0, 30.0, 0.0), (1e-4, 1e-3, 1e-8), (0.0, 1.0, 1.0)])
def test_chunks_of_any_magnitude(mp, stream, xs, bs, ss):
    r = np.random.default_rng(31)
    s, starts, slots, resume = chunked(r, [200, 90], (2, 64, 128, 1))
    s.xbc[:, :s.inner] = (s.xbc[:, :s.inner].astype(np.float32) * xs).astype(np.float16)
    s.xbc[:, s.inner:s.inner + s.bc] = (s.xbc[:, s.inner:s.inner + s.bc].astype(np.float32) * bs).astype(np.float16)
    s.states *= np.float32(ss)
    if xs == 1e-4:      # x and B are r16 subnormal values: their products are exact all the same
        s.xbc[5] = np.float16(6e-8)
    s.check(s.go(mp, stream, slots, resume, starts), starts, slots, resume)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("what", ["x", "B", "C", "raw", "state", "neighbour"])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_chunks_with_an_infinity(mp, stream, long, what, value):
    """What is not finite goes where the recurrence takes it, and nowhere else."""
    r = np.random.default_rng(40)
    lens = [700, 30] if long else [150, 130, 30]
    s, starts, slots, resume = chunked(r, lens, (2, 64, 128, 1))
    resume[:] = 1
    at = starts[1] + (20 if what == "neighbour" else -57)
    if what in ("x", "neighbour"):
        s.xbc[at, 5] = value
    elif what == "B":
        s.xbc[at, s.inner + 9] = value
    elif what == "C":
        s.xbc[at, s.inner + s.bc + 9] = value
    elif what == "raw":
        s.zx[at, 3] = value
    else:
        s.states[slots[0], 0, 3, 7] = value
    y, states = s.go(mp, stream, slots, resume, starts)
    with np.errstate(all="ignore"):
        wy, ysize, ws, ssize, ysteps, ssteps = s.want(starts, slots, resume)
    H, P, N, G = s.dims
    y = y[:, :s.inner].reshape(-1, H, P)
    for got, want, size, steps, out in ((y[:starts[-1]], wy[:starts[-1]], ysize, ysteps, True), (states[slots], ws[slots], ssize, ssteps, False)):
        got = got.astype(np.float64)
        size, steps = (size[:starts[-1]], steps[:starts[-1]]) if out else (size[slots], steps[slots])
        assert np.array_equal(np.isfinite(got), np.isfinite(want)) and np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
        fine = np.isfinite(want)
        with np.errstate(all="ignore"):
            tol = np.broadcast_to(ref.scan_tolerance("r16", want, size, steps, N, out), want.shape)
        within(got[fine], want[fine], tol[fine], "finite part")


@pytest.mark.parametrize("sfx,shape", [("r16", (2, 64, 40, 1)), ("r16", (2, 64, 77, 1)), ("r32", (2, 33, 77, 1)), ("r32", (2, 64, 128, 1)), ("r64", (2, 16, 5, 2)), ("r32", (1, 8, 200, 1))])
@pytest.mark.parametrize("lens", [[37, 5], [700, 3]])
@pytest.mark.parametrize("what", ["x", "rate"])
def test_infinities_beside_padding(mp, stream, sfx, shape, lens, what):
    """State sizes that fill no tile: an infinite x among positive B and C makes y infinite, not undefined; a head that forgets at once (its decay
    is exactly zero) keeps the last step only."""
    r = np.random.default_rng(sum(shape))
    starts, slots, resume, rows = ref.packed(r, lens, 3)
    resume[:] = 1
    s = Scan(r, sfx, rows, 3, *shape, behind=8)
    s.xbc[:, s.inner:] = np.abs(s.xbc[:, s.inner:]) + NP_OF[sfx](0.125)
    if what == "x":
        s.xbc[starts[1] - 2, 1] = np.inf
    else:
        s.A_log[0] = np.inf
    y, states = s.go(mp, stream, slots, resume, starts)
    with np.errstate(all="ignore"):
        wy, ysize, ws, ssize, ysteps, ssteps = s.want(starts, slots, resume)
    H, P, N, G = s.dims
    y = y[:, :s.inner].reshape(-1, H, P)
    with np.errstate(all="ignore"):
        ytol, stol = ref.scan_tolerance(sfx, wy, ysize, ysteps, N, True), ref.scan_tolerance(sfx, ws, ssize, ssteps, N, False)
    for got, want, tol in ((y[:starts[-1]], wy[:starts[-1]], np.broadcast_to(ytol, wy.shape)[:starts[-1]]), (states[slots], ws[slots], np.broadcast_to(stol, ws.shape)[slots])):
        got = got.astype(np.float64)
        assert np.array_equal(np.isinf(got), np.isinf(want)) and not np.isnan(got).any()
        fine = np.isfinite(want)
        within(got[fine], want[fine], tol[fine], "finite part")


@pytest.mark.parametrize("sfx", TYPES)
def test_ranges_begin_with_the_kept_state(mp, stream, sfx):
    """Long prompts that go on from a state, the last range of a single step: the first range begins with the state that was kept, not with the one
    that the last range leaves.  The same bits every time."""
    r = np.random.default_rng(50)
    lens = [1024 * 2 + 1, 1537]
    starts, slots, resume, rows = ref.packed(r, lens, 3)
    resume[:] = 1
    s = Scan(r, sfx, rows, 3, 2, 64, 128, 1, behind=8)
    s.states *= 30
    first = s.go(mp, stream, slots, resume, starts)
    s.check(first, starts, slots, resume)
    for _ in range(4):
        again = s.go(mp, stream, slots, resume, starts)
        assert np.array_equal(again[0], first[0]) and np.array_equal(again[1], first[1])


# ---------------------------------------------------------------------------------------------------- selection
def select(mp, stream, sfx, logits, scores, finished, eos, picks, off=0):
    import torch
    batch, beams, vocab = logits.shape
    pitch = vocab + off
    buf = np.full((batch * beams, pitch), np.nan, NP_OF[sfx])
    buf[:, off:] = logits.reshape(-1, vocab)
    acc = torch_dtype("r64" if sfx == "r64" else "r32")
    out = [torch.full((batch, picks), -9, dtype=t, device="cuda") for t in (acc, torch.int32, torch.int32, torch.int32)]
    nbytes = mp.lib().mpBeamSelectScratchBytes(TYPES.index(sfx), batch, beams, vocab, picks)
    scratch = torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda")
    d = dev(buf)
    run(mp, stream, "beam_select", sfx, d.data_ptr() + off * d.element_size(), pitch, dev(scores), None if finished is None else dev(finished), eos, *out, scratch,
        batch, beams, vocab, picks)
    return [host(t) for t in out]


def check_select(got, logits, scores, finished, eos, picks, sfx):
    s, p, t, f = ref.select(logits, scores, finished, eos, picks)
    assert np.array_equal(got[1], p), (got[1], p)
    assert np.array_equal(got[2], t), (got[2], t)
    if eos < logits.shape[2]:
        assert np.array_equal(got[3], f)
    # exp(v - max) to 2^-22 and its exponent's rounding, (1 + ln vocab) of them weighted by the exponential, and a lane's own sum of vocab / 32 terms
    u = ref.U_ACC[sfx]
    tol = 4 * u * (1 + np.log(logits.shape[2])) + u * (logits.shape[2] / 32 + 8) + u * np.abs(s)
    with np.errstate(invalid="ignore"):
        same = (got[0].astype(np.float64) == s) | (np.abs(got[0].astype(np.float64) - s) <= tol)
    assert same.all(), (got[0], s)


@pytest.mark.parametrize("sfx", TYPES)
@pytest.mark.parametrize("batch,beams,vocab,picks,off", [(1, 1, 5, 1, 0), (3, 4, 1024, 8, 0), (2, 5, 4999, 7, 0), (1, 12, 333, 32, 3), (2, 64, 50, 32, 1), (1, 3, 32, 32, 0),
                                                         (70, 2, 101, 4, 5), (1, 2, 50280, 16, 0)])
def test_select(mp, stream, sfx, batch, beams, vocab, picks, off):
    r = np.random.default_rng(vocab + beams)
    logits = ref.storage(r, (batch, beams, vocab), sfx, 2.0)
    scores = r.uniform(-20, 0, (batch, beams)).astype(ref.ACC[sfx])
    finished = (r.random((batch, beams)) < 0.2).astype(np.int32)
    for fin, eos in ((None, vocab), (finished, vocab // 2), (finished, 0), (None, vocab - 1)):
        check_select(select(mp, stream, sfx, logits, scores, fin, eos, picks, off), logits, scores, fin, eos, picks, sfx)


@pytest.mark.parametrize("sfx", TYPES)
def test_select_ties(mp, stream, sfx):
    """Equal logits: the lowest token; equal beams: the lowest beam.  Rows of one value, of few values, rising and falling ones."""
    r = np.random.default_rng(3)
    vocab, picks = 3001, 20
    rows = [np.zeros(vocab), np.full(vocab, -2.5), r.integers(0, 3, vocab), np.arange(vocab) // 8 * 0.25 - 300, -(np.arange(vocab) // 8 * 0.25), r.integers(0, 3, vocab)]
    logits = np.array(rows).reshape(2, 3, vocab).astype(NP_OF[sfx])
    logits[1, 2] = logits[0, 2]
    for scores in (np.zeros((2, 3)), np.array([[-1.0, -1.0, -9.0], [-5, -6, -7]])):
        check_select(select(mp, stream, sfx, logits, scores.astype(ref.ACC[sfx]), None, vocab, picks), logits, scores, None, vocab, picks, sfx)
    same = np.repeat(logits[:, 2:3], 3, axis=1)
    scores = np.full((2, 3), -2.0, ref.ACC[sfx])
    check_select(select(mp, stream, sfx, same, scores, None, vocab, picks), same, scores, None, vocab, picks, sfx)


@pytest.mark.parametrize("sfx", TYPES)
def test_select_masked_and_impossible(mp, stream, sfx):
    r = np.random.default_rng(4)
    vocab, picks = 500, 9
    logits = ref.storage(r, (1, 8, vocab), sfx)
    low = np.finfo(NP_OF[sfx]).min
    logits[0, 0, 3:] = -np.inf                    # three tokens left
    logits[0, 1, 7] = np.nan
    logits[0, 2, 9] = np.inf
    logits[0, 3] = -np.inf
    logits[0, 4, 2:] = low                        # masks of the type's lowest value
    logits[0, 5] = low
    scores = np.array([[-1, 0, 0, 0, -2, -30, 0, 0]], ref.ACC[sfx])
    scores[0, 6], scores[0, 7] = np.nan, -np.inf
    check_select(select(mp, stream, sfx, logits, scores, None, vocab, picks), logits, scores, None, vocab, picks, sfx)
    dead = scores.copy()
    dead[0, :6] = -np.inf                         # nothing is possible: the first beam's first tokens
    check_select(select(mp, stream, sfx, logits, dead, None, vocab, picks), logits, dead, None, vocab, picks, sfx)
    done = np.ones((1, 8), np.int32)              # all have ended: each goes on with the end, the rest is impossible
    check_select(select(mp, stream, sfx, logits, scores, done, 11, picks), logits, scores, done, 11, picks, sfx)
    if sfx != "r16":
        lowest = np.full((1, 8), np.finfo(ref.ACC[sfx]).min, ref.ACC[sfx])      # scores of the lowest value swallow the logits
        check_select(select(mp, stream, sfx, logits, lowest, None, vocab, picks), logits, lowest, None, vocab, picks, sfx)


def test_select_in_place(mp, stream):
    """next_scores over scores and next_finished over finished."""
    import torch
    r = np.random.default_rng(9)
    batch, beams, vocab = 5, 4, 777
    logits = ref.storage(r, (batch, beams, vocab), "r32")
    scores, finished = r.uniform(-5, 0, (batch, beams)).astype(np.float32), (r.random((batch, beams)) < 0.3).astype(np.int32)
    want = ref.select(logits, scores, finished, 5, beams)
    ds, df = dev(scores), dev(finished)
    p, t = (torch.empty(batch, beams, dtype=torch.int32, device="cuda") for _ in range(2))
    scratch = torch.empty(mp.lib().mpBeamSelectScratchBytes(1, batch, beams, vocab, beams), dtype=torch.uint8, device="cuda")
    run(mp, stream, "beam_select", "r32", dev(logits), vocab, ds, df, 5, ds, p, t, df, scratch, batch, beams, vocab, beams)
    assert np.array_equal(host(p), want[1]) and np.array_equal(host(t), want[2]) and np.array_equal(host(df), want[3])
    assert np.allclose(host(ds), want[0], rtol=0, atol=2e-5)


# ---------------------------------------------------------------------------------------------------- reordering
@pytest.mark.parametrize("sfx", TYPES)
@pytest.mark.parametrize("layers,batch,beams,row,spare,off", [(1, 1, 1, 7, 0, 0), (2, 3, 4, 1792, 1, 0), (3, 2, 5, 33, 4, 0), (1, 40, 12, 5, 0, 1), (2, 1, 64, 130, 2, 0),
                                                              (1, 2, 33, 1001, 3, 1), (24, 1, 8, 640, 0, 0)])
def test_reorder(mp, stream, sfx, layers, batch, beams, row, spare, off):
    r = np.random.default_rng(beams * row)
    nslots = batch * beams + spare
    flat = ref.storage(r, (layers * nslots * row + off,), sfx)
    slots = r.permutation(nslots)[:batch * beams].astype(np.int32)
    parents = r.integers(0, beams, (batch, beams)).astype(np.int32)
    parents[0] = np.roll(np.arange(beams), 1)                     # a cycle through all of them
    if batch > 1:
        parents[1] = np.arange(beams)
    if batch > 2:
        parents[2, 0], parents[2, -1], slots[2 * beams + 1] = -1, beams, nslots + 2      # left as they are
    for given in (slots, None):
        use = slots if given is not None else np.arange(batch * beams)
        old = flat[off:].reshape(layers, nslots, row)
        want = old.copy()
        for b in range(batch):
            for j in range(beams):
                p = parents[b, j]
                if 0 <= p < beams and 0 <= use[b * beams + j] < nslots and 0 <= use[b * beams + p] < nslots:
                    want[:, use[b * beams + j]] = old[:, use[b * beams + p]]
        d = dev(flat)
        run(mp, stream, "reorder_states", sfx, d.data_ptr() + off * d.element_size(), None if given is None else dev(given), dev(parents), layers, batch, beams, nslots, row)
        assert np.array_equal(host(d)[off:].reshape(want.shape), want) and np.array_equal(host(d)[:off], flat[:off])


# ---------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("sfx", TYPES)
def test_prompt_then_tokens_is_one_prompt(mp, stream, sfx):
    """A prompt in two calls and then token by token: the plain form's results of the whole at once."""
    r = np.random.default_rng(12)
    n, cut, tokens = 100, 61, 4
    whole = Scan(r, sfx, n, 1, 2, 64, 128, 1)
    one = np.zeros(1, np.int32)
    wy, ysize, ws, ssize, ysteps, ssteps = whole.want(np.array([0, n]), one, one)
    ys, states = [], whole.states
    for lo, hi in [(0, cut), (cut, n - tokens)] + [(k, k + 1) for k in range(n - tokens, n)]:
        part = Scan.__new__(Scan)
        part.__dict__.update(whole.__dict__)
        part.xbc, part.zx, part.y0, part.states = whole.xbc[lo:hi], whole.zx[lo:hi], whole.y0[lo:hi], states
        y, states = part.go(mp, stream, one) if hi - lo == 1 else part.go(mp, stream, one, np.array([lo > 0], np.int32), np.array([0, hi - lo], np.int32))
        ys.append(y[:, :whole.inner])
    del wy, ws
    zero = whole.want(np.array([0, n]), one, np.zeros(1))
    within(np.concatenate(ys).reshape(zero[0].shape), zero[0], ref.scan_tolerance(sfx, zero[0], zero[1], zero[4], 128, True), "y")
    within(states, zero[2], ref.scan_tolerance(sfx, zero[2], zero[3], zero[5], 128, False), "states")


def test_captured_and_replayed(mp, stream):
    """A token's conv, scan, selection and reordering in a graph, replayed three times: what the same launches give one by one."""
    import torch
    r = np.random.default_rng(15)
    batch, beams, vocab, heads, width = 2, 3, 999, 2, 4
    n, channels = batch * beams, heads * 64 + 256
    base = dict(zx=ref.storage(r, (n, channels + heads), "r16"), w=ref.storage(r, (channels, width), "r16", 0.5), conv=ref.storage(r, (n, width - 1, channels), "r16"),
                ssm=r.standard_normal((n, heads, 64, 128)).astype(np.float32), dt_bias=np.full(heads, -3, np.float32), A_log=np.zeros(heads, np.float32),
                logits=ref.storage(r, (n, vocab), "r16", 2.0), scores=np.zeros((batch, beams), np.float32))
    lib = mp.lib()

    def fresh():
        d = {k: dev(v) for k, v in base.items()}
        d.update(xbc=torch.zeros(n, channels, dtype=torch.float16, device="cuda"), y=torch.zeros(n, heads * 64, dtype=torch.float16, device="cuda"),
                 parents=torch.zeros(batch, beams, dtype=torch.int32, device="cuda"), tokens=torch.zeros(batch, beams, dtype=torch.int32, device="cuda"),
                 scratch=torch.empty(lib.mpBeamSelectScratchBytes(0, batch, beams, vocab, beams), dtype=torch.uint8, device="cuda"))
        torch.cuda.synchronize()
        return d

    def issue(d, st):
        t = torch.float16
        mp.launch("causal_conv1d_silu_token", t, d["zx"], channels + heads, d["w"], None, d["conv"], None, d["xbc"], channels, n, n, channels, width, st)
        x = d["xbc"].data_ptr()
        mp.launch("ssd_scan_token", t, x, channels, d["zx"].data_ptr() + channels * 2, channels + heads, d["dt_bias"], d["A_log"], x + heads * 128,
                  x + heads * 128 + 256, channels, d["ssm"], None, d["y"], heads * 64, n, n, heads, 64, 128, 1, st)
        mp.launch("beam_select", t, d["logits"], vocab, d["scores"], None, vocab, d["scores"], d["parents"], d["tokens"], None, d["scratch"], batch, beams, vocab, beams, st)
        mp.launch("reorder_states", torch.float32, d["ssm"], None, d["parents"], 1, batch, beams, n, heads * 64 * 128, st)
        mp.launch("reorder_states", t, d["conv"], None, d["parents"], 1, batch, beams, n, (width - 1) * channels, st)

    plain, graphed = fresh(), fresh()
    with mp.Stream() as st:
        for _ in range(3):
            issue(plain, st)
        st.sync()
        lib.mpGraphBeginCapture(st.ctx)
        issue(graphed, st)
        graph = lib.mpGraphEndCapture(st.ctx)
        for _ in range(3):
            lib.mpGraphLaunch(C.c_void_p(graph), st.ctx)
        st.sync()
        lib.mpGraphDestroy(C.c_void_p(graph))
    for k in ("conv", "ssm", "y", "scores", "parents", "tokens"):
        assert torch.equal(plain[k], graphed[k]), k


def test_two_streams_at_once(mp, stream):
    """Two calls with buffers of their own, in flight together."""
    import torch
    r = np.random.default_rng(16)
    lens = [300, 17]
    starts, slots, resume, rows = ref.packed(r, lens, 2)
    a, b = Scan(r, "r16", rows, 2, 8, 64, 128, 1), Scan(r, "r16", rows, 2, 8, 64, 128, 1)
    alone = [s.go(mp, stream, slots, resume, starts) for s in (a, b)]
    want = [host(s.d["y0"]) for s in (a, b)]
    streams = [mp.Stream(), mp.Stream()]
    ctl = [dev(v) for v in (slots, resume, starts)]
    for s in (a, b):
        s.d["states"].copy_(dev(s.states))
        s.d["y0"].copy_(dev(s.y0))
    torch.cuda.synchronize()
    for s, st in zip((a, b), streams):
        x = s.d["xbc"].data_ptr()
        mp.launch("ssd_scan_prompt", torch.float16, x, s.xbc.shape[1], s.d["zx"].data_ptr() + 6, s.zx.shape[1], s.d["dt_bias"], s.d["A_log"], x + 2 * s.inner,
                  x + 2 * (s.inner + s.bc), s.xbc.shape[1], s.d["states"], ctl[0], ctl[1], ctl[2], s.d["y0"], s.y0.shape[1], s.scratch, 2, rows, 2, *s.dims, st)
    for st in streams:
        st.sync()
        st.close()
    for s, w, (_, states) in zip((a, b), want, alone):
        assert np.array_equal(host(s.d["y0"]), w) and np.array_equal(host(s.d["states"]), states)


@pytest.mark.parametrize("sfx", ["r16", "r32"])
def test_prompts_captured_and_replayed(mp, stream, sfx):
    """Convolution and scan of prompts (in ranges) in a graph: the bits of the same launches one by one, as often as it is replayed."""
    import torch
    r = np.random.default_rng(17)
    lens, heads, width = [700, 0, 33], 2, 4
    starts, slots, resume, rows = ref.packed(r, lens, 4)
    resume[:] = 1
    channels, t = heads * 64 + 256, torch_dtype(sfx)
    size = np.dtype(NP_OF[sfx]).itemsize
    base = dict(zx=ref.storage(r, (rows, channels + 8), sfx), w=ref.storage(r, (channels, width), sfx, 0.5), conv=ref.storage(r, (4, width - 1, channels), sfx),
                ssm=r.standard_normal((4, heads, 64, 128)).astype(np.float32), dt_bias=np.full(heads, -3, np.float32), A_log=np.zeros(heads, np.float32),
                starts=starts, slots=slots, resume=resume)
    lib = mp.lib()

    def fresh():
        d = {k: dev(v) for k, v in base.items()}
        d.update(xbc=torch.zeros(rows, channels, dtype=t, device="cuda"), y=torch.zeros(rows, heads * 64, dtype=t, device="cuda"),
                 scratch=torch.zeros(lib.mpSsdScanPromptScratchBytes(TYPES.index(sfx), 3, rows, heads, 64, 128, 1), dtype=torch.uint8, device="cuda"))
        torch.cuda.synchronize()
        return d

    def issue(d, st):
        mp.launch("causal_conv1d_silu_prompt", t, d["zx"], channels + 8, d["w"], None, d["conv"], d["slots"], d["resume"], d["starts"], d["xbc"], channels, 3, rows, 4,
                  channels, width, st)
        x = d["xbc"].data_ptr()
        mp.launch("ssd_scan_prompt", t, x, channels, d["zx"].data_ptr() + channels * size, channels + 8, d["dt_bias"], d["A_log"], x + heads * 64 * size,
                  x + (heads * 64 + 128) * size, channels, d["ssm"], d["slots"], d["resume"], d["starts"], d["y"], heads * 64, d["scratch"], 3, rows, 4, heads, 64, 128, 1, st)

    plain, graphed = fresh(), fresh()
    with mp.Stream() as st:
        for _ in range(3):
            issue(plain, st)
        st.sync()
        lib.mpGraphBeginCapture(st.ctx)
        issue(graphed, st)
        graph = lib.mpGraphEndCapture(st.ctx)
        for _ in range(3):
            lib.mpGraphLaunch(C.c_void_p(graph), st.ctx)
        st.sync()
        assert st.status() == 0
        lib.mpGraphDestroy(C.c_void_p(graph))
    for k in ("conv", "ssm", "xbc", "y"):
        assert torch.equal(plain[k], graphed[k]), k


@pytest.mark.parametrize("sfx", TYPES)
def test_select_any_offset_gives_the_same(mp, stream, sfx):
    """Rows on the 16-byte boundary and off it by every possible offset: the same bits, and equal rows tie whatever their addresses."""
    r = np.random.default_rng(23)
    vocab, beams, picks = 4003, 4, 8
    one = ref.storage(r, (1, 1, vocab), sfx, 2.0)
    logits = np.repeat(one, beams, axis=1)
    scores = np.zeros((1, beams), ref.ACC[sfx])
    want = None
    for off in range(16 // np.dtype(NP_OF[sfx]).itemsize + 1):
        got = select(mp, stream, sfx, logits, scores, None, vocab, picks, off)
        assert np.array_equal(got[1][0], np.arange(picks) % beams) and np.array_equal(got[2][0], np.repeat(got[2][0][::beams], beams)), off
        want = got if want is None else want
        assert all(np.array_equal(a, b) for a, b in zip(got[:3], want[:3])), off
