"""Performance cases of the operators that answer with a trained Mamba-2 model: the two that its blocks need, over prompts
and over single tokens, and the two of a beam search.

    conv     causal convolution + SiLU that goes on from the last width - 1 inputs of each sequence (prompt and token form)
    scan     the SSD scan that goes on from a kept state of each sequence (prompt and token form)
    select   the best continuations over the beams and the vocabulary
    reorder  the kept states follow the beams that were selected, in place

Sequences are packed: rows `starts[i] .. starts[i + 1]` are sequence i, its state lies in row `slots[i]` of the state
buffer, and it goes on from that state where `resume[i]` is not zero.  `listed()` holds fixed cases, `draw(rng)` one more
of the same ranges.  `run` computes them in elementary torch operations, or by the framework's launchers where `own` is set.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DTYPES = {"r16": torch.float16, "r32": torch.float32, "r64": torch.float64}
SIZE = {"r16": 2, "r32": 4, "r64": 8}
ACC = {"r16": torch.float32, "r32": torch.float32, "r64": torch.float64}
ACC_SIZE = {"r16": 4, "r32": 4, "r64": 8}
CHUNK = 64       # steps that the plain scan takes at a time


def listed():
    return [
        # A batch of prompts of all lengths, half of them the next turn of a conversation: the block's convolution over x, B and C.
        dict(name="conv_prompt_16_r16", kind="conv", form="prompt", dtype="r16", nseq=16, longest=1023, heads=24, headdim=64, dstate=128, groups=1, width=4),
        # The same for one new token of 64 sequences.
        dict(name="conv_token_64_r16", kind="conv", form="token", dtype="r16", nseq=64, longest=1, heads=24, headdim=64, dstate=128, groups=1, width=4),
        # One short question to the benchmark's model: latency counts.
        dict(name="scan_prompt_1x37_r16", kind="scan", form="prompt", dtype="r16", nseq=1, longest=37, heads=24, headdim=64, dstate=128, groups=1),
        # The batch of prompts through the scan of the benchmark's model.
        dict(name="scan_prompt_16_r16", kind="scan", form="prompt", dtype="r16", nseq=16, longest=1023, heads=24, headdim=64, dstate=128, groups=1),
        # A long document at the benchmark scan's width: one sequence, its length no multiple of anything.
        dict(name="scan_prompt_1x8191_r16", kind="scan", form="prompt", dtype="r16", nseq=1, longest=8191, heads=32, headdim=64, dstate=128, groups=1),
        # The tests' small model in r32, a few prompts.
        dict(name="scan_prompt_5_r32", kind="scan", form="prompt", dtype="r32", nseq=5, longest=333, heads=8, headdim=64, dstate=128, groups=2),
        # One token of one conversation.
        dict(name="scan_token_1_r16", kind="scan", form="token", dtype="r16", nseq=1, longest=1, heads=24, headdim=64, dstate=128, groups=1),
        # One token of many: the states stream through HBM.
        dict(name="scan_token_300_r16", kind="scan", form="token", dtype="r16", nseq=300, longest=1, heads=24, headdim=64, dstate=128, groups=1),
        # A search with four beams for one prompt, the benchmark's vocabulary.
        dict(name="select_1x4_r16", kind="select", dtype="r16", batch=1, beams=4, picks=4, vocab=50280),
        # Eight beams for a batch, twice as many candidates as beams so that finished ones can be set aside.
        dict(name="select_64x8_r16", kind="select", dtype="r16", batch=64, beams=8, picks=16, vocab=50280),
        # The convolution's states of 24 layers follow the beams of one search.
        dict(name="reorder_1x4_r16", kind="reorder", dtype="r16", layers=24, batch=1, beams=4, sources=2, row=3 * 1792),
        # The scan's states of 24 layers for a batch of searches.
        dict(name="reorder_8x5_r32", kind="reorder", dtype="r32", layers=24, batch=8, beams=5, sources=3, row=24 * 64 * 128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _block(rng, dtype):
    """The sizes of a Mamba-2 block's inner part."""
    groups = rng.choice((1, 1, 2, 4))
    heads = groups * _log(rng, 1, 32 // groups)
    c = dict(heads=heads, headdim=64, dstate=128, groups=groups)
    if rng.random() < 0.3:     # other head and state sizes, odd ones among them
        c.update(headdim=rng.choice((16, 32, 33, 48, 64, 80, 128)), dstate=rng.choice((16, 32, 64, 77, 96, 128, 256)))
    if dtype == "r64":
        c["heads"] = groups * max(1, min(heads // groups, 4))
    return c


def draw(rng):
    kind = rng.choice(("conv", "scan", "scan", "scan", "select", "select", "reorder"))
    dtype = rng.choice(("r16", "r16", "r16", "r32", "r32", "r64"))
    if kind == "conv":
        form = rng.choice(("prompt", "token"))
        c = dict(kind=kind, form=form, dtype=dtype, **_block(rng, dtype), width=rng.choice((2, 3, 4, 4)))
        c["nseq"] = _log(rng, 1, 300 if form == "token" else 32)
        c["longest"] = 1 if form == "token" else _log(rng, 1, 16384 // c["nseq"])
        return c
    if kind == "scan":
        form = rng.choice(("prompt", "prompt", "token"))
        c = dict(kind=kind, form=form, dtype=dtype, **_block(rng, dtype))
        share = max(1.0, c["headdim"] * c["dstate"] * c["heads"] / (64 * 128 * 24) * (8 if dtype == "r64" else 2 if dtype == "r32" else 1))
        c["nseq"] = _log(rng, 1, int((300 if form == "token" else 32) / share) + 1)
        c["longest"] = 1 if form == "token" else _log(rng, 1, max(2, min(8191, int(8191 / share / math.sqrt(c["nseq"])))))
        return c
    if kind == "select":
        beams = rng.choice((1, 2, 3, 4, 5, 8, 12))
        return dict(kind=kind, dtype=dtype, batch=_log(rng, 1, 512 // beams // (1 if dtype == "r16" else 2 if dtype == "r32" else 8)), beams=beams,
                    picks=min(32, max(1, rng.choice((beams, 2 * beams, beams + 1)))), vocab=_log(rng, 40, 50280))
    beams = rng.choice((3, 4, 5, 8, 12))
    row = _log(rng, 5, 24 * 64 * 128)
    layers = rng.choice((1, 2, 6, 24))
    return dict(kind=kind, dtype=dtype, layers=layers, batch=_log(rng, 1, max(1, min(64, 37_000_000 // (row * layers * beams * (2 if dtype == "r64" else 1))))),
                beams=beams, sources=rng.randrange(1, beams - 1), row=row)


# --------------------------------------------------------------------------------------------------------------
# what a program holds before the call
# --------------------------------------------------------------------------------------------------------------
def _lengths(c):
    """The case's sequence lengths: the longest first, the others spread over the range; of many sequences, one is empty."""
    n, most = c["nseq"], c["longest"]
    if c["form"] == "token":
        return [1] * n
    lens = [max(1, int(most * ((0.618 * i) % 1.0))) if i else most for i in range(n)]
    if n >= 8:
        lens[n // 2] = 0
    return lens


def _resumes(c):
    """Whether sequence i goes on from its state: every other one, and every one that has a token already."""
    return [1 if c["form"] == "token" else i % 2 for i in range(c["nseq"])]


class _Inputs:
    """Seeded random tensors on the device."""

    def __init__(self, seed, dtype):
        self.g, self.dtype = torch.Generator(device="cuda").manual_seed(seed), dtype

    def normal(self, *shape, scale=1.0, shift=0.0, dtype=None):
        return torch.randn(*shape, generator=self.g, device="cuda").mul_(scale).add_(shift).to(dtype or self.dtype)

    def uniform(self, *shape, lo=0.0, hi=1.0, dtype=None):
        return torch.rand(*shape, generator=self.g, device="cuda").mul_(hi - lo).add_(lo).to(dtype or self.dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").to(torch.int32)


def _sequences(c, r):
    """Packed rows: where each sequence begins, which state is its own, whether it goes on; some rows behind the last one are nobody's."""
    lens = _lengths(c)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    spare = 0 if c["form"] == "token" else 3
    nslots = c["nseq"] + 2
    return dict(lens=lens, rows=starts[-1] + spare, nslots=nslots, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                slots=r.order(nslots)[:c["nseq"]].contiguous(), resume=torch.tensor(_resumes(c), dtype=torch.int32, device="cuda"))


def _columns(c):
    """Columns of the input projection's result: [ z | x B C | dt ]."""
    inner, bc = c["heads"] * c["headdim"], c["groups"] * c["dstate"]
    return inner, bc, inner + 2 * bc


def _prepare_conv(c, r):
    s = _sequences(c, r)
    inner, bc, channels = _columns(c)
    s.update(zx=r.normal(s["rows"], inner + channels + c["heads"]), w=r.uniform(channels, c["width"], lo=-1 / math.sqrt(c["width"]), hi=1 / math.sqrt(c["width"])),
             bias=r.normal(channels, scale=0.1), states=r.normal(s["nslots"], c["width"] - 1, channels), y=torch.zeros(s["rows"], channels, dtype=r.dtype, device="cuda"))
    return s


def _prepare_scan(c, r):
    s = _sequences(c, r)
    inner, bc, channels = _columns(c)
    acc = ACC[c["dtype"]]
    dt = torch.exp(r.uniform(c["heads"], lo=math.log(1e-3), hi=math.log(1e-1), dtype=torch.float64))
    act = torch.nn.functional.silu(r.normal(s["rows"], channels, dtype=torch.float32)).to(r.dtype)   # what the convolution leaves
    s.update(xbc=act, zx=r.normal(s["rows"], inner + channels + c["heads"]), dt_bias=(dt + torch.log(-torch.expm1(-dt))).to(acc),
             A_log=torch.log(r.uniform(c["heads"], lo=1.0, hi=16.0, dtype=acc)),
             states=r.normal(s["nslots"], c["heads"], c["headdim"], c["dstate"], scale=0.3, dtype=acc),
             y=torch.zeros(s["rows"], inner, dtype=r.dtype, device="cuda"))
    return s


def _prepare_select(c, r):
    rows, vocab = c["batch"] * c["beams"], c["vocab"]
    acc = ACC[c["dtype"]]
    logits = r.normal(rows, vocab, scale=2.0, dtype=torch.float64 if c["dtype"] == "r64" else torch.float32)
    if c["dtype"] == "r64":     # the generator's values have 24 bits
        logits += r.normal(rows, vocab, scale=2.0 ** -26, dtype=torch.float64)
    banned = torch.randint(0, vocab, (rows, max(1, vocab // 100)), generator=r.g, device="cuda")
    logits.scatter_(1, banned[:, ::2].contiguous(), -math.inf)                          # tokens that a filter ruled out
    logits.scatter_(1, banned[:, 1::2].contiguous(), torch.finfo(r.dtype).min)          # or set to the lowest value
    scores = -20.0 * torch.rand(c["batch"], c["beams"], generator=r.g, device="cuda", dtype=torch.float64)
    if c["batch"] > 2:
        scores[1, 1:] = -math.inf        # a search's first step: one beam
    finished = (torch.rand(c["batch"], c["beams"], generator=r.g, device="cuda") < 0.15).to(torch.int32)
    n = (c["batch"], c["picks"])
    return dict(logits=logits.to(r.dtype), scores=scores.to(acc), finished=finished, eos=vocab // 3, next_scores=torch.zeros(n, dtype=acc, device="cuda"),
                parents=torch.zeros(n, dtype=torch.int32, device="cuda"), tokens=torch.zeros(n, dtype=torch.int32, device="cuda"),
                next_finished=torch.zeros(n, dtype=torch.int32, device="cuda"))


def _prepare_reorder(c, r):
    batch, beams, k = c["batch"], c["beams"], c["sources"]
    nslots = batch * beams + 1
    j = torch.arange(beams, device="cuda")
    far = torch.tensor([a for a in range(1, beams) if a != k], device="cuda")     # then every beam of a group that moves has another parent than itself
    a = far[torch.randint(0, far.numel(), (batch,), generator=r.g, device="cuda")]
    parents = (a[:, None] + j[None, :] % k) % beams
    parents[3::4] = j                                                                   # every fourth search keeps its beams
    return dict(states=r.normal(c["layers"], nslots, c["row"]), slots=r.order(nslots)[:batch * beams].contiguous(), parents=parents.to(torch.int32).contiguous(), nslots=nslots)


def prepare(case, seed):
    s = globals()["_prepare_" + case["kind"]](case, _Inputs(seed, DTYPES[case["dtype"]]))
    s["case"] = case
    torch.cuda.synchronize()    # the inputs were made on torch's stream
    return s


# --------------------------------------------------------------------------------------------------------------
# one pass: the plain forms
# --------------------------------------------------------------------------------------------------------------
def _padded(s):
    """Packed rows as [sequence, step] padded to whole chunks: row numbers, and which of them are steps."""
    steps = -(-max(max(s["lens"]), 1) // CHUNK) * CHUNK
    lens = (s["starts"][1:] - s["starts"][:-1]).long()
    t = torch.arange(steps, device="cuda")
    return (s["starts"][:-1, None].long() + t).clamp_(max=s["rows"] - 1), t < lens[:, None], lens


def _plain_conv(s, c):
    inner, bc, channels = _columns(c)
    K, acc, dt = c["width"], ACC[c["dtype"]], DTYPES[c["dtype"]]
    x = s["zx"][:, inner:inner + channels]
    seq = torch.repeat_interleave(torch.arange(c["nseq"], device="cuda"), (s["starts"][1:] - s["starts"][:-1]).long(), output_size=sum(s["lens"]))
    n = seq.numel()
    first, slots = s["starts"][:-1].long(), s["slots"].long()
    kept = s["states"][slots] * s["resume"][:, None, None].to(dt)          # zeros where a sequence begins
    table = torch.cat([x[:n], kept.reshape(-1, channels)])                 # every input that a step can reach
    ago = torch.arange(K - 1, -1, -1, device="cuda")
    at = (torch.arange(n, device="cuda") - first[seq])[:, None] - ago      # [row, tap]: position in its sequence
    where_ = torch.where(at >= 0, first[seq][:, None] + at, n + seq[:, None] * (K - 1) + at + K - 1)
    pre = (table[where_].to(acc) * s["w"].to(acc).T).sum(1) + s["bias"].to(acc)
    s["y"][:n] = (pre * torch.sigmoid(pre)).to(dt)
    last = (s["starts"][1:].long() - first)[:, None] - ago[1:] - 1
    where_ = torch.where(last >= 0, first[:, None] + last, n + torch.arange(c["nseq"], device="cuda")[:, None] * (K - 1) + last + K - 1)
    s["states"][slots] = table[where_]
    return dict(y=s["y"], states=s["states"])


def _plain_scan(s, c):
    """Chunks of 64 steps side by side; what each hands on to the later ones is weighted by the decay between them."""
    inner, bc, channels = _columns(c)
    S, H, P, N, G = c["nseq"], c["heads"], c["headdim"], c["dstate"], c["groups"]
    acc, slots = ACC[c["dtype"]], s["slots"].long()
    rows, live, lens = _padded(s)
    nc = rows.shape[1] // CHUNK
    shape = lambda v, *tail: torch.where(live[:, :, None], v[rows].to(acc), 0).reshape(S, nc, CHUNK, *tail)
    raw = s["zx"][:, inner + channels:].to(acc) + s["dt_bias"]
    dt = shape(torch.where(raw > 20, raw, torch.log1p(torch.exp(raw))), H).permute(0, 1, 3, 2)                       # [S, c, H, q]
    x = shape(s["xbc"][:, :inner], H, P).permute(0, 1, 3, 2, 4) * dt[..., None]                                      # [S, c, H, q, P]
    B = shape(s["xbc"][:, inner:inner + bc], G, N).permute(0, 1, 3, 2, 4).repeat_interleave(H // G, 2)
    C = shape(s["xbc"][:, inner + bc:], G, N).permute(0, 1, 3, 2, 4).repeat_interleave(H // G, 2)
    cum = torch.cumsum(dt.double() * -torch.exp(s["A_log"].double())[:, None], 3)
    below = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device="cuda").tril()
    decay = torch.exp((cum[..., :, None] - cum[..., None, :]).masked_fill_(~below, -math.inf)).to(acc)
    y = (torch.matmul(C, B.transpose(-1, -2)) * decay) @ x
    made = (x * torch.exp(cum[..., -1:] - cum).to(acc)[..., None]).transpose(-1, -2) @ B                             # [S, c, H, P, N]
    total = torch.nn.functional.pad(torch.cumsum(cum[..., -1], 1), (0, 0, 1, 0)).permute(0, 2, 1)                    # [S, H, c + 1]
    later = torch.ones(nc + 1, nc + 1, dtype=torch.bool, device="cuda").tril()
    across = torch.exp((total[..., :, None] - total[..., None, :]).masked_fill_(~later, -math.inf)).to(acc)
    begin = s["states"][slots] * s["resume"][:, None, None, None].to(acc)
    made = torch.cat([begin[:, None], made], 1).permute(0, 2, 1, 3, 4).reshape(S, H, nc + 1, P * N)
    had = (across @ made).reshape(S, H, nc + 1, P, N).transpose(1, 2)
    y = y + torch.matmul(C * torch.exp(cum).to(acc)[..., None], had[:, :-1].transpose(-1, -2))
    s["y"][rows[live]] = y.permute(0, 1, 3, 2, 4).reshape(S, nc * CHUNK, inner)[live].to(s["y"].dtype)
    s["states"][slots] = had[:, -1]
    return dict(y=s["y"], states=s["states"])


def _plain_step(s, c):
    inner, bc, channels = _columns(c)
    S, H, P, N, G = c["nseq"], c["heads"], c["headdim"], c["dstate"], c["groups"]
    acc, slots = ACC[c["dtype"]], s["slots"].long()
    raw = s["zx"][:, inner + channels:].to(acc) + s["dt_bias"]
    dt = torch.where(raw > 20, raw, torch.log1p(torch.exp(raw)))
    x = s["xbc"][:, :inner].to(acc).reshape(S, H, P, 1) * dt[..., None, None]
    B, C = (v.to(acc).reshape(S, G, 1, N).repeat_interleave(H // G, 1) for v in (s["xbc"][:, inner:inner + bc], s["xbc"][:, inner + bc:]))
    state = s["states"][slots] * torch.exp(dt * -torch.exp(s["A_log"]))[..., None, None] + x * B
    s["states"][slots] = state
    s["y"].copy_((state * C).sum(-1).reshape(S, inner))
    return dict(y=s["y"], states=s["states"])


def _plain_select(s, c):
    """Within a beam by the logit (equal ones: the lowest token), between beams by the score (equal ones: the lowest beam).  A finished beam
    goes on with the end token alone; where a row's probabilities are no numbers, or its score is, nothing of it is possible."""
    batch, beams, picks, vocab, eos = c["batch"], c["beams"], c["picks"], c["vocab"], s["eos"]
    logits = s["logits"].reshape(batch * beams, vocab)
    wide = logits.double()
    top = wide.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(wide - top).sum(1, keepdim=True))
    had = s["scores"].double().reshape(-1, 1)
    only = torch.full((vocab,), -math.inf, dtype=torch.float64, device="cuda")
    only[eos] = 0
    done = s["finished"].reshape(-1, 1) != 0
    rank = torch.where(done, only, wide)
    score = had + torch.where(done, only, wide - lse)
    never = torch.isnan(had) | (had == -math.inf) | ~done & ~torch.isfinite(lse)
    rank, score = rank.masked_fill(never, 0), score.masked_fill(never, -math.inf)
    order = torch.sort(rank, dim=1, descending=True, stable=True)[1][:, :picks]
    best, at = torch.sort(score.gather(1, order).reshape(batch, beams * picks), dim=1, descending=True, stable=True)
    at = at[:, :picks]
    s["parents"].copy_(at // picks)
    s["tokens"].copy_(order.reshape(batch, beams * picks).gather(1, at))
    s["next_scores"].copy_(best[:, :picks])
    s["next_finished"].copy_((s["finished"].gather(1, at // picks) != 0) | (s["tokens"] == eos))
    return {k: s[k] for k in ("next_scores", "parents", "tokens", "next_finished")}


def _plain_reorder(s, c):
    batch, beams = c["batch"], c["beams"]
    slots = s["slots"].long().reshape(batch, beams)
    s["states"][:, slots.reshape(-1)] = s["states"][:, slots.gather(1, s["parents"].long()).reshape(-1)]
    return dict(states=s["states"])


# --------------------------------------------------------------------------------------------------------------
# one pass: the framework's launchers
# --------------------------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _stream():
    """The program's stream, opened once."""
    import metaphor_b200 as mp
    return mp.Stream()


def _scratch(s, nbytes):
    """The program's workspace, kept with its buffers."""
    if "scratch" not in s:
        s["scratch"] = torch.empty(max(16, nbytes), dtype=torch.uint8, device="cuda")
    return s["scratch"]


def _own_conv(s, c):
    import metaphor_b200 as mp
    inner, bc, channels = _columns(c)
    x = s["zx"].data_ptr() + inner * SIZE[c["dtype"]]
    if c["form"] == "token":
        mp.launch("causal_conv1d_silu_token", DTYPES[c["dtype"]], x, s["zx"].stride(0), s["w"], s["bias"], s["states"], s["slots"], s["y"], channels,
                  c["nseq"], s["nslots"], channels, c["width"], _stream())
    else:
        mp.launch("causal_conv1d_silu_prompt", DTYPES[c["dtype"]], x, s["zx"].stride(0), s["w"], s["bias"], s["states"], s["slots"], s["resume"], s["starts"],
                  s["y"], channels, c["nseq"], s["rows"], s["nslots"], channels, c["width"], _stream())
    return dict(y=s["y"], states=s["states"])


def _own_scan(s, c):
    import metaphor_b200 as mp
    inner, bc, channels = _columns(c)
    size, st = SIZE[c["dtype"]], _stream()
    x = s["xbc"].data_ptr()
    raw = s["zx"].data_ptr() + (inner + channels) * size
    shape = (c["heads"], c["headdim"], c["dstate"], c["groups"])
    ins = (x, channels, raw, s["zx"].stride(0), s["dt_bias"], s["A_log"], x + inner * size, x + (inner + bc) * size, channels, s["states"], s["slots"])
    if c["form"] == "token":
        mp.launch("ssd_scan_token", DTYPES[c["dtype"]], *ins, s["y"], inner, c["nseq"], s["nslots"], *shape, st)
    else:
        scratch = _scratch(s, mp.lib().mpSsdScanPromptScratchBytes(tuple(SIZE).index(c["dtype"]), c["nseq"], s["rows"], *shape))
        mp.launch("ssd_scan_prompt", DTYPES[c["dtype"]], *ins, s["resume"], s["starts"], s["y"], inner, scratch, c["nseq"], s["rows"], s["nslots"], *shape, st)
    return dict(y=s["y"], states=s["states"])


def _own_select(s, c):
    import metaphor_b200 as mp
    dims = (c["batch"], c["beams"], c["vocab"], c["picks"])
    scratch = _scratch(s, mp.lib().mpBeamSelectScratchBytes(tuple(SIZE).index(c["dtype"]), *dims))
    mp.launch("beam_select", DTYPES[c["dtype"]], s["logits"], c["vocab"], s["scores"], s["finished"], s["eos"], s["next_scores"], s["parents"], s["tokens"],
              s["next_finished"], scratch, *dims, _stream())
    return {k: s[k] for k in ("next_scores", "parents", "tokens", "next_finished")}


def _own_reorder(s, c):
    import metaphor_b200 as mp
    mp.launch("reorder_states", DTYPES[c["dtype"]], s["states"], s["slots"], s["parents"], c["layers"], c["batch"], c["beams"], s["nslots"], c["row"], _stream())
    return dict(states=s["states"])


def run(state):
    c = state["case"]
    if own:
        return globals()["_own_" + c["kind"]](state, c)
    return globals()["_plain_step" if c["kind"] == "scan" and c["form"] == "token" else "_plain_" + c["kind"]](state, c)


# --------------------------------------------------------------------------------------------------------------
# the work that a pass cannot do without, and its results in 64 bits
# --------------------------------------------------------------------------------------------------------------
def work(case):
    c, e, a = case, SIZE[case["dtype"]], ACC_SIZE[case["dtype"]]
    if c["kind"] in ("conv", "scan"):
        inner, bc, channels = _columns(c)
        rows, read, n = sum(_lengths(c)), sum(_resumes(c)), c["nseq"]
        if c["kind"] == "conv":
            state = (c["width"] - 1) * channels * e
            return dict(bytes=e * (2 * rows * channels + channels * (c["width"] + 1)) + state * (read + n), flops=rows * channels * (2 * c["width"] + 5))
        state = inner * c["dstate"]
        # per step and state element: the decay, the outer product's multiply and add, the output's multiply and add
        return dict(bytes=e * rows * (inner + channels + c["heads"]) + state * a * (read + n), flops=5 * rows * state)
    if c["kind"] == "select":
        rows = c["batch"] * c["beams"]
        return dict(bytes=e * rows * c["vocab"] + rows * (a + 4) + c["batch"] * c["picks"] * (a + 12), flops=4 * rows * c["vocab"])
    moving = c["batch"] - c["batch"] // 4
    return dict(bytes=c["layers"] * moving * c["row"] * e * (c["sources"] + c["beams"]) + 8 * c["batch"] * c["beams"], flops=0)


def _sequence_rows(s):
    first = s["starts"].tolist()
    return [(i, first[i], first[i + 1], int(slot), bool(go)) for i, (slot, go) in enumerate(zip(s["slots"].tolist(), s["resume"].tolist()))]


def _exact_conv(s, c):
    """Sequence by sequence, over the kept inputs and the new ones in a row."""
    inner, bc, channels = _columns(c)
    K, w = c["width"], s["w"].double()
    y, states = torch.zeros(s["rows"], channels, dtype=torch.float64, device="cuda"), s["states"].double()
    for i, lo, hi, slot, go in _sequence_rows(s):
        line = torch.cat([states[slot] if go else torch.zeros_like(states[slot]), s["zx"][lo:hi, inner:inner + channels].double()])
        pre = s["bias"].double() + sum(w[:, k] * line[k:k + hi - lo] for k in range(K))
        y[lo:hi] = pre / (1 + torch.exp(-pre))
        states[slot] = line[line.shape[0] - (K - 1):]
    return dict(y=y, states=states)


def _exact_scan(s, c):
    """The recurrence, step by step, every sequence that still has one at once."""
    inner, bc, channels = _columns(c)
    H, P, N, G = c["heads"], c["headdim"], c["dstate"], c["groups"]
    per_step = c["nseq"] * H * P * N * 8 * 8 / 4e12 + 1e-4
    if per_step * c["longest"] > 15:
        return None
    f = torch.float64
    A = -torch.exp(s["A_log"].to(f))
    dt = torch.nn.functional.softplus(s["zx"][:, inner + channels:].to(f) + s["dt_bias"].to(f), threshold=1000)
    x, B, C = s["xbc"][:, :inner].to(f), s["xbc"][:, inner:inner + bc].to(f), s["xbc"][:, inner + bc:].to(f)
    y, states = torch.zeros(s["rows"], inner, dtype=f, device="cuda"), s["states"].to(f)
    seqs = sorted(_sequence_rows(s), key=lambda q: q[1] - q[2])       # the longest first
    lens = [hi - lo for _, lo, hi, _, _ in seqs]
    where_ = torch.tensor([slot for _, _, _, slot, _ in seqs], device="cuda")
    lo = torch.tensor([q[1] for q in seqs], device="cuda")
    h = states[where_] * torch.tensor([float(q[4]) for q in seqs], dtype=f, device="cuda")[:, None, None, None]
    heads_of = lambda v: v.reshape(-1, G, 1, N).expand(-1, G, H // G, N).reshape(-1, H, 1, N)
    for t in range(max(lens)):
        n = sum(1 for k in lens if k > t)
        r = lo[:n] + t
        d = dt[r][:, :, None, None]
        h[:n].mul_(torch.exp(d * A[:, None, None])).addcmul_(d * x[r].reshape(n, H, P, 1), heads_of(B[r]))
        y[r] = torch.matmul(h[:n], heads_of(C[r]).transpose(2, 3)).reshape(n, inner)
    states[where_] = h
    return dict(y=y, states=states)


def _exact_select(s, c):
    """Beam by beam in the order of the score; only the scores are compared as numbers, so they are what is given."""
    f = torch.float64
    logp = torch.log_softmax(s["logits"].to(f), 1).reshape(c["batch"], c["beams"], c["vocab"])
    done = s["finished"] != 0
    logp[done] = -math.inf
    logp[..., s["eos"]] = torch.where(done, 0.0, logp[..., s["eos"]])
    total = torch.nan_to_num(s["scores"].to(f)[..., None] + logp, nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    return dict(next_scores=total.flatten(1).topk(c["picks"], 1)[0], parents=None, tokens=None, next_finished=None)


def _exact_reorder(s, c):
    states, slots = s["states"].double(), s["slots"].tolist()
    new = states.clone()
    for b, row in enumerate(s["parents"].tolist()):
        for j, p in enumerate(row):
            new[:, slots[b * c["beams"] + j]] = states[:, slots[b * c["beams"] + p]]
    return dict(states=new)


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](prepare(case, seed), case)
