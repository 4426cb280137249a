"""The order between a generator's stream and torch's: on the CPU with streams that write down what is asked of them, on the device beside work of
torch's that is still running."""
import numpy as np
import pytest

from metaphor_b200.generate import Generator
from metaphor_b200.mamba_lm import LMConfig, init_weights

CFG = LMConfig(d_model=64, n_layer=1, vocab=101, chunk=128)


class TorchStream:
    def __init__(self, name, log):
        self.name, self.log = name, log

    def wait_stream(self, other):
        self.log.append(f"{self.name} waits for {other.name}")

    def synchronize(self):
        self.log.append(f"{self.name} done")


class OwnStream:
    def __init__(self, log):
        self.log, self.inner = log, TorchStream("own", log)

    def torch_stream(self):
        return self.inner

    def sync(self):
        self.log.append("own done")


@pytest.fixture
def bare(monkeypatch):
    import torch
    log = []
    current = TorchStream("torch", log)
    real = torch.empty

    def empty(*size, device=None, **more):
        log.append("allocate")
        return real(*size, **more)
    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: current)
    g = Generator.__new__(Generator)
    g.cfg, g.sequences, g.max_rows, g.stream, g.scratch = CFG, 4, 10, OwnStream(log), None
    g._graph, g._graph_of = None, None
    g.logits, g.last = torch.zeros(4, 1), torch.zeros(4, 1)
    g.ids = g.starts = g.slots = g.last_rows = None
    g._upload = lambda dst, values: log.append("launch")
    g._layers = lambda *a: log.append("launch")
    g._head = lambda *a: log.append("launch")
    g._L = lambda *a: log.append("launch")
    g._lib = type("Lib", (), {"mpSsdScanPromptScratchBytes": staticmethod(lambda *a: 256)})
    return g, log


def test_scratch_waits_for_torch(bare):
    """Memory that torch frees on its stream can be handed out before the kernels there are done with it."""
    g, log = bare
    g._room(100)
    assert log == ["own done", "allocate", "torch done"]
    g._room(50)
    assert len(log) == 3 and g.scratch.numel() == 100
    g._room(101)
    assert log[3:] == ["own done", "allocate", "torch done"]


def ordered(log):
    launches = [k for k, what in enumerate(log) if what == "launch"]
    assert "own waits for torch" in log[:launches[0]], log
    assert "torch waits for own" in log[launches[-1]:], log
    if "allocate" in log:
        k = log.index("allocate")
        assert log[k + 1] == "torch done", log


def test_prompt_takes_its_turn(bare):
    g, log = bare
    g.prompt([[1, 2], [3]])
    ordered(log)


def test_token_takes_its_turn(bare):
    g, log = bare

    class Tokens:      # of a device tensor, what is looked at
        import torch
        dtype, is_cuda = torch.int32, True

        def numel(self):
            return 2

        def is_contiguous(self):
            return True
    g.token(Tokens())
    ordered(log)


@pytest.mark.gpu
def test_beside_torch(mp):
    """Nothing is synchronised by hand: tokens and scratch come behind late work of torch's, logits are read by its next operation."""
    import torch
    w = init_weights(CFG, seed=3)
    r = np.random.default_rng(1)
    prompts = [[int(v) for v in r.integers(0, CFG.vocab, n)] for n in (900, 30)]
    quiet, late = Generator(CFG, w, 2, 1000), Generator(CFG, w, 2, 1000)
    want = []
    want.append(quiet.prompt(prompts).clone())
    ids = torch.tensor([5, 7], dtype=torch.int32, device="cuda")
    for _ in range(2):
        torch.cuda.synchronize()
        want.append(quiet.token(ids).clone())
        torch.cuda.synchronize()
    nbytes = quiet.scratch.numel()
    torch.cuda.synchronize()
    temporary = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    torch.cuda._sleep(20_000_000)                     # ten milliseconds
    total = temporary.fill_(3).sum(dtype=torch.int64)
    del temporary                                     # (torch may give this memory out as scratch)
    got = [late.prompt(prompts).clone()]
    for _ in range(2):
        torch.cuda._sleep(20_000_000)
        now = ids + 0
        logits = late.token(now)
        del now
        filler = torch.full((2,), CFG.vocab - 1, dtype=torch.int32, device="cuda")      # (where the tokens were, if torch likes)
        got.append(logits.clone())
        del filler
    torch.cuda.synchronize()
    assert int(total) == 3 * nbytes
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    quiet.release(); late.release()
