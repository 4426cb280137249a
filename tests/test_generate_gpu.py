"""Answers with a Mamba-2 language model: scores of greedy and beam search against the float64 statement of the model on the sequences that were
found, and states that go on against prompts taken in at once."""
import numpy as np
import pytest

from metaphor_b200.generate import Generator, load_weights
from metaphor_b200.mamba_lm import LMConfig, MambaLM, init_weights

pytestmark = pytest.mark.gpu
CFG = LMConfig(d_model=128, n_layer=2, vocab=499, chunk=128)
TOL = 1e-2       # r16 activations against float64, relative: the tolerance of the training step's loss


@pytest.fixture(scope="module")
def weights():
    w = init_weights(CFG, seed=5)
    w["embedding"] *= 5       # logits of a spread of about one: a wrong state shows in the scores
    return w


def log_prob(w, prompt, line):
    """log p(line | prompt) in float64, with the weights as the contractions see them."""
    import torch
    from oracle import lm_oracle
    wt = {k: torch.tensor((v if k.split(".")[-1] in ("dt_bias", "A_log", "D") else v.astype(np.float16)).astype(np.float64)) for k, v in w.items()}

    def total(ids):
        if len(ids) < 2:
            return 0.0
        t = torch.tensor(ids, dtype=torch.int64)
        return -float(lm_oracle.forward_loss(CFG, wt, t[:-1], t[1:], 1, len(ids) - 1)) * (len(ids) - 1)
    return total(list(prompt) + list(line)) - total(list(prompt))


@pytest.fixture(scope="module")
def prompts():
    r = np.random.default_rng(7)
    return [[int(v) for v in r.integers(0, CFG.vocab, n)] for n in (1, 37, 5, 150)]


def test_greedy(mp, stream, weights, prompts):
    g = Generator(CFG, weights, sequences=6, max_rows=256, stream=stream)
    found = g.search(prompts, 7)
    again = g.search(prompts, 7)          # the graph of the first call, other states before it
    assert found == again and stream.status() == 0
    for p, ((line, score),) in zip(prompts, found):
        want = log_prob(weights, p, line)
        assert len(line) == 7 and abs(score - want) <= TOL * abs(want), (len(p), score, want)
    alone = g.search([prompts[3]], 7)[0][0]      # without the others beside it: the same but for the order of sums in other tiles
    assert abs(alone[1] - found[3][0][1]) <= TOL * abs(alone[1])
    g.release()


@pytest.mark.parametrize("beams,eos", [(3, None), (4, 17), (2, 17)])
def test_beams(mp, stream, weights, prompts, beams, eos):
    g = Generator(CFG, weights, sequences=len(prompts) * beams + 1, max_rows=256, stream=stream)
    for p, lines in zip(prompts, g.search(prompts, 6, beams=beams, eos=eos)):
        assert len(lines) == beams and len({tuple(line) for line, _ in lines}) == beams
        scores = [s for _, s in lines]
        assert scores == sorted(scores, reverse=True)
        for line, score in lines:
            want = log_prob(weights, p, line)
            assert (len(line) == 6 or line[-1] == eos) and (eos is None or eos not in line[:-1])
            assert abs(score - want) <= TOL * abs(want), (len(p), line, score, want)
    g.release()


def test_the_end_ends(mp, stream, weights, prompts):
    """Every first token is the end in one search or another: found with its own probability, and nothing behind it."""
    g = Generator(CFG, weights, sequences=4, max_rows=256, stream=stream)
    first = g.search([prompts[1]], 1, beams=4)[0]
    for token, score in ((line[0], s) for line, s in first):
        lines = dict((tuple(line), s) for line, s in g.search([prompts[1]], 5, beams=4, eos=token)[0])
        if (token,) in lines:      # (it may have been overtaken by longer ones that are better: only scores below are possible behind it)
            assert abs(lines[(token,)] - score) <= 1e-5 * abs(score)
    assert tuple(first[0][0]) in {tuple(line) for line, _ in g.search([prompts[1]], 5, beams=4, eos=first[0][0][0])[0]}
    g.release()


def test_tokens_go_on_where_a_prompt_ends(mp, stream, weights, prompts):
    import torch
    g = Generator(CFG, weights, sequences=3, max_rows=256, stream=stream)
    whole = [prompts[1], prompts[3][:140]]
    cut = 4
    at_once = g.prompt(whole)
    stream.sync()
    at_once = at_once.float().cpu().numpy()
    g.prompt([p[:-cut] for p in whole])
    for k in range(cut, 0, -1):
        ids = torch.tensor([p[-k] for p in whole], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        logits = g.token(ids)
        stream.sync()
    assert np.abs(logits.float().cpu().numpy() - at_once).max() <= TOL * np.abs(at_once).max()
    g.release()


def test_a_trained_model_and_its_checkpoint(mp, stream, prompts, tmp_path):
    """A model's own buffers, after a step, and the weights of its checkpoint: the same answers."""
    import torch
    m = MambaLM(CFG, 1, 128, stream=stream, loss_scale=64.0)
    r = np.random.default_rng(2)
    m.set_batch(*(torch.from_numpy(r.integers(0, CFG.vocab, 128).astype(np.int32)) for _ in range(2)))
    m.train_step(lr=1e-2)
    m.save(str(tmp_path / "m"))
    a, b = Generator(CFG, m, 4, 256), Generator(CFG, load_weights(CFG, str(tmp_path / "m")), 4, 256, stream=stream)
    assert a.search(prompts, 4) == b.search(prompts, 4)
    a.release(); b.release(); m.release()
