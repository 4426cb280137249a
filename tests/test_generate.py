"""What a generator refuses before anything reaches the device (no GPU needed)."""
import numpy as np
import pytest

from metaphor_b200.generate import Generator, load_weights
from metaphor_b200.mamba_lm import LMConfig, init_weights


def bare(sequences=4, max_rows=10):
    g = Generator.__new__(Generator)
    g.cfg, g.sequences, g.max_rows = LMConfig(d_model=64, n_layer=1, vocab=20), sequences, max_rows
    return g


@pytest.mark.parametrize("prompts,beams,what", [([], 1, "sequences"), ([[1]] * 5, 1, "sequences"), ([[1], [2]], 3, "sequences"), ([[1], []], 1, "at least one token"),
                                                ([[1] * 6, [2] * 5], 1, "buffers"), ([[1, 20]], 1, "whole numbers"), ([[-1]], 1, "whole numbers"),
                                                ([[0.5]], 1, "whole numbers"), ([[1]], 0, "beams"), ([[1]], 33, "beams")])
def test_prompts(prompts, beams, what):
    with pytest.raises(ValueError, match=what):
        bare()._check(prompts, beams)


def test_more_beams_than_tokens():
    with pytest.raises(ValueError, match="more beams"):
        bare(sequences=32)._check([[1]], 21)


@pytest.mark.parametrize("new_tokens,eos,what", [(0, None, "new token"), (3, 20, "eos"), (3, -1, "eos")])
def test_search_arguments(new_tokens, eos, what):
    with pytest.raises(ValueError, match=what):
        bare().search([[1]], new_tokens, eos=eos)


@pytest.mark.parametrize("sequences,rows,more", [(0, 5, {}), (2, 0, {}), (2, 5, dict(d_state=512)), (2, 5, dict(d_conv=5))])
def test_sizes(sequences, rows, more):
    with pytest.raises(ValueError):
        Generator(LMConfig(d_model=64, n_layer=1, vocab=20, **more), {}, sequences, rows)


def test_checkpoint_weights(tmp_path):
    cfg = LMConfig(d_model=64, n_layer=1, vocab=20)
    w = init_weights(cfg, seed=3)
    for idx, (name, _) in enumerate(cfg.param_shapes()):
        w[name].tofile(tmp_path / f"m_{idx}")
    got = load_weights(cfg, str(tmp_path / "m"))
    assert list(got) == [n for n, _ in cfg.param_shapes()] and all(np.array_equal(got[k], w[k]) for k in w)
    with pytest.raises(ValueError, match="expected"):
        load_weights(LMConfig(d_model=128, n_layer=1, vocab=20), str(tmp_path / "m"))
