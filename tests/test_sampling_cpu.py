"""Sampling settings, their random numbers, and the engine that passes them to its model, without a GPU."""
import numpy as np
import pytest
import torch

from tlaloc_b200 import __main__ as cli
from tlaloc_b200.engine import Engine
from tlaloc_b200.paging import PADDING_PAGE
from tlaloc_b200.sampling import Sampling, pack
from tlaloc_b200.step_model import StepModel


@pytest.mark.parametrize("wrong", [dict(temperature=-0.1), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_k=-1), dict(top_k=1.5), dict(top_k=2**31),
                                   dict(top_p=-0.1), dict(top_p=1.1), dict(top_p=float("nan")), dict(min_p=2), dict(min_p=float("nan")), dict(seed=2**64), dict(seed=0.5)])
def test_settings_out_of_range(wrong):
    with pytest.raises(ValueError, match=f"sampling: {list(wrong)[0]} is"):
        Sampling(**wrong)


def test_uniforms():
    """Numbers of f32 in [0, 1), the same for the same seed and index, spread evenly: of 4096 draws a sixteenth falls into each sixteenth, by five standard deviations
    (of the binomial count, sqrt(4096 / 16 * 15 / 16) = 15.5)."""
    draws = np.array([[Sampling(seed=s).uniform(i) for i in range(64)] for s in range(64)])
    assert (draws >= 0).all() and (draws < 1).all() and (draws.astype(np.float32) == draws).all()
    assert len(np.unique(draws)) > 4090  # of 2^24 values: a half pair in common is expected
    assert (np.abs(np.histogram(draws, 16, (0, 1))[0] - 256) < 78).all()
    assert Sampling(seed=3).uniform(5) == Sampling(seed=3, top_k=9).uniform(5) == draws[3, 5]
    assert Sampling(seed=-1).uniform(0) == Sampling(seed=2**64 - 1).uniform(0)


def test_packed_settings():
    some = Sampling(0.7, 50, 0.9, 0.05, seed=4)
    packed = pack([(some, 3), (None, 8)])
    assert packed.dtype == np.int32 and packed.shape == (5, 2)
    assert packed[:4, 0].view(np.float32).tolist() == np.array([some.uniform(3), 0.7, 0.9, 0.05], np.float32).tolist() and packed[4].tolist() == [50, 0]
    assert packed[1:4, 1].view(np.float32).tolist() == [0, 1, 0]
    assert pack([]).shape == (5, 0)


class Counter(StepModel):
    """Logits say how many tokens a sequence has; a draw answers with a function of that, its seed and its index."""

    def __init__(self, blocks=9):
        super().__init__(16, 4, blocks, 8, 4, 1000, "cpu")
        self.drawn, self.greedy_rows = [], 0

    def run(self, step, want):
        assert step.slot_mapping.min() >= self.block_size * (PADDING_PAGE + 1)
        return torch.tensor([[float(step.seq_lens[r])] for r in want])

    def greedy(self, logits):
        self.greedy_rows += len(logits)
        return logits[:, 0].int()

    def sample(self, logits, draws):
        assert len(draws) == len(logits)
        self.drawn += draws
        return torch.tensor([int(x) if s is None else (int(x) + int(s.uniform(i) * 500)) for x, (s, i) in zip(logits[:, 0].tolist(), draws)])

    def device_status(self):
        return 0


PROMPTS = [[1, 2, 3], list(range(17)), [4], list(range(9)), [5] * 20]


def expected(prompt, n, s):
    return [len(prompt) + i + (int(s.uniform(i) * 500) if s else 0) for i in range(n)]


@pytest.mark.parametrize("blocks", [9, 12, 40])
def test_draws_follow_seed_and_index_alone(blocks):
    """Whatever runs together, and however often a request is sent back for its pages."""
    model = Counter(blocks)
    out = Engine(model).generate(PROMPTS, 9, sampling=Sampling(0.5, seed=2**64 - 2))
    assert out == [expected(p, 9, Sampling(seed=(2**64 - 2 + i) % 2**64)) for i, p in enumerate(PROMPTS)]
    assert model.greedy_rows == 0 and all(s.temperature == 0.5 for s, _ in model.drawn) and len(model.drawn) == 45


def test_settings_of_each_prompt():
    each = [Sampling(0.5, seed=1), None, Sampling(1.0, 5, seed=1), None, Sampling(0.0)]
    model = Counter(40)
    out = Engine(model).generate(PROMPTS, 6, sampling=each)
    assert out == [expected(p, 6, s) for p, s in zip(PROMPTS, each)]
    with pytest.raises(ValueError, match="1 sampling settings for 5 prompts"):
        Engine(model).generate(PROMPTS, 6, sampling=each[:1])


def test_without_settings_every_token_is_greedy():
    model = Counter(40)
    assert Engine(model).generate(iter(PROMPTS), 4) == [expected(p, 4, None) for p in PROMPTS]
    assert model.drawn == [] and model.greedy_rows == 20


def test_command_line_refuses_settings_out_of_range(capsys):
    with pytest.raises(SystemExit):
        cli.main(["generate", "--model", "nowhere", "--prompt", "1,2", "--temperature", "0.5", "--top-p", "1.5"])
    assert "top_p is in [0, 1], not 1.5" in capsys.readouterr().err


def test_a_vocabulary_split_over_ranks_is_not_sampled():
    from tlaloc_b200.decoder import Decoder

    part = Decoder.__new__(Decoder)
    part.world = 2
    with pytest.raises(NotImplementedError, match="its part of the vocabulary"):
        part.sample(torch.zeros(1, 8), [(Sampling(), 0)])
