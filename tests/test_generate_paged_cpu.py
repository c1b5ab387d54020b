"""generate_paged and score_paged around a cache and a model that are stand-ins (no GPU)."""
import pytest
import torch

from llama.generation import Generation

VOCAB = 11


class Letters:
    eos_id, pad_id = -1, 0

    def encode(self, text, bos, eos):
        return [1] * bool(bos) + [2 + ord(c) % 9 for c in text]

    def decode(self, tokens):
        return " ".join(map(str, tokens))


class Cache:
    def __init__(self, refused):
        self.refused = refused

    def append(self, new, n):
        return None

    def release(self, finished):
        pass

    def fork(self, parents):
        return torch.tensor([r != self.refused for r in range(parents.shape[0])])


class Model(Generation):
    def __init__(self, refused=None):
        super().__init__()
        self.refused = refused

    def paged_cache(self, pages, page_size, max_requests, max_len, bits):
        self.requests = max_requests
        return Cache(self.refused)

    def forward_paged(self, tokens, step, cache, max_new, whole_prompts=False):
        return torch.zeros(self.requests, VOCAB)


def test_a_refused_sample_is_an_error():
    args = (Letters(), ["ab", "c"], 3, 0.0, 1.0, "cpu")
    assert len(Model().generate_paged(*args, samples=3)) == 6
    with pytest.raises(RuntimeError, match="refused"):
        Model(refused=4).generate_paged(*args, samples=3)
    assert len(Model(refused=1).generate_paged(*args)) == 2  # (one answer per prompt forks nothing)


@pytest.mark.parametrize("rows", [0, -1, -1024])
def test_no_rows_of_logits(rows, monkeypatch):
    """(They gave results without log probabilities.)"""
    monkeypatch.setattr("llama.generation.hidden_paged", lambda *a, **k: torch.zeros(2, 4))
    with pytest.raises(ValueError, match="rows"):
        Model().score_paged(Letters(), ["a"], "cpu", rows=rows)
