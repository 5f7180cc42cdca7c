"""generate.score before anything reaches a device: a model that only keeps the book of its calls."""
from types import SimpleNamespace

import pytest
import torch

from flint_amd import generate


class Model:
    """Transformer's part in score, with a rope table of `block` positions."""

    def __init__(self, block=64, vocab=50):
        self.device = torch.device("cpu")
        self.config = SimpleNamespace(vocab_size=vocab, dim=16)
        self.packed = SimpleNamespace(rope=torch.zeros(block, 2))
        self.room, self.fed = 0, []

    def setup_caches(self, batch, length):
        length = (length + 7) // 8 * 8
        if length > self.packed.rope.shape[0]:
            raise ValueError("max_seq_length exceeds block_size (rope table)")
        self.room = max(self.room, length)

    def _feed(self, tokens, pos):
        assert pos + tokens.numel() <= self.room
        self.fed.append((pos, tokens.tolist()))

    def verify(self, tokens, pos, depth=None, amask=None, logits=None, feat=None, tokens_out=None):
        self._feed(tokens, pos)
        return None, torch.zeros(tokens.numel(), self.config.vocab_size), None

    def prefill_features(self, tokens, pos, token_out=None):
        self._feed(tokens, pos)
        return torch.zeros(tokens.numel(), self.config.dim)


@pytest.fixture
def given(monkeypatch):
    """What score asks log probabilities of."""
    asked = []

    def note(rows, tokens, top):
        asked.extend(tokens.tolist())
        return generate._logprob_outputs(rows.shape[0], tokens, top, rows.device)

    monkeypatch.setattr(generate, "logprobs", lambda logits, tokens, top: note(logits, tokens, top))
    monkeypatch.setattr(generate, "head_logprobs", lambda feat, w, s, tokens, top: note(feat, tokens, top))
    return asked


HEAD = SimpleNamespace(weight=torch.zeros(50, 16, dtype=torch.int8), scales=torch.ones(50))


@pytest.mark.parametrize("head", [None, HEAD])
@pytest.mark.parametrize("block,n", [(64, 2), (64, 33), (64, 64), (64, 65), (67, 65), (128, 65)])
def test_a_text_as_long_as_the_positions_allow(given, head, block, n):
    """The last token takes no position: a text of one token more than there are positions can be scored. Where there is
    one, the cache has room for the last token, so that decoding can go on from it."""
    model, tokens = Model(block), torch.arange(n)
    out = generate.score(model, tokens % 50, 0, head)
    assert out.logprob.shape == (n - 1,) and given == (tokens[1:] % 50).tolist()
    assert sum((t for _, t in model.fed), []) == (tokens[:-1] % 50).tolist()
    assert model.room >= min(n, block // 8 * 8)


@pytest.mark.parametrize("head", [None, HEAD])
def test_a_longer_text_is_refused(given, head):
    model = Model(64)
    with pytest.raises(ValueError):
        generate.score(model, torch.zeros(66, dtype=torch.int32), 0, head)
    assert model.fed == []


@pytest.mark.parametrize("head", [None, HEAD])
@pytest.mark.parametrize("top", [-1, 33, 51])
def test_alternatives_that_are_refused_are_refused_first(given, head, top):
    """Before the model has run, which takes the time of a prompt and overwrites its cache."""
    model = Model(64)
    with pytest.raises(ValueError):
        generate.score(model, torch.zeros(40, dtype=torch.int32), top, head)
    assert model.fed == [] and model.room == 0


@pytest.mark.parametrize("head", [None, HEAD])
def test_64_bit_ids_outside_the_vocabulary_stay_outside(given, head):
    """As in logprobs: an id beyond 32 bits is not the one that its low bits make."""
    model = Model(64)
    generate.score(model, torch.tensor([1, 2 ** 32 + 5, -2 ** 40, 3, 2 ** 33 + 7]), 0, head)
    fed = sum((t for _, t in model.fed), [])
    assert len(given) == 4 and len(fed) == 4
    outside = lambda t: not 0 <= t < 50  # noqa: E731
    assert [outside(t) for t in given] == [True, True, False, True]
    assert [outside(t) for t in fed] == [False, True, True, False]
