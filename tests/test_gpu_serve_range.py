"""The operators around the 4-bit cache at the ends of their ranges, against their definitions in 64 bits (ref_serve.py): temperatures, rows that are alike, tables and groups that end early."""

import numpy as np
import pytest

import ref_serve as V
from test_gpu_serve import TYPES, drafted, verify

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def weights_that_count_as_nothing(monkeypatch):
    """Weights below 2^-960 of a row's largest count as 0, where numbers of 64 bits go on to 2^-1074: at temperatures as small as here's that is what all others of a row have."""
    full = V.softmax

    def softmax(x, t):
        w = full(x, t)
        if w is None:
            return None
        w = np.where(w < 2.0 ** -960 * w.max(), 0.0, w)
        return w / w.sum()

    monkeypatch.setattr(V, "softmax", softmax)


@pytest.mark.parametrize("with_draft", [True, False])
def test_tokens_without_weight_are_not_accepted(lib, cuda, with_draft):
    """A drafted token so far below the largest logit of both models that it has no weight in either: 0 < 0 is false, whatever u."""
    rng = np.random.default_rng(72)
    drafts, vocab = [1] * 24, 4001
    target, draft, _, u, v = drafted(rng, "f32", vocab, drafts)
    tokens = rng.integers(0, vocab, 24).astype(np.int32)
    target[2 * np.arange(24), tokens], draft[np.arange(24), tokens] = -30.0, -30.0
    u[::4] = 0.0
    verify(lib, "f32", target, draft if with_draft else None, drafts, tokens, np.float32([40.0, 1e3, 1e4] * 8), u, v)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("vocab", [3, 900, 20001])
def test_rows_that_are_alike_leave_the_targets_weights(lib, cuda, type_, vocab):
    """Draft and target have equal rows, and the token cannot be accepted (none, outside of the vocabulary, masked in both): of max(p - q, 0) nothing is left, p is drawn from."""
    rng = np.random.default_rng(73)
    drafts = [1] * 48
    target, _, _, u, v = drafted(rng, type_, vocab, drafts)
    target[::6, 1] = -np.inf
    draft = target[::2].copy()
    tokens = np.array([1 if i % 3 == 0 else -1 if i % 3 == 1 else vocab + i for i in range(48)], dtype=np.int32)
    verify(lib, type_, target, draft, drafts, tokens, rng.choice([1.0, 0.7, 1.4], 48), u, v)
