"""The operators around the 4-bit cache at the ends of their ranges, against their definitions in 64 bits (ref_serve.py): temperatures, rows that are alike, tables and groups that end early."""

import numpy as np
import pytest

from test_gpu_serve import TYPES, drafted, verify

pytestmark = pytest.mark.gpu


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
