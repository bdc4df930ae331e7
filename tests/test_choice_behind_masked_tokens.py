"""The choice of tokens where a vocabulary's first tokens are masked: many rows of a long vocabulary, each read by one block in batches of 16,384 tokens."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_answers_of_one_prompt import call_choice, ops, plain_choice  # noqa: F401  (ops: the fixture)

VOCAB, ROWS = 128256, 160   # more rows than a B200 has SMs: a block of its own to each
TOP_K = (2, 50, 200, 201, 300, 512)


def masked_rows(first: int, masked: float):
    """Rows whose first ``first`` tokens are masked; of some, few tokens behind these are left in a batch or two, and of some everything up to the last tokens is masked."""
    g = torch.Generator().manual_seed(first)
    logits = torch.randn(ROWS, VOCAB, generator=g) * 3
    logits[:, :first] = masked
    logits[3::8, first + 10 : 90000] = masked
    logits[5::8, : VOCAB - 700] = masked
    logits[7::8, : VOCAB - 1] = masked
    options = [(0.9 + 0.1 * (r % 3), TOP_K[r % len(TOP_K)], 0.9 if r % 4 < 2 else 1.0, 0.0) for r in range(ROWS)]
    return logits, options, torch.rand(ROWS, generator=g).tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("masked", [-float("inf"), float("nan")], ids=["minus infinity", "nan"])
@pytest.mark.parametrize("first", [16383, 16384, 20000, 40000, 70000])
def test_top_k_behind_masked_tokens(ops, first, masked):  # noqa: F811
    logits, options, uniforms = masked_rows(first, masked)
    columns = [list(c) for c in zip(*options)]
    logits = logits.cuda()
    together = call_choice(ops, logits, *columns, uniforms)
    for at in range(0, ROWS, 20):   # the same rows in clusters of blocks
        assert call_choice(ops, logits[at : at + 20], *[c[at : at + 20] for c in columns], uniforms[at : at + 20]) == together[at : at + 20]
    checked = 0
    for r in range(first % 7, ROWS, 7):
        want, _, close = plain_choice(logits[r].cpu(), *[float(np.float32(x)) if i != 1 else x for i, x in enumerate(options[r])], float(np.float32(uniforms[r])))
        if not close:
            assert together[r] == want, (r, options[r], uniforms[r])
            checked += 1
    assert checked >= 16
