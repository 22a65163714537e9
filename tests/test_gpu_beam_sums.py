"""Sums of weights of the choice over beams and vocabulary, to the bits that ordinary rows have."""
import math

import pytest
import torch

from test_gpu_beams import K, _agree, _best, _select  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", ["ordinary", "a word is no number", "large"])
def test_sums_of_long_flat_rows(K, what):  # noqa: F811
    """Rows of 50,021 nearly equal weights, 196 a thread: summed in 32 bits one after the other they would be off by up to 3e-6.  The running
    score makes up for the log-sum, so that a score's own rounding is small.  Bound: a weight is off by its 2 ulp (2^-22) and by its
    argument's rounding (below 2 in size: 2^-24, times log 2), sixteen of them are added in 32 bits in five rounded steps (2^-24 each), all
    else is 64-bit; together below 10 * 2^-24.  The score is rounded once."""
    rows, vocab, picks = 200, 50021, 8
    level = torch.linspace(-0.7, 0.7, rows, device="cuda")
    if what == "large":                                    # one word 0.7 above the others, far beyond 65,536
        logits = (70000.0 + torch.arange(rows, device="cuda"))[:, None].repeat(1, vocab)
        logits[:, 1:] -= 0.703125
    else:
        logits = level[:, None].repeat(1, vocab)
    if what == "a word is no number":
        logits[:, 4000] = math.nan
    scores = torch.full((rows,), math.log(vocab), device="cuda")
    got, want = _select(K, logits, scores, 1, picks), _best(logits.cpu().numpy(), scores.cpu().numpy(), 1, picks)
    _agree(got, want, vocab)
    assert (abs(got[0] - want[0]) <= 2.0 ** -24 * abs(want[0]) + 10 * 2.0 ** -24).all()


@pytest.mark.parametrize("top", [65537.0, 65540.0, 65600.0])
def test_rows_with_slices_on_both_sides_of_what_is_large(K, top):  # noqa: F811
    """Weights are summed by differences in the slices whose largest logit is beyond 65,536 and by powers of two in the others; a row's
    continuations hang on both."""
    vocab = 40000
    logits = torch.full((6, vocab), -100.0, device="cuda")
    for r in range(6):
        logits[r, 5 + r] = top
        logits[r, 39000 - 5000 * r] = 65536.0 - r / 128
    scores = torch.zeros(6, device="cuda")
    _agree(_select(K, logits, scores, 3, 6), _best(logits.cpu().numpy(), scores.cpu().numpy(), 3, 6), vocab)
