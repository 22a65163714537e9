"""Length penalties that a search can count with."""
import math

import pytest

from rustinfer_b200.engine.beam import BeamParams, _Search


@pytest.mark.parametrize("penalty,max_tokens", [(300.0, 16), (-300.0, 16), (1e308, 2), (-1e308, 2), (80.0, 4096)])
def test_penalties_that_leave_the_range_of_64_bits_are_refused(penalty, max_tokens):
    with pytest.raises(ValueError, match="length_penalty"):
        BeamParams(length_penalty=penalty, max_tokens=max_tokens).validate()


@pytest.mark.parametrize("penalty,max_tokens", [(216.0, 16), (-216.0, 16), (70.0, 4096), (1e308, 1), (-3.0, 100000)])
def test_hypotheses_of_every_length_are_worth_a_finite_number(penalty, max_tokens):
    p = BeamParams(beams=1, length_penalty=penalty, max_tokens=max_tokens)
    p.validate()
    for n in sorted({1, 2, max_tokens // 2, max_tokens} & set(range(1, max_tokens + 1))):
        s = _Search([0], max_tokens, tokens=[[5] * (n - 1)], scores=[-2.0 * n])
        s.advance([(-2.0 * n, 0, 9)], p, {9})
        assert s.ended and math.isfinite(s.ended[0].score) and s.ended[0].score < 0
        s = _Search([0], max_tokens, tokens=[[5] * (n - 1)], scores=[-2.0 * n])
        s.advance([(-2.0 * n, 0, 5)], p, {9})
        assert len(s.tokens[0]) == n
