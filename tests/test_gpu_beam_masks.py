"""The choice over beams and vocabulary where words are masked by large finite numbers, and where a row's weights are summed by
differences: against the formula in 64 bits, to the bound of the other rows."""
import pytest
import torch

from test_gpu_beams import K, _agree, _best, _select  # noqa: F401

pytestmark = pytest.mark.gpu

MASKS = [-f * 10.0 ** e for e in range(5, 39) for f in (1.0, 3.3)] + [-65504.0, -65536.0, -65537.0, torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min]


@pytest.mark.parametrize("vocab", [300, 5000, 50021])
@pytest.mark.parametrize("what", ["a few words left", "a tail", "half of all", "one thread's"])
def test_choice_among_words_masked_by_finite_numbers(K, vocab, what):  # noqa: F811
    """A row for every mask, each beside a row without one: the words left are chosen by the scores that they have without the masked ones.
    (No more picks than words are left, so that none of equal -1e30 is to be put in order.)"""
    beams, picks = 2, 6
    masks = torch.tensor([m for m in MASKS if m >= torch.finfo(torch.float32).min], dtype=torch.float64).float().cuda()
    groups = masks.numel()
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = torch.randn((groups, beams, vocab), generator=g, device="cuda")
    scores = -torch.rand(groups * beams, generator=g, device="cuda")
    at = torch.arange(vocab, device="cuda")
    if what == "a few words left":
        masked = torch.ones(vocab, dtype=torch.bool, device="cuda")
        masked[torch.randperm(vocab, generator=g, device="cuda")[:9]] = False
    elif what == "a tail":                                 # a vocabulary padded to a round size
        masked = at >= vocab - vocab // 5
    elif what == "half of all":
        masked = torch.rand(vocab, generator=g, device="cuda") < 0.5
    else:                                                  # words that lie 1,024 apart, four by four
        masked = at // 4 % 256 == 7
    logits[:, 0] = torch.where(masked, masks[:, None], logits[:, 0])
    logits = logits.view(-1, vocab)
    _agree(_select(K, logits, scores, beams, picks), _best(logits.cpu().numpy(), scores.cpu().numpy(), beams, picks), vocab)


@pytest.mark.parametrize("vocab", [5000, 128256])
def test_choice_where_all_words_but_those_of_one_slice_are_masked(K, vocab):  # noqa: F811
    masks = [-1e10, -1e18, -1e20, -1e29, -1e38]
    logits = torch.randn((len(masks), vocab), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    for r, m in enumerate(masks):
        logits[r, 200 * r + 100:] = m
        logits[r, : 200 * r] = m
    scores = torch.full((len(masks),), -2.0, device="cuda")
    _agree(_select(K, logits, scores, 1, 8), _best(logits.cpu().numpy(), scores.cpu().numpy(), 1, 8), vocab)
