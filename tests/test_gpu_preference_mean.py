"""The preference loss is the mean of the pairs' losses, rounded once, however many pairs there are."""
import pytest
import torch

from rgpt_b200 import native as nv

pytestmark = pytest.mark.gpu


def loss_of(x, labels, ref, **kw):
    B, T = labels.shape
    n = lambda *s: torch.empty(*s, device=x.device)  # noqa: E731
    out = dict(token_logps=n(B, T), lse=n(B, T), seq_logps=n(B), margins=n(B // 2), coef=n(B), loss=n(1))
    nv.preference_loss(x, labels, ref, **out, **kw)
    return out["loss"], out["margins"]


def aligned(x):
    """The same logits in rows of a multiple of 16 bytes: rows of equal alignment are summed in the same order."""
    held = torch.zeros(*x.shape[:-1], 304, device=x.device)
    held[..., :x.shape[-1]] = x
    return held[..., :x.shape[-1]]


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "squared"])
@pytest.mark.parametrize("T,pairs", [(7, 16), (7, 256), (300, 2), (300, 32), (1, 64)])
def test_equal_pairs_have_the_loss_of_one(cuda, kind, T, pairs):
    """Powers of two of the same pair: the sum and its division are exact, so the bits are those of one pair."""
    differ = 0
    for seed in range(12):
        g = torch.Generator(device=cuda).manual_seed(100 * T + seed)
        x = 2.0 * torch.randn(2, T, 301, device=cuda, generator=g)
        labels = torch.randint(0, 301, (2, T), device=cuda, generator=g)
        ref = torch.randn(2, device=cuda, generator=g)
        one, h = loss_of(aligned(x), labels, ref, kind=kind, beta=0.37)
        many, hs = loss_of(aligned(x.repeat_interleave(pairs, 0)), labels.repeat_interleave(pairs, 0), ref.repeat_interleave(pairs),
                           kind=kind, beta=0.37)
        assert torch.equal(hs, h.expand(pairs))
        differ += not torch.equal(one, many)
    assert differ == 0
