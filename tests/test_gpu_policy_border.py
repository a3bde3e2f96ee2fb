"""Ratios at the policy loss's clip borders, where gradient and statistics have to decide alike."""
import pytest
import torch

from rgpt_b200 import native as nv

pytestmark = pytest.mark.gpu


def policy(x, labels, old, adv, ref=None, grad=True, **kw):
    B, T = labels.shape
    n = lambda *s: torch.empty(*s, device=x.device)  # noqa: E731
    out = dict(token_logps=n(B, T), counts=torch.empty(B, device=x.device, dtype=torch.int32), stats=n(4), coef=n(B, T),
               dlogits=torch.empty_like(x) if grad else None)
    nv.policy_loss(x, labels, old, adv, ref, **out, **kw)
    return out


@pytest.mark.parametrize("side", [1.0, -1.0])
@pytest.mark.parametrize("B,T,V", [(3000, 1, 64), (6, 170, 64), (300, 1, 9000), (16, 1000, 33)])
def test_the_clipped_share_counts_the_tokens_whose_gradient_is_cut(cuda, B, T, V, side):
    g = torch.Generator(device=cuda).manual_seed(V)
    x = 2.0 * torch.randn(B, T, V, device=cuda, generator=g)
    labels = torch.randint(0, V, (B, T), device=cuda, generator=g)
    adv = torch.full((B,), side, device=cuda)
    lp = policy(x, labels, torch.zeros(B, T, device=cuda), adv, grad=False)["token_logps"]
    border = torch.log1p(torch.tensor(0.2 * side, dtype=torch.float64)).item()
    old = (lp.double() - border).float()  # ratios within a rounding of the border
    out = policy(x, labels, old, adv)
    cut = (out["coef"] == 0).sum().item()
    assert 0 < cut < B * T
    assert abs(out["stats"][3].item() * B * T - cut) <= 0.01
