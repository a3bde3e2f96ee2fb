"""The policy loss's KL term next to the reference, where its parts cancel. u = 2^-24, the half step of fp32."""
import pytest
import torch

from rgpt_b200 import native as nv

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def policy(x, labels, old, adv, ref=None, grad=True, **kw):
    B, T = labels.shape
    n = lambda *s: torch.empty(*s, device=x.device)  # noqa: E731
    out = dict(token_logps=n(B, T), counts=torch.empty(B, device=x.device, dtype=torch.int32), stats=n(4), coef=n(B, T),
               dlogits=torch.empty_like(x) if grad else None)
    nv.policy_loss(x, labels, old, adv, ref, **out, **kw)
    return out


@pytest.mark.parametrize("size", [1e-6, 1e-5, 1e-4, 1e-3, 1e-2, 0.1, 0.3, 0.7, 2.0])
@pytest.mark.parametrize("B", [1, 700, 12000])
def test_kl_next_to_the_reference(cuda, B, size):
    """e^q - q - 1 of q = ref - logp, logp as the call returns it: q is rounded once (2 u of the term, which goes with
    q^2), the term has 8 u, weight and sum 4 u. No term is negative, however small q."""
    g = torch.Generator(device=cuda).manual_seed(B)
    x = 2.0 * torch.randn(B, 1, 40, device=cuda, generator=g)
    labels = torch.randint(0, 40, (B, 1), device=cuda, generator=g)
    lp = policy(x, labels, torch.zeros(B, 1, device=cuda), torch.zeros(B, device=cuda), grad=False)["token_logps"]
    q = size * (0.5 + torch.rand(B, 1, device=cuda, generator=g)) * torch.sign(torch.randn(B, 1, device=cuda, generator=g))
    ref = (lp.double() + q).float()
    out = policy(x, labels, lp, torch.zeros(B, device=cuda), ref, grad=False, kl_coef=0.1)
    assert torch.equal(out["token_logps"], lp)
    q = ref.double() - lp.double()
    # past 0.05 the 64-bit difference is exact to 2^-53 / q^2; below, eight terms of the series
    series = q * q * sum(q ** k / torch.lgamma(torch.tensor(k + 3.0, dtype=torch.float64)).exp().item() for k in range(8))
    want = torch.where(q.abs() < 0.05, series, torch.expm1(q) - q).mean().item()
    assert abs(out["stats"][2].item() - want) <= 14 * U * want
    assert abs(out["stats"][0].item() - 0.1 * want) <= 16 * U * 0.1 * want
    if B == 1:
        assert out["stats"][2].item() >= 0
