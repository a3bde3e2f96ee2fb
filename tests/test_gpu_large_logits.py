"""Rows of large logits in the policy loss, and what the log-probabilities of many rows have in common. u = 2^-24, the half
step of fp32."""
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


@pytest.mark.parametrize("B,V", [(3, 500), (1500, 500), (9, 3001), (5, 20000), (200, 20001)])
@pytest.mark.parametrize("dtype,top,step", [(torch.float32, 1e3, 0.0), (torch.float32, -3e4, 0.0), (torch.float32, 5e5, 0.0),
                                            (torch.float16, 65504.0, 32.0), (torch.float16, -1024.0, 1.0),
                                            (torch.bfloat16, 3e4, 0.0)])
def test_gradient_rows_of_large_logits(cuda, B, V, dtype, top, step):
    """p = e^{x - lse}: the difference x - lse is rounded once (u of its size, and u of log2 e and the product each), the
    sum of exponentials has (40 + V / 256) u, the exponential 4 u, the arithmetic 4 u: nothing that grows with the logits
    themselves. An element is then rounded to its type, at half a step (fp16: at least 2^-25)."""
    g = torch.Generator(device=cuda).manual_seed(V + B)
    if step:  # logits of that size lie whole steps apart: ties
        x = top - step * torch.randint(0, 4, (B, 1, V), device=cuda, generator=g).float()
    else:
        x = top + 3.0 * torch.randn(B, 1, V, device=cuda, generator=g)
    x = x.to(dtype)
    labels = torch.randint(0, V, (B, 1), device=cuda, generator=g)
    lse = torch.logsumexp(x.double(), -1)
    lp = (x.double().gather(-1, labels[..., None])[..., 0] - lse).float()
    out = policy(x, labels, lp, torch.full((B,), -float(B), device=cuda))
    p = torch.softmax(x.double(), -1)
    c = out["coef"].double()[..., None]
    want = c * (torch.zeros_like(p).scatter_(-1, labels[..., None], 1.0) - p)
    t = (x.double() - lse[..., None]).abs() * 1.4426950408889634
    tol = c.abs() * p * ((40 + V / 256) + 8 + 3 * t) * U + 2 * U * c.abs() * (want.abs() > 0)
    tol = tol + torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -25 if dtype is torch.float16 else 0.0)
    off = (out["dlogits"].double() - want).abs() - tol
    assert (off <= 0).all(), off.max()


def test_log_probabilities_have_no_common_error(cuda):
    """What is the same for every row adds up over a long sequence: the mean error of 4096 log-probabilities in (-16, -8),
    each rounded at a step of 2^-20 (a deviation of 2^-20 / sqrt 12, so five deviations of the mean are 2.2e-8), is within
    that and the 1e-8 that the sums' own corrections leave."""
    g = torch.Generator(device=cuda).manual_seed(5)
    x = torch.randn(4096, 50304, device=cuda, generator=g).bfloat16()
    labels = torch.randint(0, 50304, (4096,), device=cuda, generator=g)
    lp = torch.empty(4096, device=cuda)
    nv.token_logprobs(x, labels, lp)
    want = torch.cat([torch.log_softmax(x[i:i + 512].double(), 1).gather(1, labels[i:i + 512, None])[:, 0]
                      for i in range(0, 4096, 512)])
    assert want.min() > -16 and want.max() < -8 + 2
    assert abs((lp.double() - want).mean().item()) <= 2.2e-8 + 1e-8
