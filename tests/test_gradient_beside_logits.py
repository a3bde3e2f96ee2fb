"""Logits and their gradient in turn in one buffer: rows that interleave share no memory."""
import pytest
import torch

from rgpt_b200 import native as nv


def halves(B, T, V, gap, dtype, device, first):
    held = torch.zeros(B, T, 2 * V + gap, dtype=dtype, device=device)
    a, b = held[..., :V], held[..., V + gap:]
    return (held, a, b) if first else (held, b, a)


@pytest.mark.parametrize("B,T,V,gap", [(4, 3, 8, 0), (4, 1, 8, 0), (1, 5, 7, 1), (1, 1, 5, 0), (3, 2, 6, 3)])
@pytest.mark.parametrize("first", [True, False])
def test_interleaved_rows_pass_the_checks(B, T, V, gap, first):
    held, x, d = halves(B, T, V, gap, torch.float32, "cpu", first)
    y, o = torch.zeros(B, T, dtype=torch.int64), torch.zeros(B, T)
    for view in (lambda t: t, lambda t: t.transpose(0, 1)):
        with pytest.raises(RuntimeError, match="CUDA"):  # passed, then wants CUDA tensors
            nv.token_logprobs_bwd(view(x), view(y).contiguous(), view(o).contiguous(), view(o).contiguous(), view(d))


def test_rows_that_touch_are_refused():
    y, o = torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)
    held = torch.zeros(4, 3, 15)
    flat = torch.zeros(200)
    for x, d in ((held[..., :8], held[..., 7:]), (flat[:96].view(4, 3, 8), flat[8:104].view(4, 3, 8)),
                 (flat[:96].view(4, 3, 8), flat[95:191].view(4, 3, 8)),
                 (flat.as_strided((4, 3, 8), (30, 10, 1)), flat.as_strided((4, 3, 8), (30, 10, 1), 12)),
                 (flat.as_strided((4, 3, 8), (48, 16, 1)), flat.as_strided((4, 3, 8), (40, 12, 1), 8))):
        with pytest.raises(ValueError, match="share no memory"):
            nv.token_logprobs_bwd(x, y, o, o, d)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,V,gap", [(3, 5, 1000, 0), (2, 40, 9001, 3), (300, 1, 20000, 8), (2, 3, 50257, 0), (700, 2, 33, 1)])
def test_values(cuda, dtype, B, T, V, gap):
    """The rows and their gradients as with memory of their own: the sums may run in another order where the rows start on
    other boundaries, so a gradient of 1 - p or -p is within (80 + V / 128) 2^-24 and a step of its type."""
    g = torch.Generator(device=cuda).manual_seed(V)
    held, x, d = halves(B, T, V, gap, dtype, cuda, True)
    held.fill_(7.0)
    x.copy_(3.0 * torch.randn(B, T, V, device=cuda, generator=g))
    own, want = x.clone(), torch.empty(B, T, V, device=cuda, dtype=dtype)
    y = torch.randint(0, V, (B, T), device=cuda, generator=g)
    y[0, 0] = -100
    lp, lse = torch.empty(2, B, T, device=cuda)
    nv.token_logprobs(own, y, lp, lse=lse)
    nv.token_logprobs_bwd(own, y, lse, torch.ones_like(lp), want)
    nv.token_logprobs(x, y, lp, lse=lse)
    nv.token_logprobs_bwd(x, y, lse, torch.ones_like(lp), d)
    assert torch.equal(x, own) and (held[..., V:V + gap] == 7).all()
    tol = (80 + V / 128) * 2.0 ** -24 + torch.finfo(dtype).eps * want.float().abs() + (2.0 ** -24 if dtype is torch.float16 else 0)
    assert ((d.float() - want.float()).abs() <= tol).all()
    st = torch.empty(4, device=cuda)
    out = dict(token_logps=lp, counts=torch.empty(B, device=cuda, dtype=torch.int32), stats=st)
    adv = torch.full((B,), -1.0, device=cuda)
    old = torch.full((B, T), -9.0, device=cuda)
    want2 = torch.empty_like(want)
    nv.policy_loss(own, y, old, adv, clip_high=1e9, dlogits=want2, **out)
    nv.policy_loss(x, y, old, adv, clip_high=1e9, dlogits=d, **out)
    assert torch.equal(x, own) and (held[..., V:V + gap] == 7).all()
    size = want2.float().abs().amax(-1, keepdim=True)
    tol = 2 * (80 + V / 128) * 2.0 ** -24 * (1 + 9) * size + torch.finfo(dtype).eps * want2.float().abs() + 2.0 ** -24
    assert ((d.float() - want2.float()).abs() <= tol).all()
