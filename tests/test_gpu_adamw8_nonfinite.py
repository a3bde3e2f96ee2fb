"""8-bit AdamW: a moment that is not finite makes its whole block's so, and no other block's."""
import pytest
import torch

from rgpt_b200.optimizer import Muon

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("n,at", [(5000, 700), (4096 + 131, 4096 + 130), (8192, 0)])
@pytest.mark.parametrize("by", [0, 1])
def test_whole_block(cuda, bad, n, at, by):
    def run(spoil):
        held = torch.zeros(n + by, device=cuda)
        p = torch.nn.Parameter(held[by:])
        opt = Muon([{"params": [p], "use_muon": False}], lr=1e-3, adam_state_bits=8)
        for step in range(3):
            p.grad = torch.randn(n, generator=torch.Generator().manual_seed(step)).cuda()
            if step == 1 and spoil:
                p.grad[at] = bad
            opt.step()
        return (p.detach().clone(), *opt.adam_moments(p))

    (p, m, v), clean = run(True), run(False)
    lo, hi = at // 256 * 256, min(n, at // 256 * 256 + 256)
    assert not torch.isfinite(m[lo:hi]).any() and not torch.isfinite(v[lo:hi]).any()
    if bad != bad:
        assert v[lo:hi].isnan().all()
    assert p[at].isnan()
    for a, b in zip((p, m, v), clean):
        assert torch.equal(a[:lo], b[:lo]) and torch.equal(a[hi:], b[hi:])
