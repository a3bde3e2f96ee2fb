"""8-bit AdamW takes second-moment decays that its codes can follow, and refuses slower ones."""
import pytest
import torch

from rgpt_b200.optimizer import ADAM8_MAX_BETA2, Muon


def params():
    big, small = torch.nn.Parameter(torch.zeros(5000)), torch.nn.Parameter(torch.zeros(10))
    big.grad, small.grad = torch.zeros(5000), torch.zeros(10)
    return big, small


def build(betas=(0.9, 0.95), bits=8, which=slice(None), **group):
    return Muon([{"params": list(params()[which]), "use_muon": False, **group}], adam_state_bits=bits, adam_betas=betas)


@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.9, 0.99), (0.9, ADAM8_MAX_BETA2 + 1e-4)])
def test_slow_decays_are_refused(betas):
    with pytest.raises(ValueError, match="beta2"):
        build(betas)
    with pytest.raises(ValueError, match="beta2"):  # a group's own
        build(adam_betas=betas)
    opt = build()
    opt.param_groups[0]["adam_betas"] = betas  # changed later
    with pytest.raises(ValueError, match="beta2"):
        opt.step()
    opt = build(betas, bits=32)
    opt.param_groups[0]["adam_state_bits"] = 8
    with pytest.raises(ValueError, match="beta2"):
        opt.step()
    opt = build()
    opt._hp_dev, opt._hp_done, opt._hp_slot, opt._hp_host = torch.zeros(1), [None], 0, [torch.zeros(64)]
    opt.param_groups[0]["adam_betas"] = betas
    with pytest.raises(ValueError, match="beta2"):
        opt.stage_device_hparams()


def test_what_keeps_fp32_moments_takes_any_decay():
    build((0.9, 0.999), bits=32)
    build((0.9, 0.999), which=slice(1, None))  # below 4096 elements
    p = torch.nn.Parameter(torch.zeros(64, 64))
    Muon([{"params": [p], "use_muon": True}], adam_state_bits=8, adam_betas=(0.9, 0.999))
    build((0.9, 0.95))
    build((0.9, ADAM8_MAX_BETA2))


def codes(r):
    """sqrt(v) rounded to the 8-bit codes of its block of 256 and back (3 bits of exponent, 5 of mantissa)."""
    b = r.view(-1, 256).amax(1, keepdim=True)
    y = r.view(-1, 256) / b * 1.96875
    step = 2.0 ** (torch.floor(torch.log2(y.clamp_min(2.0 ** -6))) - 5)
    q = torch.round(y / step) * step
    return (torch.where(y > 0, q.clamp_min(2.0 ** -11), q) * b / 1.96875).view(-1)


def test_the_codes_follow_the_largest_decay_taken():
    """The gradient of every second element falls to a tenth: after eight times 1 / (1 - beta2) steps the 8-bit second
    moment of these is within a quarter of the fp32 one for 19 of 20 (a code's half step is 3% of it; the median within
    5%), where 0.999 leaves the median more than 50 times too large."""
    for beta2, ok in ((0.95, True), (ADAM8_MAX_BETA2, True), (0.999, False)):
        tau, n = round(1 / (1 - beta2)), 2048
        g = torch.Generator().manual_seed(0)
        size = torch.exp(0.5 * torch.randn(n, generator=g))
        r, v = torch.zeros(n), torch.zeros(n)
        for t in range(14 * tau):
            d = size * torch.randn(n, generator=g)
            if t >= 6 * tau:
                d[1::2] *= 0.1
            v = beta2 * v + (1 - beta2) * d * d
            r = codes(torch.sqrt(beta2 * r * r + (1 - beta2) * d * d))
        ratio = (r * r / v)[1::2]
        if ok:
            assert abs(ratio.median() - 1) < 0.05 and ratio.quantile(0.95) < 1.25
        else:
            assert ratio.median() > 50
