"""AdamW with 8-bit moments: the moments bit for bit what the same formulas give in fp32 torch operations on the CPU
(every operation one rounding), the parameters within the rounding of a step's last operations, and both within the
codes' rounding of AdamW with fp32 moments."""
import copy
import math

import numpy as np
import pytest
import torch

from rgpt_b200 import native as nv
from rgpt_b200.graph import GraphedTrainStep  # noqa: F401  (the hp path is what graphed steps use)
from rgpt_b200.optimizer import Muon

pytestmark = pytest.mark.gpu

BLOCK = nv.ADAM8_BLOCK


def f(v):
    return float(np.float32(v))


def blocks(v):
    return torch.nn.functional.pad(v, (0, -v.numel() % BLOCK)).view(-1, BLOCK)


def table_r():
    q = torch.arange(256, dtype=torch.float64)
    return torch.where(q < 32, q / 2048, 2.0 ** (torch.floor(q / 32) - 7) * (1 + (q % 32) / 32)).float()


def pack(m, r):
    n = m.numel()
    m, r = blocks(m), blocks(r)
    a, b = m.abs().amax(1, keepdim=True), r.amax(1, keepdim=True)
    a, b = torch.where(a > 2.0 ** -100, a, 0.0 * a), torch.where(b > 2.0 ** -100, b, 0.0 * b)
    mq = (m * torch.where(a > 0, a.reciprocal() * 448.0, a)).to(torch.float8_e4m3fn).view(torch.uint8)
    y = (r * torch.where(b > 0, b.reciprocal() * 1.96875, b)).double()
    # nearest code, ties to even: 5 bits of mantissa in each binade, steps of 2^-11 below 2^-6
    e = torch.floor(torch.log2(y.clamp_min(2.0 ** -6)))
    step = 2.0 ** (e - 5)
    q = torch.round(y / step) + torch.where(y >= 2.0 ** -6, (e + 6) * 32, torch.zeros_like(e))
    q = q.clamp(0, 255)
    q = torch.where(r > 0, q.clamp_min(1), q)
    return [mq.reshape(-1)[:n].contiguous(), (a * f(1 / 448)).reshape(-1), q.to(torch.uint8).reshape(-1)[:n].contiguous(),
            (b * f(1 / 1.96875)).reshape(-1)]


def unpack(q):
    n = q[0].numel()
    m = (blocks(q[0].view(torch.float8_e4m3fn).float()) * q[1][:, None]).reshape(-1)[:n]
    r = (blocks(table_r()[q[2].long()]) * q[3][:, None]).reshape(-1)[:n]
    return m, r * r


def cpu_step(p, g, q, step, lr, wd, b1, b2, eps):
    b1, b2 = np.float32(b1), np.float32(b2)
    m, v = unpack(q)
    m = m * float(b1) + g * float(np.float32(1) - b1)
    v = v * float(b2) + (g * g) * float(np.float32(1) - b2)
    # correctly rounded: the double root's 53 bits exceed 2 * 24 + 2, so rounding it again is rounding once (the CPU's
    # vectorised fp32 root is not always the nearest)
    r = v.double().sqrt().float()
    u = (m / (r * f(1 / math.sqrt(1 - float(b2) ** step)) + f(eps))) * f(1 / (1 - float(b1) ** step))
    return p * f(np.float32(1) - np.float32(lr) * np.float32(wd)) - u * f(lr), pack(m, r)


def moved(t, by):
    """t's values in a contiguous tensor whose base is `by` elements past a 256-byte boundary."""
    held = torch.zeros(t.numel() + by, device="cuda", dtype=t.dtype)
    held[by:] = t.reshape(-1)
    return held[by:].view(t.shape)


def gradients(n, step):
    g = torch.Generator().manual_seed(1000 * step + n)
    scale = torch.exp(2.0 * torch.randn(n, generator=torch.Generator().manual_seed(n))) * 1e-3
    v = scale * torch.randn(n, generator=g)
    if step == 3:
        v.zero_()                 # a step without gradient: the moments decay
    if n > 600:
        v[256:512] = 0.0          # a block that never sees one
        v[1] = 0.0
    return v


@pytest.mark.parametrize("sizes,by", [((4096, 5001, 16384 + 255), 0), ((4097,), 1), ((70000, 4096), 4), ((8192,), 3)])
@pytest.mark.parametrize("shadow", [False, True])
def test_steps_equal_the_formulas_bit_for_bit(cuda, sizes, by, shadow):
    """The codes and scales are equal. A parameter's step lr m / (sqrt(v) c + eps) / bc1 has a division of 2 ulp (2^-22)
    and four more roundings of 2^-24 on each side, at most 2^-21 of the step in all, and each side rounds the new
    parameter twice (2^-24 of it each time): these add up over the steps."""
    ps = [0.02 * torch.randn(n, generator=torch.Generator().manual_seed(n + 5)) for n in sizes]
    params = [torch.nn.Parameter(moved(p.cuda(), by)) for p in ps]
    for p in params:
        if shadow:
            p._rgpt_shadow = moved(torch.zeros(p.shape, dtype=torch.bfloat16, device="cuda"), by)
    opt = Muon([{"params": params, "use_muon": False}], lr=3e-3, weight_decay=0.1, adam_state_bits=8)
    want = [(p, pack(torch.zeros_like(p), torch.zeros_like(p))) for p in ps]
    room = [torch.zeros_like(p, dtype=torch.float64) for p in ps]
    for step in range(1, 7):
        for i, p in enumerate(params):
            g = gradients(p.numel(), step)
            p.grad = moved(g.cuda(), by)
            before = want[i][0]
            want[i] = cpu_step(before, g, want[i][1], step, 3e-3, 0.1, 0.9, 0.95, 1e-8)
            moved_by = (want[i][0].double() - before.double() * (1 - 3e-3 * 0.1)).abs()
            room[i] += 2.0 ** -21 * moved_by + 4 * 2.0 ** -24 * before.double().abs()
        opt.step()
        for p, (wp, wq), tol in zip(params, want, room):
            st = opt.state[p]
            got = [st["exp_avg_q8"], st["exp_avg_scale"], st["exp_avg_sq_q8"], st["exp_avg_sq_scale"]]
            for a, b in zip(got, wq):
                assert torch.equal(a.cpu(), b)
            assert ((p.detach().cpu().double() - wp.double()).abs() <= tol).all()
            m, v = opt.adam_moments(p)
            wm, wv = unpack(wq)
            assert torch.equal(m.cpu(), wm) and torch.equal(v.cpu(), wv)
            if shadow:
                assert torch.equal(p._rgpt_shadow, p.detach().bfloat16())


def test_all_codes_round_trip(cuda):
    """Every code of both formats stands for the value the formats define, and encoding that value gives the code."""
    n = 256
    q = torch.arange(256, dtype=torch.uint8, device=cuda)
    one = torch.ones(1, device=cuda)
    m, v = nv.adamw8_moments(torch.empty(n, device=cuda), q, one, q, one)
    want = q.cpu().view(torch.float8_e4m3fn).float()
    assert torch.equal(torch.isnan(m.cpu()), torch.isnan(want))
    assert torch.equal(m.cpu()[~torch.isnan(want)], want[~torch.isnan(want)])
    assert torch.equal(v.cpu(), table_r() ** 2)
    back = pack(torch.zeros(256), table_r())
    assert torch.equal(back[2], q.cpu()) and back[3].item() == 1.0


def test_a_gradient_that_is_not_finite_stays_in_its_block(cuda):
    n = 5000
    runs = []
    for bad in (None, float("inf"), float("nan")):
        p = torch.nn.Parameter(0.02 * torch.randn(n, generator=torch.Generator().manual_seed(1)).cuda())
        opt = Muon([{"params": [p], "use_muon": False}], lr=1e-3, adam_state_bits=8)
        for step in range(3):
            p.grad = gradients(n, step).cuda()
            if step == 1 and bad is not None:
                p.grad[700] = bad
            opt.step()
        runs.append((p.detach().clone(), *opt.adam_moments(p)))
    for run in runs[1:]:
        assert run[0][700].isnan()
        for a, b in zip(run, runs[0]):
            assert torch.equal(a[:512], b[:512]) and torch.equal(a[768:], b[768:])


def test_near_adamw_with_fp32_moments(cuda):
    """Twenty steps on gradients of one scale. A code is within 2^-4 (first moment) of a value that is not far below its
    block's largest; the update divides by sqrt(v), whose code is within 2^-6. So an update is off by about 8% at most
    where m is not small, and the average over elements by less."""
    n = 40000
    p0 = 0.02 * torch.randn(n, generator=torch.Generator().manual_seed(1))
    res = []
    for bits in (8, 32):
        p = torch.nn.Parameter(p0.clone().cuda())
        opt = Muon([{"params": [p], "use_muon": False}], lr=1e-3, weight_decay=0.0, adam_state_bits=bits)
        for step in range(20):
            p.grad = (1e-3 * torch.randn(n, generator=torch.Generator().manual_seed(step))).cuda()
            opt.step()
        res.append((p.detach().cpu() - p0).double())
    assert ((res[0] - res[1]).norm() / res[1].norm()).item() < 2.0 ** -4 + 2.0 ** -6


def test_device_hparams_small_parameters_and_state_dict(cuda):
    def build():
        torch.manual_seed(0)
        ps = [torch.nn.Parameter(torch.randn(300, 40, device=cuda)), torch.nn.Parameter(torch.randn(100, device=cuda))]
        return ps, Muon([{"params": ps, "use_muon": False}], lr=1e-2, weight_decay=0.1, adam_state_bits=8)

    def step(ps, opt, k):
        for i, p in enumerate(ps):
            g = torch.Generator(device=cuda).manual_seed(10 * k + i)
            if p.grad is None:
                p.grad = torch.empty_like(p)
            p.grad.copy_(torch.randn(p.shape, device=cuda, generator=g))
        if opt._hp_dev is not None:
            opt.stage_device_hparams()
        opt.step()

    a, oa = build()
    b, ob = build()
    ob.use_device_hparams()
    for k in range(4):
        step(a, oa, k)
        step(b, ob, k)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert "exp_avg" in oa.state[a[1]] and "exp_avg_q8" in oa.state[a[0]]  # below 4096 elements: fp32 moments
    assert oa.adam_moments(a[1])[0] is oa.state[a[1]]["exp_avg"]
    c, oc = build()
    oc.load_state_dict(copy.deepcopy(oa.state_dict()))
    with torch.no_grad():
        for x, y in zip(c, a):
            x.copy_(y)
    st = oc.state[c[0]]
    assert st["exp_avg_q8"].dtype == torch.uint8 and st["exp_avg_scale"].dtype == torch.float32
    for k in range(4, 6):
        step(a, oa, k)
        step(c, oc, k)
    assert all(torch.equal(x, y) for x, y in zip(a, c))
    oa.param_groups[0]["adam_state_bits"] = 32
    with pytest.raises(ValueError, match="8 bits"):
        oa.step()
