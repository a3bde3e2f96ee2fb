"""Token log-probabilities, the preference loss and the policy loss against their formulas in 64 bits.

Tolerances (u = 2^-24, the half step of fp32): a sum of exponentials of V terms carries at most 4u for each hardware
exponential (relative error 2^-22), u |t| for the rounding of its exponent t = (x - max) log2 e, |t| < 30 where the
term counts, and u for each of the V/256 + 16 additions on the longest path of a CTA of at least 256 threads. So
rel(V) = (40 + V/256) u bounds the relative error of the sum and the absolute error of lse, before lse and the
log-probability are rounded to fp32 (u times their size). A gradient c (1[label] - p) adds the rounding of lse
to p (u |lse|), 4u for its own exponential and 2u for the arithmetic, then half a step of its type (for fp16 at
least 2^-25, its smallest step's half).
"""
import pytest
import torch

from rgpt_b200 import losses
from rgpt_b200 import native as nv

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
IGNORE = -100


def rel(V):
    return (40 + V / 256) * U


def make(B, T, V, dtype, layout="plain", seed=0, masked=0.3):
    """(logits view, labels): labels of some tokens ignored or outside the vocabulary."""
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * V + T)
    x = 3.0 * torch.randn(B, T, V, device="cuda", generator=g)
    if layout == "plain":
        held = torch.empty(B, T, V, device="cuda", dtype=dtype)
        view = held
    elif layout == "shifted":  # logits[:, :-1]
        held = torch.full((B, T + 1, V), 5.0, device="cuda", dtype=dtype)
        view = held[:, :-1]
    elif layout == "padded":  # rows wider than the vocabulary, base one element past a boundary
        held = torch.full((B * T * (V + 3) + 1,), 5.0, device="cuda", dtype=dtype)
        view = held[1:].view(B, T, V + 3)[..., :V]
    elif layout == "time first":
        held = torch.empty(T, B, V, device="cuda", dtype=dtype)
        view = held.transpose(0, 1)
    view.copy_(x)
    labels = torch.randint(0, V, (B, T), device="cuda", generator=g)
    drop = torch.rand(B, T, device="cuda", generator=g)
    labels[drop < masked] = IGNORE
    labels[(drop >= masked) & (drop < masked + 0.05)] = V
    labels[(drop >= masked + 0.05) & (drop < masked + 0.1)] = -1
    return view, labels


def scored(labels, V):
    return (labels >= 0) & (labels < V) & (labels != IGNORE)


def ref_logps(x, labels):
    """(lp, lse) in 64 bits, 0 where not scored."""
    V = x.shape[-1]
    on = scored(labels, V)
    xd = x.double()
    lse = torch.logsumexp(xd, -1)
    lp = xd.gather(-1, labels.clamp(0, V - 1)[..., None])[..., 0] - lse
    return torch.where(on, lp, 0.0), torch.where(on, lse, 0.0)


def check_logps(lp, want, lse, V):
    assert ((lp.double() - want).abs() <= rel(V) + U * (want.abs() + 1e-30)).all()
    return lse


def check_grad(d, x, labels, coef, coef_err=0.0):
    """d against coef * (onehot - softmax); coef_err: the coefficient's own relative error."""
    V = x.shape[-1]
    on = scored(labels, V)
    lse = torch.logsumexp(x.double(), -1)
    for b in range(x.shape[0]):  # a sequence at a time: 64-bit copies
        p = torch.softmax(x[b].double(), -1)
        hot = torch.zeros_like(p).scatter_(-1, labels[b].clamp(0, V - 1)[:, None], 1.0)
        c = torch.where(on[b], coef[b].double(), 0.0)[:, None]
        want = c * (hot - p)
        half = torch.finfo(d.dtype).eps / 2
        tol = (half + coef_err + 2 * U) * want.abs() + c.abs() * (p * (rel(V) + U * (lse[b].abs()[:, None] + 6)) + 2 * U)
        if d.dtype == torch.float16:
            tol = tol + 2.0 ** -25
        off = (d[b].double() - want).abs() - tol
        assert (off <= 0).all(), off.max()
        assert (d[b][~on[b]] == 0).all()


CASES = [
    (1, 1, 1, torch.float32, "plain"), (2, 3, 2, torch.bfloat16, "plain"), (3, 5, 7, torch.float16, "padded"),
    (2, 9, 1000, torch.bfloat16, "shifted"), (2, 6, 1001, torch.bfloat16, "shifted"), (3, 4, 4099, torch.float32, "padded"),
    (2, 8, 50304, torch.bfloat16, "plain"), (2, 5, 50257, torch.float16, "shifted"), (2, 3, 50257, torch.float32, "plain"),
    (1, 300, 515, torch.bfloat16, "time first"), (5, 40, 96, torch.float32, "time first"), (1, 2, 131071, torch.float32, "plain"),
    (1, 3, 262144, torch.bfloat16, "plain"), (40, 1, 33000, torch.bfloat16, "plain"), (700, 1, 120, torch.bfloat16, "plain"),
    (1, 5000, 65, torch.float16, "plain"),
    # many long rows
    (300, 1, 50304, torch.bfloat16, "plain"), (2, 160, 50257, torch.float16, "plain"), (3, 101, 50257, torch.float32, "plain"),
    (2, 150, 8192, torch.bfloat16, "shifted"), (2, 170, 8201, torch.float16, "shifted"), (1, 700, 4100, torch.float32, "padded"),
    (5, 70, 32768, torch.bfloat16, "time first"), (1, 300, 131071, torch.float32, "plain"), (4, 300, 16391, torch.bfloat16, "padded"),
]


@pytest.mark.parametrize("B,T,V,dtype,layout", CASES)
@pytest.mark.parametrize("inplace", [False, True])
def test_token_logprobs_forward_and_backward(cuda, B, T, V, dtype, layout, inplace):
    x, labels = make(B, T, V, dtype, layout)
    before = x.clone()
    base = x._base if x._base is not None else x
    outside = base.clone()
    lp, lse = torch.full((B, T), 9.0, device=cuda), torch.full((B, T), 9.0, device=cuda)
    nv.token_logprobs(x, labels, lp, lse=lse)
    want, want_lse = ref_logps(before, labels)
    assert ((lp.double() - want).abs() <= rel(V) + U * want.abs()).all()
    assert ((lse.double() - want_lse).abs() <= rel(V) + U * want_lse.abs()).all()
    assert torch.equal(x, before)
    g = torch.randn(B, T, device=cuda)
    d = x if inplace else torch.full((B, T, V), 3.0, device=cuda, dtype=dtype)
    nv.token_logprobs_bwd(x, labels, lse, g, d)
    check_grad(d, before, labels, g)
    if inplace:  # nothing outside the rows was written
        x.copy_(before)
    assert torch.equal(base, outside)


def test_two_dimensional_logits_are_rows(cuda):
    x, labels = make(1, 37, 777, torch.bfloat16)
    x2, y2 = x[0], labels[0]
    lp = torch.empty(37, device=cuda)
    nv.token_logprobs(x2, y2, lp)
    want, _ = ref_logps(x2, y2)
    assert ((lp.double() - want).abs() <= rel(777) + U * want.abs()).all()
    nv.token_logprobs(x2[:0], y2[:0], lp[:0])  # no rows


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V,times", [(130, 1), (50304, 1), (50304, 40), (8200, 100)])
def test_rows_of_extreme_values(cuda, dtype, V, times):
    low, inf = torch.finfo(dtype).min, float("inf")
    x = torch.randn(9, V, device=cuda).to(dtype)
    x[0] = low                      # every logit the lowest value: uniform
    x[1, : V // 2] = low            # masked half
    x[2, : V // 2] = -inf
    x[3] = -inf                     # nothing left: NaN, as log_softmax
    x[4, 5] = inf
    x[5, 6] = float("nan")
    x[6] = torch.finfo(dtype).max / 2
    x[7] = float("nan")             # not scored: must not leak
    x[8, 3] = -inf                  # the label itself is masked out
    labels = torch.full((9,), V - 1, device=cuda)
    labels[7], labels[8] = IGNORE, 3
    x, labels = x.repeat(times, 1), labels.repeat(times)
    lp, lse = torch.empty(9 * times, device=cuda), torch.empty(9 * times, device=cuda)
    nv.token_logprobs(x, labels, lp, lse=lse)
    d = torch.empty_like(x)
    nv.token_logprobs_bwd(x, labels, lse, torch.ones(9 * times, device=cuda), d)
    # the same through the policy loss, on-policy with advantage -1: the gradient is softmax - onehot over all scored
    # tokens, and the same rows give the same bits wherever they stand
    st, lp2, d2 = torch.empty(4, device=cuda), torch.empty_like(lp), torch.empty_like(x)
    old = torch.where(torch.isfinite(lp), lp, 0.0)
    n = 9 * times
    nv.policy_loss(x, labels, old, torch.full((n,), -float(8 * times), device=cuda), token_logps=lp2, stats=st,
                   counts=torch.empty(n, device=cuda, dtype=torch.int32), dlogits=d2)
    for t in (lp, lp2, d, d2):
        assert torch.equal(t.view(times, -1).nan_to_num(7.5), t.view(times, -1)[:1].nan_to_num(7.5).expand(times, -1))
    x, labels, lp, lse, d, lp2, d2 = x[:9], labels[:9], lp[:9], lse[:9], d[:9], lp2[:9], d2[:9]
    assert torch.equal(torch.isnan(lp), torch.isnan(lp2)) and lp2[8] == -inf and lp2[7] == 0 and (d2[7] == 0).all()
    assert ((lp2 - lp)[[0, 1, 2, 6]].abs() <= 2 * rel(V) + 2 * U * lp[[0, 1, 2, 6]].abs()).all()
    # a ratio of e^0 to e^{2 rel}, and the label at -inf has ratio 0
    check_grad(d2[[1, 2]][None], x[[1, 2]][None], labels[[1, 2]][None], torch.full((1, 2), 1.0, device=cuda), 3 * rel(V) + 16 * U)
    assert (d2[8] == 0).all()
    want, _ = ref_logps(x.double()[None], labels[None])
    want = want[0]
    ok = [0, 1, 2, 6]
    assert ((lp[ok].double() - want[ok]).abs() <= rel(V) + U * (want[ok].abs() + x[ok, V - 1].double().abs())).all()
    assert torch.isnan(lp[[3, 4, 5]]).all() and lp[7] == 0 and lp[8] == -inf
    assert torch.isnan(d[[3, 4, 5]]).any(1).all() and (d[7] == 0).all()
    assert torch.isfinite(d[ok]).all() and torch.isfinite(d[8]).all()
    check_grad(d[[1, 2, 8]][None], x[[1, 2, 8]][None], labels[[1, 2, 8]][None], torch.ones(1, 3, device=cuda))
    p = 1.0 / V
    assert ((d[0, 0].double() + p).abs() <= (torch.finfo(dtype).eps / 2 + rel(V)) * p + 2.0 ** -25).all()


# ------------------------------------------------------------------------------------------------ preference
def ref_preference(lp, labels, V, ref, kind, beta, smoothing, margin, average):
    on = scored(labels, V)
    P = lp.shape[0] // 2
    n = on.sum(1).clamp_min(1).double() if average else torch.ones(2 * P, device=lp.device, dtype=torch.float64)
    lp = lp.clone().requires_grad_(True)
    seq = lp.sum(1) / n
    h = seq if ref is None else seq - ref.double()
    h = beta * (h[:P] - h[P:]) - margin
    ls = torch.nn.functional.logsigmoid
    f = {"sigmoid": -(1 - smoothing) * ls(h) - smoothing * ls(-h), "hinge": torch.relu(1 - h), "squared": (h - 0.5) ** 2}[kind]
    loss = f.mean()
    (d,) = torch.autograd.grad(loss, lp)
    return loss.detach(), seq.detach(), h.detach(), torch.where(on, d, 0.0), n


PREF = [
    dict(P=1, T=1, V=11, dtype=torch.float32, kind="sigmoid"),
    dict(P=2, T=33, V=1000, dtype=torch.bfloat16, kind="hinge", beta=0.3),
    dict(P=3, T=20, V=50257, dtype=torch.float16, kind="sigmoid", smoothing=0.1, layout="shifted"),
    dict(P=2, T=17, V=50304, dtype=torch.bfloat16, kind="sigmoid", average=True, beta=2.0, margin=0.5, free=True),
    dict(P=37, T=5, V=130, dtype=torch.float32, kind="squared", beta=0.2, layout="time first"),
    dict(P=300, T=2, V=64, dtype=torch.bfloat16, kind="sigmoid"),
    dict(P=2, T=700, V=301, dtype=torch.bfloat16, kind="squared", average=True, layout="padded"),
    dict(P=2, T=9, V=500, dtype=torch.float32, kind="sigmoid", empty=True),
    dict(P=2, T=90, V=50304, dtype=torch.bfloat16, kind="sigmoid", smoothing=0.1, layout="shifted"),
    dict(P=3, T=60, V=8203, dtype=torch.float16, kind="hinge", average=True, beta=1.0),
    dict(P=160, T=1, V=20001, dtype=torch.float32, kind="squared", layout="padded"),
    dict(P=2, T=9, V=500, dtype=torch.float32, kind="hinge", average=True, empty=True),
    dict(P=100, T=5, V=250, dtype=torch.float32, kind="sigmoid", average=True, beta=1.0, smoothing=0.1),
    dict(P=512, T=1, V=501, dtype=torch.float16, kind="squared", layout="padded"),
    dict(P=1, T=450, V=1100, dtype=torch.bfloat16, kind="hinge", layout="shifted", free=True),
]


def _pref_buffers(B, T, dev):
    n = lambda *s: torch.full(s, 7.0, device=dev)  # noqa: E731
    return dict(token_logps=n(B, T), lse=n(B, T), seq_logps=n(B), margins=n(B // 2), coef=n(B), loss=n(1))


@pytest.mark.parametrize("c", PREF, ids=lambda c: "-".join(str(v) for v in c.values()))
@pytest.mark.parametrize("inplace", [False, True])
def test_preference_loss(cuda, c, inplace):
    P, T, V = c["P"], c["T"], c["V"]
    x, labels = make(2 * P, T, V, c["dtype"], c.get("layout", "plain"))
    if c.get("empty"):
        labels[0], labels[-1] = IGNORE, IGNORE  # a chosen and a rejected sequence without a scored token
    before = x.clone()
    lp, _ = ref_logps(before, labels)
    n = scored(labels, V).sum(1)
    average, beta = c.get("average", False), c.get("beta", 0.1)
    g = torch.Generator(device=cuda).manual_seed(3)
    ref = lp.sum(1) + 0.5 * n.clamp_min(1).sqrt() * torch.randn(2 * P, device=cuda, generator=g, dtype=torch.float64)
    ref = None if c.get("free") else (ref / n.clamp_min(1) if average else ref).float()
    args = dict(kind=c["kind"], beta=beta, label_smoothing=c.get("smoothing", 0.0), margin=c.get("margin", 0.0), average=average)
    loss, seq, h, coef, nn = ref_preference(lp, labels, V, ref, c["kind"], beta, c.get("smoothing", 0.0), c.get("margin", 0.0), average)
    b, b2 = _pref_buffers(2 * P, T, cuda), _pref_buffers(2 * P, T, cuda)
    nv.preference_loss(x, labels, ref, **args, **b2)  # without a gradient
    d = x if inplace else torch.full((2 * P, T, V), 3.0, device=cuda, dtype=c["dtype"])
    nv.preference_loss(x, labels, ref, dlogits=d, grad_scale=0.5, **args, **b)
    # each token's log-probability is rounded to fp32 before it is summed
    seq_tol = ((rel(V) + U * lp.abs()) * scored(labels, V)).sum(1) / nn
    assert ((b["seq_logps"].double() - seq).abs() <= seq_tol + U * seq.abs()).all()
    h_tol = beta * (seq_tol[:P] + seq_tol[P:]) + U * (h.abs() + 1)
    assert ((b["margins"].double() - h).abs() <= h_tol).all()
    slope = (2 * (h - 0.5).abs().max() + 1) if c["kind"] == "squared" else 1.0  # |f'| nearby
    assert (b["loss"][0].double() - loss).abs() <= slope * h_tol.max() + 2 * U * (loss + 1)
    # f'' is at most 2, and f' is never closer to 0 than the smallest coefficient here
    step = torch.where(coef != 0, coef.abs(), torch.inf).amin(1)  # the coefficient of each sequence
    err = 2 * beta * h_tol.repeat(2) / P / nn / step
    assert torch.isfinite(err).all()
    check_grad(d, before, labels, 0.5 * coef, (err[:, None] + 4 * U).amax())
    assert torch.allclose(b["coef"].double(), 0.5 * torch.where(step.isinf(), b["coef"].double() * 2, coef.sum(1) / n.clamp_min(1)),
                          rtol=float(err.amax() + 4 * U), atol=0)
    assert all(torch.equal(b[k], b2[k]) for k in ("loss", "seq_logps", "margins", "token_logps"))


# ------------------------------------------------------------------------------------------------ policy
def ref_policy(lp, labels, V, old, ref, adv, low, high, kl_coef, by_sequence):
    on = scored(labels, V).double()
    v = lp.clone().requires_grad_(True)
    if by_sequence:
        w = on / (on.sum(1, keepdim=True).clamp_min(1) * (on.sum(1) > 0).sum().clamp_min(1))
    else:
        w = on / on.sum().clamp_min(1)
    a = adv.double() if adv.dim() == 2 else adv.double()[:, None]
    r = torch.exp(v - torch.where(on > 0, old.double(), 0.0))
    c = r.clamp(1 - low, 1 + high)
    pg = (w * -torch.minimum(r * a, c * a)).sum()
    kl = torch.zeros_like(pg)
    if ref is not None:
        q = torch.where(on > 0, ref.double(), 0.0) - v
        kl = (w * (torch.exp(q) - q - 1)).sum()
    loss = pg + kl_coef * kl
    (d,) = torch.autograd.grad(loss, v)
    cut = (w * (c * a < r * a)).sum()
    return torch.stack([loss, pg, kl, cut]).detach(), d, w


POLICY = [
    dict(B=1, T=1, V=17, dtype=torch.float32),
    dict(B=64, T=1, V=50304, dtype=torch.bfloat16),
    dict(B=4, T=33, V=1000, dtype=torch.bfloat16, kl=0.1, by_sequence=True),
    dict(B=3, T=21, V=50257, dtype=torch.float16, kl=0.04, per_token=True, layout="shifted"),
    dict(B=2, T=7, V=70001, dtype=torch.float32, by_sequence=True, per_token=True, kl=0.5, layout="padded"),
    dict(B=700, T=3, V=65, dtype=torch.bfloat16, kl=0.01, by_sequence=True),
    dict(B=2, T=900, V=200, dtype=torch.float32, per_token=True, layout="time first"),
    dict(B=3, T=8, V=120, dtype=torch.float32, kl=0.2, by_sequence=True, empty=True),
    dict(B=4, T=90, V=50304, dtype=torch.bfloat16, kl=0.1, by_sequence=True, layout="shifted"),
    dict(B=3, T=100, V=50257, dtype=torch.float32, kl=0.04, per_token=True),
    dict(B=2, T=160, V=8203, dtype=torch.float16, by_sequence=True, kl=0.1, empty=True),
    dict(B=400, T=1, V=33000, dtype=torch.float16, layout="padded"),
    dict(B=1, T=310, V=70001, dtype=torch.float32, per_token=True),
    dict(B=300, T=2, V=130, dtype=torch.bfloat16, kl=0.1, by_sequence=True),
    dict(B=33, T=9, V=20000, dtype=torch.bfloat16, by_sequence=True, empty=True),
    dict(B=9000, T=1, V=64, dtype=torch.bfloat16, kl=0.1, by_sequence=True),
    dict(B=40, T=300, V=1201, dtype=torch.float16, kl=0.05, by_sequence=True, empty=True),
]


@pytest.mark.parametrize("c", POLICY, ids=lambda c: "-".join(str(v) for v in c.values()))
@pytest.mark.parametrize("inplace", [False, True])
def test_policy_loss(cuda, c, inplace):
    B, T, V = c["B"], c["T"], c["V"]
    x, labels = make(B, T, V, c["dtype"], c.get("layout", "plain"), masked=0.0 if T == 1 else 0.3)
    if B == 1:
        labels[0, 0] = 3
    if c.get("empty"):
        labels[1] = IGNORE
    before = x.clone()
    on = scored(labels, V)
    lp, _ = ref_logps(before, labels)
    g = torch.Generator(device=cuda).manual_seed(11)
    kl_coef, low, high = c.get("kl", 0.0), 0.2, 0.28
    # keep log ratios 1e-3 away from the clip borders, where the gradient jumps
    shift = 0.25 * torch.randn(B, T, device=cuda, generator=g, dtype=torch.float64)
    for edge in (-torch.log(torch.tensor(1 + high)).item(), -torch.log(torch.tensor(1 - low)).item()):
        shift = torch.where((shift - edge).abs() < 1e-3, shift + 4e-3, shift)
    old = (lp + shift).float()
    ref = (lp + 0.4 * torch.randn(B, T, device=cuda, generator=g)).float() if kl_coef else None
    old[~on] = float("nan")  # what masked places hold must not matter
    if ref is not None:
        ref[~on] = float("inf")
    adv = torch.randn(*((B, T) if c.get("per_token") else (B,)), device=cuda, generator=g)
    by_sequence = c.get("by_sequence", False)
    stats, coef, w = ref_policy(lp, labels, V, old, ref, adv, low, high, kl_coef, by_sequence)
    n = lambda *s: torch.full(s, 7.0, device=cuda)  # noqa: E731
    b = dict(token_logps=n(B, T), counts=torch.full((B,), -5, device=cuda, dtype=torch.int32), stats=n(4), lse=n(B, T), coef=n(B, T))
    b2 = {k: torch.empty_like(v) for k, v in b.items() if k not in ("lse", "coef")}
    nv.policy_loss(x, labels, old, adv, ref, clip_low=low, clip_high=high, kl_coef=kl_coef, by_sequence=by_sequence, **b2)
    d = x if inplace else torch.full((B, T, V), 3.0, device=cuda, dtype=c["dtype"])
    nv.policy_loss(x, labels, old, adv, ref, dlogits=d, clip_low=low, clip_high=high, kl_coef=kl_coef, by_sequence=by_sequence,
                   grad_scale=2.0, **b)
    assert torch.equal(b["counts"].long(), on.sum(1))
    tol = rel(V) + U * lp.abs()  # of a log-probability
    assert ((b["token_logps"].double() - lp).abs() <= tol).all()
    a = adv.abs().double() if adv.dim() == 2 else adv.abs().double()[:, None]
    grow = torch.exp(0.5 + shift.abs()) * (a + 1e-9)  # |d pg / d lp|
    q = torch.where(on, (ref if ref is not None else lp.float()).double(), lp) - lp
    each = w * (2 * tol + 4 * U) * (grow + (kl_coef + 1) * (torch.exp(q) + 1) * (ref is not None))
    assert ((b["stats"][:3].double() - stats[:3]).abs() <= each.sum() + 2 * U * stats[:3].abs()).all()
    assert (b["stats"][3].double() - stats[3]).abs() <= 2 * U
    # d = w (-A r + k (1 - e^q)): absolute error from lp, as a share of the coefficient where it is not 0
    err = w * (tol + 4 * U) * (grow + kl_coef * (torch.exp(q) + 1))
    assert ((b["coef"].double() - 2 * coef).abs() <= 2 * err + 2 * U * coef.abs()).all()
    check_grad(d, before, labels, b["coef"], 4 * U)  # the rows, given the coefficients checked above
    # without a gradient another kernel may serve, whose sums run in another order
    assert torch.equal(b["counts"], b2["counts"])
    assert ((b["token_logps"] - b2["token_logps"]).abs() <= 2 * tol).all()
    assert ((b["stats"] - b2["stats"]).abs()[:3] <= 2 * each.sum() + 4 * U * stats[:3].abs()).all()


def test_nothing_scored_gives_zeros(cuda):
    x = torch.full((2, 4, 33), float("nan"), device=cuda)
    labels = torch.full((2, 4), IGNORE, device=cuda)
    z = lambda *s: torch.full(s, 7.0, device=cuda)  # noqa: E731
    d = torch.empty_like(x)
    stats, lp = z(4), z(2, 4)
    nv.policy_loss(x, labels, z(2, 4), z(2), z(2, 4), token_logps=lp, counts=torch.ones(2, device=cuda, dtype=torch.int32),
                   stats=stats, dlogits=d, kl_coef=0.1, by_sequence=True)
    assert (stats == 0).all() and (lp == 0).all() and (d == 0).all()
    b = _pref_buffers(2, 4, cuda)
    nv.preference_loss(x, labels, None, dlogits=d, average=True, **b)
    assert (b["seq_logps"] == 0).all() and (b["margins"] == 0).all() and (d == 0).all()
    assert abs(b["loss"].item() - 0.6931471805599453) <= 0.7 * U


# ------------------------------------------------------------------------------------------------ autograd, differences
def test_gradients_against_differences(cuda):
    """Central differences of the fp32 losses along a random direction: the error of the difference is at most
    eps^2 |f'''| / 6 (about 1e-4 of the slope for eps = 0.01 here) plus 2 u |f| / eps (1.2e-5)."""
    x, labels = make(4, 6, 50, torch.float32, masked=0.2)
    old, _ = ref_logps(x, labels)
    adv, ref = torch.randn(4, device=cuda), (old + 0.3 * torch.randn_like(old)).float()
    funcs = [
        lambda t: losses.preference_loss(t, labels, beta=0.5, kind="sigmoid", label_smoothing=0.1)[0],
        lambda t: losses.preference_loss(t, labels, ref.sum(1), beta=0.3, kind="squared")[0],
        lambda t: losses.policy_loss(t, labels, old.float(), adv, ref, kl_coef=0.3, clip_low=0.5, clip_high=0.5)[0],
        lambda t: losses.token_logprobs(t, labels).mean(),
    ]
    for f in funcs:
        leaf = x.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(f(leaf) * 3.0, leaf)
        way = torch.randn_like(x)
        slope = (g.double() * way.double()).sum() / 3.0
        eps = 0.01
        diff = (f(x + eps * way).double() - f(x - eps * way).double()) / (2 * eps)
        assert (diff - slope).abs() <= 1e-2 * slope.abs() + 1e-3, (diff, slope)


def test_autograd_functions_match_the_fused_gradient(cuda):
    x, labels = make(6, 11, 1003, torch.bfloat16, "shifted")
    old, _ = ref_logps(x, labels)
    old = (old + 0.1).float()
    adv = torch.randn(6, device=cuda)
    fused = torch.empty(6, 11, 1003, device=cuda, dtype=torch.bfloat16)
    n = lambda *s: torch.empty(*s, device=cuda)  # noqa: E731
    nv.policy_loss(x, labels, old, adv, token_logps=n(6, 11), counts=torch.empty(6, device=cuda, dtype=torch.int32), stats=n(4),
                   dlogits=fused)
    leaf = x.detach().requires_grad_(True)
    loss, stats, logps = losses.policy_loss(leaf, labels, old, adv)
    loss.backward()
    tol = 2.0 ** -7 * fused.float().abs() + 1e-9  # both are half a bf16 step from the same fp32 number
    assert ((leaf.grad.float() - fused.float()).abs() <= tol).all()
    assert not stats.requires_grad and not logps.requires_grad
    with pytest.raises(RuntimeError):
        (g,) = torch.autograd.grad(losses.token_logprobs(leaf, labels).sum(), leaf, create_graph=True)
        g.sum().backward()


def test_repeats_streams_and_graphs_give_equal_bits(cuda):
    x, labels = make(4, 30, 5003, torch.bfloat16)
    old = torch.randn(4, 30, device=cuda) - 8
    adv = torch.randn(4, device=cuda)

    def call(out):
        n = lambda *s: torch.empty(*s, device=cuda)  # noqa: E731
        st, d, d2, b = n(4), torch.empty_like(x), torch.empty_like(x), _pref_buffers(4, 30, cuda)
        nv.policy_loss(x, labels, old, adv, token_logps=n(4, 30), counts=torch.empty(4, device=cuda, dtype=torch.int32), stats=st, dlogits=d)
        nv.preference_loss(x, labels, None, dlogits=d2, **b)
        out += [st, d, d2, b["loss"], b["margins"]]

    first = []
    call(first)
    torch.cuda.synchronize()
    s1, s2, got = torch.cuda.Stream(), torch.cuda.Stream(), ([], [])
    for s, g in ((s1, got[0]), (s2, got[1])):
        with torch.cuda.stream(s):
            call(g)
    torch.cuda.synchronize()
    graphs, kept = [], []
    for _ in range(2):  # two graphs over the same inputs
        g, out = torch.cuda.CUDAGraph(), []
        with torch.cuda.graph(g):
            call(out)
        graphs.append(g)
        kept.append(out)
    for g in graphs + graphs[::-1]:
        g.replay()
    torch.cuda.synchronize()
    for other in (*got, *kept):
        assert all(torch.equal(a, b) for a, b in zip(first, other))


def test_rows_past_32_bit_offsets(cuda):
    B, T, V = 2, 22000, 50304  # 2.2e9 elements
    x = torch.zeros(B, T, V, device=cuda, dtype=torch.bfloat16)
    labels = torch.full((B, T), IGNORE, device=cuda)
    at = [(0, 0), (1, 20800), (1, T - 1)]
    for b, t in at:
        x[b, t] = torch.randn(V, device=cuda).bfloat16()
        labels[b, t] = V - 1
    lp, lse = torch.empty(B, T, device=cuda), torch.empty(B, T, device=cuda)
    nv.token_logprobs(x, labels, lp, lse=lse)
    rows = torch.stack([x[b, t] for b, t in at])[None].clone()
    ys = torch.full((1, 3), V - 1, device=cuda)
    want, _ = ref_logps(rows, ys)
    assert ((torch.stack([lp[b, t] for b, t in at]).double() - want[0]).abs() <= rel(V) + U * want[0].abs()).all()
    nv.token_logprobs_bwd(x, labels, lse, torch.ones(B, T, device=cuda), x)
    check_grad(torch.stack([x[b, t] for b, t in at])[None], rows, ys, torch.ones(1, 3, device=cuda))
    assert (x[1, 20799] == 0).all() and (x[1, 20801] == 0).all()
