"""The two ways the post-training operators check their arguments, in one C++ step and in Python, give the kernels the
same arguments and refuse the same calls."""
import pytest
import torch

from rgpt_b200 import native as nv

pytestmark = pytest.mark.gpu
BF, F16, F, L, D, I32, U8 = (torch.bfloat16, torch.float16, torch.float32, torch.int64, torch.float64, torch.int32,
                             torch.uint8)


def z(*s, dt=F):
    return torch.zeros(*s, dtype=dt, device="cuda")


def logits(kind):
    if kind == "rows":
        return z(6, 11, dt=BF)
    if kind == "one column":
        return z(4, 3, 2, dt=F16)[..., :1]
    if kind == "time first":
        return z(3, 4, 9).transpose(0, 1)
    if kind == "shifted":
        return z(4, 4, 9, dt=BF)[:, :-1]
    if kind == "one":
        return z(2, 1, 1)
    return z(4, 3, 10, dt=F16)[..., 1:]


KINDS = ["rows", "one column", "time first", "shifted", "one", "odd start"]


def grads(x):
    return [None, x, torch.empty_like(x), z(*x.shape, dt=x.dtype), z(*x.shape[:-1], x.shape[-1] + 5, dt=x.dtype)[..., 2:-3]]


def calls():
    for kind in KINDS:
        x = logits(kind)
        s, B = x.shape[:-1], x.shape[0]
        y = z(*s, dt=L)
        for lse in (None, z(*s)):
            yield f"token {kind}", lambda z, x=x, y=y, s=s, lse=lse: nv.token_logprobs(x, y, z(*s), lse=lse, ignore_index=7)
        for i, d in enumerate(grads(x)):
            if d is not None:
                yield f"token bwd {kind} {i}", lambda z, x=x, y=y, s=s, d=d: nv.token_logprobs_bwd(x, y, z(*s), z(*s), d)
            for per_token in (False, True):
                yield f"policy {kind} {i}", lambda z, x=x, y=y, s=s, B=B, d=d, t=per_token: nv.policy_loss(
                    x, y, z(*s), z(*s) if t else z(B), z(*s) if t else None, token_logps=z(*s), counts=z(B, dt=I32), stats=z(4),
                    lse=z(*s) if t else None, coef=None if t else z(*s), dlogits=d, by_sequence=t, kl_coef=0.1 * t)
            if len(s) == 2:
                yield f"preference {kind} {i}", lambda z, x=x, y=y, s=s, B=B, d=d, i=i: nv.preference_loss(
                    x, y, z(B) if i % 2 else None, token_logps=z(*s), lse=z(*s), seq_logps=z(B), margins=z(B // 2),
                    coef=z(B), loss=z(1), dlogits=d, scratch=z(*s, dt=D), average=bool(i % 2))
    for M, V, K, ld in ((1, 1, 8, 8), (5, 300, 72, 80), (3, 129, 5, 16)):
        x, w = z(M, ld, dt=BF)[:, :K], z(V, ld, dt=BF)[:, :K]
        for lse in (None, z(M)):
            yield "linear", lambda z, x=x, w=w, M=M, V=V, lse=lse: nv.linear_logprobs(
                x, w, z(M, dt=L), z(M), lse=lse, part=z(4 * M * ((V + 127) // 128) + 3), round_bf16=lse is None)
    for n in (1, 256, 300):
        b = (n + 255) // 256
        yield "moments", lambda z, n=n, b=b: nv.adamw8_moments(z(n), z(n, dt=U8), z(b), z(n, dt=U8), z(b))


def recorded(monkeypatch, call, pack, held):
    """What the call hands to the library; the tensors that it makes are those of `held`, as far as there are any."""
    got, made = [], iter(list(held))

    def again(*s, dt=F):
        t = next(made, None)
        if t is None:
            t = z(*s, dt=dt)
            held.append(t)
        return t

    with monkeypatch.context() as m:
        m.setattr(nv, "_call_on", lambda index, name, *args, kernels=1: got.append((index, name, list(args), kernels)))
        fast = nv._pack if pack else lambda kinds, tensors: None
        m.setattr(nv, "_pack", lambda *a: got.append(fast(*a)) or got[-1])
        call(again)
    return got


def test_same_arguments(cuda, monkeypatch):
    from rgpt_b200 import _fastargs  # built with the kernels
    assert nv._pack is _fastargs.pack
    for name, call in calls():
        held = []
        (packed, a), (_, b) = recorded(monkeypatch, call, True, held), recorded(monkeypatch, call, False, held)
        assert packed is not None, f"{name}: refused by the C++ checks"
        if name == "moments":  # makes its outputs itself
            a[2][4:6] = b[2][4:6] = [0, 0]
        assert a == b, name


def refused():
    x, y, o = z(4, 3, 8), z(4, 3, dt=L), z(4, 3)
    for bad in (z(4, 3, 16)[..., ::2], z(4, 3, 8, dt=D), z(8), torch.zeros(4, 3, 8), z(4, 3, 0)):
        yield lambda bad=bad: nv.token_logprobs(bad, y, o)
    for bad in (z(4, 3, dt=I32), z(3, 4, dt=L).t(), z(12, dt=L), torch.zeros(4, 3, dtype=L)):
        yield lambda bad=bad: nv.token_logprobs(x, bad, o)
    for bad in (z(4, 3, dt=BF), z(4, 6)[:, ::2], z(4), torch.zeros(4, 3)):
        yield lambda bad=bad: nv.token_logprobs(x, y, bad)
        yield lambda bad=bad: nv.token_logprobs(x, y, o, lse=bad)
        yield lambda bad=bad: nv.token_logprobs_bwd(x, y, bad, o, x)
    held = z(200)
    h = held[:96].view(4, 3, 8)
    for bad in (held[8:104].view(4, 3, 8), held[:64].view(2, 4, 8)[:1, :3].expand(4, 3, 8), z(4, 3, 8, dt=BF), z(4, 24),
                torch.zeros(4, 3, 8), z(4, 3, 16)[..., ::2], h.view(3, 4, 8).transpose(0, 1)):
        yield lambda bad=bad: nv.token_logprobs_bwd(h, y, o, o, bad)
        yield lambda bad=bad: nv.policy_loss(h, y, o, z(4), token_logps=o, counts=z(4, dt=I32), stats=z(4), dlogits=bad)
    good = dict(token_logps=o, counts=z(4, dt=I32), stats=z(4))
    for k, bad in (("counts", z(4)), ("counts", z(3, dt=I32)), ("stats", z(8)[::2]), ("stats", z(3)), ("lse", z(4)),
                   ("coef", z(4, 3, dt=F16))):
        yield lambda k=k, bad=bad: nv.policy_loss(x, y, o, z(4), **{**good, k: bad})
    for adv in (z(3), z(4, 3, dt=BF), z(1), torch.zeros(4)):
        yield lambda adv=adv: nv.policy_loss(x, y, o, adv, **good)
    pref = dict(token_logps=o, lse=o, seq_logps=z(4), margins=z(2), coef=z(4), loss=z(1))
    for k, bad in (("margins", z(4)), ("loss", z(2)), ("scratch", z(4, 3)), ("scratch", z(4, 2, dt=D)), ("coef", z(2)),
                   ("seq_logps", z(4, dt=D))):
        yield lambda k=k, bad=bad: nv.preference_loss(x, y, **{**pref, k: bad})
    yield lambda: nv.preference_loss(x, y, z(2), **pref)
    yield lambda: nv.preference_loss(z(3, 3, 8), z(3, 3, dt=L), **pref)
    yield lambda: nv.preference_loss(z(4, 8), z(4, dt=L), token_logps=z(4), lse=z(4), seq_logps=z(4), margins=z(2), coef=z(4),
                                     loss=z(1))
    for a, w in ((z(4, 12, dt=BF), z(9, 12, dt=BF)), (z(4, 8, dt=BF), z(9, 16, dt=BF)), (z(1, 8, dt=BF).expand(4, 8), z(9, 8, dt=BF)),
                 (z(4, 8, dt=BF), z(8, 9, dt=BF).t()), (z(4, 8), z(9, 8)), (z(4, 8, dt=BF), torch.zeros(9, 8, dtype=BF)),
                 (z(4, 8, dt=BF), z(0, 8, dt=BF))):
        yield lambda a=a, w=w: nv.linear_logprobs(a, w, z(4, dt=L), z(4))
    yield lambda: nv.linear_logprobs(z(4, 8, dt=BF), z(9, 8, dt=BF), z(4, dt=L), z(4), part=z(15))
    yield lambda: nv.adamw8_moments(z(300), z(300, dt=U8), z(1), z(300, dt=U8), z(2))
    yield lambda: nv.adamw8_moments(z(300), z(299, dt=U8), z(2), z(300, dt=U8), z(2))


def test_same_refusals(cuda, monkeypatch):
    for pack in (True, False):
        for i, call in enumerate(refused()):
            with pytest.raises((ValueError, TypeError, RuntimeError)):
                recorded(monkeypatch, lambda z: call(), pack, [])
                pytest.fail(f"call {i} went through")


def test_linear_gradients_share_no_memory_with_what_they_read(cuda):
    x, w = z(4, 8, dt=BF), z(9, 8, dt=BF)
    y, o = z(4, dt=L), z(4)
    for dx, dw in ((x, None), (None, w), (x[:, :], z(9, 8)), (z(1, 8).expand(4, 8), None)):
        with pytest.raises(ValueError, match="share no memory|row stride"):
            nv.linear_logprobs_bwd(x, w, y, o, o, dx, dw)


def test_launches_are_counted(cuda):
    """Few tokens are counted by the row kernel, others by kernels of their own; few pairs' mean needs no kernel of its
    own."""
    for P, T, grad, want in ((1, 5, False, 2), (8, 5, True, 3), (9, 5, True, 4), (2, 300, True, 4), (1, 300, True, 3)):
        before = nv._lib.launch_count
        x, m, loss = torch.randn(2 * P, T, 40, device="cuda"), z(P), z(1)
        nv.preference_loss(x, z(2 * P, T, dt=L), token_logps=z(2 * P, T), lse=z(2 * P, T), seq_logps=z(2 * P), margins=m,
                           coef=z(2 * P), loss=loss, dlogits=x if grad else None, kind="squared")
        assert nv._lib.launch_count - before == want
        assert loss.item() == pytest.approx(((m.double() - 0.5) ** 2).mean().item(), rel=1e-6)
    for B, T, by_sequence, want in ((2, 9, False, 2), (33, 2, True, 4), (33, 2, False, 2), (5, 300, False, 4)):
        before = nv._lib.launch_count
        x = torch.randn(B, T, 40, device="cuda")
        st, cn = z(4), z(B, dt=I32)
        nv.policy_loss(x, z(B, T, dt=L), z(B, T), z(B), token_logps=z(B, T), counts=cn, stats=st, by_sequence=by_sequence)
        assert nv._lib.launch_count - before == want
        assert (cn == T).all() and nv._lib.device_error() == 0
