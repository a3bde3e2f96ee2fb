"""Arguments that the post-training operators refuse, checked on the host before anything is launched (CPU tensors
suffice: a call that passed the checks would fail for having no CUDA tensors)."""
import pytest
import torch

from rgpt_b200 import native as nv
from rgpt_b200.optimizer import DistMuon, Muon

F, L = torch.float32, torch.int64


def z(*s, dt=F):
    return torch.zeros(*s, dtype=dt)


def pref(B=4, T=3, V=8, **kw):
    a = dict(logits=z(B, T, V), labels=z(B, T, dt=L), ref_logps=z(B), token_logps=z(B, T), lse=z(B, T), seq_logps=z(B),
             margins=z(B // 2), coef=z(B), loss=z(1))
    a.update(kw)
    nv.preference_loss(a.pop("logits"), a.pop("labels"), a.pop("ref_logps"), **a)


def policy(B=4, T=3, V=8, **kw):
    a = dict(logits=z(B, T, V), labels=z(B, T, dt=L), old_logps=z(B, T), advantages=z(B), ref_logps=z(B, T),
             token_logps=z(B, T), counts=z(B, dt=torch.int32), stats=z(4))
    a.update(kw)
    ins = [a.pop(k) for k in ("logits", "labels", "old_logps", "advantages", "ref_logps")]
    nv.policy_loss(*ins, **a)


@pytest.mark.parametrize("kw,what", [
    (dict(kind="other"), "kind"), (dict(label_smoothing=0.6), "label_smoothing"),
    (dict(kind="hinge", label_smoothing=0.1), "label_smoothing"), (dict(beta=0.0), "beta"), (dict(beta=float("inf")), "beta"),
    (dict(logits=z(3, 3, 8)), "pair"), (dict(logits=z(0, 3, 8)), "pair"), (dict(logits=z(4, 0, 8)), "pair"),
    (dict(logits=z(4, 8)), "pair"), (dict(logits=z(4, 3, 16)[..., ::2]), "unit stride"), (dict(labels=z(4, 2, dt=L)), "labels"),
    (dict(labels=z(3, 4, dt=L).t()), "labels"), (dict(ref_logps=z(2)), "ref_logps"), (dict(margins=z(4)), "margins"),
    (dict(dlogits=z(4, 3, 9)), "dlogits"), (dict(dlogits=z(1, 3, 8).expand(4, 3, 8)), "overlap"),
])
def test_preference_loss_refuses(kw, what):
    with pytest.raises(ValueError, match=what):
        pref(**kw)


@pytest.mark.parametrize("kw", [dict(logits=z(4, 3, 8, dt=torch.float64)), dict(labels=z(4, 3, dt=torch.int32)),
                                dict(token_logps=z(4, 3, dt=torch.bfloat16))])
def test_preference_loss_refuses_types(kw):
    with pytest.raises(TypeError):
        pref(**kw)


@pytest.mark.parametrize("kw,what", [
    (dict(clip_low=-0.1), "clip_low"), (dict(clip_low=1.1), "clip_low"), (dict(clip_high=-1.0), "clip_high"),
    (dict(kl_coef=0.1, ref_logps=None), "ref_logps"), (dict(advantages=z(3)), "advantages"), (dict(old_logps=z(4)), "old_logps"),
    (dict(stats=z(3)), "stats"), (dict(coef=z(4)), "coef"), (dict(dlogits=z(4, 3, 8).transpose(0, 1)), "dlogits"),
])
def test_policy_loss_refuses(kw, what):
    with pytest.raises(ValueError, match=what):
        policy(**kw)


def test_policy_loss_refuses_types_and_no_tokens():
    with pytest.raises(TypeError):
        policy(counts=z(4, dt=L))
    with pytest.raises(ValueError, match="token"):
        policy(B=0)
    with pytest.raises(ValueError, match="token"):
        policy(T=0)


def test_gradient_memory_is_the_logits_or_apart():
    held = z(2 * 4 * 3 * 8)
    x = held[:96].view(4, 3, 8)
    policy_args = dict(logits=x)
    with pytest.raises(ValueError, match="share no memory"):
        policy(**policy_args, dlogits=held[8:104].view(4, 3, 8))
    for d in (x, held[96:].view(4, 3, 8), x.view(4, 3, 8)):  # passes the checks, then wants CUDA tensors
        with pytest.raises(RuntimeError, match="CUDA"):
            policy(**policy_args, dlogits=d)
    wide = z(3, 4, 8).transpose(0, 1)  # time-first memory is fine for both
    with pytest.raises(RuntimeError, match="CUDA"):
        policy(logits=wide, dlogits=wide)


def test_token_logprobs_refuses():
    x, y, o = z(4, 8), z(4, dt=L), z(4)
    with pytest.raises(ValueError, match="labels"):
        nv.token_logprobs(x, z(5, dt=L), o)
    with pytest.raises(ValueError, match="logps"):
        nv.token_logprobs(x, y, z(8)[::2])
    with pytest.raises(ValueError, match=r"\[M, V\]"):
        nv.token_logprobs(z(8), y, o)
    with pytest.raises(TypeError):
        nv.token_logprobs_bwd(x, y, o, z(4, dt=torch.float64), x)
    with pytest.raises(RuntimeError, match="CUDA"):
        nv.token_logprobs(x, y, o)


@pytest.mark.parametrize("x,w,what", [
    (z(4, 8, dt=torch.bfloat16), z(9, 16, dt=torch.bfloat16), "share K"), (z(4, 12, dt=torch.bfloat16), z(9, 12, dt=torch.bfloat16), "multiple of 8"),
    (z(8, 4, dt=torch.bfloat16).t(), z(9, 8, dt=torch.bfloat16), "unit stride"), (z(4, 8, dt=torch.bfloat16), z(0, 8, dt=torch.bfloat16), "V >= 1"),
    (z(1, 8, dt=torch.bfloat16).expand(4, 8), z(9, 8, dt=torch.bfloat16), "row stride"),
])
def test_linear_logprobs_refuses(x, w, what):
    with pytest.raises(ValueError, match=what):
        nv.linear_logprobs(x, w, z(x.shape[0], dt=L), z(x.shape[0]))


def test_linear_logprobs_refuses_types_scratch_and_outputs():
    x, w, y, o = z(4, 8, dt=torch.bfloat16), z(9, 8, dt=torch.bfloat16), z(4, dt=L), z(4)
    with pytest.raises(TypeError):
        nv.linear_logprobs(x.float(), w, y, o)
    with pytest.raises(ValueError, match="part"):
        nv.linear_logprobs(x, w, y, o, part=z(7))
    with pytest.raises(ValueError, match="dx"):
        nv.linear_logprobs_bwd(x, w, y, o, o, z(4, 9), None)
    with pytest.raises(ValueError, match="dw"):
        nv.linear_logprobs_bwd(x, w, y, o, o, None, z(9, 8, dt=torch.float16))
    for dx, dw in ((x, None), (None, w)):
        with pytest.raises(ValueError, match="share no memory"):
            nv.linear_logprobs_bwd(x, w, y, o, o, dx, dw)
    with pytest.raises(ValueError, match="row stride"):
        nv.linear_logprobs_bwd(x, w, y, o, o, z(1, 8).expand(4, 8), None)
    with pytest.raises(ValueError, match="chunk_rows"):
        nv.linear_logprobs_bwd(x, w, y, o, o, None, None, chunk_rows=0)


def test_adamw8_moments_refuses():
    p, q, s = z(300), z(300, dt=torch.uint8), z(2)
    for bad in ((p, q[:299], s, q, s), (p, q, z(1), q, s), (p, q, s, q, z(3))):
        with pytest.raises(ValueError, match="codes|scales"):
            nv.adamw8_moments(*bad)
    with pytest.raises(TypeError):
        nv.adamw8_moments(p, q.int(), s, q, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        nv.adamw8_moments(p, q, s, q, s)


def test_adam_state_bits():
    p = torch.nn.Parameter(z(8))
    with pytest.raises(ValueError, match="adam_state_bits"):
        Muon([{"params": [p], "use_muon": False}], adam_state_bits=16)
    opt = Muon([{"params": [p], "use_muon": False, "adam_state_bits": 4}])
    p.grad = z(8)
    with pytest.raises(ValueError, match="adam_state_bits"):
        opt.step()
    with pytest.raises(ValueError, match="sharded_state"):
        DistMuon([{"params": [p], "use_muon": False}], sharded_state=True, adam_state_bits=8)
    with pytest.raises(ValueError, match="no AdamW moments"):
        opt.adam_moments(p)
