"""The post-training operators as a run uses them together: a frozen reference and the sampling policy score labels
without logits, the policy trains on the preference or the policy loss, and AdamW holds its moments in 8 bits."""
import copy

import pytest
import torch

from rgpt_b200 import losses
from rgpt_b200.model import GPT
from rgpt_b200.optimizer import Muon, trainer_param_groups

pytestmark = pytest.mark.gpu

CFG = dict(name="t", d_model=128, n_heads=2, n_layers=2, vocab_size=512, max_seq_len=64, dropout=0.0, norm_type="rmsnorm",
           norm_eps=1e-6, qk_normtype="f_rmsnorm", activation_type="squared_relu", use_layer_scale=False, g1_gate=True,
           n_recur=1, cal_halt_loss=False, detach_recur=False, tie_word_embeddings=False, pad_token_id=-100)


def build(cuda, **kw):
    torch.manual_seed(0)
    return GPT(**{**CFG, **kw}).to(cuda).train()


def batch(cuda, B=4, T=31):
    g = torch.Generator(device=cuda).manual_seed(1)
    ids = torch.randint(0, 512, (B, T + 1), device=cuda, generator=g)
    labels = ids[:, 1:].clone()
    labels[:, :9] = -100
    labels[1, 20:] = -100
    return ids[:, :-1], labels


@pytest.mark.parametrize("recur", [1, 3])
def test_model_losses_match_autograd_over_its_logits(cuda, recur):
    """Same logits, same kernels: values equal; the fused gradient enters the same native backward as the bf16 gradient
    of the logits that autograd hands over, each half a bf16 step (2^-8) from the same number, so weight gradients
    (sums of such terms) agree to 2^-7 of their size, with room for the sums' own bf16 roundings: 2^-6."""
    model = build(cuda, n_recur=recur, cal_halt_loss=recur > 1)
    ids, labels = batch(cuda)
    ref = torch.randn(4, device=cuda) * 3 - 120
    old, adv = model.token_logprobs(ids, labels), torch.randn(4, device=cuda)
    fused = [lambda: model.preference_loss(ids, labels, ref, beta=0.3),
             lambda: model.policy_loss(ids, labels, old, adv, old - 0.1, kl_coef=0.2, by_sequence=True)]
    plain = [lambda x: losses.preference_loss(x, labels, ref, beta=0.3),
             lambda x: losses.policy_loss(x, labels, old, adv, old - 0.1, kl_coef=0.2, by_sequence=True)]
    for f, p in zip(fused, plain):
        out = f()
        model.engine().zero_grad()
        (2.0 * out[0]).backward()
        got = {n: q.grad.clone() for n, q in model.named_parameters()}
        model.engine().zero_grad()
        want = p(model(ids)[0])
        (2.0 * want[0]).backward()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        for n, q in model.named_parameters():
            assert (got[n] - q.grad).norm() <= 2.0 ** -6 * q.grad.norm() + 1e-9, n
        assert got["lm_head.weight"].norm() > 0
        with torch.no_grad():
            quiet = f()
        assert all(torch.equal(a, b) for a, b in zip(out, quiet))


def test_token_logprobs_agree_with_the_losses_and_with_token_losses(cuda):
    model = build(cuda)
    ids, labels = batch(cuda)
    lp = model.token_logprobs(ids, labels)
    _, stats, seen = model.policy_loss(ids, labels, lp, torch.ones(4, device=cuda))
    u = 2.0 ** -24
    tol = 2 * (40 + 512 / 128) * u + 2 * u * lp.abs()  # only the order of the sums differs
    assert ((lp - seen).abs() <= tol).all()
    assert abs(stats[0].item() + 1.0) <= 2 * tol.max().item() + 2 * u and stats[3] == 0  # on-policy: ratios of 1
    ce = model.eval().token_losses(ids, labels)
    assert ((lp + ce).abs() <= tol + 4 * u * ce.abs()).all()


def test_preference_training_together(cuda):
    policy = build(cuda)
    reference = copy.deepcopy(policy).eval()
    ids, labels = batch(cuda)
    opt = Muon(trainer_param_groups(policy), lr=1e-3, weight_decay=0.0, muon_lr_multiplier=20.0, adam_state_bits=8)
    ref = reference.token_logprobs(ids, labels).sum(1)
    margins = []
    for _ in range(6):
        loss, seq, h = policy.preference_loss(ids, labels, ref, beta=0.1)
        loss.backward()
        opt.step()
        opt.zero_grad()
        margins.append(h.mean().item())
    # the first step starts at the reference: log-probabilities that differ in the order of their sums alone
    assert abs(margins[0]) <= 0.1 * 64 * 2 ** -16
    assert all(torch.isfinite(p).all() for p in policy.parameters())
    moments = [opt.adam_moments(p) for g in opt.param_groups if not g["use_muon"] for p in g["params"]]
    assert all(torch.isfinite(m).all() and (v >= 0).all() for m, v in moments)
    assert any("exp_avg_q8" in s for s in opt.state.values())
    assert torch.equal(policy.engine().lm_w, policy.lm_head.weight.bfloat16())
    # the frozen reference is as it was
    assert torch.equal(reference.token_logprobs(ids, labels).sum(1), ref)


def test_policy_training_step_in_a_graph(cuda):
    """Forward, loss, backward and an 8-bit AdamW + Muon step captured once and replayed equal the eager steps."""
    ids, labels = batch(cuda)
    adv = torch.tensor([1.0, -1.0, 0.5, -0.5], device=cuda)

    def run(graphed):
        model = build(cuda)
        opt = Muon(trainer_param_groups(model), lr=1e-3, adam_state_bits=8)
        opt.use_device_hparams()
        old = model.token_logprobs(ids, labels)

        def step():
            opt.zero_grad()
            loss, stats, _ = model.policy_loss(ids, labels, old, adv, old, kl_coef=0.1)
            loss.backward()
            opt.step()
            return stats

        for _ in range(2):
            opt.stage_device_hparams()
            step()
        g = None
        for _ in range(3):
            opt.stage_device_hparams()
            if not graphed:
                stats = step()
                continue
            if g is None:
                torch.cuda.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    stats = step()
            g.replay()
        torch.cuda.synchronize()
        return model, stats.clone()

    (a, sa), (b, sb) = run(False), run(True)
    # split-K weight gradients are summed by fp32 atomics, whose order differs between runs
    assert (sa - sb).abs().max() <= 1e-4 * sa.abs().max()
    for p, q in zip(a.parameters(), b.parameters()):
        assert (p - q).norm() <= 1e-2 * p.norm()
