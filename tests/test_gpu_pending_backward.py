"""Passes of one model that come between a loss and its backward. The engine keeps one set of activations a batch shape:
a loss whose activations another pass has replaced refuses its backward, one whose activations are still there gives the
gradient that it would have given at once."""
import pytest
import torch

from rgpt_b200.graph import GraphedTrainStep
from rgpt_b200.model import GPT
from rgpt_b200.optimizer import Muon, trainer_param_groups

pytestmark = pytest.mark.gpu

CFG = dict(name="t", d_model=128, n_heads=2, n_layers=2, vocab_size=512, max_seq_len=64, dropout=0.0, norm_type="rmsnorm",
           norm_eps=1e-6, qk_normtype="f_rmsnorm", activation_type="squared_relu", use_layer_scale=False, g1_gate=True,
           n_recur=1, cal_halt_loss=False, detach_recur=False, tie_word_embeddings=False, pad_token_id=-100)


def build(cuda, **kw):
    torch.manual_seed(0)
    return GPT(**{**CFG, **kw}).to(cuda).train()


def batch(cuda, B=4, T=31, seed=1):
    g = torch.Generator(device=cuda).manual_seed(seed)
    ids = torch.randint(0, 512, (B, T + 1), device=cuda, generator=g)
    labels = ids[:, 1:].clone()
    labels[:, : T // 4] = -100
    return ids[:, :-1], labels


def losses_of(model, ids, labels):
    old, adv = torch.full(labels.shape, -6.0, device=ids.device), torch.linspace(-1, 1, ids.shape[0], device=ids.device)
    return {"preference": lambda: model.preference_loss(ids, labels, beta=0.3)[0],
            "policy": lambda: model.policy_loss(ids, labels, old, adv)[0],
            "loss": lambda: model.forward_loss(ids, labels)[0],
            "logits": lambda: model(ids)[0].float().square().mean()}


def passes(model, ids, labels):
    quiet = {k: f for k, f in losses_of(model, ids, labels).items()}

    def without_grad(f):
        with torch.no_grad():
            return f()

    out = {"scores": lambda: model.token_logprobs(ids, labels), "losses": lambda: model.token_losses(ids, labels)}
    out.update({f"{k} with gradient": f for k, f in quiet.items()})
    out.update({k: lambda f=f: without_grad(f) for k, f in quiet.items()})
    return out


@pytest.mark.parametrize("kind", ["preference", "policy", "loss", "logits"])
def test_a_replaced_pass_refuses_its_backward(cuda, kind):
    model = build(cuda)
    ids, labels = batch(cuda)
    other = batch(cuda, seed=2)
    for name, between in passes(model, *other).items():
        loss = losses_of(model, ids, labels)[kind]()
        kept = between()
        with pytest.raises(RuntimeError, match="another pass"):
            loss.backward()
        if "gradient" in name:  # the later pass still has its activations
            kept.backward()
    first, second = losses_of(model, ids, labels)[kind](), losses_of(model, *other)["loss"]()
    with pytest.raises(RuntimeError, match="another pass"):
        (first + 0.5 * second).backward()


def test_losses_of_one_step_add_up(cuda):
    """Each backward before the next forward: the gradients add up. Split-K weight gradients are summed by fp32 atomics,
    whose order differs between runs: 2^-12 of a gradient's norm leaves room for thousands of roundings of 2^-24."""
    model = build(cuda)
    ids, labels = batch(cuda)
    want = {n: torch.zeros_like(p) for n, p in model.named_parameters()}
    for kind in ("preference", "loss"):
        model.engine().zero_grad()
        losses_of(model, ids, labels)[kind]().backward()
        for n, p in model.named_parameters():
            want[n] += p.grad
    model.engine().zero_grad()
    for kind in ("preference", "loss"):
        losses_of(model, ids, labels)[kind]().backward()
    for n, p in model.named_parameters():
        assert (p.grad - want[n]).norm() <= 2.0 ** -12 * want[n].norm() + 1e-12, n


@pytest.mark.parametrize("recur", [1, 3])
@pytest.mark.parametrize("first,then", [((2, 12), (4, 31)), ((4, 31), (1, 9))])
def test_a_pass_of_another_shape_changes_nothing(cuda, recur, first, then):
    """The other shape has activations, ids and dropout masks of its own, the halting heads included."""
    model = build(cuda, n_recur=recur, cal_halt_loss=recur > 1, dropout=0.1)
    eng = model.engine()
    ids, labels = batch(cuda, *first)
    other = batch(cuda, *then, seed=2)
    for kind in ("preference", "policy", "loss"):
        grads = []
        for interrupted in (False, True):
            eng.zero_grad()
            eng.drop_seed.fill_(12345)
            loss = losses_of(model, ids, labels)[kind]()
            if interrupted:
                model.token_logprobs(*other)
                model.forward_loss(*other)
                model.eval()
                model.token_losses(*other)
                model.train()
            loss.backward()
            grads.append({n: p.grad.clone() for n, p in model.named_parameters()})
        for n in grads[0]:
            assert (grads[0][n] - grads[1][n]).norm() <= 2.0 ** -12 * grads[0][n].norm() + 1e-12, (kind, n)
        assert grads[0]["embs.weight"].norm() > 0


def test_a_replayed_step_replaces_the_activations_too(cuda):
    model = build(cuda)
    ids, labels = batch(cuda, 2, 31)
    step = GraphedTrainStep(model, Muon(trainer_param_groups(model), lr=0.0), 2, 31, warmup=1)
    tokens = torch.randint(0, 512, (1, 2, 32), device=cuda)
    for _ in range(2):  # eager, then captured: no other graph of the same leaves may be alive during a capture
        step(tokens)
    for _ in range(2):
        loss = losses_of(model, ids, labels)["policy"]()
        step(tokens)
        with pytest.raises(RuntimeError, match="another pass"):
            loss.backward()
    losses_of(model, ids, labels)["policy"]().backward()
    torch.cuda.synchronize()
    step.release()
