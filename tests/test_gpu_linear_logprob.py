"""Log-probabilities straight from hidden states against the same in 64 bits, and their gradients.

Tolerances: the products accumulate in fp32 on the tensor cores; K terms of size |x||w| carry at most K 2^-23 of
their absolute sum (truncating adds included). That bound, the largest over a row's logits, moves lse by as much
and the label's logit by as much; the sum of exponentials adds (40 + V/128) 2^-24 as in the row kernels, the
additions being one after another within a tile of at most 256 columns. The gradient rows are rounded to bf16
(half a step, 2^-8 of each element: bf16 holds 8 bits), and the GEMMs that follow add K 2^-23 of their absolute sums and half a step
of their own output type.
"""
import pytest
import torch

from rgpt_b200 import losses
from rgpt_b200 import native as nv

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
IGNORE = -100


def make(M, V, K, seed=0, stride=0):
    g = torch.Generator(device="cuda").manual_seed(seed + M + V + K)
    x = torch.randn(M, K + stride, device="cuda", generator=g).bfloat16()[:, :K]
    w = (torch.randn(V, K + stride, device="cuda", generator=g) * 2.0 / K ** 0.5).bfloat16()[:, :K]
    labels = torch.randint(0, V, (M,), device="cuda", generator=g)
    drop = torch.rand(M, device="cuda", generator=g)
    labels[drop < 0.2] = IGNORE
    labels[(drop > 0.2) & (drop < 0.25)] = V
    if M == 1:
        labels[0] = V // 2
    return x, w, labels


def ref(x, w, labels):
    V = w.shape[0]
    on = (labels >= 0) & (labels < V)
    z = x.double() @ w.double().t()
    size = 2 * x.shape[1] * U * (x.double().abs() @ w.double().abs().t()).amax(1)
    lse = torch.logsumexp(z, 1)
    lp = torch.where(on, z.gather(1, labels.clamp(0, V - 1)[:, None])[:, 0] - lse, 0.0)
    return on, z, lse, lp, size


SHAPES = [(1, 1, 8, 0), (1, 50304, 512, 0), (3, 130, 64, 0), (16, 50257, 512, 0), (128, 129, 72, 8), (257, 1000, 1024, 0),
          (300, 4097, 128, 64), (1000, 383, 512, 0), (513, 33000, 1032, 0), (5000, 300, 64, 0),
          # many tiles of K from 6 to 8 blocks of 64 (hidden states kept on chip), and one block less
          (2100, 50304, 512, 0), (1601, 50257, 449, 7), (4500, 20001, 384, 8), (7000, 12800, 328, 0), (2100, 40000, 320, 0)]


@pytest.mark.parametrize("M,V,K,stride", SHAPES)
def test_forward(cuda, M, V, K, stride):
    x, w, labels = make(M, V, K, stride=stride)
    lp, lse = torch.full((M,), 5.0, device=cuda), torch.full((M,), 5.0, device=cuda)
    nv.linear_logprobs(x, w, labels, lp, lse=lse)
    on, z, want_lse, want, size = ref(x, w, labels)
    tol = size + (40 + V / 128) * U
    assert ((lse.double() - want_lse).abs() <= tol + U * want_lse.abs()).all()
    assert ((lp.double() - want).abs() <= 2 * tol + U * want.abs()).all()
    assert (lp[~on] == 0).all()
    assert nv._lib.device_error() == 0


@pytest.mark.parametrize("M,V,K", [(130, 1000, 64), (700, 50304, 512), (5, 50257, 512), (2100, 50304, 1024), (2100, 50304, 512)])
def test_rounded_products_give_what_stored_logits_give(cuda, M, V, K):
    """The same fp32 accumulators rounded the same way, so only the sums' own order differs."""
    x, w, labels = make(M, V, K)
    a, b = torch.empty(M, device=cuda), torch.empty(M, device=cuda)
    nv.linear_logprobs(x, w, labels, a, round_bf16=True)
    ld = (V + 7) // 8 * 8
    logits = torch.empty(M, ld, device=cuda, dtype=torch.bfloat16)[:, :V]
    nv.gemm(x, w, logits)
    nv.token_logprobs(logits, labels, b)
    assert ((a.double() - b.double()).abs() <= 2 * (40 + V / 128) * U + 2 * U * b.double().abs()).all()


@pytest.mark.parametrize("M,V,K,stride,chunk", [(1, 9, 8, 0, None), (7, 50257, 512, 0, None), (300, 1001, 72, 8, None),
                                               (300, 1001, 64, 0, 128), (1025, 5000, 512, 0, 256), (2047, 777, 1024, 0, 1000),
                                               # few output tiles and a long contraction, for dx and for dw
                                               (88, 33001, 408, 0, None), (3, 20480, 72, 8, None), (129, 9999, 30, 2, 100),
                                               (5000, 130, 72, 0, None), (4097, 129, 9, 7, None)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_backward(cuda, M, V, K, stride, chunk, out):
    x, w, labels = make(M, V, K, stride=stride)
    lp, lse = torch.empty(M, device=cuda), torch.empty(M, device=cuda)
    nv.linear_logprobs(x, w, labels, lp, lse=lse)
    g = torch.randn(M, device=cuda) / M
    ld = (K + 7) // 8 * 8
    dx = torch.full((M, ld), 5.0, device=cuda, dtype=out)[:, :K]
    dw = torch.full((V, ld), 0.25, device=cuda, dtype=out)[:, :K]
    nv.linear_logprobs_bwd(x, w, labels, lse, g, dx, dw, chunk_rows=chunk)
    on, z, want_lse, _, size = ref(x, w, labels)
    d = torch.softmax(z, 1)
    d[torch.arange(M, device=cuda), labels.clamp(0, V - 1)] -= 1.0
    d *= torch.where(on, -g.double(), 0.0)[:, None]
    # of each gradient element: half a bf16 step (2^-8), and its softmax's relative error
    err = d.abs() * (2.0 ** -8 * 1.01) + (g.double().abs() * on)[:, None] * torch.softmax(z, 1) * (
        2 * size + (40 + V / 128 + 8) * U + U * want_lse.abs())[:, None] + g.double().abs()[:, None] * 2 * U
    half = torch.finfo(out).eps / 2
    for got, want, e, mag, terms in (
            (dx, d @ w.double(), err @ w.double().abs(), d.abs() @ w.double().abs(), V),
            (dw, d.t() @ x.double() + (0.25 if out == torch.float32 else 0.0), err.t() @ x.double().abs(),
             d.abs().t() @ x.double().abs() + 0.25, M)):
        tol = e + 2 * terms * U * mag + half * want.abs() * 1.01
        if out == torch.bfloat16 and chunk is not None:
            tol = tol + half * want.abs()
        off = (got.double() - want).abs() - tol
        assert (off <= 0).all(), off.max()
    assert nv._lib.device_error() == 0


@pytest.mark.parametrize("K", [64, 61])
def test_autograd_and_no_rows(cuda, K):
    x, w, labels = make(70, 513, K, stride=64 - K)
    x.requires_grad_(True), w.requires_grad_(True)
    lp = losses.linear_logprobs(x, w, labels)
    (lp * torch.linspace(-1, 1, 70, device=cuda)).sum().backward()
    xr, wr = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    on = (labels >= 0) & (labels < 513)
    z = torch.log_softmax(xr @ wr.t(), 1).gather(1, labels.clamp(0, 512)[:, None])[:, 0]
    (torch.where(on, z, 0.0) * torch.linspace(-1, 1, 70, device=cuda, dtype=torch.float64)).sum().backward()
    for got, want in ((x.grad, xr.grad), (w.grad, wr.grad)):
        # bf16 gradient rows and a bf16 result: 2^-8 of the largest sum's size
        assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -8 * want.abs().max()).all()
    nv.linear_logprobs(x.detach()[:0], w.detach(), labels[:0], torch.empty(0, device=cuda))
    dw = torch.ones(513, 64, device=cuda, dtype=torch.bfloat16)[:, :K]
    nv.linear_logprobs_bwd(x.detach()[:0], w.detach(), labels[:0], torch.empty(0, device=cuda), torch.empty(0, device=cuda), None, dw)
    assert (dw == 0).all()
