"""Equal calls of the linear log-probabilities and of their backward give equal bits, into whatever the gradients go."""
import pytest
import torch

from rgpt_b200 import native as nv

pytestmark = pytest.mark.gpu

BF, F = torch.bfloat16, torch.float32


def call(x, w, labels, g, out, chunk):
    M, K = x.shape
    V, ld = w.shape[0], (K + 7) // 8 * 8
    lp, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    nv.linear_logprobs(x, w, labels, lp, lse=lse)
    dx = torch.zeros(M, ld, device="cuda", dtype=out)[:, :K]
    dw = torch.full((V, ld), 0.5, device="cuda", dtype=out)[:, :K]
    nv.linear_logprobs_bwd(x, w, labels, lse, g, dx, dw, chunk_rows=chunk)
    return lp, lse, dx, dw


@pytest.mark.parametrize("M,V,K,chunk", [(5000, 130, 72, None), (4097, 129, 9, None), (1025, 5000, 512, 256),
                                         (300, 1001, 64, 128), (2047, 777, 1024, 1000), (9000, 2999, 256, None),
                                         (16368, 60, 512, 8000), (3000, 6001, 1024, 1024), (1, 9, 8, None)])
@pytest.mark.parametrize("out", [BF, F])
def test_equal_bits(cuda, M, V, K, chunk, out):
    g = torch.Generator(device="cuda").manual_seed(M + V)
    ld = (K + 7) // 8 * 8
    x = torch.randn(M, ld, device=cuda, generator=g).to(BF)[:, :K]
    w = (torch.randn(V, ld, device=cuda, generator=g) * K ** -0.5).to(BF)[:, :K]
    labels = torch.randint(0, V, (M,), device=cuda, generator=g)
    d = torch.randn(M, device=cuda, generator=g) / M
    first = call(x, w, labels, d, out, chunk)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for i in range(6):
        if i < 3:
            again = call(x, w, labels, d, out, chunk)
        else:
            with torch.cuda.stream(s):
                again = call(x, w, labels, d, out, chunk)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again)), i
