"""What the backward of the linear log-probabilities launches."""
import pytest
import torch

from rgpt_b200 import native as nv

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def test_no_library_kernel_in_the_backward(cuda):
    """Several chunks with a bf16 dw: the sum over the chunks starts, grows and is rounded by the framework's kernels."""
    M, V, K = 1025, 3001, 264
    x, w = torch.randn(M, K, device=cuda).to(BF), torch.randn(V, K, device=cuda).to(BF)
    labels = torch.randint(0, V, (M,), device=cuda)
    lp, lse, g = (torch.empty(M, device=cuda) for _ in range(3))
    nv.linear_logprobs(x, w, labels, lp, lse=lse)
    g.fill_(1.0 / M)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    nv.linear_logprobs_bwd(x, w, labels, lse, g, dx, dw, chunk_rows=300)
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        nv.linear_logprobs_bwd(x, w, labels, lse, g, dx, dw, chunk_rows=300)
    seen = {e.key for e in prof.key_averages() if e.key.startswith("aten::")}
    assert seen <= {"aten::empty", "aten::empty_strided"}, seen
