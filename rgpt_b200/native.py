"""Torch-tensor wrappers over the C ABI (include/rgpt.h).

Each function validates shapes/dtypes on the host, then enqueues one or more
native kernels on the current CUDA stream. None of them has a fallback.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import ptr

EPI_STORE_BF16 = 0
EPI_STORE_F32 = 1
EPI_ACCUM_F32 = 2
EPI_ACT_FWD = 3
EPI_ACT_BWD = 4
EPI_RESID_F32 = 5
EPI_POLY_BF16 = 6
EPI_BIAS_SIGMOID_BF16 = 7
EPI_POLY_F32 = 8
EPI_ARGMAX_BF16 = 9
EPI_LSE_F32 = 10             # linear_logprobs only
EPI_SOFTMAX_GRAD_BF16 = 11   # linear_logprobs_bwd only

ACTIVATIONS = {"none": 0, "identity": 0, "squared_relu": 1, "gelu": 2, "silu": 3, "mish": 4}
ACT_SQRELU = 1
ACT_SQRELU_POST = 5  # squared ReLU with the post-activation as the only forward output and the backward's C


def act_id(name: str) -> int:
    try:
        return ACTIVATIONS[name]
    except KeyError as e:
        raise ValueError(f"unknown activation {name!r}") from e


class Drop:
    """Dropout of one site: keep bits are drawn from Philox4x32-10 under the device seed (int64 [1])
    and the site number, and stored in `mask` (int32 words) for the backward; p is the drop rate."""

    __slots__ = ("mask", "seed", "site", "p")

    def __init__(self, mask: torch.Tensor, seed: torch.Tensor | None, site: int, p: float):
        if mask.dtype != torch.int32 or not mask.is_contiguous():
            raise ValueError("dropout masks are contiguous int32 words")
        if seed is not None and (seed.dtype != torch.int64 or seed.numel() != 1):
            raise ValueError("dropout seed is a device int64 [1]")
        if not 0.0 <= p < 1.0:
            raise ValueError(f"dropout p must be in [0, 1), got {p}")
        self.mask, self.seed, self.site, self.p = mask, seed, int(site), float(p)


def _drop_args(drop: "Drop | None", seed_needed: bool = True):
    if drop is None:
        return None, None, 0, 0.0
    if seed_needed and drop.seed is None:
        raise ValueError("this dropout call draws new bits and needs the seed")
    return ptr(drop.mask), ptr(drop.seed) if drop.seed is not None else None, drop.site & 0xFFFFFFFF, drop.p


def gemm_argmax(A: torch.Tensor, B: torch.Tensor, part_val: torch.Tensor, part_idx: torch.Tensor,
                argmax: torch.Tensor) -> None:
    """argmax[m] = first index of the maximum of bf16(A @ B^T)[m, :] without writing the product.

    A [M, K], B [N, K] bf16 with unit stride on K; part_val (fp32) / part_idx (int32) [M, >= ceil(N/128)]
    hold the per-column-tile partial results; argmax int32 [M]."""
    M, K = A.shape
    N = B.shape[0]
    for t, n in ((A, "A"), (B, "B")):
        if t.dtype != torch.bfloat16 or t.stride(-1) != 1 or t.dim() != 2:
            raise ValueError(f"gemm_argmax: {n} must be 2-D bf16 with unit stride on K")
    if part_val.dtype != torch.float32 or part_idx.dtype != torch.int32 or argmax.dtype != torch.int32:
        raise TypeError("gemm_argmax: partial values fp32, partial indices and argmax int32")
    ld = part_val.stride(0)
    if part_idx.stride(0) != ld or part_val.shape[0] < M or part_val.shape[1] < (N + 127) // 128:
        raise ValueError("gemm_argmax: partial buffers must be [M, >= ceil(N/128)] with equal row strides")
    _lib.call("rgpt_gemm_argmax", ptr(A), A.stride(0), ptr(B), B.stride(0), M, N, K, ptr(part_val), ptr(part_idx),
              ld, ptr(argmax), _lib.stream_ptr(A.device))


def drop_mask_rows(drop: Drop, M: int, N: int) -> None:
    """Fill drop.mask [M, ceil(N/32)] with the residual-branch keep bits of (seed, site)."""
    if drop.mask.dim() != 2 or drop.mask.shape[0] < M:
        raise ValueError("row dropout mask must be [M, ceil(N/32)] words")
    dm, ds, dsite, dp = _drop_args(drop)
    _lib.call("rgpt_drop_mask", dm, drop.mask.stride(0), ds, dsite, dp, M, N, _lib.stream_ptr(drop.mask.device))


def attn_drop_mask(drop: Drop, B: int, T: int, H: int) -> None:
    """Fill drop.mask [B*H, ceil(T/32), T] with the attention-probability keep bits of (seed, site)."""
    if drop.mask.numel() < B * H * ((T + 31) // 32) * T:
        raise ValueError("attention dropout mask must hold [B*H, ceil(T/32), T] words")
    dm, ds, dsite, dp = _drop_args(drop)
    _lib.call("rgpt_attn_drop_mask", dm, ds, dsite, dp, B, T, H, _lib.stream_ptr(drop.mask.device))


def _operand(t: torch.Tensor):
    """(mn_major, ld, bstride) for a logical [.., rows, K] bf16 operand view."""
    if t.dtype != torch.bfloat16:
        raise TypeError(f"GEMM operands must be bf16, got {t.dtype}")
    if t.stride(-1) == 1:
        mn, ld = 0, t.stride(-2)
    elif t.stride(-2) == 1:
        mn, ld = 1, t.stride(-1)
    else:
        raise ValueError(f"GEMM operand needs a unit stride in one of its last two dims, got {t.stride()}")
    bstride = t.stride(0) if t.dim() == 3 else 0
    return mn, ld, bstride


def _out(t: torch.Tensor | None):
    if t is None:
        return None, 0, 0
    if t.stride(-1) != 1:
        raise ValueError("GEMM outputs/epilogue inputs must have unit column stride")
    return ptr(t), t.stride(-2), (t.stride(0) if t.dim() == 3 else 0)


# Optional GEMM timing hook: when set to a list, every gemm() call appends
# (start_event, end_event, flops, (epi, M, N, K, batch)) recorded on the launching stream.
gemm_events: list | None = None


def gemm(A: torch.Tensor, B: torch.Tensor, out: torch.Tensor, *, epi: int = EPI_STORE_BF16,
         act: int = 0, alpha: float = 1.0, beta: float = 0.0, out2: torch.Tensor | None = None,
         c: torch.Tensor | None = None, colscale: torch.Tensor | None = None, splitk: int = 1,
         alpha_dev: torch.Tensor | None = None, drop: Drop | None = None) -> torch.Tensor:
    """out = epilogue(A @ B^T) for logical A [(b,) M, K] and B [(b,) N, K] (bf16).

    drop (RESID_F32 only): branch dropout whose mask drop_mask_rows filled.

    Either operand may be K-major (unit stride on K) or MN-major (unit stride
    on M/N), e.g. ``gemm(dy.t(), x.t(), dw, epi=EPI_ACCUM_F32)`` computes
    dW += dy^T x without materialising a transpose.
    """
    if A.dim() != B.dim() or A.dim() not in (2, 3):
        raise ValueError("A and B must both be 2-D or both 3-D")
    M, K = A.shape[-2], A.shape[-1]
    N, K2 = B.shape[-2], B.shape[-1]
    if K != K2:
        raise ValueError(f"inner dims differ: {K} vs {K2}")
    batch = A.shape[0] if A.dim() == 3 else 1
    if out.shape[-2:] != (M, N):
        raise ValueError(f"out has shape {tuple(out.shape)}, expected [..., {M}, {N}]")
    a_mn, lda, abs_ = _operand(A)
    b_mn, ldb, bbs = _operand(B)
    d, ldd, dbs = _out(out)
    d2, ldd2, d2bs = _out(out2)
    cp, ldc, cbs = _out(c)
    ev = gemm_events
    if ev is not None:
        e0 = torch.cuda.Event(enable_timing=True)
        e1 = torch.cuda.Event(enable_timing=True)
        e0.record()
    if drop is None:
        _lib.call("rgpt_gemm_bf16",
                  ptr(A), a_mn, lda, abs_, ptr(B), b_mn, ldb, bbs,
                  M, N, K, batch, epi, act, float(alpha), float(beta),
                  d, ldd, dbs, d2, ldd2, d2bs, cp, ldc, cbs,
                  ptr(colscale), splitk, ptr(alpha_dev), _lib.stream_ptr(out.device))
    else:
        dm, _, _, dp = _drop_args(drop, seed_needed=False)
        _lib.call("rgpt_gemm_bf16_dropout",
                  ptr(A), a_mn, lda, abs_, ptr(B), b_mn, ldb, bbs,
                  M, N, K, batch, epi, act, float(alpha), float(beta),
                  d, ldd, dbs, d2, ldd2, d2bs, cp, ldc, cbs,
                  ptr(colscale), splitk, ptr(alpha_dev), dm, drop.mask.shape[-1], dp,
                  _lib.stream_ptr(out.device))
    if ev is not None:
        e1.record()
        ev.append((e0, e1, 2.0 * M * N * K * batch, (epi, M, N, K, batch)))
    return out


# ----------------------------------------------------------------------------- attention
def _check(t, dtype, name):
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must have unit column stride")


def attn_fwd(qk: torch.Tensor, qkv: torch.Tensor, gate: torch.Tensor | None, o: torch.Tensor,
             og: torch.Tensor | None, lse: torch.Tensor, B: int, T: int, H: int, drop: Drop | None = None) -> None:
    """Causal attention over token-major q/k (qk [B*T, 2d]) and v (qkv[:, 2d:3d]).

    Writes o [B*T, d] (bf16), og = o * gate (if gate given) and lse [B, H, T] (fp32).
    drop: attention-probability dropout; its mask must have been filled by attn_drop_mask."""
    d = H * 64
    for t, n in ((qk, "qk"), (qkv, "qkv"), (o, "o")):
        _check(t, torch.bfloat16, n)
    if qk.shape != (B * T, 2 * d) or qkv.shape != (B * T, 3 * d) or o.shape != (B * T, d):
        raise ValueError("attention shapes do not match [B*T, 2d] / [B*T, 3d] / [B*T, d]")
    if lse.dtype != torch.float32 or lse.numel() != B * H * T:
        raise ValueError("lse must be fp32 [B, H, T]")
    if drop is not None and drop.mask.numel() < B * H * ((T + 31) // 32) * T:
        raise ValueError("attention dropout mask must hold [B*H, ceil(T/32), T] words")
    dm, _, _, dp = _drop_args(drop, seed_needed=False)
    _lib.call("rgpt_attn_fwd", ptr(qk), ptr(qkv), ptr(gate), ptr(o), ptr(og), ptr(lse), B, T, H, d,
              dm, dp, _lib.stream_ptr(o.device))


def attn_bwd_prep(dog: torch.Tensor, o: torch.Tensor, gate: torch.Tensor | None, do: torch.Tensor,
                  dgate_pre: torch.Tensor | None, D: torch.Tensor, B: int, T: int, H: int,
                  dq_zero: torch.Tensor | None = None) -> None:
    """do = dog*gate, dgate_pre = dog*o*gate*(1-gate), D = rowsum(do*o) per (token, head);
    dq_zero (the fp32 [B*T, d] dq accumulator of attn_bwd), when given, is zeroed in the same pass."""
    d = H * 64
    if dq_zero is not None and (dq_zero.dtype != torch.float32 or not dq_zero.is_contiguous()
                                or dq_zero.numel() != B * T * d):
        raise RuntimeError("attn_bwd_prep: dq_zero must be a contiguous fp32 [B*T, d] tensor")
    _lib.call("rgpt_attn_bwd_prep", ptr(dog), ptr(o), ptr(gate), ptr(do), ptr(dgate_pre), ptr(D), ptr(dq_zero),
              B, T, H, d, _lib.stream_ptr(o.device))


def attn_bwd(qk: torch.Tensor, qkv: torch.Tensor, do: torch.Tensor, lse: torch.Tensor, D: torch.Tensor,
             dq: torch.Tensor, dk: torch.Tensor, dv: torch.Tensor, B: int, T: int, H: int,
             drop: Drop | None = None) -> None:
    """dq (fp32, accumulated: caller zeroes), dk (fp32) and dv (bf16, may be a strided column view).

    drop: the forward's attention dropout (its mask is read back; no new bits are drawn)."""
    d = H * 64
    if dq.dtype != torch.float32 or dk.dtype != torch.float32 or dv.dtype != torch.bfloat16:
        raise TypeError("dq/dk must be fp32 and dv bf16")
    if drop is not None and drop.mask.numel() < B * H * ((T + 31) // 32) * T:
        raise ValueError("attention dropout mask must hold [B*H, ceil(T/32), T] words")
    dm, _, _, dp = _drop_args(drop, seed_needed=False)
    _lib.call("rgpt_attn_bwd", ptr(qk), ptr(qkv), ptr(do), ptr(lse), ptr(D), ptr(dq), ptr(dk), dk.stride(0),
              ptr(dv), dv.stride(0), B, T, H, d, dm, dp, _lib.stream_ptr(do.device))


# ----------------------------------------------------------------------------- norms
NORM_IDENTITY, NORM_RMS_AFFINE, NORM_RMS, NORM_L2_TEMP, NORM_L2, NORM_ELASTIC, NORM_ELASTICBALL, NORM_HYPERBALL = range(8)
FLT_EPS = 1.1920928955078125e-07  # torch.finfo(torch.float32).eps


def rownorm_fwd(x: torch.Tensor, y: torch.Tensor, kind: int, eps: float, *, w: torch.Tensor | None = None,
                temp: float = 1.0, alpha: float = 0.5, stat: torch.Tensor | None = None,
                qw: torch.Tensor | None = None, qb: torch.Tensor | None = None,
                qout: torch.Tensor | None = None) -> None:
    M, d = x.shape
    _lib.call("rgpt_rownorm_fwd", ptr(x), ptr(y), ptr(stat), ptr(w), float(temp), kind, float(eps), float(alpha),
              M, d, ptr(qw), ptr(qb), ptr(qout), _lib.stream_ptr(x.device))


def rownorm_bwd(x: torch.Tensor, dy: torch.Tensor | None, kind: int, eps: float, g_out: torch.Tensor, *,
                w: torch.Tensor | None = None, temp: float = 1.0, alpha: float = 0.5,
                g_in: torch.Tensor | None = None, g_bf16: torch.Tensor | None = None,
                ls: torch.Tensor | None = None, raw: torch.Tensor | None = None, dls: torch.Tensor | None = None,
                dw: torch.Tensor | None = None, dtemp: torch.Tensor | None = None,
                dq: torch.Tensor | None = None, qw: torch.Tensor | None = None, h: torch.Tensor | None = None,
                dqw: torch.Tensor | None = None, dqb: torch.Tensor | None = None, drop: Drop | None = None) -> None:
    """drop: the dropout of the branch whose gradient g_bf16 is (its mask, read back; no new bits)."""
    M, d = x.shape
    if drop is not None and drop.mask.numel() < M * (d // 32):
        raise ValueError("branch dropout mask must hold [M, d/32] words")
    dm, _, _, dp = _drop_args(drop, seed_needed=False)
    _lib.call("rgpt_rownorm_bwd", ptr(x), ptr(dy), ptr(w), float(temp), kind, float(eps), float(alpha), M, d,
              ptr(g_in), ptr(g_out), ptr(g_bf16), ptr(ls), ptr(raw), ptr(dls), ptr(dw), ptr(dtemp),
              ptr(dq), ptr(qw), ptr(h), ptr(dqw), ptr(dqb), dm, dp, _lib.stream_ptr(x.device))


# ----------------------------------------------------------------------------- standalone modules
def _rows_f32(t: torch.Tensor, name: str) -> None:
    if t.dtype != torch.float32 or t.dim() != 2 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous fp32 [M, d] tensor")


def rownorm_any_fwd(x: torch.Tensor, y: torch.Tensor, kind: int, eps: float, *, w: torch.Tensor | None = None,
                    alpha: float = 0.5) -> None:
    """y = norm(x) over rows of any length (fp32 [M, d] both); w: RMSNorm weight [d] or L2Norm temp [1]."""
    _rows_f32(x, "x")
    _rows_f32(y, "y")
    if y.shape != x.shape:
        raise ValueError("rownorm_any_fwd: y must have x's shape")
    M, d = x.shape
    _lib.call("rgpt_rownorm_any_fwd", ptr(x), ptr(y), ptr(w), kind, float(eps), float(alpha), M, d,
              _lib.stream_ptr(x.device))


def rownorm_any_bwd(x: torch.Tensor, dy: torch.Tensor, kind: int, eps: float, dx: torch.Tensor, *,
                    w: torch.Tensor | None = None, alpha: float = 0.5, dw: torch.Tensor | None = None,
                    dtemp: torch.Tensor | None = None) -> None:
    """dx = norm'(x)^T dy (written); dw (RMSNorm weight) and dtemp (L2Norm temp) are accumulated."""
    for t, n in ((x, "x"), (dy, "dy"), (dx, "dx")):
        _rows_f32(t, n)
    M, d = x.shape
    _lib.call("rgpt_rownorm_any_bwd", ptr(x), ptr(dy), ptr(w), kind, float(eps), float(alpha), M, d, ptr(dx),
              ptr(dw), ptr(dtemp), _lib.stream_ptr(x.device))


def rope(inp: torch.Tensor, out: torch.Tensor, inv_freq: torch.Tensor, backward: bool = False) -> None:
    """out (contiguous fp32 [B, H, T, D]) = RoPE(inp) for fp32 inp [B, H, T, D] with unit stride on D."""
    if inp.dtype != torch.float32 or inp.dim() != 4 or inp.stride(-1) != 1:
        raise ValueError("rope input must be a 4-D fp32 [B, H, T, D] tensor with unit stride on D")
    if out.dtype != torch.float32 or out.shape != inp.shape or not out.is_contiguous():
        raise ValueError("rope output must be a contiguous fp32 tensor of the input's shape")
    B, H, T, D = inp.shape
    if inv_freq.dtype != torch.float32 or inv_freq.numel() != D // 2 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous fp32 [D/2] tensor")
    sb, sh, st, _ = inp.stride()
    _lib.call("rgpt_rope", ptr(inp), sb, sh, st, ptr(out), ptr(inv_freq), B, H, T, D, int(backward),
              _lib.stream_ptr(inp.device))


# ----------------------------------------------------------------------------- QKV prep
def qkv_prep_fwd(qkv, qk, qn, inv_freq, qk_kind, eps, alpha, M, T, H, *, wq=None, wk=None,
                 tq=1.0, tk=1.0, sq=1.0, sk=1.0) -> None:
    _lib.call("rgpt_qkv_prep_fwd", ptr(qkv), ptr(qk), ptr(qn), ptr(inv_freq), qk_kind, float(eps), float(alpha),
              ptr(wq), ptr(wk), float(tq), float(tk), float(sq), float(sk), M, T, H, _lib.stream_ptr(qkv.device))


def qkv_prep_bwd(qkv, dq, dk, dqn_gate, dgp, dqkv, inv_freq, qk_kind, eps, alpha, M, T, H, *, dbg=None,
                 dwq=None, dwk=None, dtq=None, dtk=None, wq=None, wk=None, tq=1.0, tk=1.0, sq=1.0, sk=1.0) -> None:
    _lib.call("rgpt_qkv_prep_bwd", ptr(qkv), ptr(dq), ptr(dk), ptr(dqn_gate), ptr(dgp), ptr(dqkv), ptr(dbg),
              ptr(dwq), ptr(dwk), ptr(dtq), ptr(dtk), ptr(inv_freq), qk_kind, float(eps), float(alpha), ptr(wq),
              ptr(wk), float(tq), float(tk), float(sq), float(sk), M, T, H, _lib.stream_ptr(qkv.device))


# ----------------------------------------------------------------------------- embedding / loss
def embedding_fwd(ids: torch.Tensor, emb: torch.Tensor, x: torch.Tensor, drop: Drop | None = None) -> None:
    M = ids.numel()
    V, d = emb.shape
    if drop is not None and drop.mask.numel() < M * (d // 32):
        raise ValueError("embedding dropout mask must hold [M, d/32] words")
    _lib.call("rgpt_embedding_fwd", ptr(ids), ptr(emb), ptr(x), M, d, V, *_drop_args(drop), _lib.stream_ptr(x.device))


def embedding_bwd(ids: torch.Tensor, dx: torch.Tensor, demb: torch.Tensor, drop: Drop | None = None) -> None:
    M = ids.numel()
    V, d = demb.shape
    if drop is not None and drop.mask.numel() < M * (d // 32):
        raise ValueError("embedding dropout mask must hold [M, d/32] words")
    dm, _, _, dp = _drop_args(drop, seed_needed=False)
    _lib.call("rgpt_embedding_bwd", ptr(ids), ptr(dx), ptr(demb), M, d, V, dm, dp, _lib.stream_ptr(dx.device))


def cross_entropy(logits: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100, grad_scale: float = 1.0,
                  loss_rows: torch.Tensor | None = None, argmax: torch.Tensor | None = None,
                  scale_buf: torch.Tensor | None = None, loss_out: torch.Tensor | None = None,
                  write_grad: bool = False) -> None:
    M, V = logits.shape
    nk = 1 + (scale_buf is not None) + (loss_out is not None and loss_rows is not None)
    _lib.call("rgpt_cross_entropy", ptr(logits), logits.stride(0), M, V, ptr(labels), int(ignore_index),
              float(grad_scale), ptr(loss_rows), ptr(argmax), ptr(scale_buf), ptr(loss_out), int(write_grad),
              _lib.stream_ptr(logits.device), kernels=nk)


def halt_losses(q: torch.Tensor, argmax: torch.Tensor, labels: torch.Tensor, dq: torch.Tensor,
                losses: torch.Tensor, grad_scale: float = 1.0) -> None:
    R, M = q.shape[0], q.shape[1]
    _lib.call("rgpt_halt_losses", ptr(q), ptr(argmax), ptr(labels), R, M, float(grad_scale), ptr(dq), ptr(losses),
              _lib.stream_ptr(q.device))


# ----------------------------------------------------------------------------- post-training losses
LOGIT_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
PREFERENCE_KINDS = {"sigmoid": 0, "hinge": 1, "squared": 2}


_entries: dict = {}  # bound entry points by name
# (a torch without CUDA has neither, and no tensor that would need them)
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _call_on(index: int, name: str, *args, kernels: int = 1) -> None:
    """_lib.call on the current stream of device `index`, with that device current (the library launches on the current
    device's context). The stream is the call's last argument."""
    if index < 0:
        raise RuntimeError("librgpt_kernels only takes CUDA tensors (no CPU path)")
    if index != _current_device():
        with torch.cuda.device(index):
            return _call_on(index, name, *args, kernels=kernels)
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    rc = fn(*args, _current_stream(index))
    if rc != 0:
        raise RuntimeError(f"{name} failed (status {rc}): {_lib.last_error()}")
    _lib.launch_count += kernels


# The operators below check their arguments twice over: _fastargs.pack (csrc/fastargs.cpp) in one step, giving the
# entry point's arguments when all is well, and otherwise here, where a refusal says what was wrong. (Where only the
# kernel library has been built, the checks here serve alone.) The extension is loaded by the first call, as the kernel
# library is: importing this module maps neither.
def _load_pack():
    global _pack
    try:
        from ._fastargs import pack as _pack
    except ImportError:
        def _pack(kinds: str, tensors: tuple):
            return None
    return _pack


def __getattr__(name: str):
    if name == "_pack":
        return _load_pack()
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def _packed(kinds: str, tensors: tuple):
    """The entry point's arguments, or None where the checks here have to say what is wrong."""
    try:
        return _pack(kinds, tensors)
    except NameError:
        return _load_pack()(kinds, tensors)


def _flat(t: torch.Tensor, name: str, shape, dtype: torch.dtype, index: int) -> int:
    """Address of a contiguous tensor of the given shape, type and device (-1: host memory, which _call_on refuses)."""
    if t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous():
        return t.data_ptr()
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, expected device {index}")
    raise ValueError(f"{name} must be a contiguous tensor of shape {tuple(shape)}, got {tuple(t.shape)}"
                     f" with strides {t.stride()}")


def _opt(t: torch.Tensor | None, name: str, shape, dtype: torch.dtype, index: int) -> int | None:
    return None if t is None else _flat(t, name, shape, dtype, index)


def _logit_rows(t: torch.Tensor, name: str):
    """(dtype id, batch stride, token stride, B, T, V) of logits [B, T, V], or [M, V] as M sequences of one token."""
    dt = LOGIT_DTYPES.get(t.dtype)
    if dt is None:
        raise TypeError(f"{name} must be bf16, fp16 or fp32, got {t.dtype}")
    shape, stride = t.shape, t.stride()
    if len(shape) == 3:
        B, T, V = shape
        sb, st, sv = stride
    elif len(shape) == 2:
        (B, V), T = shape, 1
        (sb, sv), st = stride, 0
    else:
        raise ValueError(f"{name} must be [M, V] or [B, T, V], got {tuple(shape)}")
    if V > 1 and sv != 1:
        raise ValueError(f"{name} must have unit stride along the vocabulary, got strides {stride}")
    if B * T >= 2 ** 31 or V > 2 ** 30:
        raise ValueError(f"{name} must have fewer than 2^31 rows and at most 2^30 columns, got {tuple(shape)}")
    return dt, sb, st, B, T, V


def _end(t: torch.Tensor) -> int:
    """The address behind a tensor's last element."""
    last = 1
    for n, s in zip(t.shape, t.stride()):
        last += (n - 1) * s
    return t.data_ptr() + last * t.element_size()


def _rows_apart(sb: int, st: int, B: int, T: int, width: int) -> bool:
    """Whether rows of `width` elements at these strides share no element, batch first or time first."""
    return ((T == 1 or st >= width) and (B == 1 or sb >= (T - 1) * st + width)) or (sb >= width and st >= (B - 1) * sb + width)


def _grad_rows(dlogits: torch.Tensor | None, logits: torch.Tensor):
    """(address, batch stride, token stride) of the gradient's rows: the logits themselves, or memory apart from them
    (elsewhere, or in turn with their rows at the same strides)."""
    if dlogits is None:
        return None, 0, 0
    if dlogits.dtype is not logits.dtype or dlogits.shape != logits.shape or dlogits.get_device() != logits.get_device():
        raise ValueError("dlogits must have the logits' type, shape and device")
    _, sb, st, B, T, V = _logit_rows(dlogits, "dlogits")
    at, of = dlogits.data_ptr(), logits.data_ptr()
    if dlogits.is_contiguous():
        end = at + B * T * V * dlogits.element_size()
    else:
        if not _rows_apart(sb, st, B, T, V):
            raise ValueError(f"the rows of dlogits overlap (strides {dlogits.stride()})")
        end = _end(dlogits)
    if (at != of or dlogits.stride() != logits.stride()) and at < _end(logits) and of < end:
        off, odd = divmod(abs(at - of), dlogits.element_size())
        if dlogits.stride() != logits.stride() or odd or off < V or not _rows_apart(sb, st, B, T, off + V):
            raise ValueError("dlogits must be the logits themselves or share no memory with them")
    return at, sb, st


def token_logprobs(logits: torch.Tensor, labels: torch.Tensor, logps: torch.Tensor, *, lse: torch.Tensor | None = None,
                   ignore_index: int = -100) -> None:
    """logps = log softmax(logits)[label], 0 for tokens that are not scored (label ignore_index or outside the
    vocabulary); lse (optional, for token_logprobs_bwd) = logsumexp. logits [M, V] or [B, T, V] in bf16, fp16 or fp32
    with unit stride along the vocabulary and any other strides; labels int64, logps and lse fp32 of the leading shape."""
    p = _packed("LyfF", (logits, labels, logps, lse))
    if p is not None:
        return _call_on(p[10], "rgpt_token_logprobs", *p[:8], int(ignore_index), p[8], p[9])
    dt, sb, st, B, T, V = _logit_rows(logits, "logits")
    dev, shape = logits.get_device(), logits.shape[:-1]
    args = (_flat(labels, "labels", shape, torch.int64, dev), int(ignore_index),
            _flat(logps, "logps", shape, torch.float32, dev), _opt(lse, "lse", shape, torch.float32, dev))
    if B * T == 0:
        return
    if V == 0:
        raise ValueError("token_logprobs: the vocabulary is empty")
    _call_on(dev, "rgpt_token_logprobs", logits.data_ptr(), dt, sb, st, B, T, V, *args)


def token_logprobs_bwd(logits: torch.Tensor, labels: torch.Tensor, lse: torch.Tensor, dlogps: torch.Tensor,
                       dlogits: torch.Tensor, *, ignore_index: int = -100) -> None:
    """dlogits = dlogps * (onehot(label) - softmax(logits)), zero rows for tokens that are not scored. dlogits: the
    logits themselves (overwritten) or another tensor of their type and shape."""
    p = _packed("LyffG", (logits, labels, lse, dlogps, dlogits))
    if p is not None and dlogits is not None:
        return _call_on(p[13], "rgpt_token_logprobs_bwd", *p[:8], int(ignore_index), *p[8:13])
    dt, sb, st, B, T, V = _logit_rows(logits, "logits")
    dev, shape = logits.get_device(), logits.shape[:-1]
    args = (_flat(labels, "labels", shape, torch.int64, dev), int(ignore_index),
            _flat(lse, "lse", shape, torch.float32, dev), _flat(dlogps, "dlogps", shape, torch.float32, dev))
    grad = _grad_rows(dlogits, logits)
    if B * T == 0 or V == 0:
        return
    _call_on(dev, "rgpt_token_logprobs_bwd", logits.data_ptr(), dt, sb, st, B, T, V, *args, *grad)


def _preference_kernels(P: int, T: int, dlogits: torch.Tensor | None) -> int:
    """Launches of preference_loss: rows, pairs (a warp or a CTA each), their mean unless one CTA has them all, gradient."""
    return 2 + (P > (8 if T <= 256 else 1)) + (dlogits is not None)


def preference_loss(logits: torch.Tensor, labels: torch.Tensor, ref_logps: torch.Tensor | None = None, *,
                    token_logps: torch.Tensor, lse: torch.Tensor, seq_logps: torch.Tensor, margins: torch.Tensor,
                    coef: torch.Tensor, loss: torch.Tensor, dlogits: torch.Tensor | None = None,
                    scratch: torch.Tensor | None = None, kind: str = "sigmoid", beta: float = 0.1,
                    label_smoothing: float = 0.0, margin: float = 0.0, average: bool = False,
                    ignore_index: int = -100, grad_scale: float = 1.0) -> None:
    """Paired preference loss from logits [2P, T, V]: sequences 0..P-1 are the chosen ones, P..2P-1 the rejected ones.

    h = beta * ((s_chosen - ref_chosen) - (s_rejected - ref_rejected)) - margin with s the sum of a sequence's scored
    log-probabilities (their mean with `average`) and ref_logps [2P] the same of a frozen reference (None: 0);
    kind "sigmoid" (with label_smoothing), "hinge" max(0, 1 - h) or "squared" (h - 1/2)^2; loss [1] is the pairs' mean.
    Written: token_logps, lse [2P, T], seq_logps [2P], margins [P] (h), coef [2P] (grad_scale * d loss / d each scored
    log-probability), loss [1], and dlogits = grad_scale * d loss / d logits when given (the logits themselves, or
    another tensor of their type and shape). scratch: fp64 [2P, T] (allocated when None)."""
    if kind not in PREFERENCE_KINDS:
        raise ValueError(f"preference_loss: kind must be one of {sorted(PREFERENCE_KINDS)}, got {kind!r}")
    if not 0.0 <= label_smoothing <= 0.5 or (label_smoothing and kind != "sigmoid"):
        raise ValueError("preference_loss: label_smoothing must be in [0, 0.5], and 0 unless kind is 'sigmoid'")
    if not 0.0 < beta < float("inf"):
        raise ValueError(f"preference_loss: beta must be positive and finite, got {beta}")
    p = _packed("LyRffbhb1WG", (logits, labels, ref_logps, token_logps, lse, seq_logps, margins, coef, loss, scratch,
                              dlogits))
    if p is not None and logits.dim() == 3:
        pairs, T = p[4] // 2, p[5]
        return _call_on(p[19], "rgpt_preference_loss", *p[:4], pairs, *p[5:8], int(ignore_index), p[8],
                        PREFERENCE_KINDS[kind], float(beta), float(margin), float(label_smoothing), int(bool(average)),
                        float(grad_scale), *p[9:19], kernels=_preference_kernels(pairs, T, dlogits))
    dt, sb, st, B, T, V = _logit_rows(logits, "logits")
    if logits.dim() != 3 or B % 2 or B == 0 or T == 0 or V == 0:
        raise ValueError(f"preference_loss needs logits [2P, T, V] of at least one pair and token, got {tuple(logits.shape)}")
    dev, P, f32 = logits.get_device(), B // 2, torch.float32
    lab = _flat(labels, "labels", (B, T), torch.int64, dev)
    ref = _opt(ref_logps, "ref_logps", (B,), f32, dev)
    outs = (_flat(token_logps, "token_logps", (B, T), f32, dev), _flat(lse, "lse", (B, T), f32, dev),
            _flat(seq_logps, "seq_logps", (B,), f32, dev), _flat(margins, "margins", (P,), f32, dev),
            _flat(coef, "coef", (B,), f32, dev), _flat(loss, "loss", (1,), f32, dev))
    grad = _grad_rows(dlogits, logits)
    if scratch is None:
        scratch = torch.empty(B, T, device=logits.device, dtype=torch.float64)
    _flat(scratch, "scratch", (B, T), torch.float64, dev)
    _call_on(dev, "rgpt_preference_loss", logits.data_ptr(), dt, sb, st, P, T, V, lab, int(ignore_index), ref,
             PREFERENCE_KINDS[kind], float(beta), float(margin), float(label_smoothing), int(bool(average)),
             float(grad_scale), *outs, scratch.data_ptr(), *grad,
             kernels=_preference_kernels(P, T, dlogits))


def _policy_kernels(B: int, T: int, by_sequence: bool) -> int:
    """Launches of policy_loss: few tokens are counted by the row kernel, others by two kernels of their own."""
    return 2 if B * T <= 1024 and (not by_sequence or B <= 32) else 4


def policy_loss(logits: torch.Tensor, labels: torch.Tensor, old_logps: torch.Tensor, advantages: torch.Tensor,
                ref_logps: torch.Tensor | None = None, *, token_logps: torch.Tensor, counts: torch.Tensor,
                stats: torch.Tensor, lse: torch.Tensor | None = None, coef: torch.Tensor | None = None,
                dlogits: torch.Tensor | None = None, clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
                by_sequence: bool = False, ignore_index: int = -100, grad_scale: float = 1.0) -> None:
    """Clipped policy loss with a KL term from logits [B, T, V] (or [M, V]: sequences of one token).

    Per scored token with ratio r = exp(logp - old_logps): -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A)
    + kl_coef * (exp(q) - q - 1), q = ref_logps - logp; averaged over the scored tokens, or with by_sequence over each
    sequence's tokens first and then over the sequences that have any. advantages A: [B], or one per token [B, T].
    Written: token_logps [B, T], counts [B] int32 (scored tokens), stats [4] = (loss, policy term, KL, clipped share),
    lse and coef [B, T] when given (coef = grad_scale * d loss / d logp, for token_logprobs_bwd), and dlogits =
    grad_scale * d loss / d logits when given (the logits themselves, or another tensor of their type and shape)."""
    if not 0.0 <= clip_low <= 1.0 or not 0.0 <= clip_high < float("inf"):
        raise ValueError(f"policy_loss: clip_low must be in [0, 1] and clip_high >= 0, got {clip_low} and {clip_high}")
    if kl_coef != 0.0 and ref_logps is None:
        raise ValueError("policy_loss: kl_coef needs ref_logps")
    p = _packed("LyfFafc4FFG", (logits, labels, old_logps, ref_logps, advantages, token_logps, counts, stats, lse, coef,
                              dlogits))
    if p is not None:
        return _call_on(p[20], "rgpt_policy_loss", *p[:8], int(ignore_index), *p[8:12], float(clip_low),
                        float(clip_high), float(kl_coef), int(bool(by_sequence)), float(grad_scale), *p[12:20],
                        kernels=_policy_kernels(p[4], p[5], by_sequence))
    dt, sb, st, B, T, V = _logit_rows(logits, "logits")
    dev, shape, f32 = logits.get_device(), logits.shape[:-1], torch.float32
    per_token = advantages.shape != (B,)
    adv = _flat(advantages, "advantages", shape if per_token else (B,), f32, dev)
    ins = (_flat(labels, "labels", shape, torch.int64, dev), int(ignore_index),
           _flat(old_logps, "old_logps", shape, f32, dev), _opt(ref_logps, "ref_logps", shape, f32, dev))
    outs = (_flat(token_logps, "token_logps", shape, f32, dev), _flat(counts, "counts", (B,), torch.int32, dev),
            _flat(stats, "stats", (4,), f32, dev), _opt(lse, "lse", shape, f32, dev), _opt(coef, "coef", shape, f32, dev))
    grad = _grad_rows(dlogits, logits)
    if B * T == 0 or V == 0:
        raise ValueError(f"policy_loss needs at least one token, got logits {tuple(logits.shape)}")
    _call_on(dev, "rgpt_policy_loss", logits.data_ptr(), dt, sb, st, B, T, V, *ins, adv, int(per_token), float(clip_low),
             float(clip_high), float(kl_coef), int(bool(by_sequence)), float(grad_scale), *outs, *grad,
             kernels=_policy_kernels(B, T, by_sequence))


def _linear_operands(x: torch.Tensor, w: torch.Tensor):
    for t, n in ((x, "x"), (w, "w")):
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{n} must be bf16, got {t.dtype}")
        if t.dim() != 2 or t.stride(1) != 1 or t.stride(0) % 8 or t.stride(0) < t.shape[1]:
            raise ValueError(f"{n} must be [rows, K] with unit stride along K and a row stride that is a multiple of 8,"
                             f" got {tuple(t.shape)} with strides {t.stride()}")
    (M, K), (V, K2) = x.shape, w.shape
    if K != K2 or K == 0 or V == 0 or w.device != x.device:
        raise ValueError(f"x {tuple(x.shape)} and w {tuple(w.shape)} must share K >= 1 and the device, with V >= 1")
    if M >= 2 ** 31 or V >= 2 ** 31:
        raise ValueError("linear_logprobs needs fewer than 2^31 rows and columns")
    return M, V, K


def linear_logprobs(x: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, logps: torch.Tensor, *,
                    lse: torch.Tensor | None = None, part: torch.Tensor | None = None, ignore_index: int = -100,
                    round_bf16: bool = False) -> None:
    """logps [M] = log softmax(x @ w^T)[label] (0 where not scored) without storing the logits: x [M, K], w [V, K] bf16.

    lse [M] (optional, for linear_logprobs_bwd) is written for every row. round_bf16: the products are rounded to bf16
    first, which gives what token_logprobs gives on stored bf16 logits. part: fp32 scratch of at least
    4 * M * ceil(V/128) elements (allocated when None)."""
    p = _packed("XXyPfF", (x, w, labels, part, logps, lse))
    if p is not None:
        return _call_on(p[9], "rgpt_linear_logprobs", *p[:4], *x.shape[:1], *w.shape, p[4], int(ignore_index),
                        int(bool(round_bf16)), *p[5:9], kernels=2)
    M, V, K = _linear_operands(x, w)
    dev = x.get_device()
    need = 4 * M * ((V + 127) // 128)
    lab = _flat(labels, "labels", (M,), torch.int64, dev)
    outs = (_flat(logps, "logps", (M,), torch.float32, dev), _opt(lse, "lse", (M,), torch.float32, dev))
    if part is not None and (part.numel() < need or part.dtype != torch.float32 or not part.is_contiguous()
                             or part.get_device() != dev):
        raise ValueError(f"linear_logprobs: part must be a contiguous fp32 tensor of at least {need} elements")
    if M == 0:
        return
    if part is None:
        part = torch.empty(need, device=x.device, dtype=torch.float32)
    _call_on(dev, "rgpt_linear_logprobs", x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), M, V, K, lab, int(ignore_index),
             int(bool(round_bf16)), part.data_ptr(), part.numel(), *outs, kernels=2)


def _product(dev: int, A: tuple, B: tuple, M: int, N: int, C: int, D: tuple, *, batch: int = 1, epi: int, splitk: int = 1):
    """D = A @ B^T, [M, N] over C: A and B are (address, 1 if rows are the contiguous side, row stride, batch stride), D is
    (address, row stride, batch stride). gemm() without its checks, which take longer than a few rows' product."""
    _call_on(dev, "rgpt_gemm_bf16", *A, *B, M, N, C, batch, epi, 0, 1.0, 0.0, *D, None, 0, 0, None, 0, 0, None, splitk, None)


def _cuts(M: int, N: int, C: int, sms: int, add: bool) -> int:
    """Parts that _product_long cuts a contraction of C into."""
    tiles = -(-M // 128) * -(-N // 256)
    if 2 * tiles <= sms:
        return min(sms // tiles, C // 1024)
    if not add:
        return 1
    # More tiles: rounds of them (0.43 us for 64 of C, and eight such for the epilogue) against the join (4 us, and 2.4e-6
    # an element and 0.45e-6 for each of its parts). dw of 5000 x 1024 over 16368, 160 tiles on 148 SMs: 221 us in one part,
    # 154 + 25 in four; of 10000 x 1024 over 12000, 316 tiles: 252 in one, 205 + 42 in four.
    def us(s: int) -> float:
        return -(-tiles * s // sms) * (-(-C // (64 * s)) + 8) * 0.43 + (s > 1) * (4 + M * N * (2.4e-6 + 0.45e-6 * s))

    return min(range(1, max(1, min(8, C // 1024, LINEAR_CHUNK_ELEMS // (2 * M * N))) + 1), key=us)


def _product_long(out: torch.Tensor, dev: int, A: tuple, B: tuple, M: int, N: int, C: int, D: int, ldd: int,
                  add: bool = False) -> None:
    """D = A @ B^T as _product, written in out's type, or with `add` (fp32) added to D. Where D has tiles for half of the SMs
    at most and C is long, C is cut into parts whose fp32 products are joined in order (88 rows x 408 columns over 116602
    take 536 us otherwise, the whole backward of such rows 112). Each element of D gets one sum, in a fixed order: equal calls
    give equal bits (the GEMM's own split of C adds its parts as they arrive)."""
    splits = _cuts(M, N, C, torch.cuda.get_device_properties(dev).multi_processor_count, add)
    f32 = out.dtype is torch.float32
    if splits < 2:
        return _product(dev, (*A, 0), (*B, 0), M, N, C, (D, ldd, 0),
                        epi=EPI_ACCUM_F32 if add else EPI_STORE_F32 if f32 else EPI_STORE_BF16)
    each = C // splits if A[1] and B[1] else C // (8 * splits) * 8  # of a K-major operand a part starts on 16 bytes
    whole, splits, ld = C // each, -(-C // each), (N + 3) // 4 * 4  # equal parts, and perhaps what is left of fewer than 8 * splits
    part = torch.empty(splits * M * ld, device=out.device, dtype=torch.float32)
    step = [each * (ldo if mn else 1) for _, mn, ldo in (A, B)]  # elements from one part to the next
    P, size = part.data_ptr(), M * ld
    _product(dev, (*A, step[0]), (*B, step[1]), M, N, each, (P, ld, size), batch=whole, epi=EPI_STORE_F32)
    if whole < splits:
        A, B = ((at + 2 * whole * st, mn, ldo, 0) for (at, mn, ldo), st in zip((A, B), step))
        _product(dev, A, B, M, N, C - whole * each, (P + 4 * whole * size, ld, 0), epi=EPI_STORE_F32)
    _call_on(dev, "rgpt_gemm_join", P, splits, M, N, D, ldd, int(f32), int(add))


# Gradient rows of linear_logprobs_bwd in flight: at most this many bf16 logit gradients (1 GiB) at a time.
LINEAR_CHUNK_ELEMS = 1 << 29


def linear_logprobs_bwd(x: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, lse: torch.Tensor, dlogps: torch.Tensor,
                        dx: torch.Tensor | None, dw: torch.Tensor | None, *, ignore_index: int = -100,
                        chunk_rows: int | None = None) -> None:
    """The gradients of linear_logprobs (round_bf16=False): dx [M, K] written in bf16 or fp32; dw [V, K] written when
    bf16, ACCUMULATED when fp32. Either may be None. The logits' gradient exists for chunk_rows rows at a time (default:
    as many as fit 1 GiB): its tiles come from the recomputed product, rounded to bf16 for the two GEMMs that follow, as the
    cross entropy's gradient is (the tensor cores' type; an element in two bf16 halves would double both products, for 2.3e-3
    of error in dx and dw against 64 bits, of which their own bf16 makes 1.7e-3). Equal calls give equal bits."""
    M, V, K = _linear_operands(x, w)
    dev = x.device
    for t, n, dtype in ((labels, "labels", torch.int64), (lse, "lse", torch.float32), (dlogps, "dlogps", torch.float32)):
        _flat(t, n, (M,), dtype, x.get_device())
    for t, n, shape in ((dx, "dx", (M, K)), (dw, "dw", (V, K))):
        if t is None:
            continue
        if (tuple(t.shape) != shape or t.dtype not in (torch.bfloat16, torch.float32) or t.stride(1) != 1
                or t.stride(0) % 8 or t.stride(0) < K or t.device != dev):
            raise ValueError(f"{n} must be a bf16 or fp32 {shape} tensor with unit column stride and a row stride that is"
                             f" a multiple of 8")
        for o in (x, w):  # both are read until the end
            if t.numel() and o.numel() and t.data_ptr() < _end(o) and o.data_ptr() < _end(t):
                raise ValueError(f"{n} must share no memory with x and w")
    if chunk_rows is not None and chunk_rows < 1:
        raise ValueError("linear_logprobs_bwd: chunk_rows must be at least 1")
    if M == 0:
        if dw is not None and dw.dtype == torch.bfloat16:
            dw.zero_()
        return
    index = x.get_device()
    if index < 0:
        raise RuntimeError("librgpt_kernels only takes CUDA tensors (no CPU path)")
    ld = (V + 7) // 8 * 8
    rows = min(M, chunk_rows or max(256, LINEAR_CHUNK_ELEMS // ld // 256 * 256))
    dl = torch.empty(rows * ld, device=dev, dtype=torch.bfloat16)
    acc = dw
    if dw is not None and dw.dtype is torch.bfloat16 and rows < M:
        acc = torch.empty(V, (K + 3) // 4 * 4, device=dev, dtype=torch.float32)  # the sum over the chunks
    X, W, L, S, G, d = (t.data_ptr() for t in (x, w, labels, lse, dlogps, dl))
    ldx, ldw = x.stride(0), w.stride(0)
    for a in range(0, M, rows):
        n, xa = min(rows, M - a), X + 2 * a * ldx
        _call_on(index, "rgpt_linear_logprobs_dlogits", xa, ldx, W, ldw, n, V, K, L + 8 * a, int(ignore_index), S + 4 * a,
                 G + 4 * a, d, ld)
        if dx is not None:
            _product_long(dx, index, (d, 0, ld), (W, 1, ldw), n, K, V, dx.data_ptr() + dx.element_size() * a * dx.stride(0),
                          dx.stride(0))
        if acc is not None:
            _product_long(acc, index, (d, 1, ld), (xa, 1, ldx), V, K, n, acc.data_ptr(), acc.stride(0),
                          add=acc.dtype is torch.float32 and (acc is dw or a > 0))
    if acc is not dw:
        _call_on(index, "rgpt_gemm_join", acc.data_ptr(), 1, V, K, dw.data_ptr(), dw.stride(0), 0, 0)


# ----------------------------------------------------------------------------- optimizer
# hp: optional device pointer (int) to a parameter group's block of RGPT_HP_FLOATS scalars; when
# given, the kernels read this step's lr / betas / bias corrections from it instead of the arguments.
HP_FLOATS = 8


def adamw(table: torch.Tensor, chunk_tensor: torch.Tensor, chunk_start: torch.Tensor, chunk_elems: int,
          lr: float, wd: float, beta1: float, beta2: float, eps: float, step: int, hp: int | None = None) -> None:
    _lib.call("rgpt_adamw", ptr(table), ptr(chunk_tensor), ptr(chunk_start), chunk_tensor.numel(), chunk_elems,
              float(lr), float(wd), float(beta1), float(beta2), float(eps), int(step), hp,
              _lib.stream_ptr(table.device))


ADAM8_BLOCK = 256  # elements that share a scale


def adamw8(table: torch.Tensor, chunk_tensor: torch.Tensor, chunk_start: torch.Tensor, chunk_elems: int, lr: float,
           wd: float, beta1: float, beta2: float, eps: float, step: int, hp: int | None = None) -> None:
    """adamw with both moments in 8 bits; table rows: p, g, m codes, m scales, v codes, v scales, shadow, n."""
    _lib.call("rgpt_adamw8", ptr(table), ptr(chunk_tensor), ptr(chunk_start), chunk_tensor.numel(), chunk_elems,
              float(lr), float(wd), float(beta1), float(beta2), float(eps), int(step), hp,
              _lib.stream_ptr(table.device))


def adamw8_moments(p: torch.Tensor, mq: torch.Tensor, m_scale: torch.Tensor, vq: torch.Tensor, v_scale: torch.Tensor):
    """(m, v), fp32 of p's shape: the moments of parameter p that 8-bit codes and their scales stand for."""
    a = _packed("zususNN", (p, mq, m_scale, vq, v_scale, None, None))
    if a is not None:
        _call_on(a[6], "rgpt_adamw8_moments", *a[:6], mq.shape[0])
        return a[7], a[8]
    n, dev, f32 = p.numel(), p.get_device(), torch.float32
    blocks = (n + ADAM8_BLOCK - 1) // ADAM8_BLOCK
    args = (_flat(mq, "m codes", (n,), torch.uint8, dev), _flat(m_scale, "m scales", (blocks,), f32, dev),
            _flat(vq, "v codes", (n,), torch.uint8, dev), _flat(v_scale, "v scales", (blocks,), f32, dev))
    if dev < 0:
        raise RuntimeError("librgpt_kernels only takes CUDA tensors (no CPU path)")
    m, v = (torch.empty(p.shape, device=p.device, dtype=f32) for _ in range(2))
    _call_on(dev, "rgpt_adamw8_moments", *args, m.data_ptr(), v.data_ptr(), n)
    return m, v


def muon_prep(table, n, R, C, X, beta, nesterov, sumsq, hp: int | None = None) -> None:
    _lib.call("rgpt_muon_prep", ptr(table), n, R, C, ptr(X), X.stride(0), X.stride(1), float(beta), int(nesterov),
              ptr(sumsq), hp, _lib.stream_ptr(X.device))


def ns_scale(X, rows, cols, n, sumsq) -> None:
    _lib.call("rgpt_ns_scale", ptr(X), X.stride(0), X.stride(1), rows, cols, n, ptr(sumsq), _lib.stream_ptr(X.device))


def _ns_src(src: torch.Tensor):
    """(is_bf16, batch/row/col element strides) of a 3-D [n, rows, cols] source view."""
    if src.dim() != 3 or src.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("Newton-Schulz source must be a 3-D fp32/bf16 [n, rows, cols] view")
    return int(src.dtype == torch.bfloat16), src.stride(0), src.stride(1), src.stride(2)


def ns_sumsq(src: torch.Tensor, sumsq: torch.Tensor) -> None:
    """sumsq[b] += ||src[b]||_F^2 (fp32 accumulation)."""
    bf, sb, si, sj = _ns_src(src)
    n, rows, cols = src.shape
    _lib.call("rgpt_ns_sumsq", ptr(src), bf, sb, si, sj, rows, cols, n, ptr(sumsq), _lib.stream_ptr(src.device))


def ns_split(src: torch.Tensor, *, sumsq: torch.Tensor | None = None, xout: torch.Tensor | None = None,
             dst: torch.Tensor | None = None, nblk: int = 0, blk_off: int = 0, lo_mask: int = 0) -> None:
    """v = src / max(||src||_F, 1e-7) (if sumsq given) -> xout (fp32) and nblk bf16 hi/lo blocks of dst.

    Block k starts blk_off elements after dst's first element and holds bf16(v - bf16(v)) if bit k of
    lo_mask is set, else bf16(v). dst and xout share src's [n, rows, cols] indexing (their own strides)."""
    bf, sb, si, sj = _ns_src(src)
    n, rows, cols = src.shape
    if xout is not None and (xout.dtype != torch.float32 or xout.stride(2) != 1):
        raise ValueError("ns_split: xout must be fp32 with unit column stride")
    if dst is not None and (dst.dtype != torch.bfloat16 or dst.stride(2) != 1):
        raise ValueError("ns_split: dst must be bf16 with unit column stride")
    _lib.call("rgpt_ns_split", ptr(src), bf, sb, si, sj, rows, cols, n, ptr(sumsq),
              ptr(xout), xout.stride(0) if xout is not None else 0, xout.stride(1) if xout is not None else 0,
              ptr(dst), dst.stride(0) if dst is not None else 0, dst.stride(1) if dst is not None else 0,
              nblk, blk_off, lo_mask, _lib.stream_ptr(src.device))


def muon_apply(table, n, R, C, X, lr, wd, muon_lr, scale, hp: int | None = None) -> None:
    _lib.call("rgpt_muon_apply", ptr(table), n, R, C, ptr(X), X.stride(0), X.stride(1), float(lr), float(wd),
              float(muon_lr), float(scale), hp, _lib.stream_ptr(X.device))


# ----------------------------------------------------------------------------- data-parallel staging
SEG_CHUNK = 16384


def segment_table(segs, device):
    """Device table and work list of rgpt_segment_copy for segments (tensor, bf16 copy or None, buffer
    offset, element offset in the tensor, count): (table int64 [n, 4], chunk_seg int32, chunk_start int64)."""
    rows, cs, cst = [], [], []
    for i, (t, t2, off, lo, n) in enumerate(segs):
        if not t.is_contiguous() or (t2 is not None and (not t2.is_contiguous() or t2.dtype != torch.bfloat16)):
            raise ValueError("segment tensors must be contiguous (second tensors bf16)")
        rows.append([t.data_ptr() + lo * t.element_size(), t2.data_ptr() + lo * 2 if t2 is not None else 0, off, n])
        for st in range(0, n, SEG_CHUNK):
            cs.append(i)
            cst.append(st)
    if not rows:
        return None
    return (torch.tensor(rows, dtype=torch.int64).to(device), torch.tensor(cs, dtype=torch.int32).to(device),
            torch.tensor(cst, dtype=torch.int64).to(device))


def segment_copy(plan, buf: torch.Tensor, tensor_bf16: bool, scale: float = 1.0, unpack: bool = False) -> None:
    """Pack the plan's segments into buf (unpack=False) or write buf back into them (unpack=True)."""
    if plan is None:
        return
    table, cs, cst = plan
    if buf.dtype not in (torch.float32, torch.bfloat16) or not buf.is_contiguous():
        raise ValueError("staging buffers are contiguous fp32 or bf16")
    _lib.call("rgpt_segment_copy", ptr(table), ptr(cs), ptr(cst), cs.numel(), SEG_CHUNK, ptr(buf),
              int(buf.dtype == torch.bfloat16), int(tensor_bf16), float(scale), int(unpack), _lib.stream_ptr(buf.device))


def ns_chain(X: torch.Tensor, X2: torch.Tensor, A: torch.Tensor, B: torch.Tensor, xr: int, xc: int, steps: int,
             a: float, b: float, c: float, counters: torch.Tensor) -> None:
    """The whole quintic Newton-Schulz iteration of the n matrices X[:, :xr, :xc] (normalised, bf16) in one
    persistent launch; the result lands in X2 for odd `steps`, else in X. A, B [n, >=xr, >=xr] scratch,
    counters int32 [>= n * 3 * steps] (zeroed by the call)."""
    for t, nme in ((X, "X"), (X2, "X2"), (A, "A"), (B, "B")):
        if t.dtype != torch.bfloat16 or t.dim() != 3 or t.stride(2) != 1:
            raise ValueError(f"ns_chain: {nme} must be a 3-D bf16 tensor with unit column stride")
    if X2.stride() != X.stride() or B.stride() != A.stride():
        raise ValueError("ns_chain: X/X2 and A/B must share strides")
    n = X.shape[0]
    if counters.dtype != torch.int32 or counters.numel() < n * 3 * steps:
        raise ValueError("ns_chain: counters must be int32 with >= n * 3 * steps entries")
    _lib.call("rgpt_ns_chain", ptr(X), ptr(X2), ptr(A), ptr(B), n, xr, xc, X.stride(1), X.stride(0), A.stride(1),
              A.stride(0), int(steps), float(a), float(b), float(c), ptr(counters), _lib.stream_ptr(X.device))
