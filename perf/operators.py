"""The post-training operators, measured: token log-probabilities, the preference and the policy loss
(straight from logits, with their gradients), log-probabilities from hidden states without logits, and AdamW
with 8-bit states.

`run` computes each in its plain form (elementary torch operations, 32 bits, 64 for sums and ratios), or, with
`own` set, through `rgpt_b200.native` and `rgpt_b200.optimizer`. Which tokens are scored follows from the case
alone (prompt and padding lengths of each sequence), the values from the seed.
"""
import math

import numpy as np
import torch

own = False

IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 256       # elements that share one scale of the 8-bit moments
M_TOP = 448.0     # largest value of the first moment's code (float8 e4m3)
R_TOP = 1.96875   # largest value of the code of sqrt(second moment): 3 bits exponent, 5 bits mantissa, no sign
TINY = 2.0 ** -100  # a block whose largest moment is not above this holds zeros
ROWS = 2048       # rows that are made, or computed in 64 bits, at a time


def _f(v):
    return float(np.float32(v))


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a custom loss on a few fp32 logits of the reference's own, odd vocabulary: latency, a row past 16 bytes' alignment
        dict(name="logps short fp32", op="logps", dtype="fp32", B=2, T=24, V=50257, prompt=0.0, pad=0.0, shifted=False),
        # a training batch's logits shifted by one (a view with its own batch stride), prompts masked
        dict(name="logps batch bf16", op="logps", dtype="bf16", B=4, T=1023, V=50304, prompt=0.3, pad=0.1, shifted=True),
        # two pairs over a toy vocabulary (the test models' size): launches and latency
        dict(name="preference tiny", op="preference", dtype="bf16", B=4, T=48, V=1000, prompt=0.3, pad=0.2, shifted=False,
             kind="hinge", beta=0.5, smoothing=0.0, margin=0.0, average=False, free=False),
        # short answers, odd vocabulary, fp16, length-normalised and without a reference
        dict(name="preference short fp16", op="preference", dtype="fp16", B=16, T=127, V=50257, prompt=0.4, pad=0.1, shifted=False,
             kind="sigmoid", beta=2.0, smoothing=0.0, margin=0.5, average=True, free=True),
        # eight pairs at the model's full length
        dict(name="preference full bf16", op="preference", dtype="bf16", B=16, T=1023, V=50304, prompt=0.4, pad=0.1, shifted=True,
             kind="sigmoid", beta=0.1, smoothing=0.1, margin=0.0, average=False, free=False),
        # one action for each of 64 contexts
        dict(name="policy one token", op="policy", dtype="bf16", B=64, T=1, V=50304, prompt=0.0, pad=0.0, shifted=False,
             low=0.2, high=0.2, kl=0.0, per_token=False, by_sequence=False),
        # a group of sampled answers with the KL term at full length
        dict(name="policy full bf16", op="policy", dtype="bf16", B=16, T=1023, V=50304, prompt=0.2, pad=0.2, shifted=True,
             low=0.2, high=0.28, kl=0.04, per_token=False, by_sequence=True),
        # scoring the next token of 16 sequences from their last hidden states: the weight's bytes
        dict(name="linear next token", op="linear", M=16, V=50304, K=512, train=False),
        # scoring a whole batch by the frozen reference
        dict(name="linear batch", op="linear", M=16368, V=50304, K=512, train=False),
        # training through it, logits never held whole, odd rows and vocabulary, the 350M configuration's width
        dict(name="linear train", op="linear", M=4095, V=50257, K=1024, train=True),
        # a handful of small matrices and one odd vector
        dict(name="adamw8 small", op="adamw8", sizes="4096,16384,5001,262144", step=10, shadow=False),
        # the embedding and the lm_head of the small model
        dict(name="adamw8 full", op="adamw8", sizes="25755648,25755648", step=1000, shadow=True),
    ]


def _between(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.4)))))))


def draw(rng):
    op = rng.choice(["logps", "preference", "policy", "linear", "adamw8"])
    if op == "linear":
        K = 8 * _between(rng, 8, 256)
        V, M = _between(rng, 100, 66000), _between(rng, 1, 16368)
        train = rng.random() < 0.5
        while M * V * K * (4 if train else 1) > 16368 * 50304 * 512:
            M = max(1, M // 2)
        return dict(op=op, M=M, V=V, K=K, train=train)
    if op == "adamw8":
        sizes = [_between(rng, 4096, 6000000) for _ in range(rng.randint(1, 8))]
        return dict(op=op, sizes=",".join(map(str, sizes)), step=_between(rng, 1, 20000), shadow=rng.random() < 0.5)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    V = rng.choice([50304, _between(rng, 16, 131072), 8 * _between(rng, 16, 16384)])
    T, B = _between(rng, 1, 1024), 2 * _between(rng, 1, 16)
    while B * T * V * (2 if dtype == "fp32" else 1) > 16 * 1023 * 50304:
        T = max(1, T // 2)
        B = B if T > 1 else max(2, B // 4 * 2)
    c = dict(op=op, dtype=dtype, B=B, T=T, V=V, prompt=rng.choice([0.0, rng.uniform(0.0, 0.7)]), pad=rng.choice([0.0, rng.uniform(0.0, 0.6)]),
             shifted=rng.random() < 0.5)
    if op == "preference":
        c.update(kind=rng.choice(["sigmoid", "sigmoid", "hinge", "squared"]), beta=rng.choice([0.05, 0.1, 0.5]), smoothing=0.0,
                 margin=rng.choice([0.0, 0.5]), average=rng.random() < 0.4, free=False)
        if c["average"]:  # the mean over tokens goes with a larger beta, and may go without a reference
            c.update(beta=rng.choice([0.5, 2.0]), free=rng.random() < 0.5)
        if c["kind"] == "sigmoid":
            c["smoothing"] = rng.choice([0.0, 0.1])
    if op == "policy":
        c.update(low=0.2, high=rng.choice([0.2, 0.28]), kl=rng.choice([0.0, 0.01, 0.1]), per_token=rng.random() < 0.5, by_sequence=rng.random() < 0.5)
    return c


def _spans(c):
    """The scored tokens [first, last) of each sequence: prompts and padding differ from sequence to sequence; one may be left empty."""
    out = []
    for i in range(c["B"]):
        wave = 0.5 + (i * 7 % c["B"]) / c["B"]
        first = min(c["T"], int(c["T"] * c["prompt"] * wave))
        last = max(first, c["T"] - int(c["T"] * c["pad"] * (2.0 - wave)))
        out.append((first, last))
    return out


def work(c):
    if c["op"] == "linear":
        mnk = float(c["M"]) * c["V"] * c["K"]
        io = 2.0 * (c["M"] + c["V"]) * c["K"]
        return {"bytes": io * (2 if c["train"] else 1) + 16.0 * c["M"], "flops": mnk * (6 if c["train"] else 2)}
    if c["op"] == "adamw8":
        n = sum(map(int, c["sizes"].split(",")))
        blocks = sum(-(-int(s) // BLOCK) for s in c["sizes"].split(","))
        # parameter and both codes read and written, gradient read, the bf16 copy written; the moments that are returned
        return {"bytes": n * (8.0 + 4.0 + 4.0 + (2.0 if c["shadow"] else 0.0) + 8.0) + 16.0 * blocks, "flops": 20.0 * n}
    e, rows = DTYPES[c["dtype"]].itemsize, c["B"] * c["T"]
    scored = sum(b - a for a, b in _spans(c))
    per_row = {"logps": 16, "preference": 12, "policy": 24}[c["op"]]
    return {"bytes": float(e) * c["V"] * (scored + rows) + per_row * rows, "flops": 6.0 * scored * c["V"]}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(c, g):
    """Logits as a trained model's: spread 2.5, the label up to 10 above, held [B, T + 1, V] where the view is shifted."""
    B, T, V = c["B"], c["T"], c["V"]
    held = torch.empty(B, T + 1 if c["shifted"] else T, V, device="cuda", dtype=DTYPES[c["dtype"]])
    flat = held.view(-1, V)
    for r in range(0, flat.shape[0], ROWS):
        flat[r:r + ROWS] = 2.5 * torch.randn(min(ROWS, flat.shape[0] - r), V, device="cuda", generator=g)
    x = held[:, :-1] if c["shifted"] else held
    labels = torch.randint(0, V, (B, T), device="cuda", generator=g)
    at = x.gather(2, labels[..., None])
    x.scatter_(2, labels[..., None], (at.float() + 10.0 * torch.rand(at.shape, device="cuda", generator=g)).to(x.dtype))
    t = torch.arange(T, device="cuda")
    span = torch.tensor(_spans(c), device="cuda")
    labels[(t < span[:, :1]) | (t >= span[:, 1:])] = IGNORE
    return x, labels


def _behind(x, labels):
    """Log-probabilities of the labels, as another pass of the model would have given them."""
    lp = torch.empty(labels.shape, device="cuda")
    for b in range(labels.shape[0]):
        for t in range(0, labels.shape[1], ROWS):
            f = x[b, t:t + ROWS].float()
            lp[b, t:t + ROWS] = f.gather(1, labels[b, t:t + ROWS].clamp_min(0)[:, None])[:, 0] - torch.logsumexp(f, 1)
    return torch.where(labels == IGNORE, torch.zeros_like(lp), lp)


def prepare(c, seed):
    g, op = _gen(seed), c["op"]
    new = lambda *s, dt=torch.float32: torch.empty(*s, device="cuda", dtype=dt)  # noqa: E731
    if op == "linear":
        x = torch.randn(c["M"], c["K"], device="cuda", generator=g).bfloat16()  # a normalised hidden state
        w = (torch.randn(c["V"], c["K"], device="cuda", generator=g) * (2.0 / math.sqrt(c["K"]))).bfloat16()
        labels = torch.randint(0, c["V"], (c["M"],), device="cuda", generator=g)
        labels[torch.rand(c["M"], device="cuda", generator=g) < 0.1] = IGNORE
        s = dict(case=c, x=x, w=w, labels=labels, logps=new(c["M"]), lse=new(c["M"]))
        if c["train"]:
            s.update(dlogps=torch.randn(c["M"], device="cuda", generator=g) / c["M"], dx=torch.empty_like(x), dw=torch.empty_like(w))
        return s
    if op == "adamw8":
        return _prepare_adamw8(c, g)
    x, labels = _logits(c, g)
    B, T = labels.shape
    s = dict(case=c, logits=x, labels=labels, dlogits=new(B, T, c["V"], dt=x.dtype), logps=new(B, T), lse=new(B, T))
    if op == "logps":
        s["dlogps"] = torch.randn(B, T, device="cuda", generator=g) / (B * T)
    if op == "preference":
        n = (labels != IGNORE).sum(1)
        ref = (_behind(x, labels).double().sum(1) + 0.3 * n.sqrt() * torch.randn(B, device="cuda", generator=g)).float()
        s["ref"] = None if c["free"] else ref / n.clamp_min(1) if c["average"] else ref
        s.update(seq_logps=new(B), margins=new(B // 2), coef=new(B), loss=new(1))
    if op == "policy":
        lp = _behind(x, labels)
        s["old"] = lp + 0.15 * torch.randn(B, T, device="cuda", generator=g)
        s["ref"] = lp + 0.3 * torch.randn(B, T, device="cuda", generator=g) if c["kl"] else None
        s["adv"] = 0.25 + torch.randn(*((B, T) if c["per_token"] else (B,)), device="cuda", generator=g)
        s.update(counts=new(B, dt=torch.int32), stats=new(4))
    return s


def _prepare_adamw8(c, g):
    """Parameters in the middle of training: codes and scales that some hundred steps have left."""
    ps, gs, st, sh = [], [], [], []
    for n in map(int, c["sizes"].split(",")):
        size = torch.exp(0.8 * torch.randn(n, device="cuda", generator=g)) * 1e-3  # each element's own gradient scale
        m = size * torch.randn(n, device="cuda", generator=g) * 0.3
        r = size * (0.7 + 0.6 * torch.rand(n, device="cuda", generator=g))
        ps.append(0.02 * torch.randn(n, device="cuda", generator=g))
        gs.append(size * torch.randn(n, device="cuda", generator=g))
        st.append(list(_pack(m, r)))
        sh.append(ps[-1].bfloat16() if c["shadow"] else None)
    s = dict(case=c, p=ps, g=gs, st=st, sh=sh, step=c["step"], lr=3e-4, wd=0.1, betas=(0.9, 0.95), eps=1e-8)
    if own:  # the optimizer that a training program holds, resumed at this step
        from rgpt_b200.optimizer import Muon

        params = [torch.nn.Parameter(p) for p in ps]
        opt = Muon([{"params": params, "use_muon": False}], lr=s["lr"], weight_decay=s["wd"], adam_betas=s["betas"], adam_eps=s["eps"],
                   adam_state_bits=8)
        for p, gr, q, b in zip(params, gs, st, sh):
            p.grad = gr
            if b is not None:
                p._rgpt_shadow = b
            opt.state[p] = dict(zip(("exp_avg_q8", "exp_avg_scale", "exp_avg_sq_q8", "exp_avg_sq_scale"), q))
        opt.param_groups[0]["_adam_step"] = s["step"]
        s.update(opt=opt, params=params)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _blocks(v):
    """v in rows of one block each, zeros behind the last element."""
    n = v.numel()
    return torch.nn.functional.pad(v, (0, -n % BLOCK)).view(-1, BLOCK)


def _pack(m, r):
    """(codes, scales) of the first moment m, then of r = sqrt(second moment)."""
    n = m.numel()
    m, r = _blocks(m), _blocks(r)
    a, b = m.abs().amax(1, keepdim=True), r.amax(1, keepdim=True)
    a, b = torch.where(a > TINY, a, torch.zeros_like(a)), torch.where(b > TINY, b, torch.zeros_like(b))
    mq = (m * torch.where(a > 0, a.reciprocal() * M_TOP, a)).to(torch.float8_e4m3fn).view(torch.uint8).reshape(-1)[:n].contiguous()
    y = r * torch.where(b > 0, b.reciprocal() * R_TOP, b)
    bits = y.view(torch.int32)
    fine = ((bits + 0x1FFFF + ((bits >> 18) & 1)) >> 18) - (120 << 5)  # 5 bits of mantissa, ties to even
    q = torch.where(y >= 2.0 ** -6, fine, torch.round(y * 2048.0).to(torch.int32)).clamp(0, 255)
    q = torch.where(r > 0, q.clamp_min(1), q)  # a moment above zero stays above zero
    return mq, (a * _f(1.0 / M_TOP)).reshape(-1), q.to(torch.uint8).reshape(-1)[:n].contiguous(), (b * _f(1.0 / R_TOP)).reshape(-1)


def _unpack(q):
    """The moments that codes and scales stand for."""
    mq, ms, rq, rs = q
    n = mq.numel()
    m = (_blocks(mq.view(torch.float8_e4m3fn).float()) * ms[:, None]).reshape(-1)[:n]
    code = rq.to(torch.int32)
    y = torch.where(code >= 32, ((code + (120 << 5)) << 18).view(torch.float32), code.float() * 2.0 ** -11)
    r = (_blocks(y) * rs[:, None]).reshape(-1)[:n]
    return m, r * r


def _adamw8(s):
    """One step; every operation rounded to 32 bits by itself, since the codes jump at the borders between two values."""
    s["step"] += 1
    b1, b2 = np.float32(s["betas"][0]), np.float32(s["betas"][1])
    c1, c2 = 1.0 - float(b1) ** s["step"], 1.0 - float(b2) ** s["step"]
    decay = _f(np.float32(1.0) - np.float32(s["lr"]) * np.float32(s["wd"]))
    out = []
    for p, g, q, sh in zip(s["p"], s["g"], s["st"], s["sh"]):
        m, v = _unpack(q)
        m = m * float(b1) + g * float(np.float32(1.0) - b1)
        v = v * float(b2) + (g * g) * float(np.float32(1.0) - b2)
        r = v.sqrt()
        u = (m / (r * _f(1.0 / math.sqrt(c2)) + _f(s["eps"]))) * _f(1.0 / c1)
        p.copy_(p * decay - u * _f(s["lr"]))
        for old, new in zip(q, _pack(m, r)):
            old.copy_(new)
        if sh is not None:
            sh.copy_(p)
        out += [p, *_unpack(q)] + ([sh] if sh is not None else [])
    return out


def _stats(x, labels):
    """Scored rows in 32 bits: (mask, label, exp(x - max), its sum, log-probability and log-sum-exp in 64 bits)."""
    mask = labels != IGNORE
    safe = torch.where(mask, labels, torch.zeros_like(labels))
    f = x.float()
    top = f.amax(-1, keepdim=True)
    e = torch.exp(f - top)
    z = e.sum(-1, keepdim=True)
    lse = top.double() + torch.log(z.double())
    lp = torch.where(mask, (f.gather(-1, safe[..., None]).double() - lse)[..., 0], torch.zeros_like(lse[..., 0]))
    return mask, safe, e, z, lp, lse[..., 0]


def _grad(x, mask, safe, e, z, coef):
    """coef * (onehot - softmax), zero rows where nothing is scored."""
    coef = torch.where(mask, coef, torch.zeros_like(coef)).float()[..., None]
    d = e * (-coef / z)
    d.scatter_add_(-1, safe[..., None], coef)
    return d.to(x.dtype)


def _softplus(h):
    return torch.clamp_min(h, 0.0) + torch.log1p(torch.exp(-h.abs()))


def _sigmoid(h):
    e = torch.exp(-h.abs())
    return torch.where(h >= 0, 1.0 / (1.0 + e), e / (1.0 + e))


def _preference_terms(c, h):
    """(loss, d loss / d h) of each pair."""
    if c["kind"] == "hinge":
        return torch.clamp_min(1.0 - h, 0.0), torch.where(h < 1.0, -torch.ones_like(h), torch.zeros_like(h))
    if c["kind"] == "squared":
        return (h - 0.5) ** 2, 2.0 * (h - 0.5)
    s = c["smoothing"]
    return (1.0 - s) * _softplus(-h) + s * _softplus(h), -(1.0 - s) * _sigmoid(-h) + s * _sigmoid(h)


def _preference(c, lp, mask, ref):
    P = c["B"] // 2
    n = mask.sum(1).clamp_min(1) if c["average"] else torch.ones(c["B"], device=lp.device)
    seq = lp.sum(1) / n
    ratio = seq if ref is None else seq - ref.double()
    h = c["beta"] * (ratio[:P] - ratio[P:]) - c["margin"]
    loss, dh = _preference_terms(c, h)
    dh = dh * c["beta"] / P
    return loss.mean(), seq, h, torch.cat([dh, -dh]) / n


def _policy(c, lp, mask, old, ref, adv):
    """(loss, policy term, KL, clipped share), and d loss / d logp of each token."""
    lp = lp.double()
    old = old.double()
    adv = (adv if c["per_token"] else adv[:, None]).double().expand_as(lp)
    n = mask.sum(1, keepdim=True)
    w = 1.0 / (n.clamp_min(1) * (n > 0).sum().clamp_min(1)) if c["by_sequence"] else 1.0 / n.sum().clamp_min(1)
    w = torch.where(mask, torch.ones_like(lp) * w, torch.zeros_like(lp))
    r = torch.exp(lp - old)
    cut = torch.where(adv >= 0, (r > 1.0 + c["high"]) & (adv > 0), r < 1.0 - c["low"])
    bound = torch.where(adv >= 0, torch.full_like(r, 1.0 + c["high"]), torch.full_like(r, 1.0 - c["low"]))
    pg = -torch.where(cut, bound, r) * adv
    d = torch.where(cut, torch.zeros_like(r), -r * adv)
    kl = torch.zeros_like(r)
    if ref is not None:
        q = ref.double() - lp
        kl = torch.exp(q) - q - 1.0
        d = d + c["kl"] * (1.0 - torch.exp(q))
    pg, kl, cut = ((w * torch.where(mask, v, torch.zeros_like(w))).sum() for v in (pg, kl, cut.double()))
    return torch.stack([pg + c["kl"] * kl, pg, kl, cut]), w * d


def _plain(s):
    c = s["case"]
    if c["op"] == "adamw8":
        return _adamw8(s)
    if c["op"] == "linear":
        x, w = s["x"].float(), s["w"].float()
        mask, safe, e, z, lp, _ = _stats(x @ w.t(), s["labels"])
        if not c["train"]:
            return lp.float()
        d = _grad(x, mask, safe, e, z, s["dlogps"])
        return lp.float(), (d @ w).to(s["x"].dtype), (d.t() @ x).to(s["w"].dtype)
    x = s["logits"]
    mask, safe, e, z, lp, _ = _stats(x, s["labels"])
    if c["op"] == "logps":
        return lp.float(), _grad(x, mask, safe, e, z, s["dlogps"])
    if c["op"] == "preference":
        loss, seq, h, coef = _preference(c, lp, mask, s["ref"])
        return loss.float(), seq.float(), h.float(), _grad(x, mask, safe, e, z, coef[:, None].expand_as(lp))
    stats, coef = _policy(c, lp, mask, s["old"], s["ref"], s["adv"])
    return stats.float(), lp.float(), _grad(x, mask, safe, e, z, coef)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    from rgpt_b200 import native as nv

    c = s["case"]
    if c["op"] == "adamw8":
        s["opt"].step()
        out = []
        for p, sh in zip(s["params"], s["sh"]):
            out += [p.detach(), *s["opt"].adam_moments(p)] + ([sh] if sh is not None else [])
        return out
    if c["op"] == "linear":
        nv.linear_logprobs(s["x"], s["w"], s["labels"], s["logps"], lse=s["lse"])
        if not c["train"]:
            return s["logps"]
        nv.linear_logprobs_bwd(s["x"], s["w"], s["labels"], s["lse"], s["dlogps"], s["dx"], s["dw"])
        return s["logps"], s["dx"], s["dw"]
    if c["op"] == "logps":
        nv.token_logprobs(s["logits"], s["labels"], s["logps"], lse=s["lse"])
        nv.token_logprobs_bwd(s["logits"], s["labels"], s["lse"], s["dlogps"], s["dlogits"])
        return s["logps"], s["dlogits"]
    if c["op"] == "preference":
        nv.preference_loss(s["logits"], s["labels"], s["ref"], token_logps=s["logps"], lse=s["lse"], seq_logps=s["seq_logps"], margins=s["margins"],
                           coef=s["coef"], loss=s["loss"], dlogits=s["dlogits"], kind=c["kind"], beta=c["beta"], label_smoothing=c["smoothing"],
                           margin=c["margin"], average=c["average"])
        return s["loss"][0], s["seq_logps"], s["margins"], s["dlogits"]
    nv.policy_loss(s["logits"], s["labels"], s["old"], s["adv"], s["ref"], token_logps=s["logps"], counts=s["counts"], stats=s["stats"],
                   dlogits=s["dlogits"], clip_low=c["low"], clip_high=c["high"], kl_coef=c["kl"], by_sequence=c["by_sequence"])
    return s["stats"], s["logps"], s["dlogits"]


def run(s):
    return _own(s) if own else _plain(s)


# ------------------------------------------------------------------------------------------------ 64 bits, from the definitions
def _exact_rows(rows, labels):
    """log softmax of the labels, row after row: rows(a, b) gives the logits of rows a to b in 64 bits."""
    lp = torch.zeros(labels.numel(), device="cuda", dtype=torch.float64)
    for a in range(0, labels.numel(), ROWS):
        y = labels[a:a + ROWS]
        v = torch.log_softmax(rows(a, a + ROWS), 1).gather(1, y.clamp_min(0)[:, None])[:, 0]
        lp[a:a + ROWS] = torch.where(y == IGNORE, 0.0, v)
    return lp


def _exact_grad(rows, labels, coef, take):
    for a in range(0, labels.numel(), ROWS):
        y = labels[a:a + ROWS]
        k = torch.where(y == IGNORE, 0.0, coef[a:a + ROWS])
        p = torch.softmax(rows(a, a + ROWS), 1)
        p[torch.arange(y.numel(), device="cuda"), y.clamp_min(0)] -= 1.0
        take(a, p.mul_(-k[:, None]))


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "adamw8":
        return _exact_adamw8(s)
    if c["op"] == "linear":
        x, w, y = s["x"].double(), s["w"].double(), s["labels"]
        rows = lambda a, b: x[a:b] @ w.t()  # noqa: E731
        lp = _exact_rows(rows, y)
        if not c["train"]:
            return lp
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)

        def take(a, d):
            dx[a:a + ROWS] = d @ w
            dw.addmm_(d.t(), x[a:a + ROWS])

        _exact_grad(rows, y, s["dlogps"].double(), take)
        return lp, dx, dw
    B, T, V = s["logits"].shape
    y = s["labels"].reshape(-1)
    flat = s["logits"].reshape(-1, V)
    rows = lambda a, b: flat[a:b].double()  # noqa: E731
    lp = _exact_rows(rows, y)
    by = lp.view(B, T)
    on = (y != IGNORE).view(B, T).double()
    if c["op"] == "logps":
        first, coef = [lp.view(B, T)], s["dlogps"].double().reshape(-1)
    elif c["op"] == "preference":
        seq = by.sum(1) / (on.sum(1).clamp_min(1.0) if c["average"] else 1.0)
        seq.requires_grad_(True)
        P = B // 2
        h = seq[:P] - seq[P:]
        if s["ref"] is not None:
            h = h - (s["ref"][:P].double() - s["ref"][P:].double())
        h = c["beta"] * h - c["margin"]
        k = c["smoothing"]
        log_sig = torch.nn.functional.logsigmoid
        f = {"sigmoid": lambda: -(1 - k) * log_sig(h) - k * log_sig(-h), "hinge": lambda: torch.relu(1 - h), "squared": lambda: (h - 0.5).square()}[c["kind"]]()
        loss = f.sum() / P
        (ds,) = torch.autograd.grad(loss, seq)
        if c["average"]:
            ds = ds / on.sum(1).clamp_min(1.0)
        first, coef = [loss.detach(), seq.detach(), h.detach()], ds[:, None].expand(B, T).reshape(-1)
    else:
        v = by.clone().requires_grad_(True)
        w = on / (on.sum(1, keepdim=True).clamp_min(1.0) * (on.sum(1) > 0).sum().clamp_min(1)) if c["by_sequence"] else on / on.sum().clamp_min(1.0)
        a = s["adv"].double() if c["per_token"] else s["adv"].double()[:, None]
        r = torch.exp(v - s["old"].double())
        lo, hi = 1.0 - c["low"], 1.0 + c["high"]
        pg = (w * -torch.minimum(r * a, r.clamp(lo, hi) * a)).sum()
        kl = (w * (torch.exp(s["ref"].double() - v) - (s["ref"].double() - v) - 1.0)).sum() if s["ref"] is not None else pg.detach() * 0.0
        cut = (w * (r.clamp(lo, hi) * a < r * a)).sum()
        loss = pg + c["kl"] * kl
        (dv,) = torch.autograd.grad(loss, v)
        first, coef = [torch.stack([loss, pg, kl, cut]).detach(), by], dv.reshape(-1)
    d = torch.empty(B * T, V, device="cuda", dtype=torch.float64)

    def put(a, g):
        d[a:a + ROWS] = g

    _exact_grad(rows, y, coef, put)
    return (*first, d.view(B, T, V))


def _exact_adamw8(s):
    """The parameters; the moments' codes have no 64-bit value: they jump where 32 bits round the other way."""
    out, t = [], s["step"] + 1
    b1, b2 = (float(np.float32(b)) for b in s["betas"])
    lr, wd, eps = _f(s["lr"]), _f(s["wd"]), _f(s["eps"])
    e4m3 = torch.arange(256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()
    code = torch.arange(256, device="cuda", dtype=torch.float64)
    e3m5 = torch.where(code < 32, code * 2.0 ** -11, 2.0 ** (torch.floor(code / 32) - 7) * (1 + (code % 32) / 32))
    for p, g, (mq, ms, rq, rs), sh in zip(s["p"], s["g"], s["st"], s["sh"]):
        blk = torch.arange(p.numel(), device="cuda") // BLOCK
        m = e4m3[mq.long()] * ms.double()[blk]
        v = (e3m5[rq.long()] * rs.double()[blk]) ** 2
        m = b1 * m + (1 - b1) * g.double()
        v = b2 * v + (1 - b2) * g.double() ** 2
        new = p.double() * (1 - lr * wd) - lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
        out += [new, None, None] + ([new] if sh is not None else [])
    return out
