"""Cases of the decoder-step operators that stand around the SSA attention: the LM head with its
cross entropy, the gated feed-forward, the per-head norm with the rotation of queries and keys, and
the global gradient norm with clipping. Each has a plain form in elementary torch operations and
the call a user makes of the framework's kernel.

    linear_ce  loss of hidden @ weight^T against targets, and with "train" the gradients of both
    gated_ffn  silu(x Wg^T) * (x Wu^T), and with "train" the gradients of x and the weights
    qk_rope    q, k = rotate(rmsnorm(q, k)) out of the packed qkv projection, and with "train" the
               gradient of qkv and of the two norm weights
    grad_clip  the 2-norm over many gradient tensors, and the gradients scaled into the optimizer's
               fp32 buffer (or, with "norm_only", the norm alone)
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-5


def _framework():
    root = str(Path(__file__).resolve().parent.parent / "luciole-1b_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    from SSA.ssa_gated_ffn import ssa_gated_ffn
    from SSA.ssa_grad_clip import ssa_clip_grad_norm, ssa_grad_norm
    from SSA.ssa_qk_norm_rope import ssa_qk_norm_rope
    return (ssa_linear_cross_entropy, ssa_gated_ffn, ssa_qk_norm_rope, ssa_clip_grad_norm,
            ssa_grad_norm)


# --------------------------------------------------------------------------------------- cases
def listed():
    return [
        # The Luciole-1B training step's head: 4 sequences of 2048, vocabulary 65,536.
        dict(name="ce_train", op="linear_ce", n=8192, h=2048, v=65536, dtype="bf16", train=True,
             reduction="mean", ignored=0.02),
        # Per-token log-likelihood of one scored sequence (2049 tokens, shifted by one).
        dict(name="ce_score", op="linear_ce", n=2048, h=2048, v=65536, dtype="bf16", train=False,
             reduction="none", ignored=0.1),
        # A small decoder's step with a vocabulary that is no multiple of anything.
        dict(name="ce_train_odd", op="linear_ce", n=511, h=512, v=50257, dtype="fp16", train=True,
             reduction="mean", ignored=0.3),
        # The Luciole-1B step's feed-forward.
        dict(name="ffn_train", op="gated_ffn", n=8192, h=2048, f=5632, dtype="bf16", train=True),
        # The same layer run on one token.
        dict(name="ffn_token", op="gated_ffn", n=1, h=2048, f=5632, dtype="bf16", train=False),
        # A small decoder's layer on a ragged batch, inner width 8/3 of the hidden size.
        dict(name="ffn_train_odd", op="gated_ffn", n=1337, h=512, f=1365, dtype="fp16",
             train=True),
        # Queries and keys of the Luciole-1B step, with per-head norms.
        dict(name="rope_train", op="qk_rope", b=4, s=2048, hq=32, hkv=8, d=64, dtype="bf16",
             train=True, norm=True, packed=False, far=0),
        # 65,536 packed tokens, positions restart at each document, rotation alone.
        dict(name="rope_packed", op="qk_rope", b=1, s=65536, hq=32, hkv=8, d=64, dtype="bf16",
             train=False, norm=False, packed=True, far=0),
        # Three single tokens of different sequences, far into their contexts, wide heads.
        dict(name="rope_token", op="qk_rope", b=1, s=3, hq=32, hkv=8, d=128, dtype="fp16",
             train=False, norm=True, packed=True, far=30000),
        # All gradients of the 16-layer model clipped into the fp32 master gradients.
        dict(name="clip_model", op="grad_clip", layers=16, h=2048, hq=32, hkv=8, f=5632, v=65536,
             dtype="bf16", norm_only=False, clipped=True),
        # A two-layer model's gradients: many small tensors, latency counts.
        dict(name="clip_small", op="grad_clip", layers=2, h=128, hq=4, hkv=2, f=341, v=509,
             dtype="fp32", norm_only=False, clipped=True),
        # The norm that a training log shows, of one layer and the embedding, in fp32.
        dict(name="norm_log", op="grad_clip", layers=1, h=2048, hq=32, hkv=8, f=5632, v=16384,
             dtype="fp32", norm_only=True, clipped=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["linear_ce", "gated_ffn", "qk_rope", "grad_clip"])
    train = rng.random() < 0.6
    if op == "linear_ce":
        return dict(op=op, n=_log(rng, 1, 8192), h=8 * _log(rng, 8, 256), v=_log(rng, 100, 65536),
                    dtype=rng.choice(["bf16", "bf16", "fp16"]), train=train,
                    reduction=rng.choice(["mean", "sum", "none"]),
                    ignored=rng.choice([0.0, 0.1, 0.5]))
    if op == "gated_ffn":
        return dict(op=op, n=_log(rng, 1, 8192), h=8 * _log(rng, 8, 256), f=_log(rng, 96, 5632),
                    dtype=rng.choice(["bf16", "bf16", "fp16"]), train=train)
    if op == "qk_rope":
        hq, hkv = rng.choice([(32, 8), (24, 8), (16, 2), (8, 8), (6, 2), (5, 1), (1, 1)])
        d = rng.choice([16, 32, 64, 64, 128])
        packed = rng.random() < 0.5
        b = 1 if packed else rng.choice([1, 2, 4])
        cap = min(65536, 32 * 65536 // (hq * b))
        return dict(op=op, b=b, s=_log(rng, 1, cap if d <= 64 else cap // 2), hq=hq, hkv=hkv, d=d,
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), train=train,
                    norm=rng.random() < 0.6, packed=packed,
                    far=rng.choice([0, 0, 1000, 100000]))
    return dict(op=op, layers=_log(rng, 1, 16), h=8 * _log(rng, 8, 200), hq=8, hkv=2,
                f=_log(rng, 96, 4096), v=_log(rng, 100, 50000),
                dtype=rng.choice(["bf16", "fp16", "fp32"]), norm_only=not train,
                clipped=rng.random() < 0.7)


def _grad_shapes(c):
    """The gradient tensors of a decoder of these sizes."""
    h, d = c["h"], max(1, c["h"] // c["hq"])
    layer = [(h,), ((c["hq"] + 2 * c["hkv"]) * d, h), (h, c["hq"] * d), (h,), (2 * c["f"], h),
             (h, c["f"]), (c["hq"],)]
    return [(c["v"], h)] + layer * c["layers"] + [(h,), (c["v"], h)]


# --------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, dt, c = "cuda", _DT[case["dtype"]], case
    train = bool(c.get("train"))

    def rand(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    if c["op"] == "linear_ce":
        # normed hidden states; a head whose logits spread a few units; frequent and rare tokens
        x, w = rand(c["n"], c["h"]), rand(c["v"], c["h"], scale=2.0 / math.sqrt(c["h"]))
        u = torch.rand(c["n"], generator=g, device=dev)
        t = (u ** 3 * c["v"]).long().clamp_(max=c["v"] - 1)
        skip = torch.rand(c["n"], generator=g, device=dev) < c["ignored"]
        skip[0] = False
        t = torch.where(skip, torch.full_like(t, -100), t)
        grad = None
        if train:
            x.requires_grad_(True)
            w.requires_grad_(True)
            # fp16 training multiplies the mean loss, so that small gradients stay normal numbers
            scaled = c["dtype"] == "fp16" and c["reduction"] == "mean"
            grad = torch.rand(c["n"], generator=g, device=dev) + 0.5 if c["reduction"] == "none" \
                else torch.full((), 1024.0 if scaled else 1.0, device=dev)
        return dict(case=c, x=x, w=w, t=t, grad=grad)
    if c["op"] == "gated_ffn":
        x, w = rand(c["n"], c["h"]), rand(2 * c["f"], c["h"], scale=1.0 / math.sqrt(c["h"]))
        dh = rand(c["n"], c["f"]) if train else None
        if train:
            x.requires_grad_(True)
            w.requires_grad_(True)
        return dict(case=c, x=x, w=w, dh=dh)
    if c["op"] == "qk_rope":
        b, s, d, hq, hkv = c["b"], c["s"], c["d"], c["hq"], c["hkv"]
        pos, span = None, s
        if c["packed"]:
            # documents of up to 4096 tokens; "far": each begins somewhere inside its context
            start = torch.randint(0, c["far"] + 1, (1,), generator=g, device=dev)
            pos = ((torch.arange(s, device=dev) % 4096) + start).to(torch.int32)
            span = 4096 + c["far"]
        ang = torch.arange(span, device=dev, dtype=torch.float64)[:, None] / 10000.0 ** (
            torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
        ang = torch.cat([ang, ang], dim=-1)
        lead = (s,) if c["packed"] else (b, s)
        qkv = rand(*lead, (hq + 2 * hkv) * d)
        wq, wk = ((1.0 + 0.1 * rand(d, dtype=torch.float32)).to(dt) for _ in range(2)) \
            if c["norm"] else (None, None)
        grads = [rand(*lead, n, d) for n in (hq, hkv, hkv)] if train else None
        for t in (qkv, wq, wk) if train else ():
            if t is not None:
                t.requires_grad_(True)
        return dict(case=c, qkv=qkv, pos=pos, cos=ang.cos().float(), sin=ang.sin().float(), wq=wq,
                    wk=wk, grads=grads)
    shapes = _grad_shapes(c)
    sizes = [math.prod(s) for s in shapes]
    total = sum(sizes)
    grads = [(torch.randn(s, generator=g, device=dev, dtype=dt if dt != torch.float16 else
                          torch.float32) * 1e-2).to(dt) for s in shapes]
    # the optimizer's fp32 gradient buffer, one tensor with a view for each parameter
    flat = torch.zeros(1 if c["norm_only"] else total, device=dev)
    out = None if c["norm_only"] else [v.view(s) for v, s in zip(flat.split(sizes), shapes)]
    norm = 1e-2 * math.sqrt(total)
    return dict(case=c, grads=grads, flat=flat, out=out,
                max_norm=norm * (0.37 if c["clipped"] else 3.0))


# --------------------------------------------------------------------------------------- passes
def _rms(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * w


def _halves(x):
    return x[..., : x.shape[-1] // 2], x[..., x.shape[-1] // 2:]


def _rotate(x, c, s):
    a, b = _halves(x)
    return x * c + torch.cat([-b, a], dim=-1) * s


def _rotate_grad(g, c, s):
    a, b = _halves(g * s)
    return g * c + torch.cat([b, -a], dim=-1)


def _rms_grad(x, w, g):
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
    n = x * r
    gw = g * w
    return r * (gw - n * (gw * n).mean(-1, keepdim=True)), (g * n).reshape(-1, x.shape[-1])


def _plain_ce(st):
    c, x, w, t = st["case"], st["x"].detach().float(), st["w"].detach().float(), st["t"]
    keep = t != -100
    at = t.clamp(min=0)
    logits = x @ w.t()
    top = logits.amax(-1, keepdim=True)
    e = (logits - top).exp()
    z = e.sum(-1, keepdim=True)
    rows = (top + z.log())[:, 0] - logits.gather(1, at[:, None])[:, 0]
    rows = torch.where(keep, rows, torch.zeros_like(rows))
    count = keep.sum()
    loss = rows if c["reduction"] == "none" else rows.double().sum().float()
    if c["reduction"] == "mean":
        loss = loss / count
    if not c["train"]:
        return [loss]
    g = st["grad"] * torch.ones_like(rows)
    if c["reduction"] == "mean":
        g = g / count
    g = torch.where(keep, g, torch.zeros_like(g))[:, None]
    d = e.div_(z)
    d.scatter_add_(1, at[:, None], torch.full_like(g, -1.0))
    d = d.mul_(g)
    return [loss, (d @ w).to(st["x"].dtype), (d.t() @ x).to(st["w"].dtype)]


def _plain_ffn(st):
    c, x, w = st["case"], st["x"].detach().float(), st["w"].detach().float()
    gate, up = (x @ w.t()).split(c["f"], dim=-1)
    sig = 1.0 / (1.0 + (-gate).exp())
    h = (gate * sig * up).to(st["x"].dtype)
    if not c["train"]:
        return [h]
    dh = st["dh"].float()
    d = torch.cat([dh * up * sig * (1.0 + gate * (1.0 - sig)), dh * gate * sig], dim=-1)
    return [h, (d @ w).to(st["x"].dtype), (d.t() @ x).to(st["w"].dtype)]


def _plain_rope(st):
    c, dt = st["case"], st["qkv"].dtype
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    x = st["qkv"].detach().unflatten(-1, (hq + 2 * hkv, d)).float()
    q, k, v = x.split([hq, hkv, hkv], dim=-2)
    pos = st["pos"].long() if c["packed"] else torch.arange(c["s"], device=x.device)
    cos, sin = (t[pos][:, None, :] for t in (st["cos"], st["sin"]))
    wq, wk = (None if t is None else t.detach().float() for t in (st["wq"], st["wk"]))
    qn, kn = (_rms(q, wq), _rms(k, wk)) if c["norm"] else (q, k)
    out = [_rotate(qn, cos, sin).to(dt), _rotate(kn, cos, sin).to(dt), v.to(dt)]
    if not c["train"]:
        return out
    gq, gk = (_rotate_grad(t.float(), cos, sin) for t in st["grads"][:2])
    if c["norm"]:
        (gq, dwq), (gk, dwk) = _rms_grad(q, wq, gq), _rms_grad(k, wk, gk)
        out += [t.double().sum(0).to(dt) for t in (dwq, dwk)]
    return out + [torch.cat([gq, gk, st["grads"][2].float()], dim=-2).flatten(-2).to(dt)]


def _plain_clip(st):
    c = st["case"]
    squares = [g.float().square().sum(dtype=torch.float64) for g in st["grads"]]
    norm = torch.stack(squares).sum().sqrt().float()
    if c["norm_only"]:
        return [norm]
    coef = (st["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    [o.copy_(g.float() * coef) for g, o in zip(st["grads"], st["out"])]
    return [norm, st["flat"]]


def run(state):
    st, c = state, state["case"]
    if not own:
        return {"linear_ce": _plain_ce, "gated_ffn": _plain_ffn, "qk_rope": _plain_rope,
                "grad_clip": _plain_clip}[c["op"]](st)
    linear_ce, gated_ffn, qk_norm_rope, clip_grad_norm, grad_norm = _framework()
    if c["op"] == "linear_ce":
        loss = linear_ce(st["x"], st["w"], st["t"], reduction=c["reduction"])
        if not c["train"]:
            return [loss]
        return [loss.detach(), *torch.autograd.grad(loss, (st["x"], st["w"]), st["grad"])]
    if c["op"] == "gated_ffn":
        h = gated_ffn(st["x"], st["w"])
        if not c["train"]:
            return [h]
        return [h.detach(), *torch.autograd.grad(h, (st["x"], st["w"]), st["dh"])]
    if c["op"] == "qk_rope":
        out = qk_norm_rope(st["qkv"], c["hq"], c["hkv"], st["cos"], st["sin"], q_weight=st["wq"],
                           k_weight=st["wk"], eps=_EPS, positions=st["pos"])
        if not c["train"]:
            return list(out)
        if c["norm"]:
            dqkv, dwq, dwk = torch.autograd.grad(out, (st["qkv"], st["wq"], st["wk"]), st["grads"])
            return [t.detach() for t in out] + [dwq, dwk, dqkv]
        return [t.detach() for t in out] + list(torch.autograd.grad(out, (st["qkv"],),
                                                                    st["grads"]))
    if c["norm_only"]:
        return [grad_norm(st["grads"])]
    return [clip_grad_norm(st["grads"], st["max_norm"], out=st["out"]), st["flat"]]


# --------------------------------------------------------------------------------------- work
def work(case):
    c = case
    es = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "linear_ce":
        n, h, v = c["n"], c["h"], c["v"]
        inputs, flops = es * h * (n + v) + 8 * n, 2.0 * n * h * v
        outputs = 4 * (n if c["reduction"] == "none" else 1)
        return dict(bytes=inputs + outputs + (es * h * (n + v) if c["train"] else 0),
                    flops=flops * (3 if c["train"] else 1))
    if c["op"] == "gated_ffn":
        n, h, f = c["n"], c["h"], c["f"]
        fwd = es * (n * h + 2 * f * h + n * f)
        return dict(bytes=fwd + (es * (n * f + n * h + 2 * f * h) if c["train"] else 0),
                    flops=4.0 * n * h * f * (3 if c["train"] else 1))
    if c["op"] == "qk_rope":
        # queries and keys in and out (values stay where they are); backward: the gradients of
        # all three in, the gradient of qkv out, and with the norm the queries and keys again
        rows = c["b"] * c["s"]
        qk, full = rows * (c["hq"] + c["hkv"]) * c["d"], rows * (c["hq"] + 2 * c["hkv"]) * c["d"]
        table = 8 * c["d"] * min(rows, c["s"] if not c["packed"] else 4096)
        total = 2 * qk * es + table
        if c["train"]:
            total += 2 * full * es + table + (qk * es if c["norm"] else 0)
        return dict(bytes=total, flops=(12.0 if c["train"] else 6.0) * qk)
    n = sum(math.prod(s) for s in _grad_shapes(c))
    return dict(bytes=n * es + (0 if c["norm_only"] else 4 * n),
                flops=(2.0 if c["norm_only"] else 3.0) * n)


# --------------------------------------------------------------------------------------- exact
def exact(case, seed):
    st, c = prepare(case, seed), case
    if c["op"] == "linear_ce":
        x, w, t = st["x"].detach().double(), st["w"].detach().double(), st["t"]
        keep = t != -100
        logits = torch.einsum("nh,vh->nv", x, w)
        lse = torch.logsumexp(logits, 1)
        rows = torch.zeros(c["n"], dtype=torch.float64, device=x.device)
        idx = keep.nonzero()[:, 0]
        rows[idx] = lse[idx] - logits[idx, t[idx]]
        scale = 1.0 / len(idx) if c["reduction"] == "mean" else 1.0
        loss = rows if c["reduction"] == "none" else rows.sum() * scale
        if not c["train"]:
            return [loss]
        d = torch.exp(logits.sub_(lse[:, None]))
        d[idx, t[idx]] -= 1.0
        d *= (keep * scale * st["grad"].double())[:, None]
        return [loss, torch.einsum("nv,vh->nh", d, w), torch.einsum("nv,nh->vh", d, x)]
    if c["op"] == "gated_ffn":
        x, w = st["x"].detach().double(), st["w"].detach().double()
        wg, wu = w[: c["f"]], w[c["f"]:]
        a, b = torch.einsum("nh,fh->nf", x, wg), torch.einsum("nh,fh->nf", x, wu)
        s = torch.sigmoid(a)
        out = [a * s * b]
        if c["train"]:
            dh = st["dh"].double()
            da, db = dh * b * (s + a * s * torch.sigmoid(-a)), dh * a * s
            out += [torch.einsum("nf,fh->nh", da, wg) + torch.einsum("nf,fh->nh", db, wu),
                    torch.cat([torch.einsum("nf,nh->fh", da, x),
                               torch.einsum("nf,nh->fh", db, x)])]
        return out
    if c["op"] == "qk_rope":
        lead = st["qkv"].shape[:-1]
        d, half, rows = c["d"], c["d"] // 2, c["b"] * c["s"]
        x = st["qkv"].detach().double().reshape(rows, c["hq"] + 2 * c["hkv"], d)
        at = (st["pos"].long() if c["packed"] else
              torch.arange(c["s"], device=x.device).repeat(c["b"]))
        co, si = (t.double()[at, None, :half] for t in (st["cos"], st["sin"]))
        first, last, dw, dx = 0, 0, [], []
        out = []
        for i, (n, w) in enumerate(((c["hq"], st["wq"]), (c["hkv"], st["wk"]))):
            first, last = last, last + n
            y = x[:, first:last]
            inv = 1.0
            wd = torch.ones(d, dtype=torch.float64, device=x.device)
            if c["norm"]:
                inv = 1.0 / torch.sqrt((y * y).sum(-1, keepdim=True) / d + _EPS)
                wd = w.detach().double()
            z = y * inv * wd
            z = torch.complex(z[..., :half], z[..., half:]) * torch.complex(co, si)
            out.append(torch.cat([z.real, z.imag], -1).reshape(*lead, n, d))
            if c["train"]:
                gr = st["grads"][i].double().reshape(rows, n, d)
                gz = torch.complex(gr[..., :half], gr[..., half:]) * torch.complex(co, -si)
                gy = torch.cat([gz.real, gz.imag], -1)
                if c["norm"]:
                    dw.append(torch.einsum("rnd,rnd->d", gy, y * inv))
                    gy = gy * wd
                    gy = inv * gy - y * inv ** 3 * (gy * y).sum(-1, keepdim=True) / d
                dx.append(gy)
        out.append(x[:, last:].reshape(*lead, c["hkv"], d))
        if c["train"]:
            dx.append(st["grads"][2].double().reshape(rows, c["hkv"], d))
            out += dw + [torch.cat(dx, 1).reshape(*lead, -1)]
        return out
    norm = math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in st["grads"]))
    if c["norm_only"]:
        return [norm]
    scale = min(1.0, st["max_norm"] / (norm + 1e-6))
    return [norm, torch.cat([g.double().reshape(-1) * scale for g in st["grads"]])]
