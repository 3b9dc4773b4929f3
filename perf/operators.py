"""The operators at the two ends of a training step and between them, as cases to time and compare.

``logprobs``  log probabilities of given tokens, with entropy and top alternatives, and their gradient
              (``ops.nn.token_logprobs``)
``embed``     embedding lookup with scaling, its gradient by sorted tokens (``ops.nn.scaled_embedding``)
``pack``      activations held in 8 bits and brought back (``ops.nn.pack_activation``)
``swiglu``    SwiGLU that keeps its input in 8 bits for its backward pass (``ops.nn.swiglu(..., save_bits=8)``)

``run`` computes the plain form with elementary torch operations, or, where ``own`` is true, calls the framework.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORE = -100


def _logprobs(rows, vocab, dtype, **kw):
    case = {"op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "pad": 64, "top_k": 0,
            "entropy": False, "temperature": 1.0, "ignored": 0.0, "masked": 0.0, "grad": True}
    case.update(kw)
    return case


def _embed(tokens, vocab, width, dtype, **kw):
    case = {"op": "embed", "tokens": tokens, "vocab": vocab, "width": width, "dtype": dtype, "scale": 1.0,
            "zipf": False, "padded": 0.0, "grad": "dense"}
    case.update(kw)
    return case


def listed():
    return [
        # one position of a decoded sequence: its token, the uncertainty and five alternatives
        dict(_logprobs(1, 50257, "bf16", top_k=5, entropy=True, grad=False), name="logprobs one position"),
        # a batch of sequences scored, twenty alternatives each, the vocabulary of the 8B shape
        dict(_logprobs(96, 128256, "bf16", top_k=20, entropy=True, grad=False), name="logprobs score batch"),
        # a policy gradient's step over eight sequences of GPT-2 small; a tenth are prompt positions
        dict(_logprobs(8192, 50257, "fp16", ignored=0.1), name="logprobs train 8x1024"),
        # the same with entropy bonus and alternatives to distil from, the vocabulary of the 8B shape
        dict(_logprobs(2048, 128256, "bf16", top_k=8, entropy=True), name="logprobs train entropy top8"),
        # an fp32 model, odd rows without padding, a third of the vocabulary masked away, a temperature
        dict(_logprobs(1021, 32003, "fp32", pad=1, entropy=True, temperature=0.7, masked=0.33), name="logprobs fp32 masked odd"),
        # the next tokens of a few sequences
        dict(_embed(32, 128256, 4096, "bf16", scale=64.0, grad="none"), name="embed 32 tokens"),
        # GPT-2 small's micro-batch, natural token frequencies, the gradient added into the engine's buffer
        dict(_embed(16384, 50257, 768, "fp16", zipf=True, grad="arena"), name="embed arena 16x1024"),
        # the 8B shape's micro-batch, uniform tokens as in its benchmark, a gradient of its own
        dict(_embed(4096, 128256, 4096, "bf16", scale=64.0), name="embed dense 1x4096"),
        # the residual stream that a checkpointed GPT-2 XL block keeps
        {"op": "pack", "rows": 4096, "width": 1600, "dtype": "bf16", "name": "pack 4x1024x1600"},
        # an fp32 model's, odd in both directions
        {"op": "pack", "rows": 999, "width": 1111, "dtype": "fp32", "name": "pack fp32 odd"},
        # the feed-forward of the 8B shape
        {"op": "swiglu", "rows": 4096, "width": 14336, "dtype": "bf16", "name": "swiglu 4096x14336"},
        # a small model's, with a width that fills neither a vector nor a block
        {"op": "swiglu", "rows": 517, "width": 1365, "dtype": "fp16", "name": "swiglu 517x1365"},
    ]


def _size(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "embed", "embed", "pack", "swiglu"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "logprobs":
        vocab = _size(rng, 1000, 131072)
        rows = _size(rng, 1, min(8192, (1 << 27) // vocab))
        return _logprobs(rows, vocab, dtype, pad=rng.choice([1, 64]), top_k=rng.choice([0, 0, 1, 5, 20, 32]),
                         entropy=rng.random() < 0.5, temperature=rng.choice([1.0, 1.0, 0.7, 1.3]),
                         ignored=rng.choice([0.0, 0.0, 0.25]), masked=rng.choice([0.0, 0.0, 0.5]),
                         grad=rng.random() < 0.6)
    if op == "embed":
        vocab = _size(rng, 500, 131072)
        width = _size(rng, 64, 4096)
        if rng.random() < 0.7:
            width = -(-width // 8) * 8
        tokens = _size(rng, 1, min(65536, (1 << 25) // width))
        grad = rng.choice(["none", "dense", "arena"])
        if dtype == "fp32" and vocab * width > 1 << 27:
            dtype = "bf16"
        return _embed(tokens, vocab, width, dtype, scale=rng.choice([1.0, 0.5, round(math.sqrt(width), 3)]),
                      zipf=rng.random() < 0.5, padded=rng.choice([0.0, 0.0, 0.3]), grad=grad)
    width = _size(rng, 48, 14336)
    if rng.random() < 0.6:
        width = -(-width // 32) * 32
    rows = _size(rng, 1, min(16384, (1 << (24 if dtype == "fp32" else 25)) // width))
    return {"op": op, "rows": rows, "width": width, "dtype": dtype}


# ---------------------------------------------------------------- inputs
def _tokens(g, n, vocab, zipf):
    if not zipf:
        return torch.randint(0, vocab, (n,), device="cuda", generator=g)
    # frequency falls as 1 / rank, ranks dealt out over the ids
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    rank = ((vocab + 1.0) ** u).long().clamp_(1, vocab) - 1
    return torch.randperm(vocab, device="cuda", generator=g)[rank]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = dict(case)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=g).mul_(std)

    if case["op"] == "logprobs":
        m, v = case["rows"], case["vocab"]
        ld = -(-v // case["pad"]) * case["pad"]
        x = torch.empty(m, ld, device="cuda", dtype=dt)[:, :v]
        for r in range(0, m, 1024):  # logits of a trained model: a few tokens stand out
            x[r:r + 1024] = normal(min(1024, m - r), v, std=2.0)
        tok = torch.randint(0, v, (m,), device="cuda", generator=g)
        if case["masked"]:
            x.masked_fill_(torch.rand(v, device="cuda", generator=g) < case["masked"], float("-inf"))
            x[torch.arange(m, device="cuda"), tok] = normal(m).to(dt)
        tok[torch.rand(m, device="cuda", generator=g) < case["ignored"]] = IGNORE
        unit = (65536.0 if dt == torch.float16 else 1.0) / m  # a mean's gradient, under fp16's loss scale
        st.update(x=x.requires_grad_(case["grad"]), tok=tok, g_lp=normal(m, std=unit))
        st["g_h"] = normal(m, std=unit) if case["entropy"] else None
        st["g_top"] = normal(m, case["top_k"], std=unit) if case["top_k"] else None
    elif case["op"] == "embed":
        n, v, c = case["tokens"], case["vocab"], case["width"]
        w = torch.nn.Parameter(normal(v, c, std=0.02).to(dt))
        idx = _tokens(g, n, v, case["zipf"])
        st["padding_idx"] = v // 2 if case["padded"] else None
        if case["padded"]:
            idx[torch.rand(n, device="cuda", generator=g) < case["padded"]] = v // 2
        st.update(w=w, idx=idx)
        if case["grad"] == "none":
            w.requires_grad_(False)
        else:
            st["dout"] = normal(n, c, std=0.1).to(dt)
        if case["grad"] == "arena":  # what the parameter's gradient holds already (a tied head's part)
            st["before"] = normal(v, c, std=0.1).to(dt)
            w.grad = torch.empty_like(w)
    else:
        m, f = case["rows"], case["width"]
        cols = f if case["op"] == "pack" else 2 * f
        x = normal(m, cols)
        x.mul_(torch.exp(normal(cols, std=0.5)))  # channels of different size, as activations have them
        st["x"] = x.to(dt).requires_grad_(case["op"] == "swiglu")
        if case["op"] == "swiglu":
            st["dh"] = normal(m, f, std=0.1).to(dt)
    return st


# ----------------------------------------------------------- plain forms
def _plain_logprobs(st):
    x, tok, T = st["x"].detach().float() / st["temperature"], st["tok"], st["temperature"]
    k, m, v = st["top_k"], *st["x"].shape
    keep = tok != IGNORE
    at = tok.clamp(min=0)[:, None]
    e = torch.exp(x - x.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    logp = x - x.amax(-1, keepdim=True) - torch.log(e.sum(-1, keepdim=True))
    out = {"logprobs": torch.where(keep, logp.gather(1, at)[:, 0], 0.0)}
    h = None
    finite = logp.clamp(min=-1e30)  # a masked place has probability zero and adds nothing
    if st["entropy"]:
        h = -(p * finite).sum(-1, keepdim=True)
        out["entropy"] = torch.where(keep, h[:, 0], 0.0)
    top = None
    if k:
        # values in their order as whole numbers, the lower index first among equals
        bits = (st["x"].detach().float() + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        top = torch.topk(order * (1 << 20) - torch.arange(v, device=x.device), k, dim=-1).indices
        out["top_logprobs"] = torch.where(keep[:, None], logp.gather(1, top), 0.0)
        out["top_tokens"] = torch.where(keep[:, None], top, -1)
    if st["grad"]:
        d = torch.zeros_like(p).scatter_(1, at, st["g_lp"][:, None])
        total = st["g_lp"][:, None]
        if k:
            d.scatter_add_(1, top, st["g_top"])
            total = total + st["g_top"].sum(-1, keepdim=True)
        d -= p * total
        if st["entropy"]:
            d -= st["g_h"][:, None] * p * (finite + h)
        out["dlogits"] = torch.where(keep[:, None], d / T, 0.0).to(st["x"].dtype)
    return out


def _plain_embed(st):
    w, idx = st["w"].detach(), st["idx"]
    out = {"out": (w[idx].float() * st["scale"]).to(w.dtype)}
    if st["grad"] != "none":
        rows = st["dout"].float() * st["scale"]
        if st["padding_idx"] is not None:
            rows = torch.where((idx == st["padding_idx"])[:, None], 0.0, rows)
        acc = torch.zeros(w.shape, device=w.device).index_add_(0, idx, rows)
        if st["grad"] == "arena":
            acc += st["before"].float()
        out["dweight"] = acc.to(w.dtype)
    return out


def _plain_restored(x):
    """``x`` by blocks of 32 of its last axis as whole numbers in [-127, 127] times a power of two."""
    n = x.shape[-1]
    b = torch.nn.functional.pad(x.float(), (0, -n % 32)).unflatten(-1, (-1, 32))
    field = (b.abs().amax(-1, keepdim=True).view(torch.int32) >> 23).sub(6).clamp(min=0)
    scale = torch.exp2((field - 127).double())
    q = torch.round(b.double() / scale).clamp(-127, 127)
    return (q * scale).float().flatten(-2)[..., :n]


def _plain_swiglu(st):
    x, f = st["x"].detach(), st["width"]
    g, u = x[:, :f].float(), x[:, f:].float()
    out = {"h": (g / (1 + torch.exp(-g)) * u).to(x.dtype)}
    g, u = _plain_restored(x[:, :f]), _plain_restored(x[:, f:])
    d, s = st["dh"].float(), 1 / (1 + torch.exp(-g))
    out["dx"] = torch.cat([d * u * s * (1 + g * (1 - s)), d * g * s], -1).to(x.dtype)
    return out


# ------------------------------------------------------ the framework's
def _own_logprobs(ops, st):
    r = ops.token_logprobs(st["x"], st["tok"], temperature=st["temperature"], entropy=st["entropy"],
                           top_k=st["top_k"], ignore_index=IGNORE)
    out = {"logprobs": r.logprobs}
    ys, gs = [r.logprobs], [st["g_lp"]]
    if st["entropy"]:
        out["entropy"] = r.entropy
        ys.append(r.entropy)
        gs.append(st["g_h"])
    if st["top_k"]:
        out["top_logprobs"], out["top_tokens"] = r.top_logprobs, r.top_tokens
        ys.append(r.top_logprobs)
        gs.append(st["g_top"])
    if st["grad"]:
        (out["dlogits"],) = torch.autograd.grad(ys, st["x"], gs)
    return out


def _own_embed(ops, st):
    w = st["w"]
    y = ops.scaled_embedding(st["idx"], w, scale=st["scale"], padding_idx=st["padding_idx"])
    out = {"out": y}
    if st["grad"] == "dense":
        (out["dweight"],) = torch.autograd.grad(y, w, st["dout"])
    elif st["grad"] == "arena":
        w.grad.copy_(st["before"])
        y.backward(st["dout"])
        out["dweight"] = w.grad
    return out


def _own_swiglu(ops, st):
    h = ops.swiglu(st["x"], save_bits=8)
    (dx,) = torch.autograd.grad(h, st["x"], st["dh"])
    return {"h": h, "dx": dx}


def run(state):
    op = state["op"]
    if own:
        from minispeed_b200.ops import nn as ops

        if op == "logprobs":
            return _own_logprobs(ops, state)
        if op == "embed":
            return _own_embed(ops, state)
        if op == "swiglu":
            return _own_swiglu(ops, state)
        return {"restored": ops.pack_activation(state["x"]).unpack()}
    if op == "logprobs":
        return _plain_logprobs(state)
    if op == "embed":
        return _plain_embed(state)
    if op == "swiglu":
        return _plain_swiglu(state)
    return {"restored": _plain_restored(state["x"]).to(state["x"].dtype)}


# ----------------------------------------------------------------- work
def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "logprobs":
        m, v, k = case["rows"], case["vocab"], case["top_k"]
        read = (1 - case["ignored"]) * m * v
        small = m * (8 + 4 + 4 * case["entropy"] + 12 * k)
        if case["grad"]:
            small += m * (4 + 4 * case["entropy"] + 4 * k)
        return {"bytes": read * e + small + case["grad"] * m * v * e,
                "flops": read * (6 + 2 * case["entropy"] + case["grad"] * (4 + 3 * case["entropy"]))}
    if case["op"] == "embed":
        n, v, c = case["tokens"], case["vocab"], case["width"]
        share = np.diff(np.log(np.arange(1, v + 2)) / np.log(v + 1)) if case["zipf"] else np.full(v, 1 / v)
        distinct = float((1 - (1 - share) ** max(1, n * (1 - case["padded"]))).sum())
        moved = distinct * c * e + n * c * e + 8 * n
        if case["grad"] != "none":
            moved += n * (1 - case["padded"]) * c * e + v * c * e
            if case["grad"] == "arena":
                moved += v * c * e
        return {"bytes": moved, "flops": n * c * (1 + (case["grad"] != "none"))}
    m, f = case["rows"], case["width"]
    if case["op"] == "pack":
        return {"bytes": 2 * m * f * e, "flops": 4 * m * f}
    return {"bytes": m * f * e * (2 + 1 + 1 + 2), "flops": 30 * m * f}


# ---------------------------------------------------------------- exact
def _exact_logprobs(case, st):
    x, tok, k, T = st["x"].detach(), st["tok"], case["top_k"], case["temperature"]
    parts = []
    for r in range(0, x.shape[0], 256):
        z, t = x[r:r + 256].double() / T, tok[r:r + 256]
        on = (t != IGNORE).double()[:, None]
        lse = torch.logsumexp(z, -1, keepdim=True)
        lp = z - lse
        pr = lp.exp()
        # -p log p, zero where p is
        plogp = torch.special.entr(pr)
        h = plogp.sum(-1, keepdim=True)
        pos = t.clamp(min=0)[:, None]
        o = {"logprobs": (lp.gather(1, pos) * on)[:, 0]}
        if case["entropy"]:
            o["entropy"] = (h * on)[:, 0]
        if k:
            o["top_logprobs"] = lp.topk(k, -1).values * on
        if case["grad"]:
            hot = torch.zeros_like(pr).scatter_(1, pos, 1.0)
            d = st["g_lp"][r:r + 256, None].double() * (hot - pr)
            if case["entropy"]:
                d += st["g_h"][r:r + 256, None].double() * (plogp - pr * h)
            if k:
                # which positions the alternatives are: by value, then by index
                _, byval = torch.sort(x[r:r + 256].double(), dim=-1, descending=True, stable=True)
                gt = st["g_top"][r:r + 256].double()
                d = d.scatter_add(1, byval[:, :k], gt) - pr * gt.sum(-1, keepdim=True)
            o["dlogits"] = d / T * on
        parts.append(o)
    out = {key: torch.cat([p[key] for p in parts]) for key in parts[0]}
    if k:
        out["top_tokens"] = None
    return out


def _exact_restored(x):
    n = x.shape[-1]
    b = torch.cat([x.double(), x.new_zeros(x.shape[0], -n % 32, dtype=torch.float64)], -1).view(x.shape[0], -1, 32)
    biggest = b.abs().max(-1, keepdim=True).values
    power = (torch.frexp(biggest).exponent - 7).clamp(min=-127)
    power = torch.where(biggest == 0, -127, power)
    steps = torch.ldexp(b, -power)
    return torch.ldexp(steps.round().clamp(-127, 127), power).view(x.shape[0], -1)[:, :n]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(case, st)
    if case["op"] == "embed":
        w, idx = st["w"].detach(), st["idx"]
        out = {"out": w.index_select(0, idx).double() * case["scale"]}
        if case["grad"] != "none":
            live = idx != (-1 if st["padding_idx"] is None else st["padding_idx"])
            base = st["before"].double() if case["grad"] == "arena" else torch.zeros(w.shape, dtype=torch.float64, device=w.device)
            out["dweight"] = base.index_add(0, idx[live], st["dout"][live].double(), alpha=case["scale"])
        return out
    if case["op"] == "pack":
        return {"restored": _exact_restored(st["x"])}
    f = case["width"]
    x, dh = st["x"].detach(), st["dh"].double()
    silu = lambda t: t * torch.sigmoid(t)  # noqa: E731
    h = silu(x[:, :f].double()) * x[:, f:].double()
    g, u = _exact_restored(x[:, :f]), _exact_restored(x[:, f:])
    s = torch.sigmoid(g)
    return {"h": h, "dx": torch.cat([dh * u * (s + g * s * (1 - s)), dh * silu(g)], -1)}
