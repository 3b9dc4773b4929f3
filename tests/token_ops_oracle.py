"""64-bit definitions of the token and 8-bit operators, and bounds on what fp32
arithmetic may be off by, for their tests."""

import math

import torch

U32 = 2.0 ** -24   # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def logprobs(x, tok, T=1.0, k=0, ignore=-100, g_lp=None, g_ent=None, g_top=None):
    """dict of lp, ent, top_lp, top, dx and, as lp_tol, ent_tol and dx_tol, how
    far an fp32 computation rounded to x's type may be from them."""
    dtype, V = x.dtype, x.shape[-1]
    x64 = x.detach().double().reshape(-1, V)
    tok = tok.reshape(-1)
    keep = tok != ignore
    at = torch.where(keep, tok, 0)[:, None]
    empty = (x64 == -math.inf).all(-1, keepdim=True)
    z = torch.where(empty, 0.0, x64 / T)
    logp = torch.log_softmax(z, -1)
    p = torch.where(empty, 0.0, logp.exp())
    live = torch.where(logp == -math.inf, 0.0, logp)
    H = -(p * live).sum(-1, keepdim=True)
    on = keep[:, None]

    def settle(v, of_empty):
        return torch.where(on, torch.where(empty, of_empty, v), 0.0)

    top = torch.sort(x64, dim=-1, descending=True, stable=True).indices[:, :k]
    out = {"lp": settle(logp.gather(1, at), -math.inf)[:, 0], "ent": settle(H, 0.0)[:, 0],
           "top_lp": settle(logp.gather(1, top), -math.inf), "top": torch.where(on, top, -1)}
    # the exponent of every term that counts is off by a few half steps of |x| / T
    # (of nothing where that reaches 2^24 ln 2 and differences are taken first), a sum
    # of V terms over at least 256 running sums by V / 256 half steps, exp2 by four
    counts = (logp > -100) & (x64.abs() / T < 2 ** 24 * math.log(2))
    size = torch.where(counts, x64.abs(), 0.0).amax(-1, keepdim=True) / T
    tol = U32 * (V / 256 + 64 + 16 * size)
    # a log probability is itself rounded, and a difference of logits before it
    far = lambda v: tol + 8 * U32 * torch.where(torch.isfinite(v), v.abs(), 0.0)  # noqa: E731
    out["lp_tol"] = far(out["lp"][:, None])[:, 0]
    out["top_tol"] = far(out["top_lp"])
    out["ent_tol"] = tol[:, 0] * (2 + math.log2(V + 1))

    def rows(g, n):
        return torch.zeros(x64.shape[0], n, dtype=torch.float64, device=x.device) if g is None \
            else g.detach().double().reshape(-1, n)

    gl, ge, gt = rows(g_lp, 1), rows(g_ent, 1), rows(g_top, k)
    hot = torch.zeros_like(p).scatter_(1, at, gl).scatter_add_(1, top, gt)
    G = gl + gt.sum(-1, keepdim=True)
    dx = (hot - p * G - ge * p * (live + H)) / T
    out["dx"] = torch.where(on & ~empty, dx, 0.0)
    scale = (hot.abs() + p * (gl.abs() + gt.abs().sum(-1, keepdim=True)
                              + ge.abs() * (live.abs() + H + 1))) / T
    # exp2 of an exponent under -126 is 0
    flushed = 2.0 ** -126 * (gl.abs() + gt.abs().sum(-1, keepdim=True) + ge.abs() * (130 + H)) / T
    out["dx_tol"] = (half_step(dtype) * out["dx"].abs() + 4 * (tol + k * U32) * scale + flushed
                     + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps)
    return out


def embedding_grad(dout, idx, V, scale=1.0, padding=None, before=None):
    """(gradient, how far fp32 sums rounded once to dout's type may be off)."""
    C = dout.shape[-1]
    d, i = dout.double().reshape(-1, C), idx.reshape(-1)
    live = (i >= 0) & (i < V)
    if padding is not None:
        live &= i != padding
    d, i = d[live], i[live]
    zero = torch.zeros(V, C, dtype=torch.float64, device=d.device)
    grad = zero.index_add(0, i, d) * scale
    size = zero.index_add(0, i, d.abs()) * abs(scale)
    count = torch.zeros(V, dtype=torch.float64, device=d.device).index_add_(
        0, i, torch.ones_like(i, dtype=torch.float64))
    if before is not None:
        grad, size = grad + before.double(), size + before.double().abs()
    # of n terms summed one after another n - 1 sums round, and the scale and the addition
    tol = (U32 * (count[:, None] + 2) * size + half_step(dout.dtype) * grad.abs()
           + torch.finfo(dout.dtype).smallest_normal * torch.finfo(dout.dtype).eps)
    return grad, tol


def restored(x):
    """x by blocks of 32 of its last axis in 8 bits and back, in 64 bits."""
    D = x.shape[-1]
    b = torch.nn.functional.pad(x.double(), (0, -D % 32)).unflatten(-1, (-1, 32))
    big = b.abs().amax(-1, keepdim=True)
    power = torch.where(big == 0, -127, (torch.frexp(big).exponent - 7).clamp(min=-127))
    v = torch.ldexp(torch.ldexp(b, -power).round().clamp(-127, 127), power)
    return torch.where(torch.isfinite(big), v, math.nan).flatten(-2)[..., :D]


def swiglu(gu, dh):
    """h, its tolerance, and the gradient at the restored input with its."""
    F = gu.shape[-1] // 2
    g, u = gu.double()[..., :F], gu.double()[..., F:]
    h = g * torch.sigmoid(g) * u
    tiny = torch.finfo(gu.dtype).smallest_normal * torch.finfo(gu.dtype).eps
    half = half_step(gu.dtype)
    # exp of g: half steps of |g|; the quotient and products a few more
    h_tol = half * h.abs() + U32 * (16 + 4 * g.abs()) * h.abs() + tiny
    g, u, d = restored(gu[..., :F]), restored(gu[..., F:]), dh.double()
    s = torch.sigmoid(g)
    dx = torch.cat([d * u * (s + g * s * (1 - s)), d * g * s], -1)
    size = torch.cat([(d * u).abs() * s * (1 + g.abs()), (d * g).abs() * s], -1)
    soft = U32 * (32 + 4 * torch.cat([g, g], -1).abs())
    return h, h_tol, dx, half * dx.abs() + soft * size + tiny


def close(got, want, tol):
    """got is want within tol, with the same infinities and NaN; what is beyond
    the largest value of got's type is an infinity there."""
    beyond = want.abs() > torch.finfo(got.dtype).max
    want = torch.where(beyond, want.sign() * math.inf, want)
    got = got.detach().double().reshape(want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    off = ((got - want).abs() - tol.expand_as(want))[fine]
    assert not off.numel() or float(off.max()) <= 0, \
        f"off by {float((got - want)[fine].abs().max()):.3g}, {int((off > 0).sum())} places"
