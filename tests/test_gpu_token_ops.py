"""The kernels of token log probabilities, scaled embedding and 8-bit
activations against their 64-bit definitions."""

import math

import pytest
import torch
import torch.autograd.forward_ad as fwad
import torch.nn as nn

import token_ops_oracle as oracle
from minispeed_b200.activation_checkpointing import checkpoint
from minispeed_b200.ops import _ext
from minispeed_b200.ops import nn as ops

pytestmark = pytest.mark.gpu
DT = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, seed=0, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=_gen(seed)) * std).to(dtype)


# ------------------------------------------------- token log probabilities
def _check_logprobs(x, tok, T=1.0, k=0, entropy=True, seed=5):
    x = x.detach().requires_grad_()
    n = tok.numel()
    r = ops.token_logprobs(x, tok, temperature=T, entropy=entropy, top_k=k)
    gs = [_randn(n, seed=seed), _randn(n, seed=seed + 1) if entropy else None,
          _randn(n, k, seed=seed + 2) if k else None]
    want = oracle.logprobs(x, tok, T, k, g_lp=gs[0], g_ent=gs[1], g_top=gs[2])
    oracle.close(r.logprobs, want["lp"], want["lp_tol"])
    ys, gy = [r.logprobs], [gs[0].view(tok.shape)]
    if entropy:
        oracle.close(r.entropy, want["ent"], want["ent_tol"])
        ys.append(r.entropy)
        gy.append(gs[1].view(tok.shape))
    else:
        assert r.entropy is None
    if k:
        assert torch.equal(r.top_tokens.view(n, k), want["top"])
        oracle.close(r.top_logprobs, want["top_lp"], want["top_tol"])
        ys.append(r.top_logprobs)
        gy.append(gs[2].view(*tok.shape, k))
    else:
        assert r.top_tokens is None and r.top_logprobs is None
    (dx,) = torch.autograd.grad(ys, x, gy)
    assert dx.shape == x.shape and dx.dtype == x.dtype
    oracle.close(dx, want["dx"], want["dx_tol"])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (1, 2, 2), (3, 7, 5), (2, 33, 32), (5, 1000, 20),
                                      (1, 50257, 5), (2, 131071, 32), (37, 4097, 1),
                                      (300, 2050, 8), (700, 515, 0)])
def test_logprobs_sizes(dtype, rows, V, k):
    x = _randn(rows, V, seed=V, dtype=dtype, std=3.0)
    tok = torch.randint(0, V, (rows,), device="cuda", generator=_gen(1))
    tok[rows // 2] = -100 if rows > 2 else tok[rows // 2]
    _check_logprobs(x, tok, T=0.7 if rows % 2 else 1.0, k=k)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("V", [50, 3001])
def test_logprobs_masks(dtype, V):
    x = _randn(10, V, seed=2, dtype=dtype, std=3.0)
    x[1, torch.rand(V, device="cuda", generator=_gen(3)) < 0.9] = -math.inf
    x[2] = -math.inf                                   # empty
    x[3] = torch.finfo(dtype).min                      # uniform, at the lowest value
    x[4] = 1.25                                        # ties everywhere
    x[5, 3:] = -math.inf                               # fewer tokens than alternatives
    x[6, V // 2:] = torch.finfo(dtype).min             # a mask of the lowest value
    x[7, : V // 2] = -math.inf
    x[7, V // 2:] = torch.finfo(dtype).min
    x[8] = 0.0
    x[8, ::2] = -0.0                                   # equal to +0: lower index first
    x[9] = torch.arange(V, device="cuda").to(dtype) / V  # ascending, with ties in 16 bits
    tok = torch.tensor([0, 1, 2, 3, 4, 1, 7, V - 1, 9, 0], device="cuda")
    for k in (0, 1, 20):
        _check_logprobs(x, tok, T=0.7, k=k)
    _check_logprobs(x.flip(0), tok.flip(0), T=1.0, k=32, entropy=False)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("V", [50, 3001, 40003])
def test_logprobs_masks_of_any_size(dtype, V):
    """Masks from -1e4 to -1e38, and offsets of as much above zero: in part of a
    row, for whole threads, in all of it."""
    sizes = [v for v in (1e4, 1e6, 3e7, 1e9, 1e10, 1e20, 1e30, 1e38)
             if v < torch.finfo(dtype).max]
    x = _randn(4 * len(sizes), V, seed=2, dtype=dtype, std=3.0)
    for i, v in enumerate(sizes):
        x[4 * i, torch.rand(V, device="cuda", generator=_gen(i)) < 0.95] = -v
        x[4 * i + 1, 8:] = -v
        x[4 * i + 2] = -v
        x[4 * i + 2, 3] = -2 * v if 2 * v < torch.finfo(dtype).max else -v
        x[4 * i + 3, V // 2:] = v
    tok = torch.arange(4 * len(sizes), device="cuda") % 7
    _check_logprobs(x, tok, k=3)
    _check_logprobs(x, tok, T=0.3, k=0)


def test_logprobs_temperatures_at_their_limits():
    x = _randn(3, 300, seed=2)
    tok = x.argmax(-1)
    r = ops.token_logprobs(x, tok, temperature=1e-30, entropy=True, top_k=2)
    assert r.logprobs.tolist() == [0, 0, 0] and r.entropy.tolist() == [0, 0, 0]
    assert bool((r.top_logprobs[:, 1] < -1e25).all())
    r = ops.token_logprobs(x, tok, temperature=1e30, entropy=True)
    assert r.logprobs.tolist() == pytest.approx([-math.log(300)] * 3, rel=1e-6)
    assert r.entropy.tolist() == pytest.approx([math.log(300)] * 3, rel=1e-6)


@pytest.mark.parametrize("dtype", DT)
def test_logprobs_masks_of_rows_shared_by_blocks(dtype):
    """Few long rows, each read by several blocks: everything that counts in one
    block's part, in the last values behind its vectors, or nowhere."""
    V = 40003
    x = _randn(7, V, seed=2, dtype=dtype, std=3.0)
    x[0, : V - 3] = -math.inf
    x[1, 5:] = torch.finfo(dtype).min
    x[2] = torch.finfo(dtype).min
    x[3] = -math.inf
    x[4] = 2.0
    x[5, 20000:20600] = 9.0                            # more ties than are kept
    x[6] = -torch.arange(V, device="cuda").to(dtype) / V
    tok = torch.tensor([V - 1, 0, 7, 8, 9, 20100, -100], device="cuda")
    for k in (0, 32):
        _check_logprobs(x, tok, T=1.0, k=k)
    _check_logprobs(x[:, 1:], (tok - 1).clamp(min=0), T=0.7, k=3)


def test_logprobs_alternatives_in_sorted_and_crowded_rows():
    """Rows whose best values lie beside one another, in one thread's vectors, or
    all within a narrow band: the threshold lets many through."""
    V = 128 * 256
    x = torch.zeros(6, V, device="cuda")
    x[0] = torch.arange(V, device="cuda") / V
    x[1] = -torch.arange(V, device="cuda") / V
    one = (torch.arange(V, device="cuda") // 4 % 256 == 77).float()   # thread 77's fp32 vectors
    x[2] = one * (1 + torch.arange(V, device="cuda") / V)
    x[3] = torch.where(one > 0, 1.0, -torch.rand(V, device="cuda", generator=_gen(1)))
    x[4] = torch.rand(V, device="cuda", generator=_gen(2)).half().float()
    x[5] = (torch.arange(V, device="cuda") % 7).float()
    tok = torch.arange(6, device="cuda")
    for dtype in DT:
        for k in (1, 8, 32):
            _check_logprobs(x.to(dtype), tok, k=k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logprobs_largest_values(dtype):
    """Finite logits at both ends of the type."""
    big = torch.finfo(dtype).max
    x = torch.full((4, 77), -big, device="cuda", dtype=dtype)
    x[0, 5] = big
    x[1, 5:8] = big
    x[2] = big
    x[3, 9] = 0.0
    _check_logprobs(x, torch.tensor([5, 6, 70, 9], device="cuda"), k=4)
    _check_logprobs(x, torch.tensor([6, 0, 0, 0], device="cuda"), T=2.5, k=7)


@pytest.mark.parametrize("copies", [1, 40])
@pytest.mark.parametrize("sign", [-1, 1])
def test_logprobs_at_the_limit_of_wide_rows(sign, copies):
    """Logits on both sides of 2^24 / log2(e), where differences are taken before
    the scaling: parts of rows shared by blocks (few rows) or read by one block
    (many).  A shift changes no probability, so the values are those of the
    small distances from the limit, which fp32 holds exactly here."""
    V, limit = 40003, sign * 11629080
    half = torch.arange(V, device="cuda") < V // 2
    step = [torch.randint(0, 20, (V,), device="cuda", generator=_gen(i)) for i in range(4)]
    rows = [torch.where(half, 0, 1), torch.where(half, 1, 0), torch.where(half, -step[0], 3 - step[1]),
            -step[2], 1 - step[3], torch.where(half, -1, 0)]
    rows[3][-1] = 2          # alone above the limit, behind the vectors of the last block
    off = torch.stack(rows).repeat(copies, 1).float()
    n = len(off)
    x = (off + limit).requires_grad_()
    assert torch.equal(x.detach() - limit, off)
    tok = torch.arange(n, device="cuda") * 7919 % V
    r = ops.token_logprobs(x, tok, entropy=True, top_k=3)
    gs = [_randn(n, seed=1), _randn(n, seed=2), _randn(n, 3, seed=3)]
    want = oracle.logprobs(off, tok, k=3, g_lp=gs[0], g_ent=gs[1], g_top=gs[2])
    oracle.close(r.logprobs, want["lp"], want["lp_tol"])
    oracle.close(r.entropy, want["ent"], want["ent_tol"])
    assert torch.equal(r.top_tokens, want["top"])
    oracle.close(r.top_logprobs, want["top_lp"], want["top_tol"])
    (dx,) = torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], x, gs)
    oracle.close(dx, want["dx"], want["dx_tol"])


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("V", [77, 5000])
def test_logprobs_not_finite(bad, V):
    x = _randn(4, V, seed=3)
    x[1, V // 3] = bad
    x[2] = bad
    x.requires_grad_()
    tok = torch.tensor([1, 2, 3, 4], device="cuda")
    r = ops.token_logprobs(x, tok, entropy=True, top_k=3)
    (dx,) = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), x)
    for v in (r.logprobs, r.entropy, r.top_logprobs[:, 0], dx[:, 0], dx[:, V - 1]):
        assert torch.isnan(v).tolist() == [False, True, True, False]
    assert bool(((r.top_tokens >= 0) & (r.top_tokens < V)).all())


def test_logprobs_layouts():
    base = _randn(6, 40, 2100, seed=4, dtype=torch.bfloat16)
    tok = torch.randint(0, 1000, (6, 40), device="cuda", generator=_gen(2))
    for x, t in [(base[..., 37:1037], tok), (base[:, ::3, :1000], tok[:, ::3]),
                 (base[..., ::2][..., :1000], tok), (base.transpose(0, 1)[..., 1:1001], tok.T),
                 (base[0, 0, 5:1005], tok[0, 0]), (base[:1, :1, 3:1003].expand(1, 5, 1000), tok[:1, :5])]:
        _check_logprobs(x, t, k=3)


def test_logprobs_padded_rows_give_a_padded_gradient():
    h = _randn(64, 128, dtype=torch.bfloat16).requires_grad_()
    w = _randn(1003, 128, seed=1, dtype=torch.bfloat16)
    logits = ops.linear(h, w, pad_out=64)
    assert logits.stride(0) == 1024
    seen = []
    logits.register_hook(lambda g: seen.append(g.stride()))
    ops.token_logprobs(logits, torch.arange(64, device="cuda")).logprobs.sum().backward()
    assert seen == [(1024, 1)] and torch.isfinite(h.grad).all()


def test_logprobs_token_outside_the_vocabulary():
    x = _randn(3, 100, seed=1).requires_grad_()
    r = ops.token_logprobs(x, torch.tensor([100, 5, -7], device="cuda"))
    assert torch.isnan(r.logprobs).tolist() == [True, False, True]
    (dx,) = torch.autograd.grad(r.logprobs.sum(), x)
    assert not dx[0].any() and not dx[2].any() and dx[1].any()
    _ext.bounds_status(reset=True)   # the debug build has recorded them


def test_logprobs_of_nothing():
    x = torch.zeros(0, 50, device="cuda", requires_grad=True)
    r = ops.token_logprobs(x, torch.zeros(0, dtype=torch.int64, device="cuda"), entropy=True, top_k=4)
    assert r.logprobs.shape == (0,) and r.top_tokens.shape == (0, 4)
    r.logprobs.sum().backward()
    assert x.grad.shape == (0, 50)


def test_logprobs_parts_of_the_gradient():
    """Only some results used: the others add nothing; none: no gradient."""
    x = _randn(9, 700, seed=7).requires_grad_()
    tok = torch.randint(0, 700, (9,), device="cuda", generator=_gen(4))
    r = ops.token_logprobs(x, tok, entropy=True, top_k=4)
    for y, kw in ((r.logprobs, "g_lp"), (r.entropy, "g_ent"), (r.top_logprobs, "g_top")):
        (dx,) = torch.autograd.grad(y.sum(), x, retain_graph=True)   # an expanded gradient
        want = oracle.logprobs(x, tok, 1.0, 4, **{kw: torch.ones_like(y)})
        oracle.close(dx, want["dx"], want["dx_tol"])


def test_logprobs_same_bits_each_time_and_logits_untouched():
    x = _randn(500, 3001, seed=8, dtype=torch.bfloat16)
    kept = x.clone()
    x.requires_grad_()
    tok = torch.randint(0, 3001, (500,), device="cuda", generator=_gen(4))
    got = []
    for _ in range(2):
        r = ops.token_logprobs(x, tok, entropy=True, top_k=9)
        (dx,) = torch.autograd.grad([r.logprobs, r.entropy], x,
                                    [torch.ones(500, device="cuda")] * 2)
        got.append((*r, dx))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert torch.equal(x.detach(), kept)


def test_logprobs_beyond_32_bit_offsets():
    """The last rows of logits of more than 2^32 values."""
    M, V = 33000, 131072
    x = torch.zeros(M, V, device="cuda", dtype=torch.bfloat16)
    x[-3:] = _randn(3, V, dtype=torch.bfloat16, std=3.0)
    x.requires_grad_()
    tok = torch.full((M,), -100, device="cuda")
    tok[-3:] = torch.tensor([5, V - 1, 77], device="cuda")
    tok[0] = 3
    r = ops.token_logprobs(x, tok, entropy=True, top_k=4)
    g = _randn(M)
    (dx,) = torch.autograd.grad(r.logprobs, x, g)
    want = oracle.logprobs(x[-3:], tok[-3:], k=4, g_lp=g[-3:])
    oracle.close(r.logprobs[-3:], want["lp"], want["lp_tol"])
    oracle.close(r.entropy[-3:], want["ent"], want["ent_tol"])
    assert torch.equal(r.top_tokens[-3:], want["top"])
    oracle.close(dx[-3:], want["dx"], want["dx_tol"])
    assert not dx[1:100].any() and not dx[-100:-3].any()
    assert float(r.logprobs[0].detach()) == pytest.approx(-math.log(V), rel=1e-5)


# ------------------------------------------------------- scaled embedding
def _check_embedding(idx, V, C, dtype, scale=1.0, padding=None, offset=0):
    w = _randn(V * C + offset, seed=C, dtype=dtype)[offset:].view(V, C).requires_grad_()
    y = ops.scaled_embedding(idx, w, scale, padding)
    assert y.shape == (*idx.shape, C)
    assert torch.equal(y, (w.detach()[idx].float() * scale).to(dtype))
    d = _randn(idx.numel() * C + offset, seed=C + 1, dtype=dtype)[offset:].view(*idx.shape, C)
    (dw,) = torch.autograd.grad(y, w, d)
    want, tol = oracle.embedding_grad(d, idx, V, scale, padding)
    oracle.close(dw, want, tol)
    return dw


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,V,C", [(1, 1, 8), (1, 50257, 768), (31, 2, 1), (32, 3, 257), (33, 511, 72),
                                   (64, 512, 255), (65, 513, 256), (1025, 70000, 264),
                                   (4099, 300, 40), (9000, 262144, 16), (20000, 97, 24)])
def test_embedding_sizes(dtype, n, V, C):
    idx = torch.randint(0, V, (n,), device="cuda", generator=_gen(n))
    _check_embedding(idx, V, C, dtype, scale=0.625)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [100, 2048, 10007])
def test_embedding_long_runs(dtype, n):
    """One token everywhere, two halves, a run ending at a chunk's edge, padding."""
    one = torch.full((n,), 3, dtype=torch.int64, device="cuda")
    _check_embedding(one, 5, 136, dtype)
    half = one.clone()
    half[: n // 2] = 1
    _check_embedding(half, 5, 136, dtype, scale=3.0)
    edge = torch.arange(n, device="cuda") // 32 % 4
    _check_embedding(edge, 4, 33, dtype)
    mixed = torch.where(torch.rand(n, device="cuda", generator=_gen(n)) < 0.6, one,
                        torch.randint(0, 900, (n,), device="cuda", generator=_gen(n)))
    dw = _check_embedding(mixed, 900, 136, dtype, padding=3)
    assert not dw[3].any()
    assert not _check_embedding(one, 5, 136, dtype, padding=3).any()


@pytest.mark.parametrize("n", [1, 8, 33, 5000])
@pytest.mark.parametrize("V,C", [(3, 8), (70000, 8), (1025, 264), (9, 50000), (4000, 33)])
def test_embedding_clears_the_other_rows(n, V, C):
    """Every row of a new gradient is written, whatever was in its memory."""
    idx = torch.randint(0, V, (n,), device="cuda", generator=_gen(n)) // 2 * 2 % V
    for _ in range(2):
        junk = torch.full((V, C), math.nan, device="cuda", dtype=torch.bfloat16)
        del junk
        _check_embedding(idx, V, C, torch.bfloat16)


def test_embedding_beyond_32_bit_offsets():
    V, C = 1100000, 4096
    w = torch.zeros(V, C, device="cuda", dtype=torch.bfloat16)
    w[-2:] = _randn(2, C, dtype=torch.bfloat16)
    w.requires_grad_()
    idx = torch.tensor([V - 1, 0, V - 2, V - 1], device="cuda")
    y = ops.scaled_embedding(idx, w, 2.0)
    assert torch.equal(y, (w.detach()[idx].float() * 2).bfloat16())
    d = _randn(4, C, seed=3, dtype=torch.bfloat16)
    (dw,) = torch.autograd.grad(y, w, d)
    assert torch.equal(dw[-1], ((d[0].float() + d[3].float()) * 2).bfloat16())
    assert torch.equal(dw[-2], (d[2].float() * 2).bfloat16())
    assert torch.equal(dw[0], (d[1].float() * 2).bfloat16())
    assert not dw[1:-2].any()


def test_embedding_lookup_of_more_than_2_31_values():
    """Places behind the end, in the last turn of a launch, whose number times eight
    passes 31 bits, read nothing."""
    n, V, C = 600001, 37, 4096
    w = _randn(V, C, dtype=torch.bfloat16)
    idx = torch.randint(0, V, (n,), device="cuda", generator=_gen(1))
    y = ops.scaled_embedding(idx, w, 2.0)
    want = (w.float() * 2).bfloat16()
    for i in range(0, n, 100000):
        assert torch.equal(y[i:i + 100000], want[idx[i:i + 100000]])


@pytest.mark.parametrize("offset", [1, 4])
def test_embedding_unaligned(offset):
    idx = torch.randint(0, 40, (3, 50), device="cuda", generator=_gen(1))
    _check_embedding(idx, 40, 64, torch.bfloat16, offset=offset)


def test_embedding_indices_of_any_shape():
    idx = torch.randint(0, 40, (4, 5, 6), device="cuda", generator=_gen(1))
    _check_embedding(idx.transpose(0, 2), 40, 16, torch.float16)
    _check_embedding(idx[0, 0, 0], 40, 16, torch.float16)
    _check_embedding(idx[:, :0], 40, 16, torch.float16)


def test_embedding_tokens_outside_the_table():
    w = _randn(60, 16, dtype=torch.float16)
    table = w[:50].requires_grad_()
    idx = torch.tensor([49, 50, -1, 3, 1 << 40, 49], device="cuda")
    y = ops.scaled_embedding(idx, table, 2.0)
    assert not y[1].any() and not y[2].any() and not y[4].any()
    (dw,) = torch.autograd.grad(y, table, torch.ones_like(y))
    want = torch.zeros(50, 16, device="cuda", dtype=torch.float16)
    want[49], want[3] = 4.0, 2.0
    assert torch.equal(dw, want)
    _ext.bounds_status(reset=True)   # the debug build has recorded them


@pytest.mark.parametrize("dtype", DT)
def test_embedding_adds_into_the_bound_gradient(dtype):
    p = nn.Parameter(_randn(700, 40, dtype=dtype))
    before = _randn(700, 40, seed=1, dtype=dtype)
    p.grad = before.clone()
    kept = p.grad
    idx = torch.randint(0, 200, (3000,), device="cuda", generator=_gen(2))
    d = _randn(3000, 40, seed=2, dtype=dtype)
    ops.scaled_embedding(idx, p, 0.5, padding_idx=-690).backward(d)
    assert p.grad is kept
    want, tol = oracle.embedding_grad(d, idx, 700, 0.5, 10, before)
    oracle.close(p.grad, want, tol)
    assert torch.equal(p.grad[200:], before[200:])


def test_embedding_gradient_is_the_difference():
    """As on the CPU: exactly, in whole numbers."""
    w = torch.randint(-8, 9, (900, 136), device="cuda", generator=_gen(1)).float().requires_grad_()
    step = torch.randint(-8, 9, (900, 136), device="cuda", generator=_gen(2)).float()
    idx = torch.randint(0, 900, (3000,), device="cuda", generator=_gen(3)) ** 2 // 900
    d = torch.randint(-8, 9, (3000, 136), device="cuda", generator=_gen(4)).float()
    y = ops.scaled_embedding(idx, w, 3.0)
    (dw,) = torch.autograd.grad(y, w, d)
    change = ops.scaled_embedding(idx, w.detach() + step, 3.0) - y.detach()
    assert float((change.double() * d.double()).sum()) == float((dw.double() * step.double()).sum())


def test_embedding_backward_twice_from_one_lookup():
    w = _randn(50, 264).requires_grad_()
    y = ops.scaled_embedding(torch.randint(0, 50, (500,), device="cuda", generator=_gen(3)), w)
    d = _randn(500, 264, seed=1)
    (a,) = torch.autograd.grad(y, w, d, retain_graph=True)
    (b,) = torch.autograd.grad(y, w, d)
    assert torch.equal(a, b)


def test_embedding_gradient_is_the_same_each_time():
    idx = torch.randint(0, 50, (30000,), device="cuda", generator=_gen(2)) ** 2 // 50
    w = _randn(50, 264, dtype=torch.bfloat16).requires_grad_()
    d = _randn(30000, 264, seed=1, dtype=torch.bfloat16)
    grads = [torch.autograd.grad(ops.scaled_embedding(idx, w), w, d)[0] for _ in range(3)]
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])


def test_one_column_with_any_stride():
    """An axis of one element may have any stride."""
    x = _randn(1, 9)
    for v in (x.T, x.T.unsqueeze(1), _randn(9, 5)[:, 2:3], x[:, :1].expand(9, 1)):
        assert torch.equal(ops.pack_activation(v).unpack(), oracle.restored(v).float())
        _check_logprobs(v, torch.zeros(v.shape[:-1], dtype=torch.int64, device="cuda"), k=1)
    w = x.T.detach().requires_grad_()
    y = ops.scaled_embedding(torch.tensor([3, 3, 8], device="cuda"), w, 2.0)
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert dw[:, 0].tolist() == [0, 0, 0, 4, 0, 0, 0, 0, 2]


# ------------------------------------------------------ 8-bit activations
def _awkward(dtype, rows, D, seed=0):
    x = _randn(rows, D, seed=seed) * torch.exp(_randn(rows, 1, seed=seed + 1) * 4)
    x = x.to(dtype)
    x[0] = 0
    x[1, 0] = torch.finfo(dtype).max
    x[2] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    x[3] = torch.arange(D, device="cuda").to(dtype) / 2
    x[4, -1] = torch.finfo(dtype).min
    return x


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,D", [(5, 1), (6, 7), (6, 8), (7, 31), (9, 32), (300, 40), (11, 257),
                                    (64, 1600), (1000, 1111)])
def test_pack_is_exact(dtype, rows, D):
    x = _awkward(dtype, rows, D)
    p = ops.pack_activation(x)
    y = p.unpack()
    assert y.dtype == dtype
    torch.testing.assert_close(y, oracle.restored(x).to(dtype), rtol=0, atol=0, equal_nan=True)
    # the same bytes as on the CPU, but for the codes of blocks that come back as NaN
    q = ops.pack_activation(x.cpu())
    assert torch.equal(p.scales.cpu(), q.scales)
    live = (q.scales != 255).repeat_interleave(32, -1)
    assert torch.equal(p.codes.cpu()[live], q.codes[live])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("D", [64, 70])
def test_pack_not_finite(dtype, D):
    x = torch.ones(3, D, device="cuda", dtype=dtype)
    x[0, 5], x[1, 40], x[2, D - 1] = math.inf, math.nan, -math.inf
    want = oracle.restored(x).to(dtype)
    y = ops.pack_activation(x).unpack()
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(y.nan_to_num(9.0), want.nan_to_num(9.0))


def test_pack_layouts():
    base = _randn(5, 6, 200, dtype=torch.bfloat16)
    for x in (base.transpose(0, 1), base[..., 3:], base[..., :64], base[..., 8:72], base[:, ::2],
              base[..., ::2], base[0, 0], base[:, :0], base[:1].expand(4, 6, 200)):
        assert torch.equal(ops.pack_activation(x).unpack(), oracle.restored(x).to(x.dtype))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,F", [(6, 1), (7, 31), (6, 32), (9, 48), (40, 1000), (300, 45),
                                    (17, 14336)])
def test_swiglu_8bit(dtype, rows, F):
    x = _awkward(dtype, rows, 2 * F, seed=F).clamp(-30, 30).requires_grad_()
    dh = _randn(rows, F, seed=3, dtype=dtype)
    h = ops.swiglu(x, save_bits=8)
    with torch.no_grad():
        assert torch.equal(h, ops.swiglu(x, save_bits=8))   # nothing saved, the same result
    hw, ht, dw, dt = oracle.swiglu(x.detach(), dh)
    oracle.close(h, hw, ht)
    (dx,) = torch.autograd.grad(h, x, dh)
    oracle.close(dx, dw, dt)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("F", [64, 45])
def test_swiglu_8bit_output_is_the_plain_one(dtype, F):
    """Gates from the one end of the exponential's range to the other.  In fp32
    bit for bit the output of SwiGLU without 8-bit saves; in 16 bits rounded
    from within 2^-16 of it, so at most one step apart (and a subnormal one)."""
    g = torch.linspace(-100, 100, 300 * F, device="cuda").view(300, F).to(dtype)
    u = _randn(300, F, seed=1, dtype=dtype)
    even = torch.cat([nn.functional.pad(v, (0, -F % 8)) for v in (g, u)], -1)   # its widths
    want = ops.swiglu(even)[:, :F]
    h = ops.swiglu(torch.cat([g, u], -1), save_bits=8)
    if dtype == torch.float32:
        assert torch.equal(h, want)
    else:
        f = torch.finfo(dtype)
        off = (h.double() - want.double()).abs()
        assert bool((off <= f.eps * want.double().abs() + f.smallest_normal * f.eps).all())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("F", [64, 45])
def test_swiglu_8bit_gates_far_from_zero(dtype, F):
    """Down to the last gates whose sigmoid fp32 holds in full, with small
    upstream gradients."""
    x = torch.cat([torch.linspace(-87, 87, 300 * F, device="cuda").view(300, F),
                   40 * _randn(300, F)], -1).to(dtype).requires_grad_()
    dh = _randn(300, F, seed=3, dtype=dtype, std=2.0 ** -12)
    h = ops.swiglu(x, save_bits=8)
    hw, ht, dw, dt = oracle.swiglu(x.detach(), dh)
    oracle.close(h, hw, ht)
    (dx,) = torch.autograd.grad(h, x, dh)
    oracle.close(dx, dw, dt)


def test_swiglu_8bit_layouts_and_nothing():
    base = _randn(4, 6, 300, dtype=torch.bfloat16).requires_grad_()
    for x in (base[..., 1:129], base.transpose(0, 1), base[:, ::2, :64], base[:, :0]):
        h = ops.swiglu(x, save_bits=8)
        dh = _randn(*h.shape, seed=3, dtype=h.dtype)
        hw, ht, dw, dt = oracle.swiglu(x.detach(), dh)
        oracle.close(h, hw, ht)
        (dx,) = torch.autograd.grad(h, x, dh)
        oracle.close(dx, dw, dt)
    h = ops.swiglu(base, save_bits=8)
    (dx,) = torch.autograd.grad(h, base, torch.ones((), device="cuda", dtype=h.dtype).expand_as(h))
    oracle.close(dx, *oracle.swiglu(base.detach(), torch.ones_like(h))[2:])


def test_swiglu_8bit_holds_half_the_memory():
    x = _randn(2048, 4096, dtype=torch.bfloat16).requires_grad_()
    y = x * 1
    torch.cuda.synchronize()
    h = ops.swiglu(y, save_bits=8)
    kept = torch.cuda.memory_allocated()
    del y
    freed = kept - torch.cuda.memory_allocated()
    assert freed == 2048 * 4096 * 2     # the exact input is not kept
    h.sum().backward()


def test_checkpoint_8bit_cuda_random_state_and_gradient():
    leaf = _randn(64, 96, dtype=torch.bfloat16).requires_grad_()
    torch.manual_seed(5)
    y = checkpoint(lambda t: nn.functional.dropout(t * t, 0.5), leaf * 1, save_bits=8)
    torch.rand(100, device="cuda")
    y.backward(torch.ones_like(y))
    xr = oracle.restored(leaf.detach()).to(leaf.dtype)
    want = torch.where(y == 0, torch.zeros_like(xr), 4 * xr)   # 2 x / (1 - 0.5)
    assert torch.equal(leaf.grad, want)


# ------------------------------------------- derivatives without a kernel
_DIFFERENTIABLE = {
    "token_logprobs": (lambda x: ops.token_logprobs(x, torch.arange(3, device="cuda")).logprobs, (3, 8)),
    "scaled_embedding": (lambda w: ops.scaled_embedding(torch.tensor([1, 2, 1], device="cuda"), w), (5, 8)),
    "swiglu": (lambda x: ops.swiglu(x, save_bits=8), (3, 16)),
}


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("op", _DIFFERENTIABLE)
def test_forward_mode_is_refused(op, grad):
    call, shape = _DIFFERENTIABLE[op]
    x = _randn(*shape).requires_grad_(grad)
    with fwad.dual_level():
        dual = fwad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)
        assert torch.equal(call(fwad.unpack_dual(dual).primal), call(x))


@pytest.mark.parametrize("op", _DIFFERENTIABLE)
def test_second_derivatives_are_refused(op):
    call, shape = _DIFFERENTIABLE[op]
    x = _randn(*shape).requires_grad_()
    y = call(x * 1)
    (dx,) = torch.autograd.grad(y.sum(), x, retain_graph=True)
    with pytest.raises(NotImplementedError, match="create_graph"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], dx)


def test_second_derivatives_leave_the_bound_gradient_alone():
    p = nn.Parameter(_randn(5, 8))
    p.grad = _randn(5, 8, seed=1)
    before = p.grad.clone()
    y = ops.scaled_embedding(torch.tensor([1, 2, 1], device="cuda"), p)
    with pytest.raises(NotImplementedError, match="create_graph"):
        y.sum().backward(create_graph=True)
    assert torch.equal(p.grad, before)


# ----------------------------------------------- streams, graphs, together
def _all_of_them(st):
    h = ops.scaled_embedding(st["idx"], st["table"], 3.0, padding_idx=0)
    h = checkpoint(lambda t: ops.swiglu(ops.linear(t, st["w"]), save_bits=8), h, save_bits=8)
    logits = ops.linear(h, st["head"], pad_out=64)
    r = ops.token_logprobs(logits, st["next"], entropy=True, top_k=3, temperature=0.9)
    loss = -(r.logprobs.mean() + 0.01 * r.entropy.mean() + 0.1 * r.top_logprobs.sum(-1).mean())
    grads = torch.autograd.grad(loss, [st["table"], st["w"], st["head"]])
    return [loss.detach(), *grads]


def _all_state(seed):
    bf = torch.bfloat16
    return {"idx": torch.randint(0, 211, (4, 60), device="cuda", generator=_gen(seed)),
            "next": torch.randint(0, 211, (4, 60), device="cuda", generator=_gen(seed + 1)),
            "table": _randn(211, 64, seed=1, dtype=bf).requires_grad_(),
            "w": _randn(256, 64, seed=2, dtype=bf, std=0.1).requires_grad_(),
            "head": _randn(211, 128, seed=3, dtype=bf, std=0.1).requires_grad_()}


def test_together_on_a_stream_of_their_own():
    want = _all_of_them(_all_state(9))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        st = _all_state(9)
        got = _all_of_them(st)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_together_on_two_streams_at_once():
    want = [_all_of_them(_all_state(9)), _all_of_them(_all_state(29))]
    states = [_all_state(9), _all_state(29)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for st, stream in zip(states, streams):
            with torch.cuda.stream(stream):
                got.append(_all_of_them(st))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % 2]))


def test_together_captured_twice_and_replayed_with_new_tokens():
    states = [_all_state(9), _all_state(19)]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for st in states:
            _all_of_them(st)          # the GEMM plans are tuned outside a capture
    side.synchronize()
    for st in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(_all_of_them(st))
        graphs.append(g)
    fresh = _all_state(33)
    for st in states:
        st["idx"].copy_(fresh["idx"])
        st["next"].copy_(fresh["next"])
    for g in graphs:
        g.replay()
    for g in reversed(graphs):
        g.replay()
    torch.cuda.synchronize()
    want = _all_of_them(fresh)
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    for g in graphs:
        g.reset()


def test_together_against_plain_operations():
    """One pass of the four against the same in PyTorch operations on the
    packed values, in fp32 from the same bf16 weights: every bf16 result is
    rounded once (half a step, 2^-8 of the value), five of them on the way."""
    st = _all_state(9)
    got = _all_of_them(st)
    ps = {k: v.detach().float().requires_grad_() if v.is_floating_point() else v
          for k, v in st.items()}

    def plain(round_):
        h = ps["table"][ps["idx"]] * 3.0
        h = round_(h)
        hr = h + (oracle.restored(h.detach()).float() - h).detach()   # the recompute's input
        def mlp(t):
            return round_(t @ ps["w"].T)
        exact, packed = mlp(h), mlp(hr)
        pr = packed + (torch.cat([oracle.restored(p) for p in packed.detach().chunk(2, -1)], -1).float()
                       - packed).detach()
        act = lambda v: nn.functional.silu(v[..., :128]) * v[..., 128:]  # noqa: E731
        a = act(pr) + (act(exact) - act(pr)).detach()
        logits = round_(round_(a) @ ps["head"].T)
        logp = torch.log_softmax(logits / 0.9, -1)
        lp = logp.gather(-1, ps["next"][..., None])[..., 0]
        ent = -(logp.exp() * logp).sum(-1)
        top = torch.sort(logits.detach(), dim=-1, descending=True, stable=True).indices[..., :3]
        return -(lp.mean() + 0.01 * ent.mean() + 0.1 * logp.gather(-1, top).sum(-1).mean())

    class Round(torch.autograd.Function):
        @staticmethod
        def forward(ctx, v):
            return v.bfloat16().float()

        @staticmethod
        def backward(ctx, g):
            return g.bfloat16().float()

    loss = plain(Round.apply)
    grads = list(torch.autograd.grad(loss, [ps["table"], ps["w"], ps["head"]]))
    grads[0][0] = 0        # the padding token
    assert float(got[0]) == pytest.approx(float(loss.detach()), rel=5 * 2 ** -8)
    for a, b in zip(got[1:], grads):
        assert float((a.float() - b).norm() / b.norm()) < 5 * 2 ** -8


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_a_device_that_is_not_the_current_one():
    want = _all_of_them(_all_state(9))
    st = {k: v.detach().to("cuda:1").requires_grad_(v.requires_grad) for k, v in _all_state(9).items()}
    got = _all_of_them(st)
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(got, want))


# -------------------------------------------------------- through the engine
def _engine(graph, dtype="bf16"):
    import minispeed_b200 as ms
    from minispeed_b200.models import Llama, LlamaConfig, init_llama_

    torch.manual_seed(0)
    m = init_llama_(Llama(LlamaConfig(vocab_size=517, block_size=128, n_layer=2, n_head=4,
                                      n_kv_head=2, n_embd=256, ffn_hidden=360, embed_scale=16.0,
                                      activation_checkpointing=True, checkpoint_bits=8,
                                      swiglu_save_bits=8)))
    return ms.initialize(model=m, config={
        "train_micro_batch_size_per_gpu": 2, "gradient_accumulation_steps": 2, "dtype": dtype,
        "gradient_clipping": 1.0, "zero_optimization": {"stage": 2},
        "optimizer": {"type": "AdamW", "params": {"lr": 1e-3}},
        "b200": {"cuda_graph": graph}})


def _batches():
    return [torch.randint(0, 517, (2, 128), device="cuda", generator=_gen(i)) for i in range(6)]


def test_engine_on_log_probabilities_and_in_a_graph():
    """Losses of eager micro-steps, of graph replays of the same batches, and
    from the token log probabilities: the same mean, whose bf16 results on the
    way are rounded in the same places (attention adds its query gradients in
    an order of its own, so weights differ by a few roundings after a step)."""
    runs = []
    for graph in (False, True):
        e = _engine(graph)
        runs.append([float(e.train_batch(x, targets=torch.roll(x, -1, 1))) for x in _batches()])
    e = _engine(False)
    own = []
    for x in _batches():
        r = e(x, targets=torch.roll(x, -1, 1), logprobs={})
        loss = -r.logprobs.mean()
        e.backward(loss)
        e.step()
        own.append(float(loss.detach()))
    for other in (runs[1], own):
        assert other == pytest.approx(runs[0], rel=2 ** -8)
    assert all(math.isfinite(v) for v in own)


# ------------------------------------------------ the bounds-checked build
def test_debug_build_records_tokens_out_of_range():
    """Both builds skip the access; the debug build records it.  The access
    would have stayed in allocated memory: the tables are parts of larger ones."""
    import importlib

    try:
        dbg = importlib.import_module("minispeed_b200._C_debug")
    except ImportError:
        pytest.skip("debug build not built (MSB_DEBUG_BUILD=1 python setup.py build_ext --inplace)")
    _ext.bounds_status(reset=True, mod=dbg)
    V = 100
    w = _randn(V + 8, 64, dtype=torch.float16)[:V]
    idx = torch.tensor([3, V + 2, 5, 7], device="cuda")
    for sort in (False, True):
        out, _ = dbg.scaled_embedding_fwd(idx, w, 1.0, -1, sort)
        rec = {r["unit"]: r for r in _ext.bounds_status(reset=True, mod=dbg)}["embedding"]
        assert (rec["count"], rec["site"], rec["index"], rec["limit"]) == (1, 1, V + 2, V)
        assert not out[1].any() and torch.equal(out[2], w[5])
    x = _randn(4, 128)[:, :V]
    tok = torch.tensor([3, V + 2, -100, 7], device="cuda")
    lp = dbg.logprob_fwd(x, tok, 1.0, True, 3, -100)[0]
    rec = {r["unit"]: r for r in _ext.bounds_status(reset=True, mod=dbg)}["logprob"]
    assert (rec["count"], rec["site"], rec["index"], rec["limit"]) == (1, 8, V + 2, V)
    assert torch.isnan(lp).tolist() == [False, True, False, False]
