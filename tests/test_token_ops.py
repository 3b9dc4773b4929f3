"""Token log probabilities, scaled embedding, 8-bit activations: refusals, and
the CPU definitions against 64 bits."""

import math

import pytest
import torch
import torch.nn as nn

import token_ops_oracle as oracle
import minispeed_b200 as ms
from minispeed_b200.activation_checkpointing import checkpoint
from minispeed_b200.models import GPT, GPTConfig, Llama, LlamaConfig, init_gpt2_, init_llama_
from minispeed_b200.ops import nn as ops

DT = [torch.float32, torch.float16, torch.bfloat16]


# --------------------------------------------------------------- refusals
@pytest.mark.parametrize("kw,err", [
    (dict(logits=torch.zeros(2, 5, dtype=torch.float64)), TypeError),
    (dict(tokens=torch.zeros(2, dtype=torch.int32)), TypeError),
    (dict(tokens=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(logits=torch.zeros(2, 0)), ValueError),
    (dict(top_k=-1), ValueError),
    (dict(top_k=6), ValueError),
    (dict(logits=torch.zeros(2, 99), top_k=33), ValueError),
    (dict(temperature=0.0), ValueError),
    (dict(temperature=math.nan), ValueError),
    (dict(temperature=-1.0), ValueError),
    (dict(temperature=1e-31), ValueError),
    (dict(temperature=math.inf), ValueError),
    (dict(tokens=torch.tensor([1, 5])), IndexError),
    (dict(tokens=torch.tensor([1, -1])), IndexError),
])
def test_token_logprobs_refuses(kw, err):
    call = {"logits": torch.zeros(2, 5), "tokens": torch.zeros(2, dtype=torch.int64), **kw}
    with pytest.raises(err):
        ops.token_logprobs(call.pop("logits"), call.pop("tokens"), **call)


@pytest.mark.parametrize("idx,kw,err", [
    (torch.zeros(2, dtype=torch.int32), {}, TypeError),
    (torch.zeros(2, dtype=torch.int64), dict(weight=torch.zeros(3, 4, dtype=torch.float64)), TypeError),
    (torch.zeros(2, dtype=torch.int64), dict(weight=torch.zeros(3)), ValueError),
    (torch.zeros(2, dtype=torch.int64), dict(weight=torch.zeros(0, 4)), ValueError),
    (torch.zeros(2, dtype=torch.int64), dict(scale=math.inf), ValueError),
    (torch.zeros(2, dtype=torch.int64), dict(scale=math.nan), ValueError),
    (torch.zeros(2, dtype=torch.int64), dict(scale=1e39), ValueError),
    (torch.zeros(2, dtype=torch.int64), dict(padding_idx=3), ValueError),
    (torch.tensor([0, 3]), {}, IndexError),
    (torch.tensor([0, -1]), {}, IndexError),
])
def test_scaled_embedding_refuses(idx, kw, err):
    call = {"weight": torch.zeros(3, 4), **kw}
    with pytest.raises(err):
        ops.scaled_embedding(idx, **call)


def test_8bit_refusals():
    with pytest.raises(TypeError):
        ops.pack_activation(torch.zeros(3, dtype=torch.float64))
    with pytest.raises(ValueError):
        ops.pack_activation(torch.tensor(1.0))
    with pytest.raises(ValueError, match="save_bits"):
        ops.swiglu(torch.zeros(2, 8), save_bits=4)
    with pytest.raises(ValueError):
        ops.swiglu(torch.zeros(2, 7), save_bits=8)
    with pytest.raises(TypeError):
        ops.swiglu(torch.zeros(2, 8, dtype=torch.float64), save_bits=8)
    with pytest.raises(ValueError, match="save_bits"):
        checkpoint(torch.sin, torch.zeros(3), save_bits=16)
    with pytest.raises(ValueError, match="use_reentrant"):
        checkpoint(torch.sin, torch.zeros(3), save_bits=8, use_reentrant=True)


def test_backward_kernels_are_reached_through_their_forward_only():
    """They trust the sizes and lists that their forward left: a list of tokens
    read for a table of another size would name rows that are not there."""
    from minispeed_b200.ops import _ext

    mod = _ext.load()
    assert hasattr(mod, "token_logprobs") and hasattr(mod, "scaled_embedding")
    for name in ("logprob_bwd", "scaled_embedding_bwd", "swiglu8_bwd", "swiglu8_fwd", "pack8"):
        assert not hasattr(mod, name)


# ---------------------------------------------------- CPU definitions
def _logits(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(8, 50, generator=g) * 3).to(dtype)
    x[1, ::2] = -math.inf
    x[2] = -math.inf                           # an empty row
    x[3] = torch.finfo(dtype).min              # uniform, at the type's lowest value
    x[4] = x[4, 0]                             # ties everywhere
    tok = torch.tensor([3, 4, 5, 6, 7, -100, 0, 49])
    return x, tok


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T", [1.0, 0.7])
def test_token_logprobs_cpu(dtype, T):
    x, tok = _logits(dtype)
    x.requires_grad_()
    r = ops.token_logprobs(x, tok, temperature=T, entropy=True, top_k=7)
    g = torch.Generator().manual_seed(1)
    gs = [torch.randn(8, generator=g), torch.randn(8, generator=g), torch.randn(8, 7, generator=g)]
    want = oracle.logprobs(x, tok, T, 7, g_lp=gs[0], g_ent=gs[1], g_top=gs[2])
    oracle.close(r.logprobs, want["lp"], want["lp_tol"])
    oracle.close(r.entropy, want["ent"], want["ent_tol"])
    oracle.close(r.top_logprobs, want["top_lp"], want["top_tol"])
    assert torch.equal(r.top_tokens, want["top"])
    (dx,) = torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], x, gs)
    oracle.close(dx, want["dx"], want["dx_tol"])


def test_oracle_gradient_is_the_difference_quotient():
    """The closed-form gradient of the 64-bit definition against central
    differences: their error is the third derivative's, under h^2 of the
    values, plus the rounding of the values over h."""
    x, tok = _logits(torch.float32)
    x = x.double()
    g = torch.Generator().manual_seed(2)
    gl, ge, gt = (torch.randn(8, n, generator=g).double() for n in (1, 1, 5))
    gl[1] = 0   # row 1's token is masked: its log probability is -inf
    want = oracle.logprobs(x, tok, 0.8, 5, g_lp=gl, g_ent=ge, g_top=gt)

    def total(v):
        o = oracle.logprobs(v, tok, 0.8, 5)
        lp = torch.log_softmax(torch.where(torch.isinf(v).all(-1, keepdim=True), 0.0, v / 0.8), -1) \
            .gather(1, want["top"].clamp(min=0))
        fin = lambda t: torch.where(torch.isfinite(t), t, 0.0)  # noqa: E731
        keep = (tok != -100).double()
        return ((gl[:, 0] * fin(o["lp"]) + ge[:, 0] * o["ent"]) * keep
                + (gt * fin(lp)).sum(-1) * keep)

    h = 1e-5
    for row, col in [(0, 3), (0, 10), (1, 1), (4, 7), (4, 20), (5, 0), (6, 0), (7, 49)]:
        up, down = x.clone(), x.clone()
        up[row, col] += h
        down[row, col] -= h
        num = float((total(up) - total(down))[row] / (2 * h))
        assert num == pytest.approx(float(want["dx"][row, col]), abs=1e-8)


@pytest.mark.parametrize("dtype", DT)
def test_scaled_embedding_cpu(dtype):
    g = torch.Generator().manual_seed(0)
    w = torch.randn(11, 5, generator=g).to(dtype).requires_grad_()
    idx = torch.tensor([[0, 3, 3], [10, 2, 3]])
    y = ops.scaled_embedding(idx, w, 2.5, padding_idx=2)
    assert torch.equal(y, (w.detach()[idx].float() * 2.5).to(dtype))
    d = torch.randn(2, 3, 5, generator=g).to(dtype)
    (dw,) = torch.autograd.grad(y, w, d)
    want, tol = oracle.embedding_grad(d, idx, 11, 2.5, 2)
    oracle.close(dw, want, tol)


@pytest.mark.parametrize("shape", [(0,), (2, 0), (0, 3)])
def test_scaled_embedding_cpu_of_nothing(shape):
    w = torch.randn(5, 4, requires_grad=True)
    y = ops.scaled_embedding(torch.zeros(shape, dtype=torch.int64), w, 2.0)
    assert y.shape == (*shape, 4)
    (dw,) = torch.autograd.grad(y.sum(), w)
    assert torch.equal(dw, torch.zeros(5, 4))


def test_scaled_embedding_cpu_uses_the_sink_or_autograd():
    p = nn.Parameter(torch.randn(6, 4))
    p.grad = torch.ones(6, 4)
    ops.scaled_embedding(torch.tensor([1, 1, 5]), p, 2.0).sum().backward()
    want = torch.ones(6, 4)
    want[1] += 4
    want[5] += 2
    assert torch.equal(p.grad, want)


def _awkward(dtype, rows, D, seed=0):
    """Blocks of every kind: zeros, one large value, subnormals, the type's
    largest value, halves of a step."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, D, generator=g) * torch.exp(torch.randn(rows, 1, generator=g) * 4)
    x = x.to(dtype)
    x[0] = 0
    x[1, 0] = torch.finfo(dtype).max
    x[2] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    x[3] = torch.arange(D).to(dtype) / 2
    x[4, -1] = torch.finfo(dtype).min
    return x


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("D", [1, 31, 32, 33, 200])
def test_pack_cpu(dtype, D):
    x = _awkward(dtype, 6, D)
    p = ops.pack_activation(x)
    y = p.unpack()
    want = oracle.restored(x)
    assert y.dtype == dtype and y.shape == x.shape
    assert torch.equal(y, want.to(dtype))
    # half a step, or a whole one where a value rounds to 128
    f = torch.nn.functional.pad(x.double(), (0, -D % 32)).unflatten(-1, (-1, 32))
    step = torch.ldexp(torch.ones(6, p.scales.shape[1], 1), p.scales[..., None].int() - 127).double()
    off = (want - x.double()).abs()
    off = torch.nn.functional.pad(off, (0, -D % 32)).unflatten(-1, (-1, 32))
    assert bool((off <= torch.where(f.abs() >= 127.5 * step, step, step / 2)).all())
    assert bool(torch.isfinite(y).all())   # 127 steps are finite in the type, whatever the block


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_pack_marks_blocks_that_are_not_finite(bad):
    x = torch.ones(2, 70)
    x[0, 40] = bad
    y = ops.pack_activation(x).unpack()
    assert bool(torch.isnan(y[0, 32:64]).all())
    assert torch.equal(y[0, :32], x[0, :32]) and torch.equal(y[0, 64:], x[0, 64:])
    assert torch.equal(y[1], x[1])


def test_pack_of_nothing_and_of_views():
    e = ops.pack_activation(torch.zeros(3, 0, 4))
    assert e.unpack().shape == (3, 0, 4) and e.nbytes == 0
    x = torch.randn(4, 6, 64)
    for v in (x.transpose(0, 1), x[:, ::2], x[..., 3:40], x[0, 0]):
        assert torch.equal(ops.pack_activation(v).unpack(), oracle.restored(v).float())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("F", [1, 32, 45])
def test_swiglu_8bit_cpu(dtype, F):
    x = _awkward(dtype, 6, 2 * F, seed=F)
    x = x.clamp(-30, 30).requires_grad_()
    dh = torch.randn(6, F).to(dtype)
    h = ops.swiglu(x, save_bits=8)
    assert torch.equal(h, ops.swiglu(x.detach()))
    (dx,) = torch.autograd.grad(h, x, dh)
    hw, ht, dw, dt = oracle.swiglu(x.detach(), dh)
    oracle.close(h, hw, ht)
    oracle.close(dx, dw, dt)


@pytest.mark.parametrize("dtype", DT)
def test_swiglu_8bit_cpu_gates_far_from_zero(dtype):
    """As on the GPU: down to the last gates whose sigmoid fp32 holds in full."""
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.linspace(-87, 87, 300 * 45).view(300, 45),
                   40 * torch.randn(300, 45, generator=g)], -1).to(dtype).requires_grad_()
    dh = (torch.randn(300, 45, generator=g) * 2.0 ** -12).to(dtype)
    h = ops.swiglu(x, save_bits=8)
    (dx,) = torch.autograd.grad(h, x, dh)
    _, _, dw, dt = oracle.swiglu(x.detach(), dh)
    oracle.close(dx, dw, dt)


@pytest.mark.parametrize("of_dh", [False, True])
def test_swiglu_8bit_cpu_refuses_second_derivatives(of_dh):
    x = torch.randn(2, 64, requires_grad=True)
    dh = torch.randn(2, 32, requires_grad=of_dh)
    h = ops.swiglu(x, save_bits=8)
    with pytest.raises(NotImplementedError, match="create_graph"):
        torch.autograd.grad(h, x, dh, create_graph=True)


def test_swiglu_oracle_gradient_is_the_difference_quotient():
    """At inputs that 8 bits hold exactly, against central differences of the
    64-bit output: off by h^2 of the third derivatives (under 2 here) and the
    output's rounding over h."""
    g = torch.Generator().manual_seed(4)
    x = torch.randint(-127, 128, (2, 64), generator=g).float() / 32
    x[:, ::32] = 127 / 32        # every block's largest: the steps are 1 / 32
    assert torch.equal(oracle.restored(x).float(), x)
    dh = torch.randn(2, 32, generator=g)
    _, _, dx, _ = oracle.swiglu(x, dh)
    h = 1e-5
    for i in range(0, 64, 7):
        up, down = x.double(), x.double()
        up[:, i] += h
        down[:, i] -= h
        f = lambda v: (v[:, :32] * torch.sigmoid(v[:, :32]) * v[:, 32:] * dh.double()).sum(-1)  # noqa: E731
        torch.testing.assert_close((f(up) - f(down)) / (2 * h), dx[:, i], rtol=0, atol=1e-8)


def test_scaled_embedding_gradient_is_the_difference():
    """The lookup is linear: its change with the table is the gradient's product
    with that change, exactly in whole numbers."""
    g = torch.Generator().manual_seed(5)
    w = torch.randint(-8, 9, (13, 6), generator=g).float().requires_grad_()
    step = torch.randint(-8, 9, (13, 6), generator=g).float()
    idx = torch.randint(0, 13, (50,), generator=g)
    d = torch.randint(-8, 9, (50, 6), generator=g).float()
    y = ops.scaled_embedding(idx, w, 3.0)
    (dw,) = torch.autograd.grad(y, w, d)
    change = ops.scaled_embedding(idx, w.detach() + step, 3.0) - y.detach()
    assert float((change * d).sum()) == float((dw * step).sum())


# -------------------------------------------------------- checkpoint
class _Gate(nn.Module):
    def __init__(self, n):
        super().__init__()
        self.a = nn.Linear(n, n)
        self.seen = []

    def forward(self, x, other, table, flag):
        self.seen.append(x.detach().clone())
        return torch.tanh(self.a(x) * table) + other, flag


def test_checkpoint_8bit_recomputes_from_the_packed_argument():
    torch.manual_seed(0)
    m = _Gate(40)
    leaf = torch.randn(3, 40, requires_grad=True)
    x, other = leaf * 1.5, leaf.sin()
    table = torch.randn(40)
    y, flag = checkpoint(m, x, other, table, "kept", save_bits=8)
    exact, _ = m(x, other, table, None)
    assert flag == "kept" and torch.equal(y, exact)
    y.sum().backward()
    assert len(m.seen) == 3
    assert torch.equal(m.seen[0], x.detach())
    assert torch.equal(m.seen[2], oracle.restored(x.detach()).float())
    # the gradient is that of tanh(a(x) * table) with x restored inside
    xr = oracle.restored(x.detach()).float().requires_grad_()
    ref = torch.tanh(m.a(xr) * table)
    gx, gw = torch.autograd.grad(ref.sum(), [xr, m.a.weight])
    got = leaf.grad - leaf.detach().cos()
    torch.testing.assert_close(got, gx * 1.5, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(m.a.weight.grad, gw, rtol=1e-5, atol=1e-6)


def test_checkpoint_8bit_without_gradients_is_the_function():
    m = _Gate(8)
    x = torch.randn(2, 8)
    with torch.no_grad():
        y, _ = checkpoint(m, x, x, torch.ones(8), 0, save_bits=8)
        assert torch.equal(y, m(x, x, torch.ones(8), 0)[0])


def test_checkpoint_8bit_drops_the_exact_argument():
    import gc
    import weakref

    leaf = torch.randn(4, 64, requires_grad=True)
    x = leaf * 2
    w = torch.randn(64, 64, requires_grad=True)
    ref = weakref.ref(x)
    y = checkpoint(lambda t: (t @ w).tanh(), x, save_bits=8)
    del x
    gc.collect()
    assert ref() is None
    y.sum().backward()
    assert leaf.grad is not None and w.grad is not None


def test_checkpoint_8bit_keeps_the_random_state():
    torch.manual_seed(3)
    leaf = torch.ones(64, 64, requires_grad=True)
    y = checkpoint(lambda t: nn.functional.dropout(t, 0.5), leaf * 1, save_bits=8)
    y.sum().backward()
    assert torch.equal(leaf.grad != 0, y.detach() != 0)


@pytest.mark.parametrize("order", [(1, 0, 2), (0, 2, 1), (2, 1, 0)])
def test_checkpoint_8bit_keeps_the_order_of_axes(order):
    """A transposed argument is one in the recompute too: the function may rely
    on a view of it."""
    back = [order.index(i) for i in range(3)]
    leaf = torch.randn(3, 4, 32, requires_grad=True)

    def flat_cube(t):
        return (t.permute(back).view(12, 32) ** 3).sum()

    checkpoint(flat_cube, (leaf * 1).permute(order), save_bits=8).backward()
    moved = leaf.detach().permute(order)     # its blocks lie along its own last axis
    want = 3 * oracle.restored(moved).float().permute(back) ** 2
    torch.testing.assert_close(leaf.grad, want, rtol=1e-6, atol=0)


def test_checkpoint_8bit_of_views_that_are_not_dense():
    base = torch.randn(5, 8, 64, requires_grad=True)
    for view in (lambda t: t[:, ::2, :40], lambda t: t[:1].expand(3, 8, 64),
                 lambda t: t.transpose(0, 1)[..., ::2]):
        x = view(base * 1)
        y = checkpoint(lambda t: (t * t).sum(), x, save_bits=8)
        (got,) = torch.autograd.grad(y, x)
        assert torch.equal(got, 2 * oracle.restored(x.detach()).float())


def test_checkpoint_8bit_twice_backward():
    leaf = torch.randn(4, 32, requires_grad=True)
    y = checkpoint(lambda t: (t * t).sum(), leaf * 1, save_bits=8)
    (a,) = torch.autograd.grad(y, leaf, retain_graph=True)
    (b,) = torch.autograd.grad(y, leaf)
    assert torch.equal(a, b) and torch.equal(a, 2 * oracle.restored(leaf.detach()).float())


# ------------------------------------------------------------- the models
def _models(**kw):
    torch.manual_seed(0)
    size = dict(vocab_size=97, block_size=32, n_layer=2, n_head=4, n_embd=64)
    gpt_kw = {k: v for k, v in kw.items() if k in GPTConfig.__dataclass_fields__}
    return [init_gpt2_(GPT(GPTConfig(**size, **gpt_kw))),
            init_llama_(Llama(LlamaConfig(n_kv_head=2, ffn_hidden=96, **size, **kw)))]


@pytest.mark.parametrize("which", [0, 1])
def test_model_logprobs_are_the_losses_of_the_targets(which):
    m = _models()[which]
    x = torch.randint(0, 97, (2, 20))
    y = torch.roll(x, -1, 1)
    y[:, -1] = -100
    r = m(x, targets=y, logprobs={"entropy": True, "top_k": 2})
    assert r.logprobs.shape == (2, 20) and r.top_tokens.shape == (2, 20, 2)
    torch.testing.assert_close(-r.logprobs.sum() / 38, m(x, targets=y), rtol=1e-5, atol=1e-6)
    assert m(x, targets=y, logprobs={}).entropy is None
    with pytest.raises(ValueError, match="targets"):
        m(x, logprobs={})


def test_model_options_change_only_what_they_say():
    """The loss of a model with 8-bit saves and a scale of 1 is that of the
    plain one; its gradients are near it: an input kept in 8 bits is off by
    2^-7 of its block at most, some ten such on the way of a gradient."""
    x = torch.randint(0, 97, (2, 32))
    for which in (0, 1):
        a = _models()[which]
        b = _models(activation_checkpointing=True, checkpoint_bits=8, swiglu_save_bits=8,
                    embed_scale=1.0)[which]
        la, lb = (m(x, targets=torch.roll(x, -1, 1)) for m in (a, b))
        torch.testing.assert_close(lb, la, rtol=1e-6, atol=1e-6)
        la.backward()
        lb.backward()
        for p, q in zip(a.parameters(), b.parameters()):
            assert float((p.grad - q.grad).norm()) <= 10 * 2 ** -7 * float(p.grad.norm()) + 1e-9


@pytest.mark.parametrize("stage", [0, 2, 3])
def test_engine_trains_on_log_probabilities(stage):
    m = _models(activation_checkpointing=True, checkpoint_bits=8, swiglu_save_bits=8,
                embed_scale=8.0)[1]
    engine = ms.initialize(model=m, config={
        "train_micro_batch_size_per_gpu": 2, "gradient_accumulation_steps": 2, "dtype": "fp32",
        "zero_optimization": {"stage": stage},
        "optimizer": {"type": "AdamW", "params": {"lr": 1e-3}}})
    before = m.embed.weight.detach().clone()
    x = torch.randint(0, 97, (2, 16))
    for _ in range(2):
        r = engine(x, targets=torch.roll(x, -1, 1), logprobs={"entropy": True})
        engine.backward(-(r.logprobs.mean() + 0.01 * r.entropy.mean()))
        engine.step()
    after = m.embed.weight.detach()
    assert torch.isfinite(after).all() and not torch.equal(after, before)
