"""Autograd operators of the model zoo over the sm_100a kernels.

Every op has two definitions of the same math: the CUDA path (the kernels of
``minispeed_b200._C``) and a PyTorch path used for CPU tensors, which is
also the fp32 oracle of the GPU numerics tests.

Ops:
  ``add_norm``        fused residual add + LayerNorm/RMSNorm (returns the new
                      residual stream and the normalized activations)
  ``norm``            LayerNorm/RMSNorm without a residual
  ``linear``          x @ W^T + b through :mod:`.gemm`
  ``linear_gelu``     gelu(x @ W^T + b) (exact erf GELU, saves the pre-activation)
  ``swiglu``          silu(gate) * up on a fused [gate | up] projection; can keep its
                      input in 8 bits for backward
  ``pack_activation`` a tensor in 8 bits with a scale per 32 values, and back
  ``cross_entropy``   fused softmax cross-entropy on model-dtype logits
  ``token_logprobs``  log probabilities of given tokens, entropy, top alternatives
  ``embedding``       token (+ learned position) embedding
  ``scaled_embedding`` token embedding times a scale; its gradient summed in a
                      fixed order, by sorted tokens
  ``rope_``           rotary embedding on q/k views

Reference: the layers of the example model (``examples/train_lm.py:62-115``:
``nn.Linear`` projections, ``nn.LayerNorm`` at ``:84``, ``:86`` and ``:105``,
``nn.GELU`` MLP at ``:88``, token + position embeddings) and its loss
(``F.cross_entropy`` at ``:246``).  ``swiglu``, RMSNorm and ``rope_`` serve the
Llama family, which the reference has no model for.
"""

from __future__ import annotations

import math
from contextlib import contextmanager
from typing import NamedTuple, Optional, Tuple

import torch
import torch.nn.functional as F

from . import _ext, gemm

_COLSUM_CHUNKS = 256   # row chunks of a column-sum reduction
_NORM_BLOCKS = 296     # row chunks (blocks) of the norm-backward dw/db column sums


def _C():
    return _ext.get()


def _tc(x: torch.Tensor) -> bool:
    """GEMM-bearing ops run the tcgen05 kernels for 16-bit CUDA tensors; fp32
    models (a debugging configuration of the reference's GPU tests) run
    PyTorch's fp32 GEMM, since tcgen05 ``kind::f16`` takes 16-bit operands."""
    return x.is_cuda and x.dtype in (torch.float16, torch.bfloat16)


def _scratch(device, n: int) -> torch.Tensor:
    return torch.empty(n, dtype=torch.float32, device=device)


def as_matrix(t: torch.Tensor, n: int) -> torch.Tensor:
    """``t`` viewed as a row-major [rows, n] matrix with unit column stride;
    copies only when no such view exists (a padded leading dimension is kept)."""
    m = t.reshape(-1, n)
    if m.stride(-1) != 1 or (m.shape[0] > 1 and m.stride(0) < n):
        m = m.contiguous()
    return m


def grad_sink(p: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """The parameter's existing ``.grad`` if gradients can be accumulated into
    it in place (the engine binds every ``p.grad`` to a view of its flat
    gradient arena), else None.

    Backward kernels write into a sink directly (GEMM epilogue accumulate,
    column-sum accumulate) and report no gradient to autograd for that input,
    which is what autograd's own accumulation would have produced."""
    if p is None or not isinstance(p, torch.nn.Parameter):
        return None
    g = p.grad
    if g is None or g.dtype != p.dtype or g.shape != p.shape or not g.is_contiguous():
        return None
    return g


class _FinishQueue:
    """Column-sum finishes into gradient sinks, batched.

    A bias or norm-weight gradient is the column sum of fp32 partial rows
    that its backward kernel leaves; the finish that adds them into the
    gradient is a launch of its own, tiny and latency-bound (a GPT-2 small
    step has 98 of them).  Inside :func:`batched_colsums` (the engine's
    backward) finishes into sinks are queued instead and run together by
    ``colsum_finish_many``: one launch per flush.  A flush happens when the
    context exits normally, before a gradient bucket is handed to the
    collectives (:func:`flush_colsums`), when ``_BATCH`` finishes are queued,
    and before a finish whose sink, stream or dtype conflicts with the queue
    (two finishes into one sink in one launch would race).  The queue keeps
    each partial buffer alive until its flush has been launched.

    Autograd runs CUDA backward functions on its own thread while the caller
    waits in ``backward()``; the queue is shared module state, touched by one
    thread at a time."""

    _BATCH = 48

    def __init__(self):
        self.depth = 0
        self.clear()

    def clear(self):
        self.parts, self.nparts, self.outs = [], [], []
        self.sinks = set()
        self.stream = None

    def add(self, part: torch.Tensor, nparts: int, sink: torch.Tensor) -> None:
        st = torch.cuda.current_stream(sink.device)
        key = sink.data_ptr()
        if self.outs and (key in self.sinks or st != self.stream
                          or sink.dtype != self.outs[0].dtype):
            self.flush()
        if not self.outs:
            self.stream = st
        self.parts.append(part)
        self.nparts.append(int(nparts))
        self.outs.append(sink)
        self.sinks.add(key)
        if len(self.outs) >= self._BATCH:
            self.flush()

    def flush(self) -> None:
        if not self.outs:
            return
        with torch.cuda.stream(self.stream):
            _C().colsum_finish_many(self.parts, self.nparts, self.outs,
                                    [True] * len(self.outs))
        self.clear()


_finishes = _FinishQueue()


@contextmanager
def batched_colsums():
    """Queue column-sum finishes into gradient sinks while the block runs
    (a backward pass) and launch them batched; nests."""
    _finishes.depth += 1
    ok = False
    try:
        yield
        ok = True
    finally:
        _finishes.depth -= 1
        if _finishes.depth == 0:
            if ok:
                _finishes.flush()
            else:
                _finishes.clear()


def flush_colsums() -> None:
    """Launch the queued finishes now (the gradients they complete are about
    to be read)."""
    _finishes.flush()


def _finish_into(part: torch.Tensor, nparts: int, sink: torch.Tensor) -> None:
    """sink += the column sums of ``part``'s first ``nparts`` rows."""
    if _finishes.depth > 0:
        _finishes.add(part, nparts, sink)
    else:
        _C().colsum_finish(part, nparts, sink, True)


def _colsum(a2d: torch.Tensor, dtype, sink: Optional[torch.Tensor] = None
            ) -> Optional[torch.Tensor]:
    """Column sums of a [M, N] CUDA matrix (bias gradients); accumulated into
    ``sink`` (returns None) or returned as a new tensor."""
    n = a2d.shape[-1]
    part = _scratch(a2d.device, _COLSUM_CHUNKS * n)
    nb = _C().colsum_partial(a2d, part, _COLSUM_CHUNKS)
    if sink is not None:
        _finish_into(part, nb, sink)
        return None
    out = torch.empty(n, dtype=dtype, device=a2d.device)
    _C().colsum_finish(part, nb, out, False)
    return out


def _wgrad(dy2: torch.Tensor, x2: torch.Tensor, w: torch.Tensor) -> Optional[torch.Tensor]:
    """dW = dy^T x, accumulated into w's gradient sink when it has one."""
    sink = grad_sink(w)
    if sink is not None:
        gemm.linear_wgrad(dy2, x2, out=sink.view(sink.shape[0], -1), accumulate=True)
        return None
    return gemm.linear_wgrad(dy2, x2)


# --------------------------------------------------------------- norms
class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, w, b, eps, rms):
        C = x.shape[-1]
        M = x.numel() // C
        y = torch.empty_like(x)
        rstd = torch.empty(M, dtype=torch.float32, device=x.device)
        mean = None if rms else torch.empty(M, dtype=torch.float32, device=x.device)
        s = torch.empty_like(x) if delta is not None else None
        _C().add_norm_fwd(x, delta, w, b, s, y, mean, rstd, eps, rms)
        saved = s if s is not None else x
        ctx.save_for_backward(saved, w, mean, rstd)
        ctx.params = (w, b)
        ctx.rms = rms
        ctx.has_delta = delta is not None
        ctx.has_bias = b is not None
        if s is not None:
            return s, y
        return y

    @staticmethod
    def backward(ctx, *grads):
        if ctx.has_delta:
            ds, dy = grads
        else:
            (dy,) = grads
            ds = None
        s, w, mean, rstd = ctx.saved_tensors
        C = s.shape[-1]
        dy = dy.contiguous()
        dx = torch.empty_like(s)
        dw_part = _scratch(s.device, _NORM_BLOCKS * C)
        db_part = None if ctx.rms else _scratch(s.device, _NORM_BLOCKS * C)
        if ds is not None:
            ds = ds.contiguous()
        nb = _C().norm_bwd(dy, s, w, mean, rstd, ds, dx, dw_part, db_part, ctx.rms,
                           _NORM_BLOCKS)
        w_p, b_p = ctx.params
        dw = db = None
        sink = grad_sink(w_p)
        if sink is not None:
            _finish_into(dw_part, nb, sink)
        else:
            dw = torch.empty_like(w)
            _C().colsum_finish(dw_part, nb, dw, False)
        if ctx.has_bias:
            sink = grad_sink(b_p)
            if sink is not None:
                _finish_into(db_part, nb, sink)
            else:
                db = torch.empty_like(w)
                _C().colsum_finish(db_part, nb, db, False)
        if ctx.has_delta:
            return dx, dx, dw, db, None, None
        return dx, None, dw, db, None, None


def _norm_torch(x, w, b, eps, rms):
    xf = x.float()
    if rms:
        y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.float()
    else:
        y = F.layer_norm(xf, (x.shape[-1],), w.float(), None if b is None else b.float(), eps)
    return y.to(x.dtype)


def add_norm(x: torch.Tensor, delta: torch.Tensor, w, b, eps: float = 1e-5,
             rms: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """(s, y) with s = x + delta (residual stream) and y = norm(s)."""
    if x.is_cuda:
        return _AddNorm.apply(x.contiguous(), delta.contiguous(), w, b, eps, rms)
    s = x + delta
    return s, _norm_torch(s, w, b, eps, rms)


def norm(x: torch.Tensor, w, b, eps: float = 1e-5, rms: bool = False) -> torch.Tensor:
    if x.is_cuda:
        return _AddNorm.apply(x.contiguous(), None, w, b, eps, rms)
    return _norm_torch(x, w, b, eps, rms)


# -------------------------------------------------------------- linears
class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, pad):
        shp = x.shape
        x2 = as_matrix(x, shp[-1])
        N = w.shape[0]
        out = None
        if pad:
            # leading dimension rounded up to a multiple of `pad` elements so
            # that every row starts 16-byte aligned (TMA / vector access)
            ld = -(-N // pad) * pad
            out = torch.empty(x2.shape[0], ld, dtype=x.dtype, device=x.device)[:, :N]
        out = gemm.linear_fwd(x2, w, b, out=out)
        ctx.save_for_backward(x2, w)
        ctx.params = (w, b)
        ctx.shape = shp
        return out.view(*shp[:-1], N)

    @staticmethod
    def backward(ctx, dy):
        x2, w = ctx.saved_tensors
        w_p, b_p = ctx.params
        dy2 = as_matrix(dy, w.shape[0])
        dx = gemm.linear_dgrad(dy2, w) if ctx.needs_input_grad[0] else None
        dw = _wgrad(dy2, x2, w_p)
        db = _colsum(dy2, w.dtype, grad_sink(b_p)) if b_p is not None else None
        if dx is not None:
            dx = dx.view(ctx.shape)
        return dx, dw, db, None


class _MlpGelu(torch.autograd.Function):
    """fc2(gelu(fc(x))) with both GELU passes fused into GEMM epilogues:
    forward  fc : u = x W1^T + b1 and a = gelu(u) written by one epilogue
    backward fc2-dgrad: du = (dout W2) * gelu'(u) written by one epilogue."""

    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2):
        shp = x.shape
        x2 = as_matrix(x, shp[-1])
        M, F_ = x2.shape[0], w1.shape[0]
        u = torch.empty(M, F_, dtype=x.dtype, device=x.device)
        a = torch.empty_like(u)
        gemm.gemm(x2, w1, a_kmajor=True, b_kmajor=True, bias=b1, out=u,
                  mode=gemm.EPI_BIAS_GELU, aux=a)
        out = gemm.linear_fwd(a, w2, b2)
        ctx.save_for_backward(x2, w1, u, a, w2)
        ctx.params = (w1, b1, w2, b2)
        ctx.shape = shp
        return out.view(*shp[:-1], w2.shape[0])

    @staticmethod
    def backward(ctx, dout):
        x2, w1, u, a, w2 = ctx.saved_tensors
        w1_p, b1_p, w2_p, b2_p = ctx.params
        d2 = as_matrix(dout, w2.shape[0])
        dw2 = _wgrad(d2, a, w2_p)
        db2 = _colsum(d2, w2.dtype, grad_sink(b2_p)) if b2_p is not None else None
        du = torch.empty_like(u)
        M, F_ = du.shape
        # the dGELU epilogue also leaves the column sums of du (fc bias
        # gradient), one partial row per 32 rows: no second read of du
        part = _scratch(du.device, -(-M // 32) * F_) if b1_p is not None else None
        gemm.gemm(d2, w2, a_kmajor=True, b_kmajor=False, out=du, mode=gemm.EPI_DGELU, aux=u,
                  colsum=part)
        dw1 = _wgrad(du, x2, w1_p)
        db1 = None
        if b1_p is not None:
            sink = grad_sink(b1_p)
            if sink is not None:
                _finish_into(part, -(-M // 32), sink)
            else:
                db1 = torch.empty(F_, dtype=w1.dtype, device=du.device)
                _C().colsum_finish(part, -(-M // 32), db1, False)
        dx = gemm.linear_dgrad(du, w1).view(ctx.shape) if ctx.needs_input_grad[0] else None
        return dx, dw1, db1, dw2, db2


def linear(x: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor] = None,
           pad_out: int = 0) -> torch.Tensor:
    """``x @ w.T + b``.  ``pad_out`` > 0 allocates the output with its row
    stride rounded up to a multiple of ``pad_out`` (the returned tensor is a
    view with the logical width)."""
    if _tc(x):
        return _Linear.apply(x, w, b, pad_out)
    return F.linear(x, w, b)


def mlp_gelu(x: torch.Tensor, w1: torch.Tensor, b1: Optional[torch.Tensor], w2: torch.Tensor,
             b2: Optional[torch.Tensor]) -> torch.Tensor:
    """``fc2(gelu(fc(x)))`` (exact erf GELU)."""
    if _tc(x):
        return _MlpGelu.apply(x, w1, b1, w2, b2)
    return F.linear(F.gelu(F.linear(x, w1, b1)), w2, b2)


def linear_gelu(x: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor] = None
                ) -> torch.Tensor:
    """``gelu(x @ w.T + b)`` (pre-activation kept for backward)."""
    if _tc(x):
        return _LinearGelu.apply(x, w, b)
    return F.gelu(F.linear(x, w, b))


class _LinearGelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b):
        shp = x.shape
        x2 = as_matrix(x, shp[-1])
        u = torch.empty(x2.shape[0], w.shape[0], dtype=x.dtype, device=x.device)
        h = torch.empty_like(u)
        gemm.gemm(x2, w, a_kmajor=True, b_kmajor=True, bias=b, out=u,
                  mode=gemm.EPI_BIAS_GELU, aux=h)
        ctx.save_for_backward(x2, w, u)
        ctx.params = (w, b)
        ctx.shape = shp
        return h.view(*shp[:-1], w.shape[0])

    @staticmethod
    def backward(ctx, dh):
        x2, w, u = ctx.saved_tensors
        w_p, b_p = ctx.params
        du = torch.empty_like(u)
        _C().gelu_bwd(as_matrix(dh, w.shape[0]).contiguous(), u, du)
        dw = _wgrad(du, x2, w_p)
        db = _colsum(du, w.dtype, grad_sink(b_p)) if b_p is not None else None
        dx = gemm.linear_dgrad(du, w).view(ctx.shape) if ctx.needs_input_grad[0] else None
        return dx, dw, db


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu):
        F_ = gu.shape[-1] // 2
        h = torch.empty(*gu.shape[:-1], F_, dtype=gu.dtype, device=gu.device)
        _C().swiglu_fwd(gu, h)
        ctx.save_for_backward(gu)
        return h

    @staticmethod
    def backward(ctx, dh):
        (gu,) = ctx.saved_tensors
        dgu = torch.empty_like(gu)
        _C().swiglu_bwd(dh.contiguous(), gu, dgu)
        return dgu


class _SwiGLU8CPU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu):
        F_ = gu.shape[-1] // 2
        ctx.save_for_backward(*_pack8_torch(gu.reshape(-1, F_)))
        return _swiglu_torch(gu)

    @staticmethod
    def backward(ctx, dh):
        if torch.is_grad_enabled():   # the packed values have no graph back to gu
            raise NotImplementedError("swiglu with save_bits=8: second derivatives "
                                      "(create_graph=True) are not implemented")
        F_ = dh.shape[-1]
        g, u = _unpack8_torch(*ctx.saved_tensors, F_).view(-1, 2, F_).unbind(1)
        d = dh.reshape(-1, F_).float()
        s = torch.sigmoid(g)
        dgu = torch.cat([d * u * (s * (1 + g * (1 - s))), d * (g * s)], -1)
        return dgu.view(*dh.shape[:-1], 2 * F_).to(dh.dtype)


def _swiglu_torch(gu: torch.Tensor) -> torch.Tensor:
    g, u = gu.chunk(2, dim=-1)
    return (F.silu(g.float()) * u.float()).to(gu.dtype)


def _check_save_bits(save_bits) -> bool:
    """True for 8-bit saves, False for saves as they are (None)."""
    if save_bits not in (None, 8):
        raise ValueError(f"save_bits must be None or 8, got {save_bits!r}")
    return save_bits == 8


def swiglu(gu: torch.Tensor, save_bits: Optional[int] = None) -> torch.Tensor:
    """``silu(gu[..., :F]) * gu[..., F:]`` for a fused gate/up projection.

    ``save_bits=8`` keeps ``gu`` for backward in 8 bits (the format of
    :func:`pack_activation`, gate and up in blocks of their own): about half
    the memory of a 16-bit ``gu``.  The output is that of the exact input: in
    fp32 the same bits as without, in 16 bits now and then the next value.  The
    gradient is the formula's at the packed values (NaN for the values of a
    block that holds an infinity or a NaN).  Second and forward-mode derivatives
    raise."""
    if _check_save_bits(save_bits):
        _check_packable(gu)
        if gu.shape[-1] % 2:
            raise ValueError(f"swiglu: the last axis holds [gate | up], got width {gu.shape[-1]}")
        if not gu.numel():
            return _swiglu_torch(gu)
        return _C().swiglu8(gu) if gu.is_cuda else _SwiGLU8CPU.apply(gu)
    if gu.is_cuda:
        return _SwiGLU.apply(gu.contiguous())
    return _swiglu_torch(gu)


# ---------------------------------------------------- 8-bit activations
PACK_BLOCK = 32   # values per scale

_DTYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _check_packable(x: torch.Tensor) -> None:
    if x.dtype not in _DTYPE_CODES:
        raise TypeError(f"8-bit activations: fp32, fp16 or bf16 tensors, got {x.dtype}")
    if x.dim() == 0:
        raise ValueError("8-bit activations: a tensor with at least one axis is needed")


def _pack8_torch(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes [rows, 32 * blocks] and scale bytes [rows, blocks] of a matrix."""
    f = F.pad(x.detach().float(), (0, -x.shape[-1] % PACK_BLOCK)).unflatten(-1, (-1, PACK_BLOCK))
    field = (f.view(torch.int32) & 0x7FFFFFFF).amax(-1, keepdim=True) >> 23
    b = torch.where(field == 255, field, (field - 6).clamp(min=0))
    q = torch.round(torch.ldexp(f, 127 - b)).clamp(-127, 127)
    q = torch.where(b == 255, 0.0, q)
    return q.to(torch.int8).flatten(-2), b.squeeze(-1).to(torch.uint8)


def _unpack8_torch(codes: torch.Tensor, scales: torch.Tensor, width: int) -> torch.Tensor:
    b = scales[..., None].int()
    f = torch.ldexp(codes.unflatten(-1, (-1, PACK_BLOCK)).float(), b - 127)
    return torch.where(b == 255, float("nan"), f).flatten(-2)[..., :width]


class PackedActivation:
    """A tensor held in 8 bits: one signed byte a value (``codes``, int8
    [rows, 32 * blocks]) and one byte, the exponent of a power-of-two scale, for
    every 32 values of the last axis (``scales``, uint8 [rows, blocks]; the last
    block of a row may be short); and its ``shape`` and ``dtype``."""

    __slots__ = ("codes", "scales", "shape", "dtype")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape: torch.Size,
                 dtype: torch.dtype):
        self.codes, self.scales, self.shape, self.dtype = codes, scales, shape, dtype

    def unpack(self) -> torch.Tensor:
        """The tensor again, contiguous, in its own type.  Values are off by at
        most half a step of their block's scale, 2^-7 of its largest magnitude
        (a whole step for values that round to 128 steps); a block that held an
        infinity or a NaN is all NaN."""
        if 0 in self.shape:
            return torch.empty(self.shape, dtype=self.dtype, device=self.codes.device)
        if self.codes.is_cuda:
            return _C().unpack8(self.codes, self.scales, self.shape, _DTYPE_CODES[self.dtype])
        x = _unpack8_torch(self.codes, self.scales, self.shape[-1])
        return x.to(self.dtype).view(self.shape)

    @property
    def nbytes(self) -> int:
        return self.codes.nbytes + self.scales.nbytes


def pack_activation(x: torch.Tensor) -> PackedActivation:
    """``x`` (fp32, fp16 or bf16, any shape with at least one axis) in 8 bits;
    :meth:`PackedActivation.unpack` brings it back.  No gradient flows through
    the pair: it is for what a backward pass keeps."""
    _check_packable(x)
    if not x.numel():
        empty = x.new_empty((0, 0), dtype=torch.uint8)
        return PackedActivation(empty.view(torch.int8), empty, x.shape, x.dtype)
    codes, scales = _C().pack_rows(x) if x.is_cuda else \
        _pack8_torch(as_matrix(x.detach(), x.shape[-1]))
    return PackedActivation(codes, scales, x.shape, x.dtype)


# -------------------------------------------------------- cross entropy
_LOSS_GRAD_HINT: list = [None]


@contextmanager
def expected_loss_grad(seed: Optional[torch.Tensor]):
    """Within this context, :func:`cross_entropy` on CUDA computes its
    gradient during the forward, for the upstream gradient ``seed`` (an fp32
    CUDA scalar: the backward seed the engine will use, i.e. loss scale /
    gradient-accumulation steps).  The backward then only checks the real
    upstream gradient against ``seed`` and rescales when they differ.  The
    logits are read from DRAM once instead of twice.  ``None`` turns it off."""
    prev = _LOSS_GRAD_HINT[0]
    _LOSS_GRAD_HINT[0] = seed
    try:
        yield
    finally:
        _LOSS_GRAD_HINT[0] = prev


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, ignore_index, hint):
        V = logits.shape[-1]
        l2 = as_matrix(logits, V)
        M = l2.shape[0]
        t = targets.reshape(-1).contiguous()
        lse = torch.empty(M, dtype=torch.float32, device=logits.device)
        rows = torch.empty(M, dtype=torch.float32, device=logits.device)
        loss = torch.empty((), dtype=torch.float32, device=logits.device)
        inv = torch.empty(1, dtype=torch.float32, device=logits.device)
        if hint is not None:
            # the logits buffer becomes the gradient for upstream gradient `hint`
            _C().cross_entropy_fwd_grad(l2, t, lse, rows, loss, inv, hint, ignore_index)
        else:
            _C().cross_entropy_fwd(l2, t, lse, rows, loss, inv, ignore_index)
        ctx.save_for_backward(l2, t, lse, inv)
        ctx.hint = hint
        ctx.ignore_index = ignore_index
        ctx.shape = logits.shape
        return loss

    @staticmethod
    def backward(ctx, g):
        l2, t, lse, inv = ctx.saved_tensors
        go = g.float().reshape(1).contiguous()
        if ctx.hint is not None:
            _C().cross_entropy_grad_rescale(l2, go, ctx.hint)
        else:
            # the logits buffer is consumed in place: it becomes dlogits
            _C().cross_entropy_bwd(l2, t, lse, go, inv, ctx.ignore_index)
        ctx.hint = None
        return l2.view(ctx.shape), None, None, None


def cross_entropy(logits: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100
                  ) -> torch.Tensor:
    """Mean softmax cross-entropy in fp32 math over model-dtype logits.

    On CUDA the logits tensor is overwritten by its gradient (during backward,
    or during the forward inside :func:`expected_loss_grad`): it must not be
    used after the loss is computed."""
    if logits.is_cuda:
        hint = _LOSS_GRAD_HINT[0]
        if hint is not None and not (torch.is_grad_enabled() and logits.requires_grad
                                     and hint.device == logits.device):
            hint = None
        return _CrossEntropy.apply(logits, targets, ignore_index, hint)
    return F.cross_entropy(logits.reshape(-1, logits.shape[-1]).float(), targets.reshape(-1),
                           ignore_index=ignore_index)


# ------------------------------------------------- token log probabilities
MAX_TOP_K = 32


class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` returns; what was not asked for is None."""

    logprobs: torch.Tensor                 # fp32, the tokens' shape
    entropy: Optional[torch.Tensor]        # fp32, the tokens' shape
    top_logprobs: Optional[torch.Tensor]   # fp32 [..., k], most probable first
    top_tokens: Optional[torch.Tensor]     # int64 [..., k]


def _token_logprobs_torch(logits, tokens, temperature, entropy, top_k, ignore_index):
    """The same in PyTorch operations."""
    keep = tokens != ignore_index
    at = torch.where(keep, tokens, 0)
    if bool(((at < 0) | (at >= logits.shape[-1])).any()):
        raise IndexError("token_logprobs: token outside the vocabulary")
    x = logits.float()
    empty = (x == -math.inf).all(-1, keepdim=True)
    # an empty row is computed as a row of zeros, and replaced below; the largest
    # logit is subtracted first: dividing the lowest value of fp32 overflows
    x = torch.where(empty, 0.0, x)
    logp = torch.log_softmax((x - x.detach().amax(-1, keepdim=True)) / temperature, -1)
    keep_row, empty_row = keep[..., None], empty[..., 0]

    def settle(v, k, e, of_empty):
        return torch.where(k, torch.where(e, of_empty, v), 0.0)

    lp = settle(logp.gather(-1, at[..., None])[..., 0], keep, empty_row, -math.inf)
    ent = top_lp = top = None
    if entropy:
        # p log p is zero where p is, in its gradient too
        live = torch.where(logp == -math.inf, 0.0, logp)
        ent = settle(-(logp.exp() * live).sum(-1), keep, empty_row, 0.0)
    if top_k:
        top = torch.sort(logits.detach(), dim=-1, descending=True, stable=True).indices[..., :top_k]
        top_lp = settle(logp.gather(-1, top), keep_row, empty, -math.inf)
        top = torch.where(keep_row, top, -1)
    return lp, ent, top_lp, top


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0,
                   entropy: bool = False, top_k: int = 0, ignore_index: int = -100
                   ) -> TokenLogprobs:
    """Log probabilities of ``tokens`` under softmax(``logits`` / ``temperature``),
    for a temperature between 1e-30 and 1e30.

    ``logits`` [..., V] in fp32, fp16 or bf16 (rows may be padded, as
    ``linear(pad_out=)`` leaves them) and int64 ``tokens`` [...].  All results
    are fp32 and computed in fp32.  ``entropy`` adds the entropy of every
    position, ``top_k`` (at most 32) its most probable tokens and their log
    probabilities: by logit, the lower index first among equals.

    Positions whose token is ``ignore_index`` are skipped: their results are 0
    (top tokens -1), their gradient is zero.  A logit of -inf excludes a token;
    a position where every logit is -inf has log probabilities -inf and no
    entropy or gradient, and one with a NaN or +inf is NaN throughout (its top
    tokens are then unspecified, within the vocabulary).  A token outside the
    vocabulary raises ``IndexError`` on the CPU; on CUDA, where raising would
    need a synchronization, its log probability is NaN and has no gradient.

    Gradients flow to ``logits`` from the log probabilities, the entropy and
    the top log probabilities.  Unlike :func:`cross_entropy` this leaves the
    logits as they are.  Second and forward-mode derivatives raise on CUDA."""
    if logits.dtype not in _DTYPE_CODES:
        raise TypeError(f"token_logprobs: fp32, fp16 or bf16 logits, got {logits.dtype}")
    if tokens.dtype != torch.int64:
        raise TypeError(f"token_logprobs: int64 tokens, got {tokens.dtype}")
    if logits.dim() == 0 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"token_logprobs: logits {tuple(logits.shape)} need tokens "
                         f"{tuple(logits.shape[:-1])}, got {tuple(tokens.shape)}")
    if tokens.device != logits.device:
        raise ValueError(f"token_logprobs: logits on {logits.device}, tokens on {tokens.device}")
    V = logits.shape[-1]
    if V == 0:
        raise ValueError("token_logprobs: the vocabulary is empty")
    if not 0 <= top_k <= min(MAX_TOP_K, V):
        raise ValueError(f"token_logprobs: top_k must be between 0 and {min(MAX_TOP_K, V)}, "
                         f"got {top_k}")
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"token_logprobs: temperature must be between 1e-30 and 1e30, got "
                         f"{temperature}")
    args = (float(temperature), bool(entropy), int(top_k), int(ignore_index))
    if not (logits.is_cuda and logits.numel()):
        return TokenLogprobs(*_token_logprobs_torch(logits, tokens, *args))
    r = _C().token_logprobs(logits, tokens, *args)
    return TokenLogprobs(r[0], r[1] if entropy else None, *(r[-2:] if top_k else (None, None)))


# ------------------------------------------------------------ embedding
class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, idx, wte, wpe):
        B, T = idx.shape
        C = wte.shape[1]
        out = torch.empty(B, T, C, dtype=wte.dtype, device=wte.device)
        idx = idx.contiguous()
        _C().embedding_fwd(idx, wte, wpe, out, T)
        ctx.save_for_backward(idx)
        ctx.params = (wte, wpe)
        ctx.shapes = (wte.shape, None if wpe is None else wpe.shape, wte.dtype, T)
        return out

    @staticmethod
    def backward(ctx, dout):
        (idx,) = ctx.saved_tensors
        wte_shape, wpe_shape, dtype, T = ctx.shapes
        wte_p, wpe_p = ctx.params
        acc, touched = _embedding_accumulator(dout.device, wte_shape)
        # straight into the gradient arena when the parameter has a sink
        # (tied with the LM head: added to the head GEMM's wgrad), else into
        # a fresh zero gradient
        sink_te = grad_sink(wte_p)
        sink_pe = grad_sink(wpe_p) if wpe_shape is not None else None
        dwte = sink_te if sink_te is not None else torch.zeros(wte_shape, dtype=dtype,
                                                               device=dout.device)
        dwpe = None
        if wpe_shape is not None:
            dwpe = sink_pe if sink_pe is not None else torch.zeros(wpe_shape, dtype=dtype,
                                                                   device=dout.device)
        _C().embedding_bwd(dout.contiguous(), idx, acc, touched, dwte, True, dwpe, True, T)
        return (None, None if sink_te is not None else dwte,
                None if sink_pe is not None or dwpe is None else dwpe)


_EMB_ACC = {}


def _embedding_accumulator(device, shape) -> Tuple[torch.Tensor, torch.Tensor]:
    """The persistent fp32 scatter accumulator [V, C] and touched-row flags
    [V] of a device, zero between uses (the backward kernel clears the rows
    it reads).  Created on the first (eager) backward, before any CUDA-graph
    capture of the step."""
    key = (device, tuple(shape))
    buf = _EMB_ACC.get(key)
    if buf is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("embedding backward: run one eager step before capturing")
        buf = _EMB_ACC[key] = (torch.zeros(shape, dtype=torch.float32, device=device),
                               torch.zeros(shape[0], dtype=torch.uint8, device=device))
    return buf


def embedding(idx: torch.Tensor, wte: torch.Tensor, wpe: Optional[torch.Tensor] = None
              ) -> torch.Tensor:
    """``wte[idx] (+ wpe[:T])``."""
    if wte.is_cuda:
        return _Embedding.apply(idx, wte, wpe)
    x = F.embedding(idx, wte)
    if wpe is not None:
        x = x + wpe[: idx.shape[1]]
    return x


class _ScaledEmbeddingCPU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, idx, weight, scale, padding):
        ctx.save_for_backward(idx)
        ctx.weight = weight
        ctx.args = (padding, scale)
        return (F.embedding(idx, weight).float() * scale).to(weight.dtype)

    @staticmethod
    def backward(ctx, dout):
        (idx,) = ctx.saved_tensors
        padding, scale = ctx.args
        idx = idx.reshape(-1)
        rows = dout.reshape(idx.numel(), dout.shape[-1]).float() * scale
        rows = torch.where((idx == padding)[:, None], 0.0, rows)
        dw = torch.zeros(ctx.weight.shape).index_add_(0, idx, rows)
        return None, dw.to(dout.dtype), None, None


def scaled_embedding(idx: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
                     padding_idx: Optional[int] = None) -> torch.Tensor:
    """``weight[idx] * scale`` for int64 ``idx`` of any shape and a [V, C] table.

    The gradient of a row is an fp32 sum over its positions, rounded once, in
    an order that depends on the call's tokens alone: the same from run to run
    (:func:`embedding` adds with atomics, and keeps an fp32 [V, C] accumulator,
    which this does not).  On CUDA the order is that of the positions within
    parts of the batch sorted by token, and then that of the parts; other
    tokens in the batch move the cuts, and with them last bits.  It goes into ``weight.grad`` where the engine has
    bound one.  Positions equal to ``padding_idx`` give no gradient.

    A token outside the table raises ``IndexError`` on the CPU; on CUDA it
    reads as a zero row and gives no gradient, as in :func:`embedding`.
    Forward-mode derivatives raise, on CUDA second ones too."""
    if idx.dtype != torch.int64:
        raise TypeError(f"scaled_embedding: int64 tokens, got {idx.dtype}")
    if weight.dtype not in _DTYPE_CODES:
        raise TypeError(f"scaled_embedding: an fp32, fp16 or bf16 table, got {weight.dtype}")
    if weight.dim() != 2 or not weight.numel():
        raise ValueError(f"scaled_embedding: the table must be [V, C] and not empty, got "
                         f"{tuple(weight.shape)}")
    if idx.device != weight.device:
        raise ValueError(f"scaled_embedding: tokens on {idx.device}, table on {weight.device}")
    if not abs(scale) <= torch.finfo(torch.float32).max:
        raise ValueError(f"scaled_embedding: scale must be finite in fp32, got {scale}")
    V = weight.shape[0]
    padding = -1
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"scaled_embedding: padding_idx {padding_idx} outside a table of "
                             f"{V} rows")
        padding = padding_idx % V
    if not weight.is_cuda:
        return _ScaledEmbeddingCPU.apply(idx, weight, float(scale), padding)
    return _C().scaled_embedding(idx, weight, scale, padding, isinstance(weight, torch.nn.Parameter))


# ------------------------------------------------------------------ rope
def rope_tables(T: int, D: int, theta: float, device) -> Tuple[torch.Tensor, torch.Tensor]:
    inv = 1.0 / (theta ** (torch.arange(0, D, 2, dtype=torch.float64, device=device) / D))
    ang = torch.arange(T, dtype=torch.float64, device=device)[:, None] * inv[None, :]
    return torch.cos(ang).float().contiguous(), torch.sin(ang).float().contiguous()


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, cos, sin):
        B, T, H, D = x.shape
        y = x.contiguous().clone()
        _C().rope(y, cos, sin, B * T, T, H, D, H * D, False)
        ctx.save_for_backward(cos, sin)
        return y

    @staticmethod
    def backward(ctx, dy):
        cos, sin = ctx.saved_tensors
        B, T, H, D = dy.shape
        dx = dy.contiguous().clone()
        _C().rope(dx, cos, sin, B * T, T, H, D, H * D, True)
        return dx, None, None


class _RopeQK(torch.autograd.Function):
    """Rotary embedding of the q and k heads of a fused [B, T, H+2Hkv, D]
    projection (v passes through)."""

    @staticmethod
    def forward(ctx, qkv, cos, sin, H, Hkv):
        B, T, Ht, D = qkv.shape
        y = qkv.contiguous().clone()
        _C().rope(y, cos, sin, B * T, T, H + Hkv, D, Ht * D, False)
        ctx.save_for_backward(cos, sin)
        ctx.heads = (H, Hkv)
        return y

    @staticmethod
    def backward(ctx, dy):
        cos, sin = ctx.saved_tensors
        H, Hkv = ctx.heads
        B, T, Ht, D = dy.shape
        dx = dy.contiguous().clone()
        _C().rope(dx, cos, sin, B * T, T, H + Hkv, D, Ht * D, True)
        return dx, None, None, None, None


def rope_qk(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, n_head: int,
            n_kv_head: int) -> torch.Tensor:
    """Rotate the first ``n_head + n_kv_head`` heads (q and k) of a fused
    [B, T, H+2Hkv, D] projection."""
    if qkv.is_cuda:
        return _RopeQK.apply(qkv, cos, sin, n_head, n_kv_head)
    n = n_head + n_kv_head
    return torch.cat([rope(qkv[:, :, :n], cos, sin), qkv[:, :, n:]], dim=2)


def attention_gqa(qkv: torch.Tensor, n_head: int, n_kv_head: int) -> torch.Tensor:
    """Causal GQA attention of a fused [B, T, H+2Hkv, D] projection -> [B, T, H*D]."""
    from . import attention

    return attention.attention_gqa(qkv, n_head, n_kv_head)


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Rotary embedding of ``x`` [B, T, H, D] (rotate-half convention)."""
    if x.is_cuda:
        return _Rope.apply(x, cos, sin)
    D = x.shape[-1]
    x1, x2 = x[..., : D // 2].float(), x[..., D // 2:].float()
    c = cos[: x.shape[1]][None, :, None, :]
    s = sin[: x.shape[1]][None, :, None, :]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1).to(x.dtype)


# ------------------------------------------------------------- attention
def causal_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """Causal attention over [B, T, H, D] q and [B, T, Hkv, D] k/v (GQA when
    Hkv < H); returns [B, T, H, D]."""
    from . import attention

    return attention.causal_attention(q, k, v)


def attention_qkv(qkv: torch.Tensor) -> torch.Tensor:
    """Causal attention of a fused [B, T, 3, H, D] projection -> [B, T, H*D]."""
    from . import attention

    return attention.attention_qkv(qkv)


def gelu_reference(x: torch.Tensor) -> torch.Tensor:
    return 0.5 * x * (1.0 + torch.erf(x / math.sqrt(2.0)))


def gelu_grad_reference(u: torch.Tensor) -> torch.Tensor:
    cdf = 0.5 * (1.0 + torch.erf(u / math.sqrt(2.0)))
    return cdf + u * torch.exp(-0.5 * u * u) / math.sqrt(2.0 * math.pi)
