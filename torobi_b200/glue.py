"""Fused decoder glue as differentiable ops: RMSNorm, rotary embedding and
SwiGLU, each one sm_100a kernel forward and one backward (csrc/glue.cu), and
what is read off the logits: the cross-entropy (csrc/loss.cu), the log
probabilities of given tokens with entropy and alternatives, and the
distillation from a teacher's alternatives (csrc/logits.cu).

RMSNorm is ``x * rsqrt(mean(x^2) + eps) * w`` (engine/src/interp.rs:312-319),
with a frozen gain; RoPE rotates the first half of each head against the
second (engine/src/interp.rs:350-388); SwiGLU is ``(g * sigmoid(g)) * u``
(lib/torobi/models/llama.rb:320-327).
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch
from torch.autograd.graph import increment_version

from .ops import _launch, _need_cuda, _ptr, _stream
from ._lib import TQ_DTYPE_BF16, TQ_DTYPE_F32, check, lib


def _bf16_contig(name: str, t: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16, got {t.dtype}")
    return t.contiguous()


def _bf16_tile(name: str, t: torch.Tensor) -> torch.Tensor:
    """For the kernels that copy tiles: contiguous, and on the 16-byte boundary
    that those copies start on (a view may lie off it: the gradient of a tensor
    joined behind an odd number of elements)."""
    t = _bf16_contig(name, t)
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, eps):
        _need_cuda("rms_norm", x=x, w=w)
        x = _bf16_contig("x", x)
        w = _bf16_contig("w", w)
        h = x.shape[-1]
        rows = x.numel() // h
        y = torch.empty_like(x)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        _launch("rmsnorm", lambda: lib().tq_rmsnorm_fwd(_ptr(x), _ptr(w), rows, h, float(eps),
                                                         _ptr(y), _ptr(rstd), _stream()))
        ctx.save_for_backward(x, w, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, rstd = ctx.saved_tensors
        dy = dy.contiguous()
        h = x.shape[-1]
        rows = x.numel() // h
        dx = torch.empty_like(x)
        _launch("rmsnorm", lambda: lib().tq_rmsnorm_bwd(_ptr(x), _ptr(w), _ptr(rstd), _ptr(dy),
                                                         None, rows, h, _ptr(dx), _stream()))
        return dx, None, None


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    """RMSNorm over the last axis; differentiable wrt x (the gain is frozen)."""
    return _RMSNorm.apply(x, w, eps)


class _AddRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, res, w, eps):
        _need_cuda("add_rms_norm", x=x, res=res, w=w)
        x = _bf16_contig("x", x)
        res = _bf16_contig("res", res)
        w = _bf16_contig("w", w)
        if res.shape != x.shape:
            raise ValueError(f"[add_rms_norm] res {tuple(res.shape)} must match x "
                             f"{tuple(x.shape)}")
        h = x.shape[-1]
        rows = x.numel() // h
        s = torch.empty_like(x)
        y = torch.empty_like(x)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        _launch("rmsnorm", lambda: lib().tq_add_rmsnorm_fwd(
            _ptr(x), _ptr(res), _ptr(w), rows, h, float(eps), _ptr(s), _ptr(y), _ptr(rstd),
            _stream()))
        ctx.save_for_backward(s, w, rstd)
        ctx.set_materialize_grads(False)
        return s, y

    @staticmethod
    def backward(ctx, ds, dy):
        s, w, rstd = ctx.saved_tensors
        if dy is None:
            return ds, ds, None, None
        dy = dy.contiguous()
        ds = ds.contiguous() if ds is not None else None
        h = s.shape[-1]
        rows = s.numel() // h
        dx = torch.empty_like(s)
        _launch("rmsnorm", lambda: lib().tq_rmsnorm_bwd(
            _ptr(s), _ptr(w), _ptr(rstd), _ptr(dy), _ptr(ds) if ds is not None else None, rows, h,
            _ptr(dx), _stream()))
        return dx, dx, None, None


def add_rms_norm(x: torch.Tensor, res: torch.Tensor, w: torch.Tensor, eps: float):
    """``(s, rms_norm(s, w, eps))`` with ``s = x + res`` in bf16: a pre-norm
    block's residual add and the norm after it in one kernel; its backward
    adds the residual stream's gradient inside the norm's (one kernel)."""
    return _AddRMSNorm.apply(x, res, w, eps)


class _RoPE(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, cos, sin, seq):
        _need_cuda("rope", x=x, cos=cos, sin=sin)
        x = _bf16_contig("x", x)
        tokens, heads, dim = x.shape[0] * x.shape[1], x.shape[2], x.shape[3]
        y = torch.empty_like(x)
        _launch("rope", lambda: lib().tq_rope(_ptr(x), tokens, heads, dim, seq, _ptr(cos),
                                               _ptr(sin), 0, _ptr(y), _stream()))
        ctx.save_for_backward(cos, sin)
        ctx.seq = seq
        return y

    @staticmethod
    def backward(ctx, dy):
        cos, sin = ctx.saved_tensors
        dy = dy.contiguous()
        tokens, heads, dim = dy.shape[0] * dy.shape[1], dy.shape[2], dy.shape[3]
        dx = torch.empty_like(dy)
        _launch("rope", lambda: lib().tq_rope(_ptr(dy), tokens, heads, dim, ctx.seq, _ptr(cos),
                                               _ptr(sin), 1, _ptr(dx), _stream()))
        return dx, None, None, None


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [batch, seq, heads, dim] bf16; cos/sin [seq, dim/2] f32."""
    return _RoPE.apply(x, cos.contiguous(), sin.contiguous(), x.shape[1])


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = True,
                      scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Grouped-query scaled dot-product attention (engine/src/interp.rs:405-432).

    q [batch, seq, heads, dim], k/v [batch, seq, kv_heads, dim] bf16 (dim 64
    or 128).  Returns o in q's layout and lse [batch, heads, seq] f32 (the
    natural-log log-sum-exp of each query row's scaled scores)."""
    _need_cuda("attention", q=q, k=k, v=v)
    q = _bf16_tile("q", q)
    k = _bf16_tile("k", k)
    v = _bf16_tile("v", v)
    if q.dim() != 4 or k.shape != v.shape or k.dim() != 4:
        raise ValueError(f"[attention] q {tuple(q.shape)}, k {tuple(k.shape)}, v "
                         f"{tuple(v.shape)}: want [batch, seq, heads, dim] and equal k/v")
    b, s, h, d = q.shape
    if k.shape[0] != b or k.shape[1] != s or k.shape[3] != d:
        raise ValueError(f"[attention] k {tuple(k.shape)} does not match q {tuple(q.shape)}")
    hk = k.shape[2]
    sc = float(scale) if scale is not None else d ** -0.5
    o = torch.empty_like(q)
    lse = torch.empty(b, h, s, dtype=torch.float32, device=q.device)
    _launch("attention", lambda: lib().tq_attention_fwd(
        _ptr(q), _ptr(k), _ptr(v), b, s, h, hk, d, sc, int(bool(causal)), _ptr(o), _ptr(lse),
        _stream()))
    return o, lse


def attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                       do: torch.Tensor, lse: torch.Tensor, causal: bool = True,
                       scale: float | None = None):
    """dq, dk, dv of ``attention_forward`` given the upstream gradient do
    (q's layout) and the forward's o and lse."""
    _need_cuda("attention", q=q, k=k, v=v, o=o, do=do, lse=lse)
    q, k, v, o = (_bf16_tile(n, t) for n, t in (("q", q), ("k", k), ("v", v), ("o", o)))
    do = _bf16_tile("do", do)
    if o.shape != q.shape or do.shape != q.shape:
        raise ValueError("[attention] o and do must have q's shape")
    b, s, h, d = q.shape
    hk = k.shape[2]
    if lse.dtype != torch.float32 or tuple(lse.shape) != (b, h, s):
        raise ValueError(f"[attention] lse must be f32 [{b}, {h}, {s}]")
    lse = lse.contiguous()
    sc = float(scale) if scale is not None else d ** -0.5
    nbytes = ctypes.c_size_t()
    check(lib().tq_attention_bwd_workspace_bytes(b, s, h, ctypes.byref(nbytes)))
    ws = torch.empty(max(1, nbytes.value), dtype=torch.uint8, device=q.device)
    dq = torch.empty_like(q)
    dk = torch.empty_like(k)
    dv = torch.empty_like(v)
    _launch("attention", lambda: lib().tq_attention_bwd(
        _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(do), _ptr(lse), b, s, h, hk, d, sc,
        int(bool(causal)), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), nbytes.value, _stream()))
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, scale):
        o, lse = attention_forward(q, k, v, causal, scale)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.causal, ctx.scale = causal, scale
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse = ctx.saved_tensors
        dq, dk, dv = attention_backward(q, k, v, o, do, lse, ctx.causal, ctx.scale)
        return dq, dk, dv, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = True,
              scale: float | None = None) -> torch.Tensor:
    """Differentiable grouped-query attention: q [batch, seq, heads, dim],
    k/v [batch, seq, kv_heads, dim] bf16, output in q's layout; the scale
    defaults to dim^-1/2 (engine/src/interp.rs:405-432)."""
    return _Attention.apply(q, k, v, causal, scale)


def document_spans(documents: torch.Tensor, prefix: torch.Tensor | None = None,
                   causal: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """The spans ``span_attention`` takes, of rows that pack documents:
    ``(first, last)`` int32 [batch, seq], position i seeing the positions
    ``first <= j < last``.

    documents int32 or int64 [batch, seq]: a run of equal ids is one document,
    a negative id is padding and sees nothing.  A position sees its document up
    to itself (``causal``) or whole; with ``prefix`` (int32 or int64 [batch,
    seq], causal only: the document's prompt length, at each of its positions)
    every position also sees its document's first ``prefix`` positions."""
    op = "document_spans"
    _one_device(op, documents=documents, prefix=prefix)
    if documents.dim() != 2 or documents.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"[{op}] documents must be int32 or int64 [batch, seq], got "
                         f"{documents.dtype} {tuple(documents.shape)}")
    if prefix is not None:
        if not causal:
            raise ValueError(f"[{op}] a prefix goes with causal=True")
        if prefix.shape != documents.shape or prefix.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"[{op}] prefix must be int32 or int64 {tuple(documents.shape)}, got "
                             f"{prefix.dtype} {tuple(prefix.shape)}")
        if prefix.dtype == torch.int64:
            prefix = prefix.clamp(max=2 ** 31 - 1).clamp_(min=0)
        prefix = prefix.to(torch.int32).contiguous()
    documents = documents.contiguous()
    b, s = documents.shape
    first = torch.empty(b, s, dtype=torch.int32, device=documents.device)
    last = torch.empty_like(first)
    _on(documents.device, "document_spans", lambda stream: lib().tq_document_spans(
        _ptr(documents), 8 * documents.element_size(), _ptr(prefix), b, s, int(bool(causal)),
        _ptr(first), _ptr(last), stream))
    return first, last


def _span_operands(op: str, q, k, v, first, last):
    q, k, v = (_bf16_tile(n, t) for n, t in (("q", q), ("k", k), ("v", v)))
    if q.dim() != 4 or k.shape != v.shape or k.dim() != 4:
        raise ValueError(f"[{op}] q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: "
                         "want [batch, seq, heads, dim] and equal k/v")
    b, s, _, d = q.shape
    if k.shape[0] != b or k.shape[1] != s or k.shape[3] != d:
        raise ValueError(f"[{op}] k {tuple(k.shape)} does not match q {tuple(q.shape)}")
    for name, t in (("first", first), ("last", last)):
        if t.dtype != torch.int32 or t.shape != (b, s):
            raise ValueError(f"[{op}] {name} must be int32 [{b}, {s}], got {t.dtype} "
                             f"{tuple(t.shape)}")
    return q, k, v, first.contiguous(), last.contiguous()


def _scale(scale: float | None, dim: int) -> float:
    return float(scale) if scale is not None else dim ** -0.5


def _span_forward(q, k, v, first, last, sc):
    b, s, h, d = q.shape
    o = torch.empty_like(q)
    lse = torch.empty(b, h, s, dtype=torch.float32, device=q.device)
    _on(q.device, "attention", lambda stream: lib().tq_span_attention_fwd(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), first.data_ptr(), last.data_ptr(), b, s, h,
        k.shape[2], d, sc, o.data_ptr(), lse.data_ptr(), stream))
    return o, lse


def _span_backward(q, k, v, first, last, o, do, lse, sc):
    b, s, h, d = q.shape
    hk = k.shape[2]
    nbytes = ctypes.c_size_t()
    check(lib().tq_span_attention_bwd_workspace_bytes(b, s, h, hk, ctypes.byref(nbytes)))
    ws = torch.empty(max(1, nbytes.value), dtype=torch.uint8, device=q.device)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    _on(q.device, "attention", lambda stream: lib().tq_span_attention_bwd(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), first.data_ptr(), last.data_ptr(),
        o.data_ptr(), do.data_ptr(), lse.data_ptr(), b, s, h, hk, d, sc, dq.data_ptr(),
        dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), nbytes.value, stream))
    return dq, dk, dv


def span_attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                           first: torch.Tensor, last: torch.Tensor,
                           scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``attention_forward`` with a span of keys for every query in place of
    the causal rule: query i of a row sees ``first[b, i] <= j < last[b, i]``
    (int32 [batch, seq], taken within [0, seq]); one that sees nothing gets o =
    0 and lse = -inf.  Returns o and lse."""
    op = "span_attention"
    _one_device(op, q=q, k=k, v=v, first=first, last=last)
    q, k, v, first, last = _span_operands(op, q, k, v, first, last)
    return _span_forward(q, k, v, first, last, _scale(scale, q.shape[3]))


def span_attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                            first: torch.Tensor, last: torch.Tensor, o: torch.Tensor,
                            do: torch.Tensor, lse: torch.Tensor, scale: float | None = None):
    """dq, dk, dv of ``span_attention_forward`` given the upstream gradient do
    (q's layout) and the forward's o and lse."""
    op = "span_attention"
    _one_device(op, q=q, k=k, v=v, first=first, last=last, o=o, do=do, lse=lse)
    q, k, v, first, last = _span_operands(op, q, k, v, first, last)
    o, do = _bf16_tile("o", o), _bf16_tile("do", do)
    if o.shape != q.shape or do.shape != q.shape:
        raise ValueError(f"[{op}] o and do must have q's shape")
    b, s, h, d = q.shape
    if lse.dtype != torch.float32 or tuple(lse.shape) != (b, h, s):
        raise ValueError(f"[{op}] lse must be f32 [{b}, {h}, {s}]")
    return _span_backward(q, k, v, first, last, o, do, lse.contiguous(), _scale(scale, d))


class _SpanAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, first, last, sc):
        o, lse = _span_forward(q, k, v, first, last, sc)
        ctx.save_for_backward(q, k, v, first, last, o, lse)
        ctx.scale = sc
        return o

    @staticmethod
    def backward(ctx, do):
        _once("span_attention")
        q, k, v, first, last, o, lse = ctx.saved_tensors
        do = _bf16_tile("do", do)
        return *_span_backward(q, k, v, first, last, o, do, lse, ctx.scale), None, None, None


def span_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, first: torch.Tensor,
                   last: torch.Tensor, scale: float | None = None) -> torch.Tensor:
    """Differentiable grouped-query attention in which query i sees the keys
    ``first[b, i] <= j < last[b, i]``: documents packed into one row, prompts
    seen in both directions, sliding windows, padding (``document_spans`` makes
    the first two).  q [batch, seq, heads, dim], k/v [batch, seq, kv_heads,
    dim] bf16, dim 64 or 128; first/last int32 [batch, seq]; output in q's
    layout; the scale defaults to dim^-1/2.  A query that sees nothing gets 0
    and passes no gradient.  What a query does not see still enters products
    with 0, so k and v, and q and the upstream gradient of queries that see
    nothing, must be finite (and v below 1e14 in size: probabilities are summed
    against a reference up to 2^60 below)."""
    op = "span_attention"
    _one_device(op, q=q, k=k, v=v, first=first, last=last)
    q, k, v, first, last = _span_operands(op, q, k, v, first, last)
    return _SpanAttention.apply(q, k, v, first, last, _scale(scale, q.shape[3]))


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, g, u):
        _need_cuda("swiglu", g=g, u=u)
        g = _bf16_contig("g", g)
        u = _bf16_contig("u", u)
        a = torch.empty_like(g)
        _launch("swiglu", lambda: lib().tq_swiglu_fwd(_ptr(g), _ptr(u), g.numel(), _ptr(a),
                                                       _stream()))
        ctx.save_for_backward(g, u)
        return a

    @staticmethod
    def backward(ctx, da):
        g, u = ctx.saved_tensors
        da = da.contiguous()
        dg = torch.empty_like(g)
        du = torch.empty_like(u)
        _launch("swiglu", lambda: lib().tq_swiglu_bwd(_ptr(g), _ptr(u), _ptr(da), g.numel(),
                                                       _ptr(dg), _ptr(du), _stream()))
        return dg, du


def swiglu(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    """(g * sigmoid(g)) * u."""
    return _SwiGLU.apply(g, u)


def _spend(ctx, op: str) -> None:
    """Ahead of a backward pass that writes over the logits it reads: once only.
    After it the logits' version moves on (``increment_version``), so that
    autograd refuses them to every other backward pass that needs them."""
    if ctx.inplace and ctx.spent:
        raise RuntimeError(f"[{op}] inplace=True wrote the gradient over the logits: this graph "
                           "cannot be run backward twice")
    ctx.spent = True


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, targets, inplace):
        _need_cuda("cross_entropy", z=z, targets=targets)
        z = _bf16_contig("logits", z)
        vocab = z.shape[-1]
        rows = z.numel() // vocab if vocab else 0
        t = targets.reshape(-1).to(torch.int64).contiguous()
        if t.numel() != rows:
            raise ValueError(f"targets hold {t.numel()} positions, logits {rows}")
        lse = torch.empty(rows, dtype=torch.float32, device=z.device)
        loss = torch.empty(rows, dtype=torch.float32, device=z.device)
        _launch("cross_entropy", lambda: lib().tq_cross_entropy_fwd(
            _ptr(z), _ptr(t), rows, vocab, vocab, _ptr(lse), _ptr(loss), _stream()))
        ctx.save_for_backward(z, t, lse)
        ctx.inplace = inplace
        ctx.spent = False
        return loss.view(z.shape[:-1])

    @staticmethod
    def backward(ctx, dloss):
        _spend(ctx, "cross_entropy")
        z, t, lse = ctx.saved_tensors
        vocab = z.shape[-1]
        rows = z.numel() // vocab
        dl = dloss.reshape(-1).float().contiguous()
        dz = z if ctx.inplace else torch.empty_like(z)
        _launch("cross_entropy", lambda: lib().tq_cross_entropy_bwd(
            _ptr(z), _ptr(t), _ptr(lse), rows, vocab, vocab, _ptr(dl), 1.0, _ptr(dz), _stream()))
        if ctx.inplace:
            increment_version(z)
        return dz, None, None


def cross_entropy(logits: torch.Tensor, targets: torch.Tensor,
                  inplace: bool = False) -> torch.Tensor:
    """Per-position ``logsumexp(logits) - logits[target]`` in f32 (no
    reduction, as the reference's loss node), logits bf16 [..., vocab].
    ``inplace=True`` writes the gradient over the logits in backward (no
    second [rows, vocab] buffer); the graph then cannot be run backward twice,
    nor another op of the same logits after it (autograd raises)."""
    return _CrossEntropy.apply(logits, targets, inplace)


_LOGIT_DTYPES = {torch.bfloat16: TQ_DTYPE_BF16, torch.float32: TQ_DTYPE_F32}


def _one_device(op: str, **tensors) -> None:
    """Every tensor (None: none) on one CUDA device."""
    first = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not (isinstance(t, torch.Tensor) and t.is_cuda):
            _need_cuda(op, **{name: t})
        if first is None:
            first = t.device
        elif t.device != first:
            raise ValueError(f"[{op}] {name} is on {t.device}, the others on {first}")


def _on(dev: torch.device, kind: str, call) -> None:
    """Launches ``call(stream)`` on the device's current stream.  Small calls
    wait for the host, so the device is switched only if it is another one and
    the stream is asked for by its handle."""
    if torch.cuda.current_device() == dev.index:
        stream = torch._C._cuda_getCurrentRawStream(dev.index)
        _launch(kind, lambda: call(stream))
    else:
        with torch.cuda.device(dev):
            _launch(kind, lambda: call(_stream()))


def _once(op: str) -> None:
    if torch.is_grad_enabled():  # in a backward pass: create_graph=True
        raise RuntimeError(f"[{op}] has no second derivative")


def _logit_rows(op: str, z: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """``(z, rows, vocab, pitch)``: the logits as rows of one pitch, read in
    place when their strides allow it (a slice of padded rows), else copied."""
    if z.dtype not in _LOGIT_DTYPES:
        raise ValueError(f"[{op}] logits must be bfloat16 or float32, got {z.dtype}")
    if z.dim() < 1 or z.shape[-1] == 0:
        raise ValueError(f"[{op}] logits need a non-empty last axis, got {tuple(z.shape)}")
    vocab = z.shape[-1]
    rows = z.numel() // vocab
    if z.is_contiguous():
        return z, rows, vocab, vocab
    pitch = None
    span = 1  # rows below the axis looked at
    if z.stride(-1) == 1 or vocab == 1:
        for size, stride in zip(reversed(z.shape[:-1]), reversed(z.stride()[:-1])):
            if size == 1:
                continue
            if pitch is None:
                pitch = stride
            elif stride != pitch * span:
                pitch = 0
                break
            span *= size
    if pitch is None:
        pitch = vocab  # one row
        if z.stride(-1) != 1 and vocab != 1:
            pitch = 0
    if rows and pitch < vocab:
        return z.contiguous(), rows, vocab, vocab
    return z, rows, vocab, max(pitch, vocab)


def _gradient_like(z: torch.Tensor, rows: int, vocab: int,
                   pitch: int) -> tuple[torch.Tensor, int]:
    """Room for a gradient of logits, and its rows' pitch: the least that moves
    on in the 32-byte chunks of memory as the logits' does (the kernels then read
    and write whole chunks; a slice of a larger tensor has a pitch far above its
    rows)."""
    least = vocab + (pitch - vocab) % (32 // z.element_size())
    if least == vocab:
        return torch.empty_like(z, memory_format=torch.contiguous_format), vocab
    wide = torch.empty(rows, least, dtype=z.dtype, device=z.device)
    return wide.view(*z.shape[:-1], least)[..., :vocab], least


def _positions(op: str, name: str, t: torch.Tensor, z: torch.Tensor) -> torch.Tensor:
    if t.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"[{op}] {name} must be int64 or int32, got {t.dtype}")
    if t.shape != z.shape[:-1]:
        raise ValueError(f"[{op}] {name} {tuple(t.shape)} must match the logits' positions "
                         f"{tuple(z.shape[:-1])}")
    return t if t.dtype == torch.int64 and t.is_contiguous() else t.to(torch.int64).contiguous()


def _temperature(op: str, temperature: float) -> float:
    t = float(temperature)
    if not (t > 0.0 and math.isfinite(t)):
        raise ValueError(f"[{op}] temperature must be positive and finite, got {temperature}")
    return t


def _upstream(g: torch.Tensor | None) -> torch.Tensor | None:
    if g is None or (g.dtype == torch.float32 and g.is_contiguous()):
        return g
    return g.float().contiguous()


def _positions_f32(lead: torch.Size, dev: torch.device) -> torch.Tensor:
    # Sizes one by one: torch parses them in half the time of a torch.Size.
    return (torch.empty(*lead, dtype=torch.float32, device=dev) if lead else
            torch.empty((), dtype=torch.float32, device=dev))


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` answers, per position (the alternatives None
    where none were asked for)."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor | None
    top_ids: torch.Tensor | None


def _token_logprobs(z, rows, vocab, pitch, tokens, top, temperature, want_stats):
    dev = z.device
    lead = z.shape[:-1]
    logprobs = _positions_f32(lead, dev)
    entropy = torch.empty_like(logprobs)
    top_logprobs = top_ids = None
    if top:
        top_logprobs = torch.empty(*lead, top, dtype=torch.float32, device=dev)
        top_ids = torch.empty(*lead, top, dtype=torch.int64, device=dev)
    stats = torch.empty(rows, 4, dtype=torch.float32, device=dev) if want_stats else None
    _on(dev, "token_logprobs", lambda stream: lib().tq_token_logprobs_fwd(
        _ptr(z), _LOGIT_DTYPES[z.dtype], _ptr(tokens), rows, vocab, pitch, temperature, top,
        _ptr(logprobs), _ptr(entropy), _ptr(stats), _ptr(top_logprobs), _ptr(top_ids), stream))
    return logprobs, entropy, top_logprobs, top_ids, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, tokens, top, temperature, inplace):
        z, rows, vocab, pitch = _logit_rows("token_logprobs", z)
        *out, stats = _token_logprobs(z, rows, vocab, pitch, tokens, top, temperature, True)
        ctx.save_for_backward(z, tokens, stats)
        ctx.shape, ctx.temperature, ctx.inplace = (rows, vocab, pitch), temperature, inplace
        ctx.spent = False
        if top:
            ctx.mark_non_differentiable(out[2], out[3])
        ctx.set_materialize_grads(False)
        return tuple(out)

    @staticmethod
    def backward(ctx, dlogprobs, dentropy, _top, _ids):
        _once("token_logprobs")
        _spend(ctx, "token_logprobs")
        z, tokens, stats = ctx.saved_tensors
        rows, vocab, pitch = ctx.shape
        dz, ld_out = (z, pitch) if ctx.inplace else _gradient_like(z, *ctx.shape)
        dlogprobs, dentropy = _upstream(dlogprobs), _upstream(dentropy)
        _on(z.device, "token_logprobs", lambda stream: lib().tq_token_logprobs_bwd(
            _ptr(z), _LOGIT_DTYPES[z.dtype], _ptr(tokens), _ptr(stats), rows, vocab, pitch,
            ctx.temperature, _ptr(dlogprobs), _ptr(dentropy), _ptr(dz), ld_out, stream))
        if ctx.inplace:
            increment_version(z)
        return dz, None, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0,
                   temperature: float = 1.0, inplace: bool = False) -> TokenLogprobs:
    """What a model thought of given tokens: ``q = softmax(logits /
    temperature)`` over the last axis of ``logits`` (bf16 or f32 [..., vocab]),
    read once, and per position

    ``logprobs`` f32 ``ln q[token]`` (0 where the token is outside [0, vocab):
    a padding position), ``entropy`` f32 ``-sum q ln q``, and the ``top`` (0 to
    128) most likely alternatives, most likely first, equal logits by lowest
    id: ``top_logprobs`` f32 and ``top_ids`` int64 [..., top] (None for none).

    Differentiable through logprobs and entropy.  ``inplace=True`` writes the
    gradient over the logits in backward, as ``cross_entropy`` does: a backward
    pass that needs the logits after it raises.  A -inf logit has probability 0;
    a position of nothing else has no distribution (log probabilities -inf,
    entropy 0, gradient 0)."""
    op = "token_logprobs"
    _one_device(op, logits=logits, tokens=tokens)
    tokens = _positions(op, "tokens", tokens, logits)
    temperature = _temperature(op, temperature)
    if not 0 <= top <= min(128, logits.shape[-1]):
        raise ValueError(f"[{op}] top must be 0 to 128 and at most the vocabulary "
                         f"({logits.shape[-1]}), got {top}")
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, int(top), temperature,
                                                   bool(inplace)))
    z, rows, vocab, pitch = _logit_rows(op, logits)
    return TokenLogprobs(*_token_logprobs(z, rows, vocab, pitch, tokens, int(top), temperature,
                                          False)[:4])


def _distillation(z, rows, vocab, pitch, teacher, targets, temperature, want_stats):
    dev = z.device
    ids, logits = teacher
    kl = _positions_f32(z.shape[:-1], dev)
    ce = None if targets is None else torch.empty_like(kl)
    stats = torch.empty(rows, 4, dtype=torch.float32, device=dev) if want_stats else None
    _on(dev, "distillation", lambda stream: lib().tq_distill_fwd(
        _ptr(z), _LOGIT_DTYPES[z.dtype], _ptr(ids), 8 * ids.element_size(), _ptr(logits),
        _LOGIT_DTYPES[logits.dtype], ids.shape[-1], _ptr(targets), rows, vocab, pitch,
        temperature, _ptr(kl), _ptr(ce), _ptr(stats), stream))
    return kl, ce, stats


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, ids, logits, targets, temperature, inplace):
        z, rows, vocab, pitch = _logit_rows("distillation", z)
        kl, ce, stats = _distillation(z, rows, vocab, pitch, (ids, logits), targets, temperature,
                                      True)
        ctx.save_for_backward(z, ids, logits, targets, stats)
        ctx.shape, ctx.temperature, ctx.inplace = (rows, vocab, pitch), temperature, inplace
        ctx.spent = False
        ctx.set_materialize_grads(False)
        return kl if ce is None else (kl, ce)

    @staticmethod
    def backward(ctx, dkl, dce=None):
        _once("distillation")
        _spend(ctx, "distillation")
        z, ids, logits, targets, stats = ctx.saved_tensors
        rows, vocab, pitch = ctx.shape
        dz, ld_out = (z, pitch) if ctx.inplace else _gradient_like(z, *ctx.shape)
        dkl, dce = _upstream(dkl), _upstream(dce)
        _on(z.device, "distillation", lambda stream: lib().tq_distill_bwd(
            _ptr(z), _LOGIT_DTYPES[z.dtype], _ptr(ids), 8 * ids.element_size(), _ptr(logits),
            _LOGIT_DTYPES[logits.dtype], ids.shape[-1], _ptr(targets), _ptr(stats), rows,
            vocab, pitch, ctx.temperature, _ptr(dkl), _ptr(dce), _ptr(dz), ld_out, stream))
        if ctx.inplace:
            increment_version(z)
        return dz, None, None, None, None, None


def distillation(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                 targets: torch.Tensor | None = None, temperature: float = 1.0,
                 inplace: bool = False):
    """The divergence from a teacher's top logits, per position and
    differentiable: ``kl = sum_i p_i (ln p_i - ln q[teacher_ids[i]])`` f32, with
    ``p = softmax(teacher_logits / temperature)`` over the position's k (1 to
    128) given alternatives and ``q = softmax(logits / temperature)`` over the
    whole vocabulary.

    logits bf16 or f32 [..., vocab]; teacher_ids int64 or int32 [..., k], an id
    outside [0, vocab) being no alternative (kl and its gradient are 0 where a
    position has none); teacher_logits bf16 or f32 [..., k], logits or log
    probabilities (``token_logprobs(..., top=k)`` gives both).  No gradient
    reaches the teacher.  With ``targets`` [...] the answer is ``(kl, ce)``:
    ``ce`` is the targets' cross-entropy at temperature 1, 0 where a target is
    outside [0, vocab); both gradients come from one pass.  A loss that mixes
    them is ``(1 - a) * ce + a * temperature**2 * kl``.  ``inplace=True``
    writes the gradient over the logits in backward, as ``cross_entropy`` does.
    Where the logits of a position are all -inf, kl and ce are +inf and the
    gradient is 0."""
    op = "distillation"
    _one_device(op, logits=logits, teacher_ids=teacher_ids, teacher_logits=teacher_logits,
                targets=targets)
    if teacher_ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"[{op}] teacher_ids must be int64 or int32, got {teacher_ids.dtype}")
    if teacher_logits.dtype not in _LOGIT_DTYPES:
        raise ValueError(f"[{op}] teacher_logits must be bfloat16 or float32, got "
                         f"{teacher_logits.dtype}")
    if (teacher_ids.shape != teacher_logits.shape or teacher_ids.dim() != logits.dim()
            or teacher_ids.shape[:-1] != logits.shape[:-1]):
        raise ValueError(f"[{op}] teacher_ids {tuple(teacher_ids.shape)} and teacher_logits "
                         f"{tuple(teacher_logits.shape)} must be [..., k] over the logits' "
                         f"positions {tuple(logits.shape[:-1])}")
    temperature = _temperature(op, temperature)
    ids, given = teacher_ids.contiguous(), teacher_logits.detach().contiguous()
    if targets is not None:
        targets = _positions(op, "targets", targets, logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _Distillation.apply(logits, ids, given, targets, temperature, bool(inplace))
    z, rows, vocab, pitch = _logit_rows(op, logits)
    kl, ce, _ = _distillation(z, rows, vocab, pitch, (ids, given), targets, temperature, False)
    return kl if ce is None else (kl, ce)
