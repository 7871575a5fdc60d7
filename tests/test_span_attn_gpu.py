"""span_attention and document_spans (csrc/span_attn.cu) against their definitions
in 64 bits.

Tolerances.  The operands are bf16 and the products are summed in f32; what is
rounded on the way is P (and dS) to bf16 before a product and the result: each
half a step, 2^-8 of the value at most.  |o| errs by at most
2^-8 (sum_j p_j |v_j| + |o|), plus the exponentials' errors and f32 sums, for
which a tenth of that bound is ample.  For the gradients the same holds with
the products' magnitudes: dv by 2^-8 (sum_i p_ij |do_i| + |dv|), dq and dk by
2^-8 times sums of |dS| |k| (or |q|), where dS's own error comes from its
rounding and from delta = sum do o, whose o is rounded to bf16:
p_ij 2^-8 sum_d |do o|.  lse: f32, within 1e-4 (room for exponentials of
relative error 7.5e-5, the polynomial of attn.cu; log is 1-Lipschitz here)
plus 4 steps of f32 of its own size and of the scores'.
"""
from __future__ import annotations

import math

import pytest

R = 2.0 ** -8 * 1.1


def _spans_reference(documents, prefix, causal):
    """first, last [batch][seq] by walking the runs."""
    firsts, lasts = [], []
    for r, row in enumerate(documents):
        first, last = [0] * len(row), [0] * len(row)
        i = 0
        while i < len(row):
            j = i
            while j < len(row) and row[j] == row[i]:
                j += 1
            for t in range(i, j):
                first[t] = i
                if row[i] < 0:
                    last[t] = i
                elif not causal:
                    last[t] = j
                else:
                    last[t] = t + 1
                    if prefix is not None:
                        last[t] = max(t + 1, min(i + max(prefix[r][t], 0), j))
            i = j
        firsts.append(first)
        lasts.append(last)
    return firsts, lasts


def _random_documents(rnd, batch, seq, mean):
    rows = []
    for _ in range(batch):
        row, n = [], 0
        while len(row) < seq:
            length = max(1, int(rnd.expovariate(1 / mean)))
            ident = -1 if rnd.random() < 0.15 else n
            row += [ident] * length
            n += 1
        rows.append(row[:seq])
    return rows


@pytest.mark.gpu
@pytest.mark.parametrize("ids", ["int32", "int64"])
@pytest.mark.parametrize("seq, mean", [(1, 1), (2, 1), (31, 3), (200, 40), (1025, 1), (4096, 300),
                                       (4099, 900), (9001, 20000), (12289, 5)])
def test_document_spans(cuda, seq, mean, ids):
    import random

    import torch

    from torobi_b200 import glue

    rnd = random.Random(seq * 7 + len(ids))
    rows = _random_documents(rnd, 3, seq, mean)
    rows[0] = [0] * seq
    prefix = [[rnd.choice([-3, 0, 1, 5, 60, 10 ** 9]) for _ in row] for row in rows]
    d = torch.tensor(rows, dtype=getattr(torch, ids), device=cuda)
    pre = torch.tensor(prefix, dtype=torch.int32, device=cuda)
    for causal, use in ((True, None), (True, pre), (False, None)):
        first, last = glue.document_spans(d, use, causal=causal)
        f, l = _spans_reference(rows, None if use is None else prefix, causal)
        assert first.tolist() == f and last.tolist() == l
    # Prompt lengths past 32 bits are lengths still, as are those below zero.
    wide = torch.where(pre == 10 ** 9, 2 ** 32 + 1, torch.where(pre < 0, -2 ** 33 + 7, pre.long()))
    for a, b in zip(glue.document_spans(d, wide), glue.document_spans(d, pre)):
        assert torch.equal(a, b)


def _reference(q, k, v, first, last, scale, do=None):
    """o, lse, the gradients and the bounds' sums, in 64 bits, a head at a time."""
    import torch

    b, s, h, d = q.shape
    hk = k.shape[2]
    qd, kd, vd = q.double(), k.double(), v.double()
    j = torch.arange(s, device=q.device)
    see = (j >= first[:, :, None].clamp(0, s)) & (j < last[:, :, None].clamp(0, s))
    o, ob = torch.zeros_like(qd), torch.zeros_like(qd)
    lse = torch.empty(b, h, s, dtype=torch.float64, device=q.device)
    g = {n: torch.zeros_like(t) for n, t in (("dq", qd), ("dk", kd), ("dv", vd))}
    gb = {n: torch.zeros_like(t) for n, t in g.items()}
    for hi in range(h):
        kv = hi // (h // hk)
        x = (qd[:, :, hi] @ kd[:, :, kv].transpose(1, 2)) * scale
        x = x.masked_fill(~see, float("-inf"))
        lse[:, hi] = x.logsumexp(2)
        p = torch.where(see.any(2, keepdim=True), x.softmax(2), 0.0)
        o[:, :, hi] = p @ vd[:, :, kv]
        ob[:, :, hi] = p @ vd[:, :, kv].abs()
        if do is None:
            continue
        up = do[:, :, hi].double()
        dp = up @ vd[:, :, kv].transpose(1, 2)
        delta = (up * o[:, :, hi]).sum(2, keepdim=True)
        wide = (up * o[:, :, hi]).abs().sum(2, keepdim=True)
        ds = p * (dp - delta) * scale
        dsb = (ds.abs() + p * wide * scale)
        g["dq"][:, :, hi] = ds @ kd[:, :, kv]
        gb["dq"][:, :, hi] = dsb @ kd[:, :, kv].abs()
        g["dk"][:, :, kv] += ds.transpose(1, 2) @ qd[:, :, hi]
        gb["dk"][:, :, kv] += dsb.transpose(1, 2) @ qd[:, :, hi].abs()
        g["dv"][:, :, kv] += p.transpose(1, 2) @ up
        gb["dv"][:, :, kv] += p.transpose(1, 2) @ up.abs()
    return o, ob, lse, g, gb


def _inputs(cuda, seed, b, s, h, hk, d, gain=1.0):
    import torch

    g = torch.Generator(device=cuda).manual_seed(seed)
    mk = lambda n, f=1.0: (torch.randn(b, s, n, d, device=cuda, generator=g) * f).bfloat16()  # noqa: E731
    return mk(h, gain), mk(hk), mk(hk), mk(h)


def _check(q, k, v, do, first, last, scale=None):
    import torch

    from torobi_b200 import device_status, glue

    sc = scale if scale is not None else q.shape[-1] ** -0.5
    o, lse = glue.span_attention_forward(q, k, v, first, last, scale)
    ro, ob, rl, g, gb = _reference(q, k, v, first, last, sc, do)
    none = (last.clamp(0, q.shape[1]) <= first.clamp(0, q.shape[1]))
    assert ((o.double() - ro).abs() <= R * (ob + ro.abs()) + 1e-30).all()
    assert (o[none] == 0).all() and (lse.transpose(1, 2)[none] == float("-inf")).all()
    seen = ~none[:, None, :].expand_as(lse)
    top = (q.double().abs().amax() * k.double().abs().amax() * q.shape[-1] * sc).item()
    assert ((lse.double() - rl).abs()[seen]
            <= 1e-4 + 2.0 ** -22 * (rl.abs()[seen] + top)).all()
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = glue.span_attention(*leaves, first, last, scale)
    assert torch.equal(out, o)
    got = torch.autograd.grad(out, leaves, do)
    for name, t in zip(("dq", "dk", "dv"), got):
        # 1e-6: where the gradient is zero (one visible key), rounding is left.
        off = (t.double() - g[name]).abs() - R * (gb[name] + g[name].abs()) - 1e-6 * top
        assert off.max().item() <= 0, (name, off.max().item())
    assert (got[0][none] == 0).all()
    assert device_status() == 0
    return o, got


def _spans(cuda, documents, prefix=None, causal=True):
    import torch

    from torobi_b200 import glue

    d = torch.tensor(documents, dtype=torch.int32, device=cuda)
    p = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=cuda)
    return glue.document_spans(d, p, causal=causal)


CASES = [
    # batch, seq, heads, kv_heads, dim, mean document, prefix, causal
    (1, 1, 2, 1, 64, 1, False, True),
    (1, 7, 2, 2, 128, 2, False, True),
    (2, 128, 4, 2, 64, 30, False, True),
    (2, 129, 4, 1, 128, 30, True, True),
    (1, 200, 4, 2, 64, 60, False, False),
    (3, 255, 6, 6, 64, 10, True, True),
    (1, 300, 8, 1, 128, 500, True, True),
    (2, 513, 14, 2, 64, 100, False, True),
    (2, 640, 2, 2, 128, 64, False, False),
    (1, 1000, 4, 4, 64, 250, True, True),
    (1, 1537, 8, 2, 128, 700, False, True),
    (2, 2048, 4, 1, 64, 40, False, True),
    # Query heads a key/value head: those a tile holds, and rows it leaves over.
    (1, 200, 3, 1, 64, 50, False, True),
    (1, 200, 5, 1, 128, 50, True, True),
    (2, 150, 11, 1, 64, 50, False, True),
    (1, 300, 12, 1, 128, 90, False, True),
    (1, 300, 14, 1, 64, 90, True, True),
    (1, 260, 16, 1, 128, 60, False, False),
    (1, 130, 34, 2, 64, 60, False, True),
    (1, 260, 32, 1, 64, 60, True, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_packed_documents(cuda, case):
    import random

    b, s, h, hk, d, mean, pre, causal = case
    rnd = random.Random(s)
    docs = _random_documents(rnd, b, s, mean)
    prefix = None
    if pre:
        prefix = [[0] * s for _ in range(b)]
        for r, row in enumerate(docs):
            for i in range(s):
                start = i == 0 or row[i] != row[i - 1]
                prefix[r][i] = rnd.randrange(0, max(2, mean)) if start else prefix[r][i - 1]
    first, last = _spans(cuda, docs, prefix, causal)
    _check(*_inputs(cuda, s + d, b, s, h, hk, d), first, last)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kind", ["window", "padding_tiles", "nothing", "far_apart", "outside",
                                  "one_key", "random", "sharp"])
def test_spans_of_other_shapes(cuda, kind, dim):
    """Spans that no document makes: sliding windows, whole tiles that see
    nothing, neighbouring tiles far apart, bounds outside the row, one key
    each, arbitrary ones; and scores that move the running maximum."""
    import torch

    b, s, h, hk = 2, 777, 4, 2
    i = torch.arange(s, device=cuda, dtype=torch.int32).expand(b, s).contiguous()
    gain = 1.0
    if kind == "window":
        first, last = (i - 150).clamp(min=0), i + 1
    elif kind == "padding_tiles":
        first, last = torch.zeros_like(i), i + 1
        dead = ((i >= 128) & (i < 400)) | (i >= 650)
        first, last = torch.where(dead, i, first), torch.where(dead, i, last)
    elif kind == "nothing":
        first, last = i.clone(), i.clone()
        last[1] += 1
    elif kind == "far_apart":  # neighbouring query tiles at opposite ends
        even = (i // 128) % 2 == 0
        first = torch.where(even, 0, s - 100).to(torch.int32)
        last = torch.where(even, 70, s).to(torch.int32)
    elif kind == "outside":
        first, last = i - 2000, i + 2000
        first[0, ::3] = 5000
        last[1, ::5] = -7
    elif kind == "one_key":
        first = (i * 37) % s
        last = first + 1
    elif kind == "random":
        g = torch.Generator(device=cuda).manual_seed(1)
        first = torch.randint(0, s, (b, s), device=cuda, generator=g, dtype=torch.int32)
        last = first + torch.randint(-50, 300, (b, s), device=cuda, generator=g, dtype=torch.int32)
    else:
        first, last, gain = (i // 300) * 300, i + 1, 12.0
    _check(*_inputs(cuda, 5 + dim, b, s, h, hk, dim, gain), first.contiguous(),
           last.contiguous())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_one_causal_document_is_causal_attention(cuda, dim):
    """One document a row: what ``attention`` gives, to the rounding of both
    (their exponentials differ by up to 7.5e-5, which may move a rounding)."""
    import torch

    from torobi_b200 import glue

    q, k, v, do = _inputs(cuda, 3, 2, 400, 8, 2, dim)
    first, last = _spans(cuda, [[0] * 400] * 2)
    a = [t.clone().requires_grad_() for t in (q, k, v)]
    c = [t.clone().requires_grad_() for t in (q, k, v)]
    x, y = glue.span_attention(*a, first, last), glue.attention(*c, True)
    for s, t in zip((x, *torch.autograd.grad(x, a, do)), (y, *torch.autograd.grad(y, c, do))):
        assert ((s - t).abs().max() / t.abs().max()).item() <= 1e-2


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_a_nan_query_is_nan_alone(cuda, dim):
    """A NaN in one query: its output and log-sum-exp are NaN, no other's are."""
    import torch

    from torobi_b200 import glue

    b, s, h, hk = 2, 300, 4, 2
    first, last = _spans(cuda, [[0] * 130 + [1] * 170] * b)
    q, k, v, _ = _inputs(cuda, 77, b, s, h, hk, dim)
    want, wlse = glue.span_attention_forward(q, k, v, first, last)
    q[1, 200, 3, 7] = float("nan")
    o, lse = glue.span_attention_forward(q, k, v, first, last)
    assert o[1, 200, 3].isnan().all() and lse[1, 3, 200].isnan()
    o[1, 200, 3], lse[1, 3, 200] = want[1, 200, 3], wlse[1, 3, 200]
    assert torch.equal(o, want) and torch.equal(lse, wlse)


@pytest.mark.gpu
def test_span_attention_past_32_bit_offsets(cuda):
    """Three rows of 262144 positions, 32 heads of 128: the last row's queries,
    outputs and gradients lie past 2^31 elements.  It gives what it gives alone."""
    import torch

    from torobi_b200 import glue

    b, s, h, hk, d = 3, 262144, 32, 8, 128
    g = torch.Generator(device=cuda).manual_seed(3)

    def mk(n):
        return torch.randn(b, s, n, d, device=cuda, dtype=torch.bfloat16, generator=g)

    q, k, v, do = mk(h), mk(hk), mk(hk), mk(h)
    i = torch.arange(s, device=cuda, dtype=torch.int32)
    docs = torch.stack([i // 190, i // 77, i // 301])
    docs[2, -50:] = -1
    first, last = glue.document_spans(docs)
    o, lse = glue.span_attention_forward(q, k, v, first, last)
    grads = glue.span_attention_backward(q, k, v, first, last, o, do, lse)
    alone = [t[2:].clone() for t in (q, k, v, first, last)]
    o1, lse1 = glue.span_attention_forward(*alone)
    assert torch.equal(o[2:], o1) and torch.equal(lse[2:], lse1)
    grads1 = glue.span_attention_backward(*alone, o1, do[2:].clone(), lse1)
    for a, c in zip(grads, grads1):
        assert torch.equal(a[2:], c)
    assert (o[2, -50:] == 0).all() and (grads[0][2, -50:] == 0).all()
    # And its last document, in a row of its own: |o| errs by R (sum p |v| + |o|).
    at = (s - 51) // 301 * 301
    part = [t[2:, at:s - 50].contiguous() for t in (q, k, v)]
    one = torch.zeros(1, s - 50 - at, dtype=torch.int32, device=cuda)
    o2, _ = _check(*part, do[2:, at:s - 50].contiguous(), *glue.document_spans(one))
    off = (o2.double() - o[2:, at:s - 50].double()).abs().max().item()
    assert off <= 2 * R * 2 * part[2].abs().max().item()


@pytest.mark.gpu
def test_a_document_does_not_see_its_neighbours(cuda):
    """A document's outputs and gradients are the same whatever stands beside
    it (bit for bit where no warp's 32 rows hold two documents: a warp moves
    its rows' running maxima together)."""
    import torch

    from torobi_b200 import glue

    q, k, v, do = _inputs(cuda, 8, 1, 500, 4, 2, 128)
    docs = [[0] * 128 + [1] * 192 + [2] * 180]
    first, last = _spans(cuda, docs)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = glue.span_attention(*leaves, first, last)
    want = [o.detach(), *torch.autograd.grad(o, leaves, do)]
    for t in (q, k, v, do):
        t[:, :128] = torch.randn_like(t[:, :128]) * 3
        t[:, 320:] = 0
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = glue.span_attention(*leaves, first, last)
    for a, c in zip(want, [o.detach(), *torch.autograd.grad(o, leaves, do)]):
        assert torch.equal(a[:, 128:320], c[:, 128:320])


@pytest.mark.gpu
def test_span_gradient_against_differences(cuda):
    """The gradients against central differences of the 64-bit definition
    along random directions."""
    import torch

    from torobi_b200 import glue

    q, k, v, do = _inputs(cuda, 9, 1, 60, 2, 1, 64)
    first, last = _spans(cuda, [[0] * 25 + [-1] * 5 + [1] * 30])
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(glue.span_attention(*leaves, first, last), leaves, do)
    gen = torch.Generator(device=cuda).manual_seed(2)
    _, _, _, g, gb = _reference(q, k, v, first, last, 0.125, do)
    for n, name in enumerate(("dq", "dk", "dv")):
        way = torch.randn(got[n].shape, device=cuda, generator=gen, dtype=torch.float64)
        step = 1e-4

        def loss(at):
            args = [t.double() for t in (q, k, v)]
            args[n] = args[n] + at * way
            o, *_ = _reference(*args, first, last, 0.125)
            return (o * do.double()).sum()

        diff = (loss(step) - loss(-step)) / (2 * step)
        along = (got[n].double() * way).sum()
        # Each element errs within its bound; the difference's own error is of
        # order step^2 and far below.
        assert (along - diff).abs() <= (R * (gb[name] + g[name].abs()) * way.abs()).sum() + 1e-5


@pytest.mark.gpu
def test_span_attention_repeats_captured_and_on_another_stream(cuda):
    """The same bits every time: run again, on a side stream, and from two
    captured graphs replayed on new inputs."""
    import torch

    from torobi_b200 import glue

    docs = torch.tensor([[0] * 100 + [1] * 300 + [-1] * 13, [5] * 413], device=cuda)
    sets = [_inputs(cuda, 30 + i, 2, 413, 4, 2, 64) for i in range(3)]

    def work(q, k, v, do):
        first, last = glue.document_spans(docs)
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = glue.span_attention(*leaves, first, last)
        return [o.detach(), *torch.autograd.grad(o, leaves, do), first, last]

    want = [work(*x) for x in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work(*sets[0])
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(other, want[0]):
        assert torch.equal(a, c)
    graphs = []
    for i in range(2):
        static = [t.clone() for t in sets[i]]
        with torch.cuda.stream(side):
            work(*static)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work(*static)
        graphs.append((graph, static, out))
    for turn in range(2):
        for i, (graph, static, out) in enumerate(graphs):
            for t, n in zip(static, sets[i + turn]):
                t.copy_(n)
            graph.replay()
        for i, (graph, static, out) in enumerate(graphs):
            for a, c in zip(out, want[i + turn]):
                assert torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 1300, 8, 2, 128), (2, 700, 14, 2, 64), (4, 2100, 4, 4, 64)],
                         ids=str)
def test_every_run_writes_every_value(cuda, shape):
    """Outputs, gradients and workspace full of NaN before each of 20 runs of
    many tiles an SM, with and without idle gaps: always the same bits."""
    import ctypes
    import random

    import torch

    from torobi_b200 import device_status, glue
    from torobi_b200._lib import lib

    b, s, h, hk, d = shape
    first, last = _spans(cuda, _random_documents(random.Random(s), b, s, 200))
    q, k, v, do = _inputs(cuda, s, b, s, h, hk, d, 6.0)
    o, lse = glue.span_attention_forward(q, k, v, first, last)
    want = o, lse, *glue.span_attention_backward(q, k, v, first, last, o, do, lse)
    got = [torch.empty_like(t) for t in want]
    need = ctypes.c_size_t()
    assert lib().tq_span_attention_bwd_workspace_bytes(b, s, h, hk, ctypes.byref(need)) == 0
    ws = torch.empty(need.value, dtype=torch.uint8, device=cuda)
    stream = torch.cuda.current_stream().cuda_stream
    at = [t.data_ptr() for t in (q, k, v, first, last)]
    for run in range(20):
        for t in got:
            t.fill_(float("nan"))
        ws.fill_(255)
        if run % 3 == 0:
            torch.cuda.synchronize()
        assert lib().tq_span_attention_fwd(*at, b, s, h, hk, d, d ** -0.5, got[0].data_ptr(),
                                           got[1].data_ptr(), stream) == 0
        assert lib().tq_span_attention_bwd(
            *at, o.data_ptr(), do.data_ptr(), lse.data_ptr(), b, s, h, hk, d, d ** -0.5,
            *[t.data_ptr() for t in got[2:]], ws.data_ptr(), need.value, stream) == 0
        assert all(torch.equal(a, c) for a, c in zip(got, want))
    assert device_status() == 0


def _outgrown(q, k, first, last, scale):
    """How often each query's sum over a 64-key tile passes 2^60 against the
    reference it has by then (the largest score of the first tile it sees, then
    of the tile where that happened), int [batch, heads, seq], in 64 bits."""
    import torch

    b, s, h, _ = q.shape
    group = h // k.shape[2]
    x = torch.einsum("bihd,bjhd->bhij", q.double(),
                     k.double().repeat_interleave(group, 2)) * (scale / math.log(2))
    j = torch.arange(s, device=q.device)
    see = (j >= first[:, None, :, None]) & (j < last[:, None, :, None])
    x = x.masked_fill(~see, float("-inf"))
    m = torch.full((b, h, s), float("-inf"), device=q.device, dtype=torch.float64)
    times = torch.zeros(b, h, s, dtype=torch.int64, device=q.device)
    for at in range(0, s, 64):
        tile = x[..., at:at + 64]
        top = tile.amax(3)
        m = torch.where(m == float("-inf"), top, m)
        total = torch.exp2(tile - m.nan_to_num(neginf=0.0)[..., None]).sum(3)
        over = total > 2.0 ** 60
        times += over
        m = torch.where(over, top, m)
    return times


def _climbing(cuda, seed, b, s, h, hk, d, docs=None):
    """Operands whose scores climb along a row: the keys lie along one direction,
    further out every 100 positions, a third of the queries with it, a third
    twice as far, a third at right angles (beside noise): a step is 70 powers of
    two for the first third."""
    import torch

    q, k, v, do = (t.float() for t in _inputs(cuda, seed, b, s, h, hk, d, 0.5))
    i = torch.arange(s, device=cuda)
    way = torch.ones(d, device=cuda)
    way[::2] = -1.0
    step = 70 * math.log(2) * d ** 0.5 / d
    far = (i // 100 % 5) * step  # and back to the start, where little weight is left
    k = 0.25 * k + far[None, :, None, None] * way
    rows = (i[:, None] + torch.arange(h, device=cuda)) % 3
    q = q + rows[None, :, :, None] * way
    return q.bfloat16(), k.bfloat16(), v.bfloat16(), do.bfloat16()


def _check_steep(q, k, v, do, first, last):
    """As _check, for scores so large that their own rounding counts.  A score is
    a sum of D products in the tensor cores' f32, 16 at a time, each sum off by at
    most a step (2^-23) of the products' sum `top`, and 4 steps more are the
    scale's, its product's and the reference's; a probability errs by as much of
    itself, twice (by its score and by the log-sum-exp)."""
    import torch

    from torobi_b200 import device_status, glue

    d = q.shape[-1]
    sc = d ** -0.5
    ro, ob, rl, g, gb = _reference(q, k, v, first, last, sc, do)
    top = (q.double().norm(dim=3).amax() * k.double().norm(dim=3).amax() * sc).item()
    score = (d / 16 + 4) * 2.0 ** -23 * top
    r = R + 2 * score
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o, lse = glue.span_attention_forward(q, k, v, first, last)
    got = glue.span_attention_backward(q, k, v, first, last, o, do, lse)
    assert ((o.double() - ro).abs() <= r * (ob + ro.abs()) + 1e-30).all()
    assert ((lse.double() - rl).abs()
            <= score + 2.0 ** -20 + 4 * 2.0 ** -24 * (rl.abs() + top)).all()
    again = glue.span_attention(*leaves, first, last)
    assert torch.equal(again, o)
    for a, c in zip(torch.autograd.grad(again, leaves, do), got):
        assert torch.equal(a, c)
    for name, t in zip(("dq", "dk", "dv"), got):
        off = (t.double() - g[name]).abs() - r * (gb[name] + g[name].abs()) - 1e-6 * top
        assert off.max().item() <= 0, (name, off.max().item())
    assert device_status() == 0


STEEP = [
    # batch, seq, heads, kv_heads, dim, positions a document (0: the whole row)
    (1, 500, 4, 2, 64, 0),
    (1, 500, 4, 2, 128, 0),
    (2, 777, 8, 2, 128, 0),
    (2, 777, 14, 2, 64, 333),     # documents that start inside a tile of others
    (1, 1025, 3, 1, 64, 420),
    (1, 900, 6, 6, 128, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", STEEP, ids=str)
def test_scores_that_outgrow_their_reference(cuda, case):
    """Scores that climb past 2^60 of the first tile's maximum, several times
    along a row, for some rows of a warp and not for others: O in tensor memory
    is scaled in place and the tile done again."""
    import torch

    b, s, h, hk, d, length = case
    i = torch.arange(s, device=cuda, dtype=torch.int32).expand(b, s)
    first = (i // length * length if length else torch.zeros_like(i)).contiguous()
    last = (i + 1).contiguous()
    q, k, v, do = _climbing(cuda, 50 + s, b, s, h, hk, d)
    times = _outgrown(q, k, first, last, d ** -0.5)
    # The first third of queries two to four times, the last third never.
    for n in (0, 1, 2, 3):
        assert (times == n).sum().item() >= 20, (n, times.unique(return_counts=True))
    _check_steep(q, k, v, do, first, last)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_steep_random_scores(cuda, dim):
    """Queries 40 times as long as a trained model's: hundreds of rows outgrow
    their reference, here and there."""
    import torch

    b, s, h, hk = 2, 777, 4, 2
    i = torch.arange(s, device=cuda, dtype=torch.int32).expand(b, s).contiguous()
    first, last = (i // 300) * 300, i + 1
    q, k, v, do = _inputs(cuda, 5 + dim, b, s, h, hk, dim, 40.0)
    assert (_outgrown(q, k, first, last, dim ** -0.5) > 0).sum().item() >= 200
    _check_steep(q, k, v, do, first, last)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("jump", [100, 130, 140, 150, 165])
def test_small_weights_outlive_a_jump(cuda, jump, dim):
    """A second tile of keys 50 powers of two above the first, a third `jump`
    above it with values of 0: o is the second's share, 2^(50 - jump) of its
    values, a normal number although the factor that takes O to the third tile's
    reference is not one."""
    import torch

    from torobi_b200 import glue

    b, s, h, hk = 2, 192, 4, 2
    q, k, v, _ = (t.float() for t in _inputs(cuda, 90 + dim, b, s, h, hk, dim))
    way = torch.ones(dim, device=cuda)
    way[::2] = -1.0
    i = torch.arange(s, device=cuda)
    step = math.log(2) / dim ** 0.5  # a power of two
    height = torch.where(i < 64, 0.0, torch.where(i < 128, 50.0, float(jump))) * step
    q = way.expand_as(q).bfloat16()
    k = (height[None, :, None, None] * way + 0.0 * k).bfloat16()
    v = torch.where(i[None, :, None, None] < 128, v, 0.0).bfloat16()
    last = (i + 1).to(torch.int32).expand(b, s).contiguous()
    first = torch.zeros_like(last)
    o, lse = glue.span_attention_forward(q, k, v, first, last)
    ro, ob, rl, _, _ = _reference(q, k, v, first, last, dim ** -0.5)
    assert 2.0 ** (45 - jump) < ro[:, 128:].abs().amax() < 2.0 ** (58 - jump)
    score = (dim / 16 + 4) * 2.0 ** -23 * jump * math.log(2) * 1.01  # as in _check_steep
    assert ((o.double() - ro).abs() <= (R + 2 * score) * (ob + ro.abs())).all()
    assert ((lse.double() - rl).abs()
            <= score + 2.0 ** -20 + 4 * 2.0 ** -24 * (rl.abs() + jump)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 1300, 8, 2, 128), (2, 700, 14, 2, 64)], ids=str)
def test_rows_that_outgrow_their_reference_repeat(cuda, shape):
    """The same over outputs full of NaN, 20 times: always the same bits."""
    import torch

    from torobi_b200 import device_status
    from torobi_b200._lib import lib

    b, s, h, hk, d = shape
    i = torch.arange(s, device=cuda, dtype=torch.int32).expand(b, s).contiguous()
    first, last = (i // 450) * 450, i + 1
    q, k, v, _ = _climbing(cuda, s, b, s, h, hk, d)
    assert (_outgrown(q, k, first, last, d ** -0.5) > 1).sum().item() >= 200
    stream = torch.cuda.current_stream().cuda_stream
    want = None
    for run in range(20):
        o = torch.full_like(q, float("nan"))
        lse = torch.full((b, h, s), float("nan"), device=cuda)
        if run % 3 == 0:
            torch.cuda.synchronize()
        assert lib().tq_span_attention_fwd(
            *[t.data_ptr() for t in (q, k, v, first, last)], b, s, h, hk, d, d ** -0.5,
            o.data_ptr(), lse.data_ptr(), stream) == 0
        if want is None:
            want = o, lse
            assert torch.isfinite(o).all() and torch.isfinite(lse).all()
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    assert device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_every_visible_key_counts_once(cuda, case):
    """Queries of zero weigh all their keys alike: the sum is their number
    exactly, the log-sum-exp its logarithm (log2f is off by at most a step, its
    product with ln 2 by half a step each of the factor and the result: 2 steps
    of 2^-23), and o the mean of their values (sums in f32 and one rounding)."""
    import random

    import torch

    from torobi_b200 import glue

    b, s, h, hk, d, mean, _, causal = case
    docs = _random_documents(random.Random(s + 1), b, s, mean)
    first, last = _spans(cuda, docs, None, causal)
    q, k, v, _ = _inputs(cuda, s + d + 1, b, s, h, hk, d)
    o, lse = glue.span_attention_forward(torch.zeros_like(q), k, v, first, last)
    n = (last - first).double()
    want = n.log()[:, None].expand_as(lse)
    fine = want.isfinite()
    assert torch.equal(lse[~fine].double(), want[~fine])
    assert ((lse.double() - want).abs()[fine] <= 2 * 2.0 ** -23 * want[fine]).all()
    sums = torch.zeros(b, s + 1, hk, d, device=cuda, dtype=torch.float64)
    size = sums.clone()
    sums[:, 1:] = v.double().cumsum(1)
    size[:, 1:] = v.double().abs().cumsum(1)

    def mean_of(c):
        at = lambda i: c.gather(1, i.long()[..., None, None].expand(b, s, hk, d))  # noqa: E731
        return ((at(last) - at(first)) / n.clamp(min=1)[..., None, None]).repeat_interleave(
            h // hk, 2)

    ro = mean_of(sums)
    # s additions in f32, and two roundings more, beside that to bf16.
    assert ((o.double() - ro).abs()
            <= 2.0 ** -8 * 1.01 * ro.abs() + (s + 2) * 2.0 ** -24 * mean_of(size) + 1e-30).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_log_sum_exp_to_f32(cuda, case):
    """lse by its own arithmetic.  A score is a sum of D products in the tensor
    cores' f32 (16 at a time, each sum off by at most a step, 2^-23, of the
    products' sum so far; 4 steps for the scale, its product and the reference's);
    the exponentials are off by 2^-22, their sum by half a step an addition (n /
    64 tiles, 16 in a tile, 3 joins), log2f by a step and the last sum and
    product by half a step each of the result."""
    import random

    import torch

    from torobi_b200 import glue

    b, s, h, hk, d, mean, _, causal = case
    docs = _random_documents(random.Random(s + 2), b, s, mean)
    first, last = _spans(cuda, docs, None, causal)
    q, k, v, _ = _inputs(cuda, s + d + 2, b, s, h, hk, d)
    sc = d ** -0.5
    _, lse = glue.span_attention_forward(q, k, v, first, last)
    _, _, want, _, _ = _reference(q, k, v, first, last, sc)
    kk = k.double().abs().repeat_interleave(h // hk, 2)
    size = torch.einsum("bihd,bjhd->bhij", q.double().abs(), kk).amax(3) * sc
    fine = want.isfinite()
    assert torch.equal(lse[~fine].double(), want[~fine])
    tol = ((d / 16 + 4) * 2.0 ** -23 * size + 2.0 ** -22 + (s / 64 + 19) * 2.0 ** -24
           + 4 * 2.0 ** -24 * (want.abs() + size))
    off = ((lse.double() - want).abs() - tol)[fine]
    assert off.numel() == 0 or off.max().item() <= 0, off.max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_one_causal_document_is_causal_attention_everywhere(cuda, dim):
    """One document a row against ``attention``, element by element: both err by
    at most R of their products' sizes and of the value (see above; R has room for
    the polynomial of attn.cu, 7.5e-5), so they differ by at most twice that."""
    import torch

    from torobi_b200 import glue

    q, k, v, do = _inputs(cuda, 4, 2, 413, 8, 2, dim)
    first, last = _spans(cuda, [[0] * 413] * 2)
    ro, ob, _, g, gb = _reference(q, k, v, first, last, dim ** -0.5, do)
    a = [t.clone().requires_grad_() for t in (q, k, v)]
    c = [t.clone().requires_grad_() for t in (q, k, v)]
    x, y = glue.span_attention(*a, first, last), glue.attention(*c, True)
    want = (ro, g["dq"], g["dk"], g["dv"])
    size = (ob, gb["dq"], gb["dk"], gb["dv"])
    for n, (s, t) in enumerate(zip((x, *torch.autograd.grad(x, a, do)),
                                   (y, *torch.autograd.grad(y, c, do)))):
        # 1e-4: dq and dk of the first position, where zero is what is left.
        assert ((s - t).double().abs()
                <= 2 * R * (size[n] + want[n].abs()) + (1e-4 if n in (1, 2) else 0)).all(), n


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["span_attention", "attention"])
def test_operands_and_gradients_off_the_16_byte_boundary(cuda, op):
    """Views that start at an odd element, and a result joined behind an odd
    number of elements, whose gradient then is such a view: the bits of the
    aligned call."""
    import torch

    from torobi_b200 import glue

    q, k, v, do = _inputs(cuda, 12, 2, 150, 4, 2, 64)
    first, last = _spans(cuda, [[0] * 150] * 2)

    def call(*t):
        return glue.span_attention(*t, first, last) if op == "span_attention" else glue.attention(*t)

    def off(t):
        room = torch.empty(t.numel() + 1, device=cuda, dtype=t.dtype)
        room[1:] = t.flatten()
        return room[1:].view_as(t)

    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = call(*leaves)
    want = [o, *torch.autograd.grad(o, leaves, do)]
    leaves = [off(t).requires_grad_() for t in (q, k, v)]
    assert all(t.data_ptr() % 16 for t in leaves)
    o = call(*leaves)
    head = torch.ones(3, device=cuda, dtype=torch.bfloat16)
    joined = torch.cat([head, o.flatten()])
    up = torch.cat([head, do.flatten()])
    for a, c in zip([o, *torch.autograd.grad(joined, leaves, up)], want):
        assert torch.equal(a, c)


@pytest.mark.gpu
def test_two_streams_at_once(cuda):
    """Forward and backward on two streams side by side, of different shapes,
    beside one another for a while: the bits of each alone."""
    import torch

    from torobi_b200 import device_status, glue

    work = []
    for n, (b, s, h, hk, d) in enumerate([(2, 1300, 8, 2, 128), (3, 900, 14, 2, 64)]):
        docs = torch.arange(s, device=cuda).expand(b, s) // (170 + 60 * n)
        work.append((*_inputs(cuda, 60 + n, b, s, h, hk, d), docs.contiguous()))

    def run(q, k, v, do, docs):
        first, last = glue.document_spans(docs)
        o, lse = glue.span_attention_forward(q, k, v, first, last)
        return o, lse, *glue.span_attention_backward(q, k, v, first, last, o, do, lse)

    want = [run(*w) for w in work]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = ([], [])
    for _ in range(15):
        for n in (0, 1):
            with torch.cuda.stream(streams[n]):
                got[n].append(run(*work[n]))
    torch.cuda.synchronize()
    for n in (0, 1):
        for out in got[n]:
            assert all(torch.equal(a, c) for a, c in zip(out, want[n]))
    assert device_status() == 0


@pytest.mark.gpu
def test_span_refusals(cuda):
    import torch

    from torobi_b200 import TqError, glue

    q, k, v, _ = _inputs(cuda, 1, 2, 16, 4, 2, 64)
    f = torch.zeros(2, 16, dtype=torch.int32, device=cuda)
    for bad in (lambda: glue.span_attention(q, k, v, f.long(), f),
                lambda: glue.span_attention(q, k, v, f[:1], f),
                lambda: glue.span_attention(q, k, v, f, f.cpu()),
                lambda: glue.span_attention(q.float(), k, v, f, f),
                lambda: glue.span_attention(q, k[:, :8], v[:, :8], f, f),
                lambda: glue.span_attention(q, k, v[:, :8], f, f),
                lambda: glue.document_spans(f[0]), lambda: glue.document_spans(f.float()),
                lambda: glue.document_spans(f, f[:1]),
                lambda: glue.document_spans(f, f.float()),
                lambda: glue.document_spans(f, f, causal=False)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TqError, match="scale"):
        glue.span_attention(q, k, v, f, f, scale=-1.0)
    with pytest.raises(TqError, match="head dim"):
        glue.span_attention(q[..., :32], k[..., :32], v[..., :32], f, f)
    # Strided spans and empty batches are taken.
    wide = torch.zeros(2, 32, dtype=torch.int32, device=cuda)
    o, lse = glue.span_attention_forward(q, k, v, wide[:, ::2], wide[:, ::2])
    assert (o == 0).all() and (lse == float("-inf")).all()
    o, _ = glue.span_attention_forward(q[:0], k[:0], v[:0], f[:0], f[:0])
    assert o.shape == (0, 16, 4, 64)
    assert glue.document_spans(f[:, :0])[0].shape == (2, 0)


P = 1 << 20  # an aligned stand-in address; nothing is dereferenced


def test_span_entry_points_refuse_on_the_host():
    import ctypes

    import torobi_b200 as tq

    L = tq.lib()

    def fwd(first=P, last=P, heads=4, kv=2, dim=64, scale=0.1, out=P, batch=2, seq=129):
        return L.tq_span_attention_fwd(P, P, P, first, last, batch, seq, heads, kv, dim, scale,
                                       out, P, None)

    def said():
        return L.tq_last_error().decode()

    assert fwd(first=None) == 1 and "null" in said()
    assert fwd(last=None) == 1 and "null" in said()
    assert fwd(first=P + 2) == 3 and "first and last" in said()
    assert fwd(kv=3) == 1 and fwd(dim=96) == 2 and fwd(scale=0.0) == 1 and fwd(out=P + 8) == 3
    assert fwd(batch=0, first=None, last=None, out=None) == 0

    need, plain = ctypes.c_size_t(), ctypes.c_size_t()
    # 4 heads over 2: 64-row tiles of 32 positions, five of them; per tile and
    # two heads 64 rows of two statistics, per tile 64 spans and two bounds.
    assert L.tq_span_attention_bwd_workspace_bytes(2, 129, 4, 2, ctypes.byref(need)) == 0
    assert need.value == 2 * 5 * (2 * 64 * 8 + 64 * 8 + 8)
    # 11 heads over one: too few rows would be filled, a tile holds one head.
    assert L.tq_span_attention_bwd_workspace_bytes(1, 65, 11, 1, ctypes.byref(plain)) == 0
    assert plain.value == 2 * (11 * 64 * 8 + 64 * 8 + 8)
    assert L.tq_span_attention_bwd_workspace_bytes(2, 129, 4, 3, ctypes.byref(plain)) == 1

    def bwd(ws_bytes=need.value, ws=P, first=P):
        return L.tq_span_attention_bwd(P, P, P, first, P, P, P, P, 2, 129, 4, 2, 64, 0.125, P, P,
                                       P, ws, ws_bytes, None)

    assert bwd(ws_bytes=need.value - 4) == 1 and "workspace" in said()
    assert bwd(ws=P + 16) == 3 and bwd(ws=None) == 1 and bwd(first=None) == 1

    def spans(docs=P, bits=32, prefix=None, batch=2, seq=8, first=P, last=P):
        return L.tq_document_spans(docs, bits, prefix, batch, seq, 1, first, last, None)

    assert spans(bits=16) == 2 and spans(docs=None) == 1 and spans(last=None) == 1
    assert spans(docs=P + 2) == 3 and spans(docs=P + 4, bits=64) == 3 and spans(prefix=P + 1) == 3
    assert spans(seq=-1) == 1 and spans(seq=1 << 31) == 1
    assert spans(batch=0, docs=None) == 0 and spans(seq=0, docs=None) == 0
