"""token_logprobs and distillation (csrc/logits.cu) against their definitions
in 64 bits.

Tolerances, from the arithmetic.  Let e = 2^-24 (half a step of f32).  A term
2^x of a row's sum has the error of x (three roundings, 3 e |x|), of the
hardware's 2^x (2^-22 = 4 e) and of the additions it passes through: at most
V / 512 + 32 in its thread's chain, and 20 in the joins.  Terms with a large
|x| weigh nothing, |x| 2^x <= 1 at its largest, so a sum's relative error is at
most E(V) = (V / 512 + 64) e.  A log probability is a difference of such a
logarithm (absolute error E + a rounding of itself) and one product: absolute
error E + 4 e (|ln q| + ln V).  The entropy is a quotient of two such sums and
a logarithm: 3 E (1 + ln V) + 4 e H.  A gradient multiplies 2^x by factors that
carry the same relative errors: (E + 8 e (|x| + ln V)) of its largest term,
plus half a step of its type (bf16: 2^-8).
"""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALF = {"bf16": 2.0 ** -8, "f32": E}
NINF = float("-inf")


def _dtype(name):
    import torch

    return {"bf16": torch.bfloat16, "f32": torch.float32}[name]


def _sum_err(vocab):
    return (vocab / 512 + 64) * E


def _logits(cuda, rows, vocab, dtype, seed, std=2.5, pad=0, shift=0):
    """[rows, vocab] with row pitch vocab + pad, starting `shift` elements past
    a 32-byte boundary."""
    import torch

    g = torch.Generator(device=cuda).manual_seed(seed)
    room = torch.zeros(rows * (vocab + pad) + shift, device=cuda, dtype=_dtype(dtype))
    z = room[shift:].view(rows, vocab + pad)
    z.copy_((torch.randn(rows, vocab + pad, device=cuda, generator=g) * std).to(z.dtype))
    return z[:, :vocab]


def _tokens(cuda, rows, vocab, seed):
    import torch

    g = torch.Generator(device=cuda).manual_seed(1000 + seed)
    t = torch.randint(0, vocab, (rows,), device=cuda, generator=g)
    if rows > 2:
        t[1] = -1
        t[2] = vocab
    return t


def _reference(z, tokens, top, temperature):
    import torch

    x = z.double() / temperature
    m = x.max(1, keepdim=True).values
    m = torch.where(m == NINF, 0.0, m)
    e = (x - m).exp()
    s = e.sum(1, keepdim=True)
    logq = (x - m) - s.log()
    dead = (s == 0).squeeze(1)
    logq = torch.where(dead[:, None], NINF, logq)
    q = torch.where(dead[:, None], 0.0, e / s)
    ent = -torch.where(q > 0, q * logq, torch.where(q.isnan(), q, 0.0)).sum(1)
    known = (tokens >= 0) & (tokens < z.shape[1])
    lp = torch.where(known, logq.gather(1, tokens.clamp(0, z.shape[1] - 1)[:, None]).squeeze(1), 0.0)
    ids = (z.double() + 0.0).sort(dim=1, descending=True, stable=True).indices[:, :top]
    return lp, ent, logq.gather(1, ids), ids, q, logq, known


def _same_specials(got, want):
    import torch

    # A log probability past f32's range is -inf there.
    want[want < -torch.finfo(torch.float32).max] = NINF
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got[inf].double(), want[inf])
    return want.isfinite()


def _check_forward(z, tokens, top, temperature, scale_err=False):
    import torch

    from torobi_b200 import glue

    vocab = z.shape[1]
    r = glue.token_logprobs(z, tokens, top=top, temperature=temperature)
    lp, ent, tlp, ids, *_ = _reference(z, tokens, top, temperature)
    lnv = math.log(vocab) + 1
    if scale_err:  # 1/T is rounded: every ln q errs by as much of the spread it came from
        lnv += float((lp.abs() + tlp.abs().amax(1)).nan_to_num(0, 0, 0).clamp(max=1e30).max())
    for name, got, want, tol in (
            ("logprobs", r.logprobs, lp, lambda w: _sum_err(vocab) + 4 * E * (w.abs() + lnv)),
            ("entropy", r.entropy, ent, lambda w: 3 * _sum_err(vocab) * lnv + 4 * E * w.abs()),
            ("top", r.top_logprobs, tlp, lambda w: _sum_err(vocab) + 4 * E * (w.abs() + lnv))):
        if got is None:
            assert top == 0
            continue
        fine = _same_specials(got, want)
        off = (got.double() - want).abs()[fine] - tol(want)[fine]
        assert off.numel() == 0 or off.max().item() <= 0, (name, off.max().item())
    if top:
        assert r.top_ids.dtype == torch.int64 and torch.equal(r.top_ids, ids)
    return r


@pytest.mark.parametrize("temperature", [1e-4, 1e-2, 50.0, 1e6, 1e30])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_token_logprobs_far_temperatures(cuda, dtype, temperature):
    """Temperatures at which the scaled logits leave every usual range, with
    ruled-out tokens: the distribution goes from one-hot to uniform."""
    import torch

    z = _logits(cuda, 7, 2003, dtype, 21).contiguous()
    z[:, ::5] = NINF
    z[3] = torch.finfo(z.dtype).min
    z[4, 1] = 200.0
    t = torch.tensor([1, 2, 3, 4, 1, 6, 7], device=cuda)
    r = _check_forward(z, t, 6, temperature, scale_err=True)
    assert (r.entropy >= 0).all() and torch.isfinite(r.entropy).all()


FORWARD = [
    # rows, vocab, dtype, top, temperature, pad, shift
    (1, 1, "bf16", 1, 1.0, 0, 0),
    (3, 2, "f32", 2, 1.0, 0, 1),
    (5, 15, "bf16", 15, 1.0, 0, 3),         # inside one or two chunks
    (4, 16, "bf16", 4, 0.5, 0, 0),
    (4, 33, "bf16", 33, 1.0, 0, 9),
    (7, 129, "f32", 128, 2.0, 0, 5),
    (37, 1000, "bf16", 8, 1.0, 0, 0),
    (37, 1001, "bf16", 8, 0.7, 0, 0),       # every row starts elsewhere in its chunk
    (37, 1001, "f32", 5, 1.3, 7, 2),
    (64, 1024, "bf16", 0, 1.0, 0, 0),
    (64, 1024, "bf16", 128, 1.0, 64, 0),
    (3, 32003, "bf16", 64, 1.0, 61, 1),     # shared by a cluster
    (2, 32003, "f32", 20, 1.0, 0, 0),
    (1, 151936, "bf16", 20, 1.0, 0, 0),
    (1, 151936, "f32", 128, 1.0, 0, 0),
    (700, 8193, "bf16", 3, 1.0, 0, 0),
    (640, 151936, "f32", 1, 1.0, 0, 0),     # many rows, chunk maxima beyond one CTA's
    (2, 1000003, "bf16", 50, 1.0, 0, 0),
]


@pytest.mark.parametrize("case", FORWARD, ids=str)
def test_token_logprobs_forward(cuda, case):
    rows, vocab, dtype, top, temperature, pad, shift = case
    z = _logits(cuda, rows, vocab, dtype, 1, pad=pad, shift=shift)
    _check_forward(z, _tokens(cuda, rows, vocab, 1), top, temperature)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [40, 5000, 151936])
@pytest.mark.parametrize("rows", [13, 600])
def test_token_logprobs_odd_rows(cuda, dtype, vocab, rows):
    """Rows built against the selection: equal logits, few values, ordered
    logits, a run of large ones in one place, masked rows, zeros of both signs."""
    import torch

    if rows * vocab > 600 * 5000:
        rows = 13
    z = _logits(cuda, rows, vocab, dtype, 2).contiguous()
    lowest = torch.finfo(z.dtype).min
    index = torch.arange(vocab, device=cuda)
    z[0] = 0.5                                       # all equal
    z[1] = (index % 3).to(z.dtype)                   # three values
    z[2] = (index / vocab * 8).to(z.dtype)           # rising
    z[3] = (-index / vocab * 8).to(z.dtype)          # falling
    z[4] = NINF
    z[4, vocab // 2:vocab // 2 + 5] = 1.0            # five tokens allowed
    z[5] = NINF                                      # nothing allowed
    z[6] = lowest                                    # nothing allowed, the finite way
    z[7] = lowest
    z[7, 7:10] = -3.0
    z[8] = -0.0
    z[8, ::2] = 0.0
    z[9, vocab // 3:vocab // 3 + max(8, vocab // 40)] = 9.0   # a stretch of equal large ones
    z[10] = lowest
    z[10, -1] = -lowest                              # the type's whole range apart
    z[11] += 300.0
    z[12] = -1000.0
    z[12, 3] = 0.0                                   # one certain token
    if rows > 13:
        z[13] = lowest                               # the finite way, and ruled out
        z[13, 1::2] = NINF
        z[14] = -1e35                                # far below any logit, and uneven
        z[14, vocab // 2] = -9e34
        z[15, ::2] = -1e34                           # such entries beside ordinary ones
    t = torch.randint(0, vocab, (rows,), device=cuda)
    t[4] = vocab // 2 + 1
    t[12] = 3
    if rows > 13:
        t[13] = 2 * (vocab // 4)
    for top in (1, 7, min(128, vocab)):
        r = _check_forward(z, t, top, 1.0)
        assert torch.isfinite(r.entropy).all() and (r.entropy >= 0).all()
        assert (r.logprobs <= 0).all()


def test_token_logprobs_nan_and_inf_rows(cuda):
    """A NaN or +inf makes its own row NaN; ids stay within the vocabulary, the
    other rows are untouched."""
    import torch

    from torobi_b200 import glue

    z = _logits(cuda, 6, 3001, "bf16", 3).contiguous()
    clean = z.clone()
    z[1, 17] = float("nan")
    z[3, 2000] = float("inf")
    z[4] = float("nan")
    t = torch.full((6,), 5, device=cuda)
    r, c = (glue.token_logprobs(x, t, top=9) for x in (z, clean))
    for i in range(6):
        if i in (1, 3, 4):
            assert r.logprobs[i].isnan() and r.entropy[i].isnan()
            assert ((r.top_ids[i] >= 0) & (r.top_ids[i] < 3001)).all()
        else:
            for a, b in zip(r, c):
                assert torch.equal(a[i], b[i])
    assert r.top_ids[1, 0] == 17 and r.top_ids[3, 0] == 2000


def _logprob_grad(z, tokens, temperature, g, h):
    import torch

    *_, q, logq, known = _reference(z, tokens, 0, temperature)
    ent = -torch.where(q > 0, q * logq, 0.0).sum(1, keepdim=True)
    g = torch.where(known, g.double(), 0.0)[:, None]
    h = h.double()[:, None]
    lq = torch.where(q > 0, logq, 0.0)
    dz = -q * (g + h * (lq + ent))
    at = tokens.clamp(0, z.shape[1] - 1)[:, None]
    dz.scatter_add_(1, at, g)
    size = q * (g.abs() + h.abs() * (lq.abs() + ent))
    size.scatter_add_(1, at, g.abs())
    x = torch.where(q > 0, lq.abs(), 0.0)
    return dz / temperature, size / temperature, x


def _check_gradient(got, want, size, x, dtype):
    vocab = want.shape[1]
    rel = _sum_err(vocab) + 8 * E * (x + math.log(vocab) + 1)
    bound = rel * size + HALF[dtype] * want.abs() * (1 + 2 ** -6) + 1e-38
    off = (got.double() - want).abs() - bound
    assert off.max().item() <= 0, (off.max().item(), want.abs().max().item())


BACKWARD = [
    # rows, vocab, dtype, temperature, pad, shift
    (1, 1, "f32", 1.0, 0, 0),
    (3, 15, "bf16", 1.0, 0, 3),
    (5, 33, "bf16", 0.5, 0, 1),
    (37, 1001, "bf16", 1.0, 0, 0),
    (37, 1001, "f32", 2.0, 7, 3),
    (64, 1024, "bf16", 1.0, 64, 0),
    (2, 151936, "bf16", 1.0, 0, 0),
    (3, 32003, "f32", 0.7, 61, 1),
    (700, 4099, "bf16", 1.0, 5, 0),
]


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("case", BACKWARD, ids=str)
def test_token_logprobs_gradient(cuda, case, inplace):
    import torch

    from torobi_b200 import glue

    rows, vocab, dtype, temperature, pad, shift = case
    z = _logits(cuda, rows, vocab, dtype, 4, pad=pad, shift=shift)
    if rows > 4:
        z[4, ::3] = NINF
        z[3] = NINF
    before = z.clone()
    tokens = _tokens(cuda, rows, vocab, 4)
    g = torch.randn(rows, device=cuda)
    h = torch.randn(rows, device=cuda)
    leaf = z.detach().requires_grad_()
    r = glue.token_logprobs(leaf, tokens, temperature=temperature, inplace=inplace)
    dz, = torch.autograd.grad((r.logprobs, r.entropy), leaf, (g, h))
    assert dz.shape == z.shape and dz.dtype == z.dtype
    assert inplace == (dz.data_ptr() == z.data_ptr())
    if not inplace:
        assert torch.equal(z, before)
    if rows > 4:
        assert (dz[3] == 0).all()
        before[3] = 0  # no distribution: nothing to compare
        dz = dz.clone()
        dz[3] = _logprob_grad(before, tokens, temperature, g, h)[0][3].to(dz.dtype)
    _check_gradient(dz, *_logprob_grad(before, tokens, temperature, g, h), dtype)


def test_token_logprobs_gradient_of_one_output(cuda):
    """Through logprobs alone and through entropy alone; the alternatives pass
    none; a second backward over logits that were overwritten is refused."""
    import torch

    from torobi_b200 import glue

    z = _logits(cuda, 9, 500, "f32", 5).contiguous()
    tokens = _tokens(cuda, 9, 500, 5)
    one, none = torch.ones(9, device=cuda), torch.zeros(9, device=cuda)
    for pick, g, h in ((0, one, none), (1, none, one)):
        leaf = z.clone().requires_grad_()
        r = glue.token_logprobs(leaf, tokens, top=3)
        assert not r.top_logprobs.requires_grad
        r[pick].sum().backward()
        _check_gradient(leaf.grad, *_logprob_grad(z, tokens, 1.0, g, h), "f32")
    leaf = z.clone().requires_grad_()
    work = leaf * 1.0
    r = glue.token_logprobs(work, tokens, inplace=True)
    torch.autograd.grad(r.logprobs.sum(), work, retain_graph=True)
    with pytest.raises(RuntimeError, match="backward twice"):
        torch.autograd.grad(r.logprobs.sum(), work)


def test_token_logprobs_gradient_against_differences(cuda):
    """The f32 gradient against central differences of the 64-bit definition."""
    import torch

    from torobi_b200 import glue

    z = _logits(cuda, 3, 40, "f32", 6).contiguous()
    tokens = torch.tensor([0, 39, 17], device=cuda)
    g = torch.randn(3, device=cuda)
    h = torch.randn(3, device=cuda)
    leaf = z.clone().requires_grad_()
    r = glue.token_logprobs(leaf, tokens, temperature=1.5)
    dz, = torch.autograd.grad((r.logprobs, r.entropy), leaf, (g, h))
    step = 1e-5

    def loss(x):
        lp, ent, *_ = _reference(x, tokens, 0, 1.5)
        return lp * g.double() + ent * h.double()

    for j in range(40):
        up, down = z.double().clone(), z.double().clone()
        up[:, j] += step
        down[:, j] -= step
        diff = (loss(up) - loss(down)) / (2 * step)
        # step^2 / 6 of third derivatives (at most 50 here), the rounding of
        # the difference, and the gradient's own error.
        assert ((dz[:, j].double() - diff).abs() <= 50 * step ** 2 + 1e-9 + 200 * E).all()


def test_rows_past_32_bit_offsets(cuda):
    """14200 x 151936 logits, over 2^31: the last rows, forward and (in place)
    backward, give what they give alone (where clusters share a row, so that
    its f32 sums come in another order)."""
    import torch

    from torobi_b200 import glue

    rows, vocab, n = 14200, 151936, 3
    g = torch.Generator(device=cuda).manual_seed(8)
    z = torch.randn(rows, vocab, device=cuda, dtype=torch.bfloat16, generator=g)
    tokens = torch.randint(0, vocab, (rows,), device=cuda, generator=g)
    tail = z[-n:].clone()
    _check_forward(tail, tokens[-n:], 8, 1.0)
    with torch.no_grad():
        top = glue.token_logprobs(z, tokens, top=8)
    ids, given = top.top_ids, top.top_logprobs * 0.5

    def run(z, t, ids, given):
        leaf = z.requires_grad_()
        r = glue.token_logprobs(leaf, t, top=8)
        kl, ce = glue.distillation(leaf, ids, given, targets=t, temperature=2.0, inplace=True)
        dz, = torch.autograd.grad(kl.sum() + ce.sum(), leaf)
        return [x.detach()[-n:] for x in (r.top_ids, r.logprobs, r.entropy, kl, ce, dz)]

    many = run(z, tokens, ids, given)
    few = run(tail, tokens[-n:], ids[-n:], given[-n:])
    assert torch.equal(many[0], few[0])
    lnv = math.log(vocab) + 1
    for a, b in zip(many[1:5], few[1:5]):
        assert ((a - b).abs() <= 6 * _sum_err(vocab) * lnv + 8 * E * (b.abs() + lnv)).all()
    # The gradient: two roundings to bf16, and where something is given a
    # difference of shares of 1.
    a, b = many[5].double(), few[5].double()
    room = torch.zeros_like(b)
    room.scatter_(1, torch.cat([ids[-n:], tokens[-n:, None]], 1), 8 * _sum_err(vocab))
    assert ((a - b).abs() <= 2 * HALF["bf16"] * 1.1 * b.abs() + room).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gradient_with_another_pitch(cuda, dtype):
    """dlogits in rows of another pitch than the logits': elements go one by
    one, with the same results, and nothing past a row is written."""
    import torch

    from torobi_b200._lib import check, lib

    rows, vocab = 5, 1003
    z = _logits(cuda, rows, vocab, dtype, 7).contiguous()
    tokens = _tokens(cuda, rows, vocab, 7)
    code = 1 if dtype == "bf16" else 0
    f = lambda *s: torch.zeros(*s, device=cuda)  # noqa: E731
    lp, ent, stats = f(rows), f(rows), f(rows, 4)
    g, h = torch.randn(rows, device=cuda), torch.randn(rows, device=cuda)
    s = torch.cuda.current_stream().cuda_stream
    check(lib().tq_token_logprobs_fwd(z.data_ptr(), code, tokens.data_ptr(), rows, vocab, vocab,
                                      1.0, 0, lp.data_ptr(), ent.data_ptr(), stats.data_ptr(),
                                      None, None, s))
    outs = []
    for pitch in (vocab, vocab + 6):
        dz = torch.full((rows, pitch), 7.0, device=cuda, dtype=z.dtype)
        check(lib().tq_token_logprobs_bwd(
            z.data_ptr(), code, tokens.data_ptr(), stats.data_ptr(), rows, vocab, vocab, 1.0,
            g.data_ptr(), h.data_ptr(), dz.data_ptr(), pitch, s))
        assert (dz[:, vocab:] == 7.0).all()
        outs.append(dz[:, :vocab])
    assert torch.equal(*outs)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [1, 1000, 1003, 1024])
def test_gradient_of_a_slice_takes_its_own_room(cuda, vocab, dtype):
    """The last positions of [batch, seq, vocab] logits, rows of a pitch of seq *
    vocab: the gradient holds the rows read and at most a chunk of 32 bytes more
    a row, not the whole tensor's room, and is right."""
    import torch

    from torobi_b200 import glue

    batch, seq = 5, 67
    full = _logits(cuda, batch * seq, vocab, dtype, 33).contiguous().view(batch, seq, vocab)
    z = full[:, -1]
    assert z.stride(0) == seq * vocab
    tokens = _tokens(cuda, batch, vocab, 33)
    ids, t = _teacher(cuda, batch, vocab, min(3, vocab), 33, torch.int64, "f32")
    g, h = torch.randn(batch, device=cuda), torch.randn(batch, device=cuda)
    leaf = z.detach().requires_grad_()
    r = glue.token_logprobs(leaf, tokens)
    kl, ce = glue.distillation(leaf, ids, t, targets=tokens, temperature=1.5)
    a, = torch.autograd.grad((r.logprobs, r.entropy), leaf, (g, h))
    b, = torch.autograd.grad((kl, ce), leaf, (g, h))
    *_, want, size, reach = _distill_reference(z, ids, t, tokens, 1.5, g, h)
    _check_gradient(a, *_logprob_grad(z, tokens, 1.0, g, h), dtype)
    _check_gradient(b, want, 2 * size, reach, dtype)
    for dz in (a, b):
        taken, row = dz.untyped_storage().nbytes(), vocab * z.element_size()
        assert dz.shape == z.shape and taken <= batch * (row + 32)


@pytest.mark.parametrize("writer", ["token_logprobs", "distillation", "cross_entropy"])
def test_logits_written_over_are_refused_to_other_backward_passes(cuda, writer):
    """inplace=True with another op of the same logits: where the writer's
    backward pass comes first, the other's raises instead of reading a gradient
    for logits; where it comes last, the sum is the sum of both gradients."""
    import torch

    from torobi_b200 import glue

    base = _logits(cuda, 9, 500, "bf16", 34).contiguous()
    tokens = _tokens(cuda, 9, 500, 34).clamp(0, 499)
    ids, t = _teacher(cuda, 9, 500, 4, 34, torch.int64, "f32")
    calls = {
        "token_logprobs": lambda z, w: glue.token_logprobs(z, tokens, inplace=w).logprobs.sum(),
        "distillation": lambda z, w: glue.distillation(z, ids, t, inplace=w).sum(),
        "cross_entropy": lambda z, w: glue.cross_entropy(z, tokens, inplace=w).sum(),
        "torch": lambda z, w: (z.float() * z).sum(),
    }

    def logits():
        leaf = base.clone().requires_grad_()
        return leaf, leaf * 1.0  # not a leaf, and nothing that its own backward reads

    for other in calls:
        if other == writer:
            continue
        # The later op's backward pass runs first.
        leaf, z = logits()
        loss = calls[other](z, False) + calls[writer](z, True)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        leaf, z = logits()
        (calls[writer](z, True) + calls[other](z, False)).backward()
        apart = []
        for name in (other, writer):
            l2, z2 = logits()
            calls[name](z2, False).backward()
            apart.append(l2.grad)
        # bf16 gradients, added in bf16 by autograd.
        assert torch.equal(leaf.grad, apart[0] + apart[1])
    leaf, z = logits()
    loss = calls[writer](z, True)
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="backward twice"):
        loss.backward()


def test_rows_without_upstream_gradient(cuda):
    """A padding position (no gradient reaches it) gets zeros even where its
    logits are NaN."""
    import torch

    from torobi_b200 import glue

    z = _logits(cuda, 6, 700, "bf16", 8).contiguous()
    z[2] = float("nan")
    z[4] = float("inf")
    tokens = torch.tensor([1, 2, -1, 3, -1, 4], device=cuda)
    leaf = z.clone().requires_grad_()
    r = glue.token_logprobs(leaf, tokens)
    assert r.logprobs[2] == 0 and r.logprobs[4] == 0
    r.logprobs.sum().backward()
    assert torch.isfinite(leaf.grad).all() and (leaf.grad[2] == 0).all()
    leaf = z.clone().requires_grad_()
    ids = torch.randint(0, 700, (6, 4), device=cuda)
    ids[2] = -1
    ids[4] = 700
    kl, ce = glue.distillation(leaf, ids, torch.randn(6, 4, device=cuda), targets=tokens)
    assert kl[2] == 0 and ce[2] == 0 and kl[4] == 0 and ce[4] == 0
    (kl + ce).sum().backward()
    assert torch.isfinite(leaf.grad).all()
    assert (leaf.grad[2] == 0).all() and (leaf.grad[4] == 0).all()


# ------------------------------------------------------------ distillation --

def _teacher(cuda, rows, vocab, k, seed, ids_dtype, dtype):
    import torch

    g = torch.Generator(device=cuda).manual_seed(seed)
    ids = torch.stack([torch.randperm(vocab, device=cuda, generator=g)[:k] for _ in range(rows)])
    t = torch.randn(rows, k, device=cuda, generator=g) * 2
    if k > 2:
        ids[0, k // 2:] = -1                 # fewer alternatives
        t[-1, 1] = NINF                      # one without weight
        ids[rows // 2, 2] = ids[rows // 2, 0]  # the same id twice
    if rows > 3:
        ids[1] = -1                          # none
        ids[3, 0] = vocab                    # outside
    return ids.to(ids_dtype), t.to(_dtype(dtype))


def _distill_reference(z, ids, t, targets, temperature, dkl, dce):
    import torch

    rows, vocab = z.shape
    ids = ids.long()
    valid = (ids >= 0) & (ids < vocab)
    at = ids.clamp(0, vocab - 1)
    x = z.double()
    logq = torch.log_softmax(x / temperature, 1)
    w = torch.where(valid, t.double() / temperature, NINF)
    any_ = valid.any(1)
    w = torch.where(any_[:, None], w, 0.0)
    logp = torch.log_softmax(w, 1)
    p = torch.where(any_[:, None], logp.exp(), 0.0)
    terms = torch.where(p > 0, p * (logp - logq.gather(1, at)), 0.0)
    kl = terms.sum(1)
    kl_size = torch.where(p > 0, p * (logp.abs() + logq.gather(1, at).abs()), 0.0).sum(1)
    u = (dkl.double() / temperature * any_)[:, None]
    dz = u * logq.exp()
    size = dz.abs()
    dz.scatter_add_(1, at, -u * p)
    size.scatter_add_(1, at, u.abs() * p)
    reach = torch.where(logq.exp() > 0, logq.abs(), 0.0)
    ce = None
    if targets is not None:
        hard = torch.log_softmax(x, 1)
        known = (targets >= 0) & (targets < vocab)
        to = targets.clamp(0, vocab - 1)[:, None]
        ce = torch.where(known, -hard.gather(1, to).squeeze(1), 0.0)
        v = torch.where(known, dce.double(), 0.0)[:, None]
        dz += v * hard.exp()
        dz.scatter_add_(1, to, -v)
        size += v.abs() * hard.exp()
        size.scatter_add_(1, to, v.abs())
        reach = torch.maximum(reach, torch.where(hard.exp() > 0, hard.abs(), 0.0))
    return kl, kl_size, ce, dz, size, reach


DISTILL = [
    # rows, vocab, k, dtype, temperature, hard, pad, shift, ids, teacher dtype
    (1, 1, 1, "f32", 1.0, True, 0, 0, "int64", "f32"),
    (5, 17, 3, "bf16", 2.0, True, 0, 3, "int32", "bf16"),
    (37, 1001, 8, "bf16", 1.0, True, 0, 0, "int64", "f32"),
    (37, 1001, 8, "bf16", 1.0, False, 0, 0, "int32", "f32"),
    (37, 1001, 20, "f32", 0.5, True, 7, 1, "int64", "bf16"),
    (64, 1024, 128, "bf16", 2.0, True, 64, 0, "int64", "f32"),
    (2, 151936, 64, "bf16", 2.0, True, 0, 0, "int32", "bf16"),
    (4, 32003, 50, "f32", 1.0, True, 61, 0, "int64", "f32"),
    (650, 4099, 5, "bf16", 3.0, False, 0, 0, "int64", "f32"),
    (3, 128256, 64, "bf16", 3.0, True, 0, 0, "int64", "f32"),   # sums at two temperatures
    (33, 5003, 8, "f32", 1.7, True, 0, 0, "int64", "f32"),
]


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("case", DISTILL, ids=str)
def test_distillation(cuda, case, inplace):
    import torch

    from torobi_b200 import glue

    rows, vocab, k, dtype, temperature, hard, pad, shift, idt, tdt = case
    z = _logits(cuda, rows, vocab, dtype, 9, pad=pad, shift=shift)
    before = z.clone()
    ids, t = _teacher(cuda, rows, vocab, k, 9, getattr(torch, idt), tdt)
    targets = None
    if hard:
        targets = _tokens(cuda, rows, vocab, 9)
        targets[0] = ids[0, 0].clamp(min=0)  # a target among the alternatives
    dkl = torch.rand(rows, device=cuda) + 0.5
    dce = torch.rand(rows, device=cuda) + 0.5
    leaf = z.detach().requires_grad_()
    got = glue.distillation(leaf, ids, t, targets=targets, temperature=temperature,
                            inplace=inplace)
    outs, ups = ((got,), (dkl,)) if not hard else (got, (dkl, dce))
    # The same without a graph, on the same memory (a copy may start elsewhere
    # in its 32-byte chunk, where the sums take another order).
    again = glue.distillation(z, ids, t, targets=targets, temperature=temperature)
    dz, = torch.autograd.grad(outs, leaf, ups)
    assert inplace == (dz.data_ptr() == z.data_ptr())
    kl, kl_size, ce, want, size, reach = _distill_reference(before, ids, t, targets, temperature,
                                                            dkl, dce)
    lnv = math.log(vocab) + 1
    tol = 2 * _sum_err(vocab) + (8 + k / 4) * E * (kl_size + lnv)
    assert ((outs[0].double() - kl).abs() <= tol).all(), (outs[0].double() - kl).abs().max()
    if hard:
        assert ((outs[1].double() - ce).abs() <= _sum_err(vocab) + 4 * E * (ce + lnv)).all()
    _check_gradient(dz, want, 2 * size, reach, dtype)
    assert torch.equal(again[0] if hard else again, outs[0])


def test_distillation_from_token_logprobs(cuda):
    """A teacher's own alternatives: with all of the vocabulary given, kl is 0
    for the teacher itself and equals the full divergence for another model."""
    import torch

    from torobi_b200 import glue

    teacher = _logits(cuda, 11, 100, "f32", 10).contiguous()
    student = _logits(cuda, 11, 100, "f32", 11).contiguous()
    r = glue.token_logprobs(teacher, _tokens(cuda, 11, 100, 10), top=100)
    self_kl = glue.distillation(teacher, r.top_ids, r.top_logprobs)
    assert self_kl.abs().max().item() <= 400 * E
    kl = glue.distillation(student, r.top_ids, r.top_logprobs, temperature=2.0)
    p = torch.log_softmax(teacher.double() / 2, 1)
    q = torch.log_softmax(student.double() / 2, 1)
    want = (p.exp() * (p - q)).sum(1)
    assert ((kl.double() - want).abs() <= 400 * E * (1 + want)).all()


def test_distillation_gradient_against_differences(cuda):
    import torch

    from torobi_b200 import glue

    rows, vocab = 4, 30
    z = _logits(cuda, rows, vocab, "f32", 12).contiguous()
    ids, t = _teacher(cuda, rows, vocab, 6, 12, torch.int64, "f32")
    targets = torch.tensor([int(ids[0, 0]), 5, -1, 29], device=cuda)
    dkl, dce = torch.rand(rows, device=cuda), torch.rand(rows, device=cuda)
    leaf = z.clone().requires_grad_()
    dz, = torch.autograd.grad(
        glue.distillation(leaf, ids, t, targets=targets, temperature=1.7), leaf, (dkl, dce))
    step = 1e-5

    def loss(x):
        kl, _, ce, *_ = _distill_reference(x, ids, t, targets, 1.7, dkl, dce)
        return kl * dkl.double() + ce * dce.double()

    for j in range(vocab):
        up, down = z.double().clone(), z.double().clone()
        up[:, j] += step
        down[:, j] -= step
        diff = (loss(up) - loss(down)) / (2 * step)
        assert ((dz[:, j].double() - diff).abs() <= 50 * step ** 2 + 1e-9 + 200 * E).all()


def test_given_at_minus_infinity_and_dead_rows(cuda):
    """A given alternative that the student rules out: kl is +inf and its
    gradient finite; a student row without a distribution likewise."""
    import torch

    from torobi_b200 import glue

    z = _logits(cuda, 4, 64, "f32", 13).contiguous()
    z[1, 7] = NINF
    z[2] = NINF
    ids = torch.tensor([[7, 8]] * 4, device=cuda)
    t = torch.zeros(4, 2, device=cuda)
    leaf = z.clone().requires_grad_()
    kl, ce = glue.distillation(leaf, ids, t, targets=torch.tensor([1, 7, 7, 1], device=cuda))
    assert kl[1] == math.inf and kl[2] == math.inf and ce[1] == math.inf and ce[2] == math.inf
    assert torch.isfinite(kl[[0, 3]]).all()
    dz, = torch.autograd.grad(kl.sum(), leaf)
    assert torch.isfinite(dz).all() and dz[1, 7] == -0.5


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 2.0, 3.0])
@pytest.mark.parametrize("vocab, dtype", [(64, "f32"), (1003, "bf16"), (40000, "bf16")])
def test_a_row_without_a_distribution_passes_no_gradient(cuda, vocab, dtype, temperature, inplace):
    """A student row of nothing but -inf: kl and ce are +inf and the gradient is
    0 everywhere, at the given ids and the target too, through kl, through ce
    and through both; the rows beside it are as they are without it."""
    import torch

    from torobi_b200 import glue

    z = _logits(cuda, 4, vocab, dtype, 14)
    ids = torch.tensor([[7, 8, vocab - 1]] * 4, device=cuda)
    t = torch.tensor([[0.0, 1.0, -1.0]] * 4, device=cuda)
    targets = torch.tensor([1, 7, 8, vocab - 2], device=cuda)
    one = torch.ones(4, device=cuda)
    for ups in ((one, None), (None, one), (one, one)):
        grads = []
        for dead in (False, True):
            x = z.clone()
            if dead:
                x[2] = NINF
            leaf = x.requires_grad_()
            out = glue.distillation(leaf, ids, t, targets=targets, temperature=temperature,
                                    inplace=inplace)
            if dead:
                assert out[0][2] == math.inf and out[1][2] == math.inf
            used = [(o, u) for o, u in zip(out, ups) if u is not None]
            grads += torch.autograd.grad([o for o, _ in used], leaf, [u for _, u in used])
        clean, dz = grads
        assert (dz[2] == 0).all() and (clean[2] != 0).any()
        keep = torch.tensor([0, 1, 3], device=cuda)
        assert torch.equal(dz[keep], clean[keep])


# ------------------------------------------------------------- how it is called --

@pytest.mark.parametrize("temperature", [1.0, 2.0, 3.0])
def test_distillation_nan_and_inf_rows(cuda, temperature):
    """A NaN or +inf anywhere makes its row's answers NaN, at any temperature;
    the rows beside it are as they were."""
    import torch

    from torobi_b200 import glue

    z = _logits(cuda, 9, 4099, "bf16", 31).contiguous()
    ids = torch.arange(9 * 6, device=cuda).view(9, 6) * 70
    given, targets = torch.randn(9, 6, device=cuda), torch.full((9,), 7, device=cuda)
    want = glue.distillation(z, ids, given, targets=targets, temperature=temperature)
    for r, (at, value) in enumerate([(0, "nan"), (4098, "nan"), (2000, "inf"), (2002, "inf"),
                                     (17, "-nan"), (33, "inf")]):
        z[r, at] = float(value)
    got = glue.distillation(z, ids, given, targets=targets, temperature=temperature)
    for a, b in zip(got, want):
        assert a[:6].isnan().all() and torch.equal(a[6:], b[6:])


def test_calls_in_a_graph_and_on_another_stream(cuda):
    """Forward and backward on a side stream, then captured with static
    buffers and replayed on new logits: the eager results bit for bit, two
    captured graphs run one after the other included."""
    import torch

    from torobi_b200 import glue

    rows, vocab, k = 33, 4099, 12
    zs = [_logits(cuda, rows, vocab, "bf16", 20 + i).contiguous() for i in range(3)]
    tokens = _tokens(cuda, rows, vocab, 20)
    ids, t = _teacher(cuda, rows, vocab, k, 20, torch.int64, "f32")
    up = torch.rand(rows, device=cuda)

    def work(z):
        leaf = z.detach().requires_grad_()
        a = glue.token_logprobs(leaf, tokens)
        b = glue.distillation(leaf, ids, t, targets=tokens, temperature=2.0)
        da, = torch.autograd.grad((a.logprobs, a.entropy), leaf, (up, up))
        db, = torch.autograd.grad(b, leaf, (up, up))
        top = glue.token_logprobs(z, tokens, top=5)
        return [a.logprobs.detach(), a.entropy.detach(), da, b[0].detach(), b[1].detach(), db,
                top.top_ids, top.top_logprobs]

    want = [work(z) for z in zs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = work(zs[0])
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(on_side, want[0]):
        assert torch.equal(a, b)
    graphs = []
    for i in range(2):
        static = zs[i].clone()
        with torch.cuda.stream(side):
            work(static)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work(static)
        graphs.append((graph, static, out))
    for turn in range(2):
        for i, (graph, static, out) in enumerate(graphs):
            static.copy_(zs[i + turn])
            graph.replay()
        for i, (graph, static, out) in enumerate(graphs):
            for a, b in zip(out, want[i + turn]):
                assert torch.equal(a, b)


def test_shapes_and_refusals(cuda):
    import torch

    from torobi_b200 import TqError, glue

    z = torch.zeros(2, 3, 8, dtype=torch.bfloat16, device=cuda)
    t = torch.zeros(2, 3, dtype=torch.int32, device=cuda)
    r = glue.token_logprobs(z, t, top=2)
    assert r.logprobs.shape == (2, 3) and r.top_ids.shape == (2, 3, 2)
    assert glue.token_logprobs(z, t).top_ids is None
    empty = glue.token_logprobs(z[:0], t[:0], top=2)
    assert empty.logprobs.shape == (0, 3) and empty.top_ids.shape == (0, 3, 2)
    leaf = torch.zeros(0, 8, device=cuda, requires_grad=True)
    glue.token_logprobs(leaf, torch.zeros(0, dtype=torch.int64, device=cuda)).logprobs.sum().backward()
    assert leaf.grad.shape == (0, 8)
    one = glue.token_logprobs(z[0, 0], t[0, 0])
    assert one.logprobs.shape == () and abs(one.logprobs.item() + math.log(8)) < 1e-6
    for bad in (lambda: glue.token_logprobs(z.half(), t), lambda: glue.token_logprobs(z, t[0]),
                lambda: glue.token_logprobs(z, t.float()), lambda: glue.token_logprobs(z, t, top=9),
                lambda: glue.token_logprobs(z, t, top=-1),
                lambda: glue.token_logprobs(z, t, temperature=0.0),
                lambda: glue.token_logprobs(z, t.cpu()),
                lambda: glue.distillation(z, z, z), lambda: glue.distillation(z, t, z),
                lambda: glue.distillation(z, t[..., None], z[..., :2]),
                lambda: glue.distillation(z, t[..., None], z[..., :1], targets=t[0])):
        with pytest.raises(ValueError):
            bad()
    wide = torch.zeros(1, 200, device=cuda)
    with pytest.raises(TqError, match="alternatives"):
        glue.distillation(wide, torch.zeros(1, 129, dtype=torch.int64, device=cuda),
                          torch.zeros(1, 129, device=cuda))
