"""Refusals of the token_logprobs and distillation entry points, which are
checked on the host before any CUDA call."""
from __future__ import annotations

import pytest

P = 1 << 20  # an aligned stand-in address; nothing is dereferenced
BF16, F32 = 1, 0


def _lib():
    import torobi_b200 as tq

    return tq.lib()


def _logprobs_fwd(z=P, dtype=BF16, tokens=P, rows=4, vocab=64, ld=64, temperature=1.0, top=3,
                  logprobs=P, entropy=P, stats=P, top_logprobs=P, top_ids=P):
    return _lib().tq_token_logprobs_fwd(z, dtype, tokens, rows, vocab, ld, temperature, top,
                                        logprobs, entropy, stats, top_logprobs, top_ids, None)


def _logprobs_bwd(z=P, dtype=BF16, tokens=P, stats=P, rows=4, vocab=64, ld=64, temperature=1.0,
                  dlp=P, dent=P, dz=2 * P, ld_out=64):
    return _lib().tq_token_logprobs_bwd(z, dtype, tokens, stats, rows, vocab, ld, temperature, dlp,
                                        dent, dz, ld_out, None)


def _distill_fwd(z=P, dtype=BF16, ids=P, bits=64, t=P, tdtype=F32, k=4, targets=P, rows=4,
                 vocab=64, ld=64, temperature=1.0, kl=P, ce=P, stats=P):
    return _lib().tq_distill_fwd(z, dtype, ids, bits, t, tdtype, k, targets, rows, vocab, ld,
                                 temperature, kl, ce, stats, None)


def _distill_bwd(z=P, dtype=BF16, ids=P, bits=64, t=P, tdtype=F32, k=4, targets=P, stats=P, rows=4,
                 vocab=64, ld=64, temperature=1.0, dkl=P, dce=P, dz=2 * P, ld_out=64):
    return _lib().tq_distill_bwd(z, dtype, ids, bits, t, tdtype, k, targets, stats, rows, vocab, ld,
                                 temperature, dkl, dce, dz, ld_out, None)


@pytest.mark.parametrize("call", [_logprobs_fwd, _logprobs_bwd, _distill_fwd, _distill_bwd])
@pytest.mark.parametrize("bad, code, word", [
    (dict(dtype=7), 2, "f32 or bf16"),
    (dict(vocab=0), 1, "vocab > 0"),
    (dict(ld=63), 1, "ld >= vocab"),
    (dict(rows=-1), 1, "rows >= 0"),
    (dict(vocab=1 << 31, ld=1 << 31), 1, "2^31"),
    (dict(rows=1 << 28), 1, "2^27"),
    (dict(temperature=0.0), 1, "temperature"),
    (dict(temperature=-1.0), 1, "temperature"),
    (dict(temperature=float("nan")), 1, "temperature"),
    (dict(temperature=float("inf")), 1, "temperature"),
    (dict(temperature=1e-39), 1, "temperature"),
    (dict(z=None), 1, "null"),
    (dict(z=P + 1), 3, "aligned"),
    (dict(z=P + 2, dtype=F32), 3, "aligned"),
    (dict(stats=P + 8), 3, "stats: 16 bytes"),
], ids=lambda v: str(v) if isinstance(v, dict) else None)
def test_refusals_of_every_entry_point(call, bad, code, word):
    assert call(**bad) == code
    assert word in _lib().tq_last_error().decode()


@pytest.mark.parametrize("call, bad, code, word", [
    (_logprobs_fwd, dict(top=-1), 1, "top"),
    (_logprobs_fwd, dict(top=129, vocab=200, ld=200), 1, "top"),
    (_logprobs_fwd, dict(top=65), 1, "top"),
    (_logprobs_fwd, dict(vocab=(1 << 21) + 64, ld=(1 << 21) + 64), 1, "vocab of at most"),
    (_logprobs_fwd, dict(dtype=F32, vocab=(1 << 20) + 64, ld=(1 << 20) + 64), 1, "vocab of at most"),
    (_logprobs_fwd, dict(top_ids=None), 1, "null"),
    (_logprobs_fwd, dict(tokens=None), 1, "null"),
    (_logprobs_fwd, dict(entropy=None), 1, "null"),
    (_logprobs_fwd, dict(top_ids=P + 4), 3, "aligned"),
    (_logprobs_fwd, dict(tokens=P + 4), 3, "aligned"),
    (_logprobs_bwd, dict(ld_out=63), 1, "ld_out"),
    (_logprobs_bwd, dict(stats=None), 1, "null"),
    (_logprobs_bwd, dict(dz=None), 1, "null"),
    (_logprobs_bwd, dict(dz=P, ld_out=80), 1, "in place"),
    (_logprobs_bwd, dict(dlp=P + 2), 3, "aligned"),
    (_distill_fwd, dict(k=0), 1, "alternatives"),
    (_distill_fwd, dict(k=129), 1, "alternatives"),
    (_distill_fwd, dict(bits=16), 2, "32- or 64-bit"),
    (_distill_fwd, dict(tdtype=5), 2, "teacher logits"),
    (_distill_fwd, dict(ids=P + 4), 3, "teacher pointer"),
    (_distill_fwd, dict(t=P + 2), 3, "teacher pointer"),
    (_distill_fwd, dict(ids=None), 1, "null"),
    (_distill_fwd, dict(ce=None), 1, "together"),
    (_distill_fwd, dict(targets=None), 1, "together"),
    (_distill_fwd, dict(kl=None), 1, "null kl"),
    (_distill_bwd, dict(k=0), 1, "alternatives"),
    (_distill_bwd, dict(targets=None), 1, "dce without targets"),
    (_distill_bwd, dict(dz=P, ld_out=80), 1, "in place"),
    (_distill_bwd, dict(ld_out=1), 1, "ld_out"),
    (_distill_bwd, dict(dkl=P + 2), 3, "aligned"),
], ids=lambda v: str(v) if isinstance(v, dict) else None)
def test_refusals_of_one_entry_point(call, bad, code, word):
    assert call(**bad) == code
    assert word in _lib().tq_last_error().decode()


def test_no_rows_is_no_call():
    """An empty batch is valid and touches nothing."""
    assert _logprobs_fwd(rows=0, z=None, tokens=None, logprobs=None) == 0
    assert _logprobs_bwd(rows=0, z=None, tokens=None, stats=None) == 0
    assert _distill_fwd(rows=0, z=None, ids=None, t=None, kl=None) == 0
    assert _distill_bwd(rows=0, z=None, ids=None, t=None, stats=None) == 0


def test_cpu_tensors_are_refused():
    import torch

    from torobi_b200 import glue

    z, t = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        glue.token_logprobs(z, t)
    with pytest.raises(ValueError, match="CUDA"):
        glue.distillation(z, t[:, None], z[:, :1])


def test_rows_read_in_place():
    """Which strides are read where they are, and which are copied."""
    import torch

    from torobi_b200.glue import _logit_rows

    def pitch(z):
        got, rows, vocab, p = _logit_rows("t", z)
        assert rows * vocab == z.numel() and vocab == z.shape[-1]
        return p if got.data_ptr() == z.data_ptr() else None

    wide = torch.zeros(3, 5, 16)
    assert pitch(wide) == 16
    assert pitch(wide[..., :13]) == 16       # padded rows
    assert pitch(wide[..., 3:]) == 16        # rows that start inside
    assert pitch(wide[:, :4]) is None        # two pitches: copied
    assert pitch(wide[:1, :4]) == 16         # one sequence: one pitch
    assert pitch(wide[:, 2]) == 80
    assert pitch(wide[1, 2]) == 16
    assert pitch(wide[1, 2, :7]) == 7
    assert pitch(wide.transpose(1, 2)) is None
    assert pitch(wide[..., ::2]) is None
    assert pitch(wide[:1].expand(3, 5, 16)) is None
    assert pitch(wide[:, :1, :].expand(3, 5, 16)) is None
    assert pitch(torch.zeros(0, 7)) == 7
    assert pitch(torch.zeros(7)) == 7
