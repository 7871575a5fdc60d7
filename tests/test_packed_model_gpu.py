"""Packed documents, scoring and distillation as a trainer uses them together:
a teacher scores packed rows and keeps its alternatives, a student is trained
on them over the same rows.

Tolerance of logits and log probabilities between two computations of one
model: some 20 roundings to bf16 (2^-9 of the value on average) stand one
behind the other in the two-layer test model, so a hidden value errs by
sqrt(20) 2^-9 = 1 % of its size (spread), a logit (standard deviation 0.3: 256
hidden values of size 1 against embeddings of 0.02) by 0.003, plus its own
rounding, up to 2^-9 * 2; ten times that, twice for a difference: 0.1.
"""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
TOL = 0.1


def _model(seed=0, **over):
    from torobi_b200.model import QLoRACausalLM, tiny_config

    return QLoRACausalLM(tiny_config(**over), seed=seed)


def _rows(cuda, lengths, seq, vocab=1024, seed=1):
    """Packed ids [batch, seq], document ids, and the documents one by one."""
    import torch

    g = torch.Generator(device=cuda).manual_seed(seed)
    ids = torch.randint(0, vocab, (len(lengths), seq), device=cuda, generator=g)
    docs = torch.full((len(lengths), seq), -1, device=cuda, dtype=torch.int32)
    parts = []
    for r, row in enumerate(lengths):
        at = 0
        for n, length in enumerate(row):
            docs[r, at:at + length] = n
            parts.append((r, at, length))
            at += length
    return ids, docs, parts


LENGTHS = [[40, 7, 1, 75], [128], [3, 100, 2]]


def test_packed_rows_score_as_their_documents_do(cuda):
    """Each document's log probabilities in a packed row are those of the
    document alone; targets across documents and in padding are 0."""
    import torch

    model = _model()
    ids, docs, parts = _rows(cuda, LENGTHS, 128)
    with torch.no_grad():
        packed = model.token_logprobs(ids, top=3, documents=docs)
        counted = torch.zeros(3, 127, dtype=torch.bool, device=cuda)
        for r, at, n in parts:
            if n < 2:
                continue
            alone = model.token_logprobs(ids[r:r + 1, at:at + n], top=3)
            for a, b in zip(alone[:3], packed[:3]):
                assert ((a[0] - b[r, at:at + n - 1]).abs() <= TOL).all()
            counted[r, at:at + n - 1] = True
    assert (packed.logprobs[~counted] == 0).all() and (packed.logprobs[counted] < 0).all()
    assert torch.isfinite(packed.entropy).all()
    # The loss is their mean.
    loss = model.loss(ids, docs)
    assert abs(loss.item() + packed.logprobs.sum().item() / counted.sum().item()) <= 1e-3


def test_prompts_are_seen_in_both_directions(cuda):
    """A prompt position sees the rest of its prompt: changing a later prompt
    token moves earlier prompt positions, changing an answer token does not;
    prompt tokens are not targets."""
    import torch

    model = _model(1)
    ids, docs, _ = _rows(cuda, [[60, 40]], 100)
    prefix = torch.zeros_like(docs)
    prefix[:, :60] = 20
    prefix[:, 60:] = 5
    with torch.no_grad():
        base = model.hidden(ids, docs, prefix)
        other = ids.clone()
        other[0, 15] = (other[0, 15] + 1) % 1024
        moved = (model.hidden(other, docs, prefix) != base).any(2)[0]
        assert moved[:60].sum() >= 55 and not moved[60:].any()
        other = ids.clone()
        other[0, 30] = (other[0, 30] + 1) % 1024
        moved = (model.hidden(other, docs, prefix) != base).any(2)[0]
        assert not moved[:30].any() and moved[30:60].any() and not moved[60:].any()
        lp = model.token_logprobs(ids, documents=docs, prefix=prefix).logprobs[0]
    zero = lp == 0
    assert zero[:19].all() and not zero[19:59].any()      # targets 1..19 in the prompt
    assert zero[59] and zero[60:64].all() and not zero[64:].any()


@pytest.mark.parametrize("longest", [2 ** 31 - 1, 2 ** 40])
def test_prompts_longer_than_their_documents(cuda, longest):
    """A prompt length past the document's end, however large: the whole
    document is a prompt, and nothing in it a target."""
    import torch

    model = _model(1)
    ids, docs, _ = _rows(cuda, [[60, 40]], 100)
    prefix = torch.zeros_like(docs, dtype=torch.int32 if longest < 2 ** 31 else torch.int64)
    prefix[:, 60:] = longest
    with torch.no_grad():
        lp = model.token_logprobs(ids, documents=docs, prefix=prefix).logprobs[0]
    assert (lp[:59] != 0).all() and (lp[59:] == 0).all()


def _plain_distill(model, ids, tids, tlogits, docs, prefix_mask, temperature, alpha):
    import torch

    with torch.no_grad():
        z = model.logits(model.hidden(ids, docs)[:, :-1]).double()
    logq = torch.log_softmax(z / temperature, -1)
    logp = torch.log_softmax(tlogits.double() / temperature, -1)
    kl = (logp.exp() * (logp - logq.gather(-1, tids))).sum(-1)
    ce = -torch.log_softmax(z, -1).gather(-1, ids[:, 1:, None])[..., 0]
    loss = (1 - alpha) * ce + alpha * temperature ** 2 * kl
    return (loss * prefix_mask).sum() / prefix_mask.sum()


@pytest.mark.parametrize("graph", [False, True])
def test_a_student_distilled_from_a_teachers_alternatives(cuda, graph):
    """teacher.token_logprobs over packed rows -> student.distill_loss in the
    trainer, micro-batched, eagerly and as a CUDA graph: the loss is the
    formula's, every adapter gets a gradient, and an optimizer step is taken."""
    import torch

    from torobi_b200.train import AdamWConfig, Trainer

    teacher, student = _model(3), _model(4, lora_targets=("q_proj", "k_proj", "v_proj", "o_proj"))
    ids, docs, _ = _rows(cuda, [[40, 60, 20], [100], [64, 64], [128]], 128)
    counted = ((docs[:, 1:] == docs[:, :-1]) & (docs[:, 1:] >= 0)).double()
    with torch.no_grad():
        t = teacher.token_logprobs(ids, top=16, documents=docs)

    def objective(rows, tids, tlogits, documents):
        return student.distill_loss(rows, tids, tlogits, documents, temperature=2.0, alpha=0.7)

    want = sum(_plain_distill(student, ids[a:a + 2], t.top_ids[a:a + 2], t.top_logprobs[a:a + 2],
                              docs[a:a + 2], counted[a:a + 2], 2.0, 0.7) for a in (0, 2)) / 2
    trainer = Trainer(student, AdamWConfig(lr=1e-3), micro_batch=2, graph=graph,
                      objective=objective)
    before = student.store.params.clone()
    loss = trainer.step(ids, t.top_ids, t.top_logprobs, docs).item()
    # Both from the same bf16 logits: only f32 sums and the eager rerun differ.
    assert abs(loss - want.item()) <= 1e-4 * abs(want.item())
    g = student.store.grads
    assert torch.isfinite(g).all() and (g != 0).any()
    assert trainer.settle() > 0 and not torch.equal(before, student.store.params)
    again = trainer.step(ids, t.top_ids, t.top_logprobs, docs).item()
    assert again == again
    with pytest.raises(ValueError, match="rows beside"):
        trainer.step(ids, docs[:1])


def test_an_objective_that_weighs_every_target_alike(cuda):
    """A sum over the micro-batch by the whole step's targets, times the number
    of micro-batches: the same loss and gradients however the rows are split."""
    import torch

    from torobi_b200.train import AdamWConfig, Trainer

    ids, docs, _ = _rows(cuda, [[40, 60, 20], [5], [64, 64], [128]], 128)
    total = ((docs[:, 1:] == docs[:, :-1]) & (docs[:, 1:] >= 0)).sum()
    seen = []
    for micro in (1, 2, 4):
        model = _model(8)

        def objective(rows, documents):
            lp = model.token_logprobs(rows, documents=documents).logprobs
            return -lp.sum() * ((4 // micro) / total)

        trainer = Trainer(model, AdamWConfig(lr=1e-3), micro_batch=micro, objective=objective)
        loss = trainer.step(ids, docs).item()
        # The trainer's own division by the micro-batches is left to the optimizer.
        seen.append((loss, model.store.grads.clone() / (4 // micro)))
    plain = _model(8)
    with torch.no_grad():
        lp = plain.token_logprobs(ids, documents=docs).logprobs
    want = -(lp.double().sum() / total).item()
    for loss, grads in seen:
        # f32 sums of 340 log probabilities of size 7.
        assert abs(loss - want) <= 1e-5 * abs(want)
        # bf16 gradients of the logits at other scales: a power of two apart.
        assert ((grads - seen[0][1]).norm() / seen[0][1].norm()).item() <= 2 ** -8


def test_a_captured_step_beside_a_score_that_keeps_its_graph(cuda):
    """The teacher's answer is held with its graph while the student's step is
    captured and replayed; the teacher's own backward still runs after."""
    import torch

    from torobi_b200.train import AdamWConfig, Trainer

    teacher, student = _model(3), _model(4)
    ids, docs, _ = _rows(cuda, [[100], [64, 64]], 128)
    held = teacher.token_logprobs(ids, top=8, documents=docs)
    assert held.logprobs.requires_grad
    trainers = [Trainer(m, AdamWConfig(lr=1e-3), micro_batch=2, graph=g, objective=m.distill_loss)
                for m, g in ((student, True), (_model(4), False))]
    for far in (1e-5, 1e-2):  # the second after a step of 1e-3 by gradients' signs
        a, b = (t.step(ids, held.top_ids, held.top_logprobs, docs).item() for t in trainers)
        assert abs(a - b) <= far * abs(a)
    teacher.store.zero_grad()
    held.logprobs.sum().backward()
    assert torch.isfinite(teacher.store.grads).all() and (teacher.store.grads != 0).any()


def test_distill_gradient_reaches_the_adapters_by_the_formula(cuda):
    """The adapters' gradients of distill_loss against those of the same loss
    written in torch operations on the model's logits."""
    import torch

    student = _model(5)
    ids, docs, _ = _rows(cuda, LENGTHS, 128)
    g = torch.Generator(device=cuda).manual_seed(9)
    tids = torch.randint(0, 1024, (3, 127, 4), device=cuda, generator=g)
    tlogits = torch.randn(3, 127, 4, device=cuda, generator=g)
    # B is 0 at first, and with it A's gradient: a step away from there.
    student.store.params.add_(torch.randn(student.store.params.shape, device=cuda, generator=g)
                              * 0.02)
    student.store.params16.copy_(student.store.params)
    student.store.refresh_bf16()
    counted = (docs[:, 1:] == docs[:, :-1]) & (docs[:, 1:] >= 0)

    def grads(loss):
        student.store.zero_grad()
        loss.backward()
        return student.store.grads.clone()

    a = grads(student.distill_loss(ids, tids, tlogits, docs, temperature=1.5, alpha=0.3))
    z = student.logits(student.hidden(ids, docs)[:, :-1]).float()
    logq = torch.log_softmax(z / 1.5, -1)
    logp = torch.log_softmax(tlogits / 1.5, -1)
    kl = (logp.exp() * (logp - logq.gather(-1, tids))).sum(-1)
    ce = -torch.log_softmax(z, -1).gather(-1, ids[:, 1:, None])[..., 0]
    b = grads((((0.7 * ce + 0.3 * 2.25 * kl) * counted).sum()) / counted.sum())
    # The logits' gradient is rounded to bf16 on both ways, 2^-9 each on average.
    assert ((a - b).norm() / b.norm()).item() <= 2 ** -7


def test_policy_gradient_through_logprobs_and_entropy(cuda):
    """A policy step (log probability times an advantage, and the entropy)
    through the model, packed: the adapters' gradients against torch's."""
    import torch

    model = _model(6)
    ids, docs, _ = _rows(cuda, LENGTHS, 128)
    adv = torch.randn(3, 127, device=cuda, generator=torch.Generator(device=cuda).manual_seed(2))
    model.store.params.add_(torch.randn_like(model.store.params) * 0.02)
    model.store.params16.copy_(model.store.params)
    model.store.refresh_bf16()
    counted = ((docs[:, 1:] == docs[:, :-1]) & (docs[:, 1:] >= 0)).float()

    def grads(loss):
        model.store.zero_grad()
        loss.backward()
        return model.store.grads.clone()

    r = model.token_logprobs(ids, documents=docs)
    a = grads(-(r.logprobs * adv + 0.1 * r.entropy * counted).sum() / 300)
    logq = torch.log_softmax(model.logits(model.hidden(ids, docs)[:, :-1]).float(), -1)
    lp = logq.gather(-1, ids[:, 1:, None])[..., 0] * counted
    ent = -(logq.exp() * logq).sum(-1)
    b = grads(-(lp * adv + 0.1 * ent * counted).sum() / 300)
    assert ((a - b).norm() / b.norm()).item() <= 2 ** -7


def test_refusals(cuda):
    import torch

    model = _model(7)
    ids, docs, _ = _rows(cuda, [[10]], 16)
    with pytest.raises(ValueError, match="must match the ids"):
        model.loss(ids, docs[:, :8])
    with pytest.raises(ValueError, match="goes with documents"):
        model.loss(ids, None, docs)
    # Rows of padding alone have no targets: a loss of 0, gradients of 0.
    loss = model.loss(ids, torch.full_like(docs, -1))
    assert loss.item() == 0.0
    model.store.zero_grad()
    loss.backward()
    assert (model.store.grads == 0).all()
