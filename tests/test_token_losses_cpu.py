"""Log-probabilities, entropy, alternatives and distillation on the CPU path: definitions in 64 bits,
gradients against the formulas and against differences, vocabulary shards, refusals."""
import math

import pytest
import torch

from eth_b200 import ops
from eth_b200.ops import raw
from helpers import oracle_tokens as oracle

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _teacher(rows, vocab, k, seed=3):
    g = torch.Generator().manual_seed(seed)
    index = torch.randint(vocab, (rows, k), generator=g)
    logit = torch.randn(rows, k, generator=g)
    for r in range(rows):
        logit[r, k - r % (k + 1):] = -math.inf       # shorter lists, an empty one every k + 1 rows
    return index, logit


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top_k,temperature", [(1, 1, 1, 1.0), (3, 7, 7, 0.5), (17, 1001, 5, 2.0)])
def test_token_logprobs(dtype, rows, vocab, top_k, temperature):
    g = torch.Generator().manual_seed(0)
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(dtype).requires_grad_(True)
    tokens = torch.randint(vocab, (rows,), generator=g)
    r = ops.token_logprobs(logits, tokens, top_k=top_k, temperature=temperature)
    lp, ent, top_lp, top_id, _ = oracle.scores(logits, tokens, top_k, temperature)
    tol = oracle.statistic_tolerance(logits, temperature)
    assert ((r.logprob - lp).abs() <= tol).all() and ((r.entropy - ent).abs() <= tol).all()
    assert torch.equal(r.top_index, top_id) and ((r.top_logprob - top_lp).abs() <= tol[:, None]).all()
    d = [torch.randn(x.shape, generator=g) for x in (r.logprob, r.entropy, r.top_logprob)]
    got, = torch.autograd.grad((r.logprob, r.entropy, r.top_logprob), logits, d)
    want = oracle.scores_grad(logits, tokens, top_id, *d, temperature)
    assert oracle.grad_error(got, want, sum(x.abs().reshape(rows, -1).sum(1) for x in d) * 2.0 ** -18) <= 1


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(4, 9, dtype=torch.float64, generator=g, requires_grad=True)
    tokens = torch.tensor([0, 8, -1, 3])

    def scores(z):
        r = ops.token_logprobs(z, tokens, top_k=3, temperature=0.7)
        return r.logprob, r.entropy, r.top_logprob
    assert torch.autograd.gradcheck(scores, (logits,))
    index, logit = _teacher(4, 9, 3)
    index[0] = 5                                      # the same id three times
    assert torch.autograd.gradcheck(lambda z: ops.topk_distillation_loss(z, index, logit.double(), temperature=1.7),
                                    (logits,))


def test_masks_and_unscored_tokens():
    low = torch.finfo(torch.float32).min
    logits = torch.randn(6, 20, generator=torch.Generator().manual_seed(2))
    logits[0, 5:] = -math.inf
    logits[1, :19] = low
    logits[2] = low                                   # nothing but the lowest value: uniform
    logits[3] = -math.inf                             # nothing at all: undefined
    tokens = torch.tensor([1, 19, 4, 0, -1, 20])
    r = ops.token_logprobs(logits.requires_grad_(True), tokens, top_k=4)
    lp, ent, _, top_id, _ = oracle.scores(logits, tokens, 4, 1.0)
    keep = [0, 1, 2, 4]
    torch.testing.assert_close(r.logprob[keep].double(), lp[keep], rtol=0, atol=4e-6)
    torch.testing.assert_close(r.entropy[[0, 1, 2]].double(), ent[[0, 1, 2]], rtol=0, atol=4e-6)
    assert torch.equal(r.top_index, top_id)
    assert r.logprob[3].isnan() and r.entropy[3].isnan() and r.logprob[5].isnan() and r.logprob[4] == 0
    g, = torch.autograd.grad(r.logprob[[0, 1, 2, 4]].sum(), logits)
    assert g.isfinite().all() and (g[[3, 4, 5]] == 0).all() and (g[0, 5:] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,k,temperature", [(1, 1, 1, 1.0), (9, 33, 4, 0.5), (5, 1001, 64, 2.0)])
def test_distillation(dtype, rows, vocab, k, temperature):
    g = torch.Generator().manual_seed(4)
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(dtype).requires_grad_(True)
    index, logit = _teacher(rows, vocab, k)
    index[logit == -math.inf] = -7                    # unused entries may hold any id
    dloss = torch.randn(rows, generator=g)
    loss = ops.topk_distillation_loss(logits, index, logit, temperature=temperature)
    want_loss, want = oracle.distill(logits, index, logit, dloss, temperature)
    assert ((loss - want_loss).abs() <= oracle.statistic_tolerance(logits, temperature)).all()
    got, = torch.autograd.grad(loss, logits, dloss)
    assert oracle.grad_error(got, want, dloss.abs() * 2.0 ** -18) <= 1
    loss2, got2 = raw.distill_step(logits.detach(), index, logit, dloss, temperature=temperature)
    assert torch.equal(loss2, loss.detach()) and torch.equal(got2, got)
    buf = logits.detach().clone()
    loss3, got3 = raw.distill_step(buf, index, logit, dloss, temperature=temperature, out=buf)
    assert got3 is buf and torch.equal(buf, got) and torch.equal(loss3, loss2)


def test_entry_outside_the_vocabulary_is_nan():
    logits = torch.randn(2, 10)
    loss = ops.topk_distillation_loss(logits, torch.tensor([[3, 10], [3, 4]]), torch.zeros(2, 2))
    assert loss[0].isnan() and loss[1].isfinite()


@pytest.mark.parametrize("world", [2, 3])
def test_vocabulary_shards(world):
    g = torch.Generator().manual_seed(6)
    rows, part, k = 7, 40, 6
    logits = (torch.randn(rows, part * world, generator=g) * 2).round(decimals=1)     # ties across shards
    logits[1, :part] = -math.inf                      # a shard without anything to say
    tokens = torch.randint(part * world, (rows,), generator=g)
    tokens[2] = -1
    index, logit = _teacher(rows, part * world, 5)
    shards = logits.split(part, 1)
    whole = ops.token_logprobs(logits, tokens, top_k=k, temperature=0.9)
    whole_loss = ops.topk_distillation_loss(logits, index, logit, temperature=0.9)
    sent = {}

    def collect(name):                                # first run: what each rank would send
        def gather(x):
            sent.setdefault(name, []).append(x)
            return x.unsqueeze(0)
        return gather
    for w, z in enumerate(shards):
        ops.token_logprobs(z, tokens, k, 0.9, w * part, collect("scores"))
        ops.topk_distillation_loss(z, index, logit, 0.9, w * part, collect("distill"))
    for w, z in enumerate(shards):
        z = z.clone().requires_grad_(True)
        r = ops.token_logprobs(z, tokens, k, 0.9, w * part, lambda x: torch.stack(sent["scores"]))
        for a, b in zip(r, whole):
            torch.testing.assert_close(a, b, rtol=0, atol=1e-5)
        assert torch.equal(r.top_index, whole.top_index)
        loss = ops.topk_distillation_loss(z, index, logit, 0.9, w * part, lambda x: torch.stack(sent["distill"]))
        torch.testing.assert_close(loss, whole_loss, rtol=0, atol=1e-5)
        full = logits.clone().requires_grad_(True)
        rf = ops.token_logprobs(full, tokens, k, 0.9)
        gf, = torch.autograd.grad(rf.logprob.sum() + rf.entropy.sum() + rf.top_logprob.sum() +
                                  ops.topk_distillation_loss(full, index, logit, 0.9).sum(), full)
        gz, = torch.autograd.grad(r.logprob.sum() + r.entropy.sum() + r.top_logprob.sum() + loss.sum(), z)
        torch.testing.assert_close(gz, gf[:, w * part:(w + 1) * part], rtol=0, atol=1e-5)


def test_row_pitch_is_kept_in_the_gradient():
    """A slice of a padded vocabulary: the gradient has the shape of the slice, whatever its pitch."""
    wide = torch.randn(5, 24, generator=torch.Generator().manual_seed(7))
    z = wide[:, :21].detach().requires_grad_(True)
    r = ops.token_logprobs(z, torch.arange(5))
    g, = torch.autograd.grad(r.logprob.sum(), z)
    want = oracle.scores_grad(z, torch.arange(5), None, torch.ones(5), None, None, 1.0)
    torch.testing.assert_close(g.double(), want, rtol=0, atol=1e-6)


def test_refusals():
    z, t = torch.randn(3, 11), torch.zeros(3, dtype=torch.long)
    index, logit = torch.zeros(3, 2, dtype=torch.long), torch.zeros(3, 2)
    for bad in (lambda: ops.token_logprobs(z[0], t), lambda: ops.token_logprobs(z.int(), t),
                lambda: ops.token_logprobs(z, t.int()), lambda: ops.token_logprobs(z, t[:2]),
                lambda: ops.token_logprobs(z, t, top_k=12), lambda: ops.token_logprobs(z, t, top_k=-1),
                lambda: ops.token_logprobs(torch.randn(3, 500), t, top_k=129),
                lambda: ops.token_logprobs(z, t, temperature=0.0), lambda: ops.token_logprobs(z, t, temperature=math.nan),
                lambda: ops.token_logprobs(z[:, :0], t),
                lambda: ops.topk_distillation_loss(z, index, logit[:, :1]),
                lambda: ops.topk_distillation_loss(z, index.int(), logit),
                lambda: ops.topk_distillation_loss(z, index, logit.half()),
                lambda: ops.topk_distillation_loss(z, index[:, :0], logit[:, :0]),
                lambda: ops.topk_distillation_loss(z, torch.zeros(3, 513, dtype=torch.long), torch.zeros(3, 513)),
                lambda: raw.distill_step(z, index, logit, torch.ones(2)),
                lambda: raw.distill_step(z, index, logit, torch.ones(3), out=z.half()),
                lambda: raw.distill_step(z[:, :10], index, logit, torch.ones(3), out=z[:, 1:])):
        with pytest.raises(ValueError):
            bad()


def test_no_rows():
    z = torch.randn(0, 11, requires_grad=True)
    r = ops.token_logprobs(z, torch.zeros(0, dtype=torch.long), top_k=2)
    assert r.logprob.shape == (0,) and r.top_index.shape == (0, 2)
    loss = ops.topk_distillation_loss(z, torch.zeros(0, 2, dtype=torch.long), torch.zeros(0, 2))
    g, = torch.autograd.grad(loss.sum() + r.entropy.sum(), z)
    assert g.shape == (0, 11)


@pytest.mark.parametrize("overwrite", [False, True])
@pytest.mark.parametrize("last", [False, True])
def test_logits_shared_with_cross_entropy(overwrite, last):
    """Cross entropy built before or after the teacher's loss; where it may overwrite, autograd must notice."""
    g = torch.Generator().manual_seed(8)
    z = torch.randn(5, 24, generator=g, requires_grad=True)
    index, logit = _teacher(5, 24, 4)
    build = [lambda: ops.vocab_parallel_cross_entropy(z, index[:, 0], overwrite_logits=overwrite),
             lambda: ops.topk_distillation_loss(z, index, logit)]
    ones = torch.ones(5)
    want = oracle.distill(z, index, logit, ones, 1.0)[1] + oracle.scores_grad(z, index[:, 0], None, -ones, None, None, 1.0)
    outs = [f() for f in (build[::-1] if last else build)]
    if overwrite and last:
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(outs, z, [ones, ones])
        return
    got, = torch.autograd.grad(outs, z, [ones, ones])
    torch.testing.assert_close(got.double(), want, rtol=0, atol=2e-6)


def test_step_into_saved_logits_is_noticed():
    z = torch.randn(4, 9, generator=torch.Generator().manual_seed(9), requires_grad=True)
    index, logit = _teacher(4, 9, 3)
    loss = ops.topk_distillation_loss(z, index, logit)
    raw.distill_step(z.detach(), index, logit, torch.ones(4), out=z.detach())
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(loss, z, torch.ones(4))


def test_gradient_of_a_token_outside_the_vocabulary():
    """NaN where the log-probability is NaN and has a gradient; the entropy's own gradient stays defined."""
    z = torch.randn(4, 9, generator=torch.Generator().manual_seed(10), requires_grad=True)
    tokens, ones = torch.tensor([9, 8, -1, 9]), torch.ones(4)
    r = ops.token_logprobs(z, tokens)
    got, = torch.autograd.grad(r.logprob, z, torch.tensor([1.0, 1.0, 1.0, 0.0]), retain_graph=True)
    assert got[0].isnan().all() and got[1].isfinite().all() and (got[2:] == 0).all()
    got, = torch.autograd.grad(r.entropy, z, ones)
    want = oracle.scores_grad(z, torch.zeros(4, dtype=torch.long), None, None, ones, None, 1.0)
    torch.testing.assert_close(got.double(), want, rtol=0, atol=1e-6)


def test_gradient_of_a_list_with_an_entry_outside_the_vocabulary():
    z = torch.randn(3, 9, generator=torch.Generator().manual_seed(11), requires_grad=True)
    index, logit = torch.tensor([[5, 9], [7, 8], [1, 9]]), torch.tensor([[0.0, -40.0], [0.0, 1.0], [0.0, -math.inf]])
    loss = ops.topk_distillation_loss(z, index, logit)
    got, = torch.autograd.grad(loss, z, torch.ones(3))
    _, step = raw.distill_step(z.detach(), index, logit, torch.ones(3))
    for t in (got, step):
        assert t[0].isnan().all() and t[1:].isfinite().all()
