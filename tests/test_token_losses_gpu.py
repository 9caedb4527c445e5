"""Vocabulary kernels (token log-probabilities with entropy and alternatives, distillation) against
their definitions in 64 bits."""
import itertools
import math

import pytest
import torch

from eth_b200 import ops
from eth_b200.ops import raw
from helpers import oracle_tokens as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
#: rows, vocabulary, row pitch beyond the vocabulary, elements before the first row
SHAPES = [(1, 1, 0, 0), (1, 50304, 0, 0), (3, 7, 0, 0), (5, 1000, 24, 0), (7, 1003, 5, 3), (40, 5003, 0, 1),
          (300, 4099, 0, 0), (297, 50257, 47, 0), (2, 131071, 0, 0)]


def _logits(rows, vocab, pad, lead, dtype, seed=0, scale=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    flat = torch.randn(lead + rows * (vocab + pad), generator=g, device=DEV).mul_(scale).to(dtype)
    return flat[lead:].view(rows, vocab + pad)[:, :vocab], g


def _teacher(rows, vocab, k, g):
    index = torch.randint(vocab, (rows, k), generator=g, device=DEV)
    logit = torch.randn(rows, k, generator=g, device=DEV)
    used = (torch.arange(rows, device=DEV) * 5 % (2 * k + 1))[:, None]       # shorter lists, empty rows
    return index, logit.masked_fill(torch.arange(k, device=DEV) >= used, -math.inf)


def _close(got, want, tol):
    """`tol` covers the statistics. A result far from 0 (a token masked with fp16's lowest value lies 65504
    below the others) also carries the roundings of its last two fp32 steps, 2^-24 of itself each."""
    return (((got - want).abs() <= tol + 2.0 ** -23 * want.abs()) | (got == want)).all()     # -inf equals -inf


def _same_scores(r, logits, tokens, top_k, temperature):
    lp, ent, top_lp, top_id, _ = oracle.scores(logits, tokens, top_k, temperature)
    tol = oracle.statistic_tolerance(logits, temperature)
    assert _close(r.logprob, lp, tol) and _close(r.entropy, ent, tol)
    if top_k:
        assert torch.equal(r.top_index, top_id) and _close(r.top_logprob, top_lp, tol[:, None])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("top_k", [0, 1, 20, 128])
def test_token_logprobs_forward(dtype, shape, top_k):
    rows, vocab = shape[:2]
    logits, g = _logits(*shape, dtype)
    top_k = min(top_k, vocab)
    tokens = torch.randint(vocab, (rows,), generator=g, device=DEV)
    for temperature in (1.0, 0.6):
        _same_scores(ops.token_logprobs(logits, tokens, top_k, temperature), logits, tokens, top_k, temperature)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [130, 5003, 50304])
@pytest.mark.parametrize("top_k", [3, 128])
def test_ties_and_masks(dtype, vocab, top_k):
    """Rows where the first bound on the k-th alternative is loose, empty or reached by everything."""
    low = torch.finfo(dtype).min
    z, g = _logits(12, vocab, 0, 0, dtype, seed=1)
    z[0] = 0                                          # all equal
    z[1] = low                                        # the type's lowest value everywhere
    z[2] = -math.inf
    z[2, vocab // 2:] = 1.0                           # many equal behind masked ones
    z[3, 1:] = -math.inf                              # one token left
    z[4] = z[4].round()                               # a handful of distinct values
    z[5] = 0
    z[5, ::2] = -0.0                                  # both zeros are one value
    z[6, 2:] = low
    z[7] = -torch.arange(vocab, device=DEV).to(dtype)
    z[8] = torch.arange(vocab, device=DEV).to(dtype) / vocab
    z[9] = torch.finfo(dtype).smallest_normal / 4     # subnormal, above, equal and below zero
    z[9, ::3] *= -1
    z[9, 5] *= 2
    z[10, :] = 1.0
    z[10, -top_k:] = 2.0
    z[11, 17:33] = 30.0
    tokens = torch.zeros(12, dtype=torch.long, device=DEV)
    _same_scores(ops.token_logprobs(z, tokens, top_k), z, tokens, top_k, 1.0)


@pytest.mark.parametrize("rows,vocab,top_k,dtype", [(150, 32768, 64, torch.bfloat16), (150, 32768, 64, torch.float16),
                                                    (150, 16384, 64, torch.float32), (150, 65536, 100, torch.bfloat16),
                                                    (3, 262144, 128, torch.bfloat16), (3, 131072, 128, torch.float32)])
def test_rows_of_whole_segments(rows, vocab, top_k, dtype):
    """Vocabularies that fill every thread's segments exactly, in rows where all of them hold candidates."""
    z, g = _logits(rows, vocab, 0, 0, dtype, seed=12)
    z[0] = -math.inf
    z[1] = 2.0
    z[2] = torch.finfo(dtype).min
    tokens = torch.randint(vocab, (rows,), generator=g, device=DEV)
    r = ops.token_logprobs(z, tokens, top_k)
    order = torch.sort(z.double(), dim=1, descending=True, stable=True).indices[:, :top_k]
    assert torch.equal(r.top_index, order)
    _same_scores(ops.token_logprobs(z[1:], tokens[1:], top_k), z[1:], tokens[1:], top_k, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_undefined_rows_and_tokens(dtype):
    z, g = _logits(7, 6000, 0, 0, dtype, seed=2)
    z[0] = -math.inf
    z[1, 77] = math.nan
    z[2, 5001] = math.inf
    z[3] = math.nan
    tokens = torch.tensor([0, 1, 2, 3, -1, 6000, 1 << 40], device=DEV)
    r = ops.token_logprobs(z, tokens, top_k=9)
    assert r.logprob[:4].isnan().all() and r.entropy[:4].isnan().all()
    assert r.logprob[4] == 0 and r.logprob[5:].isnan().all() and r.entropy[4:].isfinite().all()
    order = torch.sort(z.double(), dim=1, descending=True, stable=True).indices[:, :9]   # NaN first, as torch sorts
    assert torch.equal(r.top_index, order)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("which", ["logprob", "entropy", "top", "all"])
def test_token_logprobs_backward(dtype, shape, which):
    rows, vocab = shape[:2]
    logits, g = _logits(*shape, dtype, seed=3)
    logits.requires_grad_(True)
    top_k = min(11, vocab)
    tokens = torch.randint(-1, vocab, (rows,), generator=g, device=DEV)
    r = ops.token_logprobs(logits, tokens, top_k=top_k, temperature=0.8)
    outs = {"logprob": r[:1], "entropy": r[1:2], "top": r[2:3], "all": r[:3]}[which]
    d = [torch.randn(x.shape, generator=g, device=DEV) for x in outs]
    for x in d:
        x[rows // 2] = 0                              # a row without any gradient
    got, = torch.autograd.grad(outs, logits, d)
    full = dict(zip({"logprob": "g", "entropy": "h", "top": "u", "all": "ghu"}[which], d))
    want = oracle.scores_grad(logits, tokens, r.top_index, full.get("g"), full.get("h"), full.get("u"), 0.8)
    # p is off by 2^-22 of itself and of its exponent (up to 60); p log p by the same of at most p |log p| <= 0.37
    assert oracle.grad_error(got, want, sum(x.abs().reshape(rows, -1).sum(1) for x in d) * 2.0 ** -17) <= 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("k", [1, 32, 512])
def test_distillation(dtype, shape, k):
    rows, vocab = shape[:2]
    logits, g = _logits(*shape, dtype, seed=4)
    logits.requires_grad_(True)
    index, logit = _teacher(rows, vocab, k, g)        # 512 entries over small vocabularies list ids many times
    dloss = torch.randn(rows, generator=g, device=DEV)
    dloss[rows // 2] = 0
    for temperature in (1.0, 2.0):
        loss = ops.topk_distillation_loss(logits, index, logit, temperature)
        want_loss, want = oracle.distill(logits, index, logit, dloss, temperature)
        assert ((loss - want_loss).abs() <= oracle.statistic_tolerance(logits, temperature)).all()
        got, = torch.autograd.grad(loss, logits, dloss)
        noise = dloss.abs() * 2.0 ** -17
        assert oracle.grad_error(got, want, noise) <= 1
        loss2, got2 = raw.distill_step(logits.detach(), index, logit, dloss, temperature)
        assert ((loss2 - want_loss).abs() <= oracle.statistic_tolerance(logits, temperature)).all()
        assert oracle.grad_error(got2, want, noise) <= 1
    buf = torch.full((rows, vocab + 9), 7.0, dtype=dtype, device=DEV)
    out = buf[:, :vocab]                              # another offset and pitch than the logits
    loss3, _ = raw.distill_step(logits.detach(), index, logit, dloss, temperature, out=out)
    assert torch.equal(out, got2) and torch.equal(loss3, loss2) and (buf[:, vocab:] == 7).all()
    buf = torch.full((rows, vocab + 9), 7.0, dtype=dtype, device=DEV)
    buf[:, :vocab] = logits.detach()
    loss4, _ = raw.distill_step(buf[:, :vocab], index, logit, dloss, temperature, out=buf[:, :vocab])
    assert oracle.grad_error(buf[:, :vocab].contiguous(), want, noise) <= 1 and (buf[:, vocab:] == 7).all()


def test_low_rows_and_extreme_temperatures():
    """Rows around the floor that keeps masked logits finite, and temperatures that stretch or flatten it."""
    z, g = _logits(8, 3001, 0, 0, torch.bfloat16, seed=15)
    z -= torch.tensor([0.0, 57000.0, 57344.0, 57600.0, 59900.0, 1e6, 1e30, 1e38], device=DEV)[:, None].to(z.dtype)
    z[:, ::7] = -math.inf
    tokens = torch.full((8,), 3, device=DEV)
    for temperature in (0.01, 1.0, 1e4, 1e30):
        zr = z.clone().requires_grad_(True)
        r = ops.token_logprobs(zr, tokens, 5, temperature)
        _same_scores(r, z, tokens, 5, temperature)
        d = [torch.randn(8, generator=g, device=DEV) for _ in range(2)]
        got, = torch.autograd.grad(r[:2], zr, d)
        want = oracle.scores_grad(z, tokens, None, *d, None, temperature)
        noise = sum(x.abs() for x in d) * (2.0 ** -17 / temperature)
        assert oracle.grad_error(got, want, noise) <= 1


def test_unused_entries_and_strangers():
    z, g = _logits(4, 3000, 0, 0, torch.bfloat16)
    z.requires_grad_(True)
    index = torch.tensor([[5, -9, 1 << 40], [2999, 2999, 2999], [7, 3000, 8], [1, 2, 3]], device=DEV)
    logit = torch.tensor([[0.5, -math.inf, -math.inf], [0.0, 1.0, -1.0], [0.0, 0.0, 0.0],
                          [math.nan, 0.0, 0.0]], device=DEV)
    loss = ops.topk_distillation_loss(z, index, logit)
    want, grad = oracle.distill(z[:2], index[:2], logit[:2], torch.ones(2, device=DEV), 1.0)
    assert ((loss[:2] - want).abs() < 1e-5).all() and loss[2:].isnan().all()
    got, = torch.autograd.grad(loss[:2].sum(), z)
    assert oracle.grad_error(got[:2], grad, torch.full((2,), 2.0 ** -17, device=DEV)) <= 1 and (got[2:] == 0).all()


@pytest.mark.parametrize("world", [2, 3])
@pytest.mark.parametrize("dtype", DTYPES)
def test_vocabulary_shards(dtype, world):
    part, rows, k = 2051, 33, 40
    logits, g = _logits(rows, part * world, 0, 0, dtype, seed=6)
    logits[1, :part] = -math.inf
    logits[2] = 0.5
    tokens = torch.randint(part * world, (rows,), generator=g, device=DEV)
    index, logit = _teacher(rows, part * world, 17, g)
    shards = logits.split(part, 1)
    sent = {"scores": [], "distill": []}
    for w, z in enumerate(shards):
        for name, op, args in (("scores", ops.token_logprobs, (tokens, k)),
                               ("distill", ops.topk_distillation_loss, (index, logit))):
            op(z, *args, 0.9, w * part, lambda x: (sent[name].append(x), x.unsqueeze(0))[1])
    dloss = torch.randn(rows, generator=g, device=DEV)
    want_loss, want = oracle.distill(logits, index, logit, dloss, 0.9)
    _, _, _, top_id, _ = oracle.scores(logits, tokens, k, 0.9)
    want_z = oracle.scores_grad(logits, tokens, top_id, dloss, dloss, None, 0.9)
    for w in range(world):
        z = shards[w].detach().requires_grad_(True)
        r = ops.token_logprobs(z, tokens, k, 0.9, w * part, lambda x: torch.stack(sent["scores"]))
        _same_scores(r, logits, tokens, k, 0.9)
        loss = ops.topk_distillation_loss(z, index, logit, 0.9, w * part, lambda x: torch.stack(sent["distill"]))
        assert _close(loss, want_loss, oracle.statistic_tolerance(logits, 0.9))     # row 1 may be infinitely far off
        mine = slice(w * part, (w + 1) * part)
        got, = torch.autograd.grad(loss, z, dloss)
        assert oracle.grad_error(got, want[:, mine], dloss.abs() * 2.0 ** -17) <= 1
        got, = torch.autograd.grad((r.logprob, r.entropy), z, (dloss, dloss))
        assert oracle.grad_error(got, want_z[:, mine], dloss.abs() * 2.0 ** -16) <= 1


def test_same_bits_every_time():
    z, g = _logits(64, 50304, 0, 0, torch.bfloat16, seed=8)
    tokens = torch.randint(50304, (64,), generator=g, device=DEV)
    index, logit = _teacher(64, 50304, 100, g)
    first = None
    for _ in range(4):
        zr = z.detach().requires_grad_(True)
        r = ops.token_logprobs(zr, tokens, top_k=100)
        gz, = torch.autograd.grad((r.logprob.sum() + r.top_logprob.sum(),), zr)
        got = [*r, gz, *raw.distill_step(z, index, logit, r.logprob.detach())]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


def test_captured_and_on_another_stream():
    z, g = _logits(33, 5000, 0, 0, torch.bfloat16, seed=9)
    tokens = torch.randint(5000, (33,), generator=g, device=DEV)
    index, logit = _teacher(33, 5000, 10, g)
    dloss = torch.ones(33, device=DEV)
    logits = z.clone()

    def work():
        return [*raw.token_scores_fwd(logits, tokens, 5)[:4], *raw.distill_step(logits, index, logit, dloss)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    logits.copy_(z.flip(0))
    graph.replay()
    now = work()
    assert all(torch.equal(a, b) for a, b in zip(out, now))
    logits.copy_(z)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_offsets_beyond_32_bits():
    """3 rows, 2^30 elements apart, of one buffer: the last starts behind 2^31 elements."""
    pitch = 1 << 30
    flat = torch.empty(2 * pitch + 1024, dtype=torch.bfloat16, device=DEV)
    z = flat.as_strided((3, 1000), (pitch, 1))
    z.copy_(torch.randn(3, 1000, device=DEV))
    tokens = torch.tensor([0, 999, 500], device=DEV)
    _same_scores(ops.token_logprobs(z, tokens, 4), z.contiguous(), tokens, 4, 1.0)
    index, logit = torch.tensor([[1, 2], [3, 4], [5, 6]], device=DEV), torch.zeros(3, 2, device=DEV)
    want, grad = oracle.distill(z.contiguous(), index, logit, torch.ones(3, device=DEV), 1.0)
    loss, _ = raw.distill_step(z, index, logit, torch.ones(3, device=DEV), out=z)
    assert ((loss - want).abs() < 1e-5).all()
    assert oracle.grad_error(z.contiguous(), grad, torch.full((3,), 2.0 ** -17, device=DEV)) <= 1


def test_refusals_on_the_device():
    z, t = torch.randn(3, 11, device=DEV), torch.zeros(3, dtype=torch.long, device=DEV)
    index, logit = torch.zeros(3, 2, dtype=torch.long, device=DEV), torch.zeros(3, 2, device=DEV)
    for bad in (lambda: ops.token_logprobs(z, t.cpu()), lambda: ops.token_logprobs(z.double(), t),
                lambda: ops.topk_distillation_loss(z, index.cpu(), logit),
                lambda: ops.topk_distillation_loss(z, index, logit.cpu()),
                lambda: raw.distill_step(z, index, logit, torch.ones(3)),
                lambda: ops.token_logprobs(z[0], t), lambda: ops.token_logprobs(z.int(), t),
                lambda: ops.token_logprobs(z, t.int()), lambda: ops.token_logprobs(z, t[:2]),
                lambda: ops.token_logprobs(z, t, top_k=12), lambda: ops.token_logprobs(z, t, top_k=-1),
                lambda: ops.token_logprobs(torch.randn(3, 500, device=DEV), t, top_k=129),
                lambda: ops.token_logprobs(z, t, temperature=0.0), lambda: ops.token_logprobs(z, t, temperature=math.nan),
                lambda: ops.token_logprobs(z[:, :0], t),
                lambda: ops.token_logprobs(z, t, 2, 1.0, 0, lambda x: x),
                lambda: ops.topk_distillation_loss(z, index, logit[:, :1]),
                lambda: ops.topk_distillation_loss(z, index.int(), logit),
                lambda: ops.topk_distillation_loss(z, index, logit.half()),
                lambda: ops.topk_distillation_loss(z, index[:, :0], logit[:, :0]),
                lambda: ops.topk_distillation_loss(z, index.new_zeros(3, 513), logit.new_zeros(3, 513)),
                lambda: raw.distill_step(z, index, logit, torch.ones(2, device=DEV)),
                lambda: raw.distill_step(z, index, logit, torch.ones(3, device=DEV), out=z.half()),
                lambda: raw.distill_step(z[:, :10], index, logit, torch.ones(3, device=DEV), out=z[:, 1:])):
        with pytest.raises(ValueError):
            bad()


def _three_losses(z, order, g, **cross_entropy):
    """Label loss, teacher loss and scores of the same logits, their nodes built in `order`; with the
    gradients handed to them and the sum of the three in 64 bits (and of the magnitudes)."""
    rows, vocab = z.shape
    targets = torch.randint(vocab, (rows,), generator=g, device=DEV)
    index, logit = _teacher(rows, vocab, 9, g)
    build = {"cross entropy": lambda: ops.vocab_parallel_cross_entropy(z, targets, **cross_entropy),
             "distillation": lambda: ops.topk_distillation_loss(z, index, logit),
             "scores": lambda: ops.token_logprobs(z, targets)[:2]}
    outs, d, parts = [], [], []
    for name in order:
        out = build[name]()
        out = list(out) if name == "scores" else [out]
        dout = [torch.randn(rows, generator=g, device=DEV) for _ in out]
        outs, d = outs + out, d + dout
        if name == "distillation":
            parts.append(oracle.distill(z, index, logit, dout[0], 1.0)[1])
        elif name == "scores":
            parts.append(oracle.scores_grad(z, targets, None, *dout, None, 1.0))
        else:
            parts.append(oracle.scores_grad(z, targets, None, -dout[0], None, None, 1.0))
    return outs, d, sum(parts), sum(p.abs() for p in parts)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("order", list(itertools.permutations(("cross entropy", "distillation", "scores"))))
def test_losses_that_share_logits_with_cross_entropy(dtype, order):
    """Autograd runs the node that was built last first, so none may write over what the others have saved."""
    z, g = _logits(37, 4104, 0, 0, dtype, seed=21)
    before = z.clone()
    outs, d, want, size = _three_losses(z.requires_grad_(True), order, g)
    got, = torch.autograd.grad(outs, z, d)
    # each of the three is rounded once, and so are their two sums, which are at most `size`
    bound = torch.finfo(dtype).eps / 2 * 3.01 * size + sum(x.abs() for x in d)[:, None] * 2.0 ** -17 + 2.0 ** -23
    assert ((got.double() - want).abs() <= bound).all()
    assert torch.equal(z.detach(), before)


def test_cross_entropy_that_overwrites_is_noticed():
    """In the order that autograd can honour the results are right; in the other it raises."""
    z, g = _logits(37, 4104, 0, 0, torch.bfloat16, seed=27)
    order = ("cross entropy", "distillation", "scores")
    outs, d, want, size = _three_losses(z.requires_grad_(True), order, g, overwrite_logits=True)
    got, = torch.autograd.grad(outs, z, d)
    bound = torch.finfo(z.dtype).eps / 2 * 3.01 * size + sum(x.abs() for x in d)[:, None] * 2.0 ** -17
    assert ((got.double() - want).abs() <= bound).all()
    for order in (("distillation", "cross entropy"), ("scores", "cross entropy")):
        z = _logits(37, 4104, 0, 0, torch.bfloat16, seed=28)[0].requires_grad_(True)
        outs, d, _, _ = _three_losses(z, order, g, overwrite_logits=True)
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(outs, z, d)


def test_step_into_saved_logits_is_noticed():
    """The gradient that replaces the logits must not pass for them in a backward that comes later."""
    z, g = _logits(5, 1003, 0, 0, torch.bfloat16, seed=22)
    index, logit = _teacher(5, 1003, 4, g)
    tokens, ones = torch.zeros(5, dtype=torch.long, device=DEV), torch.ones(5, device=DEV)
    for build in (lambda x: ops.token_logprobs(x, tokens).logprob, lambda x: ops.topk_distillation_loss(x, index, logit)):
        leaf = z.clone().requires_grad_(True)
        loss = build(leaf)
        raw.distill_step(leaf.detach(), index, logit, ones, out=leaf.detach())
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(loss, leaf, ones)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_a_token_outside_the_vocabulary(dtype):
    """NaN where the log-probability is NaN and has a gradient; the entropy's own gradient stays defined."""
    z, g = _logits(5, 6000, 0, 0, dtype, seed=23)
    z.requires_grad_(True)
    tokens = torch.tensor([6000, 1 << 40, 5999, -1, 6000], device=DEV)
    r = ops.token_logprobs(z, tokens)
    assert r.logprob[[0, 1, 4]].isnan().all()
    d = torch.ones(5, device=DEV)
    d[4] = 0
    got, = torch.autograd.grad(r.logprob, z, d, retain_graph=True)
    assert got[:2].isnan().all() and got[2].isfinite().all() and (got[3:] == 0).all()
    got, = torch.autograd.grad(r.entropy, z, torch.ones(5, device=DEV))
    want = oracle.scores_grad(z, torch.zeros_like(tokens), None, None, torch.ones(5, device=DEV), None, 1.0)
    assert oracle.grad_error(got, want, torch.full((5,), 2.0 ** -17, device=DEV)) <= 1


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_a_token_outside_sharded_vocabularies(dtype):
    part, world = 3001, 2
    logits, g = _logits(4, part * world, 0, 0, dtype, seed=24)
    tokens = torch.tensor([part * world, 17, part, -1], device=DEV)
    shards, sent = logits.split(part, 1), []
    for w, z in enumerate(shards):
        ops.token_logprobs(z, tokens, 0, 1.0, w * part, lambda x: (sent.append(x), x.unsqueeze(0))[1])
    for w, z in enumerate(shards):
        z = z.detach().requires_grad_(True)
        r = ops.token_logprobs(z, tokens, 0, 1.0, w * part, lambda x: torch.stack(sent))
        got, = torch.autograd.grad(r.logprob.sum(), z)
        assert got[0].isnan().all() and got[1:3].isfinite().all() and (got[3] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_a_list_with_an_entry_outside_the_vocabulary(dtype):
    z, g = _logits(4, 3000, 0, 0, dtype, seed=25)
    index = torch.tensor([[5, 3000], [2999, -3], [7, 8], [9, 3000]], device=DEV)
    logit = torch.tensor([[0.0, -40.0], [0.5, 0.0], [0.0, 1.0], [0.0, -math.inf]], device=DEV)
    leaf = z.clone().requires_grad_(True)
    ones = torch.ones(4, device=DEV)
    loss = ops.topk_distillation_loss(leaf, index, logit)
    assert loss[:2].isnan().all() and loss[2:].isfinite().all()
    got, = torch.autograd.grad(loss, leaf, ones)
    _, step = raw.distill_step(z, index, logit, ones)
    sent, part = [], 1500
    for w, x in enumerate(z.split(part, 1)):
        ops.topk_distillation_loss(x, index, logit, 1.0, w * part, lambda s: (sent.append(s), s.unsqueeze(0))[1])
    shards = []
    for w, x in enumerate(z.split(part, 1)):
        x = x.detach().requires_grad_(True)
        loss = ops.topk_distillation_loss(x, index, logit, 1.0, w * part, lambda s: torch.stack(sent))
        shards.append(torch.autograd.grad(loss, x, ones)[0])
    for t in (got, step, torch.cat(shards, 1)):
        assert t[:2].isnan().all() and t[2:].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature", [1.0, 1e-20, 1e-30])
def test_forced_tokens(dtype, temperature):
    """One logit so far above the others that their distance in units of the temperature passes what fp32
    holds: probability 1, entropy 0 and no gradient, not NaN."""
    info = torch.finfo(dtype)
    z, g = _logits(6, 5003, 0, 0, dtype, seed=26)
    z[0, 17] = info.max
    z[1] = info.min
    z[1, 17] = info.max
    z[2, 17] = info.max / 4
    z[3, 17] = 200.0
    z[4] = -math.inf
    z[4, 17] = info.max
    z[5, 17] = 1000.0
    tokens = torch.full((6,), 17, device=DEV)
    z.requires_grad_(True)
    r = ops.token_logprobs(z, tokens, top_k=3, temperature=temperature)
    assert (r.logprob == 0).all() and (r.entropy == 0).all() and (r.top_index[:, 0] == 17).all()
    got, = torch.autograd.grad((r.logprob, r.entropy), z, [torch.ones(6, device=DEV)] * 2)
    assert (got == 0).all()
