"""Measured cases of the packed-document operators: attention over documents of different lengths packed
into one token axis, log-probabilities of given tokens with entropy and top alternatives, and the loss
against a teacher's top logits.

`run` computes an operator in its plain form (elementary torch operations in 32 bits) or, where `own` is
set, through the framework's entry points. `exact` computes the same outputs from the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a handful of short prompts scored at once: latency
        {"name": "attn_short", "op": "attn", "train": False, "docs": 12, "longest": 61, "tokens": 256, "heads": 16,
         "kv_heads": 4, "dim": 64, "causal": True, "dtype": "bf16", "spare": 5},
        # one micro-batch of the 1.3B configuration (16 heads of 128) filled with documents
        {"name": "attn_docs", "op": "attn", "train": False, "docs": 9, "longest": 2048, "tokens": 8192, "heads": 16,
         "kv_heads": 16, "dim": 128, "causal": True, "dtype": "bf16", "spare": 0},
        # one long document, grouped heads
        {"name": "attn_long_grouped", "op": "attn", "train": False, "docs": 1, "longest": 8192, "tokens": 8192,
         "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "dtype": "bf16", "spare": 0},
        # training step on the same micro-batch of documents, fp16 as the benchmark trains
        {"name": "attn_docs_train", "op": "attn", "train": True, "docs": 9, "longest": 2048, "tokens": 8192, "heads": 16,
         "kv_heads": 16, "dim": 128, "causal": True, "dtype": "fp16", "spare": 0},
        # training step, grouped heads, documents up to 4k tokens of odd lengths, a padded end
        {"name": "attn_grouped_train", "op": "attn", "train": True, "docs": 5, "longest": 4096, "tokens": 8183,
         "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "dtype": "bf16", "spare": 9},
        # many short documents, few shared heads
        {"name": "attn_ragged_train", "op": "attn", "train": True, "docs": 40, "longest": 317, "tokens": 4001,
         "heads": 16, "kv_heads": 2, "dim": 64, "causal": True, "dtype": "bf16", "spare": 0},
        # scores of the last tokens of a few prompts, with alternatives: latency; masked padding columns
        {"name": "logprob_few", "op": "logprob", "train": False, "rows": 4, "vocab": 50304, "masked": 47, "top": 8,
         "temperature": 1.0, "dtype": "bf16"},
        # a teacher scores a whole micro-batch and reports its top alternatives
        {"name": "logprob_teacher", "op": "logprob", "train": False, "rows": 8192, "vocab": 50304, "masked": 0, "top": 32,
         "temperature": 1.0, "dtype": "bf16"},
        # policy-gradient step: log-probability and entropy with their gradient
        {"name": "logprob_train", "op": "logprob", "train": True, "rows": 4096, "vocab": 51200, "masked": 0, "top": 0,
         "temperature": 0.8, "dtype": "fp16"},
        # unpadded vocabulary in 32 bits (odd row pitch), a small batch
        {"name": "distill_odd", "op": "distill", "train": True, "rows": 250, "vocab": 50257, "top": 20,
         "temperature": 1.0, "dtype": "fp32", "step": False},
        # autograd distillation of a large vocabulary
        {"name": "distill_wide", "op": "distill", "train": True, "rows": 2048, "vocab": 128000, "top": 64,
         "temperature": 2.0, "dtype": "bf16", "step": False},
        # the last stage of a training step: loss and gradient of a micro-batch in one call
        {"name": "distill_step", "op": "distill", "train": True, "rows": 8192, "vocab": 50304, "top": 32,
         "temperature": 1.0, "dtype": "bf16", "step": True},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("attn", "logprob", "distill"))
    if op == "attn":
        tokens = _log_int(rng, 48, 8192)
        docs = _log_int(rng, 1, max(1, min(64, tokens // 8)))
        longest = min(4096, tokens, max(1, int(math.ceil(tokens / docs * rng.uniform(1.0, 3.0)))))
        heads, kv_heads = rng.choice(((16, 16), (16, 4), (32, 8), (8, 1), (12, 2), (7, 7), (9, 3), (16, 2)))
        return {"op": op, "train": rng.random() < 0.5, "docs": docs, "longest": longest, "tokens": tokens, "heads": heads,
                "kv_heads": kv_heads, "dim": rng.choice((64, 128)), "causal": rng.random() < 0.8,
                "dtype": rng.choice(("bf16", "fp16")), "spare": rng.choice((0, 0, rng.randint(1, 200)))}
    vocab = _log_int(rng, 1000, 131072)
    if rng.random() < 0.5:
        vocab = (vocab + 127) // 128 * 128
    rows = _log_int(rng, 1, max(1, min(8192, 200_000_000 // vocab)))
    case = {"op": op, "rows": rows, "vocab": vocab, "temperature": rng.choice((1.0, 1.0, 0.7, 2.0)),
            "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32"))}
    if op == "logprob":
        train = rng.random() < 0.4
        return {**case, "train": train, "masked": rng.choice((0, rng.randint(1, 100))),
                "top": 0 if train else rng.choice((0, 1, rng.randint(2, 64)))}
    return {**case, "train": True, "top": rng.randint(1, 100), "step": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Document lengths of a case: they sum to `tokens`, none is longer than `longest`, and with several
    documents one has a single token where the sum allows it."""
    docs, tokens = case["docs"], case["tokens"]
    rng = np.random.default_rng((docs, tokens, case["heads"], case["dim"]))
    longest = max(case["longest"], -(-tokens // docs))
    weights = rng.exponential(1.0, docs) + 0.05
    lengths = np.minimum(np.maximum((weights / weights.sum() * tokens).astype(np.int64), 1), longest)
    if docs > 2 and tokens - 1 <= (docs - 1) * longest:
        lengths[rng.integers(docs)] = 1
    while lengths.sum() != tokens:
        short = int(tokens - lengths.sum())
        room = longest - lengths if short > 0 else lengths - 1
        free = np.nonzero(room > 0)[0]
        part = -(-abs(short) // len(free))
        for i in rng.permutation(free):
            step = min(part, int(room[i]), abs(int(tokens - lengths.sum())))
            lengths[i] += step if short > 0 else -step
    return [int(n) for n in lengths]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return torch.randn(shape, generator=g, device=DEVICE, dtype=dtype).mul_(scale)

    if case["op"] == "attn":
        lengths = _lengths(case)
        total = sum(lengths) + case["spare"]
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        # the projections of a block leave q, k and v side by side in one buffer
        qkv = normal(total, h + 2 * hk, d)
        state = {"case": case, "lengths": lengths, "q": qkv[:, :h], "k": qkv[:, h:h + hk], "v": qkv[:, h + hk:]}
        # the plain form's plan: padded positions of the packed rows
        starts = np.concatenate([[0], np.cumsum(lengths)[:-1]])
        doc = np.repeat(np.arange(len(lengths)), lengths)
        state["doc"] = torch.from_numpy(doc).to(DEVICE)
        state["pos"] = torch.from_numpy(np.arange(len(doc)) - starts[doc]).to(DEVICE)
        state["len"] = torch.tensor(lengths, device=DEVICE)
        if case["train"]:
            state["d_out"] = normal(total, h, d)
            for name in "qkv":
                state[name].requires_grad_(True)
        if own:
            from eth_b200 import ops
            state["layout"] = ops.PackedLayout(lengths, device=DEVICE, total=total)
        return state

    rows, vocab, k = case["rows"], case["vocab"], case["top"]
    logits = normal(rows, vocab, scale=2.5)
    state = {"case": case, "logits": logits}
    if case["op"] == "logprob":
        state["tokens"] = torch.randint(vocab - case["masked"], (rows,), generator=g, device=DEVICE)
        if case["masked"]:
            logits[:, vocab - case["masked"]:] = float("-inf")
        if case["train"]:
            logits.requires_grad_(True)
            state["d_logprob"] = normal(rows, dtype=torch.float32)
            state["d_entropy"] = normal(rows, scale=0.1, dtype=torch.float32)
        return state
    # the teacher's alternatives: distinct tokens of falling log-probability, some lists shorter, some rows empty
    first = torch.randint(vocab, (rows, 1), generator=g, device=DEVICE)
    state["index"] = (first + torch.arange(k, device=DEVICE) * 7) % vocab
    tl = normal(rows, k, scale=1.5, dtype=torch.float32).sort(1, descending=True).values - 2.0
    kept = torch.randint(-1, 3 * k, (rows, 1), generator=g, device=DEVICE)
    state["teacher"] = tl.masked_fill(torch.arange(k, device=DEVICE) > kept, float("-inf")).contiguous()
    state["d_loss"] = normal(rows, dtype=torch.float32).abs_().add_(0.1)
    if not case["step"]:
        logits.requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------------ plain forms
def _padded(x, s, docs, longest):
    """[documents, heads, longest, dim] in 32 bits from packed rows."""
    out = x.new_zeros((docs, longest, x.shape[1], x.shape[2]), dtype=torch.float32)
    out[s["doc"], s["pos"]] = x[:len(s["doc"])].float()
    return out.transpose(1, 2)


def _packed(x, s, like):
    """Packed rows of the type of `like`; rows behind the last document are zero."""
    out = torch.zeros_like(like, memory_format=torch.contiguous_format)
    out[:len(s["doc"])] = x.transpose(1, 2)[s["doc"], s["pos"]].to(like.dtype)
    return out


@torch.no_grad()
def _attn_plain(s):
    case = s["case"]
    docs, longest = len(s["lengths"]), max(s["lengths"])
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    scale = 1.0 / math.sqrt(d)
    q = _padded(s["q"], s, docs, longest).unflatten(1, (hk, h // hk))
    k = _padded(s["k"], s, docs, longest).unsqueeze(2)
    v = _padded(s["v"], s, docs, longest).unsqueeze(2)
    at = torch.arange(longest, device=DEVICE)
    seen = (at[None, None, :] < s["len"][:, None, None]).expand(docs, longest, longest)
    if case["causal"]:
        seen = seen & (at[None, :, None] >= at[None, None, :])
    x = (q @ k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen[:, None, None], float("-inf"))
    p = x.sub_(x.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    out = (p @ v).flatten(1, 2)
    if not case["train"]:
        return _packed(out, s, s["q"])
    do = _padded(s["d_out"], s, docs, longest).unflatten(1, (hk, h // hk))
    dv = (p.transpose(-1, -2) @ do).sum(2)
    dp = do @ v.transpose(-1, -2)
    ds = p.mul_(dp.sub_((do * out.unflatten(1, (hk, h // hk))).sum(-1, keepdim=True))).mul_(scale)
    dq = (ds @ k).flatten(1, 2)
    dk = (ds.transpose(-1, -2) @ q).sum(2)
    return {"out": _packed(out, s, s["q"]), "dq": _packed(dq, s, s["q"]), "dk": _packed(dk, s, s["k"]),
            "dv": _packed(dv, s, s["v"])}


@torch.no_grad()
def _logprob_plain(s):
    case = s["case"]
    x = s["logits"].float() / case["temperature"]
    lse = torch.log(torch.exp(x - x.amax(1, keepdim=True)).sum(1, keepdim=True)) + x.amax(1, keepdim=True)
    logp = x - lse
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(1)
    out = {"logprob": logp.gather(1, s["tokens"][:, None])[:, 0], "entropy": entropy}
    if case["top"]:
        order = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True).indices[:, :case["top"]]
        out["top_logprob"], out["top_index"] = logp.gather(1, order), order
    if case["train"]:
        dx = -p * s["d_logprob"][:, None] - torch.where(p > 0, p * (logp + entropy[:, None]), 0.0) * s["d_entropy"][:, None]
        dx.scatter_add_(1, s["tokens"][:, None], s["d_logprob"][:, None])
        out["dlogits"] = (dx / case["temperature"]).to(s["logits"].dtype)
    return out


@torch.no_grad()
def _distill_plain(s):
    case = s["case"]
    x = s["logits"].float() / case["temperature"]
    logp = x - torch.log(torch.exp(x - x.amax(1, keepdim=True)).sum(1, keepdim=True)) - x.amax(1, keepdim=True)
    t = s["teacher"] / case["temperature"]
    some = t.amax(1, keepdim=True) > float("-inf")
    e = torch.where(some, torch.exp(t - t.amax(1, keepdim=True)), 0.0)
    total = e.sum(1, keepdim=True).clamp_min(1e-30)
    q = e / total
    log_q = t - t.amax(1, keepdim=True) - torch.log(total)
    loss = torch.where(q > 0, q * (log_q - logp.gather(1, s["index"])), 0.0).sum(1)
    dx = torch.exp(logp) * q.sum(1, keepdim=True)
    dx.scatter_add_(1, s["index"], -q)
    return {"loss": loss, "dlogits": (dx * (s["d_loss"][:, None] / case["temperature"])).to(s["logits"].dtype)}


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if not own:
        return {"attn": _attn_plain, "logprob": _logprob_plain, "distill": _distill_plain}[case["op"]](state)
    from eth_b200 import ops
    if case["op"] == "attn":
        out = ops.flash_attention_packed(state["q"], state["k"], state["v"], state["layout"], causal=case["causal"])
        if not case["train"]:
            return out
        dq, dk, dv = torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["d_out"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if case["op"] == "logprob":
        r = ops.token_logprobs(state["logits"], state["tokens"], top_k=case["top"], temperature=case["temperature"])
        out = {"logprob": r.logprob.detach(), "entropy": r.entropy.detach()}
        if case["top"]:
            out["top_logprob"], out["top_index"] = r.top_logprob, r.top_index
        if case["train"]:
            out["dlogits"], = torch.autograd.grad((r.logprob, r.entropy), state["logits"],
                                                  (state["d_logprob"], state["d_entropy"]))
        return out
    if case["step"]:
        loss, dlogits = ops.raw.distill_step(state["logits"], state["index"], state["teacher"], state["d_loss"],
                                             temperature=case["temperature"])
        return {"loss": loss, "dlogits": dlogits}
    loss = ops.topk_distillation_loss(state["logits"], state["index"], state["teacher"], temperature=case["temperature"])
    dlogits, = torch.autograd.grad(loss, state["logits"], state["d_loss"])
    return {"loss": loss.detach(), "dlogits": dlogits}


def work(case):
    if case["op"] == "attn":
        lengths = np.asarray(_lengths(case), dtype=np.float64)
        pairs = float((lengths * (lengths + 1) / 2).sum() if case["causal"] else (lengths ** 2).sum())
        rows, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        moved = 2 * rows * d * (2 * h + 2 * hk)                     # q, k, v in, o out; 16-bit types
        flops = 4 * d * h * pairs                                   # scores and context
        if case["train"]:
            moved += 2 * rows * d * (2 * h + 2 * hk)                # d_out in, dq, dk, dv out
            flops += 10 * d * h * pairs                             # scores again, dP, dV, dK, dQ
        return {"bytes": moved, "flops": flops}
    n = case["rows"] * case["vocab"]
    size = 4 if case["dtype"] == "fp32" else 2
    passes = 2 if case["train"] else 1
    side = case["rows"] * (16 + 12 * case["top"])
    return {"bytes": n * size * passes + side, "flops": n * (8 if case["train"] else 5)}


# ------------------------------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attn": _attn_exact, "logprob": _logprob_exact, "distill": _distill_exact}[case["op"]](case, s)


def _attn_exact(case, s):
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    group, scale = h // hk, d ** -0.5
    total = s["q"].shape[0]
    out = torch.zeros(total, h, d, dtype=torch.float64, device=DEVICE)
    grads = [torch.zeros(total, n, d, dtype=torch.float64, device=DEVICE) for n in (h, hk, hk)]
    first = 0
    for n in s["lengths"]:
        rows = slice(first, first + n)
        first += n
        hidden = torch.ones(n, n, dtype=torch.bool, device=DEVICE).triu(1) if case["causal"] else None
        for head in range(h):
            q, k, v = (s[name][rows, i].double() for name, i in (("q", head), ("k", head // group), ("v", head // group)))
            x = scale * torch.mm(q, k.t())
            if hidden is not None:
                x[hidden] = -math.inf
            p = torch.softmax(x, 1)
            out[rows, head] = torch.mm(p, v)
            if case["train"]:
                do = s["d_out"][rows, head].double()
                dp = torch.mm(do, v.t())
                ds = scale * p * (dp - (p * dp).sum(1, keepdim=True))
                grads[0][rows, head] = torch.mm(ds, k)
                grads[1][rows, head // group] += torch.mm(ds.t(), q)
                grads[2][rows, head // group] += torch.mm(p.t(), do)
    if not case["train"]:
        return out
    return {"out": out, "dq": grads[0], "dk": grads[1], "dv": grads[2]}


def _chunks(rows, vocab):
    step = max(1, (1 << 27) // vocab)
    return [slice(i, min(rows, i + step)) for i in range(0, rows, step)]


def _logprob_exact(case, s):
    logprob, entropy, tops, grads = [], [], [], []
    for c in _chunks(case["rows"], case["vocab"]):
        z = s["logits"][c].double()
        logp = torch.log_softmax(z / case["temperature"], 1)
        p = logp.exp()
        ent = torch.special.entr(p).sum(1)
        t = s["tokens"][c]
        logprob.append(logp[torch.arange(len(t), device=DEVICE), t])
        entropy.append(ent)
        if case["top"]:
            # distinct keys: the value first, then the lower token
            rank = torch.argsort(z, dim=1, descending=True, stable=True)[:, :case["top"]]
            tops.append((torch.take_along_dim(logp, rank, 1), rank))
        if case["train"]:
            u = torch.nan_to_num(logp, neginf=0.0)
            gz = -p * (s["d_logprob"][c].double()[:, None] + s["d_entropy"][c].double()[:, None] * (u + ent[:, None]))
            gz[torch.arange(len(t), device=DEVICE), t] += s["d_logprob"][c].double()
            grads.append((gz / case["temperature"]).to(torch.float64))
    out = {"logprob": torch.cat(logprob), "entropy": torch.cat(entropy)}
    if case["top"]:
        out["top_logprob"], out["top_index"] = (torch.cat(x) for x in zip(*tops))
    if case["train"]:
        out["dlogits"] = torch.cat(grads)
    return out


def _distill_exact(case, s):
    losses = []
    grad = torch.empty(case["rows"], case["vocab"], dtype=torch.float64, device=DEVICE)
    for c in _chunks(case["rows"], case["vocab"]):
        logp = torch.log_softmax(s["logits"][c].double() / case["temperature"], 1)
        t = s["teacher"][c].double() / case["temperature"]
        empty = torch.isinf(t).all(1, keepdim=True)
        log_q = torch.log_softmax(t.masked_fill(empty, 0.0), 1)
        q = log_q.exp().masked_fill(empty, 0.0)
        picked = torch.take_along_dim(logp, s["index"][c], 1)
        losses.append((torch.xlogy(q, q) - q * picked).sum(1))
        weight = torch.zeros_like(logp).scatter_add_(1, s["index"][c], q)
        grad[c] = (logp.exp() * q.sum(1, keepdim=True) - weight) * (s["d_loss"][c].double()[:, None] / case["temperature"])
    return {"loss": torch.cat(losses), "dlogits": grad}
