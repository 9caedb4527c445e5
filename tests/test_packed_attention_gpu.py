"""Packed-document attention kernels against the definition in 64 bits, element by element."""
import contextlib
import math

import pytest
import torch

from eth_b200 import ops
from eth_b200.ops import native, raw
from helpers import oracle_packed as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16]
LENGTHS = {"one": [1], "ones": [1, 1, 1], "tile": [128], "tile+1": [129], "mixed": [127, 128, 0, 129, 1, 300],
           "blocks": [513, 64, 0, 256, 255], "long": [2048], "ragged": [17, 700, 33, 1, 90, 385, 128]}
HEADS = [(1, 1), (2, 1), (3, 1), (4, 4), (8, 2), (6, 2)]


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    native.check_status()


def _inputs(lengths, heads, kv_heads, dim, dtype, spare=0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows = sum(lengths) + spare
    qkv = torch.randn(rows, heads + 2 * kv_heads, dim, generator=g, device=DEV, dtype=dtype)
    do = torch.randn(rows, heads, dim, generator=g, device=DEV, dtype=dtype)
    return qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:], do


def _check(lengths, q, k, v, do, causal, scale=None, layout=None):
    layout = layout or ops.PackedLayout(lengths, device=DEV, total=q.shape[0])
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = ops.flash_attention_packed(*leaves, layout, scale=scale, causal=causal)
    grads = torch.autograd.grad(out, leaves, do)
    native.check_status()
    want = oracle.attention(q, k, v, lengths, causal, scale, do)
    for name, t in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)):
        assert oracle.excess(t, want[name]) <= 1, name
        assert (t[layout.used:] == 0).all(), name
    return [out.detach(), *grads]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", HEADS)
@pytest.mark.parametrize("name", list(LENGTHS))
@pytest.mark.parametrize("causal", [True, False])
def test_forward_and_backward(dtype, dim, heads, kv_heads, name, causal):
    lengths = LENGTHS[name]
    _check(lengths, *_inputs(lengths, heads, kv_heads, dim, dtype), causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads", [(16, 16), (16, 2), (32, 8)])
def test_more_tiles_than_sms(dtype, heads, kv_heads):
    lengths = [1024, 31, 700, 1, 256, 1500, 77, 129]
    _check(lengths, *_inputs(lengths, heads, kv_heads, 128, dtype, spare=3), True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (3, 3)])
def test_nothing_leaks_between_documents(causal, heads, kv_heads):
    """Infinities and NaN in one document and behind the last one leave the others bit for bit alone."""
    lengths, spare = [200, 57, 130, 1], 70
    q, k, v, do = (t.contiguous() for t in _inputs(lengths, heads, kv_heads, 128, torch.bfloat16, spare=spare))
    clean = _check(lengths, q, k, v, do, causal)
    rows = slice(200, 257)
    for t, bad in ((q, math.nan), (k, math.inf), (v, math.nan), (do, -math.inf)):
        t[rows] = bad
        t[sum(lengths):] = bad
    layout = ops.PackedLayout(lengths, device=DEV, total=q.shape[0])
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = ops.flash_attention_packed(*leaves, layout, causal=causal)
    grads = torch.autograd.grad(out, leaves, do)
    for a, b in zip((out.detach(), *grads), clean):
        assert torch.equal(a[:200], b[:200]) and torch.equal(a[257:], b[257:])


def test_growing_maximum_and_large_scores():
    lengths = [640, 257]
    q, k, v, do = (t.contiguous() for t in _inputs(lengths, 4, 2, 128, torch.bfloat16, seed=3))
    k.mul_(torch.linspace(0.2, 6.0, k.shape[0], device=DEV).view(-1, 1, 1).to(k.dtype))
    _check(lengths, q, k, v, do, True)
    _check(lengths, q, k, v, do, False, scale=0.5)


def test_layouts_of_the_operands():
    """Head-major storage, padded heads, expanded and misaligned operands, one gradient row for all."""
    lengths, h, hk, d = [150, 40], 4, 2, 64
    q, k, v, do = _inputs(lengths, h, hk, d, torch.float16, seed=4)
    rows = sum(lengths)
    want = _check(lengths, q.contiguous(), k.contiguous(), v.contiguous(), do, True)

    def padded(t):
        return torch.zeros(rows, t.shape[1], d + 8, dtype=t.dtype, device=DEV)[..., :d].copy_(t)

    def shifted(t):
        return torch.zeros(t.numel() + 3, dtype=t.dtype, device=DEV)[3:].view(t.shape).copy_(t)

    def odd(t):
        return torch.zeros(rows, t.shape[1] * d + 1, dtype=t.dtype, device=DEV)[:, 1:].view(rows, -1, d).copy_(t)
    for change in (lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), padded, shifted, odd,
                   lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
        got = _check(lengths, change(q), change(k), change(v), change(do), True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = k[:, :1].expand(-1, 2, -1)
    _check(lengths, q, one, one, do[:1].expand(rows, -1, -1), True)


def test_same_bits_every_time_and_on_another_stream():
    lengths = [300, 1, 513, 64]
    q, k, v, do = _inputs(lengths, 8, 2, 128, torch.bfloat16, seed=5)
    layout = ops.PackedLayout(lengths, device=DEV)
    first = _check(lengths, q, k, v, do, True, layout=layout)
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = _check(lengths, q, k, v, do, True, layout=layout)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("dtype", DTYPES)
def test_residue_holds_what_rounding_took(dtype):
    """At most half a step of out, and with it the gradients come closer."""
    lengths = [40, 300, 7, 128]
    q, k, v, do = _inputs(lengths, 8, 2, 64, dtype, spare=3, seed=16)
    layout = ops.PackedLayout(lengths, device=DEV, total=q.shape[0])
    out, lse, residue = raw.attention_packed_fwd(q, k, v, layout, with_residue=True)
    plain, _ = raw.attention_packed_fwd(q, k, v, layout)
    rows = slice(0, layout.used)
    assert torch.equal(out, plain)
    half = torch.finfo(dtype).eps / 2
    assert (residue[rows].float().abs() <= half * out[rows].float().abs() * 1.01 + 2.0 ** -25).all()
    want = oracle.attention(q, k, v, lengths, True, d_out=do)
    errors = []
    for r in (residue, None):
        grads = raw.attention_packed_bwd(do, q, k, v, out, lse, layout, residue=r)
        errors.append([((g.double() - want[n][0]).norm() / want[n][0].norm()).item()
                       for n, g in zip(("dq", "dk", "dv"), grads)])
    native.check_status()
    assert errors[0][0] < errors[1][0] and errors[0][1] < errors[1][1] and errors[0][2] == errors[1][2]


def test_captured_forward_and_backward():
    lengths = [300, 1, 130]
    q, k, v, do = (t.contiguous() for t in _inputs(lengths, 4, 2, 64, torch.bfloat16, spare=5, seed=6))
    layout = ops.PackedLayout(lengths, device=DEV, total=q.shape[0])

    def work():
        out, lse = raw.attention_packed_fwd(q, k, v, layout)
        return out, *raw.attention_packed_bwd(do, q, k, v, out, lse, layout)
    work()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                # two graphs over the same inputs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, work()))
    for step in range(3):
        q.copy_(torch.randn_like(q))
        v.mul_(-1)
        for graph, _ in graphs:
            graph.replay()
        eager = work()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_two_calls_at_once():
    """Forward and backward on two streams that run side by side, with few and with many units of work."""
    lengths = [1000, 3, 257, 700, 128]
    sets = [_inputs(lengths, 16, kv, 128, torch.bfloat16, seed=s) for s, kv in ((11, 16), (12, 2))]
    layout = ops.PackedLayout(lengths, device=DEV)
    alone = [_check(lengths, *x, True, layout=layout) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        outs = []
        for s, (q, k, v, do) in zip(streams, sets):
            with torch.cuda.stream(s):
                out, lse, residue = raw.attention_packed_fwd(q, k, v, layout, with_residue=True)
                outs.append([out, *raw.attention_packed_bwd(do, q, k, v, out, lse, layout, residue=residue)])
        torch.cuda.synchronize()
        native.check_status()
        for got, want in zip(outs, alone):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_autograd():
    lengths = [200, 70]
    q, k, v, do = (t.contiguous() for t in _inputs(lengths, 4, 2, 64, torch.float16, seed=13))
    layout = ops.PackedLayout(lengths, device=DEV)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]

    def work():
        out = ops.flash_attention_packed(*leaves, layout)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    with torch.no_grad():
        for t in leaves:
            t.copy_(torch.randn_like(t))
    graph.replay()
    torch.cuda.synchronize()
    native.check_status()
    want = oracle.attention(*leaves, lengths, True, d_out=do)
    for name, t in zip(("out", "dq", "dk", "dv"), got):
        assert oracle.excess(t, want[name]) <= 1, name


def test_offsets_beyond_32_bits():
    """Rows 2^24 elements apart: the last documents lie behind 2^31 elements of the buffer."""
    lengths, h, hk, d, pitch = [40, 100], 2, 1, 64, 1 << 24
    rows = sum(lengths)
    flat = torch.empty((rows - 1) * pitch + 1024, dtype=torch.bfloat16, device=DEV)
    parts = []
    for i, n in enumerate((h, hk, hk, h)):
        parts.append(flat[i * 128:].as_strided((rows, n, d), (pitch, d, 1)))
    packed = _inputs(lengths, h, hk, d, torch.bfloat16, seed=14)
    for dst, src in zip(parts, packed):
        dst.copy_(src)
    got = _check(lengths, *parts, True)
    want = _check(lengths, *packed, True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_documents():
    q, k, v, do = _inputs([0, 0], 4, 2, 64, torch.bfloat16, spare=9)
    got = _check([0, 0], q, k, v, do, True)
    assert all((t == 0).all() and t.shape[0] == 9 for t in got)
    empty = [t[:0] for t in (q, k, v, do)]
    assert _check([], *empty, True)[0].shape == (0, 4, 64)


@pytest.mark.parametrize("heads,kv_heads,spare", [(4, 2, 9), (3, 1, 700), (1, 1, 1)])
def test_lse_of_rows_behind_the_last_document(heads, kv_heads, spare):
    q, k, v, _ = _inputs([130, 5], heads, kv_heads, 64, torch.bfloat16, spare=spare)
    torch.full((heads, q.shape[0]), math.nan, device=DEV)      # what the allocator hands out next
    _, lse = raw.attention_packed_fwd(q, k, v, ops.PackedLayout([130, 5], device=DEV, total=q.shape[0]))
    assert (lse[:, 135:] == 0).all() and lse[:, :135].isfinite().all()


def test_layout_outlives_a_call_on_another_stream():
    lengths = [300, 1, 513, 64]
    q, k, v, do = _inputs(lengths, 8, 2, 128, torch.bfloat16, seed=5)
    layout = ops.PackedLayout(lengths, device=DEV)
    lists = layout.work_lists(True)[0]
    at, size = lists.untyped_storage().data_ptr(), lists.untyped_storage().nbytes()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        out = ops.flash_attention_packed(q, k, v, layout)
    del layout, lists
    again = [torch.empty(size, dtype=torch.uint8, device=DEV) for _ in range(64)]
    assert not side.query() and all(t.data_ptr() != at for t in again)
    side.synchronize()
    want = oracle.attention(q, k, v, lengths, True, None, do)
    assert oracle.excess(out, want["out"]) <= 1


@pytest.mark.parametrize("scale", [1e-30, 1e-4, 1.0])
def test_scales(scale):
    lengths = [130, 1, 257]
    _check(lengths, *_inputs(lengths, 4, 2, 64, torch.bfloat16, seed=9), True, scale=scale)


@pytest.mark.parametrize("scale", [0.0, -1.0, 1e-31, 1e31, math.inf, math.nan])
def test_scales_out_of_range(scale):
    q, k, v, _ = _inputs([5], 4, 2, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="scale"):
        ops.flash_attention_packed(q, k, v, ops.PackedLayout([5], device=DEV), scale=scale)


def test_no_second_derivative():
    q, k, v, do = (t.contiguous().requires_grad_(True) for t in _inputs([5], 4, 2, 64, torch.bfloat16))
    out = ops.flash_attention_packed(q, k, v, ops.PackedLayout([5], device=DEV))
    with pytest.raises(RuntimeError, match="differentiated"):
        torch.autograd.grad(out, q, do, create_graph=True)


def test_refusals_on_the_device():
    q, k, v, _ = _inputs([5], 4, 2, 64, torch.bfloat16)
    layout = ops.PackedLayout([5], device=DEV)
    for bad in (lambda: ops.flash_attention_packed(q, k, v, ops.PackedLayout([5])),
                lambda: ops.flash_attention_packed(q.float(), k.float(), v.float(), layout),
                lambda: ops.flash_attention_packed(q[..., :32], k[..., :32], v[..., :32], layout),
                lambda: ops.flash_attention_packed(q, k, v.cpu(), layout),
                lambda: ops.flash_attention_packed(q, k[:, :1], v, layout),
                lambda: ops.flash_attention_packed(q[:, :3], k, v, layout),
                lambda: ops.flash_attention_packed(q[:, :0], k, v, layout),
                lambda: ops.flash_attention_packed(q[0], k, v, layout),
                lambda: ops.flash_attention_packed(q[..., :0], k[..., :0], v[..., :0], layout),
                lambda: ops.flash_attention_packed(q, k, v, ops.PackedLayout([4], device=DEV)),
                lambda: ops.flash_attention_packed(q, k, v, layout, scale=0.0),
                lambda: ops.flash_attention_packed(q, k, v, layout, scale=math.nan),
                lambda: raw.attention_packed_bwd(q[:, :2], q, k, v, q, None, layout),
                lambda: raw.attention_packed_bwd(q, q, k, v, q, torch.zeros(4, 5, device=DEV), layout, residue=q[:, :2]),
                lambda: raw.attention_packed_bwd(q[:, :2], q, k, v, q, torch.zeros(4, 5, device=DEV), layout)):
        with pytest.raises((ValueError, TypeError)):
            bad()


def test_teacher_and_student_on_packed_documents():
    """The ops of this file and of the token losses as they are used together: a teacher scores packed
    documents and reports its alternatives, a student learns from them; against the same in 64 bits."""
    g = torch.Generator(device=DEV).manual_seed(7)
    lengths, hidden, h, hk, d, vocab, k = [70, 1, 200, 33], 256, 4, 2, 64, 1003, 24
    rows, dtype = sum(lengths), torch.bfloat16
    layout = ops.PackedLayout(lengths, device=DEV)
    x = torch.randn(rows, hidden, generator=g, device=DEV, dtype=dtype)
    tokens = torch.randint(vocab, (rows,), generator=g, device=DEV)

    def model():
        return [torch.randn(n, hidden, generator=g, device=DEV, dtype=dtype).mul_(hidden ** -0.5).requires_grad_(True)
                for n in ((h + 2 * hk) * d, vocab)]

    def logits_of(w):
        qkv = (x @ w[0].t()).view(rows, h + 2 * hk, d)
        out = ops.flash_attention_packed(qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:], layout)
        return out.reshape(rows, h * d) @ (w[1] * 4).t(), qkv, out

    teacher, student = model(), model()
    with torch.no_grad():
        heard = ops.token_logprobs(logits_of(teacher)[0], tokens, top_k=k)
    logits, qkv, out = logits_of(student)
    loss = ops.topk_distillation_loss(logits, heard.top_index, heard.top_logprob)
    score = ops.token_logprobs(logits, tokens)
    total = loss.mean() - 0.1 * score.logprob.mean() - 0.01 * score.entropy.mean()
    got = torch.autograd.grad(total, (logits, out, qkv, *student))
    native.check_status()

    wide = [w.detach().double().requires_grad_(True) for w in student]
    qkv64 = (x.double() @ wide[0].t()).view(rows, h + 2 * hk, d)
    outs = []
    for s in oracle.documents(lengths):
        q64, k64, v64 = (t.transpose(0, 1) for t in (qkv64[s, :h], qkv64[s, h:h + hk], qkv64[s, h + hk:]))
        a = q64 @ k64.repeat_interleave(h // hk, 0).transpose(1, 2) / math.sqrt(d)
        a = a.masked_fill(torch.ones_like(a[0], dtype=torch.bool).triu(1), -math.inf).softmax(-1)
        outs.append((a @ v64.repeat_interleave(h // hk, 0)).transpose(0, 1))
    out64 = torch.cat(outs)
    logits64 = out64.reshape(rows, h * d) @ (wide[1] * 4).t()
    logp = logits64.log_softmax(1)
    q_t = heard.top_logprob.double().softmax(1)
    loss64 = (q_t * (q_t.log() - logp.gather(1, heard.top_index))).sum(1)
    total64 = loss64.mean() - 0.1 * logp.gather(1, tokens[:, None]).mean() + 0.01 * (logp.exp() * logp).sum(1).mean()
    want = torch.autograd.grad(total64, (logits64, out64, qkv64, *wide))
    # every step rounds its result to bf16 (2^-8 of each element at most, 2^-9 root mean square); up to six
    # such steps lie between the weights and a gradient, and errors of the logits (2^-8 of values up to
    # about 10) move probabilities by 4 %: a norm-wise bound of 6 % for the chain
    assert abs(total.item() - total64.item()) < 0.01 * abs(total64.item())
    for a, b in zip(got, want):
        assert ((a.double() - b).norm() / b.norm()).item() < 0.06


def test_keys_far_below_the_maximum():
    """A probability of 2^-288 is 0 in dV, however large the gradient that comes in."""
    q, k, v, do = (torch.zeros(2, 1, 64, dtype=torch.bfloat16, device=DEV) for _ in range(4))
    q[0, 0, 0] = 1.0
    k[1, 0, 0] = -200.0
    do[0] = 2.0 ** 125
    _check([2], q, k, v, do, False, scale=1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_largest_scale(dtype, dim):
    """Scaled scores of up to x: fp32 sums of the products and an fp32 log-sum-exp are off by 2^-22 of that
    each at most, so a probability by x 2^-21 of itself, and sums over them by twice that."""
    lengths = [130, 257]
    q, k, v, do = (t.contiguous().requires_grad_(True) for t in _inputs(lengths, 4, 2, dim, dtype, seed=17))
    out = ops.flash_attention_packed(q, k, v, ops.PackedLayout(lengths, device=DEV), scale=1e3)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), do)
    want = oracle.attention(q, k, v, lengths, True, 1e3, do.detach())
    x = 1e3 * max((q[r].double().norm(dim=2).max() * k[r].double().norm(dim=2).max()).item()
                  for r in oracle.documents(lengths))
    for name, t in (("out", out), ("dv", dv)):
        value = want[name][0]
        assert ((t.double() - value).norm() / value.norm()).item() <= x * 2.0 ** -20 + torch.finfo(dtype).eps
    assert dq.isfinite().all() and dk.isfinite().all()


@pytest.mark.parametrize("scale", [1.1e3, 1e7, 1e30])
def test_scales_whose_scores_leave_fp32(scale):
    q, k, v, _ = _inputs([5], 4, 2, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="scale"):
        ops.flash_attention_packed(q, k, v, ops.PackedLayout([5], device=DEV), scale=scale)
    with pytest.raises(ValueError, match="scale"):
        ops.flash_attention_packed(q.cpu(), k.cpu(), v.cpu(), ops.PackedLayout([5]), scale=scale)


@pytest.mark.parametrize("heads,kv_heads", [(16, 2), (8, 8)])
def test_mark_of_an_earlier_kernel_does_not_cost_results(heads, kv_heads):
    """The status word tells of a wait that gave up, here or in any kernel before; only the former may leave
    results unwritten. More units of work than SMs, so that CTAs take a second one."""
    lengths = [1024, 700, 256, 1500, 77, 129, 1024]
    inputs = _inputs(lengths, heads, kv_heads, 128, torch.bfloat16, seed=18)
    q, k, v, do = inputs
    layout = ops.PackedLayout(lengths, device=DEV)
    want = _check(lengths, *inputs, True, layout=layout)
    word = native.status(q.device)
    word.fill_(7)
    try:
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = ops.flash_attention_packed(*leaves, layout)
        got = [out.detach(), *torch.autograd.grad(out, leaves, do)]
        assert word.item() == 7 and all(torch.equal(a, b) for a, b in zip(got, want))
    finally:
        word.zero_()


def test_first_call_of_a_process_inside_a_capture(monkeypatch):
    """The status word is made, and cleared, with the layout: made inside the capture it would live in the
    graph's memory and be cleared by replays only."""
    lengths = [130, 3]
    q, k, v, do = (t.contiguous() for t in _inputs(lengths, 4, 2, 64, torch.bfloat16, seed=19))
    monkeypatch.setattr(native, "_status", {})
    layout = ops.PackedLayout(lengths, device=DEV)
    assert len(native._status) == 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = raw.attention_packed_fwd(q, k, v, layout)
    assert len(native._status) == 1
    _check(lengths, q, k, v, do, True, layout=layout)       # before any replay
    graph.replay()
    assert oracle.excess(out, oracle.attention(q, k, v, lengths, True)["out"]) <= 1


@pytest.mark.parametrize("hooks", [contextlib.nullcontext, torch.autograd.graph.save_on_cpu])
def test_status_cleared_between_forward_and_backward(hooks):
    lengths = [130, 3]
    q, k, v, do = (t.contiguous().requires_grad_(True) for t in _inputs(lengths, 4, 2, 64, torch.bfloat16, seed=20))
    with hooks():
        out = ops.flash_attention_packed(q, k, v, ops.PackedLayout(lengths, device=DEV))
    native.status(q.device).zero_()
    grads = torch.autograd.grad(out, (q, k, v), do)
    want = oracle.attention(q, k, v, lengths, True, d_out=do.detach())
    for name, t in zip(("dq", "dk", "dv"), grads):
        assert oracle.excess(t, want[name]) <= 1, name
