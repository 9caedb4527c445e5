"""Packed-document attention on the CPU path, the work lists of its layout, and its refusals."""
import math
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from eth_b200 import ops
from eth_b200.ops import raw
from helpers import oracle_packed as oracle

LENGTHS = [[], [0], [1], [5, 0, 1, 9], [130, 3]]


def _inputs(lengths, heads, kv_heads, dim, dtype, spare=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    rows = sum(lengths) + spare
    return [torch.randn(rows, n, dim, generator=g, dtype=torch.float64).to(dtype) for n in (heads, kv_heads, kv_heads, heads)]


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 2), (3, 1)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forward_and_backward(lengths, heads, kv_heads, causal, dtype):
    q, k, v, do = _inputs(lengths, heads, kv_heads, 16, dtype, spare=2)
    layout = ops.PackedLayout(lengths, total=q.shape[0])
    for t in (q, k, v):
        t.requires_grad_(True)
    out = ops.flash_attention_packed(q, k, v, layout, causal=causal)
    grads = torch.autograd.grad(out, (q, k, v), do)
    want = oracle.attention(q, k, v, lengths, causal, d_out=do)
    for name, t in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)):
        assert oracle.excess(t, want[name]) <= 1, name
        assert (t[layout.used:] == 0).all()


@pytest.mark.parametrize("causal", [True, False])
def test_gradient_against_differences(causal):
    q, k, v, _ = _inputs([4, 1, 3], 4, 2, 3, torch.float64)
    layout = ops.PackedLayout([4, 1, 3])
    for t in (q, k, v):
        t.requires_grad_(True)
    assert torch.autograd.gradcheck(lambda *t: ops.flash_attention_packed(*t, layout, causal=causal), (q, k, v))


def test_equal_lengths_agree_with_the_batched_op():
    q, k, v, _ = _inputs([6, 6], 2, 2, 8, torch.float32)
    out = ops.flash_attention_packed(q, k, v, ops.PackedLayout([6, 6]))
    want = ops.flash_attention(*(t.view(2, 6, 2, 8) for t in (q, k, v)))
    torch.testing.assert_close(out.view_as(want), want, rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("lengths", [[1], [128], [129, 0, 300, 1], [5000, 257, 256, 255, 1]])
def test_work_lists(lengths):
    """Every tile of every document exactly once, in falling order of the work it stands for."""
    tables = dict(ops.PackedLayout._work_lists(np.asarray(lengths)))
    assert set(tables) == {"causal128", "full128", "keys128", "causal256", "full256"}
    starts = np.cumsum(lengths) - lengths
    for name, table in tables.items():
        rows = 256 if "256" in name else 128
        want = sorted((int(s), int(n), t) for s, n in zip(starts, lengths) for t in range(-(-n // rows)))
        assert sorted(tuple(int(x) for x in r[:3]) for r in table) == want and table.dtype == np.int32
        tiles = -(-table[:, 1] // rows)
        weight = {"causal": table[:, 2] + 1, "full": tiles, "keys": tiles - table[:, 2]}[name.rstrip("0123456789")]
        assert (np.diff(weight) <= 0).all()


def test_refusals():
    q, k, v, _ = _inputs([5], 4, 2, 8, torch.float32)
    layout = ops.PackedLayout([5])
    for bad in (lambda: ops.PackedLayout([3, -1]), lambda: ops.PackedLayout([3.5]), lambda: ops.PackedLayout([[3]]),
                lambda: ops.PackedLayout([3], total=2), lambda: ops.PackedLayout([2 ** 31]),
                lambda: ops.flash_attention_packed(q, k, v, ops.PackedLayout([4])),
                lambda: ops.flash_attention_packed(q, k[:, :1], v, layout),
                lambda: ops.flash_attention_packed(q[:, :3], k, v, layout),
                lambda: ops.flash_attention_packed(q[:, :0], k, v, layout),
                lambda: ops.flash_attention_packed(q, k.double(), v, layout),
                lambda: ops.flash_attention_packed(q[0], k, v, layout),
                lambda: ops.flash_attention_packed(q.int(), k.int(), v.int(), layout),
                lambda: ops.flash_attention_packed(q, k, v, layout, scale=0.0),
                lambda: ops.flash_attention_packed(q, k, v, layout, scale=-1.0),
                lambda: ops.flash_attention_packed(q, k, v, layout, scale=math.inf),
                lambda: layout.work_lists(True),
                lambda: raw.attention_packed_bwd(q[:, :2], q, k, v, q, None, layout)):
        with pytest.raises(ValueError):
            bad()


def test_layout_from_tensors_and_arrays():
    for lengths in (torch.tensor([3, 0, 2], dtype=torch.int32), np.array([3, 0, 2], dtype=np.uint8), (3, 0, 2)):
        layout = ops.PackedLayout(lengths, total=7)
        assert layout.lengths == (3, 0, 2) and layout.used == 5 and layout.total == 7
        assert list(layout.documents()) == [(0, 3), (3, 2)]


def test_exponential_on_the_fma_pipe():
    """`exp2_poly` of the backward kernels, restated step by step in fp32 with the coefficients of its source:
    within 2^-17 of 2^x (the oracle grants all fp32 steps together 2^-15), 0 where 2^x is no normal number."""
    source = Path(raw.__file__).parents[1].joinpath("csrc", "attention_packed_sm100.cu").read_text()
    body = source[source.index("Pair exp2_poly(Pair x)"):source.index("Pair exp2_sfu")]
    f32 = np.float32
    floor = f32(re.search(r'"f"\((-[\d.]+)f\)', body).group(1))
    coefficients = [f32(c) for c in re.findall(r"pair\((0\.\d+)f, \1f\)", body)]
    magic = f32(12582912.0)
    x = np.concatenate([np.linspace(-130, 1, 1 << 20), -np.arange(131), [-126.5, -1e4, -np.inf]]).astype(f32)
    at = np.maximum(x, floor)
    r = at + magic
    f = at + (magic - r)
    y = np.full_like(f, coefficients[0])
    for c in coefficients[1:]:
        y = (y.astype(np.float64) * f + c).astype(f32)          # fused: one rounding
    field = ((r.view(np.int32).astype(np.int64) << 23) + 0x3f800000).astype(np.uint32).view(f32)
    got, want = (y * field).astype(np.float64), np.exp2(x.astype(np.float64))
    normal = x >= -126
    assert (np.abs(got - want)[normal] <= 2.0 ** -17 * want[normal]).all()
    assert (np.abs(got - want)[~normal] <= 2.0 ** -126).all() and (got[x <= -127] == 0).all()


@pytest.mark.parametrize("lengths", [[2 ** 62, 2 ** 62], [2 ** 63 - 1, 2], [2 ** 62] * 4,
                                     np.array([2 ** 64 - 1], dtype=np.uint64), [2 ** 31]])
def test_lengths_whose_sum_wraps(lengths):
    with pytest.raises(ValueError):
        ops.PackedLayout(lengths)


def test_total_is_a_whole_number():
    for total in (7, 7.0, np.int32(7), torch.tensor(7)):
        assert ops.PackedLayout([3, 2], total=total).total == 7
    for total in (7.5, 5.999, math.nan):
        with pytest.raises(ValueError):
            ops.PackedLayout([3, 2], total=total)
