"""Windowed prefill over keys that are not finite, in every kernel that takes it:
outputs are not finite just where a query sees such a value, and 64-bit attention
elsewhere (tolerances of rows_reference)."""

import math

import pytest
import torch

from tests.rows_reference import half_step
from tinyserver_amd.kernels import flash_attn_varlen_window

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16 = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


def _cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(DEV)


def _reference(q, k, v, lens, window, sinks):
    """(output, tolerance, where it is not finite), sequence by sequence and head by head in 64 bits on the GPU."""
    out, tol = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    off = torch.zeros(q.shape, dtype=torch.bool, device=DEV)
    group, d, u, a = q.shape[1] // k.shape[1], q.shape[2], half_step(q.dtype), 0
    for n in lens:
        i, j = torch.arange(n, device=DEV)[:, None], torch.arange(n, device=DEV)[None, :]
        see = (j <= i) & ((j > i - window) | (j < sinks))
        for h in range(q.shape[1]):
            qh = q[a : a + n, h].double()
            kh, vh = (x[a : a + n, h // group].double() for x in (k, v))
            bad_k, bad_v = ~torch.isfinite(kh).all(-1), ~torch.isfinite(vh)
            kh, vh = kh.nan_to_num(0.0, 0.0, 0.0), vh.nan_to_num(0.0, 0.0, 0.0)
            s = (qh @ kh.t().contiguous()) / math.sqrt(d)
            o = torch.softmax(s.masked_fill(~see, -INF), -1).nan_to_num(0.0) @ vh
            out[a : a + n, h] = o
            seen = see.double()
            off[a : a + n, h] = ((seen @ bad_v.double()) > 0) | ((seen @ bad_k.double()[:, None]) > 0)
            size = (qh.abs() @ kh.abs().t().contiguous()).amax(-1) / math.sqrt(d)
            e = size * ((d + 2) * 2.0**-24 + 4 * 2.0**-23) + 2.0**-22
            tol[a : a + n, h] = u * o.abs() + vh.abs().max() * (u + 2 * e + 2 * n * 2.0**-24)[:, None]
        a += n
    return out, tol, off


SHAPES = [
    (4, 2, 128, BF, [70, 33, 1, 200]),       # two q-heads a kv head
    (16, 8, 128, F16, [800, 760]),           # the same, in pairs of query blocks
    (8, 2, 128, BF, [150, 31, 97]),
    (16, 2, 128, F16, [130, 64]),
    (24, 2, 128, BF, [200, 65, 3]),          # 64 queries a wave
    (6, 2, 128, F16, [90, 140]),             # a group of three
    (4, 2, 64, F16, [70, 33, 200]),
    (4, 1, 64, BF, [97, 140]),
    (8, 1, 64, F16, [160]),
    (5, 1, 64, BF, [100, 40]),
]


@pytest.mark.parametrize("hq,hkv,d,dtype,lens", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 0), (1, 2)])
def test_queries_that_see_nan_scores_alone(hq, hkv, d, dtype, lens, window, sinks):
    """A NaN in K is a NaN in every query that sees it, also where the query sees no other key."""
    g = torch.Generator(device=DEV).manual_seed(hq + d)
    n = sum(lens)
    q, k, v = (torch.randn(n, h, d, generator=g, device=DEV).to(dtype) for h in (hq, hkv, hkv))
    k[[0, 20, 21, 22, n - 1]] = NAN
    ref, tol, off = _reference(q, k, v, lens, window, sinks)
    out = flash_attn_varlen_window(q, k, v, _cu(lens), _cu(lens), max(lens), max(lens), window, sinks).double()
    assert torch.equal(torch.isnan(out), off)
    assert bool(((out - ref).abs().masked_fill(off, 0.0) <= tol).all())
