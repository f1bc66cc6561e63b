"""Windowed prefill over keys whose V (and here and there K) is not finite, in
every kernel that takes it: outputs are not finite just where a query sees such
a value (in its dim, or anywhere for K), and 64-bit attention elsewhere
(tolerances of rows_reference); and such values cost a bounded time."""

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
@pytest.mark.parametrize("window,sinks", [(1, 0), (20, 0), (40, 5), (64, 40), (33, 1000)])
@pytest.mark.parametrize("what", ["some", "rows", "all"])
def test_values(hq, hkv, d, dtype, lens, window, sinks, what):
    g = torch.Generator(device=DEV).manual_seed(hq + window + d)
    n = sum(lens)
    q, k, v = (torch.randn(n, h, d, generator=g, device=DEV).to(dtype) for h in (hq, hkv, hkv))
    if what == "some":  # one value in some of the rows, of each kind; a K row
        at = torch.rand(n, hkv, generator=g, device=DEV) < 0.04
        dim = torch.randint(0, d, (n, hkv), generator=g, device=DEV)
        kind = torch.tensor([NAN, INF, -INF], device=DEV)[torch.randint(0, 3, (n, hkv), generator=g, device=DEV)].to(dtype)
        v.scatter_(2, dim[..., None], torch.where(at, kind, v.gather(2, dim[..., None])[..., 0])[..., None])
        k[n // 2, 0] = NAN
    elif what == "rows":  # whole rows, the last keys of the sequences among them
        v[torch.rand(n, generator=g, device=DEV) < 0.02] = NAN
        v[_cu(lens)[1:].long() - 1, 0] = INF
    else:
        v[: lens[0]] = NAN
    ref, tol, off = _reference(q, k, v, lens, window, sinks)
    out = flash_attn_varlen_window(q, k, v, _cu(lens), _cu(lens), max(lens), max(lens), window, sinks).double()
    wrong = torch.isfinite(out) == off
    assert not bool(wrong.any()), f"finite or not at other places: {int(wrong.sum())} of {wrong.numel()}"
    err = (out - ref).abs().masked_fill(off, 0.0)
    worst = float((err / tol.clamp(min=1e-300)).max())
    print(f"{hq}/{hkv} x {d}, {dtype}, {window}+{sinks}, {what}: {worst:.2f} of the tolerance", flush=True)
    assert worst <= 1


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


@pytest.mark.parametrize("hq,hkv", [(16, 8), (32, 8), (64, 8), (24, 2), (40, 8)])
def test_time(hq, hkv):
    """One row of values that are not finite, in a first token or in the middle of the longest sequence, costs less than
    three more such calls (queries that all see it are right as they are; the few of the blocks where some do not are
    computed again, from memory); V of nothing else less than eleven (every query is computed again)."""
    lens = [1024, 300, 2048, 700, 128, 1500]
    g = torch.Generator(device=DEV).manual_seed(1)
    n, start = sum(lens), 1324
    q, k, v = (torch.randn(n, h, 128, generator=g, device=DEV).to(BF) for h in (hq, hkv, hkv))
    cu = _cu(lens)

    def best(x):
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(True), torch.cuda.Event(True)
            a.record()
            flash_attn_varlen_window(q, k, x, cu, cu, 2048, 2048, 512, 4)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    clean, cases = best(v), {}
    for name, rows, most in (("a first token", slice(start + 1, start + 2), 4), ("a middle token", slice(start + 1000, start + 1001), 4),
                             ("every token", slice(0, n), 12)):
        x = v.clone()
        x[rows] = NAN
        cases[name] = best(x) / clean
        print(f"{hq}/{hkv}, {name}: {cases[name]:.2f} times {clean * 1e3:.0f} us", flush=True)
        assert cases[name] <= most, (name, cases)
