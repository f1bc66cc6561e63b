"""Windowed prefill of many work items: more than 64 a workgroup, more sequences
than its item plan holds, and rows computed again in the middle of them. Rows at
tile and window edges and around a NaN value, against 64 bits (tolerances derived
in rows_reference)."""

import pytest
import torch

from tests.rows_reference import attend, check, half_step
from tinyserver_amd.kernels import flash_attn_varlen_window

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def _check(q, k, v, out, starts, lens, at, window, sinks):
    """Rows `at` ((sequence, position) pairs) of out."""
    ref, tol, rows = [], [], []
    for s, i in at:
        see = [j for j in range(min(i + 1, lens[s])) if j > i - window or j < sinks] if i < 4096 else (
            list(range(min(sinks, i - window + 1))) + list(range(i - window + 1, i + 1)))
        idx = torch.tensor(see, device=DEV) + starts[s]
        r, t = attend(q[starts[s] + i].cpu(), k[idx].cpu(), v[idx].cpu(), q.shape[2] ** -0.5, half_step(BF), half_step(BF))
        ref.append(r)
        tol.append(t)
        rows.append(starts[s] + i)
    check(out[torch.tensor(rows, device=DEV)], torch.stack(ref), torch.stack(tol), f"window {window}, {sinks}")


@pytest.mark.parametrize("hq,hkv", [(32, 8), (16, 8), (64, 4)])
@pytest.mark.parametrize("window,sinks", [(40, 5), (512, 0)])
def test_a_long_prompt(hq, hkv, window, sinks):
    n = 140000
    g = torch.Generator(device=DEV).manual_seed(window)
    q, k, v = (torch.randn(n, h, 128, generator=g, device=DEV).to(BF) for h in (hq, hkv, hkv))
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    bad = (77, 100003, 131099)
    for j in bad:
        v[j, hkv - 1] = float("nan")
    out = flash_attn_varlen_window(q, k, v, cu, cu, n, n, window, sinks)
    # the NaN rows themselves: seen by the rows from theirs to theirs + window - 1
    nan = torch.isnan(out[:, -1]).any(-1)
    want = torch.zeros(n, dtype=torch.bool, device=DEV)
    for j in bad:
        want[j : j + window] = True
    assert torch.equal(nan, want)
    assert torch.equal(torch.isnan(out[:, : hq - hq // hkv]).any(), torch.tensor(False, device=DEV))
    near = [j + d for j in bad for d in (-2, -1, window, window + 1)]
    tiles = [64 * t + d for t in (0, 1, 500, 1023, 1024, 1500, 2047, 2048, 2186) for d in (0, 31, 32, 63)]
    at = [(0, i) for i in near + tiles + [n - 1] if i < n and not bool(want[i])]
    _check(q, k, v, out, [0], [n], at, window, sinks)


@pytest.mark.parametrize("hq,hkv", [(8, 2), (4, 2), (16, 2), (12, 1), (32, 2)])
def test_many_sequences(hq, hkv):
    g = torch.Generator().manual_seed(hq)
    lens = torch.randint(0, 300, (150,), generator=g).tolist()
    lens[7], lens[149] = 1000, 1
    n = sum(lens)
    starts = torch.tensor([0] + lens).cumsum(0).tolist()
    cu = torch.tensor(starts, dtype=torch.int32, device=DEV)
    q, k, v = (torch.randn(n, h, 128, generator=g).to(BF).to(DEV) for h in (hq, hkv, hkv))
    first = [s for s in range(150) if lens[s] > 100][:60:7]
    for s in first:
        v[starts[s] + 50] = float("inf")
    out = flash_attn_varlen_window(q, k, v, cu, cu, max(lens), max(lens), 20, 3)
    at = [(s, i) for s in first for i in (0, 31, 48, 49, 70, 71, lens[s] - 1)]
    at += [(s, i) for s in range(0, 150, 5) for i in (0, lens[s] // 2, lens[s] - 1) if lens[s] and not (s in first and 50 <= i < 70)]
    _check(q, k, v, out, starts, lens, at, 20, 3)


@pytest.mark.parametrize("hq,hkv,dtype", [(12, 1, BF), (16, 1, torch.float16), (32, 2, BF)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (32, 0), (33, 33), (50, 1), (1000, 4), (16, 1000)])
@pytest.mark.parametrize("lens_q,lens_k", [([70, 5, 160], [70, 5, 160]), ([100, 64, 3], [40, 90, 0])])
def test_wide_groups(hq, hkv, dtype, window, sinks, lens_q, lens_k):
    g = torch.Generator().manual_seed(window + hq)
    q = torch.randn(sum(lens_q), hq, 128, generator=g).to(dtype)
    k, v = (torch.randn(sum(lens_k), hkv, 128, generator=g).to(dtype) for _ in range(2))
    cu_q, cu_k = (torch.tensor([0] + x).cumsum(0).to(torch.int32).to(DEV) for x in (lens_q, lens_k))
    out = flash_attn_varlen_window(q.to(DEV), k.to(DEV), v.to(DEV), cu_q, cu_k, max(lens_q), max(lens_k), window, sinks)
    ref, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    a = b = 0
    for nq, nk in zip(lens_q, lens_k):
        for i in range(nq):
            see = [b + j for j in range(min(nk, i + 1)) if j > i - window or j < sinks]
            ref[a + i], tol[a + i] = attend(q[a + i], k[see], v[see], 128**-0.5, half_step(dtype), half_step(dtype))
        a, b = a + nq, b + nk
    check(out, ref, tol, f"{hq}/{hkv}, {window}+{sinks}")


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_wide_groups_rows_that_are_not_seen(bad):
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(300, h, 128, generator=g).to(BF) for h in (16, 1, 1))
    v[50], k[121] = bad, bad
    cu = torch.tensor([0, 200, 300], dtype=torch.int32, device=DEV)
    out = flash_attn_varlen_window(q.to(DEV), k.to(DEV), v.to(DEV), cu, cu, 200, 100, 30, 3)
    sees = [(0, i) for i in range(200) if not (50 <= i < 80 or 121 <= i < 151)]
    _check(q.to(DEV), k.to(DEV), v.to(DEV), out, [0, 200], [200, 100], sees[::7] + [(0, 49), (0, 80), (0, 120), (0, 151), (1, 99)], 30, 3)
