"""Decode and varlen prefill with a sliding window and first tokens against
64-bit attention over the visible keys (tolerances derived in rows_reference):
windows of one token to past the context, first tokens that overlap the window
or reach past the length, block and page edges, split units, GQA groups, types,
page sizes, strides; keys that are not seen hold NaN and infinities and their
pages' ids are not valid ones; 8-bit caches alike."""

import pytest
import torch

from tests.rows_reference import attend, check, half_step, pool, quantize, rows, visible
from tinyserver_amd.kernels import (
    flash_attn_varlen_window,
    paged_attention_forward,
    paged_attention_quantized,
    paged_attention_window,
)

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4, I8 = torch.float8_e4m3fn, torch.int8


def _decode_case(lens, hq, hkv, d, page, dtype, window, sinks, cache=None, seed=0):
    """(inputs, reference, tolerance). Unseen slots hold NaN or infinities; pages without a seen token have ids outside
    the pool."""
    kc, vc, bt = pool(lens, hkv, d, page, seed + d + page + len(lens))
    q = torch.randn(len(lens), hq, d, generator=torch.Generator().manual_seed(seed + 1)).to(dtype)
    if cache is None:
        kc, vc = kc.to(dtype), vc.to(dtype)
        sc = None
        k64, v64 = kc, vc
    else:
        (kc, ks), (vc, vs) = quantize(kc.nan_to_num(), cache), quantize(vc.nan_to_num(), cache)
        sc = [ks, vs]
        k64, v64 = (c.to(torch.float64) * s[..., None].double() for c, s in ((kc, ks), (vc, vs)))
    ref, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for s, n in enumerate(lens):
        see = visible(n, window, sinks)
        ref[s], tol[s] = attend(q[s], rows(k64, bt[s], see), rows(v64, bt[s], see), d**-0.5, half_step(dtype),
                                half_step(dtype))
        for p in sorted(set(range(page * bt.shape[1])) - set(see)):
            if p // page * page >= n and p // page >= -(-n // page):
                continue  # not a page of the sequence
            pg, sl = int(bt[s, p // page]), p % page
            if cache is None:
                kc[pg, :, sl], vc[pg, :, sl] = float("nan"), float("inf") if p % 2 else float("nan")
            else:
                sc[0][pg, :, sl] = sc[1][pg, :, sl] = float("nan")
        for b in range(bt.shape[1]):
            if not any(p // page == b for p in see):
                bt[s, b] = -1 if b % 2 else 1 << 30
    return (q, kc, vc, sc, bt, torch.tensor(lens, dtype=torch.int32)), ref, tol


def _run_decode(case, page, window, sinks, **kw):
    q, kc, vc, sc, bt, sl = case
    if sc is None:
        return paged_attention_window(q.to(DEV), kc.to(DEV), vc.to(DEV), bt.to(DEV), page, sl.to(DEV), window, sinks, **kw)
    return paged_attention_quantized(q.to(DEV), kc.to(DEV), vc.to(DEV), sc[0].to(DEV), sc[1].to(DEV), bt.to(DEV), page,
                                     sl.to(DEV), window=window, sinks=sinks, **kw)


SHAPES = [
    (16, 8, 128, 16, BF, [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300]),
    (32, 8, 128, 16, F16, [1000, 5, 513, 64]),
    (64, 8, 128, 256, BF, [255, 256, 257, 700]),
    (8, 8, 64, 16, BF, [100, 1, 65]),
    (6, 2, 64, 32, F16, [96, 33, 400]),
    (12, 1, 128, 48, BF, [200, 47, 49]),
    (40, 1, 128, 16, BF, [200, 33]),             # 40 heads on one kv head
    (4, 2, 128, 4, F32, [9, 1, 70, 300]),
    (4, 2, 128, 4, BF, [9, 1, 70, 300]),         # pages of less than 16 tokens
    (6, 3, 80, 16, F16, [9, 1, 70]),
    (2, 1, 32, 24, BF, [60, 25]),
]


@pytest.mark.parametrize("hq,hkv,d,page,dtype,lens", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 40), (100, 7), (64, 1000), (4096, 3), (1 << 40, 0)])
def test_decode(hq, hkv, d, page, dtype, lens, window, sinks):
    case, ref, tol = _decode_case(lens, hq, hkv, d, page, dtype, window, sinks)
    check(_run_decode(case, page, window, sinks), ref, tol, f"{hq}/{hkv} x {d}, page {page}, {dtype}, {window}+{sinks}")


@pytest.mark.parametrize("cache", [E4, I8])
@pytest.mark.parametrize("hq,hkv,d,page,dtype,lens", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (33, 5)])
def test_decode_8_bits(cache, hq, hkv, d, page, dtype, lens, window, sinks):
    case, ref, tol = _decode_case(lens, hq, hkv, d, page, dtype, window, sinks, cache)
    check(_run_decode(case, page, window, sinks), ref, tol, f"{cache} {hq}/{hkv} x {d}, page {page}, {dtype}, {window}+{sinks}")


@pytest.mark.parametrize("cache", [None, E4, I8])
@pytest.mark.parametrize("hq,lens,page,window,sinks", [
    (32, [5000, 1, 3333, 129], 16, 4000, 40),
    (16, [20000], 256, 0, 0),
    (64, [2049, 2048, 2047, 31, 0], 16, 0, 0),
    (8, [9000, 100], 32, 8192, 1),
])
def test_decode_long(cache, hq, lens, page, window, sinks):
    """Units of several splits."""
    window = window or (1 << 20 if cache is None else 0)
    case, ref, tol = _decode_case(lens, hq, 2, 128, page, BF, window, sinks, cache)
    check(_run_decode(case, page, window, sinks), ref, tol, f"{cache} {hq}/2, {lens}, {window}+{sinks}")


@pytest.mark.parametrize("cache", [None, E4, I8])
@pytest.mark.parametrize("hq,hkv,d,page,dtype,batch,longest,window,sinks", [
    (16, 8, 128, 16, BF, 64, 2500, 0, 0),
    (32, 8, 64, 32, F16, 48, 3000, 0, 0),
    (16, 8, 128, 256, BF, 64, 3000, 1900, 40),
    (40, 2, 128, 16, F16, 150, 2100, 1800, 5),
    (8, 8, 128, 16, BF, 300, 1300, 0, 0),
])
def test_decode_many_tiles(cache, hq, hkv, d, page, dtype, batch, longest, window, sinks):
    """Batches whose tables hold many tiles, of sequences that are short but for one: runs that cross units, empty
    sequences, units of one tile, one that many waves share."""
    g = torch.Generator().manual_seed(batch)
    lens = (torch.rand(batch, generator=g) ** 3 * 150).long().tolist()
    lens[batch // 3], lens[0], lens[-1] = longest, 0, 17
    if cache is None and not window:
        window = 1 << 20
    case, ref, tol = _decode_case(lens, hq, hkv, d, page, dtype, window, sinks, cache)
    check(_run_decode(case, page, window, sinks), ref, tol, f"{cache} {batch} x {hq}/{hkv} x {d}, {window}+{sinks}")


def test_decode_scales_that_16_bits_do_not_hold():
    """Rows of values near 1e-6 and 1e5 in one 8-bit cache, with f16 queries."""
    lens = [300, 40]
    for size in (1e-6, 1e5):
        kc, vc, bt = pool(lens, 2, 128, 16, 3)
        (kc, ks), (vc, vs) = quantize(kc.nan_to_num(), E4), quantize(vc.nan_to_num() * size, E4)
        q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(1)).half()
        out = paged_attention_quantized(*(t.to(DEV) for t in (q.bfloat16(), kc, vc, ks, vs, bt)), 16,
                                        torch.tensor(lens, dtype=torch.int32, device=DEV))
        for s, n in enumerate(lens):
            k, v = (rows(c.double() * x[..., None].double(), bt[s], range(n)) for c, x in ((kc, ks), (vc, vs)))
            ref, tol = attend(q[s].bfloat16(), k, v, 128**-0.5, half_step(BF), half_step(BF))
            check(out[s], ref, tol, f"size {size}")


@pytest.mark.parametrize("cache", [None, E4])
def test_decode_strides_and_out(cache):
    """Query, output, pool, table and lengths with strides of their own; the same bits as from contiguous ones."""
    case, ref, tol = _decode_case([130, 77, 600], 8, 2, 128, 16, BF, 64, 5, cache)
    q, kc, vc, sc, bt, sl = (t.to(DEV) if isinstance(t, torch.Tensor) else t for t in case)
    plain = _run_decode(case, 16, 64, 5)

    def spread(t, pad):
        w = torch.zeros(*t.shape[:-1], t.shape[-1] + pad, dtype=t.dtype, device=DEV)
        w[..., : t.shape[-1]] = t
        return w[..., : t.shape[-1]]

    out = torch.full((3, 8, 256), 7.0, dtype=BF, device=DEV)
    args = [spread(q, 16), spread(kc.view(torch.uint8) if cache else kc, 32), spread(vc.view(torch.uint8) if cache else vc, 16)]
    if cache:
        args[1:] = [t.view(cache) for t in args[1:]]
        args += [spread(s.to(DEV), 5) for s in sc]
    args += [spread(bt, 3), 16, torch.stack([sl, sl], 1)[:, 0]]
    fn = paged_attention_quantized if cache else paged_attention_window
    got = fn(*args, window=64, sinks=5, out=out[..., :128])
    check(got, ref, tol, "strides")
    assert torch.equal(got, plain) and bool((out[..., 128:] == 7).all())
    got = fn(*args, window=64, sinks=5, out=out[..., ::2])  # elements apart
    check(got, ref, tol, "an output of stride 2")


def test_decode_without_a_window_is_paged_attention():
    lens = [700, 16, 33]
    kc, vc, bt = pool(lens, 8, 128, 16, 4)
    q = torch.randn(3, 32, 128).to(BF).to(DEV)
    args = [q, kc.to(BF).to(DEV), vc.to(BF).to(DEV), bt.to(DEV), 16, torch.tensor(lens, dtype=torch.int32, device=DEV)]
    a, b = paged_attention_window(*args, 1 << 30), paged_attention_forward(*args)
    assert float((a.float() - b.float()).abs().max()) <= 2.0**-7 * float(b.float().abs().max())


@pytest.mark.parametrize("cache", [None, I8])
def test_decode_lengths_past_the_table_and_below_zero(cache):
    case, ref, tol = _decode_case([64, 64], 8, 2, 128, 16, BF, 1 << 20 if cache is None else 0, 0, cache)
    q, kc, vc, sc, bt, sl = case
    case = (q, kc, vc, sc, bt, torch.tensor([1 << 30, -5], dtype=torch.int32))
    ref[1], tol[1] = 0.0, 0.0
    check(_run_decode(case, 16, 1 << 20 if cache is None else 0, 0), ref, tol, "lengths")


def _prefill_ref(q, k, v, lens_q, lens_k, window, sinks):
    ref, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    u, d = half_step(q.dtype), q.shape[2]
    a = b = 0
    for nq, nk in zip(lens_q, lens_k):
        for i in range(nq):
            see = [j for j in range(min(nk, i + 1)) if j > i - window or j < sinks]
            ref[a + i], tol[a + i] = attend(q[a + i], k[b : b + nk][see], v[b : b + nk][see], d**-0.5, u, u)
        a, b = a + nq, b + nk
    return ref, tol


def _cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(DEV)


@pytest.mark.parametrize("hq,hkv,d,dtype,lens", [
    (4, 2, 128, BF, [1, 31, 32, 33, 0, 65]),
    (8, 2, 128, BF, [70, 5, 160]),
    (16, 2, 128, F16, [100, 64]),
    (4, 1, 64, BF, [97, 40]),
    (3, 3, 128, BF, [50, 130]),
    (6, 2, 64, F16, [50, 70]),
    (4, 2, 128, F32, [40, 70]),
    (2, 1, 80, BF, [40, 9]),
])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (8, 3), (32, 0), (33, 33), (50, 1), (1000, 4), (16, 1000)])
def test_prefill(hq, hkv, d, dtype, lens, window, sinks):
    g = torch.Generator().manual_seed(d + hq + window)
    n = sum(lens)
    q, k, v = (torch.randn(n, h, d, generator=g).to(dtype) for h in (hq, hkv, hkv))
    ref, tol = _prefill_ref(q, k, v, lens, lens, window, sinks)
    out = flash_attn_varlen_window(q.to(DEV), k.to(DEV), v.to(DEV), _cu(lens), _cu(lens), max(lens), max(lens), window, sinks)
    check(out, ref, tol, f"{hq}/{hkv} x {d}, {dtype}, {window}+{sinks}")


@pytest.mark.parametrize("window,sinks", [(5, 0), (40, 3), (64, 70)])
@pytest.mark.parametrize("hq,d", [(8, 128), (4, 128), (16, 128), (4, 64)])
def test_prefill_unlike_lengths(hq, d, window, sinks):
    """More queries than keys (late queries see the first keys only, or none:
    0), more keys than queries, none of either."""
    lens_q, lens_k = [100, 20, 5, 40, 0], [30, 90, 0, 39, 7]
    g = torch.Generator().manual_seed(hq)
    q = torch.randn(sum(lens_q), hq, d, generator=g).to(BF)
    k, v = (torch.randn(sum(lens_k), 2, d, generator=g).to(BF) for _ in range(2))
    ref, tol = _prefill_ref(q, k, v, lens_q, lens_k, window, sinks)
    out = flash_attn_varlen_window(q.to(DEV), k.to(DEV), v.to(DEV), _cu(lens_q), _cu(lens_k), 100, 90, window, sinks)
    check(out, ref, tol, f"{hq} x {d}, {window}+{sinks}")


@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 128, BF), (4, 2, 128, F16), (16, 2, 128, BF), (4, 1, 64, BF), (6, 2, 128, BF)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_prefill_rows_that_are_not_seen(hq, hkv, d, dtype, bad):
    """A key whose K or V row is not finite reaches the queries that see it and
    no others, inside a block of queries too."""
    lens, window, sinks = [150, 90], 40, 5
    g = torch.Generator().manual_seed(7)
    n = sum(lens)
    q, k, v = (torch.randn(n, h, d, generator=g).to(dtype) for h in (hq, hkv, hkv))
    ref, tol = _prefill_ref(q, k, v, lens, lens, window, sinks)
    j, hits = 70, set(range(70, 110))
    v[j, 0, 3] = bad
    v[150 + 2, 0, d - 1] = bad  # a first key: every later query sees it
    k[150 + 60, hkv - 1] = float("nan")
    out = flash_attn_varlen_window(q.to(DEV), k.to(DEV), v.to(DEV), _cu(lens), _cu(lens), 150, 150, window, sinks).cpu()
    group = hq // hkv
    seen = torch.zeros(n, hq, d, dtype=torch.bool)
    for i in hits:
        seen[i, :group, 3] = True
    seen[152:, :group, d - 1] = True
    for i in range(60, min(90, 100)):
        seen[150 + i, -group:] = True
    assert not bool(torch.isfinite(out[seen].float()).any())
    check(torch.where(seen, 0, out), torch.where(seen, 0.0, ref), tol, f"{hq}/{hkv} x {d}, {bad}")


def test_prefill_strides_and_rows_behind_the_last_sequence():
    g = torch.Generator().manual_seed(3)
    lens, extra = [70, 33], 9
    n = sum(lens)
    whole = torch.randn(n + extra, 8 + 2 + 2, 128, generator=g).to(BF)
    q, k, v = whole[:, :8], whole[:, 8:10], whole[:, 10:]
    ref, tol = _prefill_ref(q[:n], k[:n], v[:n], lens, lens, 20, 3)
    w = whole.to(DEV)
    out = torch.full((n + extra, 8, 160), 5.0, dtype=BF, device=DEV)
    got = flash_attn_varlen_window(w[:, :8], w[:, 8:10], w[:, 10:], _cu(lens), _cu(lens), 70, 70, 20, 3, out=out[..., :128])
    check(got[:n], ref, tol, "one projection's views")
    assert bool((out[n:] == 5).all()) and bool((out[..., 128:] == 5).all())


def test_prefill_scale_and_long_rows():
    """A softmax scale of its own (negative too) and sequences of several hundred blocks' windows."""
    g = torch.Generator().manual_seed(5)
    lens = [700]
    q, k, v = (torch.randn(700, h, 128, generator=g).to(BF) for h in (4, 1, 1))
    for scale in (0.3, -0.05):
        out = flash_attn_varlen_window(q.to(DEV), k.to(DEV), v.to(DEV), _cu(lens), _cu(lens), 700, 700, 130, 70, scale).cpu()
        for i in (0, 69, 70, 129, 130, 131, 200, 201, 511, 699):
            see = [j for j in range(i + 1) if j > i - 130 or j < 70]
            ref, tol = attend(q[i] * (1 if scale > 0 else -1), k[see], v[see], abs(scale), half_step(BF), half_step(BF))
            check(out[i], ref, tol, f"row {i}, scale {scale}")
