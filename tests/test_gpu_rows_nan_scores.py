"""A NaN among the keys a row sees makes the row NaN in every form of the windowed
and 8-bit decode and of the draft trees, also where a row, or a whole split of its
keys, has nothing but NaN scores; rows beside it are untouched."""

import pytest
import torch

from tinyserver_amd.kernels import paged_attention_quantized, paged_attention_tree, paged_attention_window

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAN = float("nan")


def _pool(lens, hkv, d, page, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [max(1, -(-n // page)) for n in lens]
    bt = torch.zeros(len(lens), max(need), dtype=torch.int32, device=DEV)
    at = 0
    for s, n in enumerate(need):
        bt[s, :n] = torch.arange(at, at + n, dtype=torch.int32, device=DEV)
        at += n
    return *(torch.randn(at, hkv, page, d, generator=g, device=DEV) for _ in range(2)), bt, g


def _keys(cache, bt, s, lo, hi, page, value):
    """Sets rows [lo, hi) of sequence s."""
    p = torch.arange(lo, hi, device=DEV)
    cache[bt[s, p // page].long(), :, p % page] = value


@pytest.mark.parametrize("kind", [None, torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype,hq,hkv,d,page", [(BF, 8, 2, 128, 16), (F16, 16, 2, 64, 32), (BF, 4, 2, 128, 4), (F32, 4, 2, 64, 16)])
@pytest.mark.parametrize("lens,window,lo,hi", [
    ([40, 90, 33], 1, 89, 90),        # the only key of the row
    ([40, 300, 33], 0, 299, 300),     # one of many
    ([40, 300, 33], 0, 0, 300),       # all of them
    ([40, 3000, 33], 0, 0, 700),      # a split's
    ([40, 3000, 33], 0, 0, 3000),     # every split's
    ([40, 3000] + [2500] * 70, 0, 0, 3000),  # the stream's
])
def test_decode(kind, dtype, hq, hkv, d, page, lens, window, lo, hi):
    k, v, bt, g = _pool(lens, hkv, d, page, 5)
    q = torch.randn(len(lens), hq, d, generator=g, device=DEV).to(dtype)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if kind is None:
        k, v = k.to(dtype), v.to(dtype)
        call = lambda: paged_attention_window(q, k, v, bt, page, n, window or 1 << 20)  # noqa: E731
        clean = call()
        _keys(k, bt, 1, lo, hi, page, NAN)
    else:
        k, v = (x.clamp(-3, 3).mul(30).round().to(kind) for x in (k, v))
        ks, vs = (torch.full(k.shape[:3], 0.02, device=DEV) for _ in range(2))
        call = lambda: paged_attention_quantized(q, k, v, ks, vs, bt, page, n, window=window)  # noqa: E731
        clean = call()
        _keys(ks, bt, 1, lo, hi, page, NAN)
    out = call()
    assert bool(torch.isfinite(clean).all())
    assert bool(torch.isnan(out[1]).all())
    out[1] = clean[1]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("dtype,hq,hkv,d,page", [(BF, 8, 2, 128, 16), (F16, 16, 2, 64, 32), (BF, 64, 4, 128, 16), (BF, 4, 2, 128, 4)])
@pytest.mark.parametrize("ctx,lo,hi", [(0, 0, 0), (50, 0, 50), (2000, 0, 600), (2000, 0, 2000), (50, 20, 21)])
def test_tree(dtype, hq, hkv, d, page, ctx, lo, hi):
    """A context, then node 1's own key (which no other node sees, and which is all that it sees without a context)."""
    nodes, lens = [6, 5, 1], [40, ctx, 7]
    k, v, bt, g = _pool([a + b for a, b in zip(lens, nodes)], hkv, d, page, 7)
    k, v = k.to(dtype), v.to(dtype)
    q = torch.randn(sum(nodes), hq, d, generator=g, device=DEV).to(dtype)
    cu = torch.tensor([0, 6, 11, 12], dtype=torch.int32, device=DEV)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    mask = torch.tensor([1 << i for m in nodes for i in range(m)], device=DEV)  # each node itself
    call = lambda: paged_attention_tree(q, k, v, bt, page, n, cu, mask)  # noqa: E731
    clean = call()
    _keys(k, bt, 1, ctx + 1, ctx + 2, page, NAN)
    out = call()
    assert bool(torch.isfinite(clean).all()) and bool(torch.isnan(out[7]).all())
    out[7] = clean[7]
    assert torch.equal(out, clean)
    if hi > lo:
        _keys(k, bt, 1, lo, hi, page, NAN)
        out = call()
        assert bool(torch.isnan(out[6:11]).all())
        out[6:11] = clean[6:11]
        assert torch.equal(out, clean)
