"""The 8-bit paged cache: codes and scales bit-equal to the definition (prompts
and decode steps, every source type, strided sources and pools, page sizes and
head_dims either side of the wide path), what a store must leave alone, rows of
zeros, subnormals, NaN and infinities, and reading back (bit-equal to code *
scale, rounded once)."""

import pytest
import torch

from tests.rows_reference import LARGEST, quantize
from tinyserver_amd.kernels import load_kv_cache_quantized, store_kv_cache_quantized

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4, I8 = torch.float8_e4m3fn, torch.int8


def _bits(t):
    return t.detach().cpu().contiguous().view(torch.uint8 if t.element_size() == 1 else
                                              torch.int16 if t.element_size() == 2 else torch.int32)


def _same(got, want, what):
    a, b = _bits(got), _bits(want)
    assert a.shape == b.shape, what
    bad = int((a != b).sum())
    assert not bad, f"{what}: {bad} of {a.numel()} values differ"


def _state(lens, hkv, d, page, cache, seed, strided=False):
    g = torch.Generator().manual_seed(seed)
    need = [max(1, -(-n // page)) for n in lens]
    pages = sum(need) + 2
    perm, bt, at = torch.randperm(pages, generator=g), torch.full((len(lens), max(need)), -1, dtype=torch.int32), 0
    for s, n in enumerate(need):
        bt[s, :n] = perm[at : at + n]
        at += n
    pad = 16 if strided else 0
    codes = [torch.full((pages, hkv, page, d + pad), 3, dtype=torch.uint8, device=DEV).view(cache)[..., :d] for _ in range(2)]
    scales = [torch.full((pages, hkv, page + (3 if strided else 0)), -7.0, device=DEV)[..., :page] for _ in range(2)]
    return bt, codes, scales, g


def _expect(bt, codes, scales, src, seqs, pos, page):
    """The caches after a store of packed rows src (k, v), from their state before it."""
    out = []
    for c, s, x in zip(codes, scales, src):
        c, s = c.cpu().clone(), s.cpu().clone()
        q, qs = quantize(x.cpu(), c.dtype)
        for t, (i, p) in enumerate(zip(seqs, pos)):
            if p < 0 or p // page >= bt.shape[1] or not 0 <= int(bt[i, p // page]) < c.shape[0]:
                continue
            c.view(torch.uint8)[int(bt[i, p // page]), :, p % page] = q[t].view(torch.uint8)
            s[int(bt[i, p // page]), :, p % page] = qs[t]
        out.append((c, s))
    return out


@pytest.mark.parametrize("cache", [E4, I8])
@pytest.mark.parametrize("dtype,hkv,d,page,lens,strided", [
    (torch.bfloat16, 8, 128, 16, [1, 15, 16, 17, 0, 300], False),
    (torch.float16, 8, 128, 256, [700, 1, 255], False),
    (torch.bfloat16, 2, 64, 16, [33, 64, 5], False),
    (torch.float32, 3, 128, 4, [9, 1, 50], False),
    (torch.bfloat16, 1, 128, 16, [20], True),
    (torch.bfloat16, 5, 96, 7, [20, 8], False),
    (torch.float16, 2, 130, 16, [20, 8], True),
    (torch.bfloat16, 3, 256, 16, [19, 40], False),
])
def test_store_and_load(cache, dtype, hkv, d, page, lens, strided):
    bt, codes, scales, g = _state(lens, hkv, d, page, cache, d + page, strided)
    n = sum(lens)
    wide = 2 if strided else 1
    src = [(torch.randn(n, hkv, d * wide, generator=g) * torch.exp(2 * torch.randn(n, hkv, 1, generator=g))).to(dtype).to(DEV)[..., ::wide]
           for _ in range(2)]
    src[0][0] = 0.0  # rows of zeros
    src[1][-1, 0] = 0.0
    src[0][1, 0, 1:] = 0.0  # one number
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)
    seqs = [i for i, m in enumerate(lens) for _ in range(m)]
    pos = [p for m in lens for p in range(m)]
    want = _expect(bt, codes, scales, src, seqs, pos, page)
    store_kv_cache_quantized(src[0].transpose(0, 1), src[1].transpose(0, 1), *codes, *scales, bt.to(DEV), cu)
    for (c, s), gc, gs in zip(want, codes, scales):
        _same(gs, s, "scales")
        _same(gc, c, "codes")
    for to in (torch.bfloat16, torch.float16, torch.float32):
        got = load_kv_cache_quantized(*codes, *scales, bt.to(DEV), cu, n, dtype=to)
        for (c, s), x in zip(want, got):
            blk = torch.tensor([int(bt[i, p // page]) for i, p in zip(seqs, pos)])
            sl = torch.tensor([p % page for p in pos])
            _same(x, (c[blk, :, sl].float() * s[blk, :, sl][..., None]).to(to), f"rows as {to}")


@pytest.mark.parametrize("cache", [E4, I8])
def test_step_positions_and_what_is_left_alone(cache):
    """Positions (int32 and int64), tokens before the first and past the last
    sequence, pages past the table and outside the pool: skipped by the store,
    0 for the load, which rounds nothing else."""
    lens, page, hkv, d = [1, 1, 1, 1, 1], 16, 8, 128
    bt, codes, scales, g = _state([40] * 5, hkv, d, page, cache, 5)
    bt[1, 0], bt[2, 1] = -1, 1 << 30
    pos = [39, 3, 17, 999, -1]
    src = [torch.randn(9, hkv, d, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]
    cu = torch.tensor([2, 3, 4, 5, 6, 7], dtype=torch.int32, device=DEV)
    for kind in (torch.int32, torch.int64):
        where = torch.tensor([5, 5] + pos + [5, 5], dtype=kind, device=DEV)
        want = _expect(bt, codes, scales, [x[2:7] for x in src], range(5), pos, page)
        store_kv_cache_quantized(src[0].transpose(0, 1), src[1].transpose(0, 1), *codes, *scales, bt.to(DEV), cu, where)
        for (c, s), gc, gs in zip(want, codes, scales):
            _same(gs, s, "scales")
            _same(gc, c, "codes")
        k, v = load_kv_cache_quantized(*codes, *scales, bt.to(DEV), cu, 9, where)
        blk, sl = int(bt[0, 2]), 39 % page
        for x, (c, s) in zip((k, v), want):
            ref = torch.zeros(9, hkv, d)
            ref[2] = c[blk, :, sl].float() * s[blk, :, sl][:, None]
            assert torch.equal(x.cpu().float(), ref.bfloat16().float())


@pytest.mark.parametrize("cache", [E4, I8])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 128), (torch.float16, 80)])
def test_rows_that_are_not_ordinary(cache, dtype, d):
    """Rows of tiny values, of the type's largest, one infinity or NaN, ties:
    exact codes, NaN rows read back as NaN, all in one call."""
    page, info = 16, torch.finfo(dtype)
    bt, codes, scales, g = _state([10], 2, d, page, cache, 9)
    x = torch.randn(10, 2, d, generator=g)
    x = x.to(dtype)
    x[0] = info.tiny
    x[1] = info.tiny * info.eps  # the least subnormal
    x[2] = info.max
    x[3, 0, 5] = float("inf")
    x[3, 1, 7] = float("-inf")
    x[4, :, 2] = float("nan")
    x[5] = torch.linspace(-1, 1, d).to(dtype)
    x[6] = (torch.arange(d) - d // 2).to(dtype) / 2  # halves: ties of int8 where the scale is a power of two
    x[6, :, 0] = LARGEST[cache]
    x[7, 0, 1:] = info.tiny  # far below the largest
    x[7, 0, 0] = 1.0
    want = _expect(bt, codes, scales, [x, x.flip(0)], [0] * 10, range(10), page)
    cu = torch.tensor([0, 10], dtype=torch.int32, device=DEV)
    x = x.to(DEV)
    store_kv_cache_quantized(x.transpose(0, 1), x.flip(0).transpose(0, 1), *codes, *scales, bt.to(DEV), cu)
    for (c, s), gc, gs in zip(want, codes, scales):
        bad = torch.isnan(s)
        assert torch.equal(torch.isnan(gs.cpu()), bad)
        _same(gs.cpu()[~bad], s[~bad], "scales")
        _same(gc.cpu().view(torch.uint8)[~bad], c.view(torch.uint8)[~bad], "codes")
    k, _ = load_kv_cache_quantized(*codes, *scales, bt.to(DEV), cu, 10)
    assert bool(torch.isnan(k[3:5]).all()) and not bool(torch.isnan(k[5:]).any()) and not bool(torch.isnan(k[:3]).any())


def test_nothing_to_do():
    bt, codes, scales, _ = _state([3], 2, 128, 16, I8, 1)
    before = _bits(codes[0]).clone()
    z = torch.zeros(2, 0, 128, device=DEV)
    cu = torch.tensor([0, 0], dtype=torch.int32, device=DEV)
    store_kv_cache_quantized(z, z, *codes, *scales, bt.to(DEV), cu)
    k, v = load_kv_cache_quantized(*codes, *scales, bt.to(DEV), cu, 0)
    assert k.shape == v.shape == (0, 2, 128) and torch.equal(before, _bits(codes[0]))
    k, v = load_kv_cache_quantized(*codes, *scales, bt.to(DEV), cu, 3)  # tokens of no sequence
    assert not bool(k.any()) and not bool(v.any())


def test_outputs_given():
    """k_out and v_out, strided, of a type of their own."""
    bt, codes, scales, g = _state([30], 2, 128, 16, E4, 2)
    x = torch.randn(30, 2, 128, generator=g).to(DEV)
    cu = torch.tensor([0, 30], dtype=torch.int32, device=DEV)
    store_kv_cache_quantized(x.transpose(0, 1), x.transpose(0, 1), *codes, *scales, bt.to(DEV), cu)
    plain = load_kv_cache_quantized(*codes, *scales, bt.to(DEV), cu, 30, dtype=torch.float16)[0]
    whole = torch.full((30, 2, 4, 128), 9.0, dtype=torch.float16, device=DEV)
    k, v = load_kv_cache_quantized(*codes, *scales, bt.to(DEV), cu, 30, k_out=whole[:, :, 0], v_out=whole[:, :, 2])
    assert torch.equal(k, plain) and torch.equal(v, plain)
    assert bool((whole[:, :, 1::2] == 9).all())
