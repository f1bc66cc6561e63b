"""Attention of a chunk over the paged cache against 64 bits (tolerances derived in
rows_reference): contexts of no token to several splits, chunks of no token to
several row blocks, block edges, GQA groups, types, head_dims, page sizes, strides;
pages outside the pool and past the table; rows that are not computed; keys that a
row does not see may hold anything although another row sees them."""

import pytest
import torch

from tests.chunk_reference import inputs, reference
from tests.rows_reference import check
from tinyserver_amd.kernels import flash_attn_varlen_func, paged_attention_chunk, paged_attention_forward

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _cu(new):
    return torch.tensor([0] + list(new)).cumsum(0).to(torch.int32).to(DEV)


def _run(q, kc, vc, bt, ctx, new, **kw):
    return paged_attention_chunk(q.to(DEV), kc.to(DEV), vc.to(DEV), bt.to(DEV), kc.shape[2],
                                 torch.tensor(ctx, dtype=torch.int32, device=DEV), _cu(new), **kw)


def _check(ctx, new, hq, hkv, d, page, dtype, seed=0, **kw):
    q, kc, vc, bt = inputs(ctx, new, hq, hkv, d, page, dtype, seed)
    ref, tol = reference(q, kc, vc, bt, ctx, new, kw.get("softmax_scale", d**-0.5))
    check(_run(q, kc, vc, bt, ctx, new, **kw), ref, tol, f"{ctx} + {new}, {hq}/{hkv} x {d}, page {page}, {dtype}")


@pytest.mark.parametrize("ctx,new", [
    ([0], [1]), ([0, 1, 31, 32, 33, 300], [1, 2, 5, 0, 16, 17]), ([100, 7, 64], [13, 33, 8]),
    ([0, 0, 0], [70, 1, 129]), ([250, 20, 500], [130, 64, 1]), ([1000, 3], [3, 260]),
])
@pytest.mark.parametrize("hq,hkv,d,page,dtype", [
    (16, 8, 128, 16, BF), (32, 8, 128, 256, F16), (8, 1, 128, 16, F16), (2, 2, 64, 16, BF), (6, 2, 64, 48, F16),
    (20, 4, 128, 32, BF), (32, 2, 128, 16, BF), (4, 2, 128, 16, F32), (3, 1, 64, 16, F32), (4, 2, 128, 4, BF),
    (4, 2, 80, 16, BF), (2, 1, 128, 24, F32), (40, 1, 64, 16, F16),
])
def test_shapes(ctx, new, hq, hkv, d, page, dtype):
    _check(ctx, new, hq, hkv, d, page, dtype, max_seqlen=max(new))
    if page == 16:
        _check(ctx, new, hq, hkv, d, page, dtype, seed=1)  # (max_seqlen not known)


@pytest.mark.parametrize("ctx,new,hq,hkv,dtype", [
    ([20000], [3], 8, 2, BF), ([9000, 40, 5000], [40, 200, 1], 8, 1, F16), ([33000], [300], 4, 2, BF),
    ([0], [1500], 8, 2, F16), ([4000, 17, 0, 2500], [1, 1, 1, 1], 32, 8, BF), ([5000], [70], 4, 1, F32),
])
def test_long(ctx, new, hq, hkv, dtype):
    _check(ctx, new, hq, hkv, 128, 16, dtype, max_seqlen=max(new))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_sequences(dtype):
    r = torch.Generator().manual_seed(3)
    n = 1500
    ctx = torch.randint(0, 60, (n,), generator=r).tolist()
    new = torch.randint(0, 4, (n,), generator=r).tolist()
    _check(ctx, new, 4, 2, 64, 16, dtype, max_seqlen=3)


@pytest.mark.parametrize("scale", [0.3, -0.1, 0.0])
def test_scale(scale):
    _check([70, 5], [33, 9], 8, 2, 128, 16, BF, softmax_scale=scale)


@pytest.mark.parametrize("dtype,page", [(BF, 16), (F16, 32), (F32, 16), (BF, 4)])
def test_pages_that_are_not_there(dtype, page):
    """Ids outside the pool in context and chunk, tables that end before the tokens, contexts past the table, a first
    row that sees nothing."""
    ctx, new = [90, 5, 200, 3], [40, 20, 30, 9]
    q, kc, vc, bt = inputs(ctx, new, 8, 2, 128, page, dtype)
    bt[0, 1], bt[0, -(-100 // page)] = -1, kc.shape[0]
    bt[1, 0] = 1 << 30  # row 0 of sequence 1 sees nothing up to the next page
    bt[3, :] = -7
    ref, tol = reference(q, kc, vc, bt, ctx, new, 128**-0.5)
    check(_run(q, kc, vc, bt, ctx, new, max_seqlen=40), ref, tol, f"bad pages, {dtype}")
    short = bt[:, : -(-210 // page)].contiguous()  # sequence 2 ends inside its chunk
    ref, tol = reference(q, kc, vc, short, ctx, new, 128**-0.5)
    check(_run(q, kc, vc, short, ctx, new), ref, tol, f"short table, {dtype}")
    far = [90, 5, 10**6, 3]
    ref, tol = reference(q, kc, vc, short, far, new, 128**-0.5)
    check(_run(q, kc, vc, short, far, new), ref, tol, f"context past the table, {dtype}")
    back = [-5, 5, 200, 3]
    ref, tol = reference(q, kc, vc, bt, [0, 5, 200, 3], new, 128**-0.5)
    check(_run(q, kc, vc, bt, back, new), ref, tol, f"negative context, {dtype}")
    assert float(_run(q, kc, vc, bt, ctx, new)[90:].abs().max()) == 0.0
    empty = _run(q, kc[:0], vc[:0], bt, ctx, new)
    assert float(empty.abs().max()) == 0.0 and float(_run(q, kc, vc, bt[:, :0], ctx, new).abs().max()) == 0.0


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_what_a_row_does_not_see(dtype):
    """A NaN or infinity in a later token's K or V reaches the rows that see it and no others."""
    ctx, new = [61, 0], [100, 140]
    q, kc, vc, bt = inputs(ctx, new, 8, 2, 128, 16, dtype)

    def at(cache, s, p):
        return cache[int(bt[s, p // 16]), :, p % 16]

    at(vc, 0, 61 + 50)[0, 3] = float("nan")
    at(vc, 1, 100)[1, :] = float("inf")
    at(vc, 1, 101)[1, :] = float("-inf")
    ref, tol = reference(q, kc, vc, bt, ctx, new, 128**-0.5)
    out = _run(q, kc, vc, bt, ctx, new, max_seqlen=140)
    bad = torch.isnan(ref)
    assert 0 < int(bad.sum()) < bad.numel() and not bool(torch.isfinite(out.cpu()[bad]).any())
    check(torch.where(bad.to(DEV), 0.0, out.double()), ref.nan_to_num(), tol, f"V not finite, {dtype}")
    q, kc, vc, bt = inputs(ctx, new, 8, 2, 128, 16, dtype)
    clean = _run(q, kc, vc, bt, ctx, new, max_seqlen=140)
    at(kc, 0, 61 + 97)[:, 5] = float("nan")
    at(kc, 1, 139)[:, 0] = float("inf")
    out = _run(q, kc, vc, bt, ctx, new, max_seqlen=140)
    seen = torch.zeros(240, dtype=torch.bool)
    seen[97:100] = seen[239:] = True
    assert torch.isnan(out[97:100]).all() and torch.equal(out[~seen.to(DEV)], clean[~seen.to(DEV)])


@pytest.mark.parametrize("dtype,page", [(BF, 16), (F32, 16), (F16, 4)])
def test_rows_that_are_not_computed(dtype, page):
    ctx, new = [40, 100, 7], [6, 70, 40]
    q, kc, vc, bt = inputs(ctx, new, 8, 2, 128, page, dtype)
    ref, tol = reference(q, kc, vc, bt, ctx, new, 128**-0.5)
    q2 = torch.cat([q[:2], q, q[:3]]).to(DEV)
    out = torch.full(q2.shape, 7.0, dtype=dtype, device=DEV)
    cu = (_cu(new) + 2).to(torch.int32)
    got = paged_attention_chunk(q2, kc.to(DEV), vc.to(DEV), bt.to(DEV), page,
                                torch.tensor(ctx, dtype=torch.int32, device=DEV), cu, max_seqlen=33, out=out)
    assert got is out
    left = torch.ones(len(q2), dtype=torch.bool)
    for a, n in ((2, 6), (8, 33), (78, 33)):
        left[a : a + n] = False
    assert bool((out[left.to(DEV)] == 7.0).all())
    keep = ~left[2:-3]
    check(out[2:-3][keep.to(DEV)], ref[keep], tol[keep], f"max_seqlen, {dtype}")


def test_strides_and_orders():
    ctx, new = [70, 5], [33, 90]
    q, kc, vc, bt = inputs(ctx, new, 8, 2, 128, 16, BF)
    ref, tol = reference(q, kc, vc, bt, ctx, new, 128**-0.5)
    q, kc, vc, bt = (x.to(DEV) for x in (q, kc, vc, bt))
    c, cu = torch.tensor(ctx, dtype=torch.int32, device=DEV), _cu(new)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    tokens_first = kc.transpose(1, 2).contiguous().transpose(1, 2), vc.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros(*kc.shape[:3], 136, dtype=BF, device=DEV)
    wide[..., :128] = kc
    odd = torch.zeros(*kc.shape[:3], 129, dtype=BF, device=DEV)
    odd[..., 1:] = vc
    every = torch.zeros(*q.shape[:2], 256, dtype=BF, device=DEV)
    every[..., ::2] = q
    slow_out = torch.zeros(128, 8, 123, dtype=BF, device=DEV).permute(2, 1, 0)
    for name, args, kw in (("heads first", (heads_first, kc, vc), {}), ("tokens first", (q, *tokens_first), {}),
                           ("padded rows", (q, wide[..., :128], vc), {}), ("unaligned rows", (q, kc, odd[..., 1:]), {}),
                           ("every second", (every[..., ::2], kc, vc), {}), ("out", (q, kc, vc), {"out": slow_out})):
        check(paged_attention_chunk(*args, bt, 16, c, cu, **kw), ref, tol, name)
    wide_bt = torch.full((2, 40), -1, dtype=torch.int32, device=DEV)
    wide_bt[:, : 2 * bt.shape[1] : 2] = bt
    check(paged_attention_chunk(q, kc, vc, wide_bt[:, : 2 * bt.shape[1] : 2], 16, c.long(), cu.long()), ref, tol, "tables")


def test_against_decode_and_prefill():
    """One token a sequence is paged_attention_forward, and no context flash_attn_varlen_func, within roundings."""
    ctx = [700, 15, 33]
    q, kc, vc, bt = (x.to(DEV) for x in inputs(ctx, [1, 1, 1], 32, 8, 128, 16, BF))
    c = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    a, b = _run(q, kc, vc, bt, ctx, [1, 1, 1]), paged_attention_forward(q, kc, vc, bt, 16, c + 1)
    assert float((a.float() - b.float()).abs().max()) <= 2.0**-7 * float(b.float().abs().max())
    new = [100, 1, 260]
    q, kc, vc, bt = (x.to(DEV) for x in inputs([0, 0, 0], new, 32, 8, 128, 16, BF))
    rows = [(s, p) for s, n in enumerate(new) for p in range(n)]
    k, v = (torch.stack([x[int(bt[s, p // 16]), :, p % 16] for s, p in rows]) for x in (kc, vc))
    cu = _cu(new)
    a, b = _run(q, kc, vc, bt, [0, 0, 0], new), flash_attn_varlen_func(q, k, v, cu, cu, 260, 260, True)
    assert float((a.float() - b.float()).abs().max()) <= 2.0**-7 * float(b.float().abs().max())


def test_nothing_to_do():
    q, kc, vc, bt = inputs([5, 9], [3, 4], 8, 2, 128, 16, BF)
    none = torch.zeros(0, 8, 128, dtype=BF)
    assert _run(none, kc, vc, bt, [5, 9], [0, 0]).shape == (0, 8, 128)
    assert _run(none, kc, vc, bt[:0], [], []).shape == (0, 8, 128)
    out = torch.full((7, 8, 128), 3.0, dtype=BF, device=DEV)
    assert bool((_run(q, kc, vc, bt, [5, 9], [0, 0], out=out) == 3.0).all())
    assert bool((_run(q, kc, vc, bt, [5, 9], [3, 4], max_seqlen=0, out=out) == 3.0).all())
    assert _run(q[:, :0], kc, vc, bt, [5, 9], [3, 4]).shape == (7, 0, 128)
