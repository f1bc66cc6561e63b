"""Attention of drafted tokens' trees against 64-bit attention over what each node
sees (tolerances derived in rows_reference): trees of one node to several mask
words, chains, stars, random masks, masks that leave a node nothing, contexts of
no token to several splits, block edges, GQA groups, types, page sizes; rows that
are not computed keep what they held; keys that a node does not see may hold NaN
or infinities although another node sees them."""

import pytest
import torch

from tests.rows_reference import attend, check, half_step, pool, rows
from tinyserver_amd.kernels import paged_attention_forward, paged_attention_tree

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _masks(nodes, kind, g):
    """(n, n) truth values a sequence: what each node sees of its own tree."""
    out = []
    for n in nodes:
        if kind == "chain":
            m = torch.ones(n, n).tril().bool()
        elif kind == "star":
            m = torch.eye(n).bool()
            m[:, :1] = True
        elif kind == "random":
            m = torch.rand(n, n, generator=g) < 0.4
        elif kind == "none":
            m = torch.zeros(n, n).bool()
        else:  # a tree
            m = torch.eye(n).bool()
            for i in range(1, n):
                p = int(torch.randint(-1, i, (1,), generator=g))
                if p >= 0:
                    m[i] |= m[p]
        out.append(m)
    return out


def _words(masks, words):
    out = torch.zeros(sum(len(m) for m in masks), words, dtype=torch.int64)
    at = 0
    for m in masks:
        for i in range(len(m)):
            for j in torch.nonzero(m[i]).flatten().tolist():
                b = j % 64
                out[at + i, j // 64] |= (1 << b) if b < 63 else -(1 << 63)
        at += len(m)
    return out


def _case(ctx, nodes, hq, hkv, d, page, dtype, kind, seed=0):
    g = torch.Generator().manual_seed(seed + d + sum(nodes))
    kc, vc, bt = pool([a + b for a, b in zip(ctx, nodes)], hkv, d, page, seed + page)
    kc, vc = kc.to(dtype), vc.to(dtype)
    q = torch.randn(sum(nodes), hq, d, generator=g).to(dtype)
    masks = _masks(nodes, kind, g)
    ref, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    at, u = 0, half_step(dtype)
    for s, (c, n) in enumerate(zip(ctx, nodes)):
        for i in range(n):
            see = list(range(c)) + [c + j for j in torch.nonzero(masks[s][i]).flatten().tolist()]
            ref[at], tol[at] = attend(q[at], rows(kc, bt[s], see), rows(vc, bt[s], see), d**-0.5, u, u)
            at += 1
        for p in range(c + n, -(-(c + n) // page) * page):  # past the last node
            kc[int(bt[s, p // page]), :, p % page] = float("nan")
            vc[int(bt[s, p // page]), :, p % page] = float("inf")
    return q, kc, vc, bt, masks, ref, tol


def _run(q, kc, vc, bt, page, ctx, nodes, mask, **kw):
    cu = torch.tensor([0] + nodes).cumsum(0).to(torch.int32)
    return paged_attention_tree(q.to(DEV), kc.to(DEV), vc.to(DEV), bt.to(DEV), page,
                                torch.tensor(ctx, dtype=torch.int32, device=DEV), cu.to(DEV), mask.to(DEV), **kw)


@pytest.mark.parametrize("kind", ["tree", "chain", "star", "random", "none"])
@pytest.mark.parametrize("hq,hkv,d,page,dtype,ctx,nodes", [
    (16, 8, 128, 16, BF, [0, 1, 31, 32, 33, 300], [1, 2, 5, 0, 16, 17]),
    (32, 8, 128, 16, F16, [100, 7, 64], [13, 33, 8]),
    (64, 8, 128, 256, BF, [250, 20], [20, 7]),
    (4, 1, 64, 16, BF, [40, 0], [40, 64]),
    (6, 2, 64, 48, F16, [40, 90], [9, 3]),
    (3, 3, 128, 16, BF, [17, 200], [64, 1]),
    (4, 2, 128, 4, F32, [9, 30], [3, 10]),
    (4, 2, 128, 4, BF, [9, 30], [3, 10]),
    (4, 2, 80, 16, BF, [9, 30], [3, 10]),
])
def test_trees(kind, hq, hkv, d, page, dtype, ctx, nodes):
    q, kc, vc, bt, masks, ref, tol = _case(ctx, nodes, hq, hkv, d, page, dtype, kind)
    out = _run(q, kc, vc, bt, page, ctx, nodes, _words(masks, 1))
    check(out, ref, tol, f"{kind} {hq}/{hkv} x {d}, page {page}, {dtype}")


@pytest.mark.parametrize("ctx,nodes,words", [([50, 3], [100, 130], 3), ([2000, 5000], [20, 66], 2), ([0], [65], 2)])
def test_wide_and_long(ctx, nodes, words):
    q, kc, vc, bt, masks, ref, tol = _case(ctx, nodes, 8, 2, 128, 16, BF, "tree")
    check(_run(q, kc, vc, bt, 16, ctx, nodes, _words(masks, words)), ref, tol, f"{ctx} {nodes}")
    check(_run(q, kc, vc, bt, 16, ctx, nodes, _words(masks, words + 2), max_nodes=max(nodes)), ref, tol, "spare words")


def test_a_chain_of_one_is_paged_attention():
    ctx = [700, 16, 33]
    kc, vc, bt = pool([c + 1 for c in ctx], 8, 128, 16, 4)
    kc, vc = kc.to(BF).to(DEV), vc.to(BF).to(DEV)
    q = torch.randn(3, 32, 128).to(BF).to(DEV)
    a = _run(q, kc, vc, bt, 16, ctx, [1, 1, 1], torch.ones(3, dtype=torch.int64))
    b = paged_attention_forward(q, kc, vc, bt.to(DEV), 16, torch.tensor(ctx, dtype=torch.int32, device=DEV) + 1)
    assert float((a.float() - b.float()).abs().max()) <= 2.0**-7 * float(b.float().abs().max())


def test_rows_that_are_not_computed():
    """Rows outside every sequence and rows past max_nodes keep what they held; so do those past the mask's width."""
    ctx, nodes = [40, 100], [6, 70]
    q, kc, vc, bt, masks, ref, tol = _case(ctx, nodes, 8, 2, 128, 16, BF, "tree")
    mask = _words(masks, 2)
    n = sum(nodes)
    q2 = torch.cat([q[:2], q, q[:3]])
    m2 = torch.cat([mask[:2], mask, mask[:3]])
    cu = torch.tensor([2, 8, 78], dtype=torch.int32, device=DEV)

    def run(mask, **kw):
        out = torch.full((n + 5, 8, 128), 9.0, dtype=BF, device=DEV)
        paged_attention_tree(q2.to(DEV), kc.to(DEV), vc.to(DEV), bt.to(DEV), 16,
                             torch.tensor(ctx, dtype=torch.int32, device=DEV), cu, mask.to(DEV), out=out, **kw)
        return out.cpu()

    out = run(m2)
    check(out[2:-3], ref, tol, "inside")
    assert bool((out[:2] == 9).all()) and bool((out[-3:] == 9).all())
    out = run(m2, max_nodes=5)
    check(out[2:7], ref[:5], tol[:5], "first sequence")
    assert bool((out[7] == 9).all()) and bool((out[13:] == 9).all())
    out = run(m2[:, :1])  # 64 nodes
    check(out[2:8], ref[:6], tol[:6], "first sequence, one word")
    assert bool((out[72:] == 9).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("hq,hkv,d,page,dtype", [(8, 2, 128, 16, BF), (16, 2, 128, 16, F16), (4, 1, 64, 32, BF), (2, 1, 128, 4, BF)])
def test_nodes_that_are_not_seen(hq, hkv, d, page, dtype, bad):
    """A drafted token whose V (or K) row is not finite reaches the nodes that see it and no others."""
    ctx, nodes = [37], [20]
    q, kc, vc, bt, masks, ref, tol = _case(ctx, nodes, hq, hkv, d, page, dtype, "tree", seed=2)
    m, j, k = masks[0], 1, 4
    at, at2 = ctx[0] + j, ctx[0] + k
    vc[int(bt[0, at // page]), 0, at % page, 3] = bad
    kc[int(bt[0, at2 // page]), hkv - 1, at2 % page] = float("nan")
    out = _run(q, kc, vc, bt, page, ctx, nodes, _words(masks, 1)).cpu()
    seen = torch.zeros(nodes[0], hq, d, dtype=torch.bool)
    seen[m[:, j], : hq // hkv, 3] = True
    seen[m[:, k], -(hq // hkv):] = True
    assert 0 < int(m[:, j].sum()) < nodes[0]
    assert not bool(torch.isfinite(out[seen].float()).any())
    check(torch.where(seen, 0, out), torch.where(seen, 0.0, ref), tol, f"{hq}/{hkv} x {d}, {bad}")


def test_pages_outside_the_pool_and_tables_that_end():
    """A context page with an id outside the pool is not seen; nodes past the table's end are not either."""
    ctx, nodes = [60], [8]
    q, kc, vc, bt, masks, ref, tol = _case(ctx, nodes, 8, 2, 128, 16, BF, "chain")
    bt = bt[:, :4].clone()  # 64 tokens: nodes 0 .. 3
    bt[0, 1] = -1
    out = _run(q, kc, vc, bt, 16, ctx, nodes, _words(masks, 1))
    for i in range(8):
        see = list(range(60)) + [60 + j for j in range(min(i + 1, 4))]
        r, t = attend(q[i], rows(kc, bt[0], see), rows(vc, bt[0], see), 128**-0.5, half_step(BF), half_step(BF))
        check(out[i], r, t, f"node {i}")


def test_strides():
    ctx, nodes = [130, 20], [9, 30]
    q, kc, vc, bt, masks, ref, tol = _case(ctx, nodes, 8, 2, 128, 16, BF, "tree")
    wide = torch.zeros(39, 12, 128, dtype=BF)
    wide[:, 2:10] = q
    big = torch.zeros(39, 5, dtype=torch.int64)
    big[:, 1:2] = _words(masks, 1)
    cu = torch.tensor([0, 9, 39], dtype=torch.int32, device=DEV)
    out = torch.full((39, 8, 256), 3.0, dtype=BF, device=DEV)
    got = paged_attention_tree(wide.to(DEV)[:, 2:10], kc.to(DEV), vc.to(DEV), bt.to(DEV), 16,
                               torch.tensor(ctx, dtype=torch.int64, device=DEV), cu.long(), big.to(DEV)[:, 1:2], out=out[..., :128])
    check(got, ref, tol, "strides")
    assert bool((out[..., 128:] == 3).all())
