"""Windowed and 8-bit decode, draft trees and the 8-bit store and load as a server
uses them: a prompt, its cache and decode steps in one run; a draft's verification
behind qk_norm_rope_store; captured steps replayed with new inputs, two of them at
once; calls from two threads on streams of their own; repeated calls; batches past
one launch's limit; empty batches; pools and tokens past 4 GB."""

import threading

import pytest
import torch

from tests.rows_reference import attend, check, half_step, pool, rows, visible
from tinyserver_amd.kernels import (
    flash_attn_varlen_window,
    load_kv_cache_quantized,
    paged_attention_quantized,
    paged_attention_tree,
    paged_attention_window,
    qk_norm_rope_store,
    store_kv_cache_paged,
    store_kv_cache_quantized,
)

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16 = torch.bfloat16, torch.float16
E4, I8 = torch.float8_e4m3fn, torch.int8


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cache8(pages, hkv, page, d, cache):
    kc, vc = (torch.zeros(pages, hkv, page, d, dtype=torch.uint8, device=DEV).view(cache) for _ in range(2))
    ks, vs = (torch.zeros(pages, hkv, page, device=DEV) for _ in range(2))
    return kc, vc, ks, vs


@pytest.mark.parametrize("cache", [E4, I8])
def test_a_prompt_and_its_decode_steps(cache):
    hq, hkv, d, page, window, sinks, steps = 16, 8, 128, 16, 40, 5, 3
    lens = [70, 1, 33]
    g = torch.Generator().manual_seed(5)
    total = [n + steps for n in lens]
    bt = _i32([[8 * s + i for i in range(8)] for s in range(3)])
    kc, vc, ks, vs = _cache8(24, hkv, page, d, cache)
    kw, vw = (torch.zeros(24, hkv, page, d, dtype=BF, device=DEV) for _ in range(2))
    seqs = [[torch.randn(n, h, d, generator=g).to(BF) for h in (hq, hkv, hkv)] for n in total]
    q, k, v = (torch.cat([x[i][:n] for x, n in zip(seqs, lens)]).to(DEV) for i in range(3))
    cu = _i32([0, 70, 71, 104])
    out = flash_attn_varlen_window(q, k, v, cu, cu, 70, 70, window, sinks)
    store_kv_cache_quantized(k.transpose(0, 1), v.transpose(0, 1), kc, vc, ks, vs, bt, cu)
    pos = _i32([i for n in lens for i in range(n)])
    store_kv_cache_paged(k.transpose(0, 1), v.transpose(0, 1), kw, vw, bt, cu, pos)
    u = half_step(BF)
    # the prompts' last rows, by the prefill and by a decode over the cache
    last = q[torch.tensor([69, 70, 103], device=DEV)]
    dec = paged_attention_window(last, kw, vw, bt, page, _i32(lens), window, sinks)
    for s, n in enumerate(lens):
        see = visible(n, window, sinks)
        ref, tol = attend(last[s].cpu(), seqs[s][1][see], seqs[s][2][see], d**-0.5, u, u)
        check(out[int(cu[s + 1]) - 1], ref, tol, f"prefill {s}")
        check(dec[s], ref, tol, f"decode {s}")
    one = _i32([0, 1, 2, 3])
    for t in range(steps):
        q, k, v = (torch.stack([x[i][n + t] for x, n in zip(seqs, lens)]).to(DEV) for i in range(3))
        now = _i32([n + t for n in lens])
        store_kv_cache_quantized(k.transpose(0, 1), v.transpose(0, 1), kc, vc, ks, vs, bt, one, now)
        store_kv_cache_paged(k.transpose(0, 1), v.transpose(0, 1), kw, vw, bt, one, now)
        o8 = paged_attention_quantized(q, kc, vc, ks, vs, bt, page, now + 1)
        ow = paged_attention_window(q, kw, vw, bt, page, now + 1, window, sinks)
        k64, v64 = (c.cpu().double() * s.cpu()[..., None].double() for c, s in ((kc, ks), (vc, vs)))
        for s, n in enumerate(lens):
            every, see = range(n + t + 1), visible(n + t + 1, window, sinks)
            ref, tol = attend(q[s].cpu(), rows(k64, bt[s].cpu(), every), rows(v64, bt[s].cpu(), every), d**-0.5, u, u)
            check(o8[s], ref, tol, f"step {t} sequence {s} 8 bits")
            ref, tol = attend(q[s].cpu(), seqs[s][1][see], seqs[s][2][see], d**-0.5, u, u)
            check(ow[s], ref, tol, f"step {t} sequence {s} window")
    # the whole prefixes back, as attention over them would read them
    cu = _i32([0, 73, 77, 113])
    kb, vb = load_kv_cache_quantized(kc, vc, ks, vs, bt, cu, 113, dtype=torch.float32)
    for s, n in enumerate(total):
        for back, c, sc in ((kb, kc, ks), (vb, vc, vs)):
            want = rows(c.cpu().float() * sc.cpu()[..., None], bt[s].cpu(), range(n))
            assert torch.equal(back[int(cu[s]) : int(cu[s + 1])].cpu(), want)


def test_a_draft_behind_the_stored_nodes():
    hq, hkv, d, page = 16, 8, 128, 16
    ctx, nodes = [37, 0, 300], [6, 3, 1]
    parents = [[-1, 0, 0, 1, 2, 4], [-1, 0, -1], [-1]]
    g = torch.Generator().manual_seed(11)
    kc, vc, bt = pool([a + b for a, b in zip(ctx, nodes)], hkv, d, page, 3)
    kc, vc = kc.to(BF).to(DEV), vc.to(BF).to(DEV)
    n = sum(nodes)
    q, k, v = (torch.randn(n, h, d, generator=g).to(BF).to(DEV) for h in (hq, hkv, hkv))
    wq, wk = (torch.rand(d, generator=g).to(BF).to(DEV) + 0.5 for _ in range(2))
    depth, mask, at = [], [], []
    for s, ps in enumerate(parents):
        bits, dep = [], []
        for i, p in enumerate(ps):
            bits.append((1 << i) | (bits[p] if p >= 0 else 0))
            dep.append(ctx[s] + (dep[p] - ctx[s] + 1 if p >= 0 else 0))
        mask += bits
        depth += dep
        at += [ctx[s] + i for i in range(len(ps))]
    ang = torch.tensor(depth)[:, None] * 10000.0 ** (-torch.arange(0, d, 2) / d)
    cos, sin = (torch.cat([f(ang)] * 2, -1).to(BF).to(DEV) for f in (torch.cos, torch.sin))
    cu = _i32([0, 6, 9, 10])
    qr, _ = qk_norm_rope_store(q, k, v, wq, wk, cos, sin, 1e-6, kc, vc, bt.to(DEV), cu, _i32(at), return_k=False)
    out = paged_attention_tree(qr, kc, vc, bt.to(DEV), page, _i32(ctx), cu, torch.tensor(mask, device=DEV), max_nodes=6)
    row, kk, vv = 0, kc.cpu(), vc.cpu()
    for s, m in enumerate(nodes):
        for i in range(m):
            see = list(range(ctx[s])) + [ctx[s] + j for j in range(m) if mask[row] >> j & 1]
            ref, tol = attend(qr[row].cpu(), rows(kk, bt[s], see), rows(vv, bt[s], see), d**-0.5, half_step(BF), half_step(BF))
            check(out[row], ref, tol, f"sequence {s} node {i}")
            if i == 0 or all(p == j - 1 for j, p in enumerate(parents[s][: i + 1])):  # a chain so far: a decode step
                one = paged_attention_window(qr[row : row + 1], kc, vc, bt[s : s + 1].to(DEV), page, _i32([ctx[s] + i + 1]), 1 << 20)
                check(one[0], ref, tol, f"sequence {s} node {i} as decode")
            row += 1


@pytest.mark.parametrize("hq,d,dtype", [(8, 128, BF), (32, 128, BF), (4, 64, F16), (6, 80, BF)])
def test_a_node_that_sees_one_past_max_nodes(hq, d, dtype):
    """Only the first 3 rows of a sequence are computed; they may see its later nodes."""
    hkv, page, ctx, nodes = 2, 16, [30, 5], [7, 40]
    kc, vc, bt = pool([a + b for a, b in zip(ctx, nodes)], hkv, d, page, 9)
    kc, vc = kc.to(dtype), vc.to(dtype)
    g = torch.Generator().manual_seed(d)
    q = torch.randn(47, hq, d, generator=g).to(dtype)
    mask = torch.randint(0, 1 << 40, (47,), generator=g)
    mask[:7] &= 127
    out = torch.full((47, hq, d), 3.0, dtype=dtype, device=DEV)
    paged_attention_tree(q.to(DEV), kc.to(DEV), vc.to(DEV), bt.to(DEV), page, _i32(ctx), _i32([0, 7, 47]), mask.to(DEV),
                         max_nodes=3, out=out)
    for s, at in enumerate((0, 7)):
        for i in range(3):
            see = list(range(ctx[s])) + [ctx[s] + j for j in range(nodes[s]) if int(mask[at + i]) >> j & 1]
            ref, tol = attend(q[at + i], rows(kc, bt[s], see), rows(vc, bt[s], see), d**-0.5, half_step(dtype), half_step(dtype))
            check(out[at + i], ref, tol, f"sequence {s} node {i}")
        assert bool((out[at + 3 : at + nodes[s]] == 3).all())


@pytest.mark.parametrize("batch", [40, 128, 129])
@pytest.mark.parametrize("most", [3, 9, 33])
def test_many_ragged_trees(batch, most):
    """More workgroups than CUs, lengths and node counts of all kinds (none among them)."""
    hq, hkv, d, page = 16, 4, 64, 16
    g = torch.Generator().manual_seed(batch + most)
    ctx = torch.where(torch.rand(batch, generator=g) < 0.2, 0, torch.randint(1, 900, (batch,), generator=g)).tolist()
    nodes = torch.randint(0, most + 1, (batch,), generator=g).tolist()
    nodes[3], ctx[5], ctx[6] = most, 899, 899
    kc, vc, bt = pool([a + b for a, b in zip(ctx, nodes)], hkv, d, page, 4)
    kc, vc = kc.to(BF), vc.to(BF)
    n = sum(nodes)
    q = torch.randn(n, hq, d, generator=g).to(BF)
    mask = torch.randint(0, 1 << most, (n,), generator=g)
    cu = torch.tensor([0] + nodes).cumsum(0).tolist()
    out = paged_attention_tree(q.to(DEV), kc.to(DEV), vc.to(DEV), bt.to(DEV), page, _i32(ctx), _i32(cu), mask.to(DEV))
    ref, tol, at = [], [], []
    for s in range(batch):
        for i in {0, nodes[s] - 1} if nodes[s] else ():
            see = list(range(ctx[s])) + [ctx[s] + j for j in range(nodes[s]) if int(mask[cu[s] + i]) >> j & 1]
            r, t = attend(q[cu[s] + i], rows(kc, bt[s], see), rows(vc, bt[s], see), d**-0.5, half_step(BF), half_step(BF))
            ref.append(r)
            tol.append(t)
            at.append(cu[s] + i)
    check(out[torch.tensor(at, device=DEV)], torch.stack(ref), torch.stack(tol), f"{batch} trees of up to {most}")


def _step(cache, hq, batch, longest, page=16, d=128, hkv=8):
    """A decode step over an 8-bit cache, a windowed one and a draft's, on inputs that a caller overwrites."""
    g = torch.Generator(device=DEV).manual_seed(batch + longest)
    mb = -(-longest // page) + 1
    pages = batch * mb
    c8 = _cache8(pages, hkv, page, d, cache)
    kw, vw = (torch.randn(pages, hkv, page, d, generator=g, device=DEV).to(BF) for _ in range(2))
    x = dict(
        q=torch.randn(batch, hq, d, generator=g, device=DEV).to(BF),
        k=torch.randn(batch, hkv, d, generator=g, device=DEV).to(BF),
        v=torch.randn(batch, hkv, d, generator=g, device=DEV).to(BF),
        bt=torch.randperm(pages, generator=g, device=DEV).to(torch.int32).view(batch, mb),
        lens=torch.randint(1, longest, (batch,), generator=g, device=DEV, dtype=torch.int32),
        mask=torch.randint(1, 8, (3 * batch,), generator=g, device=DEV),
        qt=torch.randn(3 * batch, hq, d, generator=g, device=DEV).to(BF),
    )
    one = torch.arange(batch + 1, dtype=torch.int32, device=DEV)
    every = torch.arange(0, 3 * batch + 1, 3, dtype=torch.int32, device=DEV)
    tok = torch.arange(batch * longest, device=DEV) // longest
    prompt = torch.randn(batch * longest, hkv, d, generator=g, device=DEV).to(BF).transpose(0, 1)
    store_kv_cache_quantized(prompt, prompt, *c8, x["bt"], (one * longest).to(torch.int32))
    del tok

    def run():
        store_kv_cache_quantized(x["k"].transpose(0, 1), x["v"].transpose(0, 1), *c8, x["bt"], one, x["lens"] - 1)
        a = paged_attention_quantized(x["q"], *c8, x["bt"], page, x["lens"])
        b = paged_attention_window(x["q"], kw, vw, x["bt"], page, x["lens"], 100, 4)
        c = paged_attention_tree(x["qt"], kw, vw, x["bt"], page, x["lens"] - 1, every, x["mask"], max_nodes=3)
        k, v = load_kv_cache_quantized(*c8, x["bt"], one, batch, dtype=BF)
        f = flash_attn_varlen_window(x["qt"], x["qt"][:, :hkv], x["qt"][:, :hkv], every, every, 3, 3, 2, 1)
        return a, b, c, k, v, f

    def renew(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        for n in ("q", "k", "v", "qt"):
            x[n].copy_(torch.randn(x[n].shape, generator=g, device=DEV))
        x["lens"].copy_(torch.randint(1, longest, (batch,), generator=g, device=DEV))
        x["mask"].copy_(torch.randint(0, 8, (3 * batch,), generator=g, device=DEV))

    return run, renew


def _same(got, want, what):
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a.cpu().view(torch.int16), b.cpu().view(torch.int16)), f"{what}: output {i}"


SIZES = [(E4, 16, 4, 200), (I8, 32, 70, 1500), (E4, 64, 3, 9000)]


@pytest.mark.parametrize("cache,hq,batch,longest", SIZES)
def test_captured_steps(cache, hq, batch, longest):
    run, renew = _step(cache, hq, batch, longest)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for seed in range(5):
        renew(seed)
        want = [t.clone() for t in run()]
        graph.replay()
        torch.cuda.synchronize()
        _same(held, want, f"replay {seed}")
        graph.replay()
        graph.replay()
        run()
        torch.cuda.synchronize()
        _same(held, want, f"replay {seed}, again")


def test_two_captured_steps_at_once():
    made = []
    for cache, hq, batch, longest in SIZES[1:]:
        run, renew = _step(cache, hq, batch, longest)
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = run()
        made.append((run, renew, graph, held))
    streams = [torch.cuda.Stream() for _ in made]
    for seed in range(4):
        want = []
        for run, renew, _, _ in made:
            renew(seed)
            want.append([t.clone() for t in run()])
        torch.cuda.synchronize()
        for _ in range(3):
            for (_, _, graph, _), st in zip(made, streams):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, held), w in zip(made, want):
            _same(held, w, f"seed {seed}")


def test_two_threads_on_their_own_streams():
    steps = [_step(*s) for s in SIZES[:2]]
    want = [[t.clone() for t in run()] for run, _ in steps]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i] = steps[i][0]()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors, errors
    for i in range(2):
        _same(got[i], want[i], f"thread {i}")


@pytest.mark.parametrize("cache,hq,batch,longest", SIZES)
def test_repeated_calls_give_the_same_bits(cache, hq, batch, longest):
    run, _ = _step(cache, hq, batch, longest)
    want = [t.clone() for t in run()]
    for i in range(4):
        _same(run(), want, f"call {i}")


@pytest.mark.parametrize("hq,hkv,d", [(2, 1, 64), (4, 2, 128)])
def test_batches_past_one_launch(hq, hkv, d):
    """4500 sequences: most without a token, some over a table of several splits."""
    batch, page, mb = 4500, 16, 40
    g = torch.Generator().manual_seed(1)
    lens = torch.where(torch.rand(batch, generator=g) < 0.9, 0, torch.randint(1, 640, (batch,), generator=g))
    kc, vc = (torch.randn(64, hkv, page, d, generator=g).to(BF) for _ in range(2))
    bt = torch.randint(0, 64, (batch, mb), generator=g).to(torch.int32)
    q = torch.randn(batch, hq, d, generator=g).to(BF)
    dev = [t.to(DEV) for t in (q, kc, vc, bt, lens.to(torch.int32))]
    from tests.rows_reference import quantize

    (k8, ks), (v8, vs) = quantize(kc, E4), quantize(vc, E4)
    outs = {
        (7, 3, False): paged_attention_window(*dev[:4], page, dev[4], 7, 3),
        (1000, 0, False): paged_attention_window(*dev[:4], page, dev[4], 1000),
        (0, 0, True): paged_attention_quantized(dev[0], *(t.to(DEV) for t in (k8, v8, ks, vs)), dev[3], page, dev[4]),
    }
    some = [s for s in range(batch) if lens[s] > 0 and s % 8 == 0][:50] + [s for s in range(4090, 4500) if lens[s] > 0]
    for (window, sinks, q8), out in outs.items():
        assert not out[dev[4] == 0].any()
        k64, v64 = (k8.double() * ks[..., None].double(), v8.double() * vs[..., None].double()) if q8 else (kc, vc)
        ref, tol = zip(*(attend(q[s], rows(k64, bt[s], see), rows(v64, bt[s], see), d**-0.5, half_step(BF), half_step(BF))
                         for s in some for see in [visible(int(lens[s]), window, sinks)]))
        check(out[torch.tensor(some, device=DEV)], torch.stack(ref), torch.stack(tol), f"window {window}, {sinks}, 8 bits {q8}")


def test_nothing_there():
    """No sequence, no page in the pool, no column in the table, no node."""
    for pages, mb, batch in ((0, 2, 3), (2, 0, 3), (2, 2, 0)):
        kc, vc = (torch.randn(pages, 2, 16, 128, device=DEV).to(BF) for _ in range(2))
        c8 = _cache8(pages, 2, 16, 128, E4)
        bt = torch.zeros(batch, mb, dtype=torch.int32, device=DEV)
        lens = torch.full((batch,), 20, dtype=torch.int32, device=DEV)
        q = torch.randn(batch, 4, 128, device=DEV).to(BF)
        cu = torch.arange(batch + 1, dtype=torch.int32, device=DEV)
        outs = [paged_attention_window(q, kc, vc, bt, 16, lens, 5), paged_attention_quantized(q, *c8, bt, 16, lens),
                paged_attention_tree(q, kc, vc, bt, 16, lens, cu, torch.ones(batch, dtype=torch.int64, device=DEV))]
        store_kv_cache_quantized(q[:, :2].transpose(0, 1), q[:, :2].transpose(0, 1), *c8, bt, cu)
        outs += load_kv_cache_quantized(*c8, bt, cu, batch, dtype=BF) if not (pages and mb) else ()
        torch.cuda.synchronize()
        for o in outs:
            assert o.shape[0] == batch and not o.any()
    kc = torch.randn(2, 2, 16, 128, device=DEV).to(BF)
    bt = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    none = torch.zeros(0, 4, 128, dtype=BF, device=DEV)
    out = paged_attention_tree(none, kc, kc, bt, 16, _i32([3, 4]), _i32([0, 0, 0]), torch.zeros(0, 1, dtype=torch.int64, device=DEV))
    assert out.shape == none.shape
    out = flash_attn_varlen_window(none, kc[:0, :, 0], kc[:0, :, 0], _i32([0, 0]), _i32([0, 0]), 0, 0, 4)
    assert out.shape == none.shape
    # queries without a key
    q = torch.randn(5, 4, 128, device=DEV).to(BF)
    assert not flash_attn_varlen_window(q, q[:0, :2], q[:0, :2], _i32([0, 5]), _i32([0, 0]), 5, 0, 4, 2).any()


FORMS = [  # (heads, kv heads, head_dim, page, tokens of a sequence, sequences)
    (32, 8, 128, 16, 500, 2),     # a workgroup a unit, trees of 32 rows and more
    (32, 8, 128, 16, 20000, 9),   # the stream
    (16, 8, 64, 64, 700, 3),
    (6, 2, 80, 12, 100, 2),       # neither
]


@pytest.mark.parametrize("hq,hkv,d,page,longest,batch", FORMS)
def test_pools_past_4_gb(hq, hkv, d, page, longest, batch):
    """The same pages at the far end of a pool of more than 4 GB (2^32 bytes in 8 bits) and in one of their own."""
    mb = -(-longest // page)
    used = batch * mb
    far = (1 << 32) // (hkv * page * d) + 7  # pages before the used ones: 4 GB in 8 bits, 8 GB in 16
    g = torch.Generator(device=DEV).manual_seed(page)
    perm = torch.randperm(used, generator=g, device=DEV).to(torch.int32).view(batch, mb)
    lens = torch.randint(longest // 2, longest - 5, (batch,), generator=g, device=DEV, dtype=torch.int32)
    near = [torch.randn(used, hkv, page, d, generator=g, device=DEV).to(BF) for _ in range(2)]
    wide = []
    for c in near:
        w = torch.empty(far + used, hkv, page, d, dtype=BF, device=DEV)
        w[far:] = c
        wide.append(w)
    q = torch.randn(batch, hq, d, generator=g, device=DEV).to(BF)
    a = paged_attention_window(q, *near, perm, page, lens, longest, 0)
    b = paged_attention_window(q, *wide, perm + far, page, lens, longest, 0)
    _same([b], [a], "window")
    for m in (3, 12, 33):
        qt = torch.randn(batch * m, hq, d, generator=g, device=DEV).to(BF)
        mask = torch.randint(1, 1 << m, (batch * m,), generator=g, device=DEV)
        cu = torch.arange(0, batch * m + 1, m, dtype=torch.int32, device=DEV)
        a = paged_attention_tree(qt, *near, perm, page, lens - 40, cu, mask, max_nodes=m)
        b = paged_attention_tree(qt, *wide, perm + far, page, lens - 40, cu, mask, max_nodes=m)
        _same([b], [a], f"tree of {m}")
    del wide
    n8, w8 = _cache8(used, hkv, page, d, E4), None
    kc, vc = (torch.empty(far + used, hkv, page, d, dtype=torch.uint8, device=DEV).view(E4) for _ in range(2))
    w8 = (kc, vc, *(torch.empty(far + used, hkv, page, device=DEV) for _ in range(2)))
    cu = torch.arange(0, batch * longest + 1, longest, dtype=torch.int32, device=DEV)
    x = [torch.randn(hkv, batch * longest, d, generator=g, device=DEV).to(BF) for _ in range(2)]
    store_kv_cache_quantized(*x, *n8, perm, cu)
    store_kv_cache_quantized(*x, *w8, perm + far, cu)
    a = (paged_attention_quantized(q, *n8, perm, page, lens), *load_kv_cache_quantized(*n8, perm, cu, batch * longest, dtype=BF))
    b = (paged_attention_quantized(q, *w8, perm + far, page, lens), *load_kv_cache_quantized(*w8, perm + far, cu, batch * longest, dtype=BF))
    _same(b, a, "8 bits")


@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 128), (4, 2, 128), (8, 2, 128), (16, 2, 128), (16, 1, 128), (8, 2, 64), (4, 2, 80)])
def test_prefill_tokens_past_4_gb(hq, hkv, d):
    """Rows 2 MiB apart: the last sequences' lie past 4 GB."""
    lens, step = [1500, 700, 333], 1 << 20
    n = sum(lens)
    g = torch.Generator(device=DEV).manual_seed(d)
    near = [torch.randn(n, h, d, generator=g, device=DEV).to(BF) for h in (hq, hkv, hkv)]
    wide = []
    for x in near:
        w = torch.empty(n * step, dtype=BF, device=DEV).as_strided(x.shape, (step, d, 1))
        w.copy_(x)
        wide.append(w)
    out = torch.empty(n * step, dtype=BF, device=DEV).as_strided(near[0].shape, (step, d, 1))
    cu = _i32([0, 1500, 2200, 2533])
    a = flash_attn_varlen_window(*near, cu, cu, 1500, 1500, 300, 3)
    b = flash_attn_varlen_window(*wide, cu, cu, 1500, 1500, 300, 3, out=out)
    _same([b], [a], "prefill")
