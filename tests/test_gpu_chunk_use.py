"""Steps as a server runs them: tables off a free list, the new tokens' norm, rotation and
store, attention of the chunk over the cache and the tokens' log probabilities, in one
run and step after step; the patched model's chunk steps against the stock model;
captured steps replayed with new inputs, two of them at once; two threads on streams of
their own; repeated calls; pools, contexts and logits past 4 GB."""

import copy
import threading

import pytest
import torch

from tests.chunk_reference import inputs, reference
from tests.helpers import assert_close
from tests.qwen3_tiny import (allocate_block_tables, original_last_logits, patched_decode_logits,
                              patched_prefill_logits, prompts_last_index, tiny_models)
from tests.rows_reference import check
from tinyserver_amd.inference_context import InferenceContext, inference_context
from tinyserver_amd.kernels import (paged_attention_chunk, qk_norm_rope_store, step_tables, store_kv_cache_batched,
                                    token_logprobs)

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---- The patched model.

def _chunk_logits(model, pieces, contexts, tables):
    """Last-token logits of each sequence's piece behind its context."""
    ids = [t for p in pieces for t in p]
    pos = [c + i for p, c in zip(pieces, contexts) for i in range(len(p))]
    ctx = InferenceContext("chunk", [{"num_tokens": len(p), "context_len": c, "block_table": bt}
                                     for p, c, bt in zip(pieces, contexts, tables)])
    with torch.no_grad(), inference_context(ctx):
        out = model(input_ids=torch.tensor([ids], device=DEV), position_ids=torch.tensor([pos], device=DEV),
                    use_cache=False)
    return out.logits[0, torch.tensor(prompts_last_index(pieces), device=DEV)]


PROMPTS = [[(7 * i + 3) % 384 for i in range(n)] for n in (5, 40, 33, 1)]
CUTS = [[3, 5], [1, 40], [16, 33], [0, 1]]  # tokens there after each step; a prompt that comes later has none yet


@pytest.mark.parametrize("page", [4, 16])
def test_prompts_in_pieces_match_the_stock_model(page):
    tables = allocate_block_tables([len(p) + 3 for p in PROMPTS], page)
    base, patched = tiny_models(F32, DEV, page, sum(len(t) for t in tables) + 2)
    there = [0] * len(PROMPTS)
    for step in range(2):
        live = [i for i in range(len(PROMPTS)) if CUTS[i][step] > there[i]]
        logits = _chunk_logits(patched, [PROMPTS[i][there[i] : CUTS[i][step]] for i in live], [there[i] for i in live],
                               [tables[i] for i in live])
        for row, i in zip(logits, live):
            there[i] = CUTS[i][step]
            assert_close(row, original_last_logits(base, PROMPTS[i][: there[i]], DEV), max_abs=1e-4, mean_abs=1e-5,
                         what=f"step {step} sequence {i}")
    # two sequences decode while the others bring two tokens more; then a plain decode step of all
    seqs = [p + [11 + i] * (1 + i % 2) for i, p in enumerate(PROMPTS)]
    logits = _chunk_logits(patched, [s[n:] for s, n in zip(seqs, there)], there, tables)
    for i, s in enumerate(seqs):
        assert_close(logits[i], original_last_logits(base, s, DEV), max_abs=1e-3, mean_abs=1e-4, what=f"mixed {i}")
    logits = patched_decode_logits(patched, [5] * len(seqs), [len(s) for s in seqs], tables, DEV)
    for i, s in enumerate(seqs):
        assert_close(logits[i], original_last_logits(base, s + [5], DEV), max_abs=1e-3, mean_abs=1e-4, what=f"decode {i}")


def test_pieces_are_as_accurate_as_whole_prompts():
    """In bf16, against float32 with the same weights: as near as the patched model's whole prefill, whose roundings
    are the same ones, is (its error's mean half as much again, as for the prefill beside the stock model)."""
    page = 16
    prompts = PROMPTS[:3]
    tables = allocate_block_tables([len(p) for p in prompts], page)
    base, patched = tiny_models(BF, DEV, page, sum(len(t) for t in tables) + 2)
    exact = copy.deepcopy(base).float()
    whole = patched_prefill_logits(patched, prompts, tables, DEV)
    for half in (1, 4):
        _chunk_logits(patched, [p[:half] for p in prompts], [0] * 3, tables)
        pieces = _chunk_logits(patched, [p[half:] for p in prompts], [half] * 3, tables)
        for i, p in enumerate(prompts):
            ref = original_last_logits(exact, p, DEV)
            a, b = ((x[i].float() - ref).abs() for x in (pieces, whole))
            print(f"cut {half} sequence {i}: pieces {a.mean():.3e} {a.max():.3e}, whole {b.mean():.3e} {b.max():.3e}", flush=True)
            assert a.mean() <= 1.5 * b.mean() + 1e-4 and a.max() <= 2.0 * b.max() + 1e-3


# ---- Steps on the kernels.

class Server:
    """Requests whose tables and free list are on the GPU; run() is one step on inputs that a caller overwrites."""

    def __init__(self, dtype, hq, hkv, d, page, seqs, longest, most, vocab=1000, top=5, pages=None):
        g = torch.Generator(device=DEV).manual_seed(seqs + longest)
        self.g, self.page, self.most, self.longest, self.top = g, page, most, longest, top
        width = -(-(longest + 8 * most) // page)
        pages = pages or seqs * width
        self.kc, self.vc, self.kb, self.vb = (torch.zeros(pages, hkv, page, d, dtype=dtype, device=DEV) for _ in range(4))
        self.tables = torch.full((seqs + 3, width), -1, dtype=torch.int32, device=DEV)
        self.rows = torch.randperm(seqs + 3, generator=g, device=DEV)[:seqs].to(torch.int32)
        self.free = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        self.num_free = _ints([pages])
        self.ctx, self.new = _ints([0] * seqs), _ints([0] * seqs)
        self.tokens = seqs * most  # rows of a step, padded

        def make(*shape):
            return torch.randn(*shape, generator=g, device=DEV).to(dtype)

        self.q, self.k, self.v = make(self.tokens, hq, d), make(self.tokens, hkv, d), make(self.tokens, hkv, d)
        self.wq, self.wk = (torch.rand(d, generator=g, device=DEV).to(dtype) + 0.5 for _ in range(2))
        self.head = make(hq * d, vocab)
        self.next = torch.randint(vocab, (self.tokens,), generator=g, device=DEV)
        self.freq = 10000.0 ** (-torch.arange(0, d, 2, device=DEV) / d)

    def renew(self, seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        for x in (self.q, self.k, self.v):
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
        self.new.copy_(torch.randint(0, self.most + 1, self.new.shape, generator=g, device=DEV))
        self.next.copy_(torch.randint(self.head.shape[1], self.next.shape, generator=g, device=DEV))

    def run(self):
        st = step_tables(self.tables, self.ctx, self.new, self.page, self.tokens, rows=self.rows, free_blocks=self.free,
                         num_free=self.num_free)
        ang = st.positions[:, None] * self.freq
        cos, sin = (torch.cat([f(ang)] * 2, -1).to(self.q.dtype) for f in (torch.cos, torch.sin))
        q, k = qk_norm_rope_store(self.q, self.k, self.v, self.wq, self.wk, cos, sin, 1e-6, self.kc, self.vc,
                                  st.block_tables, st.cu_seqlens, st.positions)
        # the same rows by the tokens' pages and slots
        store_kv_cache_batched(k.transpose(0, 1), self.v.transpose(0, 1), self.kb, self.vb, st.block_mapping, st.slot_mapping)
        out = torch.zeros_like(q)
        paged_attention_chunk(q, self.kc, self.vc, st.block_tables, self.page, self.ctx, st.cu_seqlens,
                              max_seqlen=self.most, out=out)
        logits = out.flatten(1) @ self.head
        return (*st, q, k, out, logits, *token_logprobs(logits, self.next, self.top))


def _logprobs_near(got, logits, tokens, top):
    """As in the log probabilities' own tests: sums of V = 1,000 terms and a logarithm."""
    logp, entropy, top_logp, top_tok = (x.cpu() for x in got)
    x = logits.double().cpu()
    m = x.amax(-1, keepdim=True)
    ref = torch.log_softmax(x, -1)
    size = 2.0**-21 + (x.shape[1] / 64 + 64) * 2.0**-24 + 2.0**-22 * (x - m).exp().sum(-1).log().abs()
    own = ref.gather(1, tokens.cpu()[:, None])[:, 0]
    assert bool(((logp - own).abs() <= size + 2.0**-22 * own.abs()).all())
    h = -(ref.exp() * ref).sum(-1)
    assert bool(((entropy - h).abs() <= 2 * size + 2.0**-20 * h.abs()).all())
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(top_tok, order)
    ref = ref.gather(1, order)
    assert bool(((top_logp - ref).abs() <= size[:, None] + 2.0**-22 * ref.abs()).all())


@pytest.mark.parametrize("dtype,hq,hkv,d,page", [
    (BF, 16, 8, 128, 16), (F16, 32, 4, 64, 32), (F32, 8, 4, 128, 16), (BF, 4, 2, 256, 16), (F32, 4, 1, 64, 5)])
def test_steps_of_a_server(dtype, hq, hkv, d, page):
    s = Server(dtype, hq, hkv, d, page, seqs=7, longest=120, most=40)
    left = s.free.numel()
    for step in range(3):
        s.renew(step)
        if step == 1:
            s.new.copy_(_ints([1, 1, 0, 1, 40, 1, 17]))  # decodes beside two pieces
        bt, cu, lens, pos, blk, slot, free_left, q, k, out, logits, *lp = s.run()
        ctx, new = s.ctx.tolist(), s.new.tolist()
        n = sum(new)
        assert lens.tolist() == [a + b for a, b in zip(ctx, new)] and cu.tolist()[-1] == n
        assert pos.tolist()[:n] == [c + i for c, m in zip(ctx, new) for i in range(m)]
        left -= sum(-(-(c + m) // page) - -(-c // page) for c, m in zip(ctx, new))
        assert free_left.tolist() == [left]
        # every page is one request's, and both stores left the same
        used = [p for row, m in zip(bt.tolist(), lens.tolist()) for p in row[: -(-m // page)]]
        assert len(set(used)) == len(used) and all(0 <= p < s.kc.shape[0] for p in used)
        assert torch.equal(s.kc, s.kb) and torch.equal(s.vc, s.vb)
        assert torch.equal(s.kc[blk[:n].long(), :, slot[:n].long()], k[:n])
        assert torch.equal(s.vc[blk[:n].long(), :, slot[:n].long()], s.v[:n])
        ref, tol = reference(q[:n].cpu(), s.kc.cpu(), s.vc.cpu(), bt.cpu(), ctx, new, d**-0.5)
        check(out[:n], ref, tol, f"step {step}")
        assert not bool(out[n:].any())  # the padded rows are left as they were
        _logprobs_near([x[:n] for x in lp], logits[:n], s.next[:n], s.top)
        s.ctx.copy_(lens)
        s.num_free.copy_(free_left)


def test_whole_prompts_and_their_pieces_agree():
    """A prompt at once and in three pieces: the pieces' rows see the same keys, in blocks that start elsewhere; both
    are within the reference's tolerance."""
    ctx, new, hq, hkv, d, page = [0, 0], [301, 64], 16, 4, 128, 16
    q, kc, vc, bt = inputs(ctx, new, hq, hkv, d, page, BF)
    ref, tol = reference(q, kc, vc, bt, ctx, new, d**-0.5)
    q, kc, vc, bt = (x.to(DEV) for x in (q, kc, vc, bt))
    whole = paged_attention_chunk(q, kc, vc, bt, page, _ints(ctx), _ints([0, 301, 365]), max_seqlen=301)
    check(whole, ref, tol, "whole")
    got = torch.empty_like(whole)
    done = [0, 0]
    for a, b in ((5, 64), (17, 0), (279, 0)):
        rows = torch.cat([torch.arange(done[0], done[0] + a), 301 + torch.arange(done[1], done[1] + b)]).to(DEV)
        got[rows] = paged_attention_chunk(q[rows], kc, vc, bt, page, _ints(done), _ints([0, a, a + b]))
        done = [done[0] + a, done[1] + b]
    check(got, ref, tol, "pieces")


SIZES = [dict(dtype=BF, hq=16, hkv=8, d=128, page=16, seqs=5, longest=300, most=12),
         dict(dtype=F16, hq=32, hkv=4, d=128, page=16, seqs=9, longest=2500, most=130),
         dict(dtype=F32, hq=8, hkv=4, d=64, page=16, seqs=12, longest=700, most=33)]


def _server(size):
    """One with full contexts: their pages given, their rows normal."""
    s = Server(**size)
    s.ctx.copy_(torch.randint(0, s.longest, s.ctx.shape, generator=s.g, device=DEV))
    st = step_tables(s.tables, s.ctx * 0, s.ctx, s.page, 0, rows=s.rows, free_blocks=s.free, num_free=s.num_free)
    s.num_free.copy_(st.free_left)
    for x in (s.kc, s.vc):
        x.copy_(torch.randn(x.shape, generator=s.g, device=DEV))
    s.kb.copy_(s.kc)
    s.vb.copy_(s.vc)
    s.renew(1000)
    return s


def _bits(t):
    t = t.cpu()
    return t if t.dtype in (torch.int32, torch.int64) else t.view(torch.int16 if t.element_size() == 2 else torch.int32)


def _same(got, want, what):
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(_bits(a), _bits(b)), f"{what}: output {i}"


def _capture(s):
    s.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = s.run()
    return graph, held


@pytest.mark.parametrize("size", SIZES)
def test_captured_steps(size):
    s = _server(size)
    graph, held = _capture(s)
    for seed in range(5):
        s.renew(seed)
        if seed == 3:
            s.new.zero_()  # (nothing new: every row is padding)
        want = [t.clone() for t in s.run()]
        graph.replay()
        torch.cuda.synchronize()
        _same(held, want, f"replay {seed}")
        graph.replay()
        graph.replay()
        s.run()
        torch.cuda.synchronize()
        _same(held, want, f"replay {seed}, again")


def test_two_captured_steps_at_once():
    made = [(s, *_capture(s)) for s in (_server(x) for x in SIZES[1:])]
    streams = [torch.cuda.Stream() for _ in made]
    for seed in range(4):
        want = []
        for s, _, _ in made:
            s.renew(seed)
            want.append([t.clone() for t in s.run()])
        torch.cuda.synchronize()
        for _ in range(3):
            for (_, graph, _), st in zip(made, streams):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, _, held), w in zip(made, want):
            _same(held, w, f"seed {seed}")


def test_two_threads_on_their_own_streams():
    servers = [_server(x) for x in SIZES[:2]]
    want = [[t.clone() for t in s.run()] for s in servers]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i] = servers[i].run()
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


@pytest.mark.parametrize("size", SIZES)
def test_repeated_calls_give_the_same_bits(size):
    s = _server(size)
    want = [t.clone() for t in s.run()]
    for i in range(4):
        _same(s.run(), want, f"call {i}")


@pytest.mark.parametrize("dtype,hq,hkv,d,page", [(BF, 16, 8, 128, 16), (F32, 16, 8, 128, 16), (F16, 8, 8, 64, 24)])
def test_pools_past_4_gb(dtype, hq, hkv, d, page):
    """The same call on a small pool and on one whose used pages lie behind 4 GB: the same bits."""
    ctx, new = [500, 0, 77], [40, 9, 1]
    q, kc, vc, bt = inputs(ctx, new, hq, hkv, d, page, dtype)
    cu, lens = _ints([0, 40, 49, 50]), _ints(ctx)
    args = (page, lens, cu)
    small = paged_attention_chunk(q.to(DEV), kc.to(DEV), vc.to(DEV), bt.to(DEV), *args)
    used = kc.shape[0]
    first = 4_400_000_000 // (hkv * page * d * kc.element_size())
    big = [torch.empty(first + used, hkv, page, d, dtype=dtype, device=DEV) for _ in range(2)]
    for b, c in zip(big, (kc, vc)):
        b[first:] = c.to(DEV)
    out = paged_attention_chunk(q.to(DEV), *big, bt.to(DEV) + first, *args)
    assert torch.equal(_bits(out), _bits(small))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_long_context(dtype):
    ctx, new, hq, hkv, d, page = [200_000], [5], 8, 1, 128, 16
    q, kc, vc, bt = inputs(ctx, new, hq, hkv, d, page, dtype)
    ref, tol = reference(q, kc, vc, bt, ctx, new, d**-0.5)
    out = paged_attention_chunk(q.to(DEV), kc.to(DEV), vc.to(DEV), bt.to(DEV), page, _ints(ctx), _ints([0, 5]))
    check(out, ref, tol, f"{dtype}")


def test_logits_past_4_gb():
    """Rows behind 4 GB give what they give by themselves (600 rows: neither call cuts a row)."""
    n, v = 14_400, 151_936
    x = torch.zeros(n, v, dtype=BF, device=DEV)
    x[-600:] = torch.randn(600, v, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    tokens = torch.arange(n, device=DEV)
    got, want = token_logprobs(x, tokens, 7), token_logprobs(x[-600:].clone(), tokens[-600:], 7)
    _same([t[-600:] for t in got], want, "last rows")
    assert torch.equal(got.top_tokens[:-600].cpu(), torch.arange(7).expand(n - 600, 7))
