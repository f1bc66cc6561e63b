"""A step of chunked prefill, from request lengths to scored tokens, as cases that can be timed and checked.

Three operators beside the paged store, the paged decode, the varlen prefill and
the sampler of ``tinyserver_amd.kernels``:

* the step's block tables, positions and slots, built on the GPU from the
  requests' lengths, new pages taken off a free list;
* attention of a chunk of new tokens over a paged cache that holds them and the
  tokens before them;
* log probabilities of given tokens, with the entropy of their distribution and
  the most likely alternatives.

``listed`` gives the cases, ``draw`` more of the same ranges; ``prepare`` makes
what a program holds before the call; ``run`` makes the call (``own``) or
computes the same with elementary torch operations in 32 bits; ``exact``
computes it in 64 bits.

Shapes are the package's: 8 kv heads, 2, 4 or 8 query heads per kv head,
head_dim 128 (now and then 64), pages of 16 tokens or the server's 256, a
vocabulary of 151,936.
"""

import math
import random

import torch

own = False

HKV = 8
VOCAB = 151936
DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# The costliest listed work, which drawn cases stay under.
MAX_PAIRS = 64 * 2048 * 32768  # (q-head, query, key) pairs of one call in 16 bits
MAX_PAIRS_F32 = 16 * 4 * 128 * 1024
MAX_CACHE_TOKENS = 1 << 19
MAX_LOGITS = 4096 * VOCAB
MAX_LOGITS_F32 = 512 * VOCAB
MAX_STEP_TOKENS = 65536


def listed():
    return [
        # A few short chats of a small model, each with a few more tokens: latency.
        dict(name="chunk_0.6b_bs4", kind="chunk", dtype="f16", seqs=4, singles=0, heads=16, lo=16, hi=512, new_lo=1,
             new_hi=8, page=256, dim=128, lens=1),
        # One step of continuous batching: 28 sequences decode a token each,
        # four bring a piece of their prompts.
        dict(name="chunk_8b_step_bs32", kind="chunk", dtype="bf16", seqs=32, singles=28, heads=32, lo=512, hi=4096,
             new_lo=128, new_hi=512, page=16, dim=128, lens=2),
        # Prompts whose first part is in the cache already.
        dict(name="chunk_8b_cached_16seq", kind="chunk", dtype="bf16", seqs=16, singles=0, heads=32, lo=512, hi=4096,
             new_lo=64, new_hi=512, page=16, dim=128, lens=3),
        # The last chunk of a long document on the largest model.
        dict(name="chunk_32b_2048_32k", kind="chunk", dtype="bf16", seqs=1, singles=0, heads=64, lo=30720, hi=30720,
             new_lo=2048, new_hi=2048, page=16, dim=128, lens=4),
        # A follow-up question of a few tokens over a long document.
        dict(name="chunk_32b_few_32k", kind="chunk", dtype="f16", seqs=2, singles=0, heads=64, lo=24000, hi=32768,
             new_lo=12, new_hi=40, page=256, dim=128, lens=5),
        # Chunks of a model kept in float32.
        dict(name="chunk_0.6b_f32", kind="chunk", dtype="f32", seqs=4, singles=0, heads=16, lo=100, hi=1024, new_lo=16,
             new_hi=128, page=16, dim=128, lens=6),
        # A default server's decode step: 8 sequences, one token each.
        dict(name="step_bs8", kind="step", seqs=8, rows=64, lo=16, hi=4096, new_lo=1, new_hi=1, page=256, pad=0, lens=7),
        # A large step: 512 requests with 1 to 128 new tokens, the token count
        # rounded up as a captured graph has it.
        dict(name="step_bs512", kind="step", seqs=512, rows=1024, lo=0, hi=8192, new_lo=1, new_hi=128, page=16,
             pad=1024, lens=8),
        # The sampled tokens of a few chats with five alternatives: latency.
        dict(name="logprobs_bs4", kind="logprobs", dtype="f16", rows=4, vocab=VOCAB, top=5, masked=0.0),
        # A busy server's step; a quarter of its rows follow a grammar.
        dict(name="logprobs_bs64", kind="logprobs", dtype="bf16", rows=64, vocab=VOCAB, top=20, masked=0.25),
        # A packed prompt's tokens scored.
        dict(name="logprobs_prompt_4096", kind="logprobs", dtype="bf16", rows=4096, vocab=VOCAB, top=5, masked=0.0),
        # The same of logits in float32.
        dict(name="logprobs_prompt_512_f32", kind="logprobs", dtype="f32", rows=512, vocab=VOCAB, top=20, masked=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["chunk", "chunk", "chunk", "chunk", "step", "logprobs", "logprobs"])
    if kind == "logprobs":
        c = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), vocab=_log_int(rng, 1000, 160000))
        most = (MAX_LOGITS_F32 if c["dtype"] == "f32" else MAX_LOGITS) // c["vocab"]
        c["rows"] = _log_int(rng, 1, min(4096, most))
        c["top"], c["masked"] = rng.choice([0, 1, 5, 20, 20, 50]), rng.choice([0.0, 0.0, 0.3])
        return c
    c = dict(kind=kind, lens=rng.randrange(1, 1 << 20), page=rng.choice([16, 16, 256]))
    if kind == "step":
        c["seqs"] = _log_int(rng, 1, 1024)
        c["rows"] = c["seqs"] + rng.choice([0, 3, 200])
        c["new_hi"] = min(_log_int(rng, 1, 4096), MAX_STEP_TOKENS // c["seqs"])
        c["new_lo"] = rng.choice([1, c["new_hi"], 0]) if c["new_hi"] > 1 else 1
        c["hi"] = _log_int(rng, 16, 8192)
        c["lo"], c["pad"] = rng.choice([0, c["hi"] // 8]), rng.choice([0, 256])
        return c
    c["dtype"], c["dim"] = rng.choice(["bf16", "bf16", "f16", "f16", "f32"]), rng.choice([128, 128, 128, 64])
    c["heads"] = rng.choice([16, 32, 64])
    c["seqs"] = _log_int(rng, 1, 64)
    c["singles"] = rng.choice([0, 0, c["seqs"] // 2, c["seqs"]])
    c["hi"] = min(_log_int(rng, 16, 32768), MAX_CACHE_TOKENS // c["seqs"])
    c["new_hi"] = min(_log_int(rng, 1, 4096), MAX_STEP_TOKENS // c["seqs"])
    most = MAX_PAIRS_F32 if c["dtype"] == "f32" else MAX_PAIRS
    while c["heads"] * c["seqs"] * c["new_hi"] * (c["hi"] + c["new_hi"]) > most:
        k = "new_hi" if c["new_hi"] > max(1, c["hi"] // 8) else "hi"
        c[k] = max(1, c[k] * 3 // 4)
    c["lo"] = max(0, c["hi"] // rng.choice([1, 4, 16]) - 1)
    c["new_lo"] = max(1, c["new_hi"] // rng.choice([1, 4, 16]))
    return c


# ------------------------------------------------------------------ inputs --
def _counts(case, lo, hi, salt):
    """Numbers in [lo, hi], one per sequence: fixed by the case, the same for every seed."""
    r = random.Random(1000003 * case["lens"] + 17 * hi + case["seqs"] + salt)
    return [r.randint(lo, hi) for _ in range(case["seqs"])]


def _lengths(case):
    """Cached and new tokens of each sequence."""
    ctx, new = _counts(case, case["lo"], case["hi"], 0), _counts(case, case["new_lo"], case["new_hi"], 7919)
    for i in range(case.get("singles", 0)):  # sequences that decode, spread among the others
        new[i * case["seqs"] // case["singles"]] = 1
    return ctx, new


def _randn(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEVICE)


def _cu(lens):
    return _ints([0] + torch.tensor(lens).cumsum(0).tolist())


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind = case["kind"]
    s = {"kind": kind}
    if kind == "logprobs":
        n, v = case["rows"], case["vocab"]
        # Each row has a spread of its own, a few likely tokens and a long tail.
        s["logits"] = torch.empty(n, v, dtype=DTYPES[case["dtype"]], device=DEVICE)
        for i in range(0, n, 256):
            m = min(256, n - i)
            x = _randn(gen, m, v, dtype=torch.float32) * (1.5 + 1.5 * torch.rand(m, 1, generator=gen, device=DEVICE))
            likely = torch.randint(v, (m, 12), generator=gen, device=DEVICE)
            x.scatter_(1, likely, 8 + 4 * _randn(gen, m, 12, dtype=torch.float32))
            held = torch.rand(m, 1, generator=gen, device=DEVICE) < case["masked"]
            allowed = torch.rand(m, v, generator=gen, device=DEVICE) * v < 40  # (about 40 of a grammar's tokens)
            allowed.scatter_(1, likely[:, :2], True)
            s["logits"][i : i + m] = x.masked_fill_(held & ~allowed, float("-inf"))
            if i == 0:
                best = []
            best.append(torch.where(torch.rand(m, generator=gen, device=DEVICE) < 0.5, likely[:, 0],
                                    likely[:, 1]))
        s["tokens"], s["top"] = torch.cat(best), case["top"]
        return s
    ctx, new = _lengths(case)
    page = s["page"] = case["page"]
    s["context_lens"] = _ints(ctx)
    s["num_tokens"] = sum(new)
    if kind == "step":
        s["query_lens"] = _ints(new)
        s["rows"] = torch.randperm(case["rows"], generator=gen, device=DEVICE)[: len(ctx)].to(torch.int32)
        have = [-(-a // page) for a in ctx]
        need = [-(-(a + b) // page) for a, b in zip(ctx, new)]
        s["width"] = max(1, max(need))
        pages = sum(need) + 8
        perm = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
        s["tables"] = torch.zeros(case["rows"], s["width"] + 4, dtype=torch.int32, device=DEVICE)
        col = torch.arange(s["width"] + 4, device=DEVICE)
        start = _ints([0] + torch.tensor(have).cumsum(0).tolist())[:-1]
        used = col < _ints(have)[:, None]
        s["tables"][s["rows"].long()] = torch.where(used, perm[(start[:, None] + col).clamp(max=pages - 1)], 0)
        s["free_blocks"] = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
        s["free_blocks"][: pages - sum(have)] = perm[sum(have):]
        s["num_free"] = _ints([pages - sum(have)])
        if case["pad"]:
            s["num_tokens"] = -(-s["num_tokens"] // case["pad"]) * case["pad"]
        return s
    dt, d = DTYPES[case["dtype"]], case["dim"]
    need = [-(-(a + b) // page) for a, b in zip(ctx, new)]
    pages = math.ceil(sum(need) * 1.1)
    perm = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    start = torch.tensor([sum(need[:i]) for i in range(len(need))], device=DEVICE)
    col = torch.arange(max(need), device=DEVICE)
    used = col < torch.tensor(need, device=DEVICE)[:, None]
    s["tables"] = torch.where(used, perm[(start[:, None] + col).clamp(max=pages - 1)], 0).to(torch.int32).contiguous()
    # Keys have channels that stand out and heads of unlike magnitude, as trained models' do.
    k_size = torch.exp(0.5 * torch.randn(HKV, 1, d, generator=gen, device=DEVICE))
    v_size = torch.exp(0.7 * torch.randn(HKV, 1, 1, generator=gen, device=DEVICE))
    s["k_cache"], s["v_cache"] = (torch.empty(pages, HKV, page, d, dtype=dt, device=DEVICE) for _ in range(2))
    step = max(1, (1 << 27) // (HKV * page * d))  # pieces that bound the 32-bit copies
    for i in range(0, pages, step):
        n = min(step, pages - i)
        s["k_cache"][i : i + n] = _randn(gen, n, HKV, page, d, dtype=torch.float32).mul_(k_size)
        s["v_cache"][i : i + n] = _randn(gen, n, HKV, page, d, dtype=torch.float32).mul_(v_size)
    s["q"] = _randn(gen, sum(new), case["heads"], d, dtype=dt)
    s["cu"], s["ctx"], s["new"] = _cu(new), ctx, new  # (on the host too: the scheduler's)
    return s


# --------------------------------------------------------------- the calls --
def run(s):
    if own:
        return _run_own(s)
    return {"chunk": _chunk, "step": _step, "logprobs": _logprobs}[s["kind"]](s)


def _run_own(s):
    from tinyserver_amd import kernels

    if s["kind"] == "chunk":
        return kernels.paged_attention_chunk(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["page"],
                                             s["context_lens"], s["cu"], max_seqlen=max(s["new"]))
    if s["kind"] == "step":
        t = kernels.step_tables(s["tables"], s["context_lens"], s["query_lens"], s["page"], s["num_tokens"],
                                rows=s["rows"], width=s["width"], free_blocks=s["free_blocks"],
                                num_free=s["num_free"])
        return {"tables": s["tables"], **t._asdict()}
    return kernels.token_logprobs(s["logits"], s["tokens"], s["top"])._asdict()


def _chunk(s):
    """Sequence by sequence, in blocks of queries that bound the scores."""
    t, hq, d = s["q"].shape
    out, start = torch.empty_like(s["q"]), 0
    for i, (ctx, new) in enumerate(zip(s["ctx"], s["new"])):
        n = ctx + new
        used = s["tables"][i, : -(-n // s["page"])].long()
        k, v = (s[x][used].transpose(0, 1).reshape(HKV, -1, d)[:, :n].float() for x in ("k_cache", "v_cache"))
        kt = k.transpose(1, 2).contiguous()
        step = max(1, (1 << 28) // (hq * n))
        for a in range(0, new, step):
            b = min(new, a + step)
            q = s["q"][start + a : start + b].float().reshape(b - a, HKV, -1, d).permute(1, 2, 0, 3)
            sc = torch.matmul(q.reshape(HKV, -1, d), kt).div_(math.sqrt(d)).reshape(HKV, -1, b - a, n)
            later = torch.arange(n, device=DEVICE) > torch.arange(ctx + a, ctx + b, device=DEVICE)[:, None]
            sc.masked_fill_(later, float("-inf"))
            p = sc.sub_(sc.amax(-1, keepdim=True)).exp_()
            total = p.sum(-1, keepdim=True)
            o = torch.matmul(p.reshape(HKV, -1, n), v).reshape(HKV, -1, b - a, d) / total
            out[start + a : start + b] = o.permute(2, 0, 1, 3).reshape(b - a, hq, d).to(out.dtype)
        start += new
    return out


def _step(s):
    b, width, page, t = s["rows"].shape[0], s["width"], s["page"], s["num_tokens"]
    ctx, new, rows = s["context_lens"].long(), s["query_lens"].long(), s["rows"].long()
    cu = torch.zeros(b + 1, dtype=torch.int64, device=DEVICE)
    cu[1:] = new.cumsum(0)
    have = (ctx + page - 1) // page
    need = (ctx + new + page - 1) // page
    taken = (need - have).cumsum(0)
    col = torch.arange(s["tables"].shape[1], device=DEVICE)
    fresh = (col >= have[:, None]) & (col < need[:, None])
    at = s["num_free"].long() - 1 - ((taken - (need - have))[:, None] + col - have[:, None])
    pages = torch.where(at >= 0, s["free_blocks"][at.clamp(0, s["free_blocks"].shape[0] - 1)], -1)
    full = torch.where(fresh, pages, s["tables"][rows])
    s["tables"][rows] = full
    full = torch.where(col < need[:, None], full, 0)
    tok = torch.arange(t, device=DEVICE)
    seq = torch.searchsorted(cu[1:], tok, right=True)
    real = seq < b
    seq = seq.clamp(max=b - 1)
    pos = torch.where(real, ctx[seq] + tok - cu[seq], 0)
    return {"tables": s["tables"], "block_tables": full[:, :width].contiguous(), "cu_seqlens": cu.to(torch.int32),
            "seq_lens": (ctx + new).to(torch.int32), "positions": pos.to(torch.int32),
            "block_mapping": torch.where(real, full[seq, pos // page], -1),
            "slot_mapping": torch.where(real, pos % page, -1).to(torch.int32),
            "free_left": (s["num_free"] - taken[-1]).to(torch.int32)}


def _logprobs(s):
    n, v = s["logits"].shape
    logp, entropy, top_logp, top = [], [], [], []
    for i in range(0, n, 256):  # (rows that bound the 32-bit copies)
        x = s["logits"][i : i + 256].float()
        m = x.amax(-1, keepdim=True)
        y = x - m
        e = torch.exp(y)
        total = e.sum(-1, keepdim=True)
        lse = torch.log(total)
        logp.append((y.gather(1, s["tokens"][i : i + 256, None]) - lse)[:, 0])
        entropy.append((lse - torch.where(e > 0, e * y, 0.0).sum(-1, keepdim=True) / total)[:, 0])
        # By value, the lowest index first where values tie: one whole number a logit that orders so.
        bits = (x + 0.0).view(torch.int32)
        key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 20) - torch.arange(v, device=DEVICE)
        best = key.topk(s["top"], dim=-1).indices
        top.append(best)
        top_logp.append(y.gather(1, best) - lse)
    return {"logprobs": torch.cat(logp), "entropy": torch.cat(entropy), "top_logprobs": torch.cat(top_logp),
            "top_tokens": torch.cat(top)}


def work(case):
    if case["kind"] == "logprobs":
        n, v = case["rows"], case["vocab"]
        # A logit: less the maximum, exponential, its sum and the weighted one.
        return {"bytes": n * v * (4 if case["dtype"] == "f32" else 2) + n * (16 + 12 * case["top"]), "flops": 5 * n * v}
    ctx, new = _lengths(case)
    page, t = case["page"], sum(new)
    used = sum(-(-(a + b) // page) for a, b in zip(ctx, new))
    if case["kind"] == "step":
        # Lengths and rows, table entries or free pages in; the tables, and three numbers a token.
        return {"bytes": 4 * (3 * len(ctx) + used + len(ctx) * max(-(-(a + b) // page) for a, b in zip(ctx, new))
                              + 2 * len(ctx) + 1 + 3 * t), "flops": 4 * t}
    hq, d, eb = case["heads"], case["dim"], 4 if case["dtype"] == "f32" else 2
    pairs = sum(b * a + b * (b + 1) // 2 for a, b in zip(ctx, new))
    rows = sum(ctx) + t
    return {"bytes": eb * d * (2 * HKV * rows + 2 * hq * t) + 4 * (used + 2 * len(ctx)), "flops": 4 * d * hq * pairs}


# ------------------------------------------------------- the same in 64 bits --
def exact(case, seed):
    """From the definitions, in 64 bits: head by head, request by request, row by row."""
    s = prepare(case, seed)
    if case["kind"] == "step":
        return None  # whole numbers, nothing to round
    if case["kind"] == "logprobs":
        n, v = case["rows"], case["vocab"]
        out = {k: [] for k in ("logprobs", "entropy", "top_logprobs", "top_tokens")}
        for i in range(0, n, 64):
            x = s["logits"][i : i + 64].double()
            lp = torch.log_softmax(x, dim=-1)
            out["logprobs"].append(lp.gather(1, s["tokens"][i : i + 64, None]).squeeze(1))
            out["entropy"].append(torch.special.entr(torch.softmax(x, dim=-1)).sum(-1))
            # All that reach the last place's value, in order of index, then of value, then of row.
            k = case["top"]
            if not k:
                best = torch.zeros(x.shape[0], 0, dtype=torch.int64, device=DEVICE)
            else:
                row, idx = (x >= x.topk(k, dim=-1).values[:, -1:]).nonzero(as_tuple=True)
                order = torch.sort(x[row, idx], descending=True, stable=True).indices
                order = order[torch.sort(row[order], stable=True).indices]
                first = torch.searchsorted(row[order], torch.arange(x.shape[0], device=DEVICE))
                best = idx[order][first[:, None] + torch.arange(k, device=DEVICE)]
            out["top_tokens"].append(best)
            out["top_logprobs"].append(lp.gather(1, best))
        return {k: torch.cat(x) for k, x in out.items()}
    hq, d, page = case["heads"], case["dim"], case["page"]
    ctx, new = _lengths(case)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    start = 0
    for i, (c, m) in enumerate(zip(ctx, new)):
        pos = torch.arange(c + m, device=DEVICE)
        block, slot = s["tables"][i, pos // page].long(), pos % page
        for h in range(HKV):
            k, v = s["k_cache"][block, h, slot].double(), s["v_cache"][block, h, slot].double()
            for g in range(h * hq // HKV, (h + 1) * hq // HKV):
                sc = torch.mm(s["q"][start : start + m, g].double(), k.t().contiguous()) * d**-0.5
                sc.masked_fill_(pos[None, :] > pos[c:, None], float("-inf"))
                out[start : start + m, g] = torch.mm(torch.softmax(sc, dim=-1), v)
        start += m
    return out
