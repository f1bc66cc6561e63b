"""Attention over long and compressed contexts, as cases that can be timed and checked.

Three operators beside the paged decode, the varlen prefill and the paged store
of ``tinyserver_amd.kernels``:

* a paged K/V cache held in 8 bits (e4m3 or int8, one float32 scale per token
  and kv head): written, read back, and attended to by the decode step;
* attention with a sliding window and a few first tokens that stay visible, for
  decode over the paged cache and for varlen prefill;
* attention of a tree of drafted tokens over the paged cache.

``listed`` gives the cases, ``draw`` more of the same ranges; ``prepare`` makes
what a program holds before the call; ``run`` makes the call (``own``) or
computes the same with elementary torch operations in 32 bits; ``exact``
computes it in 64 bits.

Shapes are the package's: 8 kv heads, 2, 4 or 8 query heads per kv head,
head_dim 128 (now and then 64), pages of 16 tokens or the server's 256.
"""

import math
import random

import torch

own = False

HKV = 8
DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
CACHES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"e4m3": 448.0, "int8": 127.0}

# The costliest listed work, which drawn cases stay under.
MAX_CACHE_TOKENS = 32 * 32768  # cache tokens one decode batch attends to
MAX_WINDOW_PAIRS = 64 * 16384 * 4096  # (q-head, query, key) pairs of one windowed prefill
MAX_TREE_PAIRS = 64 * 8 * 64 * 8192  # the same of one verification step
MAX_STORE_TOKENS = 16 * 2048


def listed():
    return [
        # One decode step's new tokens of a default server (8 sequences) into
        # an int8 cache of 256-token pages. Launch latency is all of it.
        dict(name="store_int8_step_bs8", kind="store", cache="int8", dtype="f16", seqs=8, lo=300, hi=4096, step=True,
             page=256, dim=128, lens=1),
        # The keys and values of 16 packed prompts into an e4m3 cache.
        dict(name="store_e4m3_16seq", kind="store", cache="e4m3", dtype="bf16", seqs=16, lo=128, hi=2048, step=False,
             page=16, dim=128, lens=2),
        # Cached prefixes of 8 sequences read back as packed 16-bit rows, as a
        # chunked prefill needs them.
        dict(name="load_int8_8seq", kind="load", cache="int8", dtype="bf16", seqs=8, lo=512, hi=4096, page=16, dim=128,
             lens=3),
        # A few short chats, two query heads per kv head: latency.
        dict(name="decode_int8_0.6b_bs4", kind="decode8", cache="int8", dtype="f16", batch=4, heads=16, lo=16, hi=512,
             page=256, dim=128, window=0, sinks=0, lens=4),
        # A busy server's decode attention over an e4m3 cache.
        dict(name="decode_e4m3_8b_bs64", kind="decode8", cache="e4m3", dtype="bf16", batch=64, heads=32, lo=512,
             hi=4096, page=16, dim=128, window=0, sinks=0, lens=5),
        # Long contexts on the largest model, the largest cache read.
        dict(name="decode_e4m3_32b_32k", kind="decode8", cache="e4m3", dtype="bf16", batch=32, heads=64, lo=32768,
             hi=32768, page=16, dim=128, window=0, sinks=0, lens=6),
        # The same busy server, each token seeing the last 1024 and the first 4.
        dict(name="window_decode_8b_bs64", kind="window", dtype="bf16", batch=64, heads=32, lo=512, hi=8192, page=16,
             dim=128, window=1024, sinks=4, lens=7),
        # A few very long chats with a wide window on 256-token pages.
        dict(name="window_decode_32b_bs8_32k", kind="window", dtype="f16", batch=8, heads=64, lo=8000, hi=32768,
             page=256, dim=128, window=4096, sinks=64, lens=8),
        # Varlen prefill of 16 packed prompts with a window of 512.
        dict(name="window_prefill_8b_16seq", kind="prefill", dtype="bf16", seqs=16, heads=32, lo=128, hi=2048, dim=128,
             window=512, sinks=4, lens=9),
        # One long document on the largest model, window 4096.
        dict(name="window_prefill_32b_16k", kind="prefill", dtype="bf16", seqs=1, heads=64, lo=16384, hi=16384,
             dim=128, window=4096, sinks=16, lens=10),
        # Verifying small draft trees of a busy server's sequences.
        dict(name="tree_8b_bs64", kind="tree", dtype="bf16", batch=64, heads=32, lo=512, hi=4096, nodes_lo=4,
             nodes_hi=16, page=16, dim=128, lens=11),
        # Wide trees on the largest model: 64 nodes, 512 rows per kv head.
        dict(name="tree_32b_bs8_64", kind="tree", dtype="f16", batch=8, heads=64, lo=2000, hi=8192, nodes_lo=40,
             nodes_hi=64, page=16, dim=128, lens=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "load", "decode8", "decode8", "window", "window", "prefill", "prefill", "tree", "tree"])
    c = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16"]), dim=rng.choice([128, 128, 128, 64]),
             lens=rng.randrange(1, 1 << 20))
    if kind != "prefill":
        c["page"] = rng.choice([16, 16, 256])
    if kind in ("store", "load", "decode8"):
        c["cache"] = rng.choice(["e4m3", "int8"])
    if kind in ("store", "load"):
        c["seqs"] = _log_int(rng, 1, 32)
        c["hi"] = min(_log_int(rng, 8, 8192), MAX_STORE_TOKENS // c["seqs"])
        c["lo"] = max(1, c["hi"] // rng.choice([1, 4, 16]))
        if kind == "store":
            c["step"] = rng.random() < 0.4
        return c
    c["heads"] = rng.choice([16, 32, 64])
    if kind == "prefill":
        c["window"], c["sinks"] = _log_int(rng, 32, 8192), rng.choice([0, 1, 4, 16, 40, 64])
        c["seqs"] = _log_int(rng, 1, 32)
        c["hi"] = _log_int(rng, 16, 16384)
        while c["seqs"] > 1 and c["seqs"] * c["hi"] > 32768:
            c["seqs"] //= 2
        while c["heads"] * c["seqs"] * c["hi"] * (min(c["hi"], c["window"]) + c["sinks"]) > MAX_WINDOW_PAIRS:
            c["hi"] = c["hi"] * 3 // 4
        c["lo"] = max(1, c["hi"] // rng.choice([1, 4, 16]))
        return c
    c["batch"] = _log_int(rng, 1, 128)
    c["hi"] = min(_log_int(rng, 64, 32768), MAX_CACHE_TOKENS // 2 // c["batch"])
    if kind == "tree":
        c["nodes_hi"] = _log_int(rng, 1, 64)
        c["nodes_lo"] = max(1, c["nodes_hi"] // rng.choice([1, 2, 8]))
        c["hi"] = max(16, min(c["hi"], MAX_TREE_PAIRS // (c["heads"] * c["nodes_hi"] * c["batch"])))
    else:
        c["window"] = 0 if kind == "decode8" and rng.random() < 0.6 else _log_int(rng, 32, 8192)
        c["sinks"] = rng.choice([0, 1, 4, 16, 40, 64]) if c["window"] else 0
    c["lo"] = max(1, c["hi"] // rng.choice([1, 4, 16]))
    return c


# ------------------------------------------------------------------ inputs --
def _counts(case, lo, hi, salt):
    """Numbers in [lo, hi], one per sequence: fixed by the case, the same for every seed."""
    n = case["batch"] if "batch" in case else case["seqs"]
    r = random.Random(1000003 * case["lens"] + 17 * hi + n + salt)
    return [r.randint(lo, hi) for _ in range(n)]


def _lengths(case):
    return _counts(case, case["lo"], case["hi"], 0)


def _nodes(case):
    return _counts(case, case["nodes_lo"], case["nodes_hi"], 7919)


def _randn(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)


def _quantize(x, cache):
    """8-bit rows and their scales: scale = the row's largest magnitude over the type's, q = x / scale rounded
    once (both quotients as float32 rounds them, which the 64-bit ones, rounded, give)."""
    x = x.double()
    scale = (x.abs().amax(-1, keepdim=True) / LARGEST[cache]).float()
    q = torch.where(scale > 0, x / scale.double(), 0.0).float().clamp(-LARGEST[cache], LARGEST[cache])
    return (q.round() if cache == "int8" else q).to(CACHES[cache]), scale.squeeze(-1)


def _tables(gen, lens, page):
    """Shuffled pages of a pool with a tenth of it free, and the zero-padded block tables."""
    need = [-(-n // page) for n in lens]
    pages = math.ceil(sum(need) * 1.1)
    perm = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    starts = torch.tensor([sum(need[:i]) for i in range(len(need))], device=DEVICE)
    col = torch.arange(max(need), device=DEVICE)
    used = col[None, :] < torch.tensor(need, device=DEVICE)[:, None]
    idx = (starts[:, None] + col[None, :]).clamp(max=pages - 1)
    return torch.where(used, perm[idx], 0).to(torch.int32).contiguous(), pages


def _cu(lens):
    cu = torch.zeros(len(lens) + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor(lens), 0).to(torch.int32)
    return cu.to(DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, dt, d = case["kind"], DTYPES[case["dtype"]], case["dim"]
    s = {"kind": kind, "cache": case.get("cache"), "window": case.get("window"), "sinks": case.get("sinks")}
    lens = _lengths(case)
    # Keys have channels that stand out and heads of unlike magnitude, as trained models' do.
    k_size = torch.exp(0.5 * torch.randn(HKV, d, generator=gen, device=DEVICE))
    v_size = torch.exp(0.7 * torch.randn(HKV, 1, generator=gen, device=DEVICE))
    if kind == "prefill":
        t = sum(lens)
        s["cu"], s["max_len"] = _cu(lens), max(lens)
        s["q"] = _randn(gen, t, case["heads"], d, dtype=dt)
        s["k"] = (_randn(gen, t, HKV, d, dtype=torch.float32) * k_size).to(dt)
        s["v"] = (_randn(gen, t, HKV, d, dtype=torch.float32) * v_size).to(dt)
        return s
    page = s["page"] = case["page"]
    nodes = _nodes(case) if kind == "tree" else [0] * len(lens)
    s["tables"], pages = _tables(gen, [a + b for a, b in zip(lens, nodes)], page)
    # The pool, in pieces that bound the 32-bit copies.
    shape = (pages, HKV, page, d)
    step = max(1, (1 << 27) // (HKV * page * d))
    if kind in ("store", "load", "decode8"):
        s["k_cache"], s["v_cache"] = (torch.zeros(shape, dtype=CACHES[case["cache"]], device=DEVICE) for _ in range(2))
        s["k_scale"], s["v_scale"] = (torch.zeros(shape[:3], device=DEVICE) for _ in range(2))
    else:
        s["k_cache"], s["v_cache"] = (torch.empty(shape, dtype=dt, device=DEVICE) for _ in range(2))
    if kind != "store":
        for i in range(0, pages, step):
            n = min(step, pages - i)
            k = _randn(gen, n, HKV, page, d, dtype=torch.float32).mul_(k_size[:, None])
            v = _randn(gen, n, HKV, page, d, dtype=torch.float32).mul_(v_size[:, None])
            if kind in ("load", "decode8"):
                s["k_cache"][i : i + n], s["k_scale"][i : i + n] = _quantize(k, case["cache"])
                s["v_cache"][i : i + n], s["v_scale"][i : i + n] = _quantize(v, case["cache"])
            else:
                s["k_cache"][i : i + n], s["v_cache"][i : i + n] = k, v
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    if kind == "store":
        # A prefill's tokens take their places in the sequences from 0 on, a decode step's one each its last place.
        n = len(lens) if case["step"] else sum(lens)
        s["cu"] = _cu([1] * len(lens) if case["step"] else lens)
        s["positions"] = s["seq_lens"] - 1 if case["step"] else None
        s["k"] = (_randn(gen, n, HKV, d, dtype=torch.float32) * k_size).to(dt)
        s["v"] = (_randn(gen, n, HKV, d, dtype=torch.float32) * v_size).to(dt)
    elif kind == "load":
        s["cu"], s["tokens"], s["dtype"] = _cu(lens), sum(lens), dt
    elif kind == "tree":
        # Each node's parent is an earlier node of its tree or the context's end; a node sees its ancestors and itself.
        b, most = len(lens), max(nodes)
        parent = (torch.rand(b, most, generator=gen, device=DEVICE) * (torch.arange(most, device=DEVICE) + 1)).long() - 1
        link = torch.nn.functional.one_hot(parent + 1, most + 1)[:, :, 1:].float()
        sees = link + torch.eye(most, device=DEVICE)
        for _ in range(max(1, most.bit_length())):
            sees = (torch.matmul(sees, sees) > 0).float()
        held = torch.arange(most, device=DEVICE)[None, :] < torch.tensor(nodes, device=DEVICE)[:, None]
        bits = (sees.long() << torch.arange(most, device=DEVICE)).sum(-1)
        s["cu"], s["most"] = _cu(nodes), most
        s["tree_mask"] = bits[held].reshape(-1, 1).contiguous()
        s["q"] = _randn(gen, sum(nodes), case["heads"], d, dtype=dt)
    else:
        s["q"] = _randn(gen, len(lens), case["heads"], d, dtype=dt)
    return s


# --------------------------------------------------------------- the calls --
def run(s):
    if own:
        return _run_own(s)
    kind = s["kind"]
    if kind == "store":
        return _store(s)
    if kind == "load":
        return _load(s)
    if kind == "prefill":
        return _prefill(s)
    if kind == "tree":
        return _tree(s)
    return _decode(s)


def _run_own(s):
    from tinyserver_amd import kernels

    kind = s["kind"]
    if kind == "store":
        kernels.store_kv_cache_quantized(s["k"].transpose(0, 1), s["v"].transpose(0, 1), s["k_cache"], s["v_cache"],
                                         s["k_scale"], s["v_scale"], s["tables"], s["cu"], s["positions"])
        return {n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    if kind == "load":
        k, v = kernels.load_kv_cache_quantized(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["tables"],
                                               s["cu"], s["tokens"], dtype=s["dtype"])
        return {"k": k, "v": v}
    if kind == "decode8":
        return kernels.paged_attention_quantized(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                                                 s["tables"], s["page"], s["seq_lens"], window=s["window"],
                                                 sinks=s["sinks"])
    if kind == "window":
        return kernels.paged_attention_window(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["page"], s["seq_lens"],
                                              s["window"], s["sinks"])
    if kind == "prefill":
        return kernels.flash_attn_varlen_window(s["q"], s["k"], s["v"], s["cu"], s["cu"], s["max_len"], s["max_len"],
                                                s["window"], s["sinks"])
    return kernels.paged_attention_tree(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["page"], s["seq_lens"],
                                        s["cu"], s["tree_mask"], max_nodes=s["most"])


def _places(s, tokens):
    """(page, slot) of each packed token, from its sequence and its position there."""
    t = torch.arange(tokens, device=DEVICE)
    seq = torch.searchsorted(s["cu"][1:], t.to(torch.int32), right=True)
    pos = t - s["cu"][seq] if s.get("positions") is None else s["positions"].long()
    return s["tables"][seq, pos // s["page"]].long(), pos % s["page"]


def _store(s):
    block, slot = _places(s, s["k"].shape[0])
    s["k_cache"][block, :, slot], s["k_scale"][block, :, slot] = _quantize(s["k"], s["cache"])
    s["v_cache"][block, :, slot], s["v_scale"][block, :, slot] = _quantize(s["v"], s["cache"])
    return {n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}


def _rows(s, name, block, slot):
    """Cache rows in 32 bits, with their scales where it has any: (..., HKV, D)."""
    x = s[name + "_cache"][block, :, slot].float()
    return x * s[name + "_scale"][block, :, slot][..., None] if name + "_scale" in s else x


def _load(s):
    block, slot = _places(s, s["tokens"])
    return {n: _rows(s, n, block, slot).to(s["dtype"]) for n in ("k", "v")}


def _attend(q, k, v, sees):
    """softmax(q k^T / sqrt(D)) v in 32 bits: q (B, R, Hq, D), k and v (B, L, HKV, D), sees (B, R, L)."""
    b, r, hq, d = q.shape
    q = q.float().reshape(b, r, HKV, -1, d).permute(0, 2, 3, 1, 4).reshape(b, HKV, -1, d).contiguous()
    sc = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) / math.sqrt(d)
    sc = sc.reshape(b, HKV, -1, r, sc.shape[-1]).masked_fill(~sees[:, None, None], float("-inf"))
    p = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True).clamp(min=1e-30)
    p = p.reshape(b, HKV, -1, p.shape[-1])
    o = torch.matmul(p, v.permute(0, 2, 1, 3).contiguous()).reshape(b, HKV, -1, r, d) / total
    return o.permute(0, 3, 1, 2, 4).reshape(b, r, hq, d)


def _decode(s):
    lens = s["seq_lens"].long()[:, None]
    if s["window"]:  # the first tokens, then the window's
        first = torch.arange(s["sinks"], device=DEVICE).expand(lens.shape[0], -1)
        last = lens - s["window"] + torch.arange(s["window"], device=DEVICE)
        pos = torch.cat([first, last], dim=1)
        old = (first < lens - s["window"]) & (first < lens)
        sees = torch.cat([old, last >= 0], dim=1)
    else:
        pos = torch.arange(s["tables"].shape[1] * s["page"], device=DEVICE).expand(lens.shape[0], -1)
        sees = pos < lens
    pos = pos.clamp(min=0).minimum(lens - 1)
    block, slot = s["tables"].gather(1, pos // s["page"]).long(), pos % s["page"]
    o = _attend(s["q"][:, None], _rows(s, "k", block, slot), _rows(s, "v", block, slot), sees[:, None])
    return o[:, 0].to(s["q"].dtype)


def _tree(s):
    b, most = s["tables"].shape[0], s["most"]
    ctx, cu = s["seq_lens"].long()[:, None], s["cu"].long()
    node = torch.arange(most, device=DEVICE)
    held = node[None, :] < (cu[1:] - cu[:-1])[:, None]
    at = (cu[:-1, None] + node).clamp(max=s["q"].shape[0] - 1)  # packed node of (sequence, node)
    pos = torch.arange(s["tables"].shape[1] * s["page"], device=DEVICE).expand(b, -1)
    block, slot = s["tables"].gather(1, pos // s["page"]).long(), pos % s["page"]
    which = pos - ctx  # a token's node, where it is one
    bits = s["tree_mask"][:, 0][at][:, :, None] >> which.clamp(0, 63)[:, None, :]
    sees = (which < 0)[:, None, :] | ((which >= 0) & (which < most))[:, None, :] & (bits & 1).bool()
    o = _attend(s["q"][at], _rows(s, "k", block, slot), _rows(s, "v", block, slot), sees)
    return o[held].to(s["q"].dtype)


def _prefill(s):
    t, hq, d = s["q"].shape
    w, n = min(s["window"], s["max_len"]), s["sinks"]
    at = torch.arange(t, device=DEVICE)
    start = s["cu"].long()[torch.searchsorted(s["cu"][1:], at.to(torch.int32), right=True)]  # its sequence's first token
    blocks = -(-t // w)
    pad = (0, 0, 0, 0, 0, blocks * w - t)
    q = torch.nn.functional.pad(s["q"].float(), pad).reshape(blocks, w, HKV, -1, d).permute(2, 0, 3, 1, 4)
    q = q.reshape(HKV, blocks, -1, d).contiguous()  # (HKV, blocks, G w, D)

    def two(x):  # each block of w keys behind the one before it: (HKV, blocks, 2 w, D)
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, w, blocks * w - t)).reshape(blocks + 1, w, HKV, d)
        return torch.cat([x[:-1], x[1:]], dim=1).permute(2, 0, 1, 3).contiguous()

    i = at.new_zeros(blocks * w) - 1
    i[:t] = at
    first = i.new_zeros(blocks * w)
    first[:t] = start
    qi = i.reshape(blocks, w, 1)
    kj = (torch.arange(2 * w, device=DEVICE) - w)[None, :] + (torch.arange(blocks, device=DEVICE) * w)[:, None]
    kj = kj[:, None, :]
    near = (kj <= qi) & (kj > qi - s["window"]) & (kj >= first.reshape(blocks, w, 1))
    sc = torch.matmul(q, two(s["k"]).transpose(2, 3).contiguous()).reshape(HKV, blocks, -1, w, 2 * w) / math.sqrt(d)
    sc.masked_fill_(~near[:, None], float("-inf"))
    # The first n tokens of each query's sequence that its window has left.
    far = first[:, None] + torch.arange(n, device=DEVICE)
    old = (far <= i[:, None] - s["window"]).reshape(blocks, 1, w, n)
    far = far.clamp(max=t - 1)
    qs = q.reshape(HKV, blocks, -1, w, d).permute(0, 1, 3, 2, 4).reshape(HKV, blocks * w, -1, d).contiguous()
    sk = s["k"].float()[far].permute(2, 0, 3, 1).contiguous()  # (HKV, blocks w, D, n)
    se = torch.matmul(qs, sk).reshape(HKV, blocks, w, -1, n).permute(0, 1, 3, 2, 4) / math.sqrt(d)
    se = se.masked_fill(~old, float("-inf"))
    top = sc.amax(-1, keepdim=True)
    top = (torch.maximum(top, se.amax(-1, keepdim=True)) if n else top).clamp(min=-1e30)
    p, pe = sc.sub_(top).exp_(), torch.exp(se - top)
    total = p.sum(-1, keepdim=True) + pe.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(HKV, blocks, -1, 2 * w), two(s["v"])).reshape(HKV, blocks, -1, w, d)
    pe = pe.permute(0, 1, 3, 2, 4).reshape(HKV, blocks * w, -1, n).contiguous()
    oe = torch.matmul(pe, s["v"].float()[far].permute(2, 0, 1, 3).contiguous())
    o = (o + oe.reshape(HKV, blocks, w, -1, d).permute(0, 1, 3, 2, 4)) / total.clamp(min=1e-30)
    return o.permute(1, 3, 0, 2, 4).reshape(blocks * w, hq, d)[:t].to(s["q"].dtype)


def work(case):
    kind, d, lens = case["kind"], case["dim"], _lengths(case)
    if kind in ("store", "load"):
        # 16-bit rows on one side, 8-bit rows and their scales on the other.
        t = len(lens) if case.get("step") else sum(lens)
        return {"bytes": 2 * t * HKV * (3 * d + 4), "flops": 2 * t * HKV * d * 2}
    hq = case["heads"]
    if kind == "prefill":
        w, n = case["window"], case["sinks"]
        # A query at i sees min(i + 1, w) keys of its window and the first n that it has left.
        pairs = sum(m * (m + 1) // 2 - max(0, m - w) * (max(0, m - w) + 1) // 2 for m in lens)
        pairs += sum(sum(min(n, max(0, i + 1 - w)) for i in range(m)) if m <= w + n else
                     n * (m - w - n) + n * (n + 1) // 2 for m in lens)
        t = sum(lens)
        return {"bytes": 2 * t * d * (2 * hq + 2 * HKV), "flops": 4 * d * hq * pairs}
    if kind == "tree":
        nodes = _nodes(case)
        t, n = sum(lens) + sum(nodes), sum(nodes)
        pairs = sum(a * b + b * (b + 1) // 2 for a, b in zip(lens, nodes))
        tables = 4 * sum(-(-(a + b) // case["page"]) for a, b in zip(lens, nodes))
        return {"bytes": 4 * t * HKV * d + 4 * n * hq * d + 8 * n + tables, "flops": 4 * d * hq * pairs}
    w = case["window"]
    t = sum(min(m, w + min(case["sinks"], max(0, m - w))) if w else m for m in lens)
    row = d + 4 if kind == "decode8" else 2 * d
    tables = 4 * sum(-(-min(m, w + case["sinks"] if w else m) // case["page"]) for m in lens) + 4 * len(lens)
    return {"bytes": 2 * t * HKV * row + 4 * len(lens) * hq * d + tables, "flops": 4 * t * hq * d}


# ------------------------------------------------------- the same in 64 bits --
def exact(case, seed):
    """Sequence by sequence from the definitions, in 64 bits."""
    s = prepare(case, seed)
    kind, d, lens = case["kind"], case["dim"], _lengths(case)

    def gather(name, seq, n):  # (HKV, n, D): a sequence's first n cache rows
        page = case["page"]
        used = s["tables"][seq, : -(-n // page)].long()
        x = s[name + "_cache"][used].double()
        if name + "_scale" in s:
            x = x * s[name + "_scale"][used].double()[..., None]
        return x.transpose(0, 1).reshape(HKV, -1, d)[:, :n].contiguous()

    def attend(q, k, v, sees):  # q (R, D), k and v (L, D), sees (R, L)
        sc = torch.mm(q, k.t().contiguous()) / math.sqrt(d)
        return torch.mm(torch.softmax(sc.masked_fill_(~sees, float("-inf")), dim=-1), v)

    if kind == "load":
        return {n: torch.cat([gather(n, i, m).transpose(0, 1) for i, m in enumerate(lens)]) for n in ("k", "v")}
    if kind == "store":
        top = LARGEST[case["cache"]]
        out = {}
        for n in ("k", "v"):
            values, scales = s[n + "_cache"].double(), s[n + "_scale"].double()
            x = s[n].double()
            size = x.abs().max(-1).values / top
            # A magnitude in [2^e, 2^(e + 1)) has steps of 2^(e - 3), one below 2^-6 those of 2^-9.
            y = x / size[..., None]
            unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
            y = torch.round(y / unit) * unit
            start = 0
            for i, m in enumerate(lens):
                at = range(m - 1, m) if case["step"] else range(m)
                pos = torch.tensor(list(at), device=DEVICE)
                block, slot = s["tables"][i, pos // case["page"]].long(), pos % case["page"]
                values[block, :, slot] = y[start : start + len(at)]
                scales[block, :, slot] = size[start : start + len(at)]
                start += len(at)
            out[n + "_cache"], out[n + "_scale"] = (values if case["cache"] == "e4m3" else None), scales
        return out
    hq = case["heads"]
    group, start = hq // HKV, 0
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for i, m in enumerate(lens):
        if kind == "prefill":
            w, n, step = case["window"], case["sinks"], 2048
            for h in range(HKV):
                k, v = (s[x][start : start + m, h].double().contiguous() for x in ("k", "v"))
                for a in range(0, m, step):
                    b = min(m, a + step)
                    lo = max(0, a - w + 1)
                    keys = torch.cat([torch.arange(min(n, lo), device=DEVICE), torch.arange(lo, b, device=DEVICE)])
                    at = torch.arange(a, b, device=DEVICE)[:, None]
                    sees = (keys[None, :] <= at) & ((keys[None, :] > at - w) | (keys[None, :] < n))
                    for g in range(group):
                        q = s["q"][start + a : start + b, h * group + g].double().contiguous()
                        out[start + a : start + b, h * group + g] = attend(q, k[keys], v[keys], sees)
            start += m
            continue
        nodes = _nodes(case)[i] if kind == "tree" else 1
        k, v = gather("k", i, m + nodes if kind == "tree" else m), gather("v", i, m + nodes if kind == "tree" else m)
        j = torch.arange(k.shape[1], device=DEVICE)
        if kind == "tree":
            bits = s["tree_mask"][start : start + nodes]
            tree = (bits >> torch.arange(nodes, device=DEVICE)) & 1
            sees = torch.cat([torch.ones(nodes, m, dtype=torch.bool, device=DEVICE), tree.bool()], dim=1)
        else:
            w = case["window"] or m
            sees = ((j >= m - w) | (j < case["sinks"]))[None, :]
        for h in range(HKV):
            q = s["q"][start : start + nodes, h * group : (h + 1) * group].double().transpose(0, 1).reshape(-1, d)
            o = attend(q.contiguous(), k[h], v[h], sees.repeat(group, 1))
            out[start : start + nodes, h * group : (h + 1) * group] = o.reshape(group, nodes, d).transpose(0, 1)
        start += nodes
    return out
