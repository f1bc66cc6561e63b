"""64-bit references and input makers for attention over part of a context, 8-bit
caches and draft trees, on the CPU.

Tolerance of an attention output, derived: it is a mean of rows of V with weights
exp(s - m) / sum. Rounding it to its type is off by at most u |o| (u = eps / 2 of
the type). Where the weights are rounded to the type for the second product, each
is off by u of itself, so the mean by u max|v|. A score is a sum of D products in
fp32, off by at most (D + 2) 2^-24 sum|q k| scale, and its exponent's argument
(|s - m| <= 2 max|s|, in log2 units) by 2^-23 of itself; an error e of the scores
moves a weight by e of itself and the mean by 2 e max|v|. The sums over n tokens
are off by at most n 2^-24 of max|v| each (fp32 exponentials: 2^-22)."""

import math

import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def pool(need_tokens, hkv, d, page, seed, free=3):
    """(k, v, block tables): normal rows in a pool of shuffled pages, NaN in the free ones."""
    g = torch.Generator().manual_seed(seed)
    need = [max(1, -(-n // page)) for n in need_tokens]
    pages = sum(need) + free
    kc, vc = (torch.randn(pages, hkv, page, d, generator=g) for _ in range(2))
    perm = torch.randperm(pages, generator=g)
    bt, at = torch.zeros(len(need), max(need), dtype=torch.int32), 0
    for s, n in enumerate(need):
        bt[s, :n] = perm[at : at + n]
        at += n
    kc[perm[at:]] = vc[perm[at:]] = float("nan")
    return kc, vc, bt


def quantize(x, dtype):
    """Codes and scales of rows x (..., D), as the definition has them."""
    x = x.double()
    top = x.abs().amax(-1)
    scale = torch.where(torch.isfinite(top), (top / torch.tensor(LARGEST[dtype], dtype=torch.float64)), math.nan).float()
    y = torch.where(scale[..., None] > 0, x / scale.double()[..., None], 0.0).float()
    y = y.clamp(-LARGEST[dtype], LARGEST[dtype])
    return (y.round() if dtype == torch.int8 else y).to(dtype), scale


def attend(q, k, v, scale, u, u_p):
    """(output, tolerance) of one row's q-heads q (Hq, D) over the visible k, v (n, Hkv, D), in 64 bits. u and u_p:
    half steps of the output's type and of the weights'."""
    hq, d = q.shape
    n, hkv = k.shape[:2]
    out, tol = torch.zeros(hq, d, dtype=torch.float64), torch.zeros(hq, d, dtype=torch.float64)
    for h in range(hq if n else 0):
        kh, vh, qh = k[:, h // (hq // hkv)].double(), v[:, h // (hq // hkv)].double(), q[h].double()
        out[h] = torch.softmax(kh @ qh * scale, 0) @ vh
        size = float((kh.abs() @ qh.abs()).max()) * scale
        e = size * ((d + 2) * 2.0**-24 + 4 * 2.0**-23) + 2.0**-22
        tol[h] = u * out[h].abs() + float(vh.abs().max()) * (u_p + 2 * e + 2 * n * 2.0**-24)
    return out, tol


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rows(cache, bt_row, positions):
    """(n, Hkv, D) rows of one sequence at these positions, those of pages outside the pool left out (and a mask of
    the kept)."""
    page = cache.shape[2]
    ids = [int(bt_row[p // page]) if p // page < len(bt_row) else -1 for p in positions]
    keep = [0 <= i < cache.shape[0] for i in ids]
    at = [(i, p % page) for i, p, ok in zip(ids, positions, keep) if ok]
    if not at:
        return cache.new_zeros(0, cache.shape[1], *cache.shape[3:])
    pg, sl = (torch.tensor(x) for x in zip(*at))
    return cache[pg, :, sl]


def visible(n, window, sinks):
    """Positions that the query at position n - 1 sees."""
    return [j for j in range(n) if (not window) or j >= n - window or j < sinks]


def check(out, ref, tol, what):
    out = out.detach().cpu().double()
    bad = torch.isnan(ref)
    assert torch.equal(torch.isnan(out), bad), f"{what}: NaN at other places"
    err = (out - ref).abs().nan_to_num()
    worst = float((err / tol.clamp(min=1e-300)).nan_to_num().max()) if err.numel() else 0.0
    print(f"{what}: max_abs={float(err.max()) if err.numel() else 0:.2e}, {worst:.2f} of the tolerance", flush=True)
    assert bool((err <= tol.nan_to_num()).all()), f"{what}: {worst:.2f} of the tolerance"
