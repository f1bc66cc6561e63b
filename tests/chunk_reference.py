"""64-bit reference of attention of a chunk over the paged cache, on the CPU, and
its tolerance (derived in rows_reference: the output's rounding, the weights' to
the type, an error of the scores, the sums)."""

import torch

from tests.rows_reference import half_step, pool


def reference(q, kc, vc, bt, ctx, new, scale):
    """(outputs, tolerances) of the packed rows q (T, Hq, D), in 64 bits: sequence s's new[s] rows at positions
    ctx[s].. over its cache rows; positions whose page is outside the pool or past the table are not seen."""
    t, hq, d = q.shape
    nb, hkv, page, _ = kc.shape
    g = hq // hkv
    u, u_p = half_step(q.dtype), 0.0 if q.dtype == torch.float32 else half_step(q.dtype)
    ref, tol = torch.zeros(t, hq, d, dtype=torch.float64), torch.zeros(t, hq, d, dtype=torch.float64)
    start = 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        cap = bt.shape[1] * page
        pos = torch.arange(min(c + n, cap))
        ids = bt[s].long()[pos // page]
        ok = (ids >= 0) & (ids < nb)
        pos, ids = pos[ok], ids[ok]
        k, v = (x[ids, :, pos % page].double() for x in (kc, vc))  # (L, Hkv, D)
        sees = pos[None, :] <= min(c, cap) + torch.arange(n)[:, None]
        for h in range(hq if n and len(pos) else 0):
            kh, vh, qh = k[:, h // g], v[:, h // g], q[start : start + n, h].double()
            # what a row does not see may hold anything
            sc = (qh @ kh.t() * scale).masked_fill(~sees, float("-inf"))
            p = torch.softmax(sc, -1).nan_to_num() if not torch.isnan(sc).any() else torch.softmax(sc, -1)
            p = torch.where(sees.any(-1, keepdim=True), p, 0.0)
            vz = torch.where(torch.isfinite(vh), vh, 0.0)
            o = p @ vz
            bad = sees.double() @ (~torch.isfinite(vh)).double() > 0
            ref[start : start + n, h] = torch.where(bad, float("nan"), o)
            size = (qh.abs() @ kh.abs().nan_to_num().t()).masked_fill(~sees, 0.0).amax(-1, keepdim=True).nan_to_num() * abs(scale)
            e = size * ((d + 2) * 2.0**-24 + 4 * 2.0**-23) + 2.0**-22
            top = torch.where(sees, vz.abs().amax(-1), 0.0).amax(-1, keepdim=True)
            tol[start : start + n, h] = u * o.abs() + top * (u_p + 2 * e + 2 * len(pos) * 2.0**-24)
        start += n
    return ref, tol


def inputs(ctx, new, hq, hkv, d, page, dtype, seed=0):
    """(q, k_cache, v_cache, block tables) on the CPU; slots behind the last token hold NaN and infinities."""
    gen = torch.Generator().manual_seed(seed + 7 * d + sum(new))
    kc, vc, bt = pool([a + b for a, b in zip(ctx, new)], hkv, d, page, seed + page)
    kc, vc = kc.to(dtype), vc.to(dtype)
    q = torch.randn(sum(new), hq, d, generator=gen).to(dtype)
    for s, (c, n) in enumerate(zip(ctx, new)):
        for p in range(c + n, -(-(c + n) // page) * page):
            kc[int(bt[s, p // page]), :, p % page] = float("nan")
            vc[int(bt[s, p // page]), :, p % page] = float("inf")
    return q, kc, vc, bt
