"""Decode over 8-bit caches whose scales lie outside f16's range or far apart
within a sequence, f16 and bf16 queries, against 64 bits.

Tolerance, derived: an output is sum_j p_j v_j / sum_j p_j. Weights off by
relative d_j move it by at most (sum_j p_j |v_j| + |o|) max d (p normalised).
d: 2^-16 for a weight times its scale as two 16-bit halves (16 significant bits),
twice the score's error and the sums' 2 n 2^-24 as in rows_reference. The output's
rounding adds u |o|, and in f16 at least half its least step, 2^-25."""

import math

import pytest
import torch

from tests.rows_reference import half_step, pool, quantize
from tinyserver_amd.kernels import paged_attention_quantized

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16 = torch.bfloat16, torch.float16
E4, I8 = torch.float8_e4m3fn, torch.int8


def _sizes(what, shape, g):
    """Magnitudes of the rows (pages, heads, slots) of K and V."""
    one = torch.ones(shape)
    pick = torch.rand(shape, generator=g)
    if what == "tiny":  # scales below f16's least number
        return one, one * 1e-6
    if what == "mixed":  # rows of 1e-6 among rows of 1e4; K of 1e-4 to 3
        return torch.where(pick < 0.3, 1e-4, torch.where(pick < 0.6, 0.1, 3.0)), torch.where(torch.rand(shape, generator=g) < 0.5, 1e-6, 1e4)
    if what == "heads":  # one head tiny, the next near f16's largest outputs
        head = (torch.arange(shape[1]) % 2 == 0)[None, :, None].expand(shape)
        return torch.where(head, 2.0, 0.01), torch.where(head, 1e-6, 1e4)
    return torch.where(pick < 0.5, 1e-6, 4.0), torch.where(pick < 0.5, 1e5, 1e-3)  # "apart": K's scale against V's


@pytest.mark.parametrize("cache", [E4, I8])
@pytest.mark.parametrize("dtype", [F16, BF])
@pytest.mark.parametrize("what", ["tiny", "mixed", "heads", "apart"])
@pytest.mark.parametrize("hq,hkv,d,page,lens", [
    (8, 2, 128, 16, [300, 40]),       # a workgroup a unit
    (16, 4, 64, 32, [1500, 7, 600]),  # splits
    (16, 8, 128, 16, [2500] + [60 + 37 * i % 700 for i in range(63)]),  # the stream
    (4, 2, 128, 4, [90, 33]),         # pages under 16 tokens
])
def test_scales(cache, dtype, what, hq, hkv, d, page, lens):
    g = torch.Generator().manual_seed(len(lens) + d)
    kc, vc, bt = pool(lens, hkv, d, page, len(lens))
    ks, vs = _sizes(what, kc.shape[:3], g)
    if dtype == F16 and what == "apart":
        vs = vs.clamp(max=2e4)  # (outputs that f16 holds)
    (kc, ks), (vc, vs) = (tuple(t.to(DEV) for t in quantize(x.nan_to_num() * s[..., None], cache)) for x, s in ((kc, ks), (vc, vs)))
    q = torch.randn(len(lens), hq, d, generator=g).to(dtype).to(DEV)
    bt = bt.to(DEV)
    out = paged_attention_quantized(q, kc, vc, ks, vs, bt, page, torch.tensor(lens, dtype=torch.int32, device=DEV))
    worst, group = 0.0, hq // hkv
    for s, n in enumerate(lens):
        pages = bt[s, : -(-n // page)].long()
        k, v = ((c[pages].double() * x[pages].double()[..., None]).transpose(0, 1).reshape(hkv, -1, d)[:, :n].contiguous()
                for c, x in ((kc, ks), (vc, vs)))
        qs = q[s].double().reshape(hkv, group, d).contiguous()
        score = torch.bmm(qs, k.transpose(1, 2).contiguous()) / math.sqrt(d)
        p = torch.softmax(score, -1)
        o = torch.bmm(p, v)
        size = torch.bmm(qs.abs(), k.abs().transpose(1, 2).contiguous()).amax(-1, keepdim=True) / math.sqrt(d)
        e = size * ((d + 2) * 2.0**-24 + 4 * 2.0**-23) + 2.0**-22
        tol = (torch.bmm(p, v.abs()) + o.abs()) * (2.0**-16 + 2 * e + 2 * n * 2.0**-24) + half_step(dtype) * o.abs()
        tol += 2.0**-25 if dtype == F16 else 0.0
        got = out[s].double().reshape(hkv, group, d)
        assert bool(torch.isfinite(got).all())
        worst = max(worst, float(((got - o).abs() / tol).max()))
    print(f"{what}, {cache}, {dtype}, {hq}/{hkv} x {d}, {len(lens)} sequences: {worst:.2f} of the tolerance", flush=True)
    assert worst <= 1
