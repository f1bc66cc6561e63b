"""Windowed prefill of as many sequences as the LDS-staged kernels count in LDS
and of one more, which takes the other kernel, against 64-bit attention of every
row (tolerances of rows_reference, with each row's largest score product bounded
over all keys)."""

import math

import pytest
import torch

from tests.rows_reference import half_step
from tinyserver_amd.kernels import flash_attn_varlen_window

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("hq,hkv,d,seqs", [
    (4, 2, 128, 1024), (4, 2, 128, 1025),
    (4, 1, 128, 2048), (4, 1, 128, 2049),
    (8, 1, 64, 2048), (8, 1, 64, 2049),
    (12, 1, 128, 2048), (12, 1, 128, 2049),
])
@pytest.mark.parametrize("window,sinks", [(2, 0), (9, 1)])
def test_sequences(hq, hkv, d, seqs, window, sinks):
    g = torch.Generator().manual_seed(seqs + hq)
    lens = torch.randint(0, 3, (seqs,), generator=g)
    lens[::97] = 40
    lens[-1] = 33
    cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).to(torch.int32).to(DEV)
    n = int(lens.sum())
    q, k, v = (torch.randn(n, h, d, generator=g).to(torch.bfloat16).to(DEV) for h in (hq, hkv, hkv))
    out = flash_attn_varlen_window(q, k, v, cu, cu, 40, 40, window, sinks).double()
    seq = torch.repeat_interleave(torch.arange(seqs), lens).to(DEV)
    i = torch.arange(n, device=DEV)
    at = i - cu.long()[seq]
    see = (seq[:, None] == seq[None, :]) & (i[None, :] <= i[:, None])
    see &= (at[None, :] > at[:, None] - window) | (at[None, :] < sinks)
    u, worst = half_step(torch.bfloat16), 0.0
    for h in range(hq):
        qh, kh, vh = (x.double() for x in (q[:, h], k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]))
        s = (qh @ kh.t().contiguous()) / math.sqrt(d)
        o = torch.softmax(s.masked_fill(~see, -math.inf), -1) @ vh
        e = (qh.abs() @ kh.abs().t().contiguous()).amax(-1) / math.sqrt(d) * ((d + 2) * 2.0**-24 + 4 * 2.0**-23) + 2.0**-22
        tol = u * o.abs() + (vh.abs().max() * (u + 2 * e + 2 * 40 * 2.0**-24))[:, None]
        worst = max(worst, float(((out[:, h] - o).abs() / tol).max()))
    print(f"{hq}/{hkv} x {d}, {seqs} sequences: {worst:.2f} of the tolerance", flush=True)
    assert worst <= 1
