"""Sequences moved from an 8-bit pool to a 16-bit one (read back, stored, then
decoded there): the 16-bit pool holds the 8-bit one's values rounded once, and the
decode over either is that of the same token (tolerance: half a step of each value
of K and V, of the weights and of both outputs, from their types)."""

import pytest
import torch

from tinyserver_amd.kernels import (
    load_kv_cache_quantized,
    paged_attention_forward,
    paged_attention_quantized,
    store_kv_cache_paged,
    store_kv_cache_quantized,
)

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("cache", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", [[1, 300, 17], [700] * 5])
def test_to_a_16_bit_pool(cache, dtype, lens):
    g = torch.Generator(device=DEV).manual_seed(len(lens))
    hq, hkv, d, page, n = 16, 4, 128, 16, sum(lens)
    need = [-(-m // page) for m in lens]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)
    bt = torch.zeros(2, len(lens), max(need), dtype=torch.int32, device=DEV)
    for pool in range(2):  # the same sequences on other pages
        perm, at = torch.randperm(sum(need), generator=g, device=DEV).to(torch.int32), 0
        for s, m in enumerate(need):
            bt[pool, s, :m] = perm[at : at + m]
            at += m
    k, v = (torch.randn(n, hkv, d, generator=g, device=DEV).to(dtype) for _ in range(2))
    codes = [torch.zeros(sum(need), hkv, page, d, dtype=cache, device=DEV) for _ in range(2)]
    scales = [torch.zeros(sum(need), hkv, page, device=DEV) for _ in range(2)]
    store_kv_cache_quantized(k.transpose(0, 1), v.transpose(0, 1), *codes, *scales, bt[0], cu)
    wide = [torch.zeros(sum(need), hkv, page, d, dtype=dtype, device=DEV) for _ in range(2)]
    k2, v2 = load_kv_cache_quantized(*codes, *scales, bt[0], cu, n, dtype=dtype)
    store_kv_cache_paged(k2.transpose(0, 1), v2.transpose(0, 1), *wide, bt[1], cu)
    for s, m in enumerate(lens):
        a, b = bt[0, s, : need[s]].long(), bt[1, s, : need[s]].long()
        for c, x, w in zip(codes, scales, wide):
            one = (c[a].float() * x[a][..., None]).to(dtype).transpose(0, 1).reshape(hkv, -1, d)[:, :m]
            assert torch.equal(one, w[b].transpose(0, 1).reshape(hkv, -1, d)[:, :m])
    q = torch.randn(len(lens), hq, d, generator=g, device=DEV).to(dtype)
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    x = paged_attention_quantized(q, *codes, *scales, bt[0], page, sl).float()
    y = paged_attention_forward(q, *wide, bt[1], page, sl).float()
    # a K value off by u of itself moves a score by u max sum|q k| scale, a weight by as much of itself and the
    # mean by twice that of max|v|; V's rounding, the weights' and the outputs' add u each
    u = torch.finfo(dtype).eps / 2
    score = float((q.float().abs().sum(-1) * k.float().abs().max()).max()) * d**-0.5
    assert float((x - y).abs().max()) <= float(v.float().abs().max()) * u * (2 * score + 4)
