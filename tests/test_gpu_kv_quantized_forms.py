"""The 8-bit store and load in the forms that long and wide batches take, and at
signed zeros: codes and scales bit-equal to the definition, values read back
bit-equal to code * scale rounded once. Calls of 2048 tokens or more give a
workgroup two kv heads (an odd one is left over), calls of more than 2048
sequences search them elsewhere."""

import pytest
import torch

from tests.rows_reference import quantize
from tests.test_gpu_kv_quantized import _same, _state
from tinyserver_amd.kernels import load_kv_cache_quantized, store_kv_cache_quantized

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4, I8 = torch.float8_e4m3fn, torch.int8


def _store_and_load(bt, codes, scales, src, lens, page):
    """Stores packed rows, compares the whole pools with the definition, and what is read back."""
    n = sum(lens)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    pos = torch.arange(n) - cu.cpu().long()[seq]
    block, slot = bt[seq, pos // page].long(), pos % page
    want = []
    for c, s, x in zip(codes, scales, src):
        c, s = c.cpu().clone(), s.cpu().clone()
        q, qs = quantize(x.cpu(), c.dtype)
        c.view(torch.uint8)[block, :, slot] = q.view(torch.uint8)
        s[block, :, slot] = qs
        want.append((c, s))
    store_kv_cache_quantized(src[0].transpose(0, 1), src[1].transpose(0, 1), *codes, *scales, bt.to(DEV), cu)
    for (c, s), gc, gs in zip(want, codes, scales):
        _same(gs, s, "scales")
        _same(gc, c, "codes")
    got = load_kv_cache_quantized(*codes, *scales, bt.to(DEV), cu, n, dtype=src[0].dtype)
    for (c, s), x in zip(want, got):
        _same(x, (c[block, :, slot].float() * s[block, :, slot][..., None]).to(src[0].dtype), "rows")


@pytest.mark.parametrize("cache", [E4, I8])
@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64), (F32, 128), (BF, 80)])
def test_signed_zeros(cache, dtype, d):
    """Negative zeros, and negative values whose quotient rounds to zero, keep their sign in e4m3 (int8 has one zero);
    all-zero rows have codes 0 of either sign of zero."""
    bt, codes, scales, g = _state([8], 3, d, 16, cache, 21)
    x = torch.randn(8, 3, d, generator=g).to(dtype)
    x[:, :, ::3] = -0.0
    x[:, :, 1::5] = 0.0
    x[2, :, 2::7] = -2.0 ** -13  # (of a row whose largest is about 3: far below half the least code)
    x[3] = -0.0
    x[4, 1] = 0.0
    _store_and_load(bt, codes, scales, [x.to(DEV), x.flip(0).to(DEV)], [8], 16)
    if cache == E4:
        assert int((codes[0].view(torch.uint8) == 0x80).sum()) > 0


@pytest.mark.parametrize("cache", [E4, I8])
@pytest.mark.parametrize("dtype,hkv,d,lens", [
    (BF, 8, 128, [2000, 60]),
    (F16, 3, 128, [700, 1, 0, 1400]),  # an odd head is left over
    (BF, 1, 64, [2300]),
    (F16, 5, 64, [1024, 1024]),        # the first call of two heads a workgroup
    (BF, 5, 64, [1024, 1023]),         # the last of one
])
def test_two_heads_a_workgroup(cache, dtype, hkv, d, lens):
    bt, codes, scales, g = _state(lens, hkv, d, 16, cache, hkv + d)
    n = sum(lens)
    src = [(torch.randn(n, hkv, d, generator=g) * torch.exp(2 * torch.randn(n, hkv, 1, generator=g))).to(dtype).to(DEV)
           for _ in range(2)]
    _store_and_load(bt, codes, scales, src, lens, 16)


@pytest.mark.parametrize("cache", [E4, I8])
@pytest.mark.parametrize("seqs", [2048, 2049])
def test_many_sequences(cache, seqs):
    """Sequences of 0 to 2 tokens, either side of the most whose starts are kept in LDS."""
    g = torch.Generator().manual_seed(seqs)
    lens = torch.randint(0, 3, (seqs,), generator=g).tolist()
    bt, codes, scales, g = _state(lens, 2, 128, 16, cache, 4)
    src = [torch.randn(sum(lens), 2, 128, generator=g).to(BF).to(DEV) for _ in range(2)]
    _store_and_load(bt, codes, scales, src, lens, 16)
