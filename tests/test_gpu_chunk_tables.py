"""Attention of a chunk under short tables, on both sides of the lengths and numbers of
sequences at which items are cut into runs, against 64 bits."""

import pytest
import torch

from tests.chunk_reference import inputs, reference
from tests.rows_reference import check
from tinyserver_amd.kernels import paged_attention_chunk

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("blocks", [8, 9, 12, 13, 16, 17])
@pytest.mark.parametrize("seqs,new", [(1, 1), (3, 5), (13, 1), (20, 7), (2, 60)])
def test_short_tables(seqs, new, blocks, dtype):
    cap, hq, hkv, d = 32 * blocks, 8, 4, 128
    lens = [cap - (i * 37) % (cap // 2) for i in range(seqs)]
    n = [max(0, new - i % 3) if i else new for i in range(seqs)]
    ctx = [a - b for a, b in zip(lens, n)]
    q, kc, vc, bt = inputs(ctx, n, hq, hkv, d, 16, dtype)
    if bt.shape[1] < 2 * blocks:
        bt = torch.nn.functional.pad(bt, (0, 2 * blocks - bt.shape[1]))
    ref, tol = reference(q, kc, vc, bt, ctx, n, d**-0.5)
    cu = torch.tensor([0] + torch.tensor(n).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    dev = [x.to(DEV) for x in (q, kc, vc, bt)]
    out = paged_attention_chunk(*dev, 16, torch.tensor(ctx, dtype=torch.int32, device=DEV), cu, max_seqlen=new)
    check(out, ref, tol, f"{seqs} x {new} under {blocks} blocks, {dtype}")
