"""Log probabilities of rows that the first tests do not have: a mask that allows about as
many consecutive tokens as the list of candidates holds (1,024)."""

import pytest
import torch

from tests.test_gpu_logprobs import _check

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,v", [(2, 151936), (600, 5003)])  # rows cut into parts, and whole ones
@pytest.mark.parametrize("allowed", [908, 909, 1000, 1024, 1025])
def test_allowed_tokens_in_one_place(allowed, n, v, dtype):
    g = torch.Generator(device=DEV).manual_seed(allowed)
    x = torch.full((n, v), float("-inf"), device=DEV).to(dtype)
    for i, start in enumerate((1600, v - 3 - allowed)):
        x[i::2, start : start + allowed] = torch.randn(x[i::2].shape[0], allowed, generator=g, device=DEV).to(dtype)
    tokens = torch.randint(1600, 1600 + allowed, (n,), generator=g, device=DEV)
    for top in (50, 64):
        _check(x, tokens, top, f"{allowed} allowed, {n} x {v}, top {top}, {dtype}")
