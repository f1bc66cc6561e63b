"""Log probabilities of rows that the first tests do not have: a mask that allows about as
many consecutive tokens as the list of candidates holds (1,024); the same rows again;
and how near sure, flat and sparse rows come to 64 bits (the tolerance:
logprobs_reference)."""

import math

import pytest
import torch

from tests.logprobs_reference import near, rows
from tests.test_gpu_logprobs import _check
from tinyserver_amd.kernels import token_logprobs

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


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("n,v", [(3, 151936), (64, 40001), (600, 5003)])
def test_the_same_again(n, v, dtype):
    """Call after call, bit for bit, whichever thread writes an alternative."""
    for seed in range(5):
        g = torch.Generator(device=DEV).manual_seed(seed)
        x = (3 * torch.randn(n, v, generator=g, device=DEV)).to(dtype)
        tokens = torch.randint(v, (n,), generator=g, device=DEV)
        first = token_logprobs(x, tokens, 20)
        for _ in range(12):
            assert all(torch.equal(a, b) for a, b in zip(first, token_logprobs(x, tokens, 20))), f"{n} x {v}, {dtype}, seed {seed}"


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("kind,n,v", [
    ("few", 600, 1003), ("few", 20, 20011), ("one_thread", 600, 5003), ("one_thread", 100, 20011), ("sure", 520, 5003),
    ("sure", 70, 151936), ("even", 5, 151936), ("plain", 8, 151936)])
def test_accuracy(kind, n, v, dtype):
    x, tokens = rows(kind, n, v, dtype, DEV)
    near(x, tokens, token_logprobs(x, tokens, 2), f"{kind}, {n} x {v}, {dtype}")


@pytest.mark.parametrize("kind", ["few", "one_thread", "sure", "even"])
def test_accuracy_of_other_strides(kind):
    x, tokens = rows(kind, 40, 5003, F32, DEV)
    near(x, tokens, token_logprobs(x.t().contiguous().t(), tokens, 2), f"{kind}, columns first", side_by_side=False)


def test_many_equal_weights():
    """2^20 logits of weights that one float32 sum over a thread's 4,096 of them rounds down at nearly every addition
    (it ends 6e-5 of itself too low): sums by piece, tile and row stay within a few of their roundings."""
    v, rest = 1 << 20, 0.99 * 2.0**-13  # weights of (1 + rest) / 2, an ulp of 2^-13 from a sum of 1,024 on
    x = torch.full((1, v), math.log1p(rest) - math.log(2.0), device=DEV)
    x[:, :1024:256] = 0.0  # each wave's largest, in its first piece
    tokens = torch.tensor([5], device=DEV)
    whole = token_logprobs(x.expand(520, -1), tokens.expand(520), 2)
    near(x, tokens, [a[:1] for a in whole], "whole rows")
    assert all(torch.equal(a, a[:1].expand_as(a)) for a in whole)
    near(x, tokens, token_logprobs(x, tokens, 2), "a row in parts")
