"""How near the log probabilities' kernels come to 64 bits, run on the CPU: rows with a sure
token, with a few allowed ones, and flat ones."""

import pytest
import torch

from tests import workgroup
from tests.logprobs_reference import near, rows
from tests.test_logprobs_workgroup import lib, pytestmark, run  # noqa: F401


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind,n,v", [
    ("few", 20, 1003), ("few", 6, 20011), ("one_thread", 40, 5003), ("one_thread", 20, 20011),
    ("sure", 4, 5003), ("sure", 2, 151936), ("even", 2, 151936), ("plain", 2, 20011)])
def test_side_by_side(lib, kind, n, v, dtype):  # noqa: F811
    x, tokens = rows(kind, n, v, dtype, "cpu")
    near(x, tokens, run(lib, x, tokens, 2, waves=1), f"{kind}, {n} x {v}, {dtype}")


@pytest.mark.parametrize("kind", ["few", "one_thread", "sure", "even"])
def test_other_strides(lib, kind):  # noqa: F811
    x, tokens = rows(kind, 8, 5003, torch.float32, "cpu")
    near(x, tokens, run(lib, x.t().contiguous().t(), tokens, 2, waves=1), f"{kind}, columns first", side_by_side=False)
