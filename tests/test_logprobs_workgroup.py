"""The choice of the most likely tokens on the CPU, each of a workgroup's waves the first
at every barrier in turn: rows with about as many candidates as the list holds, and rows
that are gone through a piece at a time. Where a wave may still read the list's count
while another one appends, the waves part here, and the list is wrong."""

import pytest
import torch

from tinyserver_amd import _lib
from tests import workgroup

pytestmark = pytest.mark.skipif(workgroup.compiler() is None, reason="no compiler for the host")
BF, F32 = torch.bfloat16, torch.float32
INF = float("inf")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    return workgroup.load("token_logprobs.hip", tmp_path_factory.mktemp("logprobs"))


def _aligned(n):
    """n bytes from a 256-byte boundary on."""
    x = torch.zeros(n + 256, dtype=torch.uint8)
    start = -x.data_ptr() % 256
    return x[start : start + n]


def run(lib, x, tokens, top, waves=4):
    """(logprobs, entropy, top_logprobs, top_tokens), the same whichever wave is the first."""
    n, v = x.shape
    first = None
    for wave in range(waves):
        out = (torch.empty(n), torch.empty(n), torch.empty(n, top), torch.empty(n, top, dtype=torch.int64))
        ws = _aligned(lib.tsa_token_logprobs_workspace_bytes(n, v, top))
        lib.wg_order(wave)
        rc = lib.tsa_token_logprobs(*map(_lib.view, (*out, x, tokens)), ws.data_ptr() if len(ws) else None, len(ws), None)
        assert rc == 0 and lib.wg_error() == b"", f"wave {wave} first: {lib.wg_error().decode()}"
        if first is None:
            first = out
        assert all(torch.equal(a.nan_to_num(7e30), b.nan_to_num(7e30)) for a, b in zip(out, first)), f"wave {wave} first"
    return first


def check(lib, x, top):
    logp, entropy, top_logp, top_tokens = run(lib, x, torch.zeros(x.shape[0], dtype=torch.int64), top)
    ref = torch.log_softmax(x.double(), -1)
    order = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(top_tokens, order)
    want = ref.gather(1, order)
    assert torch.allclose(top_logp.double().nan_to_num(neginf=-1e9), want.nan_to_num(neginf=-1e9), rtol=1e-6, atol=1e-4)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("v", [5003, 40001])  # whole rows, and rows cut into parts
@pytest.mark.parametrize("allowed", [908, 909, 1000, 1024, 1025])
@pytest.mark.parametrize("top", [50, 64])
def test_allowed_tokens_in_one_place(lib, top, allowed, v, dtype):
    """A mask of consecutive tokens, which lie in fewer groups of threads than alternatives are asked for; the list
    has 1,024 places, and up to 2 top + 16 of the masked ones are added to it."""
    g = torch.Generator().manual_seed(allowed + top)
    x = torch.full((2, v), -INF).to(dtype)
    x[0, 1600 : 1600 + allowed] = torch.randn(allowed, generator=g).to(dtype)
    x[1, v - 3 - allowed : v - 3] = torch.randn(allowed, generator=g).to(dtype)
    check(lib, x, top)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("v", [5003, 40001])
@pytest.mark.parametrize("kind", ["rising", "stairs", "few", "nan"])
def test_rows_a_piece_at_a_time(lib, kind, v, dtype):
    """Rows with more candidates than the list holds."""
    i = torch.arange(v)
    x = (i / 10000).expand(2, v).to(dtype).contiguous()
    if kind == "stairs":  # ties past the threshold
        x[:] = (i // 1500).to(dtype)
    elif kind == "few":
        x[:] = -INF
        x[:, v - 1500 :] = torch.randn(1500, generator=torch.Generator().manual_seed(1)).to(dtype)
    elif kind == "nan":  # (the order counts: no row with a NaN has log probabilities)
        x[:, ::3] = float("nan")
        got = run(lib, x, torch.zeros(2, dtype=torch.int64), 20)
        assert all(bool(torch.isnan(a).all()) for a in got[:3])
        order = torch.sort(x.float().nan_to_num(nan=-INF), dim=-1, descending=True, stable=True).indices[:, :20]
        assert torch.equal(got[3], order)
        return
    for top in (1, 20, 64):
        check(lib, x, top)
