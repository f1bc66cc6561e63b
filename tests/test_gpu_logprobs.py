"""Log probabilities of tokens, entropy and the most likely tokens against 64 bits:
vocabularies of one to 151,936, types, ties, masked rows, rows without a
distribution, sorted rows (every logit a candidate), strides and alignments.

Tolerance, derived. With t = x - m (rounded once, 2^-24 |t|), a weight exp(t) is off
by 2^-24 |t| + 2^-22 of itself, which over a row's sum is at most 2^-22 + 2^-24 of
it for the terms that count (exp(t) |t| <= 0.37), and the sum of V terms, of which
no one partial sum holds more than V / 64 + 64, by (V / 64 + 64) 2^-24. ln S then is
off by that and its own 2^-22 |ln S|; the entropy by as much of |E / S|."""

import pytest
import torch

from tinyserver_amd.kernels import token_logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _reference(x, tokens, top):
    x = x.double().cpu()
    m = x.amax(-1, keepdim=True)
    lse = (x - m).exp().sum(-1, keepdim=True).log()
    logp = (x - m) - lse
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    tokens = tokens.cpu().long()
    inside = (tokens >= 0) & (tokens < x.shape[1])
    own = torch.where(inside, logp.gather(1, tokens.clamp(0, x.shape[1] - 1)[:, None])[:, 0], float("-inf"))
    return own, entropy, logp.gather(1, order), order, lse[:, 0]


def _check(x, tokens, top, what):
    n, v = x.shape
    own, entropy, top_logp, order, lse = _reference(x, tokens, top)
    got = token_logprobs(x, tokens, top)
    e = 2.0**-21 + (v / 64 + 64) * 2.0**-24

    def near(a, b, tol, name):
        a = a.double().cpu()
        inf = torch.isinf(b)
        assert torch.equal(a[inf], b[inf]), f"{what}: {name}, infinities"
        err = torch.where(inf, 0.0, (a - b).abs().nan_to_num(1e30))
        print(f"{what}: {name} max_abs={float(err.max()) if err.numel() else 0:.1e}", flush=True)
        assert bool((err <= tol).all()), f"{what}: {name}, {float((err / tol).max()):.2f} of the tolerance"

    size = e + 2.0**-22 * lse.abs()
    near(got.logprobs, own, size + 2.0**-22 * own.abs().nan_to_num(posinf=0), "logprobs")
    near(got.entropy, entropy, 2 * size + (e + 2.0**-22) * entropy.abs(), "entropy")
    assert got.top_tokens.dtype == torch.int64 and torch.equal(got.top_tokens.cpu(), order), f"{what}: top tokens"
    near(got.top_logprobs, top_logp, size[:, None] + 2.0**-22 * top_logp.abs().nan_to_num(posinf=0), "top_logprobs")


def _rows(n, v, dtype, seed=0, size=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed + n + v)
    x = (size * torch.randn(n, v, generator=g, device=DEV)).to(dtype)
    return x, torch.randint(v, (n,), generator=g, device=DEV)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("n,v,top", [
    (1, 1, 1), (3, 2, 2), (5, 7, 0), (4, 8, 8), (3, 63, 20), (2, 64, 64), (7, 65, 5), (1, 1000, 1), (9, 1003, 64),
    (33, 4096, 20), (2, 8191, 20), (300, 2049, 5), (1, 16391, 50), (70, 151936, 20), (3, 151936, 64), (1, 151935, 5),
])
def test_shapes(dtype, n, v, top):
    x, tokens = _rows(n, v, dtype)
    _check(x, tokens, top, f"{n} x {v}, {dtype}")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "masked", "zeros", "two", "stairs", "last", "peaks"])
@pytest.mark.parametrize("n,v", [(2, 151936), (600, 5003)])
def test_ties_and_orders(kind, n, v, dtype):
    """Rows in which many logits reach the last place, or every one is larger than all before it."""
    x, tokens = _rows(n, v, dtype, 3)
    i = torch.arange(v, device=DEV)
    if kind == "equal":
        x[:] = 1.5
    elif kind == "rising":
        x[:] = (i / 10000).to(dtype)
    elif kind == "falling":
        x[:] = (-i / 10000).to(dtype)
    elif kind == "masked":  # fewer allowed tokens than alternatives
        x[:, (i % 30011) != 7] = float("-inf")
        tokens[: n // 2] = 7
    elif kind == "zeros":
        x[:] = torch.where(i % 3 == 0, -0.0, 0.0).to(dtype)
    elif kind == "two":
        x[:] = -30.0
        x[:, v // 2] = x[:, -1] = 30.0
    elif kind == "stairs":
        x[:] = (i // 64 % 5).to(dtype)
    elif kind == "last":
        x[:, -70:] = 90.0
    else:  # all the largest in one place of the row
        x[:, v // 3 : v // 3 + 500] += 20.0
    for top in (1, 20, 64):
        _check(x, tokens, top, f"{kind}, {n} x {v}, top {top}, {dtype}")


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_strides_and_alignment(dtype):
    x, tokens = _rows(6, 5008, dtype, 5)
    wide = torch.randn(6, 5100, device=DEV).to(dtype)
    for off in (0, 1, 2, 3, 5, 8):
        _check(wide[:, off : off + 4999], tokens % 4999, 20, f"offset {off}, {dtype}")
    _check(x[:, ::2], tokens % 2504, 20, "every second")
    _check(x.t().contiguous().t(), tokens, 20, "columns first")
    _check(x[::2], tokens[::2], 5, "every second row")
    _check(x[:1].expand(6, -1), tokens.int(), 5, "one row for all")
    odd = torch.randn(9 * 1003 + 1, device=DEV).to(dtype)[1:].view(9, 1003)
    _check(odd, tokens[:1].expand(9) % 1003, 9, "odd rows")


@pytest.mark.parametrize("v", [5, 1003, 151936])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_without_a_distribution(v, dtype):
    x, tokens = _rows(6, v, dtype, 9)
    x[0, v // 2] = float("nan")
    x[1, v - 1] = float("inf")
    x[2] = float("-inf")
    x[3] = float("nan")
    clean = token_logprobs(x[4:], tokens[4:], 4)
    got = token_logprobs(x, tokens, 4)
    for a in (got.logprobs[:4], got.entropy[:4], got.top_logprobs[:4]):
        assert bool(torch.isnan(a).all())
    assert all(torch.equal(a[4:], b) for a, b in zip(got, clean))
    y = torch.where(torch.isnan(x[0]), float("-inf"), x[0].float())
    assert got.top_tokens[0].tolist() == torch.sort(y, descending=True, stable=True).indices[:4].tolist()
    assert got.top_tokens[1, 0].item() == v - 1
    assert got.top_tokens[2].tolist() == got.top_tokens[3].tolist() == [0, 1, 2, 3]
    few = torch.full((1, v), float("nan"), device=DEV).to(dtype)
    few[0, v - 2] = 1.0
    assert token_logprobs(few, tokens[:1], 4).top_tokens[0].tolist() == [v - 2, 0, 1, 2]


def test_tokens_outside_the_vocabulary():
    x, _ = _rows(4, 1003, BF)
    got = token_logprobs(x, torch.tensor([-1, 1003, 1 << 40, 5], device=DEV), 2)
    assert got.logprobs[:3].tolist() == [float("-inf")] * 3 and bool(torch.isfinite(got.logprobs[3]))
    assert bool(torch.isfinite(got.entropy).all())


def test_large_values():
    """Logits past the exponential's range, far apart or all far from 0."""
    x, tokens = _rows(5, 4097, F32, 2, size=300.0)
    _check(x, tokens, 20, "far apart")
    _check(x / 100 + 60000.0, tokens, 20, "far from 0")
    _check(x / 100 - 3e38, tokens, 5, "near the lowest")
    y = x.clone()
    y[:, 1::2] = torch.finfo(torch.float32).min
    _check(y, tokens // 2 * 2, 20, "the lowest value as a mask")


def test_nothing_to_do():
    got = token_logprobs(torch.zeros(0, 50, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV), 3)
    assert [tuple(x.shape) for x in got] == [(0,), (0,), (0, 3), (0, 3)]


def test_graph_replays():
    x, tokens = _rows(3, 151936, BF, 1)
    token_logprobs(x, tokens, 20)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):  # two graphs, run in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(token_logprobs(x, tokens, 20))
        graphs.append(graph)
    for seed in range(4):
        y, t = _rows(3, 151936, BF, 10 + seed)
        x.copy_(y)
        tokens.copy_(t)
        for graph in graphs:
            graph.replay()
        want = token_logprobs(y, t, 20)
        torch.cuda.synchronize()
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
