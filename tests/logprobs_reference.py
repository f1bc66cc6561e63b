"""Log probabilities and entropies in 64 bits, on the CPU, and how far those of
``token_logprobs`` may be off, from the roundings on a weight's way to the row's sums.

With u = 2^-24, t_i = x_i - max x, pi_i the probabilities, T1 = sum pi |t|, T2 = sum pi t^2:

* A weight exp2(t log2 e) is off by 2 u of itself (the exponential) and 2.5 u |t| (t, the
  constant and the product); the largest logit's is 1.
* It is added to a piece (8 at most), a tile (8 pieces and an edge), a row's tiles, 64
  lanes (6 levels), 4 waves (3) and 12 parts (6): no addition is off by more than u of the
  sum, and those of nothing but zeros are exact, so no more count than there are logits
  above -inf. The form for other strides adds a thread's V / 256 one after the other.
* Sums move to a new largest logit: 3 u of the weights before it (exponential, product).
  That happens at most once a piece of a tile, once a tile and once a join; and at each of
  the five levels no more often than the row has other values.
* The weighted sum takes the same, and 2.5 u and two roundings a move for its terms.
* logf is off by 4 u of itself, a difference or a quotient by u.

And whatever the sizes: no log probability is above 0, no entropy below."""

import torch

U = 2.0**-24


def reference(x, tokens):
    """(log probabilities of all logits, entropies, tolerance of the logarithm of the sum, of the entropies)."""
    x = x.double().cpu()
    t = x - x.amax(-1, keepdim=True)
    lse = t.exp().sum(-1).log()
    logp = t - lse[:, None]
    pi = logp.exp()
    entropy = -torch.where(pi > 0, pi * logp, 0.0).sum(-1)
    t = torch.where(pi > 0, t, 0.0)
    return logp, entropy, lse, (pi * t.abs()).sum(-1), (pi * t * t).sum(-1), 1 - pi.amax(-1)


def near(x, tokens, got, what, side_by_side=True):
    """Asserts that got = (logprobs, entropy, top_logprobs, top_tokens) of finite rows x is as near as it has to be."""
    logp, entropy, lse, t1, t2, rest = reference(x, tokens)
    v = x.shape[1]
    row = x.double().cpu()
    finite = torch.isfinite(row).sum(-1).double()
    values = torch.tensor([r[torch.isfinite(r)].unique().numel() for r in row], dtype=torch.float64)
    if side_by_side:
        tiles = -(-v * x.element_size() // (16 * 2048))
        adds, moves = 31 + tiles, 24 + tiles
    else:
        adds, moves = -(-v // 256) + 9, 0
    adds = torch.minimum(finite - 1, torch.tensor(float(adds)))
    moves = torch.minimum(5 * (values - 1), torch.tensor(float(moves)))
    rel = U * (adds + (2 + 3 * moves) * rest + 2.5 * t1)
    tol = rel + 4 * U * lse
    tol_entropy = tol + t1 * rel + U * ((adds + 5 * moves + 12) * t1 + 5 * t2) + U * entropy

    own, h, top_logp, top_tokens = (a.cpu() for a in got)
    own_ref = logp.gather(1, tokens.cpu().long()[:, None])[:, 0]
    top_ref = logp.gather(1, top_tokens)
    for name, a, b, e in (("logprobs", own, own_ref, tol + 2 * U * own_ref.abs()), ("entropy", h, entropy, tol_entropy),
                          ("top_logprobs", top_logp, top_ref, tol[:, None] + 2 * U * top_ref.abs())):
        none = torch.isneginf(b)
        assert torch.equal(torch.isneginf(a), none), f"{what}: {name}, infinities"
        err = torch.where(none, 0.0, (a.double() - b).abs().nan_to_num(1e30))
        share = float((err / e.nan_to_num(posinf=1.0)).max()) if err.numel() else 0.0
        print(f"{what}: {name} off by {float(err.max()) if err.numel() else 0:.1e}, {share:.2f} of what it may be", flush=True)
        assert share <= 1, f"{what}: {name} off by {float(err.max()):.2e}, {share:.2f} of what it may be"
    assert not bool((own > 0).any()) and not bool((top_logp > 0).any()), f"{what}: a log probability above 0"
    assert not bool((h < 0).any()), f"{what}: an entropy below 0"


def rows(kind, n, v, dtype, device, seed=0):
    """(rows, tokens): `few`, two to four allowed tokens 0 to 20 apart anywhere; `one_thread`, two allowed tokens of one
    thread, the lower one 0 to 20 below and in an earlier 16-byte piece; `sure`, one token 10 to 16 above all
    others, late in the row; `even`, the whole vocabulary at two values, as a flat distribution; `plain`, normal ones."""
    g = torch.Generator().manual_seed(seed + n + v)
    best = v - 1 - torch.randint(max(v // 3, 1), (n,), generator=g)
    if kind == "few":
        x = torch.full((n, v), float("-inf"))
        for i in range(n):
            at = torch.randperm(v, generator=g)[: 2 + i % 3]
            x[i, at] = 20 * torch.rand(len(at), generator=g) - 5
            best[i] = at[x[i, at].argmax()]
    elif kind == "one_thread":
        x = torch.full((n, v), float("-inf"))
        a = torch.randint(2048, (n,), generator=g)
        best = a + 2048 * torch.randint(1, (v - 2048) // 2048 + 1, (n,), generator=g)
        best = torch.where(best < v, best, a + 2048)
        x[torch.arange(n), a] = 1.0
        x[torch.arange(n), best] = 1 + 20 * torch.rand(n, generator=g)
    elif kind == "sure":
        x = torch.randn(n, v, generator=g)
        x[torch.arange(n), best] = x.amax(-1) + 10 + 6 * torch.rand(n, generator=g)
    elif kind == "even":
        x = torch.where(torch.arange(v) % 2 == 0, 1.0, 1.0 - 0.4375 - 0.03125 * torch.arange(n)[:, None])
    else:
        x = 3 * torch.randn(n, v, generator=g)
    return x.to(dtype).to(device), best.to(device)
