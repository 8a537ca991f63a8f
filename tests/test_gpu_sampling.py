"""Sampling on the GPU against the float64 oracle.

An fp32 weight is within 40 * 2^-23 = 5e-6 (relative) of its value.  So the token
is the oracle's wherever the winning score leads by MARGIN = 1e-5; where moving a
cut by MARGIN of the mass changes the oracle's token, either of the two is right.
The log-probability, a logarithm of a sum of such weights and a difference of
logits, is held to TOL = 2e-5, beside what moving the cut changes in it."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import vocab_oracle as O

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TOL, MARGIN = 2e-5, 1e-5


def _rand(rows, V, seed, dtype=F32, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, V, generator=g) * scale).to(dtype).cuda()


def _noise(*shape, seed=0):
    return torch.empty(shape).exponential_(generator=torch.Generator().manual_seed(seed)).cuda()


def _rows(value, n):
    return value.reshape(-1).cpu().tolist() if isinstance(value, torch.Tensor) else [value] * n


def _check(z, noise, **kw):
    """Compares every row; at least nine in ten have to be beyond doubt in the race."""
    from matrix_b200.sampling import sample_tokens
    tokens, logprobs = sample_tokens(z, noise, **kw)
    assert tokens.dtype == torch.int32 and logprobs.dtype == F32
    assert tokens.shape == logprobs.shape == z.shape[:-1]
    n = tokens.numel()
    zz = z.double().cpu().numpy().reshape(n, -1)
    ee = noise.double().cpu().numpy().reshape(n, -1)
    names = (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))
    par = {k: _rows(kw.get(k, d), n) for k, d in names}
    tokens, logprobs, seen = tokens.reshape(-1).tolist(), logprobs.reshape(-1).tolist(), 0
    for r in range(n):
        args = {k: float(np.float32(v[r])) if k != "top_k" else v[r] for k, v in par.items()}
        want = [O.sample(zz[r], ee[r], **args, shift=s) for s in (-MARGIN, 0.0, MARGIN)]
        if want[1][2] < MARGIN:
            continue
        seen += 1
        assert tokens[r] in [w[0] for w in want], f"row {r}: token {tokens[r]}, expected {want} ({args})"
        lps = [w[1] for w in want if w[0] == tokens[r]]
        off = min(lps) - logprobs[r], logprobs[r] - max(lps)
        assert np.isnan(lps[0]) == np.isnan(logprobs[r]), f"row {r}"
        assert np.isnan(lps[0]) or max(off) <= TOL * (1 + abs(lps[0])), f"row {r}: {logprobs[r]}, expected {lps} ({args})"
    assert seen >= 0.9 * n


FILTERS = [dict(), dict(temperature=0.7), dict(temperature=0.0), dict(temperature=-1.0), dict(top_k=1), dict(top_k=5),
           dict(top_k=50, top_p=0.9), dict(top_k=3000), dict(top_k=3000, top_p=0.99, min_p=1e-4), dict(top_p=0.5),
           dict(top_p=0.0), dict(top_p=0.999), dict(min_p=0.1), dict(min_p=1.0), dict(min_p=2.0),
           dict(temperature=1.3, top_k=200, top_p=0.95, min_p=0.02), dict(temperature=50.0, top_p=0.9),
           dict(temperature=1e-3), dict(top_k=-1, top_p=2.0, min_p=-1.0), dict(top_k=10 ** 9)]


@pytest.mark.parametrize("kw", FILTERS, ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()) or "none")
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,V", [(3, 1), (4, 2), (6, 9), (20, 300), (12, 4097), (3, 40000), (1, 131072)])
def test_filters(rows, V, dtype, kw):
    _check(_rand(rows, V, V, dtype), _noise(rows, V, seed=V), **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [1000, 50001])
def test_a_batch_of_unlike_requests(V, dtype):
    n = 64
    g = torch.Generator().manual_seed(V)
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (n,), generator=g)].cuda()  # noqa: E731
    _check(_rand(n, V, 5, dtype, 3.0), _noise(n, V, seed=5), temperature=pick(0.0, 0.5, 1.0, 1.5),
           top_k=pick(0, 1, 20, 300, 5000).int(), top_p=pick(1.0, 0.3, 0.9, 0.99), min_p=pick(0.0, 0.0, 0.05, 0.5))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=4), dict(top_k=4, top_p=0.6), dict(top_p=0.6), dict(min_p=0.3),
                                dict(temperature=0.0), dict(top_k=2000, top_p=0.4)])
@pytest.mark.parametrize("V", [9, 6000, 40000])
def test_odd_rows(V, kw, dtype):
    """Rows of one value, few values, masks that leave one entry or none, infinities, NaN, the types' ends."""
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(V)
    z = torch.randn(12, V, generator=g)
    z[0] = -2.5
    z[1] = torch.randint(0, 3, (V,), generator=g).float()
    z[2] = -torch.inf
    z[3] = -torch.inf
    z[3, V // 2] = -7.0
    z[4] = low
    z[4, 3], z[4, V - 1] = 1.0, 1.0
    z[5] = low
    z[6, V // 3] = torch.nan
    z[7, 2], z[7, V - 1] = torch.inf, torch.inf
    z[8, ::2], z[8, 1::2] = 0.0, -0.0
    z[9] = torch.where(torch.rand(V, generator=g) < 0.5, -torch.inf, z[9])
    z[10] = torch.finfo(dtype).max
    z[11, 1] = torch.nan
    z[11, 2] = torch.inf
    _check(z.to(dtype).cuda(), _noise(12, V, seed=V), **kw)


def test_views_and_parameters():
    x = _rand(20, 1003, 0, BF16).view(4, 5, 1003)
    e = _noise(4, 5, 1003)
    _check(x[:, -1], e[:, -1], top_k=20)
    _check(x[:, :-1], e[:, :-1], top_p=0.9)
    _check(x[..., 1:], e[..., 1:], temperature=0.8)
    _check(x[..., :777], e[..., :777], temperature=0.8)
    _check(x[0, 0], e[0, 0])
    _check(x[0, 0].expand(6, 1003), e.view(20, 1003)[:6])
    _check(x[:, 0], e[0, 0].expand(4, 1003))
    _check(x[:, :, ::2], e[:, :, ::2])
    t = torch.linspace(0.5, 2, 20).cuda().view(4, 5)
    _check(x, e, temperature=t, top_k=torch.full((4, 5), 30, dtype=torch.int32, device="cuda"))


def test_noise_of_any_kind():
    """A number of zero wins, an infinite one loses; without a usable one there is no token."""
    from matrix_b200.sampling import sample_tokens
    z = torch.zeros(4, 100, device="cuda")
    e = torch.ones(4, 100, device="cuda")
    e[0, 37] = e[0, 90] = 0.0
    e[1] = torch.inf
    e[1, 55] = 3.0
    e[2] = torch.nan
    e[3, :99] = torch.nan
    tokens, logprobs = sample_tokens(z, e)
    assert tokens.tolist() == [37, 55, -1, 99]
    assert torch.isnan(logprobs).tolist() == [False, False, True, False]
    z[:, 10:] = -torch.inf
    e = torch.ones(4, 100, device="cuda")
    e[:, 50] = 0.0            # a masked entry stays out whatever its number
    assert sample_tokens(z, e)[0].tolist() == [0, 0, 0, 0]


def test_draws_by_weight():
    """20000 draws from a row of 50: counts within five standard deviations."""
    from matrix_b200.sampling import sample_tokens
    n, V = 20000, 50
    z = _rand(1, V, 3)
    tokens, _ = sample_tokens(z.expand(n, V), _noise(n, V, seed=11), top_k=40)
    top = torch.topk(z[0], 40).indices
    p = torch.zeros(V, device="cuda").scatter(0, top, torch.softmax(z[0, top], -1)).cpu()
    count = torch.bincount(tokens.long(), minlength=V).cpu()
    assert torch.all((count - n * p).abs() <= 5 * torch.sqrt(n * p * (1 - p)) + 1e-3)


def test_streams_graph_and_repeats():
    from matrix_b200.sampling import sample_tokens
    z, e = _rand(33, 70001, 0, BF16), _noise(33, 70001)
    kw = dict(temperature=0.9, top_k=100, top_p=0.9)
    want = sample_tokens(z, e, **kw)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(want, sample_tokens(z, e, **kw)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sample_tokens(z, e, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample_tokens(z, e, **kw)
    z.copy_(_rand(33, 70001, 1, BF16))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, sample_tokens(z, e, **kw)))
    # a row's token does not depend on its neighbours
    alone = [sample_tokens(z[r], e[r], **kw) for r in (0, 16, 32)]
    both = sample_tokens(z, e, **kw)
    assert [int(a[0]) for a in alone] == [int(both[0][r]) for r in (0, 16, 32)]


def test_refusals():
    from matrix_b200.sampling import sample_tokens
    z, e = _rand(4, 64, 0), _noise(4, 64)
    with pytest.raises(ValueError):
        sample_tokens(z, e[:, :63])
    with pytest.raises(ValueError):
        sample_tokens(z, e.cpu())
    with pytest.raises(TypeError):
        sample_tokens(z, e.double())
    with pytest.raises(TypeError):
        sample_tokens(z.half(), e)
    with pytest.raises(ValueError):
        sample_tokens(z, e, top_p=torch.ones(3, device="cuda"))
    with pytest.raises(TypeError):
        sample_tokens(z, e, top_k=torch.ones(4, device="cuda"))
    with pytest.raises(ValueError):
        sample_tokens(z, e, min_p=torch.ones(4))
    tokens, logprobs = sample_tokens(z[:0], e[:0])
    assert tokens.shape == logprobs.shape == (0,)
