"""The float64 restatements of the vocabulary operators, on the CPU: the
distillation gradient against central differences, its limits against the plain
Kullback-Leibler divergence, the sampler's filters on hand-made rows and its draw
against the probabilities; and what the entry points refuse."""

from __future__ import annotations

import ctypes as C
import os

import numpy as np
import pytest

from oracle import vocab_oracle as O


def _case(seed, V, K, listed_mass=0.7):
    rng = np.random.default_rng(seed)
    teacher = rng.standard_normal(V) * 2
    values, idx, lse = O.top_logits(teacher, K)
    return rng.standard_normal(V) * 1.5, values, idx, lse


@pytest.mark.parametrize("tail,reverse", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("temperature", [1.0, 0.7, 3.0])
def test_distill_gradient_matches_differences(tail, reverse, temperature):
    z, t, idx, _ = _case(3, 23, 6)
    teacher = np.random.default_rng(3).standard_normal(23) * 2
    t, idx, lse = O.top_logits(teacher, 6, temperature)
    kw = dict(lse=lse if tail else None, temperature=temperature, reverse=reverse, weight=1.3)
    _, g = O.distill(z, t, idx, **kw)
    h = 1e-6
    num = np.empty_like(z)
    for j in range(z.size):
        e = np.zeros_like(z)
        e[j] = h
        num[j] = (O.distill(z + e, t, idx, **kw)[0] - O.distill(z - e, t, idx, **kw)[0]) / (2 * h)
    np.testing.assert_allclose(g, num, rtol=1e-6, atol=1e-8)


def test_distill_of_everything_listed_is_the_full_divergence():
    rng = np.random.default_rng(0)
    z, teacher = rng.standard_normal(17), rng.standard_normal(17)
    t, idx, lse = O.top_logits(teacher, 17)
    lp, lq = teacher - O.logsumexp(teacher), z - O.logsumexp(z)
    full = (np.exp(lp) * (lp - lq)).sum()
    for kw in (dict(), dict(lse=lse)):
        loss, g = O.distill(z, t, idx, **kw)
        assert loss == pytest.approx(full, rel=1e-12)
        np.testing.assert_allclose(g, np.exp(lq) - np.exp(lp), atol=1e-14)
    loss, _ = O.distill(z, t, idx, lse=lse, reverse=True)
    assert loss == pytest.approx((np.exp(lq) * (lq - lp)).sum(), rel=1e-12)


def test_distill_rows_without_a_teacher_cost_nothing():
    z = np.random.default_rng(1).standard_normal(9)
    for kw in (dict(), dict(lse=0.3), dict(lse=0.3, reverse=True)):
        loss, g = O.distill(z, [5.0, 5.0], [-1, -7], **kw)
        assert loss == 0 and not g.any()
    loss, g = O.distill(np.full(9, np.nan), [5.0], [2], weight=0.0)
    assert loss == 0 and not g.any()


def test_sample_filters_on_hand_made_rows():
    z = np.log([0.4, 0.3, 0.2, 0.1])
    one = np.ones(4)
    pick = lambda token: np.where(np.arange(4) == token, 1e-9, 1.0)  # noqa: E731
    assert O.sample(z, one)[0] == 0
    assert O.sample(z, pick(3))[:1] == (3,)
    assert O.sample(z, pick(3), top_k=3)[0] == 0
    assert O.sample(z, pick(2), top_p=0.71)[0] == 2
    assert O.sample(z, pick(2), top_p=0.69)[0] == 0
    assert O.sample(z, pick(1), top_p=0.0)[0] == 0
    assert O.sample(z, pick(2), min_p=0.51)[0] == 0
    assert O.sample(z, pick(2), min_p=0.49)[0] == 2
    assert O.sample(z, pick(2), top_k=3)[1] == pytest.approx(np.log(0.2 / 0.9))
    assert O.sample(z, pick(3), temperature=0)[:2] == (0, 0.0)
    assert O.sample(np.full(4, -np.inf), one)[0] == -1
    assert O.sample(np.array([1.0, 1.0, 0.0, 1.0]), pick(3), top_k=2)[0] == 0


def test_sample_draws_by_weight():
    rng = np.random.default_rng(5)
    z = np.array([0.0, 1.0, -1.0, 2.0])
    p = np.exp(z - O.logsumexp(z))
    n = 4000
    count = np.bincount([O.sample(z, rng.exponential(size=4))[0] for _ in range(n)], minlength=4)
    # five standard deviations of a binomial count
    assert np.all(np.abs(count - n * p) < 5 * np.sqrt(n * p * (1 - p)))


# ---------------------------------------------------------------------------
# refusals: all before any CUDA call
# ---------------------------------------------------------------------------
@pytest.fixture(scope="module")
def lib():
    from matrix_b200 import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from matrix_b200 import build
        build.build()
    return _lib.load()


def _dims(**kw):
    from matrix_b200 import _lib
    d = dict(rows=2, rows_inner=2, stride_outer=0, stride_inner=64, V=64, dtype=0)
    d.update(kw)
    return _lib.LogitsDims(**d)


@pytest.mark.parametrize("bad,code", [(dict(dtype=7), -1), (dict(V=0), -1), (dict(rows=-1), -1),
                                      (dict(rows_inner=0), -1), (dict(stride_inner=-64), -1),
                                      (dict(stride_outer=-1), -1), (dict(V=393217), -2),
                                      (dict(rows=1 << 31), -2)])
def test_bad_logits_are_refused(lib, bad, code):
    from matrix_b200 import _lib
    d, p = _dims(**bad), C.c_void_p(256)
    assert lib.dwa_top_logits(None, d, p, 1, 1.0, p, p, p) == code
    assert lib.dwa_distill_fwd(None, d, _lib.DistillDims(1, 0, 1.0, 0), p, p, p, None, None, p, None, None, p, 256) == code
    assert lib.dwa_distill_bwd(None, d, _lib.DistillDims(1, 0, 1.0, 0), p, p, p, None, None, p, p, 1, p) == code
    assert lib.dwa_sample_tokens(None, d, _lib.SampleParams(), p, p, 64, p, p) == code
    assert _lib.last_error()


@pytest.mark.parametrize("k,t,code", [(0, 1.0, -1), (65, 1.0, -1), (4, 0.0, -1), (4, -1.0, -1), (4, float("nan"), -1),
                                      (4, float("inf"), -1)])
def test_bad_top_and_distill_options_are_refused(lib, k, t, code):
    from matrix_b200 import _lib
    d, p = _dims(), C.c_void_p(256)
    assert lib.dwa_top_logits(None, d, p, k, t, p, p, p) == code
    o = _lib.DistillDims(k, 0, t, 0)
    assert lib.dwa_distill_fwd(None, d, o, p, p, p, None, None, p, None, None, p, 256) == code
    assert lib.dwa_distill_bwd(None, d, o, p, p, p, None, None, p, p, 1, p) == code


def test_other_refusals(lib):
    from matrix_b200 import _lib
    p, odd = C.c_void_p(256), C.c_void_p(257)
    big = _dims(V=2048, stride_inner=2048)
    assert lib.dwa_top_logits(None, big, p, 1025, 1.0, p, p, p) == -2
    assert lib.dwa_distill_fwd(None, big, _lib.DistillDims(1025, 0, 1.0, 0), p, p, p, None, None, p, None, None, p, 256) == -2
    d, o = _dims(), _lib.DistillDims(4, 0, 1.0, 0)
    assert lib.dwa_distill_fwd(None, d, _lib.DistillDims(4, 0, 1.0, 1), p, p, p, None, None, p, None, None, p, 256) == -1
    assert "reverse" in _lib.last_error()
    assert lib.dwa_distill_fwd(None, d, _lib.DistillDims(4, 9, 1.0, 0), p, p, p, None, None, p, None, None, p, 256) == -1
    assert lib.dwa_distill_fwd(None, d, o, p, p, p, None, None, p, None, None, None, 0) == -4
    assert lib.dwa_distill_fwd(None, d, o, p, p, p, None, None, p, None, None, odd, 256) == -4
    assert lib.dwa_distill_fwd(None, d, o, p, p, p, None, None, p, None, None, p, 8) == -4
    for args in ((None, p, p), (p, None, p), (p, p, None)):
        assert lib.dwa_distill_fwd(None, d, o, *args, None, None, p, None, None, p, 256) == -1
    assert lib.dwa_distill_fwd(None, d, o, odd, p, p, None, None, p, None, None, p, 256) == -1
    assert lib.dwa_distill_bwd(None, d, o, p, p, p, None, None, None, p, 1, p) == -1
    assert lib.dwa_top_logits(None, d, None, 4, 1.0, p, p, p) == -1
    assert lib.dwa_top_logits(None, d, odd, 4, 1.0, p, p, p) == -1
    s = _lib.SampleParams()
    assert lib.dwa_sample_tokens(None, d, None, p, p, 64, p, p) == -1
    assert lib.dwa_sample_tokens(None, d, s, p, p, -1, p, p) == -1
    assert lib.dwa_sample_tokens(None, d, s, p, None, 64, p, p) == -1
    assert lib.dwa_sample_tokens(None, d, s, p, C.c_void_p(258), 64, p, p) == -1
    none = _dims(rows=0)
    assert lib.dwa_top_logits(None, none, None, 4, 1.0, None, None, None) == 0
    assert lib.dwa_distill_fwd(None, none, o, None, None, None, None, None, None, None, None, None, 0) == 0
    assert lib.dwa_sample_tokens(None, none, s, None, None, 64, None, None) == 0


def test_cpu_tensors_are_refused():
    torch = pytest.importorskip("torch")
    from matrix_b200.distill import distill_loss, top_logits
    from matrix_b200.sampling import sample_tokens
    z = torch.randn(2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        top_logits(z, 2)
    with pytest.raises(ValueError, match="CUDA"):
        distill_loss(z, z[:, :2], torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        sample_tokens(z, z)


def test_row_layouts_of_views():
    """logits_view on meta tensors: what is read in place and with which strides."""
    torch = pytest.importorskip("torch")
    from matrix_b200 import runtime

    class OnGpu(torch.Tensor):
        is_cuda = True

    def layout(t):
        v, d = runtime.logits_view("logits", t.as_subclass(OnGpu))
        return v.data_ptr() == t.data_ptr(), d.rows, d.rows_inner, d.stride_outer, d.stride_inner

    x = torch.zeros(3, 5, 16)
    assert layout(x) == (True, 15, 15, 0, 16)
    assert layout(x[:, :-1]) == (True, 12, 4, 80, 16)
    assert layout(x[:, 1:]) == (True, 12, 4, 80, 16)
    assert layout(x[..., :13]) == (True, 15, 15, 0, 16)
    assert layout(x[:, 2]) == (True, 3, 3, 0, 80)
    assert layout(x[1, 2]) == (True, 1, 1, 0, 16)
    assert layout(x[:, :, ::2])[0] is False
    assert layout(x.transpose(0, 1)) == (True, 15, 3, 16, 80)
    assert layout(torch.zeros(16).expand(4, 16)) == (True, 4, 4, 0, 0)
    y = torch.zeros(2, 3, 4, 16)[:, :2, :3]
    assert layout(y)[0] is False
    assert layout(x[:0])[1] == 0
