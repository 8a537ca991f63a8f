"""A teacher's top logits and the distillation loss on the GPU against the float64
oracle.

Tolerances, from the arithmetic: a weight exp2((z - m) c) carries two roundings
of an argument of at most 40, 40 * 2^-23 = 5e-6 relative, and a thread's sum of
at most 2048 of them 2048 * 2^-24 in the worst order but a few 2^-24 in fact:
RTOL = 2e-5 covers both.  A loss is a sum of p (log p - log q), each logarithm
off by that much: RTOL * (1 + |L|).  A gradient entry is a difference of two such
weights: RTOL times the largest entry, and half a unit of bf16 (2^-8 relative)
where it is stored in 16 bits.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import vocab_oracle as O

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

RTOL = 2e-5
F32, BF16 = torch.float32, torch.bfloat16


def _rand(rows, V, seed, dtype=F32, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, V, generator=g) * scale).to(dtype).cuda()


def _np(t):
    return t.detach().double().cpu().numpy()


def _check_top(z, k, temperature=1.0):
    from matrix_b200.distill import top_logits
    values, indices, lse = top_logits(z, k, temperature=temperature)
    assert values.dtype == z.dtype and indices.dtype == torch.int32 and lse.dtype == F32
    assert values.shape == indices.shape == (*z.shape[:-1], k) and lse.shape == z.shape[:-1]
    zz = _np(z).reshape(-1, z.shape[-1])
    values, indices, lse = _np(values).reshape(-1, k), indices.reshape(-1, k).cpu().numpy(), _np(lse).reshape(-1)
    for r, row in enumerate(zz):
        v, i, l = O.top_logits(row, k, temperature)
        np.testing.assert_array_equal(indices[r], i)
        np.testing.assert_array_equal(values[r], v)
        np.testing.assert_allclose(lse[r], l, rtol=RTOL, atol=RTOL)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (4, 8, 8), (4, 9, 1), (3, 257, 200),
                                      (2, 1024, 1024), (9, 4097, 64), (2, 33001, 1024), (40, 5003, 20),
                                      (200, 2048, 50), (2, 131072, 64), (1, 262147, 300)])
def test_top_logits(rows, V, k, dtype):
    _check_top(_rand(rows, V, rows + V, dtype), k, 1.0 if V % 2 else 0.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,k", [(9, 4), (5000, 70), (40000, 1024)])
def test_top_logits_of_odd_rows(dtype, V, k):
    """Constant rows, few values, sorted rows, zeros of both signs, infinities, NaN, the types' ends."""
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    g = torch.Generator().manual_seed(V)
    z = torch.randn(11, V, generator=g)
    z[0] = 1.25
    z[1] = torch.randint(0, 3, (V,), generator=g).float()
    z[2] = torch.linspace(-5, 5, V)
    z[3] = torch.linspace(5, -5, V)
    z[4, ::2], z[4, 1::2] = 0.0, -0.0
    z[5] = -torch.inf
    z[6] = -torch.inf
    z[6, V // 2] = 3.0
    z[7, V // 3], z[7, V - 1] = torch.inf, torch.inf
    z[8, 1] = torch.nan
    z[9] = low
    z[9, V - 2] = high
    z[10] = z[10] * 1e-40
    _check_top(z.to(dtype).cuda(), k)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_top_logits_of_views(dtype):
    x = _rand(15, 1003, 0, dtype).view(3, 5, 1003)
    _check_top(x[:, :-1], 20)
    _check_top(x[:, 1:, 1:], 20)
    _check_top(x[..., :700], 20)
    _check_top(x[1, 2], 20)
    _check_top(x.transpose(0, 1), 20)
    _check_top(x[:, :, ::3], 20)
    _check_top(x[:1, :1].expand(2, 4, 1003), 20)
    from matrix_b200.distill import top_logits
    v, i, l = top_logits(x[:0], 4)
    assert v.shape == (0, 5, 4) and i.shape == (0, 5, 4) and l.shape == (0, 5)
    for k in (0, 1004):
        with pytest.raises(Exception):
            top_logits(x, k)


def test_rows_beyond_32_bit_offsets():
    """Two rows 2^31 + 8 elements apart."""
    from matrix_b200.distill import distill_loss_and_grad
    apart, V = 2 ** 31 + 8, 1000
    buf = torch.empty(apart + V, dtype=BF16, device="cuda")
    z = buf.as_strided((2, V), (apart, 1))
    z.copy_(_rand(2, V, 3, BF16))
    _check_top(z, 30)
    idx = torch.tensor([[1, 999], [0, 500]], dtype=torch.int32, device="cuda")
    loss, g = distill_loss_and_grad(z, torch.ones(2, 2, device="cuda"), idx)
    l2, g2 = distill_loss_and_grad(z.contiguous(), torch.ones(2, 2, device="cuda"), idx)
    assert torch.equal(loss, l2) and torch.equal(g, g2)


# ---------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------
MODES = {"listed": dict(tail=False, reverse=False), "tail": dict(tail=True, reverse=False),
         "reverse": dict(tail=True, reverse=True)}


def _teacher(rows, V, k, temperature, seed, dtype=F32):
    """k logits of a random teacher, their indices, and the log-sum-exp of its row."""
    t = _rand(rows, V, seed + 1, dtype)
    v, i = torch.topk(t, k, dim=-1)
    return v, i.int(), torch.logsumexp(t.float() / temperature, -1)


def _expect(z, t, idx, lse, w, temperature, mode):
    out = []
    for r in range(z.shape[0]):
        out.append(O.distill(_np(z[r]), _np(t[r]), idx[r].cpu().numpy(),
                             float(lse[r]) if MODES[mode]["tail"] else None, temperature, MODES[mode]["reverse"],
                             1.0 if w is None else float(w[r])))
    return np.array([o[0] for o in out]), np.stack([o[1] for o in out])


def _kw(mode, lse, temperature, w):
    return dict(teacher_lse=lse if MODES[mode]["tail"] else None, temperature=temperature,
                reverse=MODES[mode]["reverse"], weights=w)


def _close_loss(got, want):
    np.testing.assert_allclose(_np(got).reshape(-1), want, rtol=RTOL, atol=RTOL)


def _close_grad(got, want, scale=1.0):
    half = 2.0 ** -8 if got.dtype == BF16 else 0.0
    g, atol = _np(got).reshape(want.shape), RTOL * scale * np.abs(want[np.isfinite(want)]).max(initial=1e-30)
    np.testing.assert_allclose(g, want, rtol=RTOL + half, atol=atol)


@pytest.mark.parametrize("mode", list(MODES))
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,V,k,temperature", [(1, 1, 1, 1.0), (2, 2, 1, 1.0), (3, 9, 9, 2.0), (5, 17, 4, 0.7),
                                                  (4, 1000, 64, 1.0), (3, 4097, 1, 4.0), (2, 33001, 1024, 1.0),
                                                  (200, 515, 20, 1.0), (2, 131072, 64, 2.0), (1, 262147, 7, 1.0)])
def test_loss_and_gradient(mode, dtype, rows, V, k, temperature):
    from matrix_b200.distill import distill_loss, distill_loss_and_grad, distill_loss_with_grad
    z = _rand(rows, V, V + k, dtype, 1.5)
    t, idx, lse = _teacher(rows, V, k, temperature, V, dtype)
    w = torch.rand(rows, generator=torch.Generator().manual_seed(1)).cuda() + 0.5
    kw = _kw(mode, lse, temperature, w)
    loss, grad = _expect(z, t, idx, lse, w, temperature, mode)
    _close_loss(distill_loss(z, t, idx, **kw), loss)
    l, g = distill_loss_and_grad(z, t, idx, **kw)
    assert g.dtype == z.dtype and g.shape == z.shape
    _close_loss(l, loss)
    _close_grad(g, grad)
    up = torch.linspace(-1, 2, rows).cuda()
    x = z.clone().requires_grad_(True)
    l = distill_loss_with_grad(x, t, idx, **kw)
    _close_loss(l, loss)
    l.backward(up)
    assert x.grad.dtype == z.dtype
    _close_grad(x.grad, grad * _np(up)[:, None])


@pytest.mark.parametrize("mode", list(MODES))
def test_gradient_matches_differences(mode):
    """A directional difference of the fp32 loss: rounding 2e-6 over 2h = 4e-2 and h^2 of a third derivative below 4."""
    from matrix_b200.distill import distill_loss, distill_loss_and_grad
    z = _rand(4, 777, 0, scale=1.0)
    t, idx, lse = _teacher(4, 777, 30, 1.0, 5)
    kw = _kw(mode, lse, 1.0, None)
    d = _rand(4, 777, 9, scale=1.0)
    h = 2e-2
    num = (distill_loss(z + h * d, t, idx, **kw) - distill_loss(z - h * d, t, idx, **kw)) / (2 * h)
    _, g = distill_loss_and_grad(z, t, idx, **kw)
    np.testing.assert_allclose(_np((g * d).sum(-1)), _np(num), atol=2e-3)


@pytest.mark.parametrize("mode", list(MODES))
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_with_little_in_them(mode, dtype):
    """Unused slots, empty teachers, masked student entries, weights of zero over garbage, types' lowest values."""
    from matrix_b200.distill import distill_loss, distill_loss_and_grad, distill_loss_with_grad
    V, k = 301, 6
    z = _rand(9, V, 1, F32, 1.5)
    t, idx, lse = _teacher(9, V, k, 1.0, 2)
    w = torch.ones(9, device="cuda")
    idx[0, 2:] = -1                      # unused slots
    idx[1] = -2 ** 31                    # nothing listed
    t[2] = -torch.inf                    # listed, but without mass
    t[3, 1:] = -torch.inf                # one entry has all of it
    z[4, idx[4, 1:].long()] = -5.0
    mask = torch.ones(V, dtype=torch.bool, device="cuda")
    mask[idx[5].long()] = False
    z[5, mask] = torch.finfo(dtype).min  # a masked student: all mass on the listed entries ...
    z[6, mask] = -torch.inf
    lse[5] = lse[6] = torch.logsumexp(t[5], -1)   # ... and a teacher that agrees
    lse[6] = torch.logsumexp(t[6], -1)
    mask6 = torch.ones(V, dtype=torch.bool, device="cuda")
    mask6[idx[6].long()] = False
    z[6] = _rand(1, V, 8)[0]
    z[6, mask6] = -torch.inf
    z[7] = torch.nan
    w[7] = 0.0                           # a row left out, whatever it holds
    z[8, 3] = torch.inf
    idx[8, 0] = 10 ** 6
    w[8] = 0.0
    z, t = z.to(dtype), t.to(dtype)
    if MODES[mode]["reverse"]:           # a teacher without mass where the student has some: infinite
        w[2] = w[3] = 0.0
    kw = _kw(mode, lse, 1.0, w)
    loss, grad = _expect(z, t, idx, lse, w, 1.0, mode)
    if MODES[mode]["tail"]:              # rounding of lse is amplified by an empty student tail: judged by sign
        z5 = distill_loss(z, t, idx, **kw)
        assert torch.isfinite(z5[6])
    rows = [0, 1, 2, 3, 4, 6, 7, 8]
    _close_loss(distill_loss(z, t, idx, **kw)[rows], loss[rows])
    l, g = distill_loss_and_grad(z, t, idx, **kw)
    _close_loss(l[rows], loss[rows])
    _close_grad(g[rows], grad[rows])
    x = z.clone().requires_grad_(True)
    distill_loss_with_grad(x, t, idx, **kw).sum().backward()
    _close_grad(x.grad[rows], grad[rows])
    from matrix_b200.runtime import raise_on_device_status
    raise_on_device_status()             # the bad index lies in a row left out


def test_bad_indices_are_reported():
    from matrix_b200 import _lib
    from matrix_b200.distill import distill_loss_and_grad, distill_loss_with_grad
    from matrix_b200.runtime import raise_on_device_status
    z = _rand(3, 100, 0)
    t, idx, lse = _teacher(3, 100, 5, 1.0, 1)
    idx[0, 3] = 100
    idx[2, 4] = idx[2, 0]
    loss, g = distill_loss_and_grad(z, t, idx)
    assert torch.isnan(loss).tolist() == [True, False, True]
    assert torch.isnan(g).all(-1).tolist() == [True, False, True] and torch.isfinite(g[1]).all()
    with pytest.raises(_lib.DwaError, match="twice"):
        raise_on_device_status()
    x = z.clone().requires_grad_(True)
    distill_loss_with_grad(x, t, idx).sum().backward()
    assert torch.isnan(x.grad).all(-1).tolist() == [True, False, True]
    with pytest.raises(_lib.DwaError):
        raise_on_device_status()
    raise_on_device_status()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_in_place_and_broadcast(dtype):
    from matrix_b200.distill import distill_loss, distill_loss_and_grad, distill_loss_with_grad
    full = _rand(12, 1003, 0, dtype).view(3, 4, 1003)
    t, idx, lse = _teacher(9, 1002, 8, 1.0, 1)
    t, idx, lse = t.view(3, 3, 8), idx.view(3, 3, 8), lse.view(3, 3)
    for z in (full[:, :-1, :1002], full[:, 1:, 1:]):
        want = distill_loss_and_grad(z.contiguous(), t, idx, teacher_lse=lse)
        got = distill_loss_and_grad(z, t, idx, teacher_lse=lse)
        _close_loss(got[0], _np(want[0]).reshape(-1))
        _close_grad(got[1], _np(want[1]))
        x = full.clone().requires_grad_(True)
        y = x[:, :-1, :1002] if z.data_ptr() == full.data_ptr() else x[:, 1:, 1:]
        distill_loss_with_grad(y, t, idx, teacher_lse=lse).sum().backward()
        pad = torch.zeros_like(full)
        (pad[:, :-1, :1002] if z.data_ptr() == full.data_ptr() else pad[:, 1:, 1:]).copy_(want[1])
        _close_grad(x.grad, _np(pad))
    z = full[:, :-1, :1002].contiguous()
    want = distill_loss_and_grad(z, t, idx, teacher_lse=lse)
    loss, g = distill_loss_and_grad(z, t, idx, teacher_lse=lse, out=z)   # over the logits
    assert g.data_ptr() == z.data_ptr()
    assert torch.equal(loss, want[0]) and torch.equal(g, want[1])
    one = full[0, 0].expand(2, 1003)     # one row for two teachers: its gradient is the sum
    x = full[0, 0].detach().clone().requires_grad_(True)
    distill_loss_with_grad(x.expand(2, 1003), t[0, :2], idx[0, :2]).sum().backward()
    parts = distill_loss_and_grad(one, t[0, :2], idx[0, :2])[1]
    _close_grad(x.grad, _np(parts).sum(0), scale=1.0 if dtype == F32 else 2.0 ** -8 / RTOL)
    assert distill_loss(full[:0], t.new_empty(0, 4, 8), idx.new_empty(0, 4, 8)).shape == (0, 4)


def test_types_shapes_and_refusals():
    from matrix_b200.distill import distill_loss, distill_loss_and_grad, distill_loss_with_grad
    z = _rand(4, 50, 0, BF16)
    t, idx, lse = _teacher(4, 50, 5, 1.0, 1, BF16)
    a = distill_loss(z, t, idx)
    assert torch.equal(a, distill_loss(z, t.float(), idx.long()))
    assert torch.equal(a, distill_loss(z[:, None], t[:, None], idx[:, None])[:, 0])
    assert distill_loss(z[0], t[0], idx[0]).shape == ()
    assert torch.equal(a[0], distill_loss(z[0], t[0], idx[0]))
    for call in (distill_loss, distill_loss_and_grad, distill_loss_with_grad):
        with pytest.raises(ValueError, match="reverse"):
            call(z, t, idx, reverse=True)
        with pytest.raises(ValueError):
            call(z, t[:3], idx[:3])
        with pytest.raises(ValueError):
            call(z, t, idx[:, :4])
        with pytest.raises(TypeError):
            call(z, t, idx.float())
        with pytest.raises(TypeError):
            call(z.half(), t, idx)
        with pytest.raises(TypeError):
            call(z, t, idx, weights=torch.ones(4, device="cuda", dtype=torch.float64))
        with pytest.raises(ValueError):
            call(z, t, idx, teacher_lse=lse[:2])
        with pytest.raises(ValueError):
            call(z, t.cpu(), idx)
        with pytest.raises(RuntimeError):
            call(z, t, idx, temperature=0.0)
    with pytest.raises(ValueError):
        distill_loss_and_grad(z, t, idx, out=torch.empty_like(z, dtype=F32))


def test_streams_repeats_and_changed_inputs():
    from matrix_b200.distill import distill_loss_and_grad, distill_loss_with_grad, top_logits
    z = _rand(37, 20011, 0, BF16)
    t, idx, lse = _teacher(37, 20011, 50, 1.0, 1, BF16)
    want = distill_loss_and_grad(z, t, idx, teacher_lse=lse)
    top = top_logits(z, 40)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = distill_loss_and_grad(z, t, idx, teacher_lse=lse)
        top2 = top_logits(z, 40)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want + top, got + top2))
    x = z.clone().requires_grad_(True)
    loss = distill_loss_with_grad(x, t, idx, teacher_lse=lse)
    t.add_(1.0)
    with pytest.raises(RuntimeError, match="modified"):
        loss.sum().backward()


def test_in_a_graph():
    from matrix_b200.distill import distill_loss_and_grad, top_logits
    z = _rand(5, 3001, 0)
    t, idx, lse = _teacher(5, 3001, 9, 1.0, 1)
    distill_loss_and_grad(z, t, idx, teacher_lse=lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        top = top_logits(z, 7)
        out = distill_loss_and_grad(z, t, idx, teacher_lse=lse)
    z.copy_(_rand(5, 3001, 2))
    graph.replay()
    want = (*top_logits(z, 7), *distill_loss_and_grad(z, t, idx, teacher_lse=lse))
    assert all(torch.equal(a, b) for a, b in zip((*top, *out), want))
