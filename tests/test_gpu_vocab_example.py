"""The vocabulary operators used together, as the example uses them: a teacher's
top logits, the student's fused loss and gradient, then sampling.

What is asserted: the first step's loss is the float64 oracle's for the
student's first logits, training lowers it, and every sampled token and its
log-probability are in range.
"""

from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import numpy as np
import pytest

from oracle import vocab_oracle as vo

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parent.parent / "examples" / "distill_and_sample.py"
    spec = importlib.util.spec_from_file_location("distill_and_sample", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("vocab,reverse", [(1000, False), (1001, True)])
def test_example_trains_and_samples(vocab, reverse):
    ex = _example()
    batch, seq, new = 4, 16, 3
    got = ex.run(vocab=vocab, steps=25, batch=batch, seq=seq, top=32, new_tokens=new, reverse=reverse, seed=3)
    assert torch.isfinite(got["losses"]).all()
    assert got["losses"][-1] < 0.7 * got["losses"][0]
    text, lp = got["tokens"], got["logprobs"]
    assert text.shape == (batch, 1 + new) and lp.shape == (batch, new)
    assert ((text >= 0) & (text < vocab)).all()
    # top_k 50 leaves at most 50 entries and the chosen one has w >= 0.02 of the largest
    assert (lp <= 0).all() and (lp >= math.log(0.02 / 50) - 1e-3).all()


def test_example_first_loss_is_the_oracles():
    ex = _example()
    vocab, batch, seq, top, T = 777, 2, 8, 16, 2.0
    got = ex.run(vocab=vocab, steps=1, batch=batch, seq=seq, top=top, new_tokens=1, temperature=T, seed=5)
    gen = torch.Generator().manual_seed(5)
    cfg = got["student"].cfg
    fresh = ex.Student(cfg, vocab, gen)
    u, v = torch.randn(vocab, 16, generator=gen).cuda(), torch.randn(vocab, 16, generator=gen).cuda()
    corpus = torch.randint(0, vocab, (batch, seq), generator=gen).cuda()
    with torch.no_grad():
        z = fresh(corpus).float().cpu().numpy().reshape(-1, vocab)
    t = (u[corpus] @ v.T).bfloat16().float().cpu().numpy().reshape(-1, vocab)
    want = []
    for zr, tr in zip(z, t):
        tv, ti, lse = vo.top_logits(tr, top, T)
        want.append(vo.distill(zr, tv, ti, lse, temperature=T)[0])
    # rows of order 1 summed in f32 by the device; inputs are the same bf16 values
    assert abs(float(got["losses"][0]) - np.mean(want)) <= 1e-5 * abs(np.mean(want)) + 1e-6
