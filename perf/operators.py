"""The vocabulary operators as they are measured: cases, inputs, plain forms and exact values.

Three operators work on rows of logits over a vocabulary:

* ``top``: the K largest logits of every row, their indices and the row's
  log-sum-exp at a temperature: what a teacher hands out.
* ``loss``, ``grad``, ``train``: the divergence of a student's logits from such
  a teacher: the rows' losses alone (evaluation), the losses with the gradient
  in one call (a training step that knows its row weights), and the same
  through autograd.
* ``sample``: one token a row under temperature, top-k, top-p and min-p, the
  draw made with given exponential random numbers (argmax of weight / number).

``own`` selects the framework's kernels; without it the plain forms below run:
elementary torch operations in 32 bits, rounded once at the end.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_PEAKS = 64          # raised logits of a peaked row

# one row of a mixed serving batch after the other: (temperature, top_k, top_p, min_p)
_REQUESTS = (
    (1.0, 50, 0.9, 0.0),      # the usual request
    (0.7, 40, 1.0, 0.0),
    (0.0, 0, 1.0, 0.0),       # greedy
    (0.8, 0, 0.95, 0.0),      # nucleus alone
    (1.0, 0, 1.0, 0.05),      # min-p alone
    (1.2, 200, 0.98, 0.02),   # everything at once
    (1.0, 0, 1.0, 0.0),       # the whole distribution
    (0.6, 20, 0.8, 0.0),
)
_FILTERS = {
    "usual": (_REQUESTS[0],),
    "mixed": _REQUESTS,
    "none": ((0.9, 0, 1.0, 0.0),),
    "nucleus": ((1.0, 0, 0.95, 0.0),),
}


def listed():
    """The cases that are always timed."""
    return [
        # a teacher answering a handful of requests: latency
        _top("top_small", 8, 32768, 20, "bf16", 1.0),
        # a teacher labelling a batch of training tokens
        _top("top_teacher", 2048, 131072, 64, "bf16", 1.0),
        # an odd vocabulary in fp32, many entries kept, softened
        _top("top_odd_f32", 333, 50001, 256, "f32", 2.0),
        # held-out loss of a small batch: latency
        _kd("loss_small", "loss", 64, 32768, 32, "bf16", 1.0, tail=False, reverse=False),
        # the training step's loss and gradient over a large vocabulary
        _kd("grad_main", "grad", 4096, 131072, 64, "bf16", 1.0, tail=True, reverse=False),
        # next-token training on logits[:, :-1] of [batch, length, vocabulary], softened, through autograd
        _kd("train_shifted", "train", 2040, 50304, 100, "bf16", 2.0, tail=False, reverse=False, shifted=8),
        # mode-seeking distillation in fp32 with an odd vocabulary
        _kd("grad_reverse_f32", "grad", 1000, 32001, 50, "f32", 1.0, tail=True, reverse=True),
        # one sequence's next token
        _draw_case("sample_one", 1, 131072, "bf16", "usual", True),
        # a serving batch of unlike requests
        _draw_case("sample_mixed", 256, 131072, "bf16", "mixed", True),
        # plain sampling at a temperature from fp32 logits, odd vocabulary
        _draw_case("sample_whole_f32", 96, 50001, "f32", "none", True),
        # a nucleus of thousands of tokens: early training, or a high temperature
        _draw_case("sample_flat", 64, 100352, "bf16", "nucleus", False),
    ]


def draw(rng):
    """One more case of the same ranges."""
    kind = rng.choice(("top", "top", "loss", "grad", "grad", "train", "sample", "sample", "sample"))
    vocab = int(math.exp(rng.uniform(math.log(1000), math.log(262144))))
    if rng.random() < 0.5:
        vocab = max(1000, vocab // 64 * 64)
    most = max(2, min(4096 if kind != "sample" else 512, 2 ** 28 // vocab))
    rows = int(math.exp(rng.uniform(0.0, math.log(most))))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    k = min(vocab // 4, int(math.exp(rng.uniform(0.0, math.log(512)))))
    temperature = rng.choice((1.0, 1.0, 2.0, 4.0))
    if kind == "top":
        c = _top("", rows, vocab, k, dtype, temperature)
    elif kind == "sample":
        c = _draw_case("", rows, vocab, dtype, rng.choice(sorted(_FILTERS)), rng.random() < 0.7)
    else:
        tail = rng.random() < 0.6
        shifted = rng.choice((0, 0, 1, 3))
        rows = max(1, rows // shifted) * shifted if shifted else rows
        c = _kd("", kind, rows, vocab, k, dtype, temperature, tail=tail, reverse=tail and rng.random() < 0.5,
                shifted=shifted)
    del c["name"]
    return c


def _top(name, rows, vocab, k, dtype, temperature):
    return dict(name=name, op="top", rows=rows, vocab=vocab, k=k, dtype=dtype, temperature=temperature)


def _kd(name, op, rows, vocab, k, dtype, temperature, *, tail, reverse, shifted=0):
    return dict(name=name, op=op, rows=rows, vocab=vocab, k=k, dtype=dtype, temperature=temperature, tail=tail,
                reverse=reverse, shifted=shifted)


def _draw_case(name, rows, vocab, dtype, filters, peaked):
    return dict(name=name, op="sample", rows=rows, vocab=vocab, dtype=dtype, filters=filters, peaked=peaked)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _random_logits(g, rows, vocab, peaked=True):
    """fp32 logits: a wide bulk and, in peaked rows, a few dozen candidates that hold most of the mass."""
    x = torch.randn((rows, vocab), generator=g, device="cuda")
    if not peaked:
        return x
    x *= 2.2
    n = min(_PEAKS, vocab)
    start = torch.randint(0, vocab, (rows, 1), generator=g, device="cuda")
    step = torch.randint(1, max(2, vocab // n), (rows, 1), generator=g, device="cuda")
    rank = torch.arange(n, device="cuda")
    height = 14.0 - 1.6 * torch.log1p(rank.float()) + 0.5 * torch.randn((rows, n), generator=g, device="cuda")
    return x.scatter_(1, (start + step * rank) % vocab, height)


def prepare(case, seed):
    """What the program has in hand: the logits, and the teacher's record or the requests' parameters."""
    g = _generator(seed)
    rows, vocab, dtype = case["rows"], case["vocab"], _DTYPES[case["dtype"]]
    if case["op"] == "top":
        return dict(case, logits=_random_logits(g, rows, vocab).to(dtype))
    if case["op"] == "sample":
        want = _FILTERS[case["filters"]]
        per_row = [want[r % len(want)] for r in range(rows)]
        column = list(zip(*per_row))
        return dict(case, logits=_random_logits(g, rows, vocab, case["peaked"]).to(dtype),
                    noise=torch.empty((rows, vocab), device="cuda").exponential_(generator=g),
                    t=torch.tensor(column[0], dtype=torch.float32, device="cuda"),
                    top_k=torch.tensor(column[1], dtype=torch.int32, device="cuda"),
                    top_p=torch.tensor(column[2], dtype=torch.float32, device="cuda"),
                    min_p=torch.tensor(column[3], dtype=torch.float32, device="cuda"))
    teacher = _random_logits(g, rows, vocab)
    student = teacher * 0.8
    student += torch.randn((rows, vocab), generator=g, device="cuda")
    teacher = teacher.to(dtype).float()
    values, indices = torch.topk(teacher, case["k"], dim=-1)
    state = dict(case, teacher=values.to(dtype), indices=indices.to(torch.int32), lse=None,
                 weights=torch.rand(rows, generator=g, device="cuda") + 0.5)
    if case["tail"]:
        state["lse"] = torch.logsumexp(teacher.div_(case["temperature"]), -1)
    student = student.to(dtype)
    if case["shifted"]:
        b = case["shifted"]
        full = torch.zeros((b, rows // b + 1, vocab), dtype=dtype, device="cuda")
        full[:, :-1] = student.view(b, rows // b, vocab)
        student = full[:, :-1]
        for name in ("teacher", "indices", "lse", "weights"):
            if state[name] is not None:
                state[name] = state[name].view(b, rows // b, *state[name].shape[1:])
    if case["op"] == "train":
        student = student.detach().requires_grad_(True)
    return dict(state, logits=student)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    """One pass through an operator and its outputs."""
    op = state["op"]
    if own:
        return _run_own(state, op)
    if op == "top":
        return _plain_top(state["logits"], state["k"], state["temperature"])
    if op == "sample":
        return _plain_sample(state["logits"], state["noise"], state["t"], state["top_k"], state["top_p"],
                             state["min_p"])
    with torch.no_grad():
        return _plain_distill(state, op != "loss")


def _run_own(state, op):
    if op == "sample":
        from matrix_b200.sampling import sample_tokens
        return sample_tokens(state["logits"], state["noise"], temperature=state["t"], top_k=state["top_k"],
                             top_p=state["top_p"], min_p=state["min_p"])
    from matrix_b200 import distill
    if op == "top":
        return distill.top_logits(state["logits"], state["k"], temperature=state["temperature"])
    args = (state["logits"], state["teacher"], state["indices"])
    kw = dict(teacher_lse=state["lse"], temperature=state["temperature"], reverse=state["reverse"],
              weights=state["weights"])
    if op == "loss":
        return distill.distill_loss(*args, **kw)
    if op == "grad":
        return distill.distill_loss_and_grad(*args, **kw)
    state["logits"].grad = None
    loss = distill.distill_loss_with_grad(*args, **kw)
    loss.sum().backward()
    return loss.detach(), state["logits"].grad


def _ordered(logits):
    """An int64 per logit whose order is: larger logit first, then lower index."""
    bits = (logits.float() + 0.0).view(torch.int32)
    key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    last = logits.shape[-1] - 1
    return (key << 32) + (last - torch.arange(last + 1, device=logits.device))


def _plain_top(logits, k, temperature):
    keys = torch.topk(_ordered(logits), k, dim=-1).values
    indices = logits.shape[-1] - 1 - (keys & 0xFFFFFFFF)
    x = logits.float() / temperature
    m = x.amax(-1, keepdim=True)
    lse = m[..., 0] + torch.log(torch.exp(x - m).sum(-1))
    return logits.gather(-1, indices), indices.to(torch.int32), lse


def _plain_distill(state, with_grad):
    z, temperature = state["logits"], state["temperature"]
    idx = state["indices"].long()
    t = state["teacher"].float() / temperature
    x = z.float() / temperature
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    log_q = x.gather(-1, idx) - m - torch.log(total)
    q = torch.exp(log_q)
    if state["tail"]:
        log_p = t - state["lse"][..., None]
        p = torch.exp(log_p)
        p_tail = (1.0 - p.sum(-1, keepdim=True)).clamp(min=2.0 ** -24)
        q_tail = e.scatter(-1, idx, 0.0).sum(-1, keepdim=True) / total
        tail_ratio = _log_rest(q_tail, q) - _log_rest(p_tail, p)
        if state["reverse"]:
            listed_ratio = log_q - log_p
            loss = (q * listed_ratio).sum(-1, keepdim=True) + q_tail * tail_ratio
            of_tail, of_listed = tail_ratio - loss, q * (listed_ratio - loss)
        else:
            loss = (p * (log_p - log_q)).sum(-1, keepdim=True) - p_tail * tail_ratio
            of_tail, of_listed = 1.0 - p_tail / q_tail, q - p
    else:
        tm = t.amax(-1, keepdim=True)
        log_p = t - tm - torch.log(torch.exp(t - tm).sum(-1, keepdim=True))
        p = torch.exp(log_p)
        loss = (p * (log_p - log_q)).sum(-1, keepdim=True)
        of_tail, of_listed = torch.ones_like(loss), q - p
    loss = loss[..., 0] * state["weights"]
    if not with_grad:
        return loss
    scale = state["weights"][..., None] / temperature
    grad = (e * (of_tail * scale / total)).scatter(-1, idx, of_listed * scale)
    return loss, grad.to(z.dtype)


def _log_rest(rest, listed):
    """log(rest) where rest = 1 - sum(listed), from whichever of the two is exact: the small one."""
    return torch.where(rest > 0.5, torch.log1p(-listed.sum(-1, keepdim=True)), torch.log(rest))


def _plain_sample(logits, noise, t, top_k, top_p, min_p):
    vocab = logits.shape[-1]
    x = logits.float()
    greedy = (t <= 0)[:, None]
    s = (x - x.amax(-1, keepdim=True)) / torch.where(greedy, torch.ones_like(t[:, None]), t[:, None])
    order = vocab - 1 - (torch.sort(_ordered(logits), dim=-1, descending=True).values & 0xFFFFFFFF)
    w = torch.exp(s).gather(-1, order)
    rank = torch.arange(vocab, device=w.device)
    limit = torch.where((top_k <= 0) | (top_k > vocab), torch.full_like(top_k, vocab), top_k)
    limit = torch.where(greedy, torch.ones_like(limit[:, None]), limit[:, None])
    keep = rank < limit
    w = w * keep
    before = w.cumsum(-1) - w
    keep &= (before < top_p[:, None] * w.sum(-1, keepdim=True)) | (top_p >= 1)[:, None] | (rank == 0)
    keep &= (w >= min_p[:, None]) & (w > 0)
    score = torch.where(keep, w / noise.gather(-1, order), torch.full_like(w, -1.0))
    token = order.gather(-1, score.argmax(-1, keepdim=True))
    logprob = s.gather(-1, token) - torch.log((w * keep).sum(-1, keepdim=True))
    return token[:, 0].to(torch.int32), logprob[:, 0]


# ---------------------------------------------------------------------------
# the work that cannot be left out, and the values in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    """Bytes and operations of one pass: every input read once, every output written once."""
    rows, vocab = case["rows"], case["vocab"]
    size = 2 if case["dtype"] == "bf16" else 4
    logits = rows * vocab * size
    if case["op"] == "top":
        return {"bytes": logits + rows * (case["k"] * (size + 4) + 4), "flops": 4 * rows * vocab}
    if case["op"] == "sample":
        want = _FILTERS[case["filters"]]
        whole = sum(want[r % len(want)][1:] == (0, 1.0, 0.0) and want[r % len(want)][0] > 0 for r in range(rows))
        return {"bytes": logits + whole * vocab * 4 + rows * 24, "flops": 4 * rows * vocab}
    record = rows * (case["k"] * (size + 4) + 4 * case["tail"] + 8)
    if case["op"] == "loss":
        return {"bytes": logits + record, "flops": 4 * rows * vocab}
    return {"bytes": 2 * logits + record, "flops": 8 * rows * vocab}


def exact(case, seed):
    """What run() returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "top":
        return _exact_top(s)
    if case["op"] == "sample":
        return _exact_sample(s)
    vocab, k = case["vocab"], case["k"]
    z, t, idx, w = (s[n].detach().reshape(-1, *s[n].shape[s["weights"].dim():])
                    for n in ("logits", "teacher", "indices", "weights"))
    lse = s["lse"].reshape(-1) if case["tail"] else None
    losses, grads = [], []
    step = max(1, 2 ** 25 // vocab)
    for a in range(0, case["rows"], step):
        b = slice(a, a + step)
        x = z[b].double().requires_grad_(case["op"] != "loss")
        loss = w[b].double() * _exact_kl(x / case["temperature"], t[b].double() / case["temperature"],
                                         idx[b].long(), lse[b].double() if case["tail"] else None, case["reverse"])
        losses.append(loss.detach())
        if x.requires_grad:
            loss.sum().backward()
            grads.append(x.grad)
    shape = s["weights"].shape
    loss = torch.cat(losses).reshape(shape)
    return loss if case["op"] == "loss" else (loss, torch.cat(grads).reshape(*shape, vocab))


def _exact_kl(x, t, idx, lse, reverse):
    """KL of two distributions over the listed entries and, given lse, one class for all others."""
    log_q = torch.log_softmax(x, -1)
    log_p = torch.log_softmax(t, -1) if lse is None else t - lse[:, None]
    a = log_q.gather(-1, idx)
    if lse is not None:
        rest = torch.logsumexp(log_q.scatter(-1, idx, -math.inf), -1, keepdim=True)
        a = torch.cat((a, rest), -1)
        p_rest = (-torch.expm1(torch.logsumexp(log_p, -1, keepdim=True))).clamp(min=2.0 ** -24)
        log_p = torch.cat((log_p, p_rest.log()), -1)
    return (a.exp() * (a - log_p) if reverse else log_p.exp() * (log_p - a)).sum(-1)


def _exact_top(s):
    values, indices = [], []
    for row in s["logits"].split(256):
        v, i = torch.sort(row.double(), dim=-1, descending=True, stable=True)
        values.append(v[:, : s["k"]])
        indices.append(i[:, : s["k"]].to(torch.int32))
    lse = torch.cat([torch.logsumexp(r.double() / s["temperature"], -1) for r in s["logits"].split(256)])
    return torch.cat(values), torch.cat(indices), lse


def _exact_sample(s):
    tokens, logprobs = [], []
    for r in range(s["rows"]):
        t, k, p, floor = (float(s[n][r]) for n in ("t", "top_k", "top_p", "min_p"))
        z, i = torch.sort(s["logits"][r].double(), descending=True, stable=True)
        if t <= 0:
            tokens.append(i[0])
            logprobs.append(torch.zeros_like(z[0]))
            continue
        if 0 < k < len(z):
            z, i = z[: int(k)], i[: int(k)]
        q = torch.softmax(z / t, -1)
        n = len(q)
        if p < 1:
            n = max(1, int((q.cumsum(0) - q < p).sum()))
        n = min(n, int((q >= floor * q[0]).sum()))
        best = (q[:n] / s["noise"][r][i[:n]].double()).argmax()
        tokens.append(i[best])
        logprobs.append(torch.log_softmax(z[:n] / t, -1)[best])
    return torch.stack(tokens).to(torch.int32), torch.stack(logprobs)
