"""Measured calls of the post-training losses on logits: token log-probabilities and their backward pass, the paired
preference loss and the clipped policy loss with a KL term, each with its gradient in the logits.

`listed()` and `draw()` give cases, `prepare()` makes one case's inputs on the GPU, `run()` is one call: the plain form in
elementary torch operations, or with `own` the call of this package. `exact()` is the definition in 64 bits.

Notation, per row (one position of one sequence) with logits z, temperature T and target y:
    x = z / T,  lse = log sum_j exp x_j,  logp = x_y - lse,  p_j = exp(x_j - lse),  dlogp/dz_j = ([j == y] - p_j) / T
A row counts when its target is >= 0 (and its weight, where there are weights, is not 0); a row that does not count has
logp = lse = 0 and a gradient of 0.

policy, per counted row: r = exp(logp - old), g = min(r A, clip(r, 1 - lo, 1 + hi) A), d = ref - logp,
    k = exp(d) - d - 1, loss = sum w (-g + c k) / D, count = sum w, kl = sum w k / D,
    clipped = sum w [clip(r) A < r A] (the rows whose ratio has no gradient)
preference, per pair (chosen i, rejected i + S/2): s = sum of a sequence's logp (its mean with `average`),
    u = beta ((s_i - ref_i) - (s_j - ref_j)), loss = sum (-(1 - e) log sigmoid(u) - e log sigmoid(-u)) / D,
    rewards = beta (s - ref)
"""

import math

import numpy as np
import torch

own = False

VOCAB = 271          # the byte tokenizer's vocabulary (mote_b200/configs.py: the 271 x 128 and 271 x 768 embeddings)
MOST = 1 << 30       # logits of the largest case
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _case(name, op, dtype, seqs, tokens, vocab, prompt=0.0, shifted=False, packed=False, masked=0, temperature=1.0,
          ref=True, weighted=False, per_token=False, average=False, smoothing=0.0):
    """`prompt`: share of each sequence whose targets are ignored; `shifted`: the logits are the view [:, :-1] of one more
    position; `packed`: sequences of different lengths one behind the other, with cu_seqlens; `masked`: that many last
    columns are -inf (a vocabulary padded to a round size)."""
    return dict(name=name, op=op, dtype=dtype, seqs=seqs, tokens=tokens, vocab=vocab, prompt=prompt, shifted=shifted,
                packed=packed, masked=masked, temperature=temperature, ref=ref, weighted=weighted, per_token=per_token,
                average=average, smoothing=smoothing)


def listed():
    return [
        # one position of a byte model, as a scorer of single answers asks for it: latency
        _case("logprobs one token", "logprobs", "fp32", 1, 1, VOCAB),
        # a training batch of the byte model scored by the reference model, next-byte shifted view
        _case("logprobs bytes", "logprobs", "bf16", 16, 2047, VOCAB, prompt=0.25, shifted=True),
        # a vocabulary of no round size: rows start at every alignment
        _case("logprobs odd vocabulary", "logprobs", "bf16", 4, 1023, 50021),
        # the first sampled token of a few prompts over a very large vocabulary: few rows, a long axis
        _case("logprobs few long rows", "logprobs", "fp32", 8, 1, 262144, temperature=0.7),
        # the backward pass under a loss of the user's own, byte model in fp32
        _case("backward bytes fp32", "backward", "fp32", 8, 2048, VOCAB, prompt=0.25),
        # the same over a large vocabulary
        _case("backward large vocabulary", "backward", "bf16", 4, 1024, 131072, prompt=0.125, masked=64),
        # two short pairs: latency of the whole loss and gradient
        _case("preference two short pairs", "preference", "bf16", 4, 64, VOCAB, prompt=0.25),
        # sixteen pairs of the byte model, ragged and packed, with rows of padding behind the last one
        _case("preference packed bytes", "preference", "bf16", 32, 2048, VOCAB, prompt=0.25, packed=True),
        # two pairs over a large vocabulary, next-token shifted view
        _case("preference large vocabulary", "preference", "bf16", 4, 2047, 65536, prompt=0.25, shifted=True,
              average=True, smoothing=0.1),
        # a group of eight short samples, fp32 logits
        _case("policy short samples", "policy", "fp32", 8, 16, VOCAB),
        # a group step of the byte model: 64 samples, weights 1 / length
        _case("policy bytes", "policy", "bf16", 64, 1024, VOCAB, prompt=0.25, weighted=True),
        # the largest: eight samples over a large vocabulary, token advantages
        _case("policy large vocabulary", "policy", "bf16", 8, 1024, 131072, prompt=0.125, masked=64, temperature=0.9,
              per_token=True),
    ]


def draw(rng):
    op = rng.choice(["logprobs", "backward", "preference", "policy"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    vocab = VOCAB if rng.random() < 0.25 else int(math.exp(rng.uniform(math.log(32), math.log(262144))))
    if rng.random() < 0.5 and vocab > 64:
        vocab -= vocab % 64
    most = min(65536, MOST // vocab // (2 if dtype == "fp32" else 1))
    rows = int(math.exp(rng.uniform(0, math.log(most))))
    seqs = min(64, int(math.exp(rng.uniform(0, math.log(rows + 1)))))
    if op == "preference":
        seqs = max(2, seqs - seqs % 2)
    tokens = max(1, min(8192, rows // seqs))
    packed = op == "preference" and rng.random() < 0.5
    case = _case("", op, dtype, seqs, tokens, vocab, prompt=rng.choice([0.0, 0.125, 0.25]),
                 shifted=not packed and rng.random() < 0.4, packed=packed,
                 masked=rng.choice([0, 0, min(64, vocab // 4)]), temperature=rng.choice([1.0, 1.0, 0.7, 1.3]),
                 ref=rng.random() < 0.75, weighted=op == "policy" and rng.random() < 0.5,
                 per_token=op == "policy" and rng.random() < 0.5, average=op == "preference" and rng.random() < 0.5,
                 smoothing=rng.choice([0.0, 0.1]) if op == "preference" else 0.0)
    del case["name"]
    return case


def _packed_rows(case):
    """Rows of a packed buffer: the sequences' mean length is 3/4 of `tokens`, and 1/16 is left for longer batches."""
    return -(-case["seqs"] * case["tokens"] * 13 // 16 // 8) * 8


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    host = np.random.default_rng(seed)
    S, T, V, dt = case["seqs"], case["tokens"], case["vocab"], TYPES[case["dtype"]]
    st = {"case": case}
    first = int(case["prompt"] * T)
    if case["packed"]:   # lengths of half to the whole of T, in a buffer of a fixed number of rows
        shape = (_packed_rows(case),)
        lens = host.integers((T + 1) // 2, T + 1, S)
        if lens.sum() > shape[0]:
            lens = lens * shape[0] // lens.sum()
        cu = np.concatenate([[0], np.cumsum(lens)])
        at = np.zeros(shape, bool)
        for i in range(S):
            at[cu[i] + int(case["prompt"] * lens[i]):cu[i + 1]] = True
        st["cu_seqlens"] = torch.from_numpy(cu.astype(np.int32)).to(dev)
    else:
        shape = (S, T)
        at = np.zeros(shape, bool)
        at[:, first:] = True
    live = torch.from_numpy(at).to(dev)
    # logits of a language model: a spread of about two, and a target somewhat likelier or less likely than the rest
    full = shape if not case["shifted"] else (S, T + 1)
    logits = torch.randn(*full, V, generator=gen, device=dev, dtype=dt).mul_(2.0)
    if case["masked"]:
        logits[..., V - case["masked"]:] = -math.inf
    if case["shifted"]:
        logits = logits[:, :-1]
    y = torch.randint(0, V - case["masked"], shape, generator=gen, device=dev)
    bump = math.log(V) + 2.0 + 2.0 * torch.randn(shape, generator=gen, device=dev) - 1.0
    logits.scatter_(-1, y[..., None], bump[..., None].to(dt))
    st["logits"], st["targets"] = logits, torch.where(live, y, -100)
    op = case["op"]
    if op == "logprobs":
        return st
    logp, lse = _plain_logprobs(logits, st["targets"], case["temperature"])
    if op == "backward":   # what the forward pass kept, and the gradient that reached the log-probabilities
        st["logprobs"], st["lse"] = logp, lse
        st["grad_logprobs"] = torch.randn(shape, generator=gen, device=dev) / logp.numel()
    elif op == "policy":   # samples of a slightly older policy, and a reference model some way off
        st["old_logprobs"] = logp + 0.15 * torch.randn(shape, generator=gen, device=dev)
        st["ref_logprobs"] = logp + 0.3 * torch.randn(shape, generator=gen, device=dev) if case["ref"] else None
        st["advantages"] = torch.randn(shape if case["per_token"] else shape[:1], generator=gen, device=dev)
        st["weights"] = (torch.full(shape[:1], 1.0 / (T - first), device=dev)
                         * (0.5 + torch.rand(shape[:1], generator=gen, device=dev))) if case["weighted"] else None
    else:
        s = _sequence_sums(logp.double(), st)
        if case["average"]:
            s = s / _sequence_sums((st["targets"] >= 0).double(), st).clamp(min=1)
        # policy and reference drift apart by about 0.1 a token, independently, besides a constant
        noise = (0.3 if case["average"] else 1.0 + 0.1 * math.sqrt(T)) * torch.randn(s.shape, generator=gen, device=dev)
        st["ref_logprobs"] = (s + noise).float() if case["ref"] else None
    return st


# ---- the plain forms: elementary torch operations in 32 bits, the values of whole rows and sequences in 64
def _plain_rows(logits, targets, temperature):
    """x, the counted rows, their targets, exp(x - max) and its sum (in 64 bits), and logp in 64 bits."""
    x = logits.float() / temperature if temperature != 1.0 else logits.float()
    live = targets >= 0
    y = torch.where(live, targets, 0)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    at = x.gather(-1, y[..., None])
    logp = ((at - m).double() - torch.log(total))[..., 0]
    return x, live, y, m, e, total, logp


def _plain_logprobs(logits, targets, temperature):
    x, live, y, m, e, total, logp = _plain_rows(logits, targets, temperature)
    lse = (m.double() + torch.log(total))[..., 0]
    return torch.where(live, logp, 0.0).float(), torch.where(live, lse, 0.0).float()


def _plain_gradient(p, y, coef, live, temperature, dtype):
    """coef ([j == y] - p_j) / T, rounded once; rows that do not count are 0 whatever they hold. p is overwritten."""
    p.scatter_add_(-1, y[..., None], torch.full_like(p[..., :1], -1.0))
    p.mul_((coef / -temperature).float()[..., None])
    return torch.where(live[..., None], p, 0.0).to(dtype)


def _row_sequence(st, rows):
    """The sequence of every packed row, and whether it lies in one."""
    cu = st["cu_seqlens"].long()
    at = torch.arange(rows, device=cu.device)
    i = torch.searchsorted(cu, at, right=True) - 1
    inside = (i >= 0) & (i < cu.numel() - 1)
    return i.clamp(0, cu.numel() - 2), inside


def _sequence_sums(v, st):
    if not st["case"]["packed"]:
        return v.sum(1)
    i, inside = _row_sequence(st, v.numel())
    return torch.zeros(st["case"]["seqs"], dtype=v.dtype, device=v.device).index_add_(0, i, torch.where(inside, v, 0.0))


def _plain_backward(st):
    c, z = st["case"], st["logits"]
    live = st["targets"] >= 0
    y = torch.where(live, st["targets"], 0)
    x = z.float() / c["temperature"] if c["temperature"] != 1.0 else z.float()
    p = torch.exp(x - st["lse"][..., None])
    return {"grad": _plain_gradient(p, y, st["grad_logprobs"], live, c["temperature"], z.dtype)}


def _plain_policy(st):
    c, z = st["case"], st["logits"]
    x, live, y, m, e, total, logp = _plain_rows(z, st["targets"], c["temperature"])
    A, w = st["advantages"].double(), st["weights"]
    A = A if A.dim() == logp.dim() else A[:, None].expand_as(logp)
    w = torch.ones_like(logp) if w is None else w.double()[:, None].expand_as(logp)
    live = live & (w != 0)
    r = torch.exp(logp - st["old_logprobs"].double())
    free, held = r * A, r.clamp(0.8, 1.2) * A
    k = torch.zeros_like(logp)
    coef = torch.where(free <= held, -free, 0.0)
    if st["ref_logprobs"] is not None:
        d = st["ref_logprobs"].double() - logp
        k = torch.exp(d) - d - 1
        coef = coef + 0.04 * (1 - torch.exp(d))
    loss = torch.minimum(free, held).neg() + 0.04 * k
    div = float(c["tokens"])
    total_of = lambda v: torch.where(live, w * v, 0.0).sum().float()  # noqa: E731
    grad = _plain_gradient(e / total.float(), y, w * coef / div, live, c["temperature"], z.dtype)
    return {"loss": total_of(loss / div), "count": total_of(torch.ones_like(w)), "kl": total_of(k / div),
            "clipped": total_of((held < free).double()), "logprobs": torch.where(live, logp, 0.0).float(), "grad": grad}


def _plain_preference(st):
    c, z = st["case"], st["logits"]
    x, live, y, m, e, total, logp = _plain_rows(z, st["targets"], c["temperature"])
    half, div, beta, eps = c["seqs"] // 2, c["seqs"] / 2, 0.1, c["smoothing"]
    if c["packed"]:
        seq, inside = _row_sequence(st, logp.numel())
        live = live & inside
    s = _sequence_sums(torch.where(live, logp, 0.0), st)
    n = _sequence_sums(live.double(), st).clamp(min=1) if c["average"] else torch.ones_like(s)
    s = s / n
    rewards = beta * (s - (st["ref_logprobs"].double() if st["ref_logprobs"] is not None else 0.0))
    u = rewards[:half] - rewards[half:]
    up, down = torch.log1p(torch.exp(-u.abs())) + (-u).clamp(min=0), torch.log1p(torch.exp(-u.abs())) + u.clamp(min=0)
    loss = ((1 - eps) * up + eps * down).sum() / div
    du = beta * (eps / (1 + torch.exp(-u)) - (1 - eps) / (1 + torch.exp(u))) / div
    coef = torch.cat([du, -du]) / n
    coef = coef[seq] if c["packed"] else coef[:, None].expand_as(logp)
    grad = _plain_gradient(e / total.float(), y, coef, live, c["temperature"], z.dtype)
    return {"loss": loss.float(), "rewards": rewards.float(), "logprobs": s.float(), "grad": grad}


def run(state):
    c = state["case"]
    if own:
        import mote_b200 as mote
        z, y, t = state["logits"], state["targets"], c["temperature"]
        if c["op"] == "logprobs":
            r = mote.token_logprobs(z, y, temperature=t)
            return {"logprobs": r.logprobs, "lse": r.lse}
        if c["op"] == "backward":
            return {"grad": mote.token_logprobs_backward(z, y, state["logprobs"], state["lse"], state["grad_logprobs"],
                                                         temperature=t)}
        if c["op"] == "policy":
            kl_coef = 0.04 if c["ref"] else 0.0   # no reference model: no KL term
            r = mote.policy_loss(z, y, state["advantages"], state["old_logprobs"], state["ref_logprobs"],
                                 weights=state["weights"], clip_low=0.2, clip_high=0.2, kl_coef=kl_coef, temperature=t,
                                 divisor=float(c["tokens"]))
            return {"loss": r.loss, "count": r.count, "kl": r.kl, "clipped": r.clipped, "logprobs": r.logprobs,
                    "grad": r.grad}
        r = mote.preference_loss(z, y, state["ref_logprobs"], cu_seqlens=state.get("cu_seqlens"), beta=0.1,
                                 label_smoothing=c["smoothing"], average=c["average"], temperature=t,
                                 divisor=c["seqs"] / 2)
        return {"loss": r.loss, "rewards": r.rewards, "logprobs": r.logprobs, "grad": r.grad}
    if c["op"] == "logprobs":
        logp, lse = _plain_logprobs(state["logits"], state["targets"], c["temperature"])
        return {"logprobs": logp, "lse": lse}
    return {"backward": _plain_backward, "policy": _plain_policy, "preference": _plain_preference}[c["op"]](state)


def work(case):
    """Counted rows are read once (twice is not needed by the definition), the gradient is written whole; per position the
    target and the few values of 4 bytes that go in and come out. Five operations for a logit's share of the sum, two more
    for its gradient."""
    rows = _packed_rows(case) if case["packed"] else case["seqs"] * case["tokens"]
    live = (0.75 * case["seqs"] * case["tokens"] if case["packed"] else rows) * (1.0 - case["prompt"])
    size = 2 if case["dtype"] == "bf16" else 4
    read, wrote = live * case["vocab"] * size, rows * case["vocab"] * size
    per = {"logprobs": 16, "backward": 20, "preference": 8, "policy": 16 + 4 * case["ref"] + 4 * case["per_token"]}[case["op"]]
    if case["op"] == "logprobs":
        return {"bytes": read + per * rows, "flops": 5 * live * case["vocab"]}
    return {"bytes": read + wrote + per * rows, "flops": (4 if case["op"] == "backward" else 7) * live * case["vocab"]}


# ---- the definition in 64 bits
def _exact_rows(z, y, live, temperature):
    """log-softmax at the target and lse of each row [N], a block of rows at a time."""
    N, V = z.shape
    logp, lse = torch.zeros(N, dtype=torch.float64, device=z.device), torch.zeros(N, dtype=torch.float64, device=z.device)
    block = max(1, (1 << 26) // V)
    for a in range(0, N, block):
        x = z[a:a + block].double() / temperature
        lse[a:a + block] = torch.logsumexp(x, -1)
        logp[a:a + block] = x.gather(1, y[a:a + block, None])[:, 0] - lse[a:a + block]
    return torch.where(live, logp, 0.0), torch.where(live, lse, 0.0)


def _exact_gradient(z, y, live, lse, coef, temperature):
    N, V = z.shape
    out = torch.zeros(N, V, dtype=torch.float64, device=z.device)
    block = max(1, (1 << 26) // V)
    for a in range(0, N, block):
        q = out[a:a + block]
        on = live[a:a + block, None]
        one = torch.nn.functional.one_hot(y[a:a + block], V)
        q += torch.where(on, coef[a:a + block, None] * (one - torch.exp(z[a:a + block].double() / temperature
                                                                          - lse[a:a + block, None])) / temperature, 0.0)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    V, t = case["vocab"], case["temperature"]
    shape = st["targets"].shape
    z, y0 = st["logits"].reshape(-1, V), st["targets"].reshape(-1)
    live, y = y0 >= 0, y0.clamp(min=0)
    if case["op"] == "policy":
        w = torch.ones(shape, dtype=torch.float64, device=z.device)
        if st["weights"] is not None:
            w = w * st["weights"].double()[:, None]
        w = w.reshape(-1)
        live = live & (w != 0)
    if case["op"] == "preference" and case["packed"]:
        cu = st["cu_seqlens"].tolist()
        live[cu[-1]:] = False
    logp, lse = _exact_rows(z, y, live, t)
    if case["op"] == "logprobs":
        return {"logprobs": logp.reshape(shape), "lse": lse.reshape(shape)}
    if case["op"] == "backward":   # of the row statistics that the forward pass kept
        g = _exact_gradient(z, y, live, st["lse"].reshape(-1).double(), st["grad_logprobs"].reshape(-1).double(), t)
        return {"grad": g.reshape(*shape, V)}
    if case["op"] == "policy":
        A = st["advantages"].double()
        A = (A if case["per_token"] else A[:, None].expand(shape)).reshape(-1)
        r = torch.exp(logp - st["old_logprobs"].reshape(-1).double())
        over = torch.where(A > 0, r > 1.2, r < 0.8) & (A != 0)
        gain = torch.where(over, torch.where(A > 0, 1.2, 0.8).double(), r) * A
        loss, slope, kl = -gain, torch.where(over, 0.0, -r * A), torch.zeros_like(r)
        if st["ref_logprobs"] is not None:
            ref = st["ref_logprobs"].reshape(-1).double()
            kl = torch.expm1(ref - logp) - (ref - logp)
            loss, slope = loss + 0.04 * kl, slope - 0.04 * torch.expm1(ref - logp)
        w = torch.where(live, w, 0.0)
        div = case["tokens"]
        g = _exact_gradient(z, y, live, lse, w * slope / div, t)
        return {"loss": (w * loss).sum() / div, "count": w.sum(), "kl": (w * kl).sum() / div, "clipped": (w * over).sum(),
                "logprobs": logp.reshape(shape), "grad": g.reshape(*shape, V)}
    if case["packed"]:
        parts = [slice(cu[i], cu[i + 1]) for i in range(case["seqs"])]
    else:
        parts = [slice(i * shape[1], (i + 1) * shape[1]) for i in range(case["seqs"])]
    n = torch.stack([live[p].sum().double().clamp(min=1) if case["average"] else torch.ones_like(logp[0]) for p in parts])
    s = torch.stack([logp[p].sum() for p in parts]) / n
    rewards = 0.1 * (s - (st["ref_logprobs"].double() if st["ref_logprobs"] is not None else 0.0))
    h, e = case["seqs"] // 2, case["smoothing"]
    u = rewards[:h] - rewards[h:]
    F = torch.nn.functional
    loss = (-(1 - e) * F.logsigmoid(u) - e * F.logsigmoid(-u)).sum() / h
    du = 0.1 * (e * torch.sigmoid(u) - (1 - e) * torch.sigmoid(-u)) / h
    per, coef = torch.cat([du, -du]) / n, torch.zeros_like(logp)
    for p, c in zip(parts, per):
        coef[p] = c
    g = _exact_gradient(z, y, live, lse, coef, t)
    return {"loss": loss, "rewards": rewards, "logprobs": s, "grad": g.reshape(*shape, V)}
