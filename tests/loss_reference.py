"""The losses on logits in 64 bits, position by position, from their definitions (include/moteopt.h), on the CPU; and how far
an fp32 kernel may be from them. Shared by the GPU tests and the CPU tests of this file itself.

Tolerances, with u = 2^-24 (half a step of fp32). A row's exponentials come from ex2.approx (at most 2 ulp, 4u of the value,
plus 2u of the argument's own rounding per unit of the exponent's size, in base e: 2u R where R is the distance from the
row's largest to its smallest finite x), summed in fp32 by a thread over at most 4096 logits in two chains of fours (a
random walk would be far less; the bound used is 512u, 32 logits a vector batch and at most 128 batches) and in trees above
(16 levels, 2u each with their factors). So
    lse, logp:  |err| <= u |value| + S,   S = (4 + 2 R + 512 + 32) u
    a probability: relative error S + (4 + 2 R) u for its own exponential, + 4u for the products
    a gradient: |err| <= |coef| (p (2 S) + [j == y] S) / T, and one rounding to the output's type (eps / 2 of the value)
"""

import math

import torch

U = 2.0 ** -24


def row_values(z, y, T):
    """logp, lse in 64 bits; 0 where y < 0, NaN where y >= V, where a logit is NaN or +inf (inf - inf) and where all are -inf.
    Differences are taken first, and where the target is the largest logp = -log1p(sum over the others of exp(x_j - x_y)),
    so that neither lowest-value logits nor sure targets lose it."""
    x = z.double() / T
    V = x.shape[-1]
    live = y >= 0
    m = x.amax(-1)
    d = x - m[..., None]
    k = y.clamp(0, V - 1)[..., None]
    l = torch.log(torch.exp(d).sum(-1))
    at = d.gather(-1, k)[..., 0]
    others = torch.exp(d.scatter(-1, k, -math.inf)).sum(-1)
    logp = torch.where(at == 0.0, -torch.log1p(others), at - l)
    lse = m + l
    good = (y < V) & torch.isfinite(m)
    logp, lse = torch.where(good, logp, math.nan), torch.where(good, lse, math.nan)
    return torch.where(live, logp, 0.0), torch.where(live, lse, 0.0)


def spread(z, T):
    """S of the rows (see the top)."""
    x = z.double() / T
    fin = torch.isfinite(x)
    hi = torch.where(fin, x, -math.inf).amax(-1)
    lo = torch.where(fin, x, math.inf).amin(-1)
    R = torch.where(torch.isfinite(hi - lo), (hi - lo).clamp(max=104.0), 0.0)   # below e^-104 an exponential is 0
    return (4 + 2 * R + 512 + 32) * U


def gradient(z, y, coef, T, live):
    """coef ([j == y] - p) / T, 0 where not live, NaN rows where y >= V; and its tolerance before the last rounding."""
    x = z.double() / T
    V = x.shape[-1]
    p = torch.softmax(x, -1)
    one = torch.zeros_like(p).scatter_(-1, y.clamp(0, V - 1)[..., None], 1.0)
    g = coef[..., None] * (one - p) / T
    S = spread(z, T)[..., None]
    tol = coef.abs()[..., None] * (p * 2 * S + one * S) / T
    g = torch.where((y >= V)[..., None], math.nan, g)
    return torch.where(live[..., None], g, 0.0), torch.where(live[..., None], tol, 0.0)


def policy(z, y, A, old, ref, w, lo, hi, c, T, div):
    logp, _ = row_values(z, y, T)
    A = (A if A.shape == y.shape else A[:, None].expand(y.shape)).double()
    w = torch.ones_like(A) if w is None else (w if w.shape == y.shape else w[:, None].expand(y.shape)).double()
    live = (y >= 0) & (w != 0)
    r = torch.exp(logp - old.double())
    free, held = r * A, r.clamp(1 - lo, 1 + hi) * A
    clipped = held < free
    loss, slope = -torch.minimum(free, held), torch.where(clipped, 0.0, -free)
    kl = torch.zeros_like(r)
    if ref is not None:
        d = ref.double() - logp
        kl = torch.exp(d) - d - 1
        if c:
            loss, slope = loss + c * kl, slope + c * (1 - torch.exp(d))
    z0 = torch.zeros_like(w)
    tot = lambda v: torch.where(live, w * v, z0).sum()  # noqa: E731
    coef = torch.where(live, w * slope / div, z0)
    g, tol = gradient(z, y, coef, T, live)
    return {"loss": tot(loss) / div, "count": tot(torch.ones_like(w)), "kl": tot(kl) / div, "clipped": tot(clipped.double()),
            "logprobs": torch.where(live, logp, z0), "grad": g, "grad_tol": tol, "live": live, "ratio": r, "w": w, "A": A,
            "coef": coef}


def preference(z, y, ref, cu, beta, eps, average, T, div):
    """z [S, T, V] (cu None) or [N, V] with cu a list of offsets."""
    logp, _ = row_values(z, y, T)
    live = y >= 0
    if cu is not None:
        inside = torch.zeros_like(live)
        inside[cu[0]:cu[-1]] = True
        live = live & inside
        parts = [(slice(a, b),) for a, b in zip(cu, cu[1:])]
    else:
        parts = [(i,) for i in range(z.shape[0])]
    S = len(parts)
    n = torch.stack([live[p].sum().double().clamp(min=1) if average else torch.ones((), dtype=torch.float64)
                     for p in parts]) if S else torch.zeros(0, dtype=torch.float64)
    s = torch.stack([torch.where(live[p], logp[p], 0.0).sum() for p in parts]) / n if S else n
    rewards = beta * (s - (ref.double() if ref is not None else 0.0))
    u = rewards[:S // 2] - rewards[S // 2:]
    F = torch.nn.functional
    loss = (-(1 - eps) * F.logsigmoid(u) - eps * F.logsigmoid(-u)).sum() / div
    du = beta * (eps * torch.sigmoid(u) - (1 - eps) * torch.sigmoid(-u)) / div
    per = torch.cat([du, -du]) / n
    coef = torch.zeros_like(logp)
    for p, c in zip(parts, per):
        coef[p] = c
    g, tol = gradient(z, y, coef, T, live)
    return {"loss": loss, "rewards": rewards, "logprobs": s, "grad": g, "grad_tol": tol, "live": live, "n": n, "u": u,
            "coef": coef}


def assert_close(got, want, tol, what):
    """|got - want| <= tol element by element; NaN and infinities have to be the same ones."""
    got, want = got.detach().cpu().double(), want.double()
    tol = torch.as_tensor(tol, dtype=torch.float64).expand(want.shape)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    odd = ~fin & ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd]), what
    off = (got - want).abs()[fin]
    bad = off > tol[fin]
    assert not bool(bad.any()), (what, int(bad.sum()), float((off / tol[fin].clamp(min=1e-300)).max()),
                                 float(off.max()))


def assert_rounded(got, want, tol, what):
    """`got` in its own type is `want` within tol, then rounded to that type."""
    half = torch.finfo(got.dtype).eps / 2
    assert_close(got, want, tol + half * (want.abs() + tol).nan_to_num(0.0) + torch.finfo(torch.float32).tiny, what)


def cpu_case(S, T, V, dtype, seed, prompt=0.25, std=2.0):
    """Logits and targets on the CPU: a few positions ignored, targets anywhere in the vocabulary."""
    gen = torch.Generator().manual_seed(seed)
    z = (torch.randn(S, T, V, generator=gen) * std).to(dtype)
    y = torch.randint(0, V, (S, T), generator=gen)
    up = torch.rand(S, T, generator=gen)
    z.scatter_add_(-1, y[..., None], (up * (math.log(V) + 3))[..., None].to(dtype))
    y[:, :int(prompt * T)] = -100
    return z, y, gen
