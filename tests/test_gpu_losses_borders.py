"""Every element of a row counts once, and nothing beside it does: one logit far above the others, in turn at each column (of
short rows) or on both sides of each place where a long row may be cut, at every alignment of a row, the target next to it, and
far larger values in the elements beside the row. A lost logit shows as an lse of -60 + log V, one counted twice as log 2, a
value from beside the row as 80 or NaN; the tolerances of rows of ordinary logits would hide one of thousands."""

import math

import pytest
import torch

from tests.loss_reference import U
from tests.test_gpu_losses import BF, F32, dev  # noqa: F401

pytestmark = pytest.mark.gpu

LOW = -60.0
S = (4 + 2 * 60 + 512 + 32) * U   # tests/loss_reference.py: the logits' range is 60
TINY = 1e6 * math.exp(LOW)        # all the other logits together


def _columns(V, size):
    """Columns to stand out: all of a short row, else both ends and 6 on each side of every 32nd line of 16 bytes (batches,
    pieces and slices of a row are cut at lines, counted from the row's first one or from its output's)."""
    if V * size <= 10000:
        return torch.arange(V)
    near = torch.arange(-14, 6)
    at = torch.arange(0, V + 1, 512 // size)[:, None] + near
    ends = torch.cat([torch.arange(24), torch.arange(V - 24, V)])
    return torch.cat([at.flatten(), ends]).clamp(0, V - 1).unique()


def _rows(cols, V, dtype, dev):  # noqa: F811
    """A row for each of `cols`, its begin 3 elements of 16 bytes' worth farther than the row before: all alignments in turn.
    The target is the next column, or the one before."""
    n = cols.numel()
    pitch = V + 24 - (V + 24) % 8 + 3
    buf = torch.full((n * pitch + 64,), 80.0, dtype=dtype, device=dev)
    z = buf.as_strided((n, V), (pitch, 1), 16)
    z.fill_(LOW)
    y = torch.where((torch.arange(n) % 2 == 0) & (cols + 1 < V) | (cols == 0), cols + 1, cols - 1).to(dev)
    c = cols.to(dev)
    z.scatter_(1, c[:, None], 0.0)
    return z, y, c


def _check(z, y, c):
    from mote_b200 import policy_loss, preference_loss, token_logprobs, token_logprobs_backward
    n = z.shape[0]
    ones = torch.ones(n, device=z.device)

    def lse_is(lse, what):
        assert float((lse - 0.0).abs().max()) <= S + TINY, (what, int((lse.abs() > S + TINY).nonzero()[0]))

    def grad_is(g, coef, what):   # coef (1 at the target, -1 at the column), all others below TINY
        half = torch.finfo(g.dtype).eps / 2
        g = g.float()
        at, top = g.gather(1, y[:, None])[:, 0], g.gather(1, c[:, None])[:, 0]
        assert float((at - coef).abs().max()) <= (2 * S + half) * 1.01 * float(coef.abs().max()) + TINY, what
        assert float((top + coef).abs().max()) <= (2 * S + half) * 1.01 * float(coef.abs().max()) + TINY, what
        g.scatter_(1, y[:, None], 0.0)
        g.scatter_(1, c[:, None], 0.0)
        assert float(g.abs().max()) <= TINY, what

    r = token_logprobs(z, y)
    lse_is(r.lse, "forward")
    lse_is(LOW - r.logprobs.double(), "forward logp")
    grad_is(token_logprobs_backward(z, y, r.logprobs, r.lse, ones), ones, "backward")
    p = policy_loss(z, y, ones, r.logprobs)
    lse_is(LOW - p.logprobs.double(), "policy logp")
    grad_is(p.grad, -ones, "policy")
    lse_is(LOW - policy_loss(z, y, ones, r.logprobs, grad=False).logprobs.double(), "policy without a gradient")
    k = n - n % 2
    if k:
        cu = torch.tensor([0, k // 2, k], dtype=torch.int32, device=z.device)
        q = preference_loss(z[:k], y[:k], cu_seqlens=cu, beta=0.001)
        u = float(q.rewards[0] - q.rewards[1])
        w = 0.001 / (1.0 + math.exp(u))
        coef = torch.full((k,), -w, device=z.device)
        coef[k // 2:] = w
        half = torch.finfo(q.grad.dtype).eps / 2
        g = q.grad.float()
        for at, sign in ((y, 1.0), (c, -1.0)):
            got = g.gather(1, at[:k, None])[:, 0]
            assert float((got - sign * coef).abs().max()) <= w * (3 * S + half + 1e-6) * 1.01, "preference"
            g.scatter_(1, at[:k, None], 0.0)
        assert float(g.abs().max()) <= TINY, "preference"


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("V", [2, 9, 17, 60, 128, 129, 271, 320, 1100, 2200, 2296, 2297, 4592, 4593, 8193, 16391, 50021, 131080,
                               262160, 600000])
def test_every_element_counts_once(dev, V, dtype):  # noqa: F811
    gen = torch.Generator().manual_seed(V)
    size = 2 if dtype == BF else 4
    cols = _columns(V, size)
    most = (1 << 29) // (V * size)             # rows a call: half a GB
    eight = cols.repeat_interleave(8)          # each at every alignment
    pick = eight if eight.numel() <= 2 * most else eight[torch.randperm(eight.numel(), generator=gen)[:2 * most].sort()[0]]
    for a in range(0, pick.numel(), most):
        _check(*_rows(pick[a:a + most], V, dtype, dev))
    # few rows at once: one cluster, slices of up to 16 blocks a row
    for n in (1, 3, 6, 30):
        for _ in range(6):
            few = cols[torch.randint(0, cols.numel(), (n,), generator=gen)]
            _check(*_rows(few, V, dtype, dev))


@pytest.mark.parametrize("V", [6000, 50021])
def test_gradients_against_differences_where_they_are_large(dev, V):  # noqa: F811
    """Six columns far apart share a long row: p is about 1/6 at each, well above what a difference is off by. h = 1/8: h^2 / 6
    times the third derivative, at most 1/4 of the coefficients, and the loss read to S over 2 h."""
    from mote_b200 import policy_loss, preference_loss, token_logprobs, token_logprobs_backward
    gen = torch.Generator().manual_seed(V)
    z = torch.full((2, 2, V), LOW)
    cols = torch.tensor([0, 5, V // 3, V // 2 + 1, V - 9, V - 1])
    z[..., cols] = 0.5 * torch.rand(2, 2, 6, generator=gen)
    z, y = z.to(dev), cols[torch.tensor([[1, 5], [0, 3]])].to(dev)
    A = torch.tensor([0.9, -1.1], device=dev)
    base = token_logprobs(z, y)
    old, gw = base.logprobs + 0.02, torch.tensor([[1.0, -0.7], [0.5, 1.3]], device=dev)
    h = 0.125
    fns = {
        "policy": (lambda x: policy_loss(x, y, A, old, old - 0.2, kl_coef=0.2, clip_low=0.9, clip_high=9.0).loss,
                   policy_loss(z, y, A, old, old - 0.2, kl_coef=0.2, clip_low=0.9, clip_high=9.0).grad, 2.0),
        "preference": (lambda x: preference_loss(x, y, beta=0.9).loss, preference_loss(z, y, beta=0.9).grad, 2.0),
        "logprobs": (lambda x: (token_logprobs(x, y).logprobs.double() * gw).sum(),
                     token_logprobs_backward(z, y, base.logprobs, base.lse, gw), 1.3),
    }
    for name, (f, grad, third) in fns.items():
        tol = third / 4 * h * h + 2 * 8 * S / (2 * h)
        for s in range(2):
            for t in range(2):
                for j in cols.tolist():
                    up, dn = z.clone(), z.clone()
                    up[s, t, j] += h
                    dn[s, t, j] -= h
                    fd, g = (float(f(up)) - float(f(dn))) / (2 * h), float(grad[s, t, j])
                    assert abs(fd - g) < tol and abs(g) > 2.5 * tol, (name, s, t, j, fd, g, tol)


@pytest.mark.parametrize("V", [271, 2200, 4700])
def test_the_mean_error_of_many_positions(dev, V):  # noqa: F811
    """ex2's own mean error of 5.05e-8 is taken out of a row's sum: over 32768 positions half of it would show. The mean's own
    noise is that of fp32's rounding of a logp between 4 and 32, at most 5.5e-7 / sqrt(32768) = 3e-9, and as much again of the
    exponents' rounding in a row."""
    from mote_b200 import policy_loss, token_logprobs
    gen = torch.Generator(device=dev).manual_seed(V)
    z = torch.randn(32768, V, generator=gen, device=dev) * 2
    y = torch.randint(0, V, (32768,), generator=gen, device=dev)
    want = torch.cat([torch.log_softmax(b.double(), -1).gather(1, t[:, None])[:, 0] for b, t in zip(z.split(4096), y.split(4096))])
    ones = torch.ones(32768, device=dev)
    for got in (token_logprobs(z, y).logprobs, policy_loss(z, y, ones, ones).logprobs):
        assert abs(float((got.double() - want).mean())) < 2.5e-8
