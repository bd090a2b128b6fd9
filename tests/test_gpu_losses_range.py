"""The losses on logits where fp32 ends: ratios and KL terms beyond e^88, logits far from 0, log-probabilities of one size and
logits of another. Tolerances: tests/loss_reference.py."""

import math

import pytest
import torch

from tests import loss_reference as ref
from tests.loss_reference import U, assert_close, assert_rounded, cpu_case
from tests.test_gpu_losses import BF, F32, dev  # noqa: F401

pytestmark = pytest.mark.gpu

# one cluster of tiles, many blocks of them, 32 lanes a row, slices of one block and of a cluster
ROWS = [(1, 24, 271), (40, 30, 271), (1, 24, 2200), (1, 24, 6000), (2, 12, 50021)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("size", ROWS, ids=str)
def test_policy_terms_beyond_fp32(dev, size, dtype):  # noqa: F811
    """Ratios of e^100 and e^300 with advantages -1, 0 and 1 and KL terms of e^100, with weights that keep what comes out of
    them in fp32's range (the coefficient of the log-probability need not be), beside ordinary rows."""
    from mote_b200 import policy_loss
    S, T, V = size
    z, y, gen = cpu_case(S, T, V, dtype, V + T, prompt=0.1)
    n = torch.arange(S * T).view(S, T)
    sure = n % 6 == 3   # a target of probability 1 - V e^-60: a coefficient of 2.7e43 times 1 - p is in range
    at = torch.where(sure, 60.0, z.float().gather(-1, y.clamp(min=0)[..., None])[..., 0])
    z.scatter_(-1, y.clamp(min=0)[..., None], at[..., None].to(dtype))
    z[..., -3:] = torch.where((y < V - 3)[..., None], -math.inf, z[..., -3:])   # columns of probability 0
    A = (n % 3 - 1).float()
    logp, _ = ref.row_values(z, y, 1.0)
    far = torch.where(n % 5 == 0, 300.0, 100.0)
    far = torch.where((A != 0) & (far > 200), 100.0, far)   # e^300 only where the advantage is 0
    ordinary = n % 4 == 1
    old = torch.where(ordinary, logp + 0.1, logp - far).float()
    rf = torch.where(ordinary | (n % 2 == 0), logp - 0.2, logp + 100.0).float()
    w = torch.where(ordinary | sure, 1.0, torch.where(n % 8 < 4, 1e-6, 1e-20)).float()   # 2.7e43 * 1e-6: above 2^112
    rf = torch.where(sure, (logp - 0.2).float(), rf)
    c, div = 0.04, 2.0
    to = lambda t: t.to(dev)  # noqa: E731
    r = policy_loss(to(z), to(y), to(A), to(old), to(rf), weights=to(w), clip_low=0.2, clip_high=0.3, kl_coef=c, divisor=div)
    want = ref.policy(z, y, A, old, rf, w, 0.2, 0.3, c, 1.0, div)
    assert bool(torch.isfinite(want["grad"]).all()) and float(want["coef"].abs().max()) > 1e43
    assert float(want["grad"].abs().max()) < 3e38 / (1 + 1 / 128)
    Sp = ref.spread(z, 1.0)
    d = torch.exp(rf.double() - logp)
    # e^x of a 64-bit difference rounded to fp32 would be off by 150 u at 300; it is of the log-probability's own error
    bend = torch.where(want["live"], want["w"] * (A.abs().double() * want["ratio"] + c * d) / div, 0.0)
    # a row's probabilities and its target's 1 - p, which its coefficient's error is multiplied by
    p = torch.softmax(z.double(), -1)
    share = torch.where(torch.arange(V) == y.clamp(min=0)[..., None], (1 - p).clamp(min=1e-12), p)
    tol = want["grad_tol"] + 2 * (bend * (Sp + 4 * U))[..., None] * share
    assert_rounded(r.grad, want["grad"], tol, "grad")
    assert not bool(r.grad[..., -3:].cpu()[(y < V - 3) & (y >= 0)].any())   # nothing times a probability of 0
    # a sure target keeps its relative accuracy, at the target and beside it
    rows = sure & (y >= 0) & (A < 0)
    assert bool(rows.any())
    # in 64 bits too a difference of 1 and p would be 0 there: 1 - p = -expm1(logp)
    exact = want["grad"].scatter(-1, y.clamp(min=0)[..., None], (-torch.expm1(logp) * want["coef"])[..., None])[rows]
    got = r.grad.cpu().double()[rows]
    rel = 8 * float(Sp.max()) + torch.finfo(dtype).eps / 2
    assert bool(((got - exact).abs() <= rel * exact.abs() + 1e-37).all())
    assert float(want["loss"]) > 1e39 and float(r.loss) == math.inf   # the sure rows' terms are no fp32 numbers
    w, div = torch.where(sure, 0.0, w), float(S * T)                  # the means of the others are
    r = policy_loss(to(z), to(y), to(A), to(old), to(rf), weights=to(w), clip_low=0.2, clip_high=0.3, kl_coef=c, divisor=div)
    want = ref.policy(z, y, A, old, rf, w, 0.2, 0.3, c, 1.0, div)
    scale = float((want["w"] * (A.abs().double() * torch.where(A < 0, want["ratio"], 1.3) + c * (d + 110)))[want["live"]].sum())
    assert_close(r.loss, want["loss"], scale / div * float(Sp.max() + 8 * U) + U * float(want["loss"].abs()), "loss")
    klt = float((want["w"] * (d + 110))[want["live"]].sum()) / div * float(Sp.max() + 8 * U)
    assert_close(r.kl, want["kl"], klt + U * float(want["kl"]), "kl")
    assert_close(r.count, want["count"], 2 * U * float(want["count"]), "count")
    assert_close(r.clipped, want["clipped"], 2 * U * float(want["clipped"]), "clipped")


@pytest.mark.parametrize("V", [271, 6000])
def test_an_advantage_of_zero_is_zero_whatever_the_ratio(dev, V):  # noqa: F811
    """A group whose rewards are all equal, with old log-probabilities that no longer fit: no loss and no gradient."""
    from mote_b200 import policy_loss
    z, y, _ = cpu_case(2, 6, V, F32, V, prompt=0.0)
    z, y = z.to(dev), y.to(dev)
    for low in (-100.0, -500.0, -2000.0, -3e38):
        r = policy_loss(z, y, torch.zeros(2, device=dev), torch.full((2, 6), low, device=dev))
        assert float(r.loss) == 0.0 and not bool(r.grad.any()) and float(r.count) == 12.0, low


def _far_rows(V, dtype, mask, gen):
    """Rows with a finite mask or far logits, and their targets."""
    z = torch.randn(1, 10, V, generator=gen)
    y = torch.randint(3, V - 3, (1, 10), generator=gen)
    z[0, 0] = mask                      # only the target
    z[0, 0, y[0, 0]] = 1.5
    z[0, 1, 3:] = mask                  # three columns, the target one of them
    y[0, 1] = 1
    z[0, 2, :2 * V // 3] = mask         # the first, the middle, the last columns
    y[0, 2] = V - 2
    z[0, 3, V // 5:4 * V // 5] = mask
    y[0, 3] = V - 1
    z[0, 4, V // 3:] = mask
    y[0, 4] = 0
    z[0, 5, y[0, 5]] = mask             # only the target is masked
    z[0, 6] = mask                      # all the same: uniform
    z[0, 7] = mask                      # a far target above a mask
    z[0, 7, y[0, 7]] = -mask
    z[0, 8, 2] = -mask                  # another column far above all
    z[0, 9] = mask                      # two of the same size above the mask
    z[0, 9, :2] = -mask
    y[0, 9] = 1
    return z.to(dtype), y


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("V", [60, 271, 2200, 6000, 50021, 300000])
@pytest.mark.parametrize("mask", [-2e5, -1e7, -1e9, -3e9, -1e10, -1e12, -1e15, -1e18, -1e30])
def test_masks_of_any_size(dev, mask, V, dtype):  # noqa: F811
    """A finite mask is as good as -inf, at every temperature: in the tiles, the pieces (whole ones that are masked), the
    slices. x = z times an fp32 reciprocal: 2 u of a difference and of lse."""
    from mote_b200 import policy_loss, preference_loss, token_logprobs, token_logprobs_backward
    z, y = _far_rows(V, dtype, mask, torch.Generator().manual_seed(V))
    zd, yd = z.to(dev), y.to(dev)
    one = torch.ones(1, 10)
    near = [0, 1, 2, 3, 4, 5]               # their lse is an ordinary number
    for T in (1.0, 0.3, 0.1):
        logp, lse = ref.row_values(z, y, T)
        S = ref.spread(z, T)
        r = token_logprobs(zd, yd, temperature=T)
        assert_close(r.logprobs, logp, 4 * U * logp.abs() + S, f"logprobs {T}")
        assert_close(r.lse, lse, 4 * U * lse.abs() + S, f"lse {T}")
        want, tol = ref.gradient(z, y, one.double(), T, y >= 0)
        kept = tol + want.abs() * 4 * U * torch.where(lse.abs() < 1e3, lse.abs() + 1, 1.0)[..., None] + 1e-30
        d = token_logprobs_backward(zd, yd, r.logprobs, r.lse, one.to(dev), temperature=T).cpu()
        assert not bool(torch.isnan(d).any()), T
        rows = near if T != 1.0 else near + [7, 8]   # at T = 1 their far lse is the logit itself, else it is a rounded number
        assert_rounded(d[:, rows], want[:, rows], kept[:, rows], f"backward {T}")
        # the policy loss at a ratio of 1: the gradient of the log-probability, and as exact where lse is far
        p = policy_loss(zd, yd, one.to(dev), r.logprobs, temperature=T, clip_high=1e9)
        ratio = want.abs() * (S + 4 * U * logp.abs().clamp(max=1.0))[..., None]
        fine = [i for i in range(10) if bool(torch.isfinite(logp[0, i])) and float(logp[0, i]) > -1e3]
        assert_rounded(p.grad.cpu()[:, fine], -want[:, fine], (tol + 2 * ratio + 1e-30)[:, fine], f"policy {T}")
        assert not bool(torch.isnan(p.grad).any()) and not bool(torch.isnan(p.loss))
        # the preference loss of two such sequences: a coefficient of 1/20 each, as far as their sums agree
        q = preference_loss(torch.cat([zd, zd]), torch.cat([yd, yd]), temperature=T)
        assert not bool(torch.isnan(q.grad).any()) and not bool(torch.isnan(q.loss))
        e = 0.1 * 2 * float(S.sum()) + 1e-6
        assert abs(float(q.loss) - math.log(2.0)) < e
        for s, sign in ((0, -0.05), (1, 0.05)):
            assert_rounded(q.grad.cpu()[s:s + 1, near], sign * want[:, near],
                           0.05 * (kept + 2 * e * want.abs())[:, near], f"preference {T}")


@pytest.mark.parametrize("V", [271, 2200, 6000, 70000])
@pytest.mark.parametrize("base,T", [(3e5, 1.0), (3e6, 1.0), (-2e4, 0.1), (3e9, 1e4)])
def test_far_logits_next_to_each_other(dev, base, T, V):  # noqa: F811
    """fp32 logits that differ by little and lie far from 0: their differences are exact, so are the results as accurate as
    those of the same logits at 0 (an fp32 product z / T would be off by half a unit of |z / T| log2 e)."""
    from mote_b200 import policy_loss, token_logprobs
    gen = torch.Generator().manual_seed(V)
    step = 2.0 ** math.floor(math.log2(abs(base)) - 23) * 2   # two units of the logits' last place
    k = torch.randint(0, 40, (2, 6, V), generator=gen)
    z = torch.tensor(base).double() + k.double() * step
    assert torch.equal(z.float().double(), z)
    y = torch.randint(0, V, (2, 6), generator=gen)
    r = token_logprobs(z.float().to(dev), y.to(dev), temperature=T)
    logp, lse = ref.row_values(z, y, T)
    S = ref.spread(z, T)
    assert_close(r.logprobs, logp, 3 * U * logp.abs() + S, "logprobs")
    assert_close(r.lse, lse, 4 * U * lse.abs() + S, "lse")
    p = policy_loss(z.float().to(dev), y.to(dev), torch.ones(2, device=dev), r.logprobs, temperature=T, clip_high=1e9)
    want, tol = ref.gradient(z, y, torch.ones(2, 6, dtype=torch.float64), T, y >= 0)
    assert_rounded(p.grad, -want, tol + (2 * S + 4 * U * logp.abs())[..., None] * want.abs(), "policy")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("size", [(4, 8, 64), (64, 32, 64), (2, 300, 256), (20, 8, 1024), (2, 4, 8192), (2, 3, 65536)], ids=str)
def test_the_preference_gradient_does_not_feel_where_the_logits_lie(dev, size, dtype):  # noqa: F811
    """Rows whose logits are one number L, around 2000: p = 1 / V, to what the kernels' exponentials are off by. An exponent
    (base 2) is rounded at most twice below 32, by 2^-20 each, here and in the sum behind lse: 4 ln 2 2^-20 in all, with 16 u
    for ex2 and the products. An fp32 lse is off by up to 2^-14, and the probabilities as much."""
    from mote_b200 import preference_loss
    S, T, V = size
    gen = torch.Generator().manual_seed(V)
    L = (2000.0 + 32 * torch.rand(S, T, 1, generator=gen)).to(dtype)
    lse = L.double() + math.log(V)
    assert float((lse.float().double() - lse).abs().max()) > 2.0 ** -17   # what an fp32 number would lose: above rel
    z = L.expand(S, T, V).contiguous()
    y = torch.randint(0, V, (S, T), generator=gen)
    r = preference_loss(z.to(dev), y.to(dev), divisor=1.0)
    coef = torch.where(torch.arange(S) < S // 2, -0.05, 0.05).double().view(S, 1, 1)
    one = torch.zeros(S, T, V, dtype=torch.float64).scatter_(-1, y[..., None], 1.0)
    want = coef * (one - 1.0 / V)
    # the coefficient: both sequences' sums are -T log V, off by T positions of S and by nothing else
    rel = 4 * math.log(2.0) * 2.0 ** -20 + 16 * U
    tol = want.abs() * (rel + 0.1 * 2 * T * rel)
    assert_rounded(r.grad, want, tol, "grad")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("V", [271, 2200, 6000, 50021, 300000])
def test_logits_farther_apart_than_fp32(dev, V, dtype):  # noqa: F811
    """A logit of 3e38 (1e36 and a temperature of 0.01) and the others ten times below it or at its negative: their difference
    in exponents is no fp32 number. The large one in the first, a middle and the last line of a row."""
    from mote_b200 import policy_loss, token_logprobs, token_logprobs_backward
    sure, lost = [0, 1, 2, 3, 4], [5, 6, 7, 8]   # rows whose target is the large one, and another
    for top, T in ((3e38, 1.0), (1e36, 0.01), (-1e35, 0.01)):
        z = torch.empty(1, 9, V)
        z[0] = top / 10 if top > 0 else top * 30
        z[0, 3:6] = -abs(top) * 10 if top < 0 else -top
        for r, j in enumerate((0, V // 2, V - 1) * 3):
            z[0, r, j] = top
        z = z.to(dtype)
        y = torch.tensor([[0, V // 2, V - 1, 0, V // 2, V - 2, V // 3, 1, 0]])
        r = token_logprobs(z.to(dev), y.to(dev), temperature=T)
        assert not bool(r.logprobs[0, sure].any()), (top, r.logprobs)   # of probability 1
        assert float(r.logprobs[0, lost].max()) <= -1e35, (top, r.logprobs)
        one = torch.ones(1, 9, device=dev)
        p = policy_loss(z.to(dev), y.to(dev), one, torch.zeros(1, 9, device=dev), temperature=T)
        assert torch.equal(p.logprobs, r.logprobs) and not bool(p.grad.any())   # the ratio is 0 where it is not sure
        d = token_logprobs_backward(z.to(dev), y.to(dev), r.logprobs, r.lse, one, temperature=T)
        if T == 1.0:   # their lse is an fp32 number
            want = torch.zeros(9, V)
            for i in lost:
                want[i, y[0, i]] = 1.0
                want[i, (0, V // 2, V - 1)[i % 3]] = -1.0
            assert torch.equal(d[0].float().cpu(), want)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("size", [(2, 6, 271), (2, 600, 60), (2, 6, 2200), (2, 6, 6000), (2, 3, 50021)], ids=str)
def test_coefficients_near_the_end_of_fp32(dev, size, dtype):  # noqa: F811
    """A gradient of 1e37 that reaches the log-probabilities, a beta of 1e37 whose pair's preference is wrong: their products
    with probabilities are fp32 numbers, 0 in columns of probability 0."""
    from mote_b200 import preference_loss, token_logprobs, token_logprobs_backward
    S, T, V = size
    z, y, _ = cpu_case(S, T, V, dtype, V, prompt=0.0)
    y = y % (V // 2)
    z[..., V // 2 + 3:] = -math.inf
    r = token_logprobs(z.to(dev), y.to(dev))
    lse = ref.row_values(z, y, 1.0)[1]
    g = torch.full((S, T), 1e37)
    want, tol = ref.gradient(z, y, g.double(), 1.0, y >= 0)
    tol = tol + want.abs() * 4 * U * (lse.abs() + 1)[..., None]
    d = token_logprobs_backward(z.to(dev), y.to(dev), r.logprobs, r.lse, g.to(dev))
    assert_rounded(d, want, tol, "backward")
    assert not bool(d[..., V // 2 + 3:].any())
    wrong = torch.tensor([1e3, -1e3], device=dev)   # u = beta (s_0 - s_1 - 2000): -beta sigmoid(-u) is -beta
    q = preference_loss(z.to(dev), y.to(dev), wrong, beta=1e37)
    sums = r.logprobs.double().sum(-1)
    assert float(sums[0] - sums[1]) < 1900
    sign = torch.tensor([-1.0, 1.0]).view(2, 1, 1)
    assert_rounded(q.grad, sign * want, tol, "preference")
    assert not bool(q.grad[..., V // 2 + 3:].any())
