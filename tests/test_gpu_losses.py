"""The losses on logits on the GPU against their definitions in 64 bits (tests/loss_reference.py, where the tolerances are
derived): token log-probabilities and their backward pass, the clipped policy loss, the paired preference loss."""

import math

import pytest
import torch

from tests import loss_reference as ref
from tests.loss_reference import U, assert_close, assert_rounded, cpu_case

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
# (sequences, positions, vocabulary): a vocabulary of one, words, warps and 16-byte lines and one beside them, the byte
# vocabulary, the limits of the warp-per-rows kernels (4592 bf16 and 2296 fp32 logits), slices of one block and of clusters
# of 2 to 16, the longest fp32 row, and so many short rows that a warp takes several and their sums go through two stages
SIZES = [(1, 1, 1), (2, 3, 1), (9, 80, 271), (10, 3500, 33), (3, 5, 2), (2, 7, 3), (4, 9, 17), (2, 33, 64), (5, 31, 271), (1, 1, 271), (3, 2, 2296),
         (3, 2, 2297), (2, 2, 1100), (2, 3, 4592), (2, 2, 4593), (1, 3, 8193), (80, 2, 16384), (1, 2, 16391), (2, 80, 50021),
         (1, 1, 131072), (1, 1, 262144), (1, 2, 262160), (1, 1, 900864)]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda", 0)


def _same(a, b):
    return torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))


def _check_rows(r, z, y, T):
    logp, lse = ref.row_values(z, y, T)
    S = ref.spread(z, T)
    assert_close(r.logprobs, logp, (U * logp.abs() + S).nan_to_num(0.0, 0.0, 0.0), "logprobs")
    assert_close(r.lse, lse, (U * lse.abs() + S).nan_to_num(0.0, 0.0, 0.0), "lse")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_token_logprobs_and_their_backward(dev, size, dtype):
    from mote_b200 import token_logprobs, token_logprobs_backward
    S, T, V = size
    z, y, gen = cpu_case(S, T, V, dtype, 11 * V + T)
    for temperature in (1.0, 0.7):
        r = token_logprobs(z.to(dev), y.to(dev), temperature=temperature)
        _check_rows(r, z, y, temperature)
        g = torch.randn(S, T, generator=gen)
        d = token_logprobs_backward(z.to(dev), y.to(dev), r.logprobs, r.lse, g.to(dev), temperature=temperature)
        assert d.dtype == dtype and d.shape == z.shape and d.is_contiguous()
        want, tol = ref.gradient(z, y, g.double(), temperature, y >= 0)
        # the kept lse is fp32: another u |lse| in every probability, and as much in the exponent's split
        _, lse = ref.row_values(z, y, temperature)
        tol = tol + (want.abs() * 4 * U * (lse.abs() + 1)[..., None])
        assert_rounded(d, want, tol, "backward")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("V", [1, 2, 13, 271, 5003, 16400, 262160])
def test_strides_shifts_and_offsets(dev, V, dtype):
    """Shifted views, transposed positions, rows at odd offsets, an expanded sequence: the same bits as a contiguous copy,
    and per-position inputs of every stride."""
    from mote_b200 import policy_loss, token_logprobs, token_logprobs_backward
    S, T = (3, 6) if V < 10000 else (2, 2)
    z, y, gen = cpu_case(S, T + 1, V, dtype, V)
    z, y = z.to(dev), y.to(dev)
    pad = torch.zeros(S * (T + 1) * (V + 5) + 3, dtype=dtype, device=dev)
    wide = pad[3:].view(S, T + 1, V + 5)
    wide[..., 2:V + 2].copy_(z)
    views = [z[:, :-1], z[:, 1:], wide[..., 2:V + 2][:, :-1], z.transpose(0, 1).contiguous().transpose(0, 1)[:, :-1],
             z[:1, :-1].expand(S, T, V)]
    labels = [y[:, 1:], y[:, :-1], y.t().contiguous().t()[:, 1:], y[:, 1:], y[:, 1:]]
    g = torch.randn(T, S, generator=gen).to(dev).t()
    for v, l in zip(views, labels):
        assert V == 1 or not v.is_contiguous()
        a, b = token_logprobs(v, l), token_logprobs(v.contiguous(), l.contiguous())
        # another alignment groups the sum in another way: equal within the rows' tolerance
        want = ref.row_values(v.cpu(), l.cpu(), 1.0)[0]
        tol = U * want.abs() + ref.spread(v.cpu(), 1.0)
        assert_close(a.logprobs, want, tol, "strided")
        assert_close(b.logprobs, want, tol, "contiguous")
        da = token_logprobs_backward(v, l, b.logprobs, b.lse, g)
        db = token_logprobs_backward(v.contiguous(), l.contiguous(), b.logprobs, b.lse, g.contiguous())
        assert da.is_contiguous() and _same(da, db)   # elementwise: the same bits whatever the alignment
        adv = torch.randn(S, generator=gen).to(dev)
        old = (b.logprobs + 0.1).t().contiguous().t()
        p = policy_loss(v, l, adv, old, old - 0.05, kl_coef=0.1)
        w = ref.policy(v.cpu(), l.cpu(), adv.cpu(), old.cpu(), (old - 0.05).cpu(), None, 0.2, 0.2, 0.1, 1.0, 1.0)
        tol = w["grad_tol"] + (w["ratio"].abs() * w["A"].abs() + 0.2)[..., None] * (U * 8 + ref.spread(v.cpu(), 1.0)[..., None]) * 2
        assert_rounded(p.grad, w["grad"], tol, "policy strided")


@pytest.mark.parametrize("V", [271, 5003, 20000])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_masked_and_extreme_logits(dev, V, dtype):
    """-inf and lowest-value columns, a single finite logit, a row of -inf, very large logits, +inf and NaN, a target on a
    masked column, sure and hopeless targets; NaN and infinities in ignored positions change nothing."""
    from mote_b200 import token_logprobs, token_logprobs_backward
    gen = torch.Generator().manual_seed(V)
    z = torch.randn(1, 14, V, generator=gen).to(dtype)
    y = torch.randint(3, V - 3, (1, 14), generator=gen)
    low = torch.finfo(dtype).min
    z[0, 0, :V // 2] = -math.inf
    y[0, 0] = V - 2
    z[0, 1, 3:] = low
    y[0, 1] = 1
    z[0, 2, :] = -math.inf
    z[0, 2, 5] = 3.0
    y[0, 2] = 5                       # the only finite logit: logp 0, gradient 0
    z[0, 3, :] = -math.inf
    z[0, 3, 5] = 3.0
    y[0, 3] = 6                       # masked target: logp -inf
    z[0, 4, :] = -math.inf            # nothing at all: NaN
    z[0, 5, 7] = math.inf             # NaN
    z[0, 6, 7] = math.nan
    z[0, 7, y[0, 7]] = math.inf       # inf - inf: NaN
    z[0, 8] *= 1000.0
    z[0, 9, y[0, 9]] = 60.0           # sure: logp of about -V e^-60
    z[0, 10, y[0, 10]] = -120.0       # hopeless
    z[0, 11, :] = math.nan
    y[0, 11] = -100
    z[0, 12, :] = low                 # all the same lowest value: uniform
    y[0, 13] = V                      # no such column
    r = token_logprobs(z.to(dev), y.to(dev))
    logp, lse = ref.row_values(z, y, 1.0)
    S = ref.spread(z, 1.0)
    S[0, [1, 8]] += 4 * U * 1000 * 8  # x - m of this size is rounded before the exponential
    assert_close(r.logprobs, logp, (U * logp.abs() + S).nan_to_num(0.0, 0.0, 0.0), "logprobs")
    assert_close(r.lse, lse, (U * lse.abs() + S).nan_to_num(0.0, 0.0, 0.0), "lse")
    # a sure target's log-probability keeps its relative accuracy
    assert abs(float(r.logprobs[0, 9]) / float(logp[0, 9]) - 1) < float(S[0, 9]) + U
    assert float(r.logprobs[0, 11]) == 0.0 and float(r.lse[0, 11]) == 0.0
    g = torch.ones(1, 14)
    d = token_logprobs_backward(z.to(dev), y.to(dev), r.logprobs, r.lse, g.to(dev)).cpu()
    fine = [0, 1, 2, 3, 9, 10, 11, 12]
    want, tol = ref.gradient(z[:, fine], y[:, fine], g[:, fine].double(), 1.0, y[:, fine] >= 0)
    l = lse[:, fine].abs().clamp(max=1e30)[..., None].nan_to_num(0.0)
    tol = tol + want.abs() * 4 * U * (torch.where(l > 1e6, 0.0, l) + 1)
    keep = torch.tensor([True] * len(fine))
    keep[fine.index(12)] = False      # lse of lowest values: fp32 cannot hold lowest + log V, the probabilities follow it
    assert_rounded(d[:, fine][:, keep], want[:, keep], tol[:, keep], "backward")
    for i in (4, 5, 6, 7, 13):
        assert bool(torch.isnan(d[0, i]).any()), i
    assert not bool(d[0, 11].float().any())


def _policy_inputs(S, T, V, dtype, seed, per_token, weighted, with_ref):
    z, y, gen = cpu_case(S, T, V, dtype, seed)
    logp, _ = ref.row_values(z, y, 1.0)
    old = (logp + 0.25 * torch.randn(S, T, generator=gen)).float()
    rf = (logp + 0.5 * torch.randn(S, T, generator=gen)).float() if with_ref else None
    A = torch.randn((S, T) if per_token else (S,), generator=gen)
    w = None
    if weighted:
        w = torch.rand((S, T) if per_token else (S,), generator=gen) + 0.1
        w.view(-1)[::3] = 0.0
    # no ratio within reach of rounding of a border: the gradient jumps there
    r = torch.exp(logp - old.double())
    for b in (0.8, 1.3):
        old = torch.where((r / b - 1).abs() < 1e-3, old + 0.01, old)
    return z, y, A, old, rf, w, gen


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("per_token,weighted,with_ref", [(False, False, True), (True, True, True), (False, True, False)])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_policy_loss(dev, size, per_token, weighted, with_ref, dtype):
    from mote_b200 import policy_loss
    S, T, V = size
    z, y, A, old, rf, w, _ = _policy_inputs(S, T, V, dtype, 7 * V + T, per_token, weighted, with_ref)
    c = 0.04 if with_ref else 0.0
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    r = policy_loss(to(z), to(y), to(A), to(old), to(rf), weights=to(w), clip_low=0.2, clip_high=0.3, kl_coef=c, divisor=3.0)
    want = ref.policy(z, y, A, old, rf, w, 0.2, 0.3, c, 1.0, 3.0)
    Sp = ref.spread(z, 1.0)
    assert_close(r.logprobs, want["logprobs"], U * want["logprobs"].abs() + Sp, "logprobs")
    # the slope's own change with logp: |d slope / d logp| <= |A| r + c e^d, times logp's error before its rounding
    d = torch.zeros_like(want["ratio"]) if rf is None else torch.exp(rf.double() - ref.row_values(z, y, 1.0)[0])
    bend = want["w"] * (want["A"].abs() * want["ratio"] + c * d) / 3.0
    rows = torch.where(want["live"], bend * (Sp + 4 * U), 0.0)
    assert_rounded(r.grad, want["grad"], want["grad_tol"] + 2 * rows[..., None], "grad")
    n = max(1, S * T)
    scale = float((want["w"] * (want["A"].abs() * want["ratio"] + c * (d + 10)))[want["live"]].sum()) if n else 0.0
    assert_close(r.loss, want["loss"], scale / 3.0 * float(Sp.max() + 8 * U) + U * float(want["loss"].abs()) + 1e-30, "loss")
    assert_close(r.count, want["count"], U * float(want["count"]) + 1e-30, "count")
    assert_close(r.clipped, want["clipped"], U * float(want["clipped"]) + 1e-30, "clipped")
    klt = float((want["w"] * (d + 1))[want["live"]].sum()) / 3.0 * float(Sp.max() + 8 * U)
    assert_close(r.kl, want["kl"], klt + U * float(want["kl"]) + 1e-30, "kl")
    e = policy_loss(to(z), to(y), to(A), to(old), to(rf), weights=to(w), clip_low=0.2, clip_high=0.3, kl_coef=c, divisor=3.0,
                    grad=False)
    assert e.grad is None and _same(e.loss, r.loss) and _same(e.logprobs, r.logprobs)


def test_policy_loss_of_nothing(dev):
    """No sequences, no positions, all ignored, all weights 0."""
    from mote_b200 import policy_loss
    for S, T in ((0, 4), (3, 0), (0, 0)):
        z = torch.zeros(S, T, 271, device=dev)
        y = torch.zeros(S, T, dtype=torch.int64, device=dev)
        r = policy_loss(z, y, torch.zeros(S, device=dev), torch.zeros(S, T, device=dev))
        assert [float(v) for v in r[:4]] == [0.0] * 4 and r.grad.shape == z.shape and r.logprobs.shape == y.shape
    for V in (271, 6000, 300000):
        z = torch.full((2, 3, V), math.nan, device=dev)
        y = torch.full((2, 3), -100, dtype=torch.int64, device=dev)
        w = None
        for k in range(2):
            r = policy_loss(z, y, torch.full((2,), math.nan, device=dev), torch.full((2, 3), math.nan, device=dev), weights=w)
            assert [float(v) for v in r[:4]] == [0.0] * 4 and not bool(r.grad.any()) and not bool(r.logprobs.any()), (V, k)
            y, w = torch.zeros_like(y), torch.zeros(2, device=dev)


def test_policy_divisors(dev):
    from mote_b200 import policy_loss
    z, y, A, old, rf, w, _ = (t.to(dev) if isinstance(t, torch.Tensor) else t
                              for t in _policy_inputs(3, 8, 271, F32, 5, False, False, True))
    a = policy_loss(z, y, A, old, rf, kl_coef=0.1, divisor=8.0)
    b = policy_loss(z, y, A, old, rf, kl_coef=0.1, divisor=torch.tensor(8, device=dev))
    c = policy_loss(z, y, A, old, rf, kl_coef=0.1)
    assert all(_same(x, t) for x, t in zip(a, b))
    # a power of two: the same bits after scaling
    assert _same(a.grad * 8, c.grad) and _same(a.loss * 8, c.loss) and _same(a.kl * 8, c.kl) and _same(a.count, c.count)
    m = policy_loss(z, y, A, old, rf, kl_coef=0.0)   # the KL is measured only
    n = policy_loss(z, y, A, old)
    assert _same(m.grad, n.grad) and _same(m.loss, n.loss) and float(m.kl) > 0 and float(n.kl) == 0


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("average,eps,with_ref", [(False, 0.0, True), (True, 0.1, True), (False, 0.3, False)])
@pytest.mark.parametrize("size", [(2, 1, 1), (2, 3, 2), (6, 31, 271), (2, 300, 17), (4, 5, 5003), (2, 2, 50021),
                                  (2, 1, 262160)], ids=str)
def test_preference_loss_padded(dev, size, average, eps, with_ref, dtype):
    from mote_b200 import preference_loss
    S, T, V = size
    z, y, gen = cpu_case(S, T, V, dtype, 3 * V + T)
    y[0] = -100 if T > 4 else y[0]   # a chosen sequence without a counted position
    _check_preference(dev, z, y, None, average, eps, with_ref, gen)


def _check_preference(dev, z, y, cu, average, eps, with_ref, gen, div=2.0):
    from mote_b200 import preference_loss
    base = ref.preference(z, y, None, cu, 0.1, eps, average, 1.0, div)
    rf = (base["logprobs"] + (0.3 if average else 3.0) * torch.randn(base["logprobs"].shape, generator=gen)).float()
    rf = rf if with_ref else None
    want = ref.preference(z, y, rf, cu, 0.1, eps, average, 1.0, div)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev)
    r = preference_loss(to(z), to(y), to(rf), cu_seqlens=cut, beta=0.1, label_smoothing=eps, average=average, divisor=div)
    S = len(want["logprobs"])
    # a sequence's error: its positions' (summed in 64 bits), then one rounding
    Sp = ref.spread(z, 1.0)
    parts = [(slice(a, b),) for a, b in zip(cu, cu[1:])] if cu is not None else [(i,) for i in range(S)]
    es = torch.stack([torch.where(want["live"][p], Sp[p], 0.0).sum() for p in parts]) / want["n"]
    assert_close(r.logprobs, want["logprobs"], U * want["logprobs"].abs() + es, "logprobs")
    assert_close(r.rewards, want["rewards"], U * want["rewards"].abs() + 0.1 * es + 1e-30, "rewards")
    eu = 0.1 * (es[:S // 2] + es[S // 2:]) + 8 * U
    assert_close(r.loss, want["loss"], float(eu.sum()) / div + U * float(want["loss"]), "loss")
    # d coef / du <= beta / 4 a position (divided as the coefficient is)
    row = torch.zeros_like(Sp)
    for k, p in enumerate(parts):
        row[p] = 0.1 / div / 4 * eu[k % (S // 2)] / want["n"][k]
    tol = want["grad_tol"] + torch.where(want["live"], row + want["coef"].abs() * 8 * U, 0.0)[..., None]
    # the probabilities come from the kept fp32 lse
    lse = ref.row_values(z, y, 1.0)[1]
    tol = tol + want["grad"].abs() * 4 * U * (lse.abs() + 1)[..., None]
    assert_rounded(r.grad, want["grad"], tol, "grad")
    e = preference_loss(to(z), to(y), to(rf), cu_seqlens=cut, beta=0.1, label_smoothing=eps, average=average, divisor=div,
                        grad=False)
    assert e.grad is None and _same(e.loss, r.loss) and _same(e.logprobs, r.logprobs)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("V,cu,rows", [(271, [0, 5, 12, 12, 40], 48), (271, [3, 3, 9, 9, 10], 10), (17, [0, 300, 301], 350),
                                       (5003, [0, 1, 3, 7, 8], 9), (3, [0, 0, 0], 4), (20000, [1, 3, 5], 6)], ids=str)
def test_preference_loss_packed(dev, V, cu, rows, dtype):
    """Sequences of one position and of none, rows in front of the first and behind the last sequence that hold NaN."""
    z, y, gen = cpu_case(1, rows, V, dtype, V + rows)
    z, y = z[0], y[0]
    z[:cu[0]] = math.nan
    z[cu[-1]:] = math.nan
    clean = z.nan_to_num(0.0)
    want = ref.preference(clean, y, None, cu, 0.1, 0.0, False, 1.0, 2.0)
    from mote_b200 import preference_loss
    r = preference_loss(z.to(dev), y.to(dev), cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev), divisor=2.0)
    assert not bool(torch.isnan(r.grad).any()) and not bool(r.grad[:cu[0]].any()) and not bool(r.grad[cu[-1]:].any())
    assert not bool(r.grad.cpu()[~want["live"]].any())
    for average, eps, with_ref in ((False, 0.0, True), (True, 0.2, False)):
        _check_preference(dev, clean, y, cu, average, eps, with_ref, gen)


def test_preference_loss_of_nothing(dev):
    from mote_b200 import preference_loss
    r = preference_loss(torch.zeros(0, 4, 9, device=dev), torch.zeros(0, 4, dtype=torch.int64, device=dev))
    assert float(r.loss) == 0.0 and r.rewards.shape == (0,) and r.grad.shape == (0, 4, 9)
    r = preference_loss(torch.zeros(4, 0, 9, device=dev), torch.zeros(4, 0, dtype=torch.int64, device=dev), divisor=2.0)
    assert abs(float(r.loss) - math.log(2.0)) < 1e-6 and not bool(r.logprobs.any())
    z = torch.full((5, 9), math.nan, device=dev)
    r = preference_loss(z, torch.zeros(5, dtype=torch.int64, device=dev),
                        cu_seqlens=torch.tensor([2], dtype=torch.int32, device=dev))
    assert float(r.loss) == 0.0 and not bool(r.grad.any())


@pytest.mark.parametrize("V", [5, 6000])
def test_gradients_against_differences(dev, V):
    """Central differences of the losses themselves, in fp32: h = 1/8 (exact in fp32), the loss read to 2^-24 of its size over
    2h, the third derivative of a sum of log-softmax terms below |coefficients|, so h^2/6 of those."""
    from mote_b200 import policy_loss, preference_loss, token_logprobs, token_logprobs_backward
    z, y, gen = cpu_case(2, 3, V, F32, 77, prompt=0.0)
    z, y = z.to(dev), y.to(dev)
    A = torch.tensor([0.7, -1.1], device=dev)
    base = token_logprobs(z, y)
    old, rf = base.logprobs + 0.02, base.logprobs - 0.3
    gw = torch.randn(2, 3, generator=gen).to(dev)
    h = 0.125
    fns = {
        "policy": (lambda x: policy_loss(x, y, A, old, rf, kl_coef=0.2, clip_low=0.9, clip_high=9.0).loss,
                   policy_loss(z, y, A, old, rf, kl_coef=0.2, clip_low=0.9, clip_high=9.0).grad, 12.0),
        "preference": (lambda x: preference_loss(x, y, beta=0.5, label_smoothing=0.1).loss,
                       preference_loss(z, y, beta=0.5, label_smoothing=0.1).grad, 4.0),
        "logprobs": (lambda x: (token_logprobs(x, y).logprobs.double() * gw).sum(),
                     token_logprobs_backward(z, y, base.logprobs, base.lse, gw), float(gw.abs().max())),
    }
    cols = list(range(min(V, 5))) + [int(c) for c in y.unique()]
    for name, (f, grad, third) in fns.items():
        size = float(f(z).abs()) + (float((base.logprobs.abs() * gw.abs()).sum()) if name == "logprobs" else 4.0)
        tol = third * h * h / 6 + size * 64 * U / (2 * h) + 6 * 544 * U / (2 * h)
        for s in range(2):
            for t in range(3):
                for j in cols[:8]:
                    up, dn = z.clone(), z.clone()
                    up[s, t, j] += h
                    dn[s, t, j] -= h
                    fd = (float(f(up)) - float(f(dn))) / (float(up[s, t, j]) - float(dn[s, t, j]))
                    assert abs(fd - float(grad[s, t, j])) < tol, (name, s, t, j, fd, float(grad[s, t, j]), tol)


@pytest.mark.parametrize("V", [271, 5003, 40000, 262160])
def test_the_same_bits_every_time_and_on_any_stream(dev, V):
    from mote_b200 import policy_loss, preference_loss
    S, T = (8, 64) if V < 10000 else (4, 3)
    z, y, A, old, rf, w, _ = (t.to(dev) if isinstance(t, torch.Tensor) else t
                              for t in _policy_inputs(S, T, V, BF, V, False, False, True))
    first = policy_loss(z, y, A, old, rf, kl_coef=0.04)
    pref = preference_loss(z, y)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(dev) for _ in range(3)]
    got = []
    for k in range(6):   # calls in flight on three streams at once
        with torch.cuda.stream(side[k % 3]):
            got.append((policy_loss(z, y, A, old, rf, kl_coef=0.04), preference_loss(z, y)))
    torch.cuda.synchronize()
    for p, q in got:
        assert all(_same(a, b) for a, b in zip(p, first)) and all(_same(a, b) for a, b in zip(q, pref))


@pytest.mark.parametrize("V", [271, 40000, 262160])
def test_two_captured_graphs(dev, V):
    """Two graphs over the same inputs, replayed in turn and against eager calls, with new inputs copied in."""
    from mote_b200 import policy_loss, preference_loss, token_logprobs
    ins = [[t.to(dev) if isinstance(t, torch.Tensor) else t for t in _policy_inputs(4, 6, V, BF, 9 + k, False, False, True)[:5]]
           for k in range(3)]
    z, y, A, old, rf = (t.clone() for t in ins[0])
    count = torch.full((), 4.0, device=dev)
    policy_loss(z, y, A, old, rf, kl_coef=0.04, divisor=count)
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        a = policy_loss(z, y, A, old, rf, kl_coef=0.04, divisor=count)
    with torch.cuda.graph(gb):
        b = preference_loss(z, y)
        c = token_logprobs(z, y)
    for k in (1, 2, 0):
        for t, s in zip((z, y, A, old, rf), ins[k]):
            t.copy_(s)
        count.fill_(2.0 ** k)
        ga.replay()
        gb.replay()
        ga.replay()
        torch.cuda.synchronize()
        ea = policy_loss(*ins[k], kl_coef=0.04, divisor=2.0 ** k)
        eb, ec = preference_loss(*ins[k][:2]), token_logprobs(*ins[k][:2])
        for x, w in ((a, ea), (b, eb), (c, ec)):
            assert all(_same(p, q) for p, q in zip(x, w)), k
    del ga, gb


def test_a_post_training_step_through_the_optimizer(dev):
    """Reference and old log-probabilities, the policy loss and the preference loss of a small model, their gradients handed
    to autograd and the summed loss divided in the fused step: the same parameters as autograd's own loss gives."""
    from mote_b200 import AdamW, fused_step, policy_loss, preference_loss, token_logprobs
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(6, 9, 32, generator=gen).to(dev)
    y = torch.randint(0, 271, (6, 9), generator=gen)
    y[:, :2] = -100
    y = y.to(dev)
    A = torch.randn(6, generator=gen).to(dev)
    W0 = (0.3 * torch.randn(271, 32, generator=gen)).to(dev)
    Wr = (0.3 * torch.randn(271, 32, generator=gen)).to(dev)
    ref_lp = token_logprobs(x @ Wr.t(), y)
    old = token_logprobs(x @ W0.t(), y)
    for kind in ("policy", "preference"):
        ws = []
        for own in (True, False):
            W = torch.nn.Parameter(W0.clone())
            opt = AdamW([W], lr=1e-2, weight_decay=0.0)
            for _ in range(3):
                logits = x @ W.t()
                if kind == "policy" and own:
                    r = policy_loss(logits.detach(), y, A, old.logprobs, ref_lp.logprobs, kl_coef=0.05)
                    logits.backward(r.grad)
                    count = r.count
                elif kind == "policy":
                    lp = torch.log_softmax(logits, -1).gather(-1, y.clamp(min=0)[..., None])[..., 0]
                    ratio, d = torch.exp(lp - old.logprobs), ref_lp.logprobs - lp
                    per = -torch.minimum(ratio * A[:, None], ratio.clamp(0.8, 1.2) * A[:, None]) + 0.05 * (torch.exp(d) - d - 1)
                    count = (y >= 0).sum().float()
                    (per * (y >= 0)).sum().backward()
                elif own:
                    r = preference_loss(logits.detach(), y, ref_lp.logprobs.sum(-1))
                    logits.backward(r.grad)
                    count = torch.tensor(3.0, device=dev)
                else:
                    lp = torch.log_softmax(logits, -1).gather(-1, y.clamp(min=0)[..., None])[..., 0]
                    s = (lp * (y >= 0)).sum(-1) - ref_lp.logprobs.sum(-1)
                    count = torch.tensor(3.0, device=dev)
                    (-torch.nn.functional.logsigmoid(0.1 * (s[:3] - s[3:]))).sum().backward()
                fused_step(opt, max_norm=1.0, grad_divisor=count)
                opt.zero_grad(set_to_none=True)
            ws.append(W.detach().clone())
        moved = float((ws[1] - W0).norm())
        assert moved > 0.1 and float((ws[0] - ws[1]).norm()) < 1e-3 * moved, kind


def test_offsets_past_32_bits(dev):
    """A gradient of more than 2^32 elements from one expanded row, short rows and long ones, and rows of logits that lie more
    than 2^32 bytes apart."""
    from mote_b200 import policy_loss, token_logprobs, token_logprobs_backward
    if torch.cuda.get_device_properties(dev).total_memory < 60e9:
        pytest.skip("needs 60 GB")
    gen = torch.Generator().manual_seed(1)
    for V, n in ((131072, 33000), (272, 15_900_000)):
        z = torch.randn(1, V, generator=gen).to(BF).to(dev).expand(n, V)
        y = torch.full((n,), V - 3, device=dev)
        r = token_logprobs(z[:2], y[:2])
        lp, ls = r.logprobs[:1].expand(n), r.lse[:1].expand(n)
        d = token_logprobs_backward(z, y, lp, ls, torch.ones(1, device=dev).expand(n))
        assert d.numel() > 2 ** 32 and bool(d[0].any())
        assert _same(d[-1], d[0]) and _same(d[n // 2], d[0])
        p = policy_loss(z, y, torch.ones(n, device=dev), lp)
        assert _same(p.grad[-1], p.grad[0]) and float(p.count) == n and float(p.logprobs[-1]) == float(r.logprobs[0])
        del d, p
    base = torch.zeros((3 << 30) + 300, dtype=BF, device=dev)
    z = base.as_strided((3, 271), ((3 << 29) + 7, 1), 5)
    z.copy_(torch.randn(3, 271, generator=gen))
    y = torch.tensor([4, 200, 270], device=dev)
    want, _ = ref.row_values(z.cpu(), y.cpu(), 1.0)
    assert_close(token_logprobs(z, y).logprobs, want, U * want.abs() + ref.spread(z.cpu(), 1.0), "far rows")


def test_refusals(dev):
    from mote_b200 import policy_loss, preference_loss, token_logprobs
    from mote_b200._lib import MoteoptError
    z, y = torch.zeros(2, 3, 8, device=dev), torch.zeros(2, 3, dtype=torch.int64, device=dev)
    f = torch.zeros(2, 3, device=dev)
    bad = [(ValueError, lambda: token_logprobs(z.cpu(), y)), (TypeError, lambda: token_logprobs(z.half(), y)),
           (TypeError, lambda: token_logprobs(z, y.int())), (ValueError, lambda: token_logprobs(z, y[:, :2])),
           (ValueError, lambda: token_logprobs(z, y.cpu())), (ValueError, lambda: token_logprobs(z.transpose(1, 2), y)),
           (ValueError, lambda: token_logprobs(z[0, 0], y[0, 0])), (ValueError, lambda: token_logprobs(z[..., :0], y)),
           (MoteoptError, lambda: token_logprobs(z, y, temperature=0.0)),
           (MoteoptError, lambda: token_logprobs(z, y, temperature=-1.0)),
           (MoteoptError, lambda: token_logprobs(z, y, temperature=math.nan)),
           (MoteoptError, lambda: token_logprobs(z, y, temperature=math.inf)),
           (MoteoptError, lambda: token_logprobs(torch.zeros(1, 900865, device=dev), y[:1, 0])),
           (MoteoptError, lambda: token_logprobs(torch.zeros(1, 1801729, dtype=BF, device=dev), y[:1, 0])),
           (TypeError, lambda: policy_loss(z, y, f.double(), f)), (ValueError, lambda: policy_loss(z, y, f, f[0])),
           (ValueError, lambda: policy_loss(z, y, f[:, 0].cpu(), f)), (ValueError, lambda: policy_loss(z, y, f, f, kl_coef=0.1)),
           (MoteoptError, lambda: policy_loss(z, y, f, f, clip_low=-0.1)),
           (MoteoptError, lambda: policy_loss(z, y, f, f, divisor=0.0)),
           (MoteoptError, lambda: policy_loss(z, y, f, f, f, kl_coef=math.nan)),
           (ValueError, lambda: policy_loss(z, y, f, f, divisor=f)),
           (ValueError, lambda: preference_loss(z[:1], y[:1])), (ValueError, lambda: preference_loss(z[0], y[0])),
           (ValueError, lambda: preference_loss(z, y, cu_seqlens=torch.zeros(3, dtype=torch.int32, device=dev))),
           (TypeError, lambda: preference_loss(z[0], y[0], cu_seqlens=torch.zeros(3, dtype=torch.int64, device=dev))),
           (ValueError, lambda: preference_loss(z[0], y[0], cu_seqlens=torch.zeros(3, dtype=torch.int32))),
           (ValueError, lambda: preference_loss(z, y, f[0])),
           (MoteoptError, lambda: preference_loss(z, y, label_smoothing=1.5)),
           (MoteoptError, lambda: preference_loss(z, y, beta=math.inf))]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
