"""Calls of the losses on logits as a user's program makes them beside the plain ones: a first call inside a capture, a captured
training step, host threads, offsets beyond the rows, many pairs, targets without probability, broadcast inputs."""

import math
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from tests import loss_reference as ref
from tests.loss_reference import U, assert_close, assert_rounded, cpu_case
from tests.test_gpu_losses import BF, F32, _check_preference, _policy_inputs, _same, dev  # noqa: F401

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("size", [(600, 1, 33), (2, 256, 271), (64, 8, 60), (4, 16, 1100), (4, 16, 2200), (20, 3, 2200),
                                  (6, 90, 1100)], ids=str)
def test_preference_pairs_of_many_shapes(dev, size, dtype):  # noqa: F811
    """More pairs than one cluster takes, the most rows that it takes and one sequence more, 32 lanes a row."""
    S, T, V = size
    z, y, gen = cpu_case(S, T, V, dtype, S + V)
    _check_preference(dev, z, y, None, False, 0.1, True, gen)


@pytest.mark.parametrize("V", [33, 6000])
def test_packed_pairs_of_no_and_of_one_position(dev, V):  # noqa: F811
    """300 pairs, every third sequence empty."""
    lengths = [0 if q % 3 == 0 else 1 for q in range(600)]
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    z, y, gen = cpu_case(1, cu[-1], V, F32, V, prompt=0.0)
    _check_preference(dev, z[0], y[0], cu, True, 0.0, True, gen)


@pytest.mark.parametrize("V", [271, 6000])
def test_offsets_are_held_to_the_rows(dev, V):  # noqa: F811
    from mote_b200 import preference_loss
    z, y, _ = cpu_case(1, 12, V, BF, V)
    z, y = z[0].to(dev), y[0].to(dev)
    cut = lambda *c: torch.tensor(c, dtype=torch.int32, device=dev)  # noqa: E731
    want = preference_loss(z, y, cu_seqlens=cut(0, 5, 12))
    for wild in (cut(-7, 5, 12), cut(0, 5, 13), cut(-(2 ** 31), 5, 2 ** 31 - 1)):
        got = preference_loss(z, y, cu_seqlens=wild)
        assert all(_same(a, b) for a, b in zip(got, want))
    none = preference_loss(z[:0], y[:0], cu_seqlens=cut(4, 5, 7))   # no rows at all: log 2
    assert abs(float(none.loss) - math.log(2.0)) < 1e-6 and none.grad.shape == (0, V)
    # not ascending: a sequence that ends before it begins is empty
    r = preference_loss(z, y, cu_seqlens=cut(8, 3, 12))
    assert float(r.logprobs[0]) == 0.0 and math.isfinite(float(r.loss)) and not bool(r.grad[:8].any())


@pytest.mark.parametrize("V", [271, 6000])
def test_a_target_without_probability(dev, V):  # noqa: F811
    """A rejected target on a -inf column: the pair is decided, its loss and gradient are 0; with smoothing the loss is
    infinite. The ratio of such a position is 0."""
    from mote_b200 import policy_loss, preference_loss
    z = torch.randn(2, 3, V, generator=torch.Generator().manual_seed(V)).to(dev)
    y = torch.tensor([[1, 2, 3], [4, 5, 6]], device=dev)
    z[1, 1, 5] = -math.inf
    r = preference_loss(z, y)
    assert float(r.loss) == 0.0 and float(r.rewards[1]) == -math.inf and not bool(r.grad.any())
    assert float(preference_loss(z, y, label_smoothing=0.1).loss) == math.inf
    r = preference_loss(z.flip(0), y.flip(0), label_smoothing=1.0)
    assert float(r.loss) == 0.0 and not bool(r.grad.any())
    assert float(preference_loss(z.flip(0), y.flip(0)).loss) == math.inf
    old = torch.full((2, 3), -5.0, device=dev)
    p = policy_loss(z, y, torch.ones(2, device=dev), old, clip_high=1e9)
    assert float(p.logprobs[1, 1]) == -math.inf and math.isfinite(float(p.loss)) and not bool(p.grad[1, 1].any())
    assert bool(torch.isfinite(p.grad).all())


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("V", [271, 6000])
def test_backward_of_broadcast_and_zero_gradients(dev, V, dtype):  # noqa: F811
    from mote_b200 import token_logprobs, token_logprobs_backward
    z, y, gen = cpu_case(3, 5, V, dtype, V, prompt=0.0)
    z, y = z.to(dev), y.to(dev)
    g = torch.randn(3, generator=gen).to(dev)
    r = token_logprobs(z, y)
    want = token_logprobs_backward(z, y, r.logprobs, r.lse, g[:, None].expand(3, 5).contiguous())
    assert _same(token_logprobs_backward(z, y, r.logprobs, r.lse, g), want)
    assert _same(token_logprobs_backward(z, y, r.logprobs, r.lse, g[:, None].expand(3, 5)), want)
    # a position without a gradient is 0 whatever its logits hold, the others keep their bits
    g2 = g[:, None].repeat(1, 5)
    g2[1] = 0.0
    z2 = z.clone()
    z2[1] = math.nan
    r2 = token_logprobs(z2, y)
    assert bool(torch.isnan(r2.logprobs[1]).all())
    d = token_logprobs_backward(z2, y, r2.logprobs, r2.lse, g2)
    assert not bool(d[1].any()) and _same(d[0], want[0]) and _same(d[2], want[2])


def test_the_same_call_from_other_kinds_of_tensors(dev):  # noqa: F811
    """Logits that require a gradient, inference mode, expanded targets, a whole number for a temperature, one label for all."""
    from mote_b200 import policy_loss, token_logprobs
    z, y, A, old, rf, _, _ = (t.to(dev) if isinstance(t, torch.Tensor) else t
                              for t in _policy_inputs(4, 6, 271, F32, 2, False, False, True))
    want = policy_loss(z, y, A, old, rf, kl_coef=0.1)
    p = torch.nn.Parameter(z.clone())
    got = policy_loss(p, y, A, old, rf, kl_coef=0.1)
    assert all(_same(a, b) for a, b in zip(got, want)) and not got.loss.requires_grad and not got.grad.requires_grad
    p.backward(got.grad)
    assert _same(p.grad, want.grad)
    w = torch.ones((), device=dev, requires_grad=True)
    (w * got.loss).backward()   # the outputs are ordinary tensors
    assert _same(w.grad, want.loss)
    with torch.inference_mode():
        assert all(_same(a, b) for a, b in zip(policy_loss(z, y, A, old, rf, kl_coef=0.1), want))
    one = torch.full((1, 1), 9, device=dev).expand(4, 6)
    a, b = token_logprobs(z, one, temperature=2), token_logprobs(z, one.contiguous(), temperature=2.0)
    assert all(_same(s, t) for s, t in zip(a, b))
    got.loss.fill_(7.0)   # the four sums share a storage and not their elements
    assert _same(got.count, want.count) and _same(got.kl, want.kl)


@pytest.mark.parametrize("V", [271, 6000, 70000])
def test_temperatures_far_from_one(dev, V):  # noqa: F811
    """x is a product with the fp32 reciprocal: u |x| away from z / T, in x_y and in the others."""
    from mote_b200 import token_logprobs
    z, y, _ = cpu_case(2, 3, V, F32, V)
    for T in (0.01, 0.05, 40.0, 1e4):
        r = token_logprobs(z.to(dev), y.to(dev), temperature=T)
        logp, lse = ref.row_values(z, y, T)
        S = ref.spread(z, T) + 3 * U * (z.double().abs() / T).amax(-1)
        assert_close(r.logprobs, logp, U * logp.abs() + S, f"logprobs {T}")
        assert_close(r.lse, lse, U * lse.abs() + S, f"lse {T}")


@pytest.mark.parametrize("V", [271, 6000])
def test_policy_clips_without_a_border_and_negative_weights(dev, V):  # noqa: F811
    from mote_b200 import policy_loss
    z, y, A, old, rf, _, gen = _policy_inputs(3, 7, V, F32, V, True, False, True)
    w = torch.randn(3, 7, generator=gen)
    for lo, hi in ((math.inf, math.inf), (1.0, math.inf), (2.0, 0.3), (0.2, 1e6)):
        r = policy_loss(z.to(dev), y.to(dev), A.to(dev), old.to(dev), weights=w.to(dev), clip_low=lo, clip_high=hi)
        want = ref.policy(z, y, A, old, None, w, lo, hi, 0.0, 1.0, 1.0)
        bend = (want["w"].abs() * want["A"].abs() * want["ratio"])
        Sp = ref.spread(z, 1.0)
        rows = torch.where(want["live"], bend * (Sp + 4 * U), 0.0)
        assert_rounded(r.grad, want["grad"], want["grad_tol"] + 2 * rows[..., None], f"grad {lo} {hi}")
        scale = float(bend[want["live"]].sum())
        assert_close(r.loss, want["loss"], scale * (float(Sp.max()) + 8 * U) + U * float(want["loss"].abs()), f"loss {lo} {hi}")


@pytest.mark.parametrize("V", [271, 20000])
def test_calls_from_several_threads(dev, V):  # noqa: F811
    from mote_b200 import policy_loss, preference_loss
    ins = [[t.to(dev) if isinstance(t, torch.Tensor) else t for t in _policy_inputs(6, 20, V, BF, 3 + k, False, False, True)[:5]]
           for k in range(3)]
    want = [(policy_loss(*i, kl_coef=0.04), preference_loss(*i[:2])) for i in ins]
    torch.cuda.synchronize()
    got = [[] for _ in ins]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream(dev)):
            for _ in range(20):
                got[k].append((policy_loss(*ins[k], kl_coef=0.04), preference_loss(*ins[k][:2])))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for k in range(3):
        assert len(got[k]) == 20
        for p, q in got[k]:
            assert all(_same(a, b) for a, b in zip(p, want[k][0])) and all(_same(a, b) for a, b in zip(q, want[k][1]))


def test_a_captured_step_with_its_backward_pass(dev):  # noqa: F811
    """Model, loss, backward pass and their replay with new inputs: the gradient of an eager step, to the bit."""
    from mote_b200 import policy_loss
    gen = torch.Generator().manual_seed(4)
    xs = [torch.randn(4, 6, 32, generator=gen).to(dev) for _ in range(3)]
    y = torch.randint(-2, 271, (4, 6), generator=gen).to(dev)
    A, old = torch.randn(4, generator=gen).to(dev), torch.full((4, 6), -5.5, device=dev)
    W = torch.nn.Parameter((0.3 * torch.randn(271, 32, generator=gen)).to(dev))
    x = xs[0].clone()

    def step():
        logits = x @ W.t()
        r = policy_loss(logits.detach(), y, A, old)
        logits.backward(r.grad)
        return r.loss

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
            W.grad = None
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    kept = W.grad
    for v in (xs[1], xs[2], xs[0]):
        x.copy_(v)
        kept.zero_()
        graph.replay()
        torch.cuda.synchronize()
        a, b = kept.clone(), loss.clone()
        W.grad = None
        want = step()
        assert _same(b, want) and _same(a, W.grad)
    del graph


_FIRST = """
import torch, mote_b200 as m
d = torch.device("cuda", 0)
gen = torch.Generator(device=d).manual_seed(1)
ins = {V: (torch.randn(4, 3, V, generator=gen, device=d), torch.randint(0, V, (4, 3), generator=gen, device=d),
           torch.ones(4, device=d), torch.full((4, 3), -5.0, device=d)) for V in (271, 900, 5000, 40000)}
torch.cuda.synchronize()
def calls():
    return [t for z, y, A, old in ins.values() for r in (m.policy_loss(z, y, A, old), m.preference_loss(z, y), m.token_logprobs(z, y))
            for t in r if t is not None]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = calls()
g.replay()
torch.cuda.synchronize()
got = [t.clone() for t in got]
want = calls()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("same")
"""


def test_the_first_call_of_a_process_may_be_captured(dev):  # noqa: F811
    r = subprocess.run([sys.executable, "-c", _FIRST], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]
