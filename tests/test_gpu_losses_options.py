"""Every combination of options that the measured calls of the losses draw from (perf/operators.py), at small sizes: the public
calls and the plain forms against the definition in 64 bits."""

import importlib.util
import itertools
from pathlib import Path

import pytest
import torch

from tests.loss_reference import U, assert_close, spread

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def _operators():
    spec = importlib.util.spec_from_file_location("measured_operators", ROOT / "perf" / "operators.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _options(op):
    """What draw() chooses between for this operator, all of it."""
    both = (False, True)
    keys = {"dtype": ("bf16", "fp32"), "masked": both, "temperature": (1.0, 0.7, 1.3), "layout": ("plain", "shifted")}
    if op in ("policy", "preference"):
        keys["ref"] = both
    if op == "policy":
        keys.update(weighted=both, per_token=both)
    if op == "preference":
        keys.update(layout=("plain", "shifted", "packed"), average=both, smoothing=(0.0, 0.1))
    for values in itertools.product(*keys.values()):
        yield dict(zip(keys, values))


def _case(op, S, T, V, o):
    return dict(op=op, dtype=o["dtype"], seqs=S, tokens=T, vocab=V, prompt=0.25, shifted=o["layout"] == "shifted",
                packed=o["layout"] == "packed", masked=min(64, V // 4) if o["masked"] else 0, temperature=o["temperature"],
                ref=o.get("ref", True), weighted=o.get("weighted", False), per_token=o.get("per_token", False),
                average=o.get("average", False), smoothing=o.get("smoothing", 0.0))


def _scales(c, st, want, S):
    """Per position: a bound of the gradient's coefficient and of its change with the log-probabilities, and what the sums
    and the rewards are off by. S: a position's logp (see tests/loss_reference.py), and u |x| three times over for the fp32
    reciprocal of the temperature, in x_y and in the others."""
    live = (st["targets"] >= 0).cpu()
    rows = torch.where(live, S, 0.0)
    if c["op"] == "logprobs":
        return None, rows, None, None
    if c["op"] == "backward":   # sum S: what the two exponentials of lse and logp are off by
        return st["grad_logprobs"].cpu().double().abs(), rows, None, None
    if c["op"] == "policy":
        lp = want["logprobs"].cpu()
        A = st["advantages"].cpu().double().abs()
        A = A if c["per_token"] else A[:, None].expand(live.shape)
        w = torch.ones_like(A) if st["weights"] is None else st["weights"].cpu().double()[:, None].expand(live.shape)
        r = torch.exp(lp - st["old_logprobs"].cpu().double())
        k = 0.04 * (1.0 + torch.exp(st["ref_logprobs"].cpu().double() - lp)) if c["ref"] else 0.0
        bound = torch.where(live, w * (A * r + k) / c["tokens"], 0.0)
        off = float((bound * (S + 8 * U)).sum())
        return bound, rows, off, off / 0.04   # the KL sum stands without its coefficient
    half = c["seqs"] / 2
    longest = c["tokens"]
    e = longest * float(rows.max())               # a sequence's sum; its mean is not farther off
    bound = torch.full(live.shape, 0.1 / half, dtype=torch.float64)   # du <= beta / D a pair
    return bound * (1.0 + 0.1 * 2 * e / 4 / float(rows.max())), rows, 0.2 * e, e


@pytest.mark.parametrize("size", [(4, 6, 40), (4, 3, 6001)], ids=str)
@pytest.mark.parametrize("op", ["logprobs", "backward", "policy", "preference"])
def test_every_combination_of_the_options(op, size):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    ops = _operators()
    n = 0
    for n, o in enumerate(_options(op)):
        c = _case(op, *size, o)
        what = str(o)
        want = ops.exact(c, n)
        st = ops.prepare(c, n)
        z, T = st["logits"].cpu(), c["temperature"]
        x = z.double() / T
        S = spread(z, T) + (3 * U * torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1) if T != 1.0 else 0.0)
        bound, rows, off, far = _scales(c, st, want, S)
        for own in (True, False):
            ops.own = own
            got = ops.run(st)
            assert got.keys() == want.keys()
            for k in got:
                w = want[k].double().cpu()
                half = U * w.abs() + 1e-30
                if k in ("logprobs", "lse") and op != "preference":
                    tol = rows + half
                elif k == "logprobs":
                    tol = far + half
                elif k == "rewards":
                    tol = 0.1 * far + half
                elif k in ("count", "clipped"):
                    tol = 4 * half
                elif k == "kl":
                    tol = far + half
                elif k == "loss":
                    tol = off + half
                else:
                    eps = torch.finfo(got[k].dtype).eps / 2
                    tol = (4 * bound * rows / T)[..., None] * (1 + eps) + eps * w.abs() + torch.finfo(torch.float32).tiny
                assert_close(got[k], w, tol, f"{'own' if own else 'plain'} {k} {what}")
    assert n + 1 == {"logprobs": 24, "backward": 24, "policy": 192, "preference": 288}[op]
