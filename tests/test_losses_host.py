"""The losses on logits without a GPU: the C structures' layout, the entry points' refusals before any device call, the
workspace sizes, the torch binding's refusals, and the GPU tests' own oracle against autograd in 64 bits."""

import ctypes as C
import math
import subprocess
from pathlib import Path

import pytest
import torch

from tests import loss_reference as ref

ROOT = Path(__file__).resolve().parent.parent


def test_ctypes_structs_match_the_c_layout(tmp_path):
    from mote_b200 import _lib
    structs = {"moteopt_logits": _lib.Logits, "moteopt_positions": _lib.Positions, "moteopt_policy": _lib.Policy,
               "moteopt_preference": _lib.Preference}
    body = ""
    for name, cls in structs.items():
        body += f'printf("{name} %zu\\n", sizeof({name}));'
        for f, _ in cls._fields_:
            body += f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));'
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "moteopt.h"\nint main(void) {' + body + "return 0; }")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "p")],
                   check=True)
    out = subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout
    for line in out.splitlines():
        name, n = line.split()
        if "." in name:
            s, f = name.split(".")
            assert getattr(structs[s], f).offset == int(n), name
        else:
            assert C.sizeof(structs[name]) == int(n), name


def _logits(L, data=256, dtype=1, seqs=2, tokens=3, vocab=8):
    return L.Logits(data, dtype, seqs, tokens, vocab, tokens * vocab, vocab)


def test_entry_points_refuse_before_any_device_call():
    """Error codes and texts; the pointers are never followed."""
    from mote_b200 import _lib as L
    lib, text = L.lib, lambda: L.lib.moteopt_last_error().decode()
    y, f = L.Positions(256, 3, 1), L.Positions(256, 3, 1)
    none = L.Positions(None, 0, 0)

    def logprobs(z=None, y=y, t=1.0, out=256):
        return lib.moteopt_token_logprobs(_logits(L) if z is None else z, y, t, out, None, None, 0, None)

    bad = [(dict(z=_logits(L, dtype=2)), -1, "fp32 or bf16"), (dict(z=_logits(L, vocab=0)), -1, "shape"),
           (dict(z=_logits(L, seqs=-1)), -1, "shape"), (dict(z=_logits(L, data=None)), -1, "null"),
           (dict(z=_logits(L, data=257)), -1, "aligned"), (dict(y=L.Positions(260, 3, 1)), -1, "aligned"),
           (dict(y=none), -1, "null"), (dict(out=None), -1, "null"), (dict(t=0.0), -1, "temperature"),
           (dict(t=-1.0), -1, "temperature"), (dict(t=math.nan), -1, "temperature"), (dict(t=math.inf), -1, "temperature"),
           (dict(t=1e-300), -1, "temperature"), (dict(t=1e300), -1, "temperature"),
           (dict(z=_logits(L, seqs=1 << 14, tokens=1 << 14)), -3, "positions"),
           (dict(z=_logits(L, vocab=1801729)), -3, "bytes"), (dict(z=_logits(L, dtype=0, vocab=900865)), -3, "bytes"),
           (dict(z=_logits(L, vocab=5000)), -1, "workspace")]
    for kw, rc, words in bad:
        assert logprobs(**kw) == rc and words in text(), (kw, text())
    assert logprobs(z=_logits(L, seqs=0)) == 0 and logprobs(z=_logits(L, tokens=0)) == 0   # nothing to do

    z = _logits(L)
    assert lib.moteopt_token_logprobs_backward(z, y, 1.0, f, none, f, 256, None) == -1 and "null" in text()
    assert lib.moteopt_token_logprobs_backward(z, y, 1.0, f, f, f, None, None) == -1

    def policy(p=None, sums=256, logp=256, ws=None, size=0):
        p = p or L.Policy(f, f, f, none, 0.2, 0.2, 0.1, 1.0, None)
        return lib.moteopt_policy_loss(z, y, p, 1.0, sums, logp, 256, ws, size, None)

    for p, words in ((L.Policy(f, f, none, none, 0.2, 0.2, 0.1, 1.0, None), "reference"),
                     (L.Policy(none, f, f, none, 0.2, 0.2, 0.1, 1.0, None), "null"),
                     (L.Policy(f, f, f, none, -0.2, 0.2, 0.1, 1.0, None), "clips"),
                     (L.Policy(f, f, f, none, 0.2, math.nan, 0.1, 1.0, None), "clips"),
                     (L.Policy(f, f, f, none, 0.2, 0.2, math.inf, 1.0, None), "finite"),
                     (L.Policy(f, f, f, none, 0.2, 0.2, 0.1, 0.0, None), "divisor"),
                     (L.Policy(f, f, f, none, 0.2, 0.2, 0.1, math.nan, None), "divisor")):
        assert policy(p) == -1 and words in text(), text()
    assert policy(sums=None) == -1 and policy(logp=None) == -1
    need = lib.moteopt_policy_loss_workspace_size(z)
    assert policy() == -1 and "workspace" in text()
    assert policy(ws=128, size=need) == -1 and "aligned" in text()
    assert policy(ws=256, size=need - 1) == -1 and "small" in text()

    def preference(p, zz=z):
        return lib.moteopt_preference_loss(zz, y, p, 1.0, 256, 256, 256, 256, None, 0, None)

    for p, words in ((L.Preference(3, None, None, 0.1, 0.0, 0, 1.0, None), "pairs"),
                     (L.Preference(4, None, None, 0.1, 0.0, 0, 1.0, None), "match"),
                     (L.Preference(2, 256, None, 0.1, 0.0, 0, 1.0, None), "match"),
                     (L.Preference(2, None, None, math.nan, 0.0, 0, 1.0, None), "beta"),
                     (L.Preference(2, None, None, 0.1, 1.5, 0, 1.0, None), "label_smoothing"),
                     (L.Preference(2, None, None, 0.1, 0.0, 0, 0.0, None), "divisor"),
                     (L.Preference(2, None, None, 0.1, 0.0, 0, 1.0, None), "workspace")):
        assert preference(p) == -1 and words in text(), text()


def test_workspace_sizes():
    from mote_b200 import _lib as L
    lib = L.lib
    z = _logits(L, seqs=10, tokens=100, vocab=271)
    assert lib.moteopt_token_logprobs_workspace_size(z) == 256                  # short rows: the header alone
    assert lib.moteopt_policy_loss_workspace_size(z) >= 256 + 32 * 1000         # at most a row of partials a position
    assert lib.moteopt_preference_loss_workspace_size(z, 10) >= 256 + (8 + 4 + 4) * 1000 + 8 * 5
    wide = _logits(L, seqs=10, tokens=100, vocab=100000)
    pieces = lib.moteopt_token_logprobs_workspace_size(wide) - 256
    assert pieces >= 1000 * 8 * (100000 * 2 // 16 // 1024)                      # one (maximum, sum) a piece
    assert lib.moteopt_preference_loss_workspace_size(wide, 10) >= lib.moteopt_preference_loss_workspace_size(z, 10) + pieces - 512
    for bad in (_logits(L, vocab=0), _logits(L, seqs=-1), _logits(L, dtype=7), _logits(L, vocab=1 << 40),
                _logits(L, seqs=1 << 40, tokens=1 << 40)):
        assert lib.moteopt_token_logprobs_workspace_size(bad) == 0
        assert lib.moteopt_policy_loss_workspace_size(bad) == 0
        assert lib.moteopt_preference_loss_workspace_size(bad, 2) == 0
    assert lib.moteopt_preference_loss_workspace_size(z, -2) == 0


def test_the_binding_refuses_cpu_tensors_and_what_is_none():
    import mote_b200 as m
    z, y, f = torch.zeros(2, 3, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    for call in (lambda: m.token_logprobs(z, y), lambda: m.policy_loss(z, y, f, f), lambda: m.preference_loss(z, y),
                 lambda: m.token_logprobs_backward(z, y, f, f, f)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: m.token_logprobs(z.tolist(), y), lambda: m.token_logprobs(z, None),
                 lambda: m.token_logprobs(z.to(torch.float16), y), lambda: m.policy_loss(z.double(), y, f, f)):
        with pytest.raises(TypeError):
            call()


def test_the_oracle_against_autograd():
    """tests/loss_reference.py in 64 bits: its losses are torch's, its gradients autograd's."""
    gen = torch.Generator().manual_seed(2)
    S, T, V = 4, 5, 7
    z = torch.randn(S, T, V, generator=gen, dtype=torch.float64, requires_grad=True)
    y = torch.randint(0, V, (S, T), generator=gen)
    y[:, 0] = -100
    A, w = torch.randn(S, generator=gen), torch.rand(S, T, generator=gen)
    old = ref.row_values(z.detach(), y, 1.3)[0].float() + 0.3 * torch.randn(S, T, generator=gen)
    rf = old + 0.2
    live = y >= 0
    lp = torch.log_softmax(z / 1.3, -1).gather(-1, y.clamp(min=0)[..., None])[..., 0]
    r, d = torch.exp(lp - old.double()), rf.double() - lp
    per = -torch.minimum(r * A[:, None], r.clamp(0.8, 1.3) * A[:, None]) + 0.1 * (torch.exp(d) - d - 1)
    loss = (per * w * live).sum() / 3.0
    (g,) = torch.autograd.grad(loss, z, retain_graph=True)
    got = ref.policy(z.detach(), y, A, old, rf, w, 0.2, 0.3, 0.1, 1.3, 3.0)
    assert abs(float(got["loss"] - loss)) < 1e-6 and torch.allclose(got["grad"], g, atol=1e-7)   # A, w, old in fp32
    s = (lp * live).sum(-1) / live.sum(-1)
    u = 0.5 * ((s[:2] - s[2:]))
    F = torch.nn.functional
    loss = (-0.9 * F.logsigmoid(u) - 0.1 * F.logsigmoid(-u)).sum() / 2
    (g,) = torch.autograd.grad(loss, z)
    got = ref.preference(z.detach(), y, None, None, 0.5, 0.1, True, 1.3, 2.0)
    assert abs(float(got["loss"] - loss)) < 1e-12 and torch.allclose(got["grad"], g, atol=1e-12)
    flat = ref.preference(z.detach().reshape(-1, V), y.reshape(-1), None, [0, 5, 10, 15, 20], 0.5, 0.1, True, 1.3, 2.0)
    assert torch.equal(flat["grad"].reshape(S, T, V), got["grad"])
    # a sure target: the log-probability that a difference of logits and lse in 64 bits would lose
    z1 = torch.tensor([[60.0, 0.0, -1.0]], dtype=torch.float64)
    lp1 = float(ref.row_values(z1, torch.tensor([0]), 1.0)[0])
    assert abs(lp1 / -(math.exp(-60) + math.exp(-61)) - 1) < 1e-12
