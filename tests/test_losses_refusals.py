"""Calls of the losses on logits that are refused on the host, without a GPU."""

import pytest
import torch


def test_tensors_that_are_not_aligned_to_their_elements_are_refused():
    """Before any device call: the pointers are never followed. One pointer of the call is off by one or two bytes at a time."""
    from mote_b200 import _lib as L
    lib, text = L.lib, lambda: L.lib.moteopt_last_error().decode()
    for dtype, off in ((0, 2), (1, 1)):   # fp32 logits and their gradient, bf16 ones
        z = L.Logits(256, dtype, 2, 3, 8, 24, 8)
        y = L.Positions(256, 3, 1)
        pos = lambda bad: L.Positions(256 + 2 * bad, 3, 1)  # noqa: E731

        def logprobs(k):
            return lib.moteopt_token_logprobs(z, y, 1.0, 256 + 2 * (k == 0), 256 + 2 * (k == 1), None, 0, None)

        def backward(k):
            return lib.moteopt_token_logprobs_backward(z, y, 1.0, pos(k == 0), pos(k == 1), pos(k == 2), 256 + off * (k == 3),
                                                       None)

        def policy(k):
            p = L.Policy(pos(k == 0), pos(k == 1), pos(k == 2), pos(k == 3), 0.2, 0.2, 0.1, 1.0, 256 + 2 * (k == 4))
            return lib.moteopt_policy_loss(z, y, p, 1.0, 256 + 2 * (k == 5), 256 + 2 * (k == 6), 256 + off * (k == 7), None, 0,
                                           None)

        def preference(k):
            p = L.Preference(2, None, 256 + 2 * (k == 0), 0.1, 0.0, 0, 1.0, 256 + 2 * (k == 1))
            return lib.moteopt_preference_loss(z, y, p, 1.0, 256 + 2 * (k == 2), 256 + 2 * (k == 3), 256 + 2 * (k == 4),
                                               256 + off * (k == 5), None, 0, None)

        def packed(k):
            p = L.Preference(2, 256 + 2 * (k == 0), None, 0.1, 0.0, 0, 1.0, None)
            return lib.moteopt_preference_loss(L.Logits(256, dtype, 1, 6, 8, 0, 8), y, p, 1.0, 256, 256, 256, 256, None, 0, None)

        # without a GPU no call gets farther than its workspace, so this is what a call with aligned pointers says
        for call, n in ((backward, 4), (policy, 8), (preference, 6), (packed, 1), (logprobs, 2)):
            for k in range(n):
                assert call(k) == -1 and "aligned" in text(), (call.__name__, k, text())
        for call in (policy, preference, packed):
            assert call(-1) == -1 and "workspace" in text(), call.__name__


def test_forward_mode_tangents_are_refused():
    """The losses have no forward mode: a tangent is not dropped without a word."""
    import torch.autograd.forward_ad as fwd

    import mote_b200 as m
    z, y, f = torch.randn(2, 3, 8), torch.zeros(2, 3, dtype=torch.int64), torch.randn(2, 3)
    with fwd.dual_level():
        zd = fwd.make_dual(z, torch.ones_like(z))
        for call in (lambda: m.token_logprobs(zd, y), lambda: m.token_logprobs_backward(zd, y, f, f, f),
                     lambda: m.policy_loss(zd, y, f, f), lambda: m.preference_loss(zd, y)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        # the logits' own check, that they are on the GPU, comes later than this one
        with pytest.raises(ValueError, match="CUDA"):
            m.token_logprobs(zd.detach(), y)


def test_views_that_negate_when_they_are_read_are_refused():
    """The imaginary part of a conjugate: torch keeps the values and a flag."""
    import mote_b200 as m
    z, y = torch.randn(2, 3, 8, dtype=torch.complex64).conj().imag, torch.zeros(2, 3, dtype=torch.int64)
    assert z.is_neg()
    with pytest.raises(ValueError, match="resolve_neg"):
        m.token_logprobs(z, y)
    with pytest.raises(ValueError, match="CUDA"):
        m.token_logprobs(z.resolve_neg(), y)


@pytest.mark.gpu
def test_views_that_negate_are_refused_from_every_argument():
    import mote_b200 as m
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    dev = torch.device("cuda", 0)
    z, y, f = torch.randn(2, 3, 8, device=dev), torch.zeros(2, 3, dtype=torch.int64, device=dev), torch.zeros(2, 3, device=dev)
    n = torch.ones(2, 3, dtype=torch.complex64, device=dev).conj().imag
    for call in (lambda: m.policy_loss(z, y, n, f), lambda: m.policy_loss(z, y, f, n), lambda: m.policy_loss(z, y, f, f, n),
                 lambda: m.policy_loss(z, y, f, f, weights=n[:, 0]), lambda: m.token_logprobs_backward(z, y, f, f, n),
                 lambda: m.preference_loss(z, y, n[:, 0]), lambda: m.policy_loss(z, y, f, f, divisor=n[0, 0])):
        with pytest.raises(ValueError, match="resolve_neg"):
            call()


@pytest.mark.gpu
def test_forward_mode_tangents_of_the_other_arguments_are_refused():
    import torch.autograd.forward_ad as fwd

    import mote_b200 as m
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    dev = torch.device("cuda", 0)
    z, y, f = torch.randn(2, 3, 8, device=dev), torch.zeros(2, 3, dtype=torch.int64, device=dev), torch.randn(2, 3, device=dev)
    one = torch.ones((), device=dev)
    with fwd.dual_level():
        fd, s, d = fwd.make_dual(f, f), fwd.make_dual(f[:, 0].contiguous(), one.expand(2)), fwd.make_dual(one, one)
        for call in (lambda: m.policy_loss(z, y, fd, f), lambda: m.policy_loss(z, y, f, fd), lambda: m.policy_loss(z, y, f, f, fd),
                     lambda: m.policy_loss(z, y, f, f, weights=fd), lambda: m.token_logprobs_backward(z, y, f, f, fd),
                     lambda: m.preference_loss(z, y, s), lambda: m.policy_loss(z, y, f, f, divisor=d)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
