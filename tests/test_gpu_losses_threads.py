"""Python threads beside calls of the losses on logits."""

import threading
import time

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_other_threads_run_while_a_call_waits_for_the_launch_queue():
    """More calls than the queue takes behind a kernel of about a second: the call that waits does not hold the interpreter."""
    from mote_b200 import policy_loss, preference_loss, token_logprobs, token_logprobs_backward
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    dev = torch.device("cuda", 0)
    z, y, f = torch.randn(2, 3, 8, device=dev), torch.zeros(2, 3, dtype=torch.int64, device=dev), torch.zeros(2, 3, device=dev)
    calls = [lambda: token_logprobs(z, y), lambda: token_logprobs_backward(z, y, f, f, f), lambda: policy_loss(z, y, f, f),
             lambda: preference_loss(z, y)]
    for call in calls:
        call()
    torch.cuda.synchronize()
    ticks, stop = [], threading.Event()

    def tick():
        while not stop.is_set():
            ticks.append(time.perf_counter())
            time.sleep(0.005)

    for call in calls:
        ticks.clear()
        stop.clear()
        t = threading.Thread(target=tick)
        t.start()
        torch.cuda._sleep(2_000_000_000)
        begin = time.perf_counter()
        for _ in range(3000):
            call()
        end = time.perf_counter()
        stop.set()
        t.join()
        torch.cuda.synchronize()
        seen = [begin] + [x for x in ticks if begin <= x <= end] + [end]
        assert end - begin > 0.5, "the queue did not fill"
        assert max(b - a for a, b in zip(seen, seen[1:])) < 0.25
