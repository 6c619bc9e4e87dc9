"""error_if_nonfinite waits for the device; other Python threads run meanwhile."""

import threading
import time

import pytest
import torch

import fussim_b200 as fb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inplace", [False, True])
def test_other_threads_run_during_the_wait(inplace):
    grads = [torch.randn(1000, device="cuda") for _ in range(3)]
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]

    def call():
        for p, g in zip(params, grads):
            p.grad = g.clone()
        if inplace:
            return fb.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
        return fb.clip_grad_norm(grads, 1.0, error_if_nonfinite=True)[1]

    want = call().item()
    ticks, done = [], threading.Event()

    def tick():
        while not done.is_set():
            ticks.append(time.monotonic())
            time.sleep(0.002)

    other = threading.Thread(target=tick)
    other.start()
    try:
        torch.cuda._sleep(1_000_000_000)  # about half a second of work on the stream
        begin = time.monotonic()
        norm = call()
        end = time.monotonic()
    finally:
        done.set()
        other.join()
    assert norm.item() == want
    assert end - begin >= 0.2
    assert sum(begin <= t <= end for t in ticks) >= 20
