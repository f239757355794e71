"""CPU: more of what the draw, the 4-bit products and the gradient norm refuse or hand on before any launch."""
import ctypes as C
import sys
import threading
import time

import pytest
import torch

import albatross_b200 as ab
from albatross_b200 import _lib


def test_gradient_norm_refuses_scales_beyond_32_bits():
    one = (_lib.Grad * 1)(_lib.Grad(4096, 4096, 8, 0, 0))
    for scale in (1e39, 3.5e38, 1e300):
        assert _lib.lib.ab_clip_grad_norm(one, 1, scale, 1.0, 256, 256, None) == -1
        assert "scale" in _lib.lib.ab_last_error().decode()


def test_the_gradient_norm_lets_other_threads_run():
    """Threads change over only where one lets the interpreter's lock go: a call that keeps it leaves the other thread's count as it was."""
    count, stop, begun = [0], threading.Event(), threading.Event()

    def other():
        begun.set()
        while not stop.is_set():
            count[0] += 1
            time.sleep(0)

    def refused():
        try:
            ab.grad_norm([])            # after the list has been taken
        except RuntimeError:
            pass

    refused()                           # (what a first call sets up may let it go)
    interval, thread, ran = sys.getswitchinterval(), threading.Thread(target=other), 0
    sys.setswitchinterval(1000.0)
    try:
        thread.start()
        begun.wait()
        for _ in range(2000):
            before = count[0]
            refused()
            ran += count[0] - before
    finally:
        sys.setswitchinterval(interval)
        stop.set()
        thread.join()
    assert ran > 0


@pytest.mark.parametrize("zeros", [False, True])
def test_a_quantised_parameter_takes_no_part_in_gradients(zeros):
    """A layer's weight as it stands in the module: the scales do not carry its graph, with which linear_int4 would refuse them."""
    w = torch.nn.Linear(256, 16, bias=False).weight
    m, plain = ab.quantize_int4(w, 64, zeros), ab.quantize_int4(w.detach(), 64, zeros)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(m, plain))
    assert not any(t is not None and t.requires_grad for t in m) and not m.dequantize().requires_grad
    turned = ab.quantize_int4(w.detach().t().contiguous().t(), 64, zeros)          # in another order of memory
    assert all(a is b is None or (torch.equal(a, b) and b.is_contiguous()) for a, b in zip(m, turned))
