"""The operators beside other Python threads."""

import sys
import threading

import pytest
import torch

from f16acc_amd import fp8, moe

CPU = torch.zeros(4, 128)


@pytest.mark.parametrize("call", [
    lambda: fp8.quantize(CPU), lambda: fp8.quantize_weight(CPU), lambda: fp8.linear(CPU, CPU), lambda: moe.route(CPU, 2),
    lambda: fp8.mm(CPU, CPU, CPU, CPU), lambda: moe.experts(*[CPU] * 7)],
    ids=["quantize", "quantize_weight", "linear", "route", "mm", "experts"])
def test_the_interpreter_is_free_during_a_call(call):
    """Checks, allocation and launch let other threads run.  The thread that waits here never asks for the
    interpreter (the switch interval is longer than the test), so it gets it only where a call gives it up."""
    lock, passed = threading.Lock(), threading.Event()
    lock.acquire()

    def wait():
        with lock:
            passed.set()

    waiting = threading.Thread(target=wait)
    waiting.start()
    before = sys.getswitchinterval()
    sys.setswitchinterval(1000.0)
    try:
        lock.release()  # `waiting` wakes, and needs the interpreter to go on
        for _ in range(3000):
            with pytest.raises(ValueError):
                call()
            if passed.is_set():
                break
        assert passed.is_set()
    finally:
        sys.setswitchinterval(before)
        waiting.join()
