"""The native host side and the interpreter's other threads."""
import ctypes
import threading
import time

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_launch_that_waits_lets_other_threads_run(cuda):
    """A stream that is held up for 0.9 seconds by a host function (libc's usleep: it needs no interpreter) takes
    about a thousand launches; the next launch waits for it on the host. Other Python threads go on meanwhile."""
    from embodied_efficiency_b200 import quantize_tokens
    cudart, libc = ctypes.CDLL("libcudart.so.12"), ctypes.CDLL(None)
    launch = cudart.cudaLaunchHostFunc
    launch.argtypes, launch.restype = [ctypes.c_void_p] * 3, ctypes.c_int
    x = torch.randn(4, 64, device=cuda).bfloat16()
    want = quantize_tokens(x)[0]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    gaps, stop = [0.0], threading.Event()

    def tick():
        last = time.perf_counter()
        while not stop.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            gaps.append(now - last)
            last = now

    other = threading.Thread(target=tick)
    other.start()
    try:
        with torch.cuda.stream(side):
            start = time.perf_counter()
            assert launch(side.cuda_stream, ctypes.cast(libc.usleep, ctypes.c_void_p), 900_000) == 0
            for _ in range(5000):
                got = quantize_tokens(x)[0]
            took = time.perf_counter() - start
    finally:
        stop.set()
        other.join()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert took > 0.6, "no launch had to wait: nothing is shown"
    assert max(gaps) < 0.3, max(gaps)
