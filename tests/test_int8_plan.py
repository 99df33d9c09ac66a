"""How the 8-bit integer product is launched (ee_int8_plan, host only)."""
import ctypes
import random

import pytest

SMS = 148
# an SM's shared memory, and what every CTA takes of it beside its own
SM_BYTES, RESERVE = 228 * 1024, 1024


@pytest.fixture(scope="module")
def plan():
    from embodied_efficiency_b200 import _lib, build
    build.build()
    lib = _lib.load()

    def f(m, n, k, sms=SMS):
        t, c, s = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_size_t()
        assert lib.ee_int8_plan(m, n, k, sms, t, c, s) == 0
        return t.value, c.value, s.value
    return f


def _sizes(count):
    rng = random.Random(7)
    for _ in range(count):
        yield tuple(int(2 ** rng.uniform(a, b)) for a, b in ((0, 17), (0, 15))) + (16 * int(2 ** rng.uniform(0, 13)),)


def test_plan_refusals(plan):
    from embodied_efficiency_b200 import _lib
    lib = _lib.load()
    t, c, s = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_size_t()
    for args, rc in (((0, 8, 64, SMS), 2), ((1, 8, 40, SMS), 2), ((1, 8, 131072, SMS), 2), ((1, 8, 64, 0), 1)):
        assert lib.ee_int8_plan(*args, t, c, s) == rc
    assert lib.ee_int8_plan(1, 8, 64, SMS, None, c, s) == 1


def test_launches_fit_the_gpu(plan):
    for m, n, k in _sizes(20000):
        tokens, ctas, smem = plan(m, n, k)
        assert tokens in (16, 32, 64, 128, 256) and ctas in (1, 2, 4, 8) and smem <= SM_BYTES - RESERVE
        assert ctas == 2 or tokens < 256
        assert (k + 127) // 128 >= ctas or tokens == 256  # every slice of K holds a k-block


def test_no_cluster_beside_a_pair(plan):
    """A pair waits for all tensor memory of two SMs. A cluster of another stream's product, one of whose CTAs held
    some of it while another waited for a pair's, would never end and neither would the pair: no CTA of the kernel
    for few tokens may share an SM with one of a pair."""
    pair = plan(8192, 8192, 2048)
    assert pair[0] == 256
    least = min(plan(m, n, k)[2] for m in (1, 16, 30) for n in (128, 1024, 4096) for k in (16, 128, 1024))
    least = min([least] + [p[2] for p in (plan(*s) for s in _sizes(5000)) if p[0] < 256])
    assert pair[2] + least + 2 * RESERVE > SM_BYTES
