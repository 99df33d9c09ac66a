"""The bounded waits inside the tensor-core attention kernel: a walk over many keys is no reason to give up, and a
launch that does give up ends with a status and leaves the GPU usable."""
import pytest
import torch

pytestmark = pytest.mark.gpu

LIMIT_NS = 300_000


@pytest.fixture
def short_waits(cuda):
    from embodied_efficiency_b200 import _lib
    from embodied_efficiency_b200.wq_gemm import gemm_status
    assert gemm_status(reset=True) == 0
    lib = _lib.load()
    assert lib.ee_prompt_attention_wait_limit(LIMIT_NS) == 0
    yield lib
    lib.ee_prompt_attention_wait_limit(0)
    gemm_status(reset=True)


@pytest.mark.parametrize("hd", [64, 128])
def test_a_walk_longer_than_the_limit(short_waits, cuda, hd):
    """One item per SM that walks 1251 blocks of keys, a millisecond or more: its second tile is empty, and the last
    block has one key, so that two roles wait for the whole walk. Weights' and result's rounding to 16 bits, fp32 sums
    of nk / 16 steps (2^-24 each), scores to 2^-22 of sum |q k|, which moves a weight twice."""
    from embodied_efficiency_b200 import prompt_attention
    from embodied_efficiency_b200.wq_gemm import gemm_status
    nq, nk, heads = 100, 160001, torch.cuda.get_device_properties(cuda).multi_processor_count
    g = torch.Generator(device=cuda).manual_seed(hd)
    q = (torch.randn(nq, heads, hd, generator=g, device=cuda) * 1.5).bfloat16()
    k, v = (torch.randn(nk, 1, hd, generator=g, device=cuda).bfloat16() for _ in range(2))
    cu_q, cu_k = (torch.tensor([0, n], device=cuda, dtype=torch.int32) for n in (nq, nk))
    wide = [x.expand(nk, heads, hd) for x in (k, v)]
    prompt_attention(q[:, :1], k, v, cu_q, cu_k, causal=False)
    t = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    t[0].record()
    out = prompt_attention(q, *wide, cu_q, cu_k, causal=False)
    t[1].record()
    assert gemm_status() == 0
    assert t[0].elapsed_time(t[1]) * 1e6 > 2 * LIMIT_NS  # longer than the limit and a sleep of 0.2 ms, or nothing is shown
    kd, vd = k[:, 0].double(), v[:, 0].double()
    for h in (0, heads // 2, heads - 1):
        qd = q[:, h].double()
        p = torch.softmax(qd @ kd.T * hd ** -0.5, -1)
        ref, mean = p @ vd, p @ vd.abs()
        d = (qd.abs() @ kd.abs().T).amax(-1, keepdim=True) * (hd ** -0.5 * 2 ** -22)
        tol = 2 ** -8 * (mean + ref.abs()) * (1 + 2 ** -6) + mean * (2 * d + 2 ** -18 + nk * 2.0 ** -28)
        assert bool(((out[:, h].double() - ref).abs() <= tol).all())


def test_a_launch_that_gives_up(short_waits, cuda):
    """A million empty sequences take the kernel longer to look through than the limit lets its other roles wait for
    the first item. The launch ends by itself, says so, and the next one is right."""
    from embodied_efficiency_b200 import _lib, prompt_attention
    from embodied_efficiency_b200.wq_gemm import gemm_status
    n, heads, hd = 1 << 20, 128, 64
    tokens = 16 * n // heads + 128  # more than 16 rows a sequence: the tensor-core kernel
    q = torch.randn(tokens, 1, hd, device=cuda).bfloat16().expand(tokens, heads, hd)
    k, v = torch.randn(1, 1, hd, device=cuda).bfloat16(), torch.randn(1, 1, hd, device=cuda).bfloat16()
    cu_q, cu_k = torch.zeros(n + 1, device=cuda, dtype=torch.int32), torch.zeros(n + 1, device=cuda, dtype=torch.int32)
    cu_q[-1], cu_k[-1] = tokens, 1
    prompt_attention(q, k, v, cu_q, cu_k, causal=False)
    assert gemm_status(reset=True) == _lib.EE_ERR_TIMEOUT
    short_waits.ee_prompt_attention_wait_limit(0)
    out = prompt_attention(q, k, v, cu_q, cu_k, causal=False)
    assert gemm_status() == 0
    assert bool((out == v).all())  # one key: its value
