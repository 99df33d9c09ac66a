"""The bounded waits of attention over a paged cache: they go by the limit that the caller sets, a walk over many keys is no
reason to give up, and a launch that does give up ends with a status and leaves the GPU usable."""
import pytest
import torch

from test_gpu_cache import codes_of
from test_gpu_prompt_waits import LIMIT_NS, short_waits  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,bits", [(64, 8), (128, 4)])
def test_a_walk_longer_than_the_limit(short_waits, cuda, hd, bits):  # noqa: F811
    """One item per SM that walks 1251 blocks of keys. Weights' and result's rounding to 16 bits, fp32 sums of nk / 16
    steps (2^-24 each), scores to 2^-22 of sum |q k|, which moves a weight twice."""
    from embodied_efficiency_b200 import KVCache, cache_attention
    from embodied_efficiency_b200.wq_gemm import gemm_status
    nq, nk, page, heads = 100, 160001, 64, torch.cuda.get_device_properties(cuda).multi_processor_count
    g = torch.Generator(device=cuda).manual_seed(hd)
    pages = -(-nk // page)
    cache = KVCache.empty(pages, heads, hd, page, bits)
    for t in (cache.k, cache.v):
        t.random_(-127, 128, generator=g) if bits == 8 else t.random_(0, 256, generator=g)
    for t in (cache.k_scale, cache.v_scale):
        t.fill_(0.0136 if bits == 8 else 0.22)  # of deviation 1
    q = (torch.randn(nq, heads, hd, generator=g, device=cuda) * 1.5).bfloat16()
    table = torch.arange(pages, device=cuda, dtype=torch.int32)[None]
    cu, kl = (torch.tensor(n, device=cuda, dtype=torch.int32) for n in ([0, nq], [nk]))
    cache_attention(q[:, :heads], cache, cu, table[:, :2], kl, causal=False)
    t = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    t[0].record()
    out = cache_attention(q, cache, cu, table, kl, causal=False)
    t[1].record()
    assert gemm_status() == 0
    assert t[0].elapsed_time(t[1]) * 1e6 > 2 * LIMIT_NS  # longer than the limit and a sleep of 0.2 ms, or nothing is shown
    for h in (0, heads // 2, heads - 1):
        kd, vd = (codes_of(c[:, h], bits).reshape(-1, hd)[:nk].double() * s[0, 0, 0].double()
                  for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        qd = q[:, h].double()
        p = torch.softmax(qd @ kd.T * hd ** -0.5, -1)
        ref, mean = p @ vd, p @ vd.abs()
        d = (qd.abs() @ kd.abs().T).amax(-1, keepdim=True) * (hd ** -0.5 * 2 ** -22)
        tol = 2 ** -8 * (mean + ref.abs()) * (1 + 2 ** -6) + mean * (2 * d + 2 ** -18 + nk * 2.0 ** -28)
        assert bool(((out[:, h].double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("prefix", [0, 1])
def test_a_launch_that_gives_up(short_waits, cuda, prefix):  # noqa: F811
    """A million empty sequences take the kernel longer to look through than the limit lets its other roles wait for the
    first item. The call ends by itself, says so, and the next one is right: one key, or two that are the same."""
    from embodied_efficiency_b200 import KVCache, _lib, cache_attention
    from embodied_efficiency_b200.wq_gemm import gemm_status
    n, heads, hd = 1 << 20, 128, 64
    tokens = 16 * n // heads + 128  # more than 16 rows a sequence: the tensor-core kernel
    q = torch.randn(tokens, 1, hd, device=cuda).bfloat16().expand(tokens, heads, hd)
    cache = KVCache.empty(1, 1, hd, 32)
    cache.k.random_(-127, 128), cache.v.random_(-127, 128)
    cache.k_scale.fill_(2.0 ** -6), cache.v_scale.fill_(2.0 ** -6)
    pre = tuple((c[0, :, :1] * 2.0 ** -6).bfloat16() for c in (cache.k, cache.v)) if prefix else None
    cu, kl = torch.zeros(n + 1, device=cuda, dtype=torch.int32), torch.zeros(n, device=cuda, dtype=torch.int32)
    table = torch.zeros(n, 1, device=cuda, dtype=torch.int32)
    cu[-1], kl[-1] = tokens, 1
    cache_attention(q, cache, cu, table, kl, causal=False, prefix=pre)
    assert gemm_status(reset=True) == _lib.EE_ERR_TIMEOUT
    short_waits.ee_prompt_attention_wait_limit(0)
    out = cache_attention(q, cache, cu, table, kl, causal=False, prefix=pre)
    assert gemm_status() == 0
    assert bool((out == (cache.v[0, :, :1] * 2.0 ** -6).bfloat16()).all())
