"""Many keys whose weights are far below the largest one: together they count, whatever 16-bit type a weight is
rounded to for its product with the values."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nq,heads", [(1, 4), (1, 4736), (40, 8), (40, 296), (300, 2)])
@pytest.mark.parametrize("at", [0, 70000, 131071])
def test_one_key_above_many(cuda, dtype, nq, heads, at):
    """One key scores 17.625 above 131071 others (2^-25.4 of its weight each) and has values of 0, the others have 1:
    the result is the others' share, 0.0029. With few heads the keys are split, and only the part with that key has
    small weights; with many a row's keys stay together. Its tolerance: the result's and the weights' rounding, half a step each;
    fp32 sums of at most nk / 16 steps; for fp16, whose steps end at 2^-24 (half: 2^-25), a weight is held at 2^7
    times its value or more beside a largest one, so nk keys are off by nk * 2^-32 together."""
    from embodied_efficiency_b200 import prompt_attention
    nk, hd, high = 1 << 17, 64, 17.625
    q = torch.zeros(nq, heads, hd, device=cuda, dtype=dtype)
    q[..., 0] = 1
    k, v = torch.zeros(nk, 1, hd, device=cuda, dtype=dtype), torch.ones(nk, 1, hd, device=cuda, dtype=dtype)
    k[at, :, 0], v[at] = high, 0
    k, v = k.expand(nk, heads, hd), v.expand(nk, heads, hd)
    cu_q, cu_k = (torch.tensor([0, n], device=cuda, dtype=torch.int32) for n in (nq, nk))
    out = prompt_attention(q, k, v, cu_q, cu_k, causal=False, scale=1.0)
    rest = (nk - 1) * math.exp(-high)
    ref = rest / (1 + rest)
    tol = torch.finfo(dtype).eps * ref * (1 + 2 ** -6) + ref * nk * 2.0 ** -28
    if dtype == torch.float16:
        tol += nk * 2.0 ** -32
    assert float((out.double() - ref).abs().max()) <= tol
