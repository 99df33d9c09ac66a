"""How far attention over a paged cache is from 64 bits: up to 16 rows a sequence and key head the result's own rounding,
above that the weights' rounding to fp16 beside it."""
import pytest
import torch

from test_gpu_cache_attention import held, make, status

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16]


def exact(q, cache, table, q_len, k_len):
    """Causal results in 64 bits, sum_j p_j |v_j| and the most that a score is off by (fp32 sums, steps and exponents 2^-22
    of sum |q k|, bf16 queries as fp16 2^-25 of the largest times sum |k|), [tokens, heads, ...]."""
    g, i, res = q.shape[1] // cache.kv_heads, 0, []
    for b, (nq, nk) in enumerate(zip(q_len, k_len)):
        kd, vd, _ = held(cache, table, b, nk)
        kd, vd = (x.transpose(0, 1).repeat_interleave(g, 0) for x in (kd, vd))
        qd = q[i:i + nq].double().transpose(0, 1)
        at = torch.arange(nk, device=q.device)[None] - torch.arange(nq, device=q.device)[:, None]
        p = torch.softmax((qd @ kd.transpose(1, 2) * q.shape[2] ** -0.5).masked_fill(at > nk - nq, float("-inf")), -1)
        d = (qd.abs() @ kd.abs().transpose(1, 2) * 2 ** -22).amax(-1, keepdim=True)
        d = (d + qd.abs().amax(-1, keepdim=True) * kd.abs().sum(-1).amax(-1)[:, None, None] * 2 ** -25) * q.shape[2] ** -0.5
        res.append([x.transpose(0, 1) for x in (p @ vd, p @ vd.abs(), d)])
        i += nq
    return [torch.cat(x) for x in zip(*res)]


def rms(x):
    return float(x.pow(2).mean().sqrt())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("hq,nq", [(4, 1), (16, 1), (8, 3), (16, 2)])
def test_few_rows_are_off_by_the_results_rounding(cuda, dtype, bits, hd, hq, nq):
    """The weights enter in two parts, 2^-16 of them is left; 2^-18 for exp2, sums and joins. Rows of one to three keys
    show it: the weights' error is the same in all their dims, with one part of 8 bits 1.4 times the result's."""
    from embodied_efficiency_b200 import cache_attention
    k_len = [nq + i % 3 for i in range(40)] + [nq + 100 * i for i in range(12)]
    q_len = [nq] * len(k_len)
    q, cache, cu, table, kl, _ = make(cuda, dtype, bits, hq, 4, hd, 64, q_len, k_len, 3)
    out = cache_attention(q, cache, cu, table, kl).double()
    ref, mean, d = exact(q, cache, table, q_len, k_len)
    half = torch.finfo(dtype).eps / 2
    tol = half * ref.abs() * (1 + 2 ** -6) + mean * (2.0 ** -16 + 2 * d + 2 ** -18) + 2.0 ** -24
    assert bool(((out - ref).abs() <= tol).all()), float(((out - ref).abs() / tol).max())
    for rows in (slice(0, 40 * nq), slice(40 * nq, None)):
        assert rms((out - ref)[rows]) <= 1.05 * rms((ref.to(dtype).double() - ref)[rows])
    assert status() == 0


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 128])
def test_first_rows_of_a_prompt(cuda, dtype, bits, hd):
    """More than 16 rows: the weights are rounded to fp16 once, by up to half a step of 2^-11 each, which rows of one to
    four keys do not average out, and lose up to 2^-25 beside a largest one of 2^7. Independent of the result's rounding
    and, in fp16, of its size: sqrt(2) of that over many rows; 1.5 leaves 6 % for the spread over 4096 of them. In bf16 the
    result's rounding is eight times that: sqrt(1 + 2^-6)."""
    from embodied_efficiency_b200 import cache_attention
    n, nq = 64, 30
    q, cache, cu, table, kl, _ = make(cuda, dtype, bits, 16, 16, hd, 64, [nq] * n, [nq] * n, 7)
    out = cache_attention(q, cache, cu, table, kl).double()
    ref, mean, d = exact(q, cache, table, [nq] * n, [nq] * n)
    half = torch.finfo(dtype).eps / 2
    tol = (2.0 ** -11 * mean + half * ref.abs()) * (1 + 2 ** -6) + mean * (2 * d + 2 ** -18) + 2.0 ** -24
    tol = tol + nq * 2.0 ** -32 * 127 * float(cache.v_scale[cache.v_scale.isfinite()].max())
    assert bool(((out - ref).abs() <= tol).all()), float(((out - ref).abs() / tol).max())
    first = torch.arange(n * nq, device=cuda) % nq < 4
    most = 1.5 if dtype == torch.float16 else 1.05
    assert rms((out - ref)[first]) <= most * rms((ref.to(dtype).double() - ref)[first])
    assert status() == 0
