"""GPU tests of attention over a paged cache whose steps span the range of fp32: what the caller, or a cache written in
bf16, may hold."""
import random

import pytest
import torch

from test_gpu_cache_attention import held, make, status

pytestmark = pytest.mark.gpu


def check_visible(out, q, cache, table, q_len, k_len, scale, prefix=None):
    """|out - exact| per value of causal fp16 calls, from what a row sees alone. With A = sum_j p_j |v_j|: the weights'
    and the result's rounding 2^-11 of A and of the result each; a score's error of d (fp32 sums, steps and exponents:
    2^-22 of sum |q k| scale) moves a weight twice; 2^-18 A covers exp2, products and sums. Weights below 2^-14 lose up to
    2^-25 each, where the row's largest (weight x excess of its step over 2^8, or 2^12) is 2^7 or more: on values of at
    most 2^15, 2^-25 of that one's weight and step, or 2^-32 of the value where no step exceeds."""
    g = q.shape[1] // cache.kv_heads
    i = 0
    for b, (nq, nk) in enumerate(zip(q_len, k_len)):
        kd, vd, there = held(cache, table, b, nk)
        step = cache.v_scale.transpose(1, 2)[table[b].long()[torch.arange(nk, device=q.device) // cache.page_size],
                                             torch.arange(nk, device=q.device) % cache.page_size].double()
        seen = there[None] & (torch.arange(nk, device=q.device)[None] <= torch.arange(nq, device=q.device)[:, None] + (nk - nq))
        if prefix is not None:
            kd, vd = torch.cat([prefix[0].double(), kd]), torch.cat([prefix[1].double(), vd])
            step = torch.cat([prefix[1].double().abs().amax(-1), step])
            seen = torch.cat([seen.new_ones(nq, len(prefix[0])), seen], 1)
        kd, vd = (x.transpose(0, 1).repeat_interleave(g, 0) for x in (kd, vd))
        step = step.T.repeat_interleave(g, 0)
        qd = q[i:i + nq].double().transpose(0, 1)
        p = torch.softmax((qd @ kd.transpose(1, 2) * scale).masked_fill(~seen, float("-inf")), -1).nan_to_num(0.0)
        ref, mean = p @ vd, p @ vd.abs()
        d = ((qd.abs() @ kd.abs().transpose(1, 2)) * seen).amax(-1, keepdim=True) * (2 ** -22 * scale)
        most = (vd.abs().amax(-1)[:, None] * seen).amax(-1, keepdim=True).clamp(max=2.0 ** 15)
        small = seen.shape[1] * (2.0 ** -25 * (p * step[:, None]).amax(-1, keepdim=True) + 2.0 ** -32 * most)
        tol = 2.0 ** -11 * (mean + ref.abs()) * (1 + 2 ** -6) + mean * (2 * d + 2 ** -18) + small + 2.0 ** -24
        got = out[i:i + nq].double().transpose(0, 1)
        err = (got - ref).abs()
        err[(ref.abs() + tol >= 65520) & got.isinf() & (got * ref > 0)] = 0  # from there on rounding gives infinity
        assert bool((err <= tol).all()), (b, nq, nk, float((err / tol).max()), int(got.isnan().sum()), int(got.isinf().sum()))
        i += nq


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("q_len,k_len,prefix", [([50], [50], 0), ([50, 20, 130], [300, 20, 131], 0), ([40], [3000], 0),
                                                ([50, 20, 60], [50, 131, 90], 100), ([30], [700], 3000), ([1, 1], [90, 300], 0)])
def test_steps_that_fp16_does_not_hold(cuda, bits, hd, q_len, k_len, prefix):
    """Values far above fp16's largest number with weights that bring the result back into its range: steps of 2^9 to
    2^20 on a tenth of the keys, whose scores are so low that they count with a weight of about a value / 2^20 .. 2^3;
    early rows must not see the later ones. Codes of both ends, -128 and -8, among them."""
    from embodied_efficiency_b200 import cache_attention
    q, cache, cu, table, kl, pre = make(cuda, torch.float16, bits, 4, 2, hd, 32, q_len, k_len, bits + hd, prefix)
    r, most, scale = random.Random(hd + len(q_len)), 127 if bits == 8 else 7, hd ** -0.5
    q[..., 0] = 16.0
    if prefix:
        pre[0][..., 0] = 0
    page = cache.page_size
    cache.k[..., 0] = 0 if bits == 8 else cache.k[..., 0] & 0xF0
    for b, n in enumerate(k_len):
        for key in range(n):
            if r.random() < 0.1 or key == n - 1 or key == n // 2:
                e, h = r.randint(9, 20), r.randrange(2)
                at = (int(table[b, key // page]), h, key % page)
                cache.v_scale[at] = 2.0 ** e * r.uniform(1, 2)
                cache.v[at][r.randrange(8)] = -128 if bits == 8 else 0x88
                # a score of -t: 2^e most e^-t is 2^3 to 2^9
                t = (e + (7 if bits == 8 else 3) - r.uniform(3, 9)) * 0.6931
                cache.k[at] = 0
                cache.k[at][0] = -most if bits == 8 else 16 - most
                cache.k_scale[at] = t / (16 * most * scale)
    out = cache_attention(q, cache, cu, table, kl, prefix=pre)
    check_visible(out, q, cache, table, q_len, k_len, scale, pre)
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nq", [3, 20])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_the_largest_steps_under_the_mask(cuda, dtype, bits, hd, nq, which):
    """A step near fp32's largest number on one key reaches no row that does not see it."""
    from embodied_efficiency_b200 import cache_attention
    q, cache, cu, table, kl, _ = make(cuda, dtype, bits, 2, 1, hd, 32, [nq], [50], 4)
    out = cache_attention(q, cache, cu, table, kl)
    getattr(cache, which)[table[0, 1], 0, 48 - 32] = 2.0 ** 127  # key 48: not seen by queries before the last but one
    assert torch.equal(cache_attention(q, cache, cu, table, kl)[:nq - 2], out[:nq - 2]) and bool(out.isfinite().all())
    assert status() == 0


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("q_len", [[50, 50, 20, 30], [1, 1, 1, 1]])
def test_steps_below_those_of_fp16(cuda, bits, hd, q_len):
    """bf16 calls whose values are far below fp16's smallest number, a sequence's all of one size (2^-20, 2^-40 and 2^-70
    of the usual, within 2^5 of one another), and a sequence of zeros as ``cache_write`` holds them. The weights' rounding
    to 2^-11, and those that it takes below 2^-14: 2^-25 each beside a largest one of 2^7 or more, on values whose parts
    that stay with them differ by up to 2^6."""
    from embodied_efficiency_b200 import cache_attention
    k_len = [50, 300, 131, 100]
    q, cache, cu, table, kl, _ = make(cuda, torch.bfloat16, bits, 4, 2, hd, 32, q_len, k_len, 5)
    for b, e in enumerate((-20, -40, -70)):
        rows = table[b][table[b] >= 0].long()
        cache.v_scale[rows] = cache.v_scale[rows].nan_to_num(1.0, 1.0) * 2.0 ** e
    rows = table[3][table[3] >= 0].long()
    cache.v[rows], cache.v_scale[rows] = 0, 1e-8
    out = cache_attention(q, cache, cu, table, kl)
    i = 0
    for b, (nq, nk) in enumerate(zip(q_len, k_len)):
        kd, vd, _ = held(cache, table, b, nk)
        at = torch.arange(nk, device=cuda)
        step = cache.v_scale.transpose(1, 2)[table[b].long()[at // 32], at % 32].double().T.repeat_interleave(2, 0)
        kd, vd = (x.transpose(0, 1).repeat_interleave(2, 0) for x in (kd, vd))
        qd = q[i:i + nq].double().transpose(0, 1)
        seen = at[None] <= torch.arange(nq, device=cuda)[:, None] + (nk - nq)
        p = torch.softmax((qd @ kd.transpose(1, 2) * hd ** -0.5).masked_fill(~seen, float("-inf")), -1)
        ref, mean = p @ vd, p @ vd.abs()
        d = (qd.abs() @ kd.abs().transpose(1, 2) * 2 ** -22).amax(-1, keepdim=True)
        d = (d + qd.abs().amax(-1, keepdim=True) * kd.abs().sum(-1).amax(-1)[:, None, None] * 2 ** -25) * hd ** -0.5
        small = nk * 2.0 ** -19 * (p * step[:, None]).amax(-1, keepdim=True)
        tol = (2.0 ** -11 * mean + 2.0 ** -8 * ref.abs()) * (1 + 2 ** -6) + mean * (2 * d + 2 ** -18) + small
        err = (out[i:i + nq].double().transpose(0, 1) - ref).abs()
        assert bool((err <= tol).all()), (b, float((err / tol).max()))
        assert b == 3 or bool(out[i:i + nq].any())
        i += nq
    assert not bool(out[sum(q_len[:3]):].any()) and status() == 0
