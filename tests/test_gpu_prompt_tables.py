"""Offset tables that break the rule (they decrease, so that two sequences claim the same rows): nothing outside the
tensors is touched, rows that one sequence claims are right, the others hold one of their sequences' results."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _ref(q, k, v, causal):
    """The result in 64 bits, and the bound of its error: half a step for the weights and for the result, 2^-18 for
    exp2, sums and merges, twice a score's 2^-22 of sum |q k|."""
    g = q.shape[1] // k.shape[1]
    qd, kd, vd = (x.double().transpose(0, 1) for x in (q, k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)))
    scale = q.shape[2] ** -0.5
    s = qd @ kd.transpose(1, 2) * scale
    if causal:
        seen = torch.arange(k.shape[0], device=q.device)[None] <= torch.arange(q.shape[0], device=q.device)[:, None] + (
            k.shape[0] - q.shape[0])
        s = s.masked_fill(~seen, float("-inf"))
    p = torch.softmax(s, -1)
    ref, mean = p @ vd, p @ vd.abs()
    d = (qd.abs() @ kd.abs().transpose(1, 2) * scale * 2 ** -22).amax(-1, keepdim=True)
    tol = 2 ** -8 * (mean + ref.abs()) * (1 + 2 ** -6) + mean * (2 * d + 2 ** -18) + 2.0 ** -24
    return ref.transpose(0, 1), tol.transpose(0, 1)


@pytest.mark.parametrize("q_end,keys", [(4, 3000), (4, 40), (300, 700)])
@pytest.mark.parametrize("causal", [True, False])
def test_decreasing_offsets(cuda, q_end, keys, causal):
    from embodied_efficiency_b200 import prompt_attention
    low = q_end // 4
    tq = q_end + low
    g = torch.Generator(device=cuda).manual_seed(q_end + keys)
    q = torch.randn(tq, 4, 64, generator=g, device=cuda).bfloat16()
    k, v = (torch.randn(2 * keys, 2, 64, generator=g, device=cuda).bfloat16() for _ in range(2))
    cu_q = torch.tensor([0, q_end, low, tq], device=cuda, dtype=torch.int32)
    cu_k = torch.tensor([0, keys, keys, 2 * keys], device=cuda, dtype=torch.int32)
    buf = torch.full((tq + 2, 4, 64), 7.0, device=cuda, dtype=torch.bfloat16)
    for _ in range(3):
        out = prompt_attention(q, k, v, cu_q, cu_k, causal=causal, out=buf[1:-1])
        assert bool((buf[0] == 7).all()) and bool((buf[-1] == 7).all())
        a, ta = _ref(q[:q_end], k[:keys], v[:keys], causal)
        b, tb = _ref(q[low:], k[keys:], v[keys:], causal)
        in_a = (out[:q_end].double() - a).abs() <= ta
        in_b = (out[low:].double() - b).abs() <= tb
        assert bool(in_a[:low].all()) and bool(in_b[q_end - low:].all())
        assert bool((in_a[low:].all(-1) | in_b[:q_end - low].all(-1)).all())
