"""The scales that prompt_attention takes: those whose product with log2(e), by which the kernels multiply, is an fp32
value above 0."""
import pytest
import torch


def test_scales_out_of_range():
    from embodied_efficiency_b200 import _lib, build, prompt_attention
    build.build()
    lib = _lib.load()
    q, cu = torch.zeros(5, 4, 64, dtype=torch.bfloat16), torch.tensor([0, 5], dtype=torch.int32)
    for scale in (2.5e38, 1e39, 1e-46, -1.0, float("nan")):
        with pytest.raises(ValueError, match="scale must be"):
            prompt_attention(q, q, q, cu, scale=scale)
    args = [16, 256, 64, 16, 256, 64, 16, 256, 64, 16, 256, 64, 16, 0, 0, 5, 5, 1, 4, 4, 64, 1]
    for scale in (2.5e38, 3e38, float("inf"), 0.0, -1.0, float("nan")):
        assert lib.ee_prompt_attention(*args, scale, _lib.EE_BF16, 0, 0, None) == 1
    for scale in (2.3e38, 1e-30):  # the next check: no GPU of this kind, or a workspace that is missing
        assert lib.ee_prompt_attention(*args, scale, _lib.EE_BF16, 0, 0, None) in (5, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [3, 200])
def test_largest_and_smallest_scales(cuda, t):
    """Queries of zeros: every key counts the same at any scale. The mean of v in 64 bits; half a step for weights and
    result, 2^-18 for the sums."""
    from embodied_efficiency_b200 import prompt_attention
    q, v = torch.zeros(t, 4, 64, device=cuda).bfloat16(), torch.randn(t, 4, 64, device=cuda).bfloat16()
    cu = torch.tensor([0, t], device=cuda, dtype=torch.int32)
    ref, mean = v.double().mean(0), v.double().abs().mean(0)
    for scale in (2.3e38, 2.0 ** -126):
        out = prompt_attention(q, v, v, cu, causal=False, scale=scale)
        assert bool(((out.double() - ref).abs() <= 2 ** -8 * (1 + 2 ** -6) * (mean + ref.abs()) + 2 ** -18 * mean).all())
