"""Forward-mode differentiation: the prompt-layer operators have no derivative of that kind either, and say so."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


def test_tangents_are_refused(cuda):
    from embodied_efficiency_b200 import int8_linear, int8_matmul, prompt_attention, quantize_tokens, rotary_embed
    g = torch.Generator(device=cuda).manual_seed(0)

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device=cuda).bfloat16()

    x, r, b = rnd(9, 64), rnd(9, 24), rnd(24)
    w = torch.randint(-127, 128, (24, 64), generator=g, device=cuda, dtype=torch.int8)
    s = torch.rand(24, generator=g, device=cuda)
    q, k, pos = rnd(9, 4, 64), rnd(9, 2, 64), torch.arange(9, device=cuda)
    cu = torch.tensor([0, 2, 9], device=cuda, dtype=torch.int32)
    xq, sx = quantize_tokens(x)
    rotary_embed(q, k, pos, (32,))
    with torch.no_grad(), fwAD.dual_level():
        def dual(t):
            return fwAD.make_dual(t, torch.ones_like(t))

        for call in (lambda: int8_linear(dual(x), w, s), lambda: int8_linear(x, w, dual(s)),
                     lambda: int8_linear(x, w, s, dual(b)), lambda: int8_linear(x, w, s, residual=dual(r)),
                     lambda: int8_matmul(xq, dual(sx), w, s), lambda: quantize_tokens(dual(x)),
                     lambda: rotary_embed(dual(q), k, pos, (32,)), lambda: rotary_embed(None, dual(k), pos, (32,)),
                     lambda: prompt_attention(dual(q), k, k, cu), lambda: prompt_attention(q, k, dual(k), cu)):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
        assert torch.equal(quantize_tokens(x)[0], xq)  # a level without tangents changes nothing
