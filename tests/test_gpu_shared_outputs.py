"""Outputs whose elements share memory: threads would write them in any order, so they are refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_outputs_that_overlap_themselves(cuda):
    from embodied_efficiency_b200 import prompt_attention, rotary_embed
    t, hd = 40, 64
    q, k = torch.randn(t, 8, hd, device=cuda).bfloat16(), torch.randn(t, 1, hd, device=cuda).bfloat16()
    pos, cu = torch.arange(t, device=cuda), torch.tensor([0, t], device=cuda, dtype=torch.int32)
    wide, row = k.expand(t, 8, hd), k[:1].expand(t, 1, hd)
    window = torch.empty(t * 8 * hd + 8 * hd, device=cuda, dtype=torch.bfloat16).as_strided((t, 8, hd), (4 * hd, hd, 1))
    for out in (wide, window):
        with pytest.raises(ValueError, match="overlap"):
            rotary_embed(q, None, pos, (32,), out=(out, None))
        with pytest.raises(ValueError, match="overlap"):
            prompt_attention(q, k, k, cu, out=out)
    with pytest.raises(ValueError, match="overlap"):  # broadcast keys turned in place
        rotary_embed(q, wide, pos, (32,), out=(q.clone(), wide))
    with pytest.raises(ValueError, match="overlap"):
        rotary_embed(None, k, pos, (32,), out=(None, row))
    assert rotary_embed(q, wide, pos, (32,))[1].is_contiguous()  # as inputs they are fine


def test_other_strided_outputs_are_filled(cuda):
    from embodied_efficiency_b200 import prompt_attention, rotary_embed
    t, hd = 40, 64
    q, k = torch.randn(t, 8, hd, device=cuda).bfloat16(), torch.randn(t, 2, hd, device=cuda).bfloat16()
    pos, cu = torch.arange(t, device=cuda), torch.tensor([0, t], device=cuda, dtype=torch.int32)
    turned, seen = rotary_embed(q, k, pos, (32,))[0], prompt_attention(q, k, k, cu)
    for make in (lambda: torch.empty(8, t, hd, device=cuda, dtype=q.dtype).transpose(0, 1),
                 lambda: torch.empty(t, 16, hd, device=cuda, dtype=q.dtype)[:, ::2],
                 lambda: torch.empty(t, 8, 2 * hd, device=cuda, dtype=q.dtype)[..., hd:]):
        assert torch.equal(rotary_embed(q, None, pos, (32,), out=(make(), None))[0], turned)
        assert torch.equal(prompt_attention(q, k, k, cu, out=make()), seen)
    one = torch.empty(1, 1, hd, device=cuda, dtype=q.dtype).expand(1, 1, hd)  # a stride of a single entry means nothing
    assert torch.equal(rotary_embed(q[:1, :1], None, pos[:1], (32,), out=(one, None))[0], turned[:1, :1])
