"""GPU parity of the multi-axis rotary positions (ee_rotary) against the rotation in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _ref(x, pos, sections, base, interleaved):
    """The rotation in 64 bits, and |a| + |b| of every pair."""
    half = x.shape[-1] // 2
    axis = sum(([i] * s for i, s in enumerate(sections)), [])
    freq = base ** (-torch.arange(half, dtype=torch.float64, device=x.device) / half)
    # the angle modulo a turn in exact integers would be the same: double keeps |pos| < 2^31 to 2^-22 turns
    ang = (pos[axis].T.double() * freq)[:, None]
    xd = x.double()
    a, b = (xd[..., 0::2], xd[..., 1::2]) if interleaved else (xd[..., :half], xd[..., half:])
    c, d, mag = a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos(), a.abs() + b.abs()
    if interleaved:
        return torch.stack([c, d], -1).flatten(-2), torch.stack([mag, mag], -1).flatten(-2)
    return torch.cat([c, d], -1), torch.cat([mag, mag], -1)


def _check(y, x, pos, sections, base, interleaved):
    """Half a step of the result, and for the angle: its 32-bit fraction of a turn and its fp32 value (2^-24 of at
    most pi), the two ulps of the sine and the reference's own double angle, together below 2^-20."""
    ref, mag = _ref(x, pos, sections, base, interleaved)
    eps = torch.finfo(y.dtype).eps / 2
    tol = eps * ref.abs() * (1 + 2 ** -10) + mag * 2 ** -20 + torch.finfo(y.dtype).smallest_normal * eps
    assert bool(((y.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,hq,hk,hd,sections", [(1, 16, 4, 128, (16, 24, 24)), (64, 16, 4, 128, (16, 24, 24)),
                                                 (5, 1, 1, 32, (16,)), (777, 16, 16, 64, (10, 11, 11)),
                                                 (33, 7, 3, 64, (1, 31)), (9, 5, 2, 256, (32, 32, 32, 32)),
                                                 (300, 40, 8, 128, (64,)), (2, 3, 1, 64, (0, 32, 0))])
@pytest.mark.parametrize("interleaved", [False, True])
def test_matches_the_rotation(cuda, dtype, t, hq, hk, hd, sections, interleaved):
    from embodied_efficiency_b200 import rotary_embed
    g = torch.Generator(device=cuda).manual_seed(t + hq)
    q = torch.randn(t, hq, hd, generator=g, device=cuda).to(dtype)
    k = torch.randn(t, hk, hd, generator=g, device=cuda).to(dtype)
    pos = torch.randint(0, 5000, (len(sections), t), generator=g, device=cuda, dtype=torch.int32)
    q2, k2 = rotary_embed(q, k, pos, sections, interleaved=interleaved)
    _check(q2, q, pos, sections, 10000.0, interleaved)
    _check(k2, k, pos, sections, 10000.0, interleaved)


def test_far_negative_and_64_bit_positions(cuda):
    from embodied_efficiency_b200 import rotary_embed
    q = torch.randn(6, 2, 64, device=cuda).half()
    pos = torch.tensor([[0, -1, 1 << 20, (1 << 31) - 1, -(1 << 31), 12345678]], device=cuda, dtype=torch.int64)
    # at 2^31 the reference's double angle is 2^-22 turns off at worst: 2^-19 of |a| + |b|; counted at 2^-20 + it
    for p in (pos, pos.to(torch.int32)):
        q2, none = rotary_embed(q, None, p, (32,), base=500000.0)
        assert none is None
        _check(q2[[0, 1, 2, 5]], q[[0, 1, 2, 5]], pos[:, [0, 1, 2, 5]], (32,), 500000.0, False)
        ref, mag = _ref(q, pos, (32,), 500000.0, False)
        assert bool(((q2.double() - ref).abs() <= 2 ** -11 * ref.abs() * 1.001 + mag * 2 ** -18 + 2 ** -25).all())
    # whole turns of exact integer steps: pos and pos + 2^40 turn pair 0 differently, position 0 not at all
    assert torch.equal(rotary_embed(q, None, torch.zeros_like(pos), (32,))[0], q)


def test_views_in_place_and_empty(cuda):
    from embodied_efficiency_b200 import rotary_embed
    t, hq, hk, hd = 50, 8, 2, 64
    qkv = torch.randn(t, (hq + 2 * hk) * hd, device=cuda).bfloat16()
    keep = qkv.clone()
    q, k = qkv[:, :hq * hd].view(t, hq, hd), qkv[:, hq * hd:(hq + hk) * hd].view(t, hk, hd)
    pos = torch.arange(t, device=cuda, dtype=torch.int32)
    q2, k2 = rotary_embed(q, k, pos, (32,))
    assert torch.equal(qkv, keep)
    _check(q2, q, pos[None], (32,), 10000.0, False)
    got = rotary_embed(q, k, pos, (32,), out=(q, k))
    assert got[0] is q and torch.equal(q, q2) and torch.equal(k, k2)
    assert torch.equal(qkv[:, (hq + hk) * hd:], keep[:, (hq + hk) * hd:])  # the values beside them
    heads_first = torch.randn(hq, t, hd, device=cuda).bfloat16().transpose(0, 1)
    _check(rotary_embed(heads_first, None, pos, (32,))[0], heads_first, pos[None], (32,), 10000.0, False)
    odd = torch.randn(t, hq, hd + 1, device=cuda).bfloat16()[..., 1:]  # off the 16-byte boundary: copied
    _check(rotary_embed(None, odd, pos.long(), (32,))[1], odd, pos[None], (32,), 10000.0, False)
    assert rotary_embed(q[:0], k[:0], pos[:0], (32,))[0].shape == (0, hq, hd)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        again = rotary_embed(keep[:, :hq * hd].view(t, hq, hd), None, pos, (32,))[0]
    torch.cuda.synchronize()
    assert torch.equal(again, q2)


def test_captured(cuda):
    """The table of frequencies has to be there before a capture; replays follow the buffers."""
    from embodied_efficiency_b200 import rotary_embed
    q, pos = torch.randn(3, 2, 64, device=cuda).half(), torch.arange(3, device=cuda, dtype=torch.int32)
    want = rotary_embed(q, q, pos, (32,))[0]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = rotary_embed(q, q, pos, (32,))
        with pytest.raises(RuntimeError, match="before the stream capture"):
            rotary_embed(q, q, pos, (32,), base=77.0)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want) and torch.equal(got[1], want)
    pos.add_(5)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], rotary_embed(q, q, pos, (32,))[0]) and not torch.equal(got[0], want)
