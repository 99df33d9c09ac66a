"""GPU parity of the norms of query and key heads with the rotation in the same pass (ee_norm_rotary)."""
import pytest
import torch

from test_gpu_rotary import _ref

pytestmark = pytest.mark.gpu


def _check(y, x, w, eps, pos, sections, interleaved, base=10000.0):
    """Half a step of the result; the angle as in the rotation's own test (2^-20 of the normalised pair's |a| + |b|);
    the norm's factor: the fp32 sum of hd squares (hd 2^-24 relative, halved by the root), the root and its rounding,
    the products with it and the weight: together below (hd / 2 + 8) 2^-24."""
    hd = x.shape[-1]
    xd = x.double()
    n = w.double() * xd / torch.sqrt(xd.pow(2).mean(-1, keepdim=True) + eps)
    ref, mag = _ref(n, pos, sections, base, interleaved)
    half = torch.finfo(y.dtype).eps / 2
    tol = half * ref.abs() * (1 + 2 ** -10) + mag * (2 ** -20 + (hd / 2 + 8) * 2 ** -24) \
        + torch.finfo(y.dtype).smallest_normal * half
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wtype", ["own", "fp32"])
@pytest.mark.parametrize("t,hq,hk,hd,sections", [(1, 16, 4, 128, (16, 24, 24)), (64, 16, 4, 128, (16, 24, 24)),
                                                 (5, 1, 1, 32, (16,)), (77, 16, 16, 64, (10, 11, 11)),
                                                 (33, 7, 3, 64, (1, 31)), (9, 5, 2, 256, (32, 32, 32, 32)),
                                                 (30, 40, 8, 128, (64,)), (2, 3, 25, 64, (0, 32, 0))])
@pytest.mark.parametrize("interleaved", [False, True])
def test_matches_norm_and_rotation(cuda, dtype, wtype, t, hq, hk, hd, sections, interleaved):
    from embodied_efficiency_b200 import norm_rotary_embed
    g = torch.Generator(device=cuda).manual_seed(t + hq)
    q = (torch.randn(t, hq, hd, generator=g, device=cuda) * 3).to(dtype)
    k = (torch.randn(t, hk, hd, generator=g, device=cuda) * 0.01).to(dtype)
    qw, kw = [(1 + 0.3 * torch.randn(hd, generator=g, device=cuda)).to(torch.float32 if wtype == "fp32" else dtype)
              for _ in range(2)]
    pos = torch.randint(0, 5000, (len(sections), t), generator=g, device=cuda, dtype=torch.int32)
    q2, k2 = norm_rotary_embed(q, k, qw, kw, pos, sections, eps=1e-5, interleaved=interleaved)
    _check(q2, q, qw, 1e-5, pos, sections, interleaved)
    _check(k2, k, kw, 1e-5, pos, sections, interleaved)
    q3, none = norm_rotary_embed(q, None, qw, None, pos, sections, eps=1e-5, interleaved=interleaved)
    assert none is None and torch.equal(q3, q2)
    none, k3 = norm_rotary_embed(None, k, None, kw, pos, sections, eps=1e-5, interleaved=interleaved)
    assert none is None and torch.equal(k3, k2)


def test_extreme_heads(cuda):
    """A head of zeros is zero, a tiny one is carried by eps, a large one is normalised, infinities and NaN stay in
    their own head."""
    from embodied_efficiency_b200 import norm_rotary_embed
    hd = 128
    x = torch.randn(7, 3, hd, device=cuda).bfloat16()
    x[0, 0] = 0
    x[1, 1] *= 1e-12
    x[2, 2] *= 1e15
    x[3, 0, 5] = float("inf")
    x[4, 1, 127] = float("nan")
    x[5, 2, 0] = -float("inf")
    w, pos = torch.ones(hd, device=cuda), torch.arange(7, device=cuda)
    y, _ = norm_rotary_embed(x, None, w, None, pos, (64,))
    bad = [(3, 0), (4, 1), (5, 2)]
    fine = torch.ones(7, 3, dtype=torch.bool)
    for i, h in bad:
        fine[i, h] = False
        assert not bool(y[i, h].isfinite().all())
    assert bool(y[fine.to(cuda)].isfinite().all()) and not bool(y[0, 0].any())
    clean = x.clone()
    for i, h in bad:
        clean[i, h] = 1
    _check(torch.where(fine.to(cuda)[..., None], y, norm_rotary_embed(clean, None, w, None, pos, (64,))[0]), clean, w,
           1e-6, pos[None], (64,), False)


def test_views_in_place_streams_and_capture(cuda):
    from embodied_efficiency_b200 import norm_rotary_embed
    t, hq, hk, hd = 50, 8, 2, 64
    qkv = torch.randn(t, (hq + 2 * hk) * hd, device=cuda).bfloat16()
    keep = qkv.clone()
    q, k = qkv[:, :hq * hd].view(t, hq, hd), qkv[:, hq * hd:(hq + hk) * hd].view(t, hk, hd)
    qw, kw = torch.rand(hd, device=cuda).bfloat16(), torch.rand(hd, device=cuda).bfloat16()
    pos = torch.arange(t, device=cuda, dtype=torch.int32)
    q2, k2 = norm_rotary_embed(q, k, qw, kw, pos, (32,))
    assert torch.equal(qkv, keep)
    _check(q2, q, qw, 1e-6, pos[None], (32,), False)
    # weights off the 16-byte boundary and strided ones: copied
    off = torch.stack([qw, qw], -1)
    assert torch.equal(norm_rotary_embed(q, k, off[:, 1], torch.cat([kw[:1], kw])[1:], pos, (32,))[0], q2)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        again = norm_rotary_embed(q, k, qw, kw, pos, (32,))
    torch.cuda.synchronize()
    assert torch.equal(again[0], q2) and torch.equal(again[1], k2)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = norm_rotary_embed(q, k, qw, kw, pos, (32,))
        with pytest.raises(RuntimeError, match="norm_rotary_embed copies its frequencies"):
            norm_rotary_embed(q, k, qw, kw, pos, (32,), base=78.0)
    qkv.mul_(2)
    gr.replay()
    torch.cuda.synchronize()
    _check(got[0], q, qw, 1e-6, pos[None], (32,), False)
    want = norm_rotary_embed(q, k, qw, kw, pos, (32,))
    assert norm_rotary_embed(q, k, qw, kw, pos, (32,), out=(q, k))[0] is q
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(qkv[:, (hq + hk) * hd:], keep[:, (hq + hk) * hd:] * 2)  # the values beside them
    assert norm_rotary_embed(q[:0], k[:0], qw, kw, pos[:0], (32,))[0].shape == (0, hq, hd)


def test_matches_the_plain_rotation(cuda):
    """Where the norm does nothing but divide by a power of two, the rotation's own kernel gives the same bits."""
    from embodied_efficiency_b200 import norm_rotary_embed, rotary_embed
    x = torch.where(torch.rand(40, 6, 128, device=cuda) < 0.5, -2.0, 2.0).half()  # mean square 4
    pos, w = torch.arange(40, device=cuda), torch.ones(128, device=cuda)
    for inter in (False, True):
        a = norm_rotary_embed(x, x, w, w, pos, (64,), eps=2.0 ** -126, interleaved=inter)
        b = rotary_embed(x / 2, x / 2, pos, (64,), interleaved=inter)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
