"""The native host side of the prompt-layer operators (lib/ee_torch.so): the usual calls give what the Python path
gives, every other call is left to it."""
import pytest
import torch


class _Off:
    """A native module that takes no call."""

    def __getattr__(self, name):
        return lambda *a: None


def test_unusual_calls_are_left_to_python():
    from embodied_efficiency_b200 import _lib, build
    build.build()
    n = _lib.native()
    x, w, s = torch.zeros(3, 64).bfloat16(), torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)
    for call in (lambda: n.int8_linear(x, w, s, None, False, None), lambda: n.int8_linear(x),
                 lambda: n.int8_linear(1, 2, 3, 4, 5, 6), lambda: n.quantize_tokens(x), lambda: n.quantize_tokens(None),
                 lambda: n.int8_matmul(w, s, w, s, None, False, None, 3),
                 lambda: n.rotary_embed(x, x, x, (32,), x, False), lambda: n.rotary_embed(x, x, x, [32], x, 0),
                 lambda: n.prompt_attention(x, x, x, s, None, None, True, None), lambda: n.prompt_attention()):
        assert call() is None


@pytest.mark.gpu
def test_native_and_python_agree(cuda, monkeypatch):
    from embodied_efficiency_b200 import _lib, int8_linear, int8_matmul, prompt_attention, quantize_tokens, rotary_embed
    g = torch.Generator(device=cuda).manual_seed(0)

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device=cuda).bfloat16()

    x, r, b = rnd(5, 7, 256), rnd(5, 7, 96), rnd(96)
    w = torch.randint(-127, 128, (96, 256), generator=g, device=cuda, dtype=torch.int8)
    s = torch.rand(96, 1, generator=g, device=cuda)
    xq, sx = quantize_tokens(x)
    qkv = rnd(9, 6 * 64)
    q, k, v = qkv[:, :256].view(9, 4, 64), qkv[:, 256:320].view(9, 1, 64), qkv[:, 320:].view(9, 1, 64)
    pos = torch.arange(27, device=cuda).view(3, 9)
    cu = torch.tensor([0, 2, 9], device=cuda, dtype=torch.int32)
    rotary_embed(q, k, pos, (8, 12, 12))  # the table of frequencies is there from here on
    calls = {
        "int8_linear": lambda: (int8_linear(x, w, s, b, gelu=True), int8_linear(x, w, s.half(), None, residual=r)),
        "int8_matmul": lambda: (int8_matmul(xq, sx, w, s, b), int8_matmul(xq, sx, w, s, dtype=torch.float16)),
        "quantize_tokens": lambda: quantize_tokens(x),
        "rotary_embed": lambda: rotary_embed(q, k, pos, (8, 12, 12)) + rotary_embed(q, k, pos[0].int(), (32,), interleaved=True),
        "prompt_attention": lambda: (prompt_attention(q, k, v, cu), prompt_attention(q, k, v, cu, cu, cu[1:] - cu[:-1], False),
                                     prompt_attention(q, k, v, cu, scale=0.5)),
    }
    native = _lib.native()
    for name, call in calls.items():
        seen = []

        class Spy(_Off):
            def __getattr__(self, n):
                def f(*a):
                    y = getattr(native, n)(*a)
                    seen.append((n, y is not None))
                    return y
                return f

        monkeypatch.setattr(_lib, "_native", Spy())
        got = call()
        assert seen and all(n == name and took for n, took in seen), (name, seen)
        monkeypatch.setattr(_lib, "_native", _Off())
        want = call()
        for u, t in zip(got, want):
            assert u.shape == t.shape and u.dtype == t.dtype and u.stride() == t.stride() and torch.equal(u, t), name
    monkeypatch.setattr(_lib, "_native", native)
    # what asks for a gradient, or for a copy, is not taken
    xg = x.clone().requires_grad_()
    for call in (lambda: int8_linear(xg, w, s), lambda: quantize_tokens(xg),
                 lambda: prompt_attention(q.clone().requires_grad_(), k, v, cu),
                 lambda: rotary_embed(q.clone().requires_grad_(), k, pos, (8, 12, 12))):
        with pytest.raises(RuntimeError, match="no backward pass"):
            call()
    with torch.no_grad():
        assert torch.equal(int8_linear(xg, w, s), int8_linear(x, w, s))
    assert torch.equal(int8_linear(x.transpose(0, 1), w, s), int8_linear(x.transpose(0, 1).contiguous(), w, s))
