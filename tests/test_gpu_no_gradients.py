"""The prompt-layer operators have no backward pass: whatever asks for a gradient is refused, never dropped."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def linear(cuda):
    g = torch.Generator(device=cuda).manual_seed(0)
    x = torch.randn(5, 64, generator=g, device=cuda).bfloat16()
    w = torch.randint(-127, 128, (24, 64), generator=g, device=cuda, dtype=torch.int8)
    return x, w, torch.rand(24, generator=g, device=cuda), torch.randn(24, generator=g, device=cuda).bfloat16()


def test_parameters_of_a_linear(cuda, linear):
    from embodied_efficiency_b200 import int8_linear, int8_matmul, quantize_tokens
    x, w, s, b = linear
    xq, sx = quantize_tokens(x)
    bias, scales = torch.nn.Parameter(b), torch.nn.Parameter(s)
    for call in (lambda: int8_linear(x, w, s, bias), lambda: int8_linear(x, w, scales, b),
                 lambda: int8_linear(x, w, s, bias, gelu=True), lambda: int8_linear(x, w, s, bias.float()),
                 lambda: int8_matmul(xq, sx, w, s, bias), lambda: int8_matmul(xq, sx, w, scales)):
        with pytest.raises(RuntimeError, match="no backward pass"):
            call()
    want = int8_linear(x, w, s, b)
    with torch.no_grad():
        assert torch.equal(int8_linear(x, w, scales, bias), want)
        assert torch.equal(int8_matmul(xq, sx, w, scales, bias), want)
    assert torch.equal(int8_linear(x, w, s, bias.detach()), want)


def test_module_counts_its_parameters_as_constants(cuda):
    """As the weight-only modules do: a call with gradients enabled gives values without a graph."""
    from embodied_efficiency_b200 import TritonQuantLinear
    lin = TritonQuantLinear(torch.nn.Linear(64, 24).to(cuda).bfloat16(), 8, act_bits=8)
    assert lin.bias.requires_grad
    x = torch.randn(5, 64, device=cuda).bfloat16().requires_grad_()
    y = lin(x)
    assert y.grad_fn is None and not y.requires_grad
    with torch.no_grad():
        assert torch.equal(lin(x), y)
