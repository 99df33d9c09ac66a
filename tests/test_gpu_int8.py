"""GPU parity of the 8-bit integer linears (ee_quantize_tokens, ee_int8_gemm, ee_int8_linear) against their
definition in 64 bits: exact codes and scales, exact integer sums, one rounding of the result."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16]


def _quant_ref(x):
    xf = x.float()
    s = (xf.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device=x.device)).clamp_min(1e-8)
    return torch.round(xf / s).to(torch.int8), s


def _check(y, xq, sx, w, sw, bias, gelu, residual):
    """|y - exact| within the result's half step and the fp32 steps of the epilogue: three products and sums of
    2^-24 relative each on the way to the pre-activation z, and for the GELU 1 + erf(z / sqrt 2) to 3 x 2^-24
    absolute (its slope is below 1.13)."""
    acc = xq.double() @ w.double().T
    prod = acc * sx.double() * sw.double().reshape(1, -1)
    z = prod if bias is None else prod + bias.double()
    ref = z
    if gelu:
        ref = 0.5 * z * torch.special.erfc(-z / 2 ** 0.5)
    if residual is not None:
        ref = z + residual.double()
    f = 2.0 ** -24
    mid = 4 * f * (prod.abs() + z.abs()) * 1.13 + (4 * f * z.abs() if gelu else 0.0)
    if residual is not None:
        mid = mid + f * ref.abs()
    eps = torch.finfo(y.dtype).eps / 2
    tol = eps * (ref.abs() + mid) + mid + torch.finfo(y.dtype).smallest_normal * eps
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def _weight(g, n, k, dev):
    w = torch.randint(-128, 128, (n, k), generator=g, device=dev, dtype=torch.int8)
    return w, (torch.rand(n, generator=g, device=dev) + 0.5) * 3e-4


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,k", [(1, 16), (3, 48), (50, 1024), (7, 2048), (129, 4096), (2, 8192), (5, 16400),
                                    (3, 40000), (1000, 1040)])
def test_quantize_tokens_is_exact(cuda, dtype, rows, k):
    from embodied_efficiency_b200 import quantize_tokens
    g = torch.Generator(device=cuda).manual_seed(rows * 31 + k)
    x = torch.randn(rows, k, generator=g, device=cuda).to(dtype)
    x[:, ::53] *= 8
    if rows > 2:
        x[1] = 0
        x[2] *= 1e-6
    q, s = quantize_tokens(x)
    qr, sr = _quant_ref(x)
    assert torch.equal(s, sr) and torch.equal(q, qr)


@pytest.mark.parametrize("dtype", DT)
def test_quantize_tokens_ties_and_non_finite_rows(cuda, dtype):
    from embodied_efficiency_b200 import int8_linear, quantize_tokens
    # amax 127: the scale is 1 and every half is a tie
    x = (torch.arange(-256, 256, device=cuda).float() / 2).clamp(-127, 127).to(dtype).repeat(6, 1)
    x[1, 5], x[2, 0], x[3, 511] = float("inf"), float("nan"), float("-inf")
    q, s = quantize_tokens(x)
    for r in (0, 4, 5):
        assert torch.equal(q[r], torch.round(x[r].float()).to(torch.int8)) and float(s[r]) == 1.0
    assert not bool(q[1:4].any()) and bool(s[1:4].isnan().all())
    w, sw = _weight(torch.Generator(device=cuda).manual_seed(1), 40, 512, cuda)
    y = int8_linear(x, w, sw)
    assert bool(y[1:4].isnan().all()) and bool(y[[0, 4, 5]].isfinite().all())


SHAPES = [(1, 64, 128), (1, 8192, 2048), (2, 7, 16), (8, 130, 2064), (17, 1000, 1040), (31, 33, 48), (50, 2048, 8192),
          (64, 1024, 1024), (65, 129, 144), (100, 257, 512), (129, 4096, 1024), (300, 1000, 1040), (513, 264, 2048),
          (1023, 1000, 1040), (2000, 1024, 4096), (5000, 520, 272)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_matches_the_definition(cuda, dtype, m, n, k):
    from embodied_efficiency_b200 import int8_linear
    g = torch.Generator(device=cuda).manual_seed(m * 7 + n * 3 + k)
    x = torch.randn(m, k, generator=g, device=cuda).to(dtype)
    w, sw = _weight(g, n, k, cuda)
    bias = torch.randn(n, generator=g, device=cuda).to(dtype)
    res = torch.randn(m, n, generator=g, device=cuda).to(dtype)
    xq, sx = _quant_ref(x)
    for b, gelu, r in ((None, False, None), (bias, True, None), (bias, False, res)):
        y = int8_linear(x, w, sw, b, gelu=gelu, residual=r)
        assert y.dtype == dtype and y.shape == (m, n)
        _check(y, xq, sx, w, sw, b, gelu, r)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,n,k", [(1, 72, 16), (37, 1000, 1040), (300, 264, 4096), (1500, 1030, 528)])
def test_matmul_extreme_codes_and_half_scales(cuda, dtype, m, n, k):
    """Sums that leave 24 bits: codes of -128 and 127 only; fp16 channel scales."""
    from embodied_efficiency_b200 import int8_matmul
    g = torch.Generator(device=cuda).manual_seed(m + n + k)
    xq = torch.where(torch.rand(m, k, generator=g, device=cuda) < 0.9, -128, 127).to(torch.int8)
    w = torch.where(torch.rand(n, k, generator=g, device=cuda) < 0.9, -128, 127).to(torch.int8)
    sx = (torch.rand(m, 1, generator=g, device=cuda) + 0.5) * 1e-3
    sw = ((torch.rand(n, generator=g, device=cuda) + 0.5) * 1e-3).half()
    _check(int8_matmul(xq, sx, w, sw, dtype=dtype), xq, sx, w, sw.float(), None, False, None)


@pytest.mark.parametrize("m", [3, 200, 3000])
def test_views_batches_and_repeats(cuda, m):
    """Strided rows, leading dimensions, an odd base address, empty calls; the same call gives the same bits."""
    from embodied_efficiency_b200 import int8_linear, int8_matmul, quantize_tokens
    g = torch.Generator(device=cuda).manual_seed(m)
    big = torch.randn(m, 3 * 512 + 8, generator=g, device=cuda).bfloat16()
    w, sw = _weight(g, 96, 512, cuda)
    for x in (big[:, 512:1024], big[:, 3:515], big[:, 512:1024].unsqueeze(1), big[:, :1024].reshape(m, 2, 512)):
        y = int8_linear(x, w, sw)
        assert y.shape == (*x.shape[:-1], 96)
        assert torch.equal(y, int8_linear(x.contiguous(), w, sw)) and torch.equal(y, int8_linear(x, w, sw))
        xq, sx = quantize_tokens(x)
        assert torch.equal(y, int8_matmul(xq, sx, w, sw))
    flat = torch.empty(96 * 512 + 1, dtype=torch.int8, device=cuda)
    odd = flat[1:].view(96, 512).copy_(w)
    assert torch.equal(int8_linear(big[:, 512:1024], odd, sw), int8_linear(big[:, 512:1024], w, sw))
    assert int8_linear(big[:0, :512], w, sw).shape == (0, 96)
    assert int8_linear(big[:, :512], w[:0], sw[:0]).shape == (m, 0)
    assert int8_matmul(torch.empty(0, 512, dtype=torch.int8, device=cuda), torch.empty(0, 1, device=cuda), w,
                       sw).shape == (0, 96)


def test_captured_and_on_another_stream(cuda):
    from embodied_efficiency_b200 import int8_linear
    from embodied_efficiency_b200.wq_gemm import gemm_status
    g = torch.Generator(device=cuda).manual_seed(5)
    x = torch.randn(600, 1024, generator=g, device=cuda).bfloat16()
    w, sw = _weight(g, 512, 1024, cuda)
    first, few = int8_linear(x, w, sw), int8_linear(x[:5], w, sw)
    graphs = []
    for _ in range(2):  # two graphs of the same call, replayed in turn
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = int8_linear(x, w, sw), int8_linear(x[:5], w, sw)
        graphs.append((gr, out))
    for gr, out in graphs + graphs:
        gr.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert torch.equal(out[0], first) and torch.equal(out[1], few)
    x2 = x.flip(0).contiguous()
    want = int8_linear(x2, w, sw)
    x.copy_(x2)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1][0], want)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    torch.cuda.synchronize()
    for i in range(6):
        with torch.cuda.stream(side[i % 2]):
            outs.append(int8_linear(x, w, sw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    assert gemm_status() == 0
