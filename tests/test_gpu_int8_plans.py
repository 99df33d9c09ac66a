"""Every way the 8-bit product is launched -- tokens per tile, slices of K, output rows on and off 16-byte boundaries --
with every epilogue, as part of int8_linear (whose product loads its weights early) and by itself; and the launches of
both kernels in one graph and on two streams at a time."""
import ctypes

import pytest
import torch
from test_gpu_int8 import _check, _quant_ref, _weight

pytestmark = pytest.mark.gpu

SIZES = [(1, 8, 16), (1, 9, 16), (622, 8, 672), (1, 4758, 688), (1, 8, 400), (16, 1023, 400), (1, 8, 912),
         (1, 1025, 1040), (2775, 8, 816), (2416, 9, 816), (1226, 8, 2640), (1229, 9, 2480), (649, 8, 3584),
         (614, 10, 3360), (318, 8, 7248), (291, 9, 6864), (4931, 8, 848), (4776, 9, 784), (2637, 8, 2560),
         (2738, 9, 2544), (1286, 8, 3568), (1268, 9, 3840), (596, 8, 7296), (618, 10, 6864), (5114, 8, 2768),
         (5074, 9, 2784), (2943, 8, 4000), (2472, 10, 3920), (1465, 8, 7792), (1546, 9, 7840), (400, 2048, 8192),
         (126, 5587, 3488), (1500, 1030, 528), (1111, 2049, 1040), (2000, 1176, 256)]
EPILOGUES = [(False, False, False), (True, True, False), (True, False, True), (False, True, False), (False, False, True)]


def _plan(m, n, k):
    from embodied_efficiency_b200 import _lib
    t, c, s = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_size_t()
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert _lib.load().ee_int8_plan(m, n, k, sms, t, c, s) == 0
    return t.value, c.value


def test_the_sizes_reach_every_launch(cuda):
    have = {(_plan(m, n, k), n % 8 == 0) for m, n, k in SIZES}
    tiles = [(16, s) for s in (1, 2, 4, 8)] + [(t, s) for t in (32, 64) for s in (1, 2, 4, 8)]
    want = {(p, vec) for p in tiles + [(128, 2), (128, 4), (128, 8), (256, 2)] for vec in (True, False)}
    assert have >= want, want - have


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_every_launch_matches_the_definition(cuda, dtype, m, n, k):
    from embodied_efficiency_b200 import int8_linear, int8_matmul
    g = torch.Generator(device=cuda).manual_seed(m + n + k)
    x = torch.randn(m, k, generator=g, device=cuda).to(dtype)
    w, sw = _weight(g, n, k, cuda)
    bias = torch.randn(n, generator=g, device=cuda).to(dtype)
    res = torch.randn(m, n, generator=g, device=cuda).to(dtype)
    xq, sx = _quant_ref(x)
    for has_bias, gelu, has_res in EPILOGUES:
        b, r = bias if has_bias else None, res if has_res else None
        y = int8_linear(x, w, sw, b, gelu=gelu, residual=r)
        _check(y, xq, sx, w, sw, b, gelu, r)
        assert torch.equal(y, int8_matmul(xq, sx, w, sw, b, dtype=dtype, gelu=gelu, residual=r))


def test_pairs_and_clusters_captured_and_on_two_streams(cuda):
    """Pairs of 256 x 256 tiles and clusters of eight slices of K: one after the other in a graph, and beside each
    other on two streams, where their tensor memory has to suffice for both."""
    from embodied_efficiency_b200 import int8_linear
    from embodied_efficiency_b200.wq_gemm import gemm_status
    g = torch.Generator(device=cuda).manual_seed(2)
    w, sw = _weight(g, 1024, 1024, cuda)
    xs = [torch.randn(m, 1024, generator=g, device=cuda).bfloat16() for m in (5000, 16)]
    assert [_plan(x.shape[0], 1024, 1024) for x in xs] == [(256, 2), (16, 8)]
    odd, sodd = _weight(g, 1027, 1024, cuda)
    want = [int8_linear(x, w, sw) for x in xs] + [int8_linear(x, odd, sodd) for x in xs]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = [int8_linear(x, w, sw) for x in xs] + [int8_linear(x, odd, sodd) for x in xs]
    for _ in range(3):
        for t in got:
            t.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for i in range(40):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs.append((j, int8_linear(xs[j], w, sw)))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[j]) for j, y in outs) and gemm_status() == 0
