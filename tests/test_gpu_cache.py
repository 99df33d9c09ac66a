"""GPU tests of the paged cache of quantised keys and values: written codes and steps exactly, read back to a rounding."""
import copy
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16]


def quantized(x, bits):
    """Codes and steps by their definition: fp32 steps, true division, ties to even."""
    f = x.float()
    amax = f.abs().amax(-1, keepdim=True)
    s = (amax / torch.full_like(amax, 2 ** (bits - 1) - 1)).clamp_min(1e-8)
    bad = ~amax.isfinite()
    c = torch.where(bad, torch.zeros_like(f), torch.round(f / s))
    return c.to(torch.int8), torch.where(bad, torch.full_like(s, float("nan")), s)[..., 0]


def codes_of(t, bits):
    if bits == 8:
        return t
    lo, hi = (t & 15).to(torch.int8), (t >> 4).to(torch.int8)
    c = torch.stack([lo, hi], -1).flatten(-2)
    return torch.where(c > 7, c - 16, c)


def fill(cache, seed):
    """Every page filled with codes and steps of its own."""
    g = torch.Generator(device=cache.device).manual_seed(seed)
    for t in (cache.k, cache.v):
        lo, hi = (-127, 128) if cache.bits == 8 else (0, 256)
        t.copy_(torch.randint(lo, hi, t.shape, generator=g, device=cache.device).to(t.dtype))
    for t in (cache.k_scale, cache.v_scale):
        t.copy_(torch.rand(t.shape, generator=g, device=cache.device) * 0.02 + 1e-3)
    return cache


def tables(k_len, page, dev, seed, extra=2, width=None):
    """A table over shuffled pages (unused places -1) and the number of pages."""
    need = [-(-max(n, 0) // page) for n in k_len]
    pages = list(range(sum(need) + extra))
    random.Random(seed).shuffle(pages)
    width = max(need + [1]) if width is None else width
    rows, at = [], 0
    for n in need:
        rows.append(pages[at:at + n] + [-1] * (width - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device=dev).view(len(k_len), width), len(pages)


def places(q_len, k_len, table, page):
    """(row, page, place) of every packed row that has one."""
    tab, out, row = table.tolist(), [], 0
    for b, (n, total) in enumerate(zip(q_len, k_len)):
        for i in range(n):
            key = total - n + i
            if key >= 0 and key // page < len(tab[b]) and tab[b][key // page] >= 0:
                out.append((row, tab[b][key // page], key % page))
            row += 1
    return torch.tensor(out, device=table.device).view(-1, 3)


def offsets(lens, dev):
    return torch.tensor([0] + list(lens), device=dev).cumsum(0).to(torch.int32)


CASES = [([1], [1], 64), ([1] * 70, list(range(1, 71)), 32), ([5, 0, 33, 64, 1], [5, 40, 33, 100, 129], 64),
         ([257, 300], [257, 1000], 128), ([0, 0, 7, 0], [0, 3, 7, 0], 256), ([40, 3], [10, 2], 32)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("kv,hd", [(1, 64), (3, 128), (16, 64), (5, 64), (8, 128)])
@pytest.mark.parametrize("q_len,k_len,page", CASES, ids=lambda v: str(v)[:12])
def test_written_and_read(cuda, dtype, bits, kv, hd, q_len, k_len, page):
    """The last case has fewer keys than tokens: rows whose key would lie before 0 go nowhere."""
    from embodied_efficiency_b200 import KVCache, cache_read, cache_write
    g = torch.Generator(device=cuda).manual_seed(kv)
    t = sum(q_len)
    table, pages = tables(k_len, page, cuda, 1)
    cache = fill(KVCache.empty(pages, kv, hd, page, bits), 2)
    before = copy.deepcopy(cache)
    assert before.k.data_ptr() != cache.k.data_ptr() and torch.equal(before.k, cache.k)
    wide = torch.randn(t, 2 * kv, hd, generator=g, device=cuda).to(dtype)
    wide[:, ::2] *= torch.rand(t, kv, 1, generator=g, device=cuda).to(dtype)
    k, v = wide[:, :kv], wide[:, kv:]  # views of one projection
    cu, lens = offsets(q_len, cuda), torch.tensor(k_len, dtype=torch.int32, device=cuda)
    assert cache_write(cache, k, v, cu, table, lens) is None
    at = places(q_len, k_len, table, page)
    for x, codes, steps, codes0, steps0 in ((k, cache.k, cache.k_scale, before.k, before.k_scale),
                                            (v, cache.v, cache.v_scale, before.v, before.v_scale)):
        c, s = quantized(x, bits)
        want_c, want_s = codes_of(codes0, bits).clone(), steps0.clone()
        want_c[at[:, 1], :, at[:, 2]] = c[at[:, 0]]
        want_s[at[:, 1], :, at[:, 2]] = s[at[:, 0]]
        assert torch.equal(codes_of(codes, bits), want_c) and torch.equal(steps, want_s)
    keep = torch.full((t, kv, hd), 7.0, dtype=dtype, device=cuda)
    outs = [keep.clone(), keep.clone()]
    got = cache_read(cache, cu, table, lens, t, dtype, out=outs)
    assert got[0] is outs[0] and got[1] is outs[1]
    new = cache_read(cache, cu, table, lens, t, dtype)
    for x, y, z in zip((k, v), got, new):
        c, s = quantized(x, bits)
        want = keep.clone()
        want[at[:, 0]] = (c.float() * s[..., None]).to(dtype)[at[:, 0]]
        assert torch.equal(y, want) and torch.equal(z[at[:, 0]], want[at[:, 0]])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", DT)
def test_extreme_values(cuda, bits, dtype):
    """Zeros, the smallest and largest values, ties, infinities and NaN; one head's do not touch another's."""
    from embodied_efficiency_b200 import KVCache, cache_read, cache_write
    fi = torch.finfo(dtype)
    x = torch.randn(8, 2, 64, device=cuda).to(dtype)
    x[0, 0] = 0
    x[1, 1] = fi.smallest_normal * torch.randn(64, device=cuda)
    x[2, 0] = fi.max
    x[3, 1] = torch.arange(64, device=cuda).to(dtype) - 31.5  # ties of a step of 1
    x[3, 1, 0] = 127 if bits == 8 else 7
    x[4, 0, 3] = float("inf")
    x[5, 1, 63] = -float("inf")
    x[6, 0, 0] = float("nan")
    x[7] = -0.0
    table = torch.zeros(1, 1, dtype=torch.int32, device=cuda)
    cache = KVCache.empty(1, 2, 64, 32, bits)
    cu, lens = offsets([8], cuda), torch.tensor([8], dtype=torch.int32, device=cuda)
    cache_write(cache, x, x, cu, table, lens)
    c, s = quantized(x, bits)
    assert torch.equal(codes_of(cache.k, bits)[0, :, :8].transpose(0, 1), c)
    assert torch.equal(cache.v_scale[0, :, :8].T.nan_to_num(-1), s.nan_to_num(-1))
    k, _ = cache_read(cache, cu, table, lens, 8, dtype)
    assert torch.equal(k.nan_to_num(9), (c.float() * s[..., None]).to(dtype).nan_to_num(9))
    assert torch.equal(s.isnan(), ~x.float().abs().amax(-1).isfinite())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", DT)
def test_every_largest_value(cuda, bits, dtype):
    """Heads with each of the type's finite magnitudes as their largest, and values at and beside the borders between
    codes under it: steps and codes are those of the true divisions."""
    from embodied_efficiency_b200 import KVCache, cache_write
    bitsets = torch.arange(1 << 15, dtype=torch.int32, device=cuda).to(torch.int16).view(dtype)
    amax = bitsets[bitsets.float().isfinite()]
    n = len(amax)
    most = 2 ** (bits - 1) - 1
    half = (torch.arange(63, device=cuda) % most + 0.5) / most  # borders, rounded to the type: on either side of them
    x = (amax.float()[:, None] * torch.cat([torch.ones(1, device=cuda), half])).to(dtype)[:, None]
    x[:, 0, 33:] *= -1
    pages = -(-n // 256)
    cache = KVCache.empty(pages, 1, 64, 256, bits)
    table = torch.arange(pages, dtype=torch.int32, device=cuda)[None]
    cache_write(cache, x, -x, offsets([n], cuda), table, torch.tensor([n], dtype=torch.int32, device=cuda))
    c, s = quantized(x, bits)
    assert torch.equal(codes_of(cache.k, bits).flatten(0, 2)[:n], c[:, 0])
    assert torch.equal(codes_of(cache.v, bits).flatten(0, 2)[:n], -c[:, 0])
    assert torch.equal(cache.k_scale.flatten()[:n], s[:, 0])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", DT)
def test_every_quotient(cuda, bits, dtype):
    """Every value of the type under every largest one, but for powers of two: all significands of the largest value (at
    one exponent, and where the step is held at 1e-8), and under each all values that do not round to a code of 0."""
    from embodied_efficiency_b200 import KVCache, cache_write
    fi = torch.finfo(dtype)
    sig = torch.arange(1, 2, fi.eps, device=cuda, dtype=torch.float64)  # significands
    low = 12 if bits == 8 else 7  # a value 2^-low of the largest is below half a code
    for scale in (1.0, 2.0 ** -21):
        under = torch.cat([sig * 2.0 ** -e for e in range(low)] + [sig * 0])
        pad = -len(under) % 63
        under = torch.cat([under, under.new_zeros(pad)]).view(-1, 63) * scale
        for part in sig.split(64):
            top = part * scale
            x = torch.minimum(under[None].expand(len(top), -1, -1), top[:, None, None])  # none above its largest
            x = torch.cat([top[:, None, None].expand(-1, under.shape[0], 1), x], -1).flatten(0, 1).to(dtype)[:, None]
            n = len(x)
            pages = -(-n // 256)
            cache = KVCache.empty(pages, 1, 64, 256, bits)
            table = torch.arange(pages, dtype=torch.int32, device=cuda)[None]
            cache_write(cache, x, -x, offsets([n], cuda), table, torch.tensor([n], dtype=torch.int32, device=cuda))
            c, s = quantized(x, bits)
            assert torch.equal(codes_of(cache.k, bits).flatten(0, 2)[:n], c[:, 0])
            assert torch.equal(codes_of(cache.v, bits).flatten(0, 2)[:n], -c[:, 0])
            assert torch.equal(cache.v_scale.flatten()[:n], s[:, 0])


def test_what_the_device_says_is_not_trusted(cuda):
    """Page numbers, offsets and lengths outside the cache and the tensors: nothing outside is touched, rows without a
    place stay, the others are right."""
    from embodied_efficiency_b200 import KVCache, cache_read, cache_write
    page, kv, hd, pages = 32, 2, 64, 4
    big = torch.full((3 * pages, kv, page, hd), 55, dtype=torch.int8, device=cuda)
    steps = torch.full((3 * pages, kv, page), 0.5, device=cuda)
    vbig, vsteps = big.clone(), steps.clone()
    cache = KVCache(big[pages:2 * pages], vbig[pages:2 * pages], steps[pages:2 * pages], vsteps[pages:2 * pages])
    x = torch.randn(200, kv, hd, device=cuda).bfloat16()
    table = torch.tensor([[1, 4, 5, -1], [2 ** 31 - 1, 3, 0, -2 ** 31]], dtype=torch.int32, device=cuda)
    for q_off, lens in (([0, 90, 200], [128, 110]), ([-5, 1000, 7], [100, 60]), ([50, 20, 2 ** 31 - 1], [4, 2 ** 31 - 1]),
                        ([3, 3, 3], [-7, -2 ** 31]), ([150, 100, 0], [70, 80])):
        cu, kl = (torch.tensor(v, dtype=torch.int32, device=cuda) for v in (q_off, lens))
        cache_write(cache, x, x, cu, table, kl)
        out = cache_read(cache, cu, table, kl, 200, out=(torch.zeros_like(x), torch.zeros_like(x)))
        torch.cuda.synchronize()
        for t, keep in ((big, 55), (vbig, 55), (steps, 0.5), (vsteps, 0.5)):
            assert bool((t[:pages] == keep).all()) and bool((t[2 * pages:] == keep).all())
        assert bool(out[0].isfinite().all())
    cu, kl = offsets([90, 110], cuda), torch.tensor([128, 110], dtype=torch.int32, device=cuda)
    cache_write(cache, x, x, cu, table, kl)
    k, v = cache_read(cache, cu, table, kl, 200, out=(torch.zeros_like(x), torch.zeros_like(x)))
    table_ok = torch.tensor([[1, -1, -1, -1], [-1, 3, 0, -1]], dtype=torch.int32, device=cuda)
    at = places([90, 110], [128, 110], table_ok, page)[:, 0]
    c, s = quantized(x, 8)
    want = torch.zeros_like(x)
    want[at] = (c.float() * s[..., None]).bfloat16()[at]
    assert torch.equal(k, want) and torch.equal(v, want) and 0 < len(at) < 200


def test_far_pages(cuda):
    """Codes beyond 2^31 bytes and beyond 2^32 from the cache's start."""
    from embodied_efficiency_b200 import KVCache, cache_read, cache_write
    page, kv, hd = 256, 8, 128
    pages = (1 << 32) // (page * kv * hd) + 40
    cache = KVCache.empty(pages, kv, hd, page)
    x = torch.randn(600, kv, hd, device=cuda).half()
    table = torch.tensor([[pages - 1, 0, pages // 2 + 30]], dtype=torch.int32, device=cuda)
    cu, kl = offsets([600], cuda), torch.tensor([600], dtype=torch.int32, device=cuda)
    cache_write(cache, x, -x, cu, table, kl)
    c, s = quantized(x, 8)
    for i, p in enumerate(table[0].tolist()):
        n = min(256, 600 - 256 * i)
        assert torch.equal(cache.k[p, :, :n], c[256 * i:256 * i + n].transpose(0, 1))
        assert torch.equal(cache.v_scale[p, :, :n], s[256 * i:256 * i + n].T)
    k, v = cache_read(cache, cu, table, kl, 600, torch.float16)
    assert torch.equal(k, (c.float() * s[..., None]).half()) and torch.equal(v, -k)


def test_streams_captures_and_odd_operands(cuda):
    from embodied_efficiency_b200 import KVCache, cache_read, cache_write
    kv, hd, page = 4, 64, 64
    q_len, k_len = [3, 9, 1], [70, 9, 64]
    table, pages = tables(k_len, page, cuda, 5)
    cu, kl = offsets(q_len, cuda), torch.tensor(k_len, dtype=torch.int32, device=cuda)
    cache = fill(KVCache.empty(pages, kv, hd, page), 1)
    x = torch.randn(13, kv, hd, device=cuda).bfloat16()
    c, s = quantized(x, 8)
    want = (c.float() * s[..., None]).bfloat16()
    # operands off the 16-byte boundary, a table with a wide row, lengths that are a view
    odd = torch.zeros(13, kv, hd + 1, device=cuda, dtype=torch.bfloat16)[..., 1:].copy_(x)
    wide = torch.full((3, 9), -1, dtype=torch.int32, device=cuda)
    wide[:, :table.shape[1]] = table
    both = torch.stack([kl, kl], 1)
    cache_write(cache, odd, odd, cu, wide[:, :table.shape[1]], both[:, 1])
    assert torch.equal(cache_read(cache, cu, wide.t().contiguous().t(), kl, 13)[1], want)
    # more rows than sequences claim: the last ones stay
    more = torch.cat([x, x])
    out = (torch.zeros_like(more), torch.zeros_like(more))
    cache_write(cache, more, more, cu, table, kl)
    cache_read(cache, cu, table, kl, 26, out=out)
    assert torch.equal(out[0][:13], want) and not bool(out[0][13:].any())
    heads_first = torch.empty(kv, 13, hd, device=cuda, dtype=torch.bfloat16).transpose(0, 1)
    assert torch.equal(cache_read(cache, cu, table, kl, 13, out=(heads_first, torch.empty_like(x)))[0], want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        cache_write(cache, -x, x, cu, table, kl)
        k, v = cache_read(cache, cu, table, kl, 13)
    torch.cuda.synchronize()
    assert torch.equal(k, -want) and torch.equal(v, want)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        cache_write(cache, x, x, cu, table, kl)
        got = cache_read(cache, cu, table, kl, 13)
    x.mul_(2)
    kl.add_(torch.tensor([1, 3, 0], dtype=torch.int32, device=cuda))
    gr.replay()
    torch.cuda.synchronize()
    c, s = quantized(x, 8)
    assert torch.equal(got[0], (c.float() * s[..., None]).bfloat16())
    for empty in (0,):
        z = x[:empty]
        cache_write(cache, z, z, torch.zeros(1, dtype=torch.int32, device=cuda), table[:0], kl[:0])
        assert cache_read(cache, torch.zeros(1, dtype=torch.int32, device=cuda), table[:0], kl[:0], 0)[0].shape == (0, kv, hd)
