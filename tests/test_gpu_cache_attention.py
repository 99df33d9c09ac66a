"""GPU parity of attention over a paged cache of quantised keys and values (ee_cache_attention), with and without a shared
prefix, against its definition in 64 bits."""
import random

import pytest
import torch

from test_gpu_cache import codes_of, fill, offsets, tables

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16]


def held(cache, table, b, n):
    """Keys and values 0..n of sequence b in 64 bits, and which of them are there."""
    at = torch.arange(n, device=cache.device)
    row = table[b].long()
    page = row[at // cache.page_size] if n else at
    there = (page >= 0) & (page < cache.pages)
    page = page.clamp(0, cache.pages - 1)
    out = []
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = codes_of(c.transpose(1, 2)[page, at % cache.page_size], cache.bits).double()
        x = x * s.transpose(1, 2)[page, at % cache.page_size].double()[..., None]
        out.append(torch.where(there[:, None, None], x, torch.zeros_like(x)))
    return out[0], out[1], there


def check(out, q, cache, table, q_len, k_len, causal, scale, prefix=None):
    """|out - exact| per value. With A = sum_j p_j |v_j| / sum_j p_j: the weights' rounding for the product with v gives
    2^-8 A (bf16) or 2^-16 A (fp16, rounded twice; behind a prefix and with more than 16 rows a sequence and key head
    rounded once, 2^-11 A, and 2^-25 absolute per weight where the largest is at least 2^-1), the result's rounding half a step of it; a score's error of d moves a weight by a factor e^d, twice
    with the sum below it: fp32 sums of hd products, the steps' and the exponent's roundings 2^-22 of sum |q k| scale,
    and bf16 queries as fp16 2^-25 of the row's largest times sum |k|; 2^-18 A covers exp2, the sums of up to a few
    thousand weights and the merges."""
    fi = torch.finfo(out.dtype)
    f16 = out.dtype == torch.float16
    g = q.shape[1] // cache.kv_heads
    i = 0
    many = sum(q_len) * g > 16 * len(q_len) and g <= 128
    for b, (nq, nk) in enumerate(zip(q_len, k_len)):
        if nq:
            kd, vd, there = held(cache, table, b, nk)
            qd = q[i:i + nq].double().transpose(0, 1)
            seen = there[None].expand(nq, nk).clone()
            if causal:
                seen &= torch.arange(nk, device=q.device)[None] <= torch.arange(nq, device=q.device)[:, None] + (nk - nq)
            if prefix is not None:
                kd, vd = torch.cat([prefix[0].double(), kd]), torch.cat([prefix[1].double(), vd])
                seen = torch.cat([seen.new_ones(nq, len(prefix[0])), seen], 1)
            kd, vd = (x.transpose(0, 1).repeat_interleave(g, 0) for x in (kd, vd))
            s = (qd @ kd.transpose(1, 2) * scale).masked_fill(~seen, float("-inf"))
            p = torch.softmax(s, -1).nan_to_num(0.0)
            ref, mean = p @ vd, p @ vd.abs()
            n = kd.shape[1]
            d = 0.0
            if n:
                d = (qd.abs() @ kd.abs().transpose(1, 2) * 2 ** -22).amax(-1, keepdim=True)
                if not f16:
                    d = d + qd.abs().amax(-1, keepdim=True) * kd.abs().sum(-1).amax(-1)[:, None, None] * 2 ** -25
                d = d * scale
            weights = 2.0 ** -8 if not f16 else (2.0 ** -11 if many or prefix is not None else 2.0 ** -16)
            tol = (weights * mean + fi.eps / 2 * ref.abs()) * (1 + 2 ** -6) + mean * (2 * d + 2 ** -18) + 2.0 ** -24
            if f16 and n and (many or prefix is not None):
                tol = tol + (n if many else len(prefix[0])) * 2.0 ** -25 * vd.abs().amax(1, keepdim=True)
            got = out[i:i + nq].double().transpose(0, 1)
            err = (got - ref).abs()
            # rounding to nearest gives infinity from the largest value and half its step on
            err[(got == ref.to(out.dtype).double()) & got.isinf()] = 0
            assert bool((err <= tol).all()), (b, nq, nk, float((err / tol).max()))
            none = ~seen.any(-1)
            assert not bool(got[:, none].any())
        i += nq


def make(dev, dtype, bits, hq, hk, hd, page, q_len, k_len, seed, prefix=0, holes=False):
    """Queries, a cache whose unused places hold NaN and infinite steps, and the tables of the call."""
    from embodied_efficiency_b200 import KVCache
    g = torch.Generator(device=dev).manual_seed(seed)
    table, pages = tables(k_len, page, dev, seed)
    cache = fill(KVCache.empty(pages, hk, hd, page, bits), seed)
    used = torch.zeros(pages, page, dtype=torch.bool, device=dev)
    for b, n in enumerate(k_len):
        at = torch.arange(max(n, 0), device=dev)
        used[table[b].long()[at // page], at % page] = True
    for s, bad in ((cache.k_scale, float("nan")), (cache.v_scale, float("inf"))):
        s.copy_(torch.where(used[:, None], s * (40 if bits == 4 else 2), torch.full_like(s, bad)))
    if holes:  # pages that are not there, in the middle of sequences
        r = random.Random(seed)
        for b in range(table.shape[0]):
            if r.random() < 0.5:
                table[b, r.randrange(table.shape[1])] = r.choice([-1, pages, 2 ** 31 - 1, -2 ** 31])
    q = (torch.randn(sum(q_len), hq, hd, generator=g, device=dev) * 1.5).to(dtype)
    pre = None
    if prefix:
        pre = tuple((torch.randn(prefix, hk, hd, generator=g, device=dev) * s).to(dtype) for s in (1.0, 0.8))
    return q, cache, offsets(q_len, dev), table, torch.tensor(k_len, dtype=torch.int32, device=dev), pre


def status():
    from embodied_efficiency_b200.wq_gemm import gemm_status
    return gemm_status()


LENS = [([1], [1]), ([1], [31]), ([1], [33]), ([1], [1000]), ([1] * 70, list(range(70))), ([1, 1, 1], [5000, 3, 257]),
        ([0, 1, 0, 1], [7, 0, 0, 64]), ([50], [816]), ([50, 50, 50], [50, 300, 64]), ([3, 17, 1, 9], [30, 17, 100, 4]),
        ([130, 5], [130, 77]), ([40], [10])]
HEADS = [(1, 1), (4, 4), (8, 2), (7, 1), (16, 2), (16, 1), (40, 2), (12, 4)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("hq,hk", HEADS)
@pytest.mark.parametrize("causal", [True, False])
def test_cache(cuda, dtype, bits, hd, hq, hk, causal):
    from embodied_efficiency_b200 import cache_attention
    for i, (q_len, k_len) in enumerate(LENS):
        page = (32, 64, 128, 256)[(i + hq) % 4]
        q, cache, cu, table, kl, _ = make(cuda, dtype, bits, hq, hk, hd, page, q_len, k_len, i + hq)
        out = cache_attention(q, cache, cu, table, kl, causal=causal)
        assert out.shape == q.shape and out.dtype == dtype
        check(out, q, cache, table, q_len, k_len, causal, hd ** -0.5)
    assert status() == 0


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("bits,hd,hq,hk", [(8, 128, 8, 2), (4, 64, 6, 2), (8, 64, 16, 1), (4, 128, 5, 5), (8, 128, 40, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_shared_prefix(cuda, dtype, bits, hd, hq, hk, causal):
    from embodied_efficiency_b200 import cache_attention
    for i, (plen, q_len, k_len) in enumerate([(1, [1], [1]), (100, [1] * 40, list(range(40))), (700, [1, 1], [0, 500]),
                                              (2000, [1] * 9, [70] * 9), (816, [50] * 3, [50, 60, 0]),
                                              (300, [0, 20, 200], [9, 3, 200]), (4100, [1], [0])]):
        q, cache, cu, table, kl, pre = make(cuda, dtype, bits, hq, hk, hd, 64, q_len, k_len, i, plen)
        out = cache_attention(q, cache, cu, table, kl, causal=causal, prefix=pre)
        check(out, q, cache, table, q_len, k_len, causal, hd ** -0.5, pre)
    # a prefix without keys is none
    none = tuple(x[:0] for x in pre)
    assert torch.equal(cache_attention(q, cache, cu, table, kl, causal=causal, prefix=none),
                       cache_attention(q, cache, cu, table, kl, causal=causal))
    assert status() == 0


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hq,hk,nq", [(4, 4, 1), (8, 1, 1), (12, 1, 1), (4, 2, 30)])
def test_many_and_long(cuda, dtype, bits, hq, hk, nq):
    """Items cut many times over, several items a share, and hundreds of sequences."""
    from embodied_efficiency_b200 import cache_attention
    r = random.Random(hq)
    for k_len in ([40000], [r.choice([0, 1, 31, 32, 33, 500, 1500]) for _ in range(300)], [20000, 1, 0, 9000, 64, 7]):
        q_len = [r.choice([nq, nq, 0]) for _ in k_len[1:]] + [nq]
        q, cache, cu, table, kl, _ = make(cuda, dtype, bits, hq, hk, 64, 64, q_len, k_len, 3, holes=True)
        check(cache_attention(q, cache, cu, table, kl, scale=0.2), q, cache, table, q_len, k_len, True, 0.2)
    assert status() == 0


def test_extreme_scores(cuda):
    """Scores hundreds apart, values of very different steps, rows of zeros and of large and tiny queries."""
    from embodied_efficiency_b200 import cache_attention
    q_len, k_len = [1] * 12, [200] * 12
    for dtype in DT:
        q, cache, cu, table, kl, _ = make(cuda, dtype, 8, 4, 2, 64, 64, q_len, k_len, 11)
        ok = cache.k_scale.isfinite()
        cache.k_scale.copy_(torch.where(ok, cache.k_scale * torch.exp(3 * torch.randn_like(cache.k_scale)), cache.k_scale))
        cache.v_scale.copy_(torch.where(ok, torch.exp(6 * torch.randn_like(cache.v_scale)) * 1e-3, cache.v_scale))
        q[0] = 0
        q[1] *= 100
        q[2] *= 1e-6
        q[3, :, ::2] *= 1e-4
        q[3, :, 0] = 60
        out = cache_attention(q, cache, cu, table, kl)
        check(out, q, cache, table, q_len, k_len, True, 0.125)
        # a NaN key reaches the rows that see it, and no others
        cache.k_scale[table[5, 1], 0, 3] = float("nan")
        cache.v_scale[table[6, 0], 1, 9] = float("nan")
        got = cache_attention(q, cache, cu, table, kl)
        assert bool(got[5, :2].isnan().all()) and bool(got[6, 2:].isnan().all())
        keep = torch.ones(12, 4, dtype=torch.bool, device=cuda)
        keep[5, :2] = keep[6, 2:] = False
        assert torch.equal(got[keep], out[keep])


def test_a_nan_key_under_the_mask(cuda):
    from embodied_efficiency_b200 import cache_attention
    q, cache, cu, table, kl, _ = make(cuda, torch.bfloat16, 8, 2, 1, 64, 32, [20], [50], 4)
    out = cache_attention(q, cache, cu, table, kl)
    for s in (cache.k_scale, cache.v_scale):
        s[table[0, 1], 0, 45 - 32] = float("nan")  # key 45: seen by queries 15 and up
    got = cache_attention(q, cache, cu, table, kl)
    assert torch.equal(got[:15], out[:15]) and bool(got[15:].isnan().all())


def test_what_the_device_says_is_not_trusted(cuda):
    """Lengths, offsets and pages outside the cache and the tensors: rows of no sequence stay, the rest is finite."""
    from embodied_efficiency_b200 import cache_attention
    for hq in (2, 16, 40):
        q, cache, _, _, _, _ = make(cuda, torch.bfloat16, 8, hq, 2, 64, 32, [64], [500], 4)
        cache.k_scale.fill_(0.01), cache.v_scale.fill_(0.01)
        table = torch.tensor([[0, 99, 3, -1], [2 ** 31 - 1, 1, 2, -2 ** 31]], dtype=torch.int32, device=cuda)
        for q_off, lens in (([0, 9, 20], [128, 110]), ([-5, 1000, 7], [2 ** 31 - 1, 60]), ([5, 2, 2 ** 31 - 1], [4, 129]),
                            ([3, 3, 3], [-7, -2 ** 31]), ([30, 10, 0], [70, 80])):
            cu, kl = (torch.tensor(v, dtype=torch.int32, device=cuda) for v in (q_off, lens))
            out = cache_attention(q, cache, cu, table, kl, out=torch.full_like(q, 3.0))
            assert bool(out.isfinite().all())
        cu, kl = offsets([9, 11], cuda), torch.tensor([128, 110], dtype=torch.int32, device=cuda)
        out = cache_attention(q, cache, cu, table, kl, out=torch.full_like(q, 3.0))
        assert bool((out[20:] == 3).all())
        check(out[:20], q[:20], cache, table, [9, 11], [128, 110], True, 0.125)
        # lengths beyond the table are cut to it
        kl = torch.tensor([4000, 129], dtype=torch.int32, device=cuda)
        check(cache_attention(q, cache, cu, table, kl)[:20], q[:20], cache, table, [9, 11], [128, 128], True, 0.125)
    assert status() == 0


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd,nq,prefix", [(64, 1, 0), (128, 1, 300), (128, 50, 0), (64, 50, 300), (64, 50, 0)])
def test_two_roundings_at_most(cuda, dtype, bits, hd, nq, prefix):
    """The weights' rounding for their product with the values and the result's: errors of one size that do not depend on
    one another, sqrt(2) of the result's alone; 1.5 leaves 6 % for the fp32 steps between them."""
    from embodied_efficiency_b200 import cache_attention
    k_len = [nq + 40 * i for i in range(6)]
    q, cache, cu, table, kl, pre = make(cuda, dtype, bits, 8, 4, hd, 64, [nq] * 6, k_len, 17, prefix)
    out = cache_attention(q, cache, cu, table, kl, prefix=pre)
    err, half = [], []
    for b, n in enumerate(k_len):
        kd, vd, _ = held(cache, table, b, n)
        if prefix:
            kd, vd = torch.cat([pre[0].double(), kd]), torch.cat([pre[1].double(), vd])
        kd, vd = (x.transpose(0, 1).repeat_interleave(2, 0) for x in (kd, vd))
        s = q[b * nq:(b + 1) * nq].double().transpose(0, 1) @ kd.transpose(1, 2) * hd ** -0.5
        at = torch.arange(kd.shape[1], device=cuda)[None] - torch.arange(nq, device=cuda)[:, None]
        ref = torch.softmax(s.masked_fill(at > n + prefix - nq, float("-inf")), -1) @ vd
        err.append(out[b * nq:(b + 1) * nq].double().transpose(0, 1) - ref)
        half.append(ref.to(dtype).double() - ref)
    rms = lambda x: float(torch.cat([y.flatten() for y in x]).pow(2).mean().sqrt())
    assert rms(err) <= 1.5 * rms(half)


@pytest.mark.parametrize("plen", [100, 2000])
@pytest.mark.parametrize("nq", [1, 30])
def test_rows_outside_the_sequences_behind_a_prefix(cuda, plen, nq):
    """Rows before the first and behind the last sequence stay as they were; captured calls repeat what eager ones give."""
    from embodied_efficiency_b200 import cache_attention
    n = 7
    q, cache, _, table, kl, pre = make(cuda, torch.bfloat16, 8, 8, 2, 128, 64, [nq] * n + [5], [40 * i for i in range(n)] + [9],
                                       8, plen)
    table, kl = table[:n], kl[:n]
    cu = torch.arange(n + 1, device=cuda, dtype=torch.int32) * nq + 3
    out = cache_attention(q, cache, cu, table, kl, prefix=pre, out=torch.full_like(q, 3.0))
    assert bool((out[:3] == 3).all()) and bool((out[3 + n * nq:] == 3).all())
    check(out[3:3 + n * nq], q[3:3 + n * nq], cache, table, [nq] * n, [40 * i for i in range(n)], True, 128 ** -0.5, pre)
    graph, held = torch.cuda.CUDAGraph(), torch.full_like(q, 3.0)
    with torch.cuda.graph(graph):
        cache_attention(q, cache, cu, table, kl, prefix=pre, out=held)
        again = cache_attention(held, cache, cu, table, kl, prefix=pre, out=torch.empty_like(q).fill_(3.0))
    for _ in range(3):
        held.fill_(3.0)
        graph.replay()
    assert torch.equal(held, out)
    assert torch.equal(again, cache_attention(out, cache, cu, table, kl, prefix=pre, out=torch.full_like(q, 3.0)))
    assert status() == 0


def test_far_pages(cuda):
    """Codes beyond 2^31 and 2^32 bytes from the cache's start."""
    from embodied_efficiency_b200 import KVCache, cache_attention, cache_write
    page, kv, hd = 256, 8, 128
    pages = (1 << 32) // (page * kv * hd) + 40
    cache = KVCache.empty(pages, kv, hd, page)
    x = torch.randn(600, kv, hd, device=cuda).half()
    table = torch.tensor([[pages - 1, 0, pages // 2 + 30]], dtype=torch.int32, device=cuda)
    cu, kl = offsets([600], cuda), torch.tensor([600], dtype=torch.int32, device=cuda)
    cache_write(cache, x, -x, cu, table, kl)
    q = torch.randn(3, 16, hd, device=cuda).half()
    check(cache_attention(q, cache, offsets([3], cuda), table, kl), q, cache, table, [3], [600], True, hd ** -0.5)
    q = torch.randn(70, 16, hd, device=cuda).half()
    check(cache_attention(q, cache, offsets([70], cuda), table, kl), q, cache, table, [70], [600], True, hd ** -0.5)


@pytest.mark.parametrize("nq", [1, 40])
def test_no_keys_at_all(cuda, nq):
    """A table of no pages, a cache of none: only the shared prefix is seen, or nothing."""
    from embodied_efficiency_b200 import KVCache, cache_attention
    q, cache, cu, table, kl, pre = make(cuda, torch.bfloat16, 8, 8, 2, 64, 32, [nq] * 3, [nq] * 3, 5, 70)
    none = KVCache.empty(0, 2, 64, 32)
    for c, t in ((cache, table[:, :0]), (none, table), (none, table[:, :0])):
        assert not bool(cache_attention(q, c, cu, t, kl).any())
        check(cache_attention(q, c, cu, t, kl, prefix=pre), q, cache, table, [nq] * 3, [0] * 3, True, 64 ** -0.5, pre)
    assert status() == 0


@pytest.mark.parametrize("hq,hk,nq", [(130, 1, 2), (300, 1, 1), (128, 1, 3), (256, 2, 1), (127, 1, 2)])
def test_wide_groups(cuda, hq, hk, nq):
    """Groups that fill or do not fit a tile of 128 rows; above, a prefix is refused."""
    from embodied_efficiency_b200 import cache_attention
    q_len, k_len = [nq, 1, 0, nq], [300, 1, 5, 64]
    q, cache, cu, table, kl, pre = make(cuda, torch.bfloat16, 4, hq, hk, 64, 64, q_len, k_len, 2, 150)
    check(cache_attention(q, cache, cu, table, kl), q, cache, table, q_len, k_len, True, 0.125)
    if hq // hk > 128:
        with pytest.raises(ValueError, match="128"):
            cache_attention(q, cache, cu, table, kl, prefix=pre)
    else:
        check(cache_attention(q, cache, cu, table, kl, prefix=pre), q, cache, table, q_len, k_len, True, 0.125, pre)
    assert status() == 0


@pytest.mark.parametrize("nq", [1, 9])
def test_thousands_of_sequences(cuda, nq):
    from embodied_efficiency_b200 import cache_attention
    r = random.Random(nq)
    k_len = [r.choice([0, 1, 9, 40, 70]) for _ in range(3000)]
    q_len = [r.choice([0, nq, nq]) for _ in k_len]
    q, cache, cu, table, kl, pre = make(cuda, torch.bfloat16, 8, 4, 2, 64, 32, q_len, k_len, 1, 40)
    check(cache_attention(q, cache, cu, table, kl), q, cache, table, q_len, k_len, True, 0.125)
    check(cache_attention(q, cache, cu, table, kl, prefix=pre), q, cache, table, q_len, k_len, True, 0.125, pre)
    assert status() == 0


def test_calls_at_once(cuda):
    """Calls of every kernel and order on four streams from four threads give what each gives by itself."""
    import threading
    from embodied_efficiency_b200 import cache_attention
    sets = [make(cuda, torch.bfloat16, 8, 8, 2, 64, 64, [n] * 20, [n + 37 * i for i in range(20)], n, 200) for n in (1, 3, 30, 60)]
    want = [[cache_attention(*s[:5], prefix=p) for p in (None, s[5])] for s in sets]
    torch.cuda.synchronize()
    bad = []

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for k in range(40):
                s = sets[(i + k) % 4]
                for j, p in enumerate((None, s[5])):
                    if not torch.equal(cache_attention(*s[:5], prefix=p), want[(i + k) % 4][j]):
                        bad.append((i, k, j))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad and status() == 0


def test_views_streams_and_captures(cuda):
    from embodied_efficiency_b200 import cache_attention
    q_len, k_len = [1, 4, 1], [700, 4, 33]
    q, cache, cu, table, kl, pre = make(cuda, torch.bfloat16, 8, 8, 2, 128, 64, q_len, k_len, 8, prefix=300)
    want, with_pre = cache_attention(q, cache, cu, table, kl), cache_attention(q, cache, cu, table, kl, prefix=pre)
    wide = torch.zeros(6, 20, 128, device=cuda, dtype=q.dtype)
    wide[:, 3:11] = q
    odd = torch.zeros(6, 8, 129, device=cuda, dtype=q.dtype)[..., 1:].copy_(q)
    fused = torch.cat([pre[0], pre[1]], 1)  # keys and values of one projection
    out = torch.zeros(8, 6, 128, device=cuda, dtype=q.dtype).transpose(0, 1)
    for got in (cache_attention(wide[:, 3:11], cache, cu, table, kl), cache_attention(odd, cache, cu, table, kl),
                cache_attention(q, cache, cu, table, kl, out=out)):
        assert torch.equal(got, want)
    assert torch.equal(cache_attention(q, cache, cu, table, kl, prefix=(fused[:, :2], fused[:, 2:])), with_pre)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        a = cache_attention(q, cache, cu, table, kl)
        b = cache_attention(q, cache, cu, table, kl, prefix=pre)
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, with_pre)
    graphs = []
    for p in (None, pre):  # two captured calls, replayed side by side
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            graphs.append((gr, cache_attention(q, cache, cu, table, kl, prefix=p)))
        graphs[-1] = (gr, graphs[-1][1])
    for _ in range(3):
        with torch.cuda.stream(side):
            graphs[0][0].replay()
        graphs[1][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], with_pre)
    kl.sub_(1)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    check(graphs[0][1], q, cache, table, q_len, [n - 1 for n in k_len], True, 128 ** -0.5)
    kl.add_(1)
    assert cache_attention(q[:0], cache, cu, table, kl).shape == (0, 8, 128)
    empty = torch.zeros(1, dtype=torch.int32, device=cuda)
    keep = torch.full_like(q, 2.0)
    assert cache_attention(q, cache, empty, table[:0], kl[:0], out=keep) is keep and bool((keep == 2).all())
    # a table of no pages: no keys
    assert not bool(cache_attention(q, cache, cu, table[:, :0], kl).any())
    for scale in (0.0, 1e-40, float("nan"), float("inf"), -0.1):
        with pytest.raises(ValueError, match="scale"):
            cache_attention(q, cache, cu, table, kl, scale=scale)
    for shared in (q[:1].expand(6, 8, 128),):
        with pytest.raises(ValueError, match="overlap"):
            cache_attention(q, cache, cu, table, kl, out=shared)


def test_calls_repeat_exactly(cuda):
    from embodied_efficiency_b200 import cache_attention
    q, cache, cu, table, kl, pre = make(cuda, torch.float16, 4, 12, 4, 64, 32, [1] * 50, list(range(1, 1000, 20)), 9, 500)
    want = cache_attention(q, cache, cu, table, kl, prefix=pre)
    for _ in range(5):
        assert torch.equal(cache_attention(q, cache, cu, table, kl, prefix=pre), want)


def test_gradients_are_refused(cuda):
    import torch.autograd.forward_ad as fwAD
    from embodied_efficiency_b200 import cache_attention, cache_write, norm_rotary_embed
    q, cache, cu, table, kl, pre = make(cuda, torch.bfloat16, 8, 4, 2, 64, 32, [3], [40], 9, 20)
    w, pos, k = torch.ones(64, device=cuda), torch.arange(3, device=cuda), q[:, :2]

    def calls(f):
        return (lambda: cache_attention(f(q), cache, cu, table, kl),
                lambda: cache_attention(q, cache, cu, table, kl, prefix=(pre[0], f(pre[1]))),
                lambda: cache_write(cache, f(k), k, cu, table, kl), lambda: cache_write(cache, k, f(k), cu, table, kl),
                lambda: norm_rotary_embed(f(q), k, w, w, pos, (32,)), lambda: norm_rotary_embed(q, k, w, f(w), pos, (32,)))

    norm_rotary_embed(q, k, w, w, pos, (32,))
    for call in calls(lambda t: t.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="no backward pass"):
            call()
    with torch.no_grad():
        for call in calls(lambda t: t.clone().requires_grad_()):
            call()
    with torch.no_grad(), fwAD.dual_level():
        for call in calls(lambda t: fwAD.make_dual(t, torch.ones_like(t))):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()


def test_native_and_python_agree(cuda, monkeypatch):
    from embodied_efficiency_b200 import KVCache, _lib, cache_attention, cache_read, cache_write, norm_rotary_embed
    q, cache, cu, table, kl, pre = make(cuda, torch.bfloat16, 8, 4, 2, 64, 32, [3, 1], [40, 7], 9, 20)
    k, w, pos = q[:, :2], torch.rand(64, device=cuda), torch.arange(4, device=cuda)
    norm_rotary_embed(q, k, w, w, pos, (32,))

    def written():
        cache_write(cache, k, q[:, 2:], cu, table, kl)
        return cache.k.clone(), cache.v.clone()

    calls = {"norm_rotary_embed": lambda: norm_rotary_embed(q, k, w, w, pos, (32,)),
             "cache_write": written, "cache_read": lambda: cache_read(cache, cu, table, kl, 4),
             "cache_attention": lambda: (cache_attention(q, cache, cu, table, kl),
                                         cache_attention(q, cache, cu, table, kl, False, 0.3, pre))}
    native = _lib.native()
    for name, call in calls.items():
        seen = []

        class Spy:
            def __getattr__(self, n):
                def f(*a):
                    y = getattr(native, n)(*a)
                    seen.append((n, y is not None))
                    return y
                return f

        class Off:
            def __getattr__(self, n):
                return lambda *a: None

        monkeypatch.setattr(_lib, "_native", Spy())
        got = call()
        assert seen and all(n == name and took for n, took in seen), (name, seen)
        monkeypatch.setattr(_lib, "_native", Off())
        for u, t in zip(got, call()):
            assert u.shape == t.shape and u.dtype == t.dtype and torch.equal(u, t), name
    monkeypatch.setattr(_lib, "_native", native)
    assert repr(cache).startswith("KVCache(") and isinstance(cache, KVCache)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hq,hk,hd", [(8, 2, 64), (16, 4, 128)])
def test_a_layer_step_by_step(cuda, bits, hq, hk, hd):
    """Norm and rotation, the cache written, attention over it: a prompt, then single tokens, then a chunk, each call
    against the definition on what the step before it gave; three sequences behind a shared prefix."""
    from embodied_efficiency_b200 import KVCache, cache_attention, cache_read, cache_write, norm_rotary_embed
    from test_gpu_norm_rotary import _check as check_rotated
    g = torch.Generator(device=cuda).manual_seed(bits)
    page, dtype, plen = 32, torch.bfloat16, 90
    qw, kw = (1 + 0.2 * torch.randn(2, hd, generator=g, device=cuda)).unbind(0)
    pre = tuple(torch.randn(plen, hk, hd, generator=g, device=cuda).to(dtype) for _ in range(2))
    table, pages = tables([300, 200, 260], page, cuda, 2)
    cache = KVCache.empty(pages, hk, hd, page, bits)
    for t in (cache.k_scale, cache.v_scale):
        t.fill_(float("nan"))
    have, everything = [0, 0, 0], [[[], []] for _ in range(3)]
    for new in ([130, 40, 71], [1, 1, 1], [1, 0, 1], [50, 50, 50], [1, 1, 1]):
        t = sum(new)
        qkv = torch.randn(t, hq + 2 * hk, hd, generator=g, device=cuda).to(dtype)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        pos = torch.cat([plen + h + torch.arange(n, device=cuda) for h, n in zip(have, new)]).to(torch.int32)
        have = [h + n for h, n in zip(have, new)]
        cu, kl = offsets(new, cuda), torch.tensor(have, dtype=torch.int32, device=cuda)
        qr, kr = norm_rotary_embed(q, k, qw, kw, pos, (hd // 2,))
        check_rotated(qr, q, qw, 1e-6, pos[None], (hd // 2,), False)
        check_rotated(kr, k, kw, 1e-6, pos[None], (hd // 2,), False)
        cache_write(cache, kr, v, cu, table, kl)
        out = cache_attention(qr, cache, cu, table, kl, prefix=pre)
        check(out, qr, cache, table, new, have, True, hd ** -0.5, pre)
        back, at = cache_read(cache, cu, table, kl, t), 0
        for b, n in enumerate(new):
            for i in range(2):
                everything[b][i].append(back[i][at:at + n])
            at += n
    # the whole cache as it was read after each step
    whole = cache_read(cache, offsets(have, cuda), table, kl, sum(have))
    for i in range(2):
        assert torch.equal(whole[i], torch.cat([torch.cat(e[i]) for e in everything]))
    # and what the codes stand for is near what was written: half a step of amax / 127 or / 7
    tail = (back[0].float() - kr.float()).abs().amax(-1) / kr.float().abs().amax(-1)
    assert float(tail.max()) <= (0.5 / 127 if bits == 8 else 0.5 / 7) + 2 ** -7
