"""GPU parity of attention over packed prompts (ee_prompt_attention) against its definition in 64 bits."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16]


def _cu(lens, dev):
    return torch.tensor([0] + list(lens), device=dev).cumsum(0).to(torch.int32)


def _check(out, q, k, v, q_len, k_len, causal, scale, k_start=None, k_used=None):
    """|out - exact| per value. With A = sum_j p_j |v_j| / sum_j p_j: the weights' rounding for the product with v
    gives eps/2 * A, the result's rounding eps/2 * |out|; a score's error of d (fp32 sums of hd products, 2^-22 of
    sum |q k| * scale) moves a weight by a factor e^d, twice with the sum below it; 2^-18 A covers exp2, the sums of up
    to a few thousand weights and the merges. fp16 weights below 2^-14 of the largest round to 2^-25 absolute."""
    i = j = 0
    eps = torch.finfo(out.dtype).eps / 2
    g = q.shape[1] // k.shape[1]
    for b, (nq, nk) in enumerate(zip(q_len, k_len)):
        j0 = j if k_start is None else k_start[b]
        nu = nk if k_used is None else k_used[b]
        if nq:
            qd = q[i:i + nq].double().transpose(0, 1)
            kd = k[j0:j0 + nu].double().transpose(0, 1).repeat_interleave(g, 0)
            vd = v[j0:j0 + nu].double().transpose(0, 1).repeat_interleave(g, 0)
            s = qd @ kd.transpose(1, 2) * scale
            if causal:
                seen = torch.arange(nu, device=q.device)[None] <= torch.arange(nq, device=q.device)[:, None] + (nu - nq)
            else:
                seen = torch.ones(nq, nu, dtype=torch.bool, device=q.device)
            p = torch.softmax(s.masked_fill(~seen, float("-inf")), -1).nan_to_num(0.0)
            ref, mean = p @ vd, p @ vd.abs()
            d = (qd.abs() @ kd.abs().transpose(1, 2) * scale * 2 ** -22).amax(-1, keepdim=True) if nu else 0.0
            tol = eps * (mean + ref.abs()) * (1 + 2 ** -6) + mean * (2 * d + 2 ** -18) + 2.0 ** -24
            if out.dtype == torch.float16 and nu:
                tol = tol + nu * 2.0 ** -25 * vd.abs().amax(1, keepdim=True)
            err = (out[i:i + nq].double().transpose(0, 1) - ref).abs()
            assert bool((err <= tol).all()), (b, nq, nk, float((err / tol).max()))
            if nu == 0:
                assert not bool(out[i:i + nq].any())
        i, j = i + nq, j + nk


def _inputs(dev, dtype, tq, tk, hq, hk, hd, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [(torch.randn(t, h, hd, generator=g, device=dev) * s).to(dtype)
            for t, h, s in ((tq, hq, 1.5), (tk, hk, 1.0), (tk, hk, 1.0))]


SELF = [[1], [2], [64], [65], [127], [128], [129], [256], [257], [0, 5, 0, 0, 130, 1, 0], [300, 1, 511, 17], [1000],
        [33] * 20, [1] * 70]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hq,hk,hd", [(4, 4, 64), (8, 2, 128), (6, 2, 64), (7, 1, 128)])
@pytest.mark.parametrize("lens", SELF, ids=lambda v: "-".join(map(str, v[:7])) + ("x%d" % len(v)))
@pytest.mark.parametrize("causal", [True, False])
def test_prompts(cuda, dtype, hq, hk, hd, lens, causal):
    from embodied_efficiency_b200 import prompt_attention
    t = sum(lens)
    q, k, v = _inputs(cuda, dtype, t, t, hq, hk, hd, t + hq)
    out = prompt_attention(q, k, v, _cu(lens, cuda), causal=causal)
    assert out.shape == q.shape and out.dtype == dtype
    _check(out, q, k, v, lens, lens, causal, hd ** -0.5)


@pytest.mark.parametrize("hq,hk,hd", [(8, 8, 64), (4, 2, 128), (12, 4, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_more_items_than_sms(cuda, hq, hk, hd, causal):
    """Several items per CTA, one after another: lengths on both sides of the tiles, sequences without queries or
    without keys among them."""
    from embodied_efficiency_b200 import prompt_attention
    r = random.Random(hq)
    q_len = [r.choice([0, 1, 20, 64, 127, 128, 129, 200, 256, 257, 300]) for _ in range(90)]
    k_len = [n if r.random() < 0.7 else r.choice([0, 1, n + 5, n + 128, max(n - 3, 0)]) for n in q_len]
    q, k, v = _inputs(cuda, torch.bfloat16, sum(q_len), sum(k_len), hq, hk, hd, 5)
    out = prompt_attention(q, k, v, _cu(q_len, cuda), _cu(k_len, cuda), causal=causal)
    _check(out, q, k, v, q_len, k_len, causal, hd ** -0.5)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hq,hk", [(5, 5), (8, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_last_tiles_that_have_no_neighbour(cuda, dtype, hq, hk, causal):
    """Heads of 64, sequences whose last query tile stands alone against one to nine blocks of keys, many of them per
    CTA and between whole pairs; rows that see nothing of the later blocks; NaN behind every sequence's keys; and
    scores whose largest lies in the first or in the last block."""
    from embodied_efficiency_b200 import prompt_attention
    r = random.Random(hq)
    tile = 128 * hk // hq
    q_len = [r.choice([tile, tile - 1, tile // 2, 2 * tile, 2 * tile + 1, 3 * tile, 3 * tile - 5]) for _ in range(150)]
    k_len = [max(n + r.choice([0, 0, 1, 100]), r.choice([1, 128, 129, 255, 256, 257, 384, 511, 640, 1100])) for n in q_len]
    room = [n + r.choice([0, 3, 200]) for n in k_len]
    q, k, v = _inputs(cuda, dtype, sum(q_len), sum(room), hq, hk, 64, 11)
    start, at = [0], 0
    for i, (n, w) in enumerate(zip(k_len, room)):
        if i % 3:  # a slope along the keys, up or down
            k[at:at + n, :, 0] += (torch.arange(n, device=cuda, dtype=dtype) * (0.125 if i % 3 == 1 else -0.125))[:, None]
        k[at + n:at + w], v[at + n:at + w] = float("nan"), float("nan")
        at += w
        start.append(at)
    q[:, :, 0] = 4.0
    used = torch.tensor(k_len, device=cuda, dtype=torch.int32)
    out = prompt_attention(q, k, v, _cu(q_len, cuda), torch.tensor(start, device=cuda, dtype=torch.int32), used,
                           causal=causal)
    keep = torch.cat([torch.arange(a, a + n) for a, n in zip(start, k_len)]).to(cuda)
    _check(out, q, k[keep], v[keep], q_len, k_len, causal, 0.125)
    assert torch.equal(out, prompt_attention(q, k, v, _cu(q_len, cuda), torch.tensor(start, device=cuda, dtype=torch.int32),
                                             used, causal=causal))


@pytest.mark.parametrize("longest", [3, 40])
def test_many_short_sequences(cuda, longest):
    """More sequences than a CTA has threads, most of them tiny or empty."""
    from embodied_efficiency_b200 import prompt_attention
    r = random.Random(longest)
    q_len = [0 if r.random() < 0.2 else r.randint(0 if longest < 9 else 20, longest) for _ in range(1300)]
    k_len = [n + r.choice([0, 0, 1, 17, 70]) for n in q_len]
    q, k, v = _inputs(cuda, torch.float16, sum(q_len), sum(k_len), 4, 2, 64, 6)
    out = prompt_attention(q, k, v, _cu(q_len, cuda), _cu(k_len, cuda))
    _check(out, q, k, v, q_len, k_len, True, 0.125)


CACHED = [([1], [1]), ([1], [777]), ([1] * 5, [1, 128, 129, 4000, 0]), ([1] * 64, list(range(1, 1300, 20))[:64]),
          ([3, 0, 1, 70], [100, 50, 1, 70]), ([50], [866]), ([50] * 3, [866, 50, 300]), ([200, 100], [700, 1500]),
          ([10, 129, 300], [4, 100, 7]), ([1], [30000]), ([5, 2], [0, 9000]), ([260], [1])]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hq,hk,hd", [(4, 4, 64), (16, 4, 128), (16, 2, 64), (7, 1, 128), (40, 1, 64)])
@pytest.mark.parametrize("q_len,k_len", CACHED, ids=["c%d" % i for i in range(len(CACHED))])
@pytest.mark.parametrize("causal", [True, False])
def test_new_tokens_behind_cached_ones(cuda, dtype, hq, hk, hd, q_len, k_len, causal):
    """Keys that reach further back than the queries, none at all, or fewer than queries (rows that see nothing)."""
    from embodied_efficiency_b200 import prompt_attention
    q, k, v = _inputs(cuda, dtype, sum(q_len), sum(k_len), hq, hk, hd, sum(k_len) + hq)
    out = prompt_attention(q, k, v, _cu(q_len, cuda), _cu(k_len, cuda), causal=causal, scale=0.11)
    _check(out, q, k, v, q_len, k_len, causal, 0.11)


@pytest.mark.parametrize("q_len", [[1, 1, 1], [2, 40, 9], [150, 300, 128]])
@pytest.mark.parametrize("causal", [True, False])
def test_what_lies_beside_the_sequences_is_not_used(cuda, q_len, causal):
    """A cache with room to grow, its unused rows full of NaN and infinities; rows before, between and behind the
    sequences keep what the output held."""
    from embodied_efficiency_b200 import prompt_attention
    cap, used = 400, [333, 300, 128]
    q, k, v = _inputs(cuda, torch.bfloat16, sum(q_len) + 9, 3 * cap, 8, 2, 64, 3)
    for x, bad in ((k, float("nan")), (v, float("inf"))):
        for b in range(3):
            x[b * cap + used[b]:(b + 1) * cap] = bad
            x[b * cap + used[b] + 1:(b + 1) * cap:2] = float("nan")
    q[sum(q_len):] = float("nan")
    out = torch.full_like(q, 7.0)
    cu_q, cu_k = _cu(q_len, cuda), torch.tensor([0, cap, 2 * cap, 3 * cap], device=cuda, dtype=torch.int32)
    res = prompt_attention(q, k, v, cu_q, cu_k, torch.tensor(used, device=cuda, dtype=torch.int32), causal=causal,
                           out=out)
    assert res is out and bool((out[sum(q_len):] == 7.0).all())
    _check(out, q, k, v, q_len, [cap] * 3, causal, 0.125, [0, cap, 2 * cap], used)


@pytest.mark.parametrize("t", [40, 300])
def test_scores_of_any_size(cuda, t):
    """Huge scores (a softmax that picks one key), keys of -inf scores, one key only, NaN kept to its own row."""
    from embodied_efficiency_b200 import prompt_attention
    q, k, v = _inputs(cuda, torch.bfloat16, t, t, 4, 4, 64, 9)
    cu = _cu([t], cuda)
    out = prompt_attention(q * 100, k, v, cu, scale=1.0)
    _check(out, q * 100, k, v, [t], [t], True, 1.0)
    # scores that grow along the keys, so that the running maximum moves in every block
    kk = (torch.arange(t, device=cuda).view(t, 1, 1) * 0.25 * torch.ones_like(k[0])).bfloat16()
    qq = torch.ones_like(q)
    _check(prompt_attention(qq, kk, v, cu, scale=1.0), qq, kk, v, [t], [t], True, 1.0)
    _check(prompt_attention(qq, kk.flip(0), v, cu, scale=1.0), qq, kk.flip(0), v, [t], [t], True, 1.0)
    k2 = k.clone()
    k2[0, :, 0], k2[0, :, 1:] = float("-inf"), 0.0
    q2 = q.abs() + 1
    out = prompt_attention(q2, k2, v, cu, causal=True)
    # key 0 scores -inf for every query: query 0 has nothing left, the others do without it
    assert not bool(out[0].any())
    g = prompt_attention(q2[1:], k2[1:], v[1:], _cu([t - 1], cuda), causal=True)
    assert float((out[1:].float() - g.float()).abs().max()) <= 2 ** -6 * float(g.float().abs().max())
    q3 = q.clone()
    q3[5, 2] = float("nan")
    out = prompt_attention(q3, k, v, cu)
    assert bool(out[5, 2].isnan().all())
    out[5, 2] = 0
    assert bool(out.isfinite().all())


@pytest.mark.parametrize("lens", [[3, 1, 9], [200, 77]])
def test_views_of_a_fused_projection_graphs_and_streams(cuda, lens):
    from embodied_efficiency_b200 import prompt_attention
    t, hq, hk, hd = sum(lens), 8, 2, 64
    qkv = torch.randn(t, (hq + 2 * hk) * hd, device=cuda).bfloat16()

    def parts(x):
        return (x[:, :hq * hd].view(t, hq, hd), x[:, hq * hd:(hq + hk) * hd].view(t, hk, hd),
                x[:, (hq + hk) * hd:].view(t, hk, hd))

    cu = _cu(lens, cuda)
    q, k, v = parts(qkv)
    out = prompt_attention(q, k, v, cu)
    _check(out, q, k, v, lens, lens, True, 0.125)
    assert torch.equal(out, prompt_attention(*(x.contiguous() for x in (q, k, v)), cu))
    heads_first = prompt_attention(*(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)), cu)
    assert torch.equal(out, heads_first)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = prompt_attention(q, k, v, cu)
        graphs.append((gr, res))
    other = torch.randn_like(qkv)
    qkv.copy_(other)
    back = _cu(lens[::-1], cuda)
    cu.copy_(back)  # replayed with other lengths
    for gr, _ in graphs + graphs:
        gr.replay()
    torch.cuda.synchronize()
    want = prompt_attention(*parts(other), back)
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    torch.cuda.synchronize()
    for i in range(6):
        with torch.cuda.stream(side[i % 2]):
            outs.append(prompt_attention(q, k, v, cu))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("t", [3, 300])
@pytest.mark.parametrize("hd", [64, 128])
def test_broadcast_and_head_major_views(cuda, t, hd):
    """Strides of 0 (heads or tokens that share their memory) and heads that lie behind one another."""
    from embodied_efficiency_b200 import prompt_attention
    q, k, v = _inputs(cuda, torch.bfloat16, t, t, 8, 1, hd, 21)
    major = q.transpose(0, 1).contiguous().transpose(0, 1)
    cu = _cu([t], cuda)
    for qq, kk, vv in ((q, k.expand(t, 4, hd), v.expand(t, 4, hd)), (q, k[:1].expand(t, 1, hd), v[:1].expand(t, 1, hd)),
                       (q[:, :1].expand(t, 8, hd), k, v), (q[:1, :1].expand(t, 8, hd), k, v), (major, k, v)):
        _check(prompt_attention(qq, kk, vv, cu), qq, kk, vv, [t], [t], True, hd ** -0.5)


def test_offsets_beyond_the_tensors_are_cut(cuda):
    """Tables that claim rows the tensors do not have read and write nothing outside them."""
    from embodied_efficiency_b200 import prompt_attention
    q, k, v = _inputs(cuda, torch.float16, 40, 90, 4, 2, 64, 1)
    cu_q = torch.tensor([0, 10, 1000], device=cuda, dtype=torch.int32)
    cu_k = torch.tensor([-5, 30, 100000], device=cuda, dtype=torch.int32)
    out = prompt_attention(q, k, v, cu_q, cu_k, torch.tensor([1 << 30, 1 << 30], device=cuda, dtype=torch.int32))
    _check(out, q, k, v, [10, 30], [30, 60], True, 0.125)


def test_long_cache_offsets_pass_32_bits(cuda):
    """A key row whose byte offset needs more than 32 bits."""
    from embodied_efficiency_b200 import prompt_attention
    rows, hk, hd = 2_300_000, 8, 64
    k = torch.empty(rows, 2 * hk, hd, device=cuda, dtype=torch.bfloat16)  # 4.7 GB: keys and values of a row together
    kk, vv = k[:, :hk], k[:, hk:]
    for lens, nq in (([700], 1), ([700], 200)):
        start = rows - 700
        k[start:].normal_()
        q = torch.randn(nq, 16, hd, device=cuda).bfloat16()
        cu_k = torch.tensor([start, rows], device=cuda, dtype=torch.int32)
        out = prompt_attention(q, kk, vv, _cu([nq], cuda), cu_k)
        _check(out, q, kk[start:], vv[start:], [nq], lens, True, 0.125)
