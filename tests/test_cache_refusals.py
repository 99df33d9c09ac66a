"""What the norm with rotation and the cache's operators refuse, on a machine without a GPU: Python arguments before any
device call, and the C ABI's error codes before any launch."""
import ctypes

import pytest
import torch

BF = torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    from embodied_efficiency_b200 import _lib, build
    build.build()
    return _lib.load()


def test_norm_rotary_arguments():
    from embodied_efficiency_b200 import norm_rotary_embed
    q, k, p = torch.zeros(5, 4, 64, dtype=BF), torch.zeros(5, 2, 64, dtype=BF), torch.zeros(5, dtype=torch.int32)
    w = torch.ones(64)
    for match, call in (
            ("q_weight must be \\[64\\]", lambda: norm_rotary_embed(q, k, w[:32], w, p, (32,))),
            ("q_weight must be \\[64\\]", lambda: norm_rotary_embed(q, k, None, w, p, (32,))),
            ("k_weight must be \\[64\\]", lambda: norm_rotary_embed(q, k, w, w[None], p, (32,))),
            ("k_weight must be fp32", lambda: norm_rotary_embed(q, k, w, w.half(), p, (32,))),
            ("q_weight is", lambda: norm_rotary_embed(q, k, w, w.to(BF), p, (32,))),
            ("eps must be", lambda: norm_rotary_embed(q, k, w, w, p, (32,), eps=0.0)),
            ("eps must be", lambda: norm_rotary_embed(q, k, w, w, p, (32,), eps=float("nan"))),
            ("eps must be", lambda: norm_rotary_embed(q, k, w, w, p, (32,), eps=float("inf"))),
            ("sum to head_dim / 2", lambda: norm_rotary_embed(q, k, w, w, p, (30,))),
            ("base must be", lambda: norm_rotary_embed(q, k, w, w, p, (32,), base=1.0)),
            ("norm_rotary_embed needs q or k", lambda: norm_rotary_embed(None, None, w, w, p, (32,)))):
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError, match="no CPU path"):
        norm_rotary_embed(q, k, w, w, p, (32,))


def _tensors(pages=3, heads=2, size=32, hd=64, dtype=torch.int8):
    return ([torch.zeros(pages, heads, size, hd, dtype=dtype) for _ in range(2)]
            + [torch.zeros(pages, heads, size) for _ in range(2)])


def test_cache_tensors():
    from embodied_efficiency_b200 import KVCache
    k, v, ks, vs = _tensors()
    for match, call in (
            ("k must be int8", lambda: KVCache(k.float(), v, ks, vs)),
            ("k must be int8", lambda: KVCache(k[0], v, ks, vs)),
            ("head_dim must be", lambda: KVCache(*_tensors(hd=32))),
            ("head_dim must be", lambda: KVCache(*_tensors(hd=128, dtype=torch.uint8))),
            ("page_size must be", lambda: KVCache(*_tensors(size=48))),
            ("at least one head", lambda: KVCache(*_tensors(heads=0))),
            ("v torch.int8", lambda: KVCache(k, v[:2], ks, vs)),
            ("k_scale must be", lambda: KVCache(k, v, ks.half(), vs)),
            ("v_scale must be", lambda: KVCache(k, v, ks, vs[..., :16])),
            ("v must be contiguous", lambda: KVCache(k, v.transpose(0, 1).contiguous().transpose(0, 1), ks, vs)),
            ("k_scale must not ask", lambda: KVCache(k, v, ks.clone().requires_grad_(), vs)),
            ("bits must be", lambda: KVCache.empty(3, 2, 64, bits=3, device="cpu"))):
        with pytest.raises(ValueError, match=match):
            call()
    for call in (lambda: KVCache(k, v, ks, vs), lambda: KVCache.empty(3, 2, 64, device="cpu")):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


@pytest.fixture
def cache(monkeypatch):
    """A record over host tensors: its calls end at the check of their device."""
    from embodied_efficiency_b200 import KVCache, _lib
    with monkeypatch.context() as m:
        m.setattr(_lib, "same_device", lambda *t: t[0].device)
        return KVCache(*_tensors())


def test_cache_arguments(cache):
    from embodied_efficiency_b200 import cache_read, cache_write
    x, cu = torch.zeros(5, 2, 64, dtype=BF), torch.tensor([0, 5], dtype=torch.int32)
    tab, kl = torch.zeros(1, 4, dtype=torch.int32), torch.tensor([9], dtype=torch.int32)
    for match, call in (
            ("must be a KVCache", lambda: cache_write(x, x, x, cu, tab, kl)),
            ("at least one offset", lambda: cache_write(cache, x, x, cu[:0], tab, kl)),
            ("cu must be int32", lambda: cache_write(cache, x, x, cu.long(), tab, kl)),
            ("k_lens must be int32 \\[1\\]", lambda: cache_write(cache, x, x, cu, tab, cu)),
            ("table must be int32 \\[1, pages\\]", lambda: cache_write(cache, x, x, cu, tab[0], kl)),
            ("table must be int32 \\[1, pages\\]", lambda: cache_write(cache, x, x, cu, tab.long(), kl)),
            ("table must be int32 \\[1, pages\\]", lambda: cache_write(cache, x, x, cu, tab.expand(2, 4), kl)),
            ("at most", lambda: cache_write(cache, x, x, cu, tab[:, :1].expand(1, 1 << 27), kl)),
            ("bf16 or fp16", lambda: cache_write(cache, x.float(), x.float(), cu, tab, kl)),
            ("must be \\[tokens, 2, 64\\]", lambda: cache_write(cache, x, x[:4], cu, tab, kl)),
            ("must be \\[tokens, 2, 64\\]", lambda: cache_write(cache, x, x.half(), cu, tab, kl)),
            ("must be \\[tokens, 2, 64\\]", lambda: cache_write(cache, x[:, :1], x[:, :1], cu, tab, kl)),
            ("dtype must be", lambda: cache_read(cache, cu, tab, kl, 5, torch.float32)),
            ("tokens must not", lambda: cache_read(cache, cu, tab, kl, -1)),
            ("must be a KVCache", lambda: cache_read(None, cu, tab, kl, 5))):
        with pytest.raises(ValueError, match=match):
            call()
    for call in (lambda: cache_write(cache, x, x, cu, tab, kl), lambda: cache_read(cache, cu, tab, kl, 5)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_attention_arguments(cache):
    from embodied_efficiency_b200 import cache_attention
    q, cu = torch.zeros(5, 4, 64, dtype=BF), torch.tensor([0, 5], dtype=torch.int32)
    tab, kl, p = torch.zeros(1, 4, dtype=torch.int32), torch.tensor([9], dtype=torch.int32), torch.zeros(7, 2, 64, dtype=BF)
    many = torch.zeros(5, 258, 64, dtype=BF)
    for match, call in (
            ("must be a KVCache", lambda: cache_attention(q, p, cu, tab, kl)),
            ("cu_q must be int32", lambda: cache_attention(q, cache, cu.long(), tab, kl)),
            ("cu_q needs at least one", lambda: cache_attention(q, cache, cu[:0], tab, kl)),
            ("k_lens must be int32 \\[1\\]", lambda: cache_attention(q, cache, cu, tab, cu)),
            ("table must be int32", lambda: cache_attention(q, cache, cu, tab.float(), kl)),
            ("q must be bf16 or fp16", lambda: cache_attention(q.float(), cache, cu, tab, kl)),
            ("must be \\[tokens, heads, 64\\]", lambda: cache_attention(q[..., :32], cache, cu, tab, kl)),
            ("not a multiple of 2", lambda: cache_attention(q[:, :3], cache, cu, tab, kl)),
            ("scale must be", lambda: cache_attention(q, cache, cu, tab, kl, scale=-1.0)),
            ("scale must be", lambda: cache_attention(q, cache, cu, tab, kl, scale=float("nan"))),
            ("prefix k", lambda: cache_attention(q, cache, cu, tab, kl, prefix=(p, p[:6]))),
            ("prefix k", lambda: cache_attention(q, cache, cu, tab, kl, prefix=(p.half(), p.half()))),
            ("prefix k", lambda: cache_attention(q, cache, cu, tab, kl, prefix=(p[:, :1], p[:, :1]))),
            ("at most 128", lambda: cache_attention(many, cache, cu, tab, kl, prefix=(p, p)))):
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError, match="no CPU path"):
        cache_attention(q, cache, cu, tab, kl, prefix=(p, p))


def test_abi_codes(lib):
    from embodied_efficiency_b200 import _lib
    assert lib.ee_struct_size(4) == ctypes.sizeof(_lib.Cache)
    sec = (ctypes.c_int32 * 2)(16, 16)
    # ee_norm_rotary(q.., q_out.., k.., k_out.., q_weight, k_weight, weight_dtype, eps, pos, pos_axis, pos_bits, freqs,
    #                tokens, n_q, n_kv, head_dim, sections, n_axes, interleaved, act, stream)
    ro = [16, 256, 64, 16, 256, 64, 16, 128, 64, 16, 128, 64, 16, 16, _lib.EE_F32, 1e-6, 16, 5, 32, 16, 5, 4, 2, 64, sec,
          2, 0, _lib.EE_BF16, None]
    for i, v, rc in ((0, 0, 1), (9, 8, 3), (12, 0, 1), (13, 0, 1), (12, 8, 3), (13, 4, 3), (14, _lib.EE_F16, 4),
                     (14, 7, 4), (15, 0.0, 1), (15, float("nan"), 1), (15, float("inf"), 1), (16, 0, 1), (23, 96, 9),
                     (27, 2, 4)):
        assert lib.ee_norm_rotary(*(ro[:i] + [v] + ro[i + 1:])) == rc, (i, v)
    assert lib.ee_norm_rotary(*(ro[:20] + [0] + ro[21:])) == 0  # no tokens
    # ee_cache_write(cache, k, tok, head, v, tok, head, cu, table, table_row, width, k_lens, tokens, n_seq, act, stream)
    good = dict(k_codes=16, v_codes=16, k_steps=16, v_steps=16, pages=3, kv_heads=2, page_size=32, head_dim=64, bits=8)
    args = [16, 128, 64, 16, 128, 64, 16, 16, 4, 4, 16, 5, 1, _lib.EE_BF16, None]
    for fn in (lib.ee_cache_write, lib.ee_cache_read):
        for f, v, rc in (("bits", 16, 9), ("head_dim", 96, 9), ("page_size", 16, 9), ("page_size", 48, 9), ("pages", -1, 2),
                         ("kv_heads", 0, 2), ("pages", 1 << 26, 2), ("k_codes", 0, 1), ("v_steps", 0, 1),
                         ("v_codes", 24, 3), ("k_steps", 4, 3)):
            assert fn(ctypes.byref(_lib.Cache(**{**good, f: v})), *args) == rc, (f, v)
        c = ctypes.byref(_lib.Cache(**good))
        assert fn(None, *args) == 1
        for i, v, rc in ((0, 0, 1), (3, 0, 1), (6, 0, 1), (7, 0, 1), (10, 0, 1), (0, 8, 3), (1, 4, 3), (5, 12, 3),
                         (6, 2, 3), (7, 18, 3), (9, -1, 2), (9, 1 << 27, 2), (11, -1, 2), (11, 1 << 31, 2), (12, -1, 2),
                         (13, 2, 4)):
            assert fn(c, *(args[:i] + [v] + args[i + 1:])) == rc, (i, v)
        for i in (9, 11, 12):
            assert fn(c, *(args[:i] + [0] + args[i + 1:])) == 0  # nothing to do
    # ee_cache_attention(cache, q, tok, head, out, tok, head, cu_q, table, table_row, width, k_lens, prefix_k, tok, head,
    #                    prefix_v, tok, head, prefix_len, tq, n_seq, n_q, causal, scale, act, workspace, bytes, stream)
    ca = [16, 256, 64, 16, 256, 64, 16, 16, 4, 4, 16, 16, 128, 64, 16, 128, 64, 7, 5, 1, 4, 1, 0.125, _lib.EE_BF16, 0, 0,
          None]
    fn = lib.ee_cache_attention
    for f, v, rc in (("bits", 16, 9), ("head_dim", 96, 9), ("page_size", 16, 9), ("k_codes", 0, 1), ("v_codes", 24, 3)):
        assert fn(ctypes.byref(_lib.Cache(**{**good, f: v})), *ca) == rc, (f, v)
    assert fn(None, *ca) == 1
    for i, v, rc in ((0, 0, 1), (3, 0, 1), (6, 0, 1), (7, 0, 1), (10, 0, 1), (11, 0, 1), (14, 0, 1), (0, 8, 3), (3, 8, 3),
                     (1, 4, 3), (5, 12, 3), (6, 2, 3), (11, 8, 3), (13, 4, 3), (9, -1, 2), (17, -1, 2), (17, 1 << 31, 2),
                     (18, -1, 2), (18, 1 << 30, 2), (19, -1, 2), (20, 3, 2), (20, 0, 2), (20, 260, 9), (22, 0.0, 1),
                     (22, float("nan"), 1), (22, 3e38, 1), (23, 2, 4)):
        assert fn(c, *(ca[:i] + [v] + ca[i + 1:])) == rc, (i, v)
    for i in (18, 19):
        assert fn(c, *(ca[:i] + [0] + ca[i + 1:])) == 0
    need = lib.ee_cache_attention_workspace_bytes
    assert need(5, 1, 4, 2, 64, 8, 128, 0) > 0 and need(5, 1, 4, 2, 64, 8, 128, 100) > need(5, 1, 4, 2, 64, 8, 128, 0)
    for bad in ((0, 1, 4, 2, 64, 8, 128, 0), (5, 1, 3, 2, 64, 8, 128, 0), (5, 1, 4, 2, 96, 8, 128, 0),
                (5, 1, 4, 2, 64, 16, 128, 0), (1 << 30, 1, 4, 2, 64, 8, 128, 0), (5, 1, 4, 2, 64, 8, 128, -1),
                (5, 1, 4, 2, 64, 8, -1, 0)):
        assert need(*bad) == 0


def test_workspace_of_calls_that_are_refused(lib):
    """Heads that a call with a prefix does not take: no workspace, and no division by their tile's tokens."""
    need = lib.ee_cache_attention_workspace_bytes
    for n_q, n_kv in ((260, 2), (129, 1), (65535, 1)):
        for tq in (1, 5, 1000):
            for bits in (8, 4):
                assert need(tq, 1, n_q, n_kv, 64, bits, 128, 7) == 0
                assert need(tq, 1, n_q, n_kv, 64, bits, 128, 0) > 0
    assert need(5, 1, 256, 2, 64, 8, 128, 7) > 0
