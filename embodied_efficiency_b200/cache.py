"""A paged cache of quantised keys and values for tokens that follow a prompt, on the
sm_100a kernels of ``libee_b200.so``: written as tokens come, read back, attended over.

Tokens are packed as in ``prompt``: [tokens, heads, head_dim], sequences one behind another without padding, int32
offsets ``cu`` of their first rows. Where a sequence's keys lie says the int32 ``table`` [sequences, width] of page
numbers, how many it has ``k_lens`` [sequences]; both live on the device, so nothing here waits for the GPU and every
call can be captured into a CUDA graph. A call's tokens are the last ones of their sequences: the same ``cu``,
``table`` and ``k_lens`` (the lengths with the new tokens in them) write a step's keys and attend over them. The
operators compute forward only.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .prompt import _MAX_SCALE, _act_dtype, _heads, _offsets, _out

PAGE_SIZES = (32, 64, 128, 256)


class KVCache:
    """Pages of ``page_size`` tokens: codes ``k`` and ``v`` [pages, kv_heads, page_size, head_dim] int8, or
    [..., head_dim / 2] uint8 with two 4-bit codes a byte (as ``_pack_int4``), and steps ``k_scale`` and ``v_scale``
    [pages, kv_heads, page_size] fp32; a value is code * step. The tensors are the caller's and stay where they are;
    ``KVCache.empty`` makes them. head_dim 64 or 128, page_size 32, 64, 128 or 256. Which pages belong to whom is the
    caller's bookkeeping."""

    def __init__(self, k, v, k_scale, v_scale):
        if k.dim() != 4 or k.dtype not in (torch.int8, torch.uint8):
            raise ValueError(f"k must be int8 [pages, kv_heads, page_size, head_dim] or uint8 [.., head_dim / 2], got "
                             f"{k.dtype} {tuple(k.shape)}")
        pages, heads, size, hd = k.shape
        self.bits = 8 if k.dtype == torch.int8 else 4
        hd *= 8 // self.bits
        if hd not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {hd}")
        if size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {size}")
        if heads < 1 or heads > 65535 or pages * heads * size > 0x7fffffff:
            raise ValueError(f"{pages} pages of {size} tokens with {heads} heads: at least one head, below 2^31 rows")
        if v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError(f"v {v.dtype} {tuple(v.shape)} does not match k {k.dtype} {tuple(k.shape)}")
        for t, n in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if t.shape != k.shape[:3] or t.dtype != torch.float32:
                raise ValueError(f"{n} must be fp32 {tuple(k.shape[:3])}, got {t.dtype} {tuple(t.shape)}")
        for t, n in ((k, "k"), (v, "v"), (k_scale, "k_scale"), (v_scale, "v_scale")):
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{n} must be contiguous and on a 16-byte boundary")
            if t.requires_grad:
                raise ValueError(f"{n} must not ask for a gradient: the cache is written in place")
        self.device = _lib.same_device(k, v, k_scale, v_scale)
        self._tensors = (k, v, k_scale, v_scale)
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, size, hd
        self._c = _lib.Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, heads, size, hd,
                             self.bits, 0)
        self._at = ctypes.addressof(self._c)  # the native host side reads the record there

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scale = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])

    def __reduce__(self):  # a copy has memory of its own, and a record of it
        return KVCache, self._tensors

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, bits: int = 8, device="cuda"):
        """A cache of its own memory; what its pages hold before they are written is undefined."""
        if bits not in (8, 4):
            raise ValueError(f"bits must be 8 or 4, got {bits}")
        shape = (pages, kv_heads, page_size)
        codes = [torch.empty(*shape, head_dim * bits // 8, dtype=torch.int8 if bits == 8 else torch.uint8, device=device)
                 for _ in range(2)]
        return cls(*codes, *(torch.empty(shape, dtype=torch.float32, device=device) for _ in range(2)))

    def __repr__(self):
        return (f"KVCache({self.pages} pages of {self.page_size}, {self.kv_heads} heads of {self.head_dim}, "
                f"{self.bits} bits, {self.device})")


def _places(cache, cu, table, k_lens, name):
    """Checked offsets, table and lengths; the number of sequences."""
    if not isinstance(cache, KVCache):
        raise ValueError(f"cache must be a KVCache, got {type(cache).__name__}")
    n = cu.numel() - 1
    if n < 0:
        raise ValueError(f"{name} needs at least one offset")
    cu, k_lens = _offsets(cu, n + 1, name), _offsets(k_lens, n, "k_lens")
    if table.dim() != 2 or table.dtype != torch.int32 or table.shape[0] != n:
        raise ValueError(f"table must be int32 [{n}, pages], got {table.dtype} {tuple(table.shape)}")
    if table.shape[1] > 0x7fff0000 // cache.page_size:
        raise ValueError(f"table names {table.shape[1]} pages a sequence: at most {0x7fff0000 // cache.page_size}")
    if table.stride(1) != 1 and table.shape[1] > 1:
        table = table.contiguous()
    return cu, table, k_lens, n


def cache_write(cache: KVCache, k, v, cu, table, k_lens) -> None:
    """Quantise new tokens into the cache (``ee_cache_write``): rows ``cu[b]`` to ``cu[b + 1]`` of ``k`` and ``v``
    [tokens, kv_heads, head_dim] become the last keys of sequence b before ``k_lens[b]``. Per token and head the step is
    ``max(amax / 127, 1e-8)`` (4 bits: ``/ 7``) and a code ``round(x / step)``; a head with an infinity or NaN gets a
    NaN step. Rows whose key would lie before 0, past the table or on a page the cache does not have are left out. The
    places written in one call have to differ: one that two tokens claim is left with either's values or a mixture.
    bf16 / fp16."""
    if type(cache) is KVCache and (_lib._native or _lib.native()).cache_write(cache.k, cache._at, k, v, cu, table, k_lens):
        return
    cu, table, k_lens, n = _places(cache, cu, table, k_lens, "cu")
    _act_dtype(k, "k and v")
    if k.dim() != 3 or k.shape != v.shape or k.dtype != v.dtype or k.shape[1:] != (cache.kv_heads, cache.head_dim):
        raise ValueError(f"k {k.dtype} {tuple(k.shape)} and v {v.dtype} {tuple(v.shape)} must be [tokens, "
                         f"{cache.kv_heads}, {cache.head_dim}]")
    dev = _lib.same_device(cache.k, k, v, cu, table, k_lens)
    _lib.no_grad_through("cache_write", k, v)
    with _lib.on_device(dev):
        (k, ks), (v, vs) = _heads(k, "k"), _heads(v, "v")
        rc = _lib.load().ee_cache_write(ctypes.byref(cache._c), k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
                                        cu.data_ptr(), table.data_ptr(), table.stride(0), table.shape[1],
                                        k_lens.data_ptr(), k.shape[0], n, _lib.act_code(k.dtype), _lib.stream_ptr(dev))
    _lib.check(rc, "ee_cache_write")


def cache_read(cache: KVCache, cu, table, k_lens, tokens: int, dtype=torch.bfloat16, out=None):
    """The way back (``ee_cache_read``): rows ``cu[b]`` to ``cu[b + 1]`` of the results k and v [``tokens``, kv_heads,
    head_dim] (new, of ``dtype``, or ``out`` = (k, v)) are sequence b's last keys before ``k_lens[b]``, code * step
    rounded once. Rows that belong to no sequence, or whose key lies before 0, past the table or on a page the cache
    does not have, are not written."""
    if out is None and type(cache) is KVCache:
        done = (_lib._native or _lib.native()).cache_read(cache.k, cache._at, cu, table, k_lens, tokens, dtype)
        if done is not None:
            return done
    cu, table, k_lens, n = _places(cache, cu, table, k_lens, "cu")
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"dtype must be bf16 or fp16, not {dtype}")
    if tokens < 0:
        raise ValueError(f"tokens must not be negative, got {tokens}")
    dev = _lib.same_device(cache.k, cu, table, k_lens)
    like = torch.empty((tokens, cache.kv_heads, cache.head_dim), dtype=dtype, device="meta")
    with _lib.on_device(dev):
        if out is None:
            k, v = (torch.empty(like.shape, dtype=dtype, device=dev) for _ in range(2))
        else:
            k, v = out
            _lib.no_grad_through("cache_read", k, v)
            for t, name in ((k, "out for k"), (v, "out for v")):
                if t.shape != like.shape or t.dtype != dtype or t.device != dev:
                    raise ValueError(f"{name} must be {dtype} {tuple(like.shape)} on {dev}")
                _out(t, t, name)
        ks, vs = k.stride(), v.stride()
        rc = _lib.load().ee_cache_read(ctypes.byref(cache._c), k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
                                       cu.data_ptr(), table.data_ptr(), table.stride(0), table.shape[1],
                                       k_lens.data_ptr(), tokens, n, _lib.act_code(dtype), _lib.stream_ptr(dev))
    _lib.check(rc, "ee_cache_read")
    return k, v


def cache_attention(q, cache: KVCache, cu_q, table, k_lens, causal: bool = True, scale: float | None = None, prefix=None,
                    out=None):
    """Attention over the cache (``ee_cache_attention``): sequence b's queries, rows ``cu_q[b]`` to ``cu_q[b + 1]`` of
    ``q`` [tokens, heads, head_dim], against its first ``k_lens[b]`` keys (at most what its row of the table covers).
    ``prefix`` = (k, v) [P, kv_heads, head_dim] in q's type are keys and values before those that every sequence shares
    and every query sees: they are read once for the whole call. heads is a multiple of kv_heads: head h reads key head
    ``h // (heads // kv_heads)``; at most 128 heads a key head with a prefix. With ``causal`` a sequence's last query
    sees its last key; a query that sees no key gives zeros. ``scale`` defaults to head_dim^-0.5. Keys past a
    sequence's length, under the mask or on pages that the cache does not have count with weight 0, whatever is there.
    One kernel serves the whole call, chosen by the mean of queries per sequence and key head: a long turn among many
    single tokens is faster in a call of its own. Lengths that the table cuts count as cut, for the mask too. For their
    product with the values the weights keep 16 bits (up to 16 queries x heads a sequence and key head) or 11 (above; then
    a key that counts less than 2^-32 of the row's first may count as 0), over the prefix those of q's type. Returns
    [tokens, heads, head_dim], new or ``out`` (which shares no memory with the inputs); rows that belong to no sequence are
    not written. Sums are fp32, of weights up to 2^15 before they are divided: values beyond 2^100 can overflow in
    them, values below 2^-100 be lost.
    bf16 / fp16."""
    if out is None and type(cache) is KVCache:
        done = (_lib._native or _lib.native()).cache_attention(cache.k, cache._at, q, cu_q, table, k_lens, causal, scale,
                                                               prefix)
        if done is not None:
            return done
    cu_q, table, k_lens, n = _places(cache, cu_q, table, k_lens, "cu_q")
    hd, hk = cache.head_dim, cache.kv_heads
    _act_dtype(q, "q")
    if q.dim() != 3 or q.shape[2] != hd:
        raise ValueError(f"q {tuple(q.shape)} must be [tokens, heads, {hd}]")
    tq, hq = q.shape[:2]
    if hq < 1 or hq % hk:
        raise ValueError(f"{hq} heads are not a multiple of {hk} key heads")
    scale = hd ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -126 <= scale <= _MAX_SCALE:
        raise ValueError(f"scale must be finite and above 0 (fp32, 2^-126 to {_MAX_SCALE:.4g}), got {scale}")
    pk = pv = None
    if prefix is not None:
        pk, pv = prefix
        if pk.dim() != 3 or pk.shape != pv.shape or pk.dtype != q.dtype or pv.dtype != q.dtype or pk.shape[1:] != (hk, hd):
            raise ValueError(f"prefix k {pk.dtype} {tuple(pk.shape)} and v {pv.dtype} {tuple(pv.shape)} must be "
                             f"{q.dtype} [P, {hk}, {hd}]")
        if pk.shape[0] and hq // hk > 128:
            raise ValueError(f"{hq // hk} heads a key head: at most 128 with a prefix")
    dev = _lib.same_device(cache.k, q, pk, pv, cu_q, table, k_lens)
    _lib.no_grad_through("cache_attention", q, pk, pv)
    lib = _lib.load()
    with _lib.on_device(dev):
        (qc, qs), (out, os_) = _heads(q, "q"), _out(out, q, "out")
        p_len, pks, pvs = 0, (0, 0), (0, 0)
        if pk is not None and pk.shape[0]:
            (pk, pks), (pv, pvs), p_len = _heads(pk, "prefix k"), _heads(pv, "prefix v"), pk.shape[0]
        nb = lib.ee_cache_attention_workspace_bytes(tq, n, hq, hk, hd, cache.bits, table.shape[1] * cache.page_size, p_len)
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        rc = lib.ee_cache_attention(
            ctypes.byref(cache._c), qc.data_ptr(), qs[0], qs[1], out.data_ptr(), os_[0], os_[1], cu_q.data_ptr(),
            table.data_ptr(), table.stride(0), table.shape[1], k_lens.data_ptr(), _lib.ptr(pk), pks[0], pks[1],
            _lib.ptr(pv), pvs[0], pvs[1], p_len, tq, n, hq, 1 if causal else 0, scale, _lib.act_code(q.dtype),
            _lib.ptr(ws), nb, _lib.stream_ptr(dev))
    _lib.check(rc, "ee_cache_attention")
    return out
