"""Attention layers of packed prompts: rotary positions with several axes (alone or
behind a norm of each head) and causal or full attention with grouped heads, on the sm_100a kernels of
``libee_b200.so``.

A prompt's queries, keys and values are rows of token-major tensors
[tokens, heads, head_dim] (views into a fused projection will do), prompts of
different lengths one behind another without padding; ``cu`` tensors hold the
int32 offsets of their first rows on the device, so nothing here waits for the
GPU and every call can be captured into a CUDA graph. The operators compute
forward only.
"""
from __future__ import annotations

import ctypes
import decimal
import functools
import math

import torch

from . import _lib


def _heads(t, name):
    """A [tokens, heads, head_dim] operand and its strides; a copy where a stride or the base is not on 16 bytes."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got {tuple(t.shape)}")
    s = t.stride()
    if s[2] != 1 or s[0] % 8 or s[1] % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        s = t.stride()
    return t, s


def _out(out, like, name):
    """An output to fill and its strides: ``out`` after checks, or a new contiguous tensor."""
    if out is None:
        out = torch.empty_like(like) if like.is_contiguous() else like.new_empty(like.shape)
        return out, out.stride()
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{name} must be {like.dtype} {tuple(like.shape)} on {like.device}")
    s = out.stride()
    if s[2] != 1 or s[0] % 8 or s[1] % 8 or out.data_ptr() % 16:
        raise ValueError(f"{name} needs a contiguous last dimension, strides of 8 elements and a 16-byte boundary")
    reach = out.shape[2]  # elements that the dimensions of smaller strides cover
    for stride, size in sorted(zip(s[:2], out.shape[:2])):
        if size > 1 and out.numel():
            if stride < reach:
                raise ValueError(f"elements of {name} overlap in memory (strides {s}): it cannot be written")
            reach += stride * (size - 1)
    return out, s


def _vector(t):
    """A contiguous vector on a 16-byte boundary; a copy where it is not."""
    if t is not None and (t.stride(0) != 1 or t.data_ptr() % 16):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _act_dtype(t, name):
    if t.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{name} must be bf16 or fp16, not {t.dtype}")


_TURNS: dict = {}
_PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def _turn_fractions(half: int, base: float) -> list:
    """round(base^(-i / half) / 2 pi * 2^64) for i < half. In 50 digits: in double, whose 53 bits end 11 short of the
    table's, a position of 2^40 would turn 2^-15 of a turn too far."""
    with decimal.localcontext(decimal.Context(prec=50)):  # of its own: a caller's may trap inexact results
        log, scale = decimal.Decimal(float(base)).ln(), decimal.Decimal(2 ** 64) / (2 * _PI)
        return [int((scale * (log * -i / half).exp()).to_integral_value()) for i in range(half)]


def _turns(device, half: int, base: float, name: str = "rotary_embed") -> torch.Tensor:
    """``_turn_fractions`` as int64 bits, a constant table per device."""
    key = (device, half, base)
    tab = _TURNS.get(key)
    if tab is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{name} copies its frequencies (head_dim {2 * half}, base {base}) to the device on "
                               "first use: call it once before the stream capture")
        host = torch.tensor(_turn_fractions(half, base), dtype=torch.int64)  # at most 2^64 / 2 pi < 2^63
        tab = _TURNS[key] = host.to(device)
    return tab


@functools.lru_cache(maxsize=64)
def _sections(sections, half: int):
    """The axes' pair counts as the ABI takes them, after checks."""
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) != half:
        raise ValueError(f"sections {sections} must be one to four counts that sum to head_dim / 2 = {half}")
    return (ctypes.c_int32 * len(sections))(*sections)


def rotary_embed(q, k, positions, sections, base: float = 10000.0, interleaved: bool = False, out=None):
    """Rotary positions with up to four axes (``ee_rotary``) of ``q`` [T, heads, head_dim] and ``k``
    [T, kv_heads, head_dim] (either may be None): pair i of the head_dim / 2 pairs turns by
    ``positions[axis][t] * base^(-2i / head_dim)``, the first ``sections[0]`` pairs by axis 0, the next
    ``sections[1]`` by axis 1 and so on. Pairs are (i, i + head_dim / 2), or (2i, 2i + 1) when ``interleaved``.
    ``positions`` is int32 or int64 [axes, T] ([T] for one axis); an angle is off by less than 2^-22 (fp32's rounding of
    angle, sine and cosine) and ``|position| * 2^-62``: as much again only from 2^40 on. Returns (q, k) turned, as new
    tensors or in ``out`` = (q_out, k_out), which may be the inputs themselves but not overlap them, or one another, in
    any other way. head_dim 32, 64, 128 or 256; bf16 / fp16. The first call for a head_dim and base on a device copies
    a small table to it and has to come before a stream capture."""
    if out is None and q is not None and k is not None:
        tab = _TURNS.get((q.device, q.shape[-1] // 2, base))
        if tab is not None:
            done = (_lib._native or _lib.native()).rotary_embed(q, k, positions, sections, tab, interleaved)
            if done is not None:
                return done
    return _rotary("rotary_embed", q, k, positions, sections, base, interleaved, out)


def norm_rotary_embed(q, k, q_weight, k_weight, positions, sections, eps: float = 1e-6, base: float = 10000.0,
                      interleaved: bool = False, out=None):
    """``rotary_embed`` of heads that are normalised first, in one pass (``ee_norm_rotary``): every head x of ``q``
    becomes ``q_weight * x / sqrt(mean(x^2) + eps)`` before it turns, every head of ``k`` the same with ``k_weight``
    ([head_dim], fp32 or of the heads' type, both the same; None for heads that are None). Squares and sums in fp32, one
    rounding at the end. ``eps`` at least 2^-126. Everything else as for ``rotary_embed``."""
    if out is None and q is not None and k is not None:
        tab = _TURNS.get((q.device, q.shape[-1] // 2, base))
        if tab is not None:
            done = (_lib._native or _lib.native()).norm_rotary_embed(q, k, q_weight, k_weight, positions, sections, tab,
                                                                     interleaved, eps)
            if done is not None:
                return done
    return _rotary("norm_rotary_embed", q, k, positions, sections, base, interleaved, out, (q_weight, k_weight, eps))


def _norm_weight(w, x, name):
    if w is None or w.dim() != 1 or w.numel() != x.shape[-1]:
        raise ValueError(f"{name} must be [{x.shape[-1]}], got {None if w is None else tuple(w.shape)}")
    if w.dtype not in (torch.float32, x.dtype):
        raise ValueError(f"{name} must be fp32 or {x.dtype}, not {w.dtype}")


def _rotary(name, q, k, positions, sections, base, interleaved, out, norm=None):
    one = q if q is not None else k
    if one is None:
        raise ValueError(f"{name} needs q or k")
    t, hd = one.shape[0], one.shape[-1]
    if type(sections) is not tuple:
        sections = tuple(sections)
    sec = _sections(sections, hd // 2)
    pshape = positions.shape if positions.dim() != 1 else (1, positions.shape[0])
    if len(pshape) != 2 or pshape[0] != len(sections) or pshape[1] != t:
        raise ValueError(f"positions have shape {tuple(positions.shape)}, expected {(len(sections), t)}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, not {positions.dtype}")
    if hd not in (32, 64, 128, 256):
        raise ValueError(f"head_dim must be 32, 64, 128 or 256, got {hd}")
    if not 1.0 < base < math.inf:
        raise ValueError(f"base must be finite and above 1, got {base}")
    _act_dtype(one, "q and k")
    if q is not None and k is not None and (k.shape[0] != t or k.shape[-1] != hd or k.dtype != q.dtype):
        raise ValueError(f"q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} do not belong together")
    if norm is not None:
        qw, kw, eps = norm
        qw, kw = (None if q is None else qw), (None if k is None else kw)
        for w, x, n in ((qw, q, "q_weight"), (kw, k, "k_weight")):
            if x is not None:
                _norm_weight(w, x, n)
        if qw is not None and kw is not None and qw.dtype != kw.dtype:
            raise ValueError(f"q_weight is {qw.dtype}, k_weight {kw.dtype}")
        if not 2.0 ** -126 <= eps <= 3.4e38:
            raise ValueError(f"eps must be finite and at least 2^-126, got {eps}")
    else:
        qw = kw = None
    dev = _lib.same_device(q, k, positions, qw, kw)
    _lib.no_grad_through(name, q, k, qw, kw)
    qo, ko = out if out is not None else (None, None)
    qs = ks = qp = kp = qop = kop = nq = nk = 0
    none = (0, 0)
    with _lib.on_device(dev):
        if q is not None:
            (q, qs), (qo, qos), nq = _heads(q, "q"), _out(qo, q, "out for q"), q.shape[1]
            qp, qop = q.data_ptr(), qo.data_ptr()
        else:
            qo, qs, qos = None, none, none
        if k is not None:
            (k, ks), (ko, kos), nk = _heads(k, "k"), _out(ko, k, "out for k"), k.shape[1]
            kp, kop = k.data_ptr(), ko.data_ptr()
        else:
            ko, ks, kos = None, none, none
        if positions.stride(-1) != 1:
            positions = positions.contiguous()
        heads = (qp, qs[0], qs[1], qop, qos[0], qos[1], kp, ks[0], ks[1], kop, kos[0], kos[1])
        rest = (positions.data_ptr(), positions.stride(0) if positions.dim() == 2 else t,
                32 if positions.dtype == torch.int32 else 64, _turns(dev, hd // 2, base, name).data_ptr(), t, nq, nk, hd,
                sec, len(sections), 1 if interleaved else 0, _lib.act_code(one.dtype), _lib.stream_ptr(dev))
        if norm is None:
            rc = _lib.load().ee_rotary(*heads, *rest)
        else:
            qw, kw = _vector(qw), _vector(kw)
            code = _lib.EE_F32 if (kw if qw is None else qw).dtype == torch.float32 else _lib.act_code(one.dtype)
            rc = _lib.load().ee_norm_rotary(*heads, _lib.ptr(qw), _lib.ptr(kw), code, eps, *rest)
    _lib.check(rc, "ee_rotary" if norm is None else "ee_norm_rotary")
    return qo, ko


def _offsets(t, n, name):
    if t.dim() != 1 or t.dtype != torch.int32 or t.numel() != n:
        raise ValueError(f"{name} must be int32 [{n}], got {t.dtype} {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


_MAX_SCALE = 2.0 ** 128 / 1.4427  # scale * log2(e) is an fp32 value


def prompt_attention(q, k, v, cu_q, cu_k=None, k_lens=None, causal: bool = True, scale: float | None = None, out=None):
    """Attention over packed prompts (``ee_prompt_attention``): sequence b's queries, rows ``cu_q[b]`` to
    ``cu_q[b + 1]`` of ``q`` [Tq, heads, head_dim], against its keys, rows ``cu_k[b]`` to ``cu_k[b + 1]`` of ``k`` and
    ``v`` [Tk, kv_heads, head_dim] -- the first ``k_lens[b]`` of them when given (a cache with room to grow);
    ``cu_k`` None means the queries' own rows. heads is a multiple of kv_heads: head h reads key head
    ``h // (heads // kv_heads)``. With ``causal`` a sequence's last query sees its last key, so queries may be the new
    tokens (or the one new token) behind a cached prompt; a query that sees no key gives zeros. ``scale`` defaults to
    head_dim^-0.5. Offsets are int32 on the device, not decreasing; what they claim beyond the tensors is cut off.
    A masked key counts with weight 0, so ``k`` may hold anything there, while ``v`` has to be finite on the keys of a
    sequence (0 * inf is NaN); beyond them, nothing is used.
    One kernel serves the whole call, chosen by the mean of queries per sequence and key head: long prompts are faster
    in a call of their own than beside many single tokens.
    Returns [Tq, heads, head_dim], new or ``out`` (which shares no memory with the inputs); rows that belong to no sequence are not written.
    head_dim 64 or 128; bf16 / fp16."""
    if out is None:
        done = (_lib._native or _lib.native()).prompt_attention(q, k, v, cu_q, cu_k, k_lens, causal, scale)
        if done is not None:
            return done
    if k.shape != v.shape or q.dtype != k.dtype or q.dtype != v.dtype:
        raise ValueError(f"q {q.dtype}, k {k.dtype} {tuple(k.shape)} and v {v.dtype} {tuple(v.shape)} do not match")
    if q.dim() != 3 or k.dim() != 3 or q.shape[2] != k.shape[2]:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must be [tokens, heads, head_dim]")
    _act_dtype(q, "q, k and v")
    tq, hq, hd = q.shape
    tk, hk, _ = k.shape
    if hd not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {hd}")
    if hk < 1 or hq < 1 or hq % hk:
        raise ValueError(f"{hq} heads are not a multiple of {hk} key heads")
    n = cu_q.numel() - 1
    if n < 0:
        raise ValueError("cu_q needs at least one offset")
    if cu_k is None and tk != tq:
        raise ValueError(f"{tk} keys for {tq} queries need offsets of their own (cu_k)")
    scale = hd ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -126 <= scale <= _MAX_SCALE:
        raise ValueError(f"scale must be finite and above 0 (fp32, 2^-126 to {_MAX_SCALE:.4g}), got {scale}")
    cu_q = _offsets(cu_q, n + 1, "cu_q")
    cu_k = None if cu_k is None else _offsets(cu_k, n + 1, "cu_k")
    k_lens = None if k_lens is None else _offsets(k_lens, n, "k_lens")
    dev = _lib.same_device(q, k, v, cu_q, cu_k, k_lens)
    _lib.no_grad_through("prompt_attention", q, k, v)
    lib = _lib.load()
    with _lib.on_device(dev):
        (qc, qs), (k, ks), (v, vs), (out, os_) = _heads(q, "q"), _heads(k, "k"), _heads(v, "v"), _out(out, q, "out")
        nb = lib.ee_prompt_attention_workspace_bytes(tq, tk, n, hq, hk, hd)
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        rc = lib.ee_prompt_attention(
            qc.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], out.data_ptr(),
            os_[0], os_[1], cu_q.data_ptr(), _lib.ptr(cu_k), _lib.ptr(k_lens), tq, tk, n, hq, hk, hd,
            1 if causal else 0, scale, _lib.act_code(q.dtype), _lib.ptr(ws), nb, _lib.stream_ptr(dev))
    _lib.check(rc, "ee_prompt_attention")
    return out
