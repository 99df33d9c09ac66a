"""Attention layers of packed prompts: rotary positions with several axes and
causal or full attention with grouped heads, on the sm_100a kernels of
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
import functools
import math

import torch

from . import _lib


def _heads(t, name):
    """Checks of a [tokens, heads, head_dim] operand; a copy where a stride or the base is not on 16 bytes."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got {tuple(t.shape)}")
    if t.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{name} must be bf16 or fp16, not {t.dtype}")
    s = t.stride()
    if s[2] != 1 or s[0] % 8 or s[1] % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _out(out, like, name):
    """An output to fill: ``out`` after checks, or a new contiguous tensor."""
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    s = out.stride()
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{name} must be {like.dtype} {tuple(like.shape)} on {like.device}")
    if out.dim() != 3 or s[2] != 1 or s[0] % 8 or s[1] % 8 or out.data_ptr() % 16:
        raise ValueError(f"{name} needs a contiguous last dimension, strides of 8 elements and a 16-byte boundary")
    return out


_TURNS: dict = {}


def _turns(device, half: int, base: float) -> torch.Tensor:
    """base^(-i / half) / 2 pi as 64-bit fractions of a turn (int64 bits), a constant table per device."""
    key = (device, half, base)
    tab = _TURNS.get(key)
    if tab is None:
        vals = [int(round(math.ldexp(base ** (-i / half) / (2.0 * math.pi), 64))) & (2 ** 64 - 1) for i in range(half)]
        host = torch.tensor([v - 2 ** 64 if v >= 2 ** 63 else v for v in vals], dtype=torch.int64)
        tab = _TURNS[key] = host.to(device)
    return tab


@functools.lru_cache(maxsize=64)
def _section_array(sections):
    return (ctypes.c_int32 * len(sections))(*sections)


def rotary_embed(q, k, positions, sections, base: float = 10000.0, interleaved: bool = False, out=None):
    """Rotary positions with up to four axes (``ee_rotary``) of ``q`` [T, heads, head_dim] and ``k``
    [T, kv_heads, head_dim] (either may be None): pair i of the head_dim / 2 pairs turns by
    ``positions[axis][t] * base^(-2i / head_dim)``, the first ``sections[0]`` pairs by axis 0, the next
    ``sections[1]`` by axis 1 and so on. Pairs are (i, i + head_dim / 2), or (2i, 2i + 1) when ``interleaved``.
    ``positions`` is int32 or int64 [axes, T] ([T] for one axis); angles stay exact to the last bits of fp32 at any
    position. Returns (q, k) turned, as new tensors or in ``out`` = (q_out, k_out), which may be the inputs
    themselves. head_dim 32, 64, 128 or 256; bf16 / fp16."""
    sections = tuple(int(s) for s in sections)
    pos = positions.unsqueeze(0) if positions.dim() == 1 else positions
    one = q if q is not None else k
    if one is None:
        raise ValueError("rotary_embed needs q or k")
    t, hd = one.shape[0], one.shape[-1]
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) != hd // 2:
        raise ValueError(f"sections {sections} must be one to four counts that sum to head_dim / 2 = {hd // 2}")
    if pos.dim() != 2 or tuple(pos.shape) != (len(sections), t):
        raise ValueError(f"positions have shape {tuple(positions.shape)}, expected {(len(sections), t)}")
    if pos.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, not {pos.dtype}")
    if hd not in (32, 64, 128, 256):
        raise ValueError(f"head_dim must be 32, 64, 128 or 256, got {hd}")
    if not base > 1.0 or math.isinf(base):
        raise ValueError(f"base must be finite and above 1, got {base}")
    if q is not None and k is not None and (k.shape[0] != t or k.shape[-1] != hd or k.dtype != q.dtype):
        raise ValueError(f"q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} do not belong together")
    dev = _lib.same_device(q, k, pos)
    _lib.no_grad_through("rotary_embed", q, k)
    with _lib.on_device(dev):
        qo, ko = out if out is not None else (None, None)
        args, res, keep = [], [], []
        for x, o, name in ((q, qo, "q"), (k, ko, "k")):
            if x is None:
                args += [0, 0, 0, 0, 0, 0]
                res.append(None)
                continue
            xs = _heads(x, name)
            o = _out(o, x, f"out for {name}")
            args += [xs.data_ptr(), xs.stride(0), xs.stride(1), o.data_ptr(), o.stride(0), o.stride(1)]
            res.append(o)
            keep.append(xs)
        if pos.stride(1) != 1:
            pos = pos.contiguous()
        _lib.check(_lib.load().ee_rotary(*args, pos.data_ptr(), pos.stride(0), 32 if pos.dtype == torch.int32 else 64,
                                         _turns(dev, hd // 2, float(base)).data_ptr(), t,
                                         0 if q is None else q.shape[1], 0 if k is None else k.shape[1], hd,
                                         _section_array(sections), len(sections), 1 if interleaved else 0,
                                         _lib.act_code(one.dtype), _lib.stream_ptr(dev)), "ee_rotary")
    return res[0], res[1]


def _offsets(t, n, name):
    if t.dim() != 1 or t.dtype != torch.int32 or t.numel() != n:
        raise ValueError(f"{name} must be int32 [{n}], got {t.dtype} {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def prompt_attention(q, k, v, cu_q, cu_k=None, k_lens=None, causal: bool = True, scale: float | None = None, out=None):
    """Attention over packed prompts (``ee_prompt_attention``): sequence b's queries, rows ``cu_q[b]`` to
    ``cu_q[b + 1]`` of ``q`` [Tq, heads, head_dim], against its keys, rows ``cu_k[b]`` to ``cu_k[b + 1]`` of ``k`` and
    ``v`` [Tk, kv_heads, head_dim] -- the first ``k_lens[b]`` of them when given (a cache with room to grow);
    ``cu_k`` None means the queries' own rows. heads is a multiple of kv_heads: head h reads key head
    ``h // (heads // kv_heads)``. With ``causal`` a sequence's last query sees its last key, so queries may be the new
    tokens (or the one new token) behind a cached prompt; a query that sees no key gives zeros. ``scale`` defaults to
    head_dim^-0.5. Offsets are int32 on the device, not decreasing; what they claim beyond the tensors is cut off.
    Returns [Tq, heads, head_dim], new or ``out``; rows that belong to no sequence are not written.
    head_dim 64 or 128; bf16 / fp16."""
    if k.shape != v.shape or q.dtype != k.dtype or q.dtype != v.dtype:
        raise ValueError(f"q {q.dtype}, k {k.dtype} {tuple(k.shape)} and v {v.dtype} {tuple(v.shape)} do not match")
    if q.dim() != 3 or k.dim() != 3 or q.shape[2] != k.shape[2]:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must be [tokens, heads, head_dim]")
    tq, hq, hd = q.shape
    tk, hk = k.shape[0], k.shape[1]
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
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be finite and above 0, got {scale}")
    cu_q = _offsets(cu_q, n + 1, "cu_q")
    cu_k = None if cu_k is None else _offsets(cu_k, n + 1, "cu_k")
    k_lens = None if k_lens is None else _offsets(k_lens, n, "k_lens")
    dev = _lib.same_device(q, k, v, cu_q, cu_k, k_lens)
    _lib.no_grad_through("prompt_attention", q, k, v)
    with _lib.on_device(dev):
        qs, ks, vs = _heads(q, "q"), _heads(k, "k"), _heads(v, "v")
        o = _out(out, q, "out")
        lib = _lib.load()
        nb = lib.ee_prompt_attention_workspace_bytes(tq, tk, n, hq, hk, hd)
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        _lib.check(lib.ee_prompt_attention(
            qs.data_ptr(), qs.stride(0), qs.stride(1), ks.data_ptr(), ks.stride(0), ks.stride(1), vs.data_ptr(),
            vs.stride(0), vs.stride(1), o.data_ptr(), o.stride(0), o.stride(1), cu_q.data_ptr(), _lib.ptr(cu_k),
            _lib.ptr(k_lens), tq, tk, n, hq, hk, hd, 1 if causal else 0, scale, _lib.act_code(q.dtype), _lib.ptr(ws),
            nb, _lib.stream_ptr(dev)), "ee_prompt_attention")
    return o
