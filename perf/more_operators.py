"""The operators of tokens that follow a cached prompt, as cases to measure: norms and rotation of query and key heads in
one pass, a paged cache of 8- or 4-bit keys and values (written, read back, attended over), and attention of a batch whose
sequences share a prefix.

``run`` computes a case in elementary torch operations (fp32, rounded once at the end), or, with ``own`` set, through
the framework's entry points. Sizes are those of the framework's experts and fleets (16 heads of 64 or 128, prefixes of
816 tokens, chunks of 50 tokens) or generic.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _norm(name, tokens, heads, kv_heads, head_dim, dtype, sections, **more):
    """sections: pairs of the time / height / width axis, as text ("16,24,24"); grid: side of each prompt's image."""
    return {"name": name, "op": "norm", "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "sections": sections, "interleaved": False, "grid": 16, "start": 0,
            **more}


def _cache(name, op, seqs, q_lo, q_hi, kv_heads, head_dim, dtype, bits, **more):
    """seqs sequences of q_lo..q_hi new tokens each, after past_lo..past_hi cached ones (and ``prefix`` shared ones)."""
    return {"name": name, "op": op, "seqs": seqs, "q_lo": q_lo, "q_hi": q_hi, "past_lo": 0, "past_hi": 0,
            "heads": kv_heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "bits": bits, "page": 64,
            "causal": True, "prefix": 0, "mix": 1, **more}


def listed():
    return [
        # one new token of each of 64 robots
        _norm("norm tokens", 64, 16, 4, 128, "bf16", "16,24,24", start=816),
        # a fleet's prompts, one axis, pairs side by side, far positions
        _norm("norm fleet", 65537, 16, 8, 64, "fp16", "32", interleaved=True, start=1000000),
        # the new token of each of 64 robots enters its cache
        _cache("write tokens", "write", 64, 1, 1, 4, 128, "bf16", 8, past_lo=1, past_hi=1632),
        # the prompts of a fleet (an image and a short text each) enter an empty cache
        _cache("write prompts", "write", 128, 257, 816, 16, 64, "bf16", 8),
        # a fleet's cached prompts, in 16 bits again
        _cache("read prompts", "read", 64, 257, 816, 16, 128, "bf16", 8),
        # one long conversation, from 4 bits
        _cache("read long", "read", 1, 32767, 32767, 4, 128, "fp16", 4),
        # one new token of each of 64 robots against its cached prompt
        _cache("attention tokens", "attention", 64, 1, 1, 4, 128, "bf16", 8, heads=16, past_lo=1, past_hi=1632),
        # two long conversations in 4 bits, one new token each
        _cache("attention long token", "attention", 2, 1, 1, 2, 64, "fp16", 4, heads=16, past_lo=30000, past_hi=32766),
        # action chunks of 64 robots against their prefixes, every token sees all
        _cache("attention chunks", "attention", 64, 50, 50, 16, 128, "bf16", 8, past_lo=257, past_hi=816,
               causal=False),
        # further turns of four conversations: many new tokens behind what is cached
        _cache("attention turns", "attention", 4, 500, 1024, 4, 128, "bf16", 8, heads=16, past_lo=1, past_hi=4096),
        # one new token of each of 64 robots with an instruction in common
        _cache("shared tokens", "attention", 64, 1, 1, 4, 128, "bf16", 8, heads=16, prefix=8192, past_lo=1, past_hi=816),
        # 128 action samples from one observation: chunks of 50 behind the prefix they share
        _cache("shared chunks", "attention", 128, 50, 50, 16, 128, "bf16", 8, prefix=816, causal=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "fp16"])
    hd = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8, 16])
    bits, page, mix = rng.choice([8, 8, 4]), rng.choice([32, 64, 128]), rng.randrange(1 << 30)
    op = rng.choice(["norm", "write", "read", "attention", "attention", "shared"])
    if op == "norm":
        heads = kv * rng.choice([g for g in (1, 2, 3, 4, 8) if g * kv <= 32])
        half = hd // 2
        a = rng.randrange(4, half - 8)
        b = rng.randrange(2, half - a)
        sections = rng.choice(["%d" % half, "%d,%d" % (a, half - a), "%d,%d,%d" % (a, b, half - a - b)])
        tokens = _log(rng, 1, 65537 * 24 * 64 // ((heads + kv) * hd))
        return _norm("", tokens, heads, kv, hd, dtype, sections, interleaved=rng.random() < 0.5,
                     grid=rng.choice([8, 14, 16]), start=_log(rng, 1, 1000000))
    if op in ("write", "read"):
        hi = _log(rng, 1, 32767)
        seqs = max(1, min(128, _log(rng, 1, 128), (1 << 26) // (hi * kv * hd)))
        past = _log(rng, 1, 2000) if op == "write" else 0
        return _cache("", op, seqs, rng.randrange(1, hi + 1), hi, kv, hd, dtype, bits, page=page, mix=mix,
                      past_lo=rng.randrange(past + 1), past_hi=past)
    group = rng.choice([g for g in (1, 2, 3, 4, 7, 8) if g * kv <= 32])
    prefix = _log(rng, 1, 8192) if op == "shared" else 0
    kind = rng.choice(["token", "token", "chunk", "turn"])
    q_hi = {"token": 1, "chunk": _log(rng, 2, 100), "turn": _log(rng, 100, 1024)}[kind]
    past = _log(rng, 1, 32766 if kind == "token" else 4096)
    seqs = max(1, min(64, _log(rng, 1, 64), (1 << 17) // past, (1 << 25) // (q_hi * kv * group * (past + prefix))))
    return _cache("", "attention", seqs, rng.randrange(1, q_hi + 1), q_hi, kv, hd, dtype, bits, heads=kv * group, page=page,
                  mix=mix, past_lo=rng.randrange(past), past_hi=past, prefix=prefix, causal=rng.random() < 0.7)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(case):
    """New tokens and keys of each sequence; a sequence's last key is its last new token."""
    rng = random.Random(case["mix"])
    n = case["seqs"]
    q = [rng.randint(case["q_lo"], case["q_hi"]) for _ in range(n)]
    past = [rng.randint(case["past_lo"], case["past_hi"]) for _ in range(n)]
    q[-1], past[0] = case["q_hi"], case["past_hi"]
    return q, [a + b for a, b in zip(q, past)]


def _sections(case):
    return tuple(int(s) for s in case["sections"].split(","))


def _pack(codes):
    """Two signed 4-bit codes a byte, the even one in the low half."""
    u = codes.to(torch.uint8) & 15
    return u[..., 0::2] | (u[..., 1::2] << 4)


def _unpack(packed):
    p = packed.to(torch.int16)
    return (((torch.stack([p & 15, p >> 4], -1).flatten(-2)) ^ 8) - 8).to(torch.int8)


def _quantize(x, bits):
    """Codes and fp32 scales of heads: x [..., hd]."""
    f = x.float()
    s = (f.abs().amax(-1, keepdim=True) / torch.full((), 2.0 ** (bits - 1) - 1, device=x.device)).clamp_min(1e-8)
    return torch.round(f / s).to(torch.int8), s[..., 0]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype, hd, kv = DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"]

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(to)

    if case["op"] == "norm":
        t = case["tokens"]
        i = torch.arange(t, device=dev, dtype=torch.int32) % 816  # prompts of 816 tokens: an image, then text
        side = case["grid"]
        image, text = i < side * side, i - side * side + side
        axes = [torch.where(image, v, text) + case["start"] for v in (torch.zeros_like(i), i // side, i % side)]
        return {"case": case, "q": normal(t, case["heads"], hd, scale=3.0), "k": normal(t, kv, hd, scale=2.0),
                "q_weight": (1 + normal(hd, scale=0.2)).to(dtype), "k_weight": (1 + normal(hd, scale=0.2)).to(dtype),
                "positions": torch.stack(axes[-len(_sections(case)):]).contiguous()}
    q_len, k_len = _lengths(case)
    page, bits = case["page"], case["bits"]
    need = [(n + page - 1) // page for n in k_len]
    # pages as a pool hands them out: in any order, some belonging to nobody, the table's unused places at -1
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=dev)[:sum(need)].to(torch.int32)
    width, counts = max(need), torch.tensor(need, device=dev)
    table = torch.full((case["seqs"], width), -1, device=dev, dtype=torch.int32)
    table[torch.arange(width, device=dev)[None] < counts[:, None]] = order
    st = {"case": case, "table": table, "longest_q": max(q_len), "longest_k": max(k_len), "rows": sum(q_len),
          "cu": torch.tensor([0] + q_len, device=dev).cumsum(0).to(torch.int32),
          "k_lens": torch.tensor(k_len, device=dev, dtype=torch.int32)}
    for n, size in (("k", 1.0), ("v", 0.7)):
        codes, scales = _quantize(normal(pages, kv, page, hd, scale=size), bits)
        st["cache_" + n], st["cache_" + n + "_scale"] = _pack(codes) if bits == 4 else codes, scales.contiguous()
    rows = sum(q_len)
    if case["op"] == "write":
        st["k"], st["v"] = normal(rows, kv, hd), normal(rows, kv, hd, scale=0.7)
    if case["op"] == "attention":
        st["q"] = normal(rows, case["heads"], hd, scale=1.5)
        if case["prefix"]:
            st["prefix_k"], st["prefix_v"] = normal(case["prefix"], kv, hd), normal(case["prefix"], kv, hd, scale=0.7)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _plain_norm(case, st):
    half = case["head_dim"] // 2
    pos, dev = st["positions"], st["q"].device
    axis = torch.repeat_interleave(torch.arange(pos.shape[0], device=dev), torch.tensor(_sections(case), device=dev),
                                   output_size=half)
    freq = 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
    angle = pos[axis].T.double() * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x, weight):
        f = x.float()
        f = f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + EPS) * weight.float()
        if case["interleaved"]:
            a, b = f[..., 0::2], f[..., 1::2]
            return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2).to(x.dtype)
        a, b = f[..., :half], f[..., half:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(x.dtype)

    return turn(st["q"], st["q_weight"]), turn(st["k"], st["k_weight"])


def _places(case, st):
    """Page and place in the page of each row: row i of a sequence's n is key k_len - n + i."""
    row = torch.arange(st["rows"], device=st["cu"].device, dtype=torch.int32)
    seq = torch.searchsorted(st["cu"][1:], row, right=True)
    key = (row - st["cu"][seq + 1] + st["k_lens"][seq]).long()
    return st["table"][seq, key // case["page"]].long(), key % case["page"]


def _values(case, st, n, page, place):
    """Keys or values of the cache in fp32."""
    codes = st["cache_" + n][page, :, place]
    if case["bits"] == 4:
        codes = _unpack(codes)
    return codes.float() * st["cache_" + n + "_scale"][page, :, place][..., None]


def _plain_write(case, st):
    page, place = _places(case, st)
    for n in ("k", "v"):
        codes, scales = _quantize(st[n], case["bits"])
        st["cache_" + n][page, :, place] = _pack(codes) if case["bits"] == 4 else codes
        st["cache_" + n + "_scale"][page, :, place] = scales
    if case["bits"] == 4:
        return _plain_read(case, st) + (st["cache_k_scale"], st["cache_v_scale"])
    return st["cache_k"], st["cache_v"], st["cache_k_scale"], st["cache_v_scale"]


def _plain_read(case, st):
    page, place = _places(case, st)
    return tuple(_values(case, st, n, page, place).to(DTYPES[case["dtype"]]) for n in ("k", "v"))


def _plain_attention(case, st):
    """Sequences padded to the longest one, whole rows of scores, a mask."""
    q, cu, nk = st["q"], st["cu"], st["k_lens"][:, None]
    dev, group = q.device, case["heads"] // case["kv_heads"]
    iq, ik = torch.arange(st["longest_q"], device=dev), torch.arange(st["longest_k"], device=dev)
    nq = (cu[1:] - cu[:-1])[:, None]
    qp = q[(cu[:-1, None] + iq).clamp(max=q.shape[0] - 1)].float()
    page = st["table"].long().clamp_min(0)[:, ik // case["page"]]
    place = (ik % case["page"]).expand_as(page)
    kp, vp = (_values(case, st, n, page, place) for n in ("k", "v"))
    b, lq = qp.shape[0], qp.shape[1]
    qp = qp.view(b, lq, -1, group, case["head_dim"]).permute(0, 2, 3, 1, 4)  # [b, kv, group, q, hd]
    kp, vp = kp.permute(0, 2, 3, 1)[:, :, None], vp.permute(0, 2, 1, 3)[:, :, None]
    s = (qp @ kp) * (1.0 / math.sqrt(case["head_dim"]))
    seen = (ik < nk)[:, None, :]
    if case["causal"]:
        seen = seen & (ik <= (iq + (nk - nq))[:, :, None])
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    if case["prefix"]:
        sp = (qp @ st["prefix_k"].float().permute(1, 2, 0)[:, None]) * (1.0 / math.sqrt(case["head_dim"]))
        top = torch.maximum(top, sp.amax(-1, keepdim=True))
    p = torch.exp(s - top)
    o, total = p @ vp, p.sum(-1, keepdim=True)
    if case["prefix"]:
        pp = torch.exp(sp - top)
        o = o + pp @ st["prefix_v"].float().permute(1, 0, 2)[:, None]
        total = total + pp.sum(-1, keepdim=True)
    o = (o / total).permute(0, 3, 1, 2, 4).reshape(b, lq, case["heads"], case["head_dim"])
    row = torch.arange(q.shape[0], device=dev, dtype=torch.int32)
    seq = torch.searchsorted(cu[1:], row, right=True)
    return o[seq, row - cu[seq]].to(q.dtype)


def run(state):
    case, st = state["case"], state
    if not own:
        return {"norm": _plain_norm, "write": _plain_write, "read": _plain_read,
                "attention": _plain_attention}[case["op"]](case, st)
    import embodied_efficiency_b200 as ee
    if case["op"] == "norm":
        return ee.norm_rotary_embed(st["q"], st["k"], st["q_weight"], st["k_weight"], st["positions"], _sections(case),
                                    eps=EPS, interleaved=case["interleaved"])
    cache = st.get("cache")
    if cache is None:  # the handle that a program keeps
        cache = st["cache"] = ee.KVCache(st["cache_k"], st["cache_v"], st["cache_k_scale"], st["cache_v_scale"])
    if case["op"] == "write":
        ee.cache_write(cache, st["k"], st["v"], st["cu"], st["table"], st["k_lens"])
        if case["bits"] == 4:
            return ee.cache_read(cache, st["cu"], st["table"], st["k_lens"], st["rows"], DTYPES[case["dtype"]]) + (
                st["cache_k_scale"], st["cache_v_scale"])
        return st["cache_k"], st["cache_v"], st["cache_k_scale"], st["cache_v_scale"]
    if case["op"] == "read":
        return ee.cache_read(cache, st["cu"], st["table"], st["k_lens"], st["rows"], DTYPES[case["dtype"]])
    prefix = (st["prefix_k"], st["prefix_v"]) if case["prefix"] else None
    return ee.cache_attention(st["q"], cache, st["cu"], st["table"], st["k_lens"], causal=case["causal"], prefix=prefix)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    hd, kv = case["head_dim"], case["kv_heads"]
    if case["op"] == "norm":
        values = case["tokens"] * (case["heads"] + kv) * hd
        return {"bytes": 4 * values + 4 * case["tokens"] * len(_sections(case)) + 4 * hd, "flops": 7 * values}
    q_len, k_len = _lengths(case)
    held = kv * (hd * case["bits"] // 8 + 4) * 2  # bytes of one cached token
    tables = 4 * (2 * case["seqs"] + 1 + sum((n + case["page"] - 1) // case["page"] for n in k_len))
    if case["op"] != "attention":
        rows = sum(q_len)
        values = 2 * rows * kv * hd
        back = 2 if case["op"] == "write" and case["bits"] == 4 else 1  # written and read back
        return {"bytes": back * (2 * values + rows * held) + tables, "flops": back * 3 * values}
    pairs = sum(a * (b - a) + a * (a + 1) // 2 if case["causal"] else a * b for a, b in zip(q_len, k_len))
    pairs += case["prefix"] * sum(q_len)
    return {"bytes": 4 * hd * case["heads"] * sum(q_len) + held * sum(k_len) + 4 * hd * kv * case["prefix"] + tables,
            "flops": 4 * hd * case["heads"] * pairs}


def exact(case, seed):
    """The definitions in 64 bits."""
    st = prepare(case, seed)
    if case["op"] == "norm":
        half = case["head_dim"] // 2
        turns, first = [], 0
        for axis, many in enumerate(_sections(case)):  # e^(i p f) for the pairs of each axis
            f = torch.exp(torch.arange(first, first + many, device="cuda", dtype=torch.float64) *
                          (-math.log(10000.0) / half))
            turns.append(torch.polar(torch.ones((), device="cuda", dtype=torch.float64).expand(case["tokens"], many),
                                     st["positions"][axis].double()[:, None] * f))
            first += many
        by = torch.cat(turns, 1)[:, None]
        res = []
        for n in ("q", "k"):
            x = st[n].double()
            x = st[n + "_weight"].double() * x / torch.sqrt(torch.einsum("thd,thd->th", x, x)[..., None] / (2 * half) + EPS)
            if case["interleaved"]:
                z = torch.view_as_complex(x.unflatten(-1, (half, 2)).contiguous()) * by
                res.append(torch.view_as_real(z).flatten(-2))
            else:
                z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * by
                res.append(torch.cat([z.real, z.imag], -1))
        return tuple(res)
    q_len, k_len = _lengths(case)
    page, hd, kv = case["page"], case["head_dim"], case["kv_heads"]
    table = st["table"].tolist()

    def held(n, b, lo, hi):
        """Keys or values lo..hi of sequence b: the codes times their steps."""
        at = torch.arange(lo, hi, device="cuda")
        pages = torch.tensor(table[b], device="cuda")[at // page]
        c = st["cache_" + n].transpose(1, 2)[pages, at % page]
        if case["bits"] == 4:
            low, high = c.to(torch.int32) % 16, c.to(torch.int32) // 16
            c = torch.stack([low, high], -1).reshape(hi - lo, kv, hd)
            c = torch.where(c > 7, c - 16, c)
        return c.double() * st["cache_" + n + "_scale"].transpose(1, 2)[pages, at % page].double()[..., None]

    if case["op"] == "read":
        return tuple(torch.cat([held(n, b, k - q, k) for b, (q, k) in enumerate(zip(q_len, k_len))]) for n in ("k", "v"))
    if case["op"] == "write":
        most = 2.0 ** (case["bits"] - 1) - 1
        scales, values = [], []
        for n in ("k", "v"):
            grid = st["cache_" + n + "_scale"].double()
            x = st[n].double()
            step = torch.clamp(x.abs().max(dim=-1).values / most, min=1e-8)
            first = 0
            for b, (q, k) in enumerate(zip(q_len, k_len)):
                at = torch.arange(k - q, k, device="cuda")
                grid.transpose(1, 2)[torch.tensor(table[b], device="cuda")[at // page], at % page] = step[first:first + q]
                first += q
            scales.append(grid)
            s32 = step.float()  # the step is an fp32 value, as the codes go by it
            values.append(torch.round(torch.div(st[n].float(), s32[..., None])).double() * s32.double()[..., None])
        return (*values, *scales) if case["bits"] == 4 else (None, None, *scales)
    if sum(a * (b + case["prefix"]) for a, b in zip(q_len, k_len)) * case["heads"] > 1 << 32:
        return None
    out, i, group = torch.empty(st["q"].shape, device="cuda", dtype=torch.float64), 0, case["heads"] // kv
    for b, (a, n) in enumerate(zip(q_len, k_len)):
        keys, vals = held("k", b, 0, n), held("v", b, 0, n)
        hidden = torch.arange(n, device="cuda")[None] - torch.arange(a, device="cuda")[:, None] > (
            n - a if case["causal"] else n)
        if case["prefix"]:
            keys, vals = torch.cat([st["prefix_k"].double(), keys]), torch.cat([st["prefix_v"].double(), vals])
            hidden = torch.cat([hidden.new_zeros(a, case["prefix"]), hidden], 1)
        qq = st["q"][i:i + a].double().unflatten(1, (kv, group)).permute(1, 2, 0, 3)
        s = torch.matmul(qq, keys.permute(1, 2, 0)[:, None]) / math.sqrt(hd)
        w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        out[i:i + a] = torch.matmul(w, vals.permute(1, 0, 2)[:, None]).permute(2, 0, 1, 3).flatten(1, 2)
        i += a
    return out
