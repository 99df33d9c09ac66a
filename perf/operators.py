"""The operators of a prompt's transformer layers, as cases to measure: 8-bit integer linears with a scale for each
token and each output channel, rotary positions with several axes, and attention over packed prompts.

``run`` computes a case in elementary torch operations (fp32, rounded once at the end), or, with ``own`` set, through
the framework's entry points. Sizes are those of the framework's experts and fleets (width 1024 and 2048, 16 heads of
64 or 128, prefixes of 256 and 816 tokens, chunks of 50 tokens) or generic.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _linear(name, m, n, k, dtype, **more):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "bias": True, "gelu": False,
            "residual": False, "quantized": False, **more}


def _rotary(name, tokens, heads, kv_heads, head_dim, dtype, sections, **more):
    """sections: pairs of the time / height / width axis, as text ("16,24,24"); grid: side of each prompt's image."""
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "sections": sections, "interleaved": False, "grid": 16, "start": 0,
            **more}


def _attention(name, seqs, q_lo, q_hi, heads, kv_heads, head_dim, dtype, **more):
    """seqs sequences of q_lo..q_hi new tokens each, after past_lo..past_hi cached ones."""
    return {"name": name, "op": "attention", "seqs": seqs, "q_lo": q_lo, "q_hi": q_hi, "past_lo": 0, "past_hi": 0,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "causal": True, "mix": 1,
            **more}


def listed():
    return [
        # one token through the up-projection of the Pi0-scale MLP: latency and weight bytes
        _linear("linear token", 1, 8192, 2048, "bf16", gelu=True),
        # an action chunk (50 tokens) through its down-projection with the residual stream
        _linear("linear chunk", 50, 2048, 8192, "fp16", residual=True),
        # a few prompts of odd total length, activations quantised once for several products; odd width
        _linear("product ragged", 1023, 1000, 1040, "bf16", quantized=True, bias=False),
        # the prefix K/V projection of eight requests of 816 tokens
        _linear("linear prefix", 6528, 4096, 2048, "bf16"),
        # the up-projection over the prefixes of 64 requests
        _linear("linear fleet", 52224, 8192, 2048, "bf16", gelu=True),
        # one new token of each of 64 robots
        _rotary("rotary tokens", 64, 16, 4, 128, "bf16", "16,24,24", start=816),
        # eight prompts of 816 tokens (an image, then text), all heads with keys of their own
        _rotary("rotary prompts", 6528, 16, 16, 128, "bf16", "16,24,24"),
        # a fleet's prompts, one axis, pairs side by side, far positions
        _rotary("rotary fleet", 65537, 16, 8, 64, "fp16", "32", interleaved=True, start=1000000),
        # one new token of each of 64 robots against its cached prompt
        _attention("attention tokens", 64, 1, 1, 16, 4, 128, "bf16", past_lo=1, past_hi=1632),
        # two long conversations, one new token each
        _attention("attention long token", 2, 1, 1, 16, 2, 64, "fp16", past_lo=30000, past_hi=32767),
        # prompts of a fleet (an image and a short text each), every token sees its whole prompt
        _attention("attention prompts", 128, 257, 816, 16, 16, 64, "fp16", causal=False),
        # one long prompt with grouped heads
        _attention("attention long", 1, 8192, 8192, 16, 4, 128, "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "fp16"])
    op = rng.choice(["linear", "linear", "rotary", "attention", "attention"])
    if op == "linear":
        m, n, k = _log(rng, 1, 52224), _log(rng, 64, 8192), 16 * _log(rng, 8, 512)
        while m * n * k > 52224 * 8192 * 2048:
            m = max(1, m // 2)
        tail = rng.choice(["none", "gelu", "residual"])
        return _linear("", m, n, k, dtype, bias=rng.random() < 0.7, gelu=tail == "gelu", residual=tail == "residual",
                       quantized=rng.random() < 0.3)
    if op == "rotary":
        hd = rng.choice([64, 128])
        kv = rng.choice([1, 2, 4, 8, 16])
        heads = kv * rng.choice([g for g in (1, 2, 3, 4, 8) if g * kv <= 32])
        half = hd // 2
        a = rng.randrange(4, half - 8)
        b = rng.randrange(2, half - a)
        sections = rng.choice(["%d" % half, "%d,%d" % (a, half - a), "%d,%d,%d" % (a, b, half - a - b)])
        tokens = _log(rng, 1, 65537 * 24 * 64 // ((heads + kv) * hd))
        return _rotary("", tokens, heads, kv, hd, dtype, sections, interleaved=rng.random() < 0.5,
                       grid=rng.choice([8, 14, 16]), start=_log(rng, 1, 1000000))
    hd = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8, 16])
    heads = kv * rng.choice([g for g in (1, 2, 3, 4, 7, 8) if g * kv <= 28])
    mix = rng.randrange(1 << 30)
    kind = rng.choice(["token", "chunk", "prompts", "prompts"])
    if kind == "prompts":
        hi = _log(rng, 2, 6000)
        seqs = max(1, min(128, _log(rng, 1, 40000) // hi, (1 << 26) // (hi * hi)))
        return _attention("", seqs, rng.randrange(1, hi + 1), hi, heads, kv, hd, dtype, mix=mix,
                          causal=rng.random() < 0.6)
    q_hi = 1 if kind == "token" else _log(rng, 2, 100)
    past = _log(rng, 1, 32767)
    seqs = max(1, min(64, _log(rng, 1, 64), (1 << 17) // past))
    return _attention("", seqs, 1, q_hi, heads, kv, hd, dtype, past_lo=rng.randrange(past), past_hi=past, mix=mix,
                      causal=rng.random() < 0.8)


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


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(to)

    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x = normal(m, k)
        x[:, :: 97] *= 6.0  # the few large channels that activations have
        st = {"weight": torch.randint(-127, 128, (n, k), generator=g, device=dev, dtype=torch.int8),
              "scales": (torch.rand(n, generator=g, device=dev) + 0.5) * (0.02 / 64),
              "bias": normal(n, scale=0.1) if case["bias"] else None,
              "residual": normal(m, n) if case["residual"] else None}
        if case["quantized"]:
            xf = x.float()
            s = xf.abs().amax(-1, keepdim=True) / 127
            st["xq"], st["x_scale"] = torch.round(xf / s).clamp(-127, 127).to(torch.int8), s
        else:
            st["x"] = x
    elif case["op"] == "rotary":
        t, hd = case["tokens"], case["head_dim"]
        i = torch.arange(t, device=dev, dtype=torch.int32) % 816  # prompts of 816 tokens: an image, then text
        side = case["grid"]
        image, text = i < side * side, i - side * side + side
        axes = [torch.where(image, v, text) + case["start"] for v in (torch.zeros_like(i), i // side, i % side)]
        st = {"q": normal(t, case["heads"], hd), "k": normal(t, case["kv_heads"], hd),
              "positions": torch.stack(axes[-len(_sections(case)):]).contiguous()}
    else:
        q_len, k_len = _lengths(case)
        tq, tk, hd = sum(q_len), sum(k_len), case["head_dim"]
        st = {"q": normal(tq, case["heads"], hd, scale=1.5), "k": normal(tk, case["kv_heads"], hd),
              "v": normal(tk, case["kv_heads"], hd), "longest_q": max(q_len), "longest_k": max(k_len),
              "cu_q": torch.tensor([0] + q_len, device=dev).cumsum(0).to(torch.int32),
              "cu_k": torch.tensor([0] + k_len, device=dev).cumsum(0).to(torch.int32)}
    return {"case": case, **st}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _plain_linear(case, st):
    if case["quantized"]:
        q, s, dtype = st["xq"].float(), st["x_scale"], DTYPES[case["dtype"]]
    else:
        x, dtype = st["x"].float(), st["x"].dtype
        s = (x.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device=x.device)).clamp_min(1e-8)
        q = torch.round(x / s)
    y = (q @ st["weight"].float().T) * s * st["scales"]
    if st["bias"] is not None:
        y = y + st["bias"].float()
    if case["gelu"]:
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return y.to(dtype)


def _plain_rotary(case, st):
    half = case["head_dim"] // 2
    pos, dev = st["positions"], st["q"].device
    axis = torch.repeat_interleave(torch.arange(pos.shape[0], device=dev), torch.tensor(_sections(case), device=dev),
                                   output_size=half)
    freq = 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
    angle = pos[axis].T.double() * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x):
        f = x.float()
        if case["interleaved"]:
            a, b = f[..., 0::2], f[..., 1::2]
            return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2).to(x.dtype)
        a, b = f[..., :half], f[..., half:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(x.dtype)

    return turn(st["q"]), turn(st["k"])


def _plain_attention(case, st):
    """Sequences padded to the longest one, whole rows of scores, a mask."""
    q, k, v, cu_q, cu_k = (st[n] for n in ("q", "k", "v", "cu_q", "cu_k"))
    dev, group = q.device, case["heads"] // case["kv_heads"]
    iq, ik = torch.arange(st["longest_q"], device=dev), torch.arange(st["longest_k"], device=dev)
    nq, nk = (cu_q[1:] - cu_q[:-1])[:, None], (cu_k[1:] - cu_k[:-1])[:, None]
    at_q, at_k = (cu_q[:-1, None] + iq).clamp(max=q.shape[0] - 1), (cu_k[:-1, None] + ik).clamp(max=k.shape[0] - 1)
    qp, kp, vp = q[at_q].float(), k[at_k].float(), v[at_k].float()
    b, lq, lk = qp.shape[0], qp.shape[1], kp.shape[1]
    qp = qp.view(b, lq, -1, group, case["head_dim"]).permute(0, 2, 3, 1, 4)  # [b, kv, group, q, hd]
    kp, vp = kp.permute(0, 2, 3, 1)[:, :, None], vp.permute(0, 2, 1, 3)[:, :, None]
    s = (qp @ kp) * (1.0 / math.sqrt(case["head_dim"]))
    seen = (ik < nk)[:, None, :]
    if case["causal"]:
        seen = seen & (ik <= (iq + (nk - nq))[:, :, None])
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = (p @ vp) / p.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, lq, case["heads"], case["head_dim"])
    row = torch.arange(q.shape[0], device=dev, dtype=torch.int32)
    seq = torch.searchsorted(cu_q[1:], row, right=True)
    return o[seq, row - cu_q[seq]].to(q.dtype)


def run(state):
    case, st = state["case"], state
    if not own:
        return {"linear": _plain_linear, "rotary": _plain_rotary, "attention": _plain_attention}[case["op"]](case, st)
    import embodied_efficiency_b200 as ee
    if case["op"] == "linear":
        if case["quantized"]:
            return ee.int8_matmul(st["xq"], st["x_scale"], st["weight"], st["scales"], st["bias"],
                                  dtype=DTYPES[case["dtype"]], gelu=case["gelu"], residual=st["residual"])
        return ee.int8_linear(st["x"], st["weight"], st["scales"], st["bias"], gelu=case["gelu"],
                              residual=st["residual"])
    if case["op"] == "rotary":
        return ee.rotary_embed(st["q"], st["k"], st["positions"], _sections(case), interleaved=case["interleaved"])
    return ee.prompt_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], causal=case["causal"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        acts = m * k * (1 if case["quantized"] else 2) + (4 * m if case["quantized"] else 0)
        ends = m * n * 2 * (2 if case["residual"] else 1) + (2 * n if case["bias"] else 0)
        return {"bytes": acts + n * k + 4 * n + ends, "flops": 2 * m * n * k}
    if case["op"] == "rotary":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        return {"bytes": 4 * values + 4 * case["tokens"] * len(_sections(case)), "flops": 3 * values}
    q_len, k_len = _lengths(case)
    pairs = sum(a * (b - a) + a * (a + 1) // 2 if case["causal"] else a * b for a, b in zip(q_len, k_len))
    hd, heads, kv = case["head_dim"], case["heads"], case["kv_heads"]
    return {"bytes": 2 * hd * (2 * heads * sum(q_len) + 2 * kv * sum(k_len)) + 8 * (case["seqs"] + 1),
            "flops": 4 * hd * heads * pairs}


def exact(case, seed):
    """The definitions in 64 bits."""
    st = prepare(case, seed)
    if case["op"] == "linear":
        if case["quantized"]:
            codes, step = st["xq"].double(), st["x_scale"].double()
        else:
            step = torch.clamp(st["x"].float().abs().max(dim=1, keepdim=True).values.div(
                torch.tensor([127.0], device="cuda")), min=1e-8)  # the step is an fp32 value, as the codes go by it
            codes = torch.round(torch.div(st["x"].float(), step)).double()
            step = step.double()
        out = torch.einsum("mk,nk->mn", codes, st["weight"].double())
        out *= step * st["scales"].double()[None]
        if st["bias"] is not None:
            out += st["bias"].double()
        if case["gelu"]:
            out *= torch.special.erfc(-out / math.sqrt(2.0)) / 2
        if st["residual"] is not None:
            out += st["residual"].double()
        return out
    if case["op"] == "rotary":
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
        for x in (st["q"].double(), st["k"].double()):
            if case["interleaved"]:
                z = torch.view_as_complex(x.unflatten(-1, (half, 2)).contiguous()) * by
                res.append(torch.view_as_real(z).flatten(-2))
            else:
                z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * by
                res.append(torch.cat([z.real, z.imag], -1))
        return tuple(res)
    q_len, k_len = _lengths(case)
    if sum(a * b for a, b in zip(q_len, k_len)) * case["heads"] > 1 << 32:
        return None
    out, i, j = torch.empty(st["q"].shape, device="cuda", dtype=torch.float64), 0, 0
    group = case["heads"] // case["kv_heads"]
    for a, b in zip(q_len, k_len):
        last = torch.arange(b - a, b, device="cuda") if case["causal"] else torch.full((a,), b - 1, device="cuda")
        hidden = torch.arange(b, device="cuda")[None] > last[:, None]
        for h in range(case["kv_heads"]):
            kk, vv = st["k"][j:j + b, h].double(), st["v"][j:j + b, h].double()
            qq = st["q"][i:i + a, h * group:(h + 1) * group].double().transpose(0, 1)
            w = torch.softmax((torch.matmul(qq, kk.T) / math.sqrt(case["head_dim"])).masked_fill(hidden, -math.inf), -1)
            out[i:i + a, h * group:(h + 1) * group] = torch.matmul(w, vv).transpose(0, 1)
        i, j = i + a, j + b
    return out
