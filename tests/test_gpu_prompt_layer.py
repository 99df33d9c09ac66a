"""The prompt-layer operators as they are used together: the attention half of a transformer layer over packed
prompts and then over one new token behind a cache; 8-bit activations and prefixes of different lengths in the
action expert, the sampler's graph and the fleet."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def _q(x):
    """The token quantiser in 64 bits of fp32 steps: what int8_linear multiplies."""
    xf = x.float()
    s = (xf.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device=x.device)).clamp_min(1e-8)
    return torch.round(xf / s).double() * s.double()


def test_a_layer_over_packed_prompts_and_a_new_token(cuda):
    """int8 q/k/v projection -> rotary positions in place -> causal attention -> int8 output projection with the
    residual stream, for three prompts at once, then for one new token of each against the cache they left. The
    reference takes the same roundings of the steps' results and 64 bits inside each step; the tolerance is the last
    step's: its input's code may differ by one where the attention's result differs by a rounding."""
    from embodied_efficiency_b200 import int8_linear, prompt_attention, rotary_embed
    g = torch.Generator(device=cuda).manual_seed(11)
    d, hq, hk, hd, cap = 512, 8, 2, 64, 320
    lens, sections = [300, 17, 129], (8, 12, 12)
    width = (hq + 2 * hk) * hd

    def lin(n, k):
        return (torch.randint(-127, 128, (n, k), generator=g, device=cuda, dtype=torch.int8),
                torch.full((n,), 0.6 / (73 * k ** 0.5), device=cuda))

    (w_in, s_in), (w_out, s_out) = lin(width, d), lin(d, hq * hd)
    cache = torch.full((3 * cap, 2, hk, hd), float("nan"), device=cuda, dtype=torch.bfloat16)
    start = [b * cap for b in range(3)]

    def step(x, q_len, past):
        t = x.shape[0]
        pos = torch.cat([torch.stack([torch.arange(p, p + n), torch.arange(p, p + n) // 16,
                                      torch.arange(p, p + n) % 16]) for n, p in zip(q_len, past)], 1).to(cuda)
        qkv = int8_linear(x, w_in, s_in)
        raw = qkv.clone()
        q, k, v = qkv.split([hq * hd, hk * hd, hk * hd], -1)
        q, k, v = (y.unflatten(-1, (-1, hd)) for y in (q, k, v))
        rotary_embed(q, k, pos, sections, out=(q, k))
        at = torch.cat([torch.arange(s + p, s + p + n) for s, p, n in zip(start, past, q_len)]).to(cuda)
        cache[at, 0], cache[at, 1] = k, v
        cu_q = torch.tensor([0] + q_len, device=cuda).cumsum(0).to(torch.int32)
        cu_k = torch.tensor(start + [3 * cap], device=cuda, dtype=torch.int32)
        used = torch.tensor([p + n for p, n in zip(past, q_len)], device=cuda, dtype=torch.int32)
        o = prompt_attention(q, cache[:, 0], cache[:, 1], cu_q, cu_k, used)
        y = int8_linear(o.reshape(t, hq * hd), w_out, s_out, residual=x)
        # the same in 64 bits, from the rounded results of the step before
        assert float((raw.double() - _q(x) @ (w_in.double().T * s_in.double())).abs().max()) <= 2 ** -8 * float(raw.abs().max())
        i = 0
        for b, (n, p) in enumerate(zip(q_len, past)):
            kk = cache[start[b]:start[b] + p + n, 0].double().repeat_interleave(hq // hk, 1).transpose(0, 1)
            vv = cache[start[b]:start[b] + p + n, 1].double().repeat_interleave(hq // hk, 1).transpose(0, 1)
            sc = q[i:i + n].double().transpose(0, 1) @ kk.transpose(1, 2) * hd ** -0.5
            hidden = torch.arange(p + n, device=cuda)[None] > torch.arange(p, p + n, device=cuda)[:, None]
            ref = (torch.softmax(sc.masked_fill(hidden, float("-inf")), -1) @ vv).transpose(0, 1)
            assert float((o[i:i + n].double() - ref).abs().max()) <= 2 ** -6 * float(vv.abs().max())
            i += n
        ref = _q(o.reshape(t, hq * hd)) @ (w_out.double().T * s_out.double()) + x.double()
        assert float((y.double() - ref).abs().max()) <= 2 ** -8 * float(ref.abs().max())
        return y

    x = torch.randn(sum(lens), d, generator=g, device=cuda).bfloat16()
    y = step(x, lens, [0, 0, 0])
    assert bool(y.isfinite().all())
    token = torch.randn(3, d, generator=g, device=cuda).bfloat16()
    first = step(token, [1, 1, 1], lens)
    # the same new tokens appended to the prompts' own pass: the last row of each
    longer = torch.cat([torch.cat([x[sum(lens[:b]):sum(lens[:b + 1])], token[b:b + 1]]) for b in range(3)])
    again = step(longer, [n + 1 for n in lens], [0, 0, 0])
    last = torch.tensor([sum(lens[:b + 1]) + b for b in range(3)], device=cuda)
    # two kernels with other summation orders: their 16-bit attention results, and so the codes, differ by a step
    assert float((again[last].float() - first.float()).abs().max()) <= 2 ** -5 * float(first.float().abs().max())


def _expert(seed=0, **kw):
    from embodied_efficiency_b200 import ActionExpert, ActionExpertConfig
    torch.manual_seed(seed)
    return ActionExpert(ActionExpertConfig(d_model=256, n_layers=2, n_heads=4, prefix_len=64, **kw)).cuda().bfloat16().eval()


def _action_error(out, ref):
    return float((out.float() - ref.float()).pow(2).mean().sqrt() / ref.float().abs().mean())


def test_expert_with_8_bit_activations(cuda):
    """The reference's fidelity gate (5 % action error against the 16-bit expert) holds, on every route."""
    from embodied_efficiency_b200 import GraphedSampler, flow_sample, quantize_model_triton
    from embodied_efficiency_b200 import fused
    base = _expert()
    m = quantize_model_triton(copy.deepcopy(base), bits=8, act_bits=8)
    lin = m.blocks[0].qkv
    assert lin.act_bits == 8 and lin.scales.shape == (768, 1) and not fused.supports(m, 2)
    assert "act_bits=8" in repr(lin)
    x = torch.randn(2, 50, 32, device=cuda).bfloat16()
    ref = flow_sample(base, x, 10, base.encode_prefix(2))
    kv = m.encode_prefix(2)
    out = flow_sample(m, x, 10, kv)
    assert _action_error(out, ref) <= 0.05
    with pytest.raises(ValueError, match="does not cover"):
        flow_sample(m, x, 10, kv, path="fused")
    gs = GraphedSampler(m, x, 10, prefix_kv=kv)
    assert not gs.fused and torch.equal(gs.run(x), out)
    y = lin(torch.randn(3, 256, device=cuda))  # fp32 in, fp32 out, as wq_linear
    assert y.dtype == torch.float32 and "_dense" not in lin.__dict__
    big = lin(torch.randn(2000, 256, device=cuda).bfloat16())
    assert big.shape == (2000, 768) and "_dense" not in lin.__dict__


def test_act_bits_refusals():
    from embodied_efficiency_b200 import TritonQuantLinear
    lin = torch.nn.Linear(256, 64)
    for kw in (dict(bits=4, act_bits=8), dict(bits=8, act_bits=4)):
        with pytest.raises(ValueError, match="act_bits"):
            TritonQuantLinear(lin, **kw)
    with pytest.raises(ValueError, match="multiple of 16"):
        TritonQuantLinear(torch.nn.Linear(40, 8), 8, act_bits=8)


@pytest.mark.parametrize("bits", [None, 8])
def test_prefixes_of_different_lengths(cuda, bits):
    """A batch with packed prefixes gives what each request gives by itself on the layer path."""
    from embodied_efficiency_b200 import GraphedSampler, flow_sample, quantize_model_triton
    m = _expert(1)
    if bits:
        quantize_model_triton(m, bits=bits)
    lens = [64, 1, 200, 37]
    pre = [torch.randn(1, n, 256, device=cuda).bfloat16() for n in lens]
    x = torch.randn(4, 50, 32, device=cuda).bfloat16()
    cu = torch.tensor([0] + lens, device=cuda).cumsum(0).to(torch.int32)
    kv = m.encode_packed(torch.cat([p[0] for p in pre]), cu)
    out = flow_sample(m, x, 4, kv)
    for i in range(4):
        ref = flow_sample(m, x[i:i + 1], 4, m.encode(pre[i]), path="layers")
        assert float((out[i].float() - ref[0].float()).abs().max()) <= 3e-2 * float(ref.float().abs().max())
    gs = GraphedSampler(m, x, 4, prefix_kv=kv)
    assert torch.equal(gs.run(x), out)
    with pytest.raises(ValueError, match="packed prefixes"):
        flow_sample(m, x[:3], 4, kv)
    with pytest.raises(ValueError, match="does not cover"):
        flow_sample(m, x, 4, kv, path="fused")


def test_fleet_of_different_prompts(cuda):
    from embodied_efficiency_b200 import flow_sample
    from embodied_efficiency_b200.fleet import FleetSampler
    m = _expert(2)
    g = torch.Generator().manual_seed(3)
    reqs = [(torch.randn(1, n, 256, generator=g), torch.randn(1, 50, 32, generator=g)) for n in (30, 64, 64, 5, 64, 64)]
    fs = FleetSampler(6, 0, 1, chunk=4, n_steps=3, expert=m, device=cuda).stage(lambda i: reqs[i])
    acts = fs.run().actions
    for i, (pre, x0) in enumerate(reqs):
        ref = flow_sample(m, x0.to(cuda).bfloat16(), 3, m.encode(pre.to(cuda)), path="layers").float().cpu()
        assert float((acts[i] - ref[0]).abs().max()) <= 3e-2 * float(ref.abs().max())


def test_offsets_first_asked_for_in_a_capture(cuda):
    """A graph's own memory holds nothing before its replay: what a capture computes is not kept for eager calls, and
    what eager calls keep serves captures and other streams."""
    from embodied_efficiency_b200.expert import PackedKV
    kv = torch.zeros(9, 2, 64, device=cuda, dtype=torch.bfloat16)
    packed = PackedKV(kv, kv, torch.tensor([0, 2, 5, 9], device=cuda, dtype=torch.int32))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = packed.queries(3, 4) + 0
    eager = packed.queries(3, 4)
    assert eager.tolist() == [0, 4, 8, 12]
    graph.replay()
    assert inside.tolist() == [0, 4, 8, 12]
    again = torch.cuda.CUDAGraph()
    with torch.cuda.graph(again):
        assert packed.queries(3, 4) is eager
        keep = eager + 0
    assert packed.queries(3, 5).tolist() == [0, 5, 10, 15]
    assert packed.queries(3, 4) is eager  # still there for the capture
    again.replay()
    assert keep.tolist() == [0, 4, 8, 12]
    with pytest.raises(ValueError):
        packed.queries(4, 4)
