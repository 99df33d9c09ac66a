"""The action expert over prefixes held as codes in a paged cache (encode_packed with kv_bits)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _expert(seed=0, **kw):
    from embodied_efficiency_b200 import ActionExpert, ActionExpertConfig
    torch.manual_seed(seed)
    cfg = dict(d_model=256, n_layers=2, n_heads=4, prefix_len=64)
    return ActionExpert(ActionExpertConfig(**{**cfg, **kw})).cuda().bfloat16().eval()


def _offsets(lens):
    return torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)


@pytest.mark.parametrize("bits,page,n_heads", [(8, 64, 4), (4, 32, 4), (8, 128, 2), (4, 256, 2)])
@pytest.mark.parametrize("horizon", [50, 1])
def test_prefixes_held_as_codes(cuda, bits, page, n_heads, horizon):
    """The sampler over a cache gives what it gives over the 16-bit values read back from it: the two differ by the
    rounding of those values and of 16-bit arithmetic, as the packed and the padded prefixes of one expert do. With 8
    bits the action error against the unquantised prefix is within the 5 % gate of quantised weights."""
    from embodied_efficiency_b200 import CachedKV, GraphedSampler, PackedKV, cache_read, flow_sample
    m = _expert(1, n_heads=n_heads)
    lens = [64, 1, 200, 0, 37]
    pre = torch.randn(sum(lens), 256, device=cuda).bfloat16()
    cu = _offsets(lens)
    x = torch.randn(5, horizon, 32, device=cuda).bfloat16()
    kv = m.encode_packed(pre, cu, kv_bits=bits, page_size=page)
    assert all(isinstance(c, CachedKV) and c.cache.bits == bits for c in kv)
    assert kv[0].cache.pages == sum(-(-n // page) for n in lens)
    back = [PackedKV(*cache_read(c.cache, cu, c.table, c.k_lens, sum(lens)), cu) for c in kv]
    exact = m.encode_packed(pre, cu)
    for c, e in zip(back, exact):  # half a step of a head's largest value, and a 16-bit rounding
        for a, b in ((c.k, e.k), (c.v, e.v)):
            big = b.float().abs().amax(-1, keepdim=True)
            assert ((a.float() - b.float()).abs() <= big * (0.5 / (127 if bits == 8 else 7) + 2 ** -8)).all()
    out, ref = flow_sample(m, x, 4, kv), flow_sample(m, x, 4, back)
    assert float((out.float() - ref.float()).abs().max()) <= 3e-2 * float(ref.float().abs().max())
    if bits == 8:
        want = flow_sample(m, x, 4, exact).float()
        assert float((out.float() - want).pow(2).mean().sqrt() / want.abs().mean()) <= 5e-2
    gs = GraphedSampler(m, x, 4, prefix_kv=kv)
    assert torch.equal(gs.run(x), out)
    with pytest.raises(ValueError, match="packed prefixes"):
        flow_sample(m, x[:3], 4, kv)
    with pytest.raises(ValueError, match="does not cover"):
        flow_sample(m, x, 4, kv, path="fused")


def test_codes_carry_no_gradient(cuda):
    m = _expert()
    kv = m.encode_packed(torch.randn(9, 256, device=cuda).bfloat16().requires_grad_(), _offsets([4, 5]), kv_bits=8)
    assert not any(t.requires_grad for t in (kv[0].cache.k_scale, kv[0].cache.v_scale))


@pytest.mark.parametrize("lens", [(30, 64, 64, 5, 64, 64), (64,) * 6])
def test_fleet_over_codes(cuda, lens):
    from embodied_efficiency_b200 import CachedKV, flow_sample
    from embodied_efficiency_b200.fleet import FleetSampler
    m = _expert(2)
    g = torch.Generator().manual_seed(3)
    reqs = [(torch.randn(1, n, 256, generator=g), torch.randn(1, 50, 32, generator=g)) for n in lens]
    fs = FleetSampler(6, 0, 1, chunk=4, n_steps=3, expert=m, device=cuda, kv_bits=8).stage(lambda i: reqs[i])
    assert all(isinstance(c[4][0], CachedKV) for c in fs._inputs)
    acts = fs.run().actions
    for i, (pre, x0) in enumerate(reqs):
        kv = m.encode_packed(pre[0].to(cuda), _offsets([lens[i]]), kv_bits=8)
        ref = flow_sample(m, x0.to(cuda).bfloat16(), 3, kv).float().cpu()
        assert float((acts[i] - ref[0]).abs().max()) <= 3e-2 * float(ref.abs().max())
