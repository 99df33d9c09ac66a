"""What the prompt-layer operators refuse, on a machine without a GPU: Python arguments before any device call, and
the C ABI's error codes before any launch."""
import ctypes

import pytest
import torch

BF = torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    from embodied_efficiency_b200 import _lib, build
    build.build()
    return _lib.load()


def test_int8_arguments():
    from embodied_efficiency_b200 import int8_linear, int8_matmul, quantize_tokens
    x, w, s = torch.zeros(3, 64, dtype=BF), torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)
    for match, call in (
            ("K=64, weight has K=48", lambda: int8_linear(x, w[:, :48], s)),
            ("weight must be int8", lambda: int8_linear(x, w.float(), s)),
            ("multiple of 16", lambda: int8_linear(x[:, :40], w[:, :40], s)),
            ("multiple of 16", lambda: int8_linear(torch.zeros(1, 131072, dtype=BF),
                                                   torch.zeros(1, 131072, dtype=torch.int8), s[:1])),
            ("outputs are bf16 or fp16", lambda: int8_linear(x.float(), w, s)),
            ("one per output channel", lambda: int8_linear(x, w, s[:7])),
            ("one per output channel", lambda: int8_linear(x, w, s.double())),
            ("bias has 7", lambda: int8_linear(x, w, s, torch.zeros(7))),
            ("residual has shape", lambda: int8_linear(x, w, s, residual=torch.zeros(3, 7))),
            ("xq must be int8", lambda: int8_matmul(x, torch.ones(3, 1), w, s)),
            ("one per token", lambda: int8_matmul(x.to(torch.int8), torch.ones(2, 1), w, s)),
            ("one per token", lambda: int8_matmul(x.to(torch.int8), torch.ones(3, 1, dtype=BF), w, s)),
            ("outputs are bf16 or fp16", lambda: int8_matmul(x.to(torch.int8), torch.ones(3), w, s,
                                                             dtype=torch.float32)),
            ("bf16 or fp16", lambda: quantize_tokens(x.float())),
            ("multiple of 16", lambda: quantize_tokens(x[:, :24]))):
        with pytest.raises(ValueError, match=match):
            call()
    for call in (lambda: int8_linear(x, w, s), lambda: int8_matmul(x.to(torch.int8), torch.ones(3, 1), w, s),
                 lambda: quantize_tokens(x)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_rotary_arguments():
    from embodied_efficiency_b200 import rotary_embed
    q, k, p = torch.zeros(5, 4, 64, dtype=BF), torch.zeros(5, 2, 64, dtype=BF), torch.zeros(3, 5, dtype=torch.int32)
    for match, call in (
            ("sum to head_dim / 2", lambda: rotary_embed(q, k, p, (10, 10, 10))),
            ("sum to head_dim / 2", lambda: rotary_embed(q, k, p, (40, -8))),
            ("one to four", lambda: rotary_embed(q, k, p, (8, 8, 8, 4, 4))),
            ("one to four", lambda: rotary_embed(q, k, p, ())),
            ("positions have shape", lambda: rotary_embed(q, k, p, (16, 16))),
            ("positions have shape", lambda: rotary_embed(q, k, p[:, :4], (10, 11, 11))),
            ("int32 or int64", lambda: rotary_embed(q, k, p.float(), (10, 11, 11))),
            ("head_dim must be", lambda: rotary_embed(q[..., :48], None, p[0], (24,))),
            ("base must be", lambda: rotary_embed(q, k, p[0], (32,), base=0.0)),
            ("do not belong together", lambda: rotary_embed(q, k[:4], p[0], (32,))),
            ("do not belong together", lambda: rotary_embed(q, k.half(), p[0], (32,))),
            ("needs q or k", lambda: rotary_embed(None, None, p[0], (32,)))):
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError, match="no CPU path"):
        rotary_embed(q, k, p, (10, 11, 11))


def test_attention_arguments():
    from embodied_efficiency_b200 import prompt_attention
    q, k, cu = torch.zeros(5, 4, 64, dtype=BF), torch.zeros(9, 2, 64, dtype=BF), torch.tensor([0, 5], dtype=torch.int32)
    for match, call in (
            ("do not match", lambda: prompt_attention(q, k, k[:8], cu, cu)),
            ("do not match", lambda: prompt_attention(q, k.half(), k.half(), cu, cu)),
            ("must be \\[tokens, heads", lambda: prompt_attention(q[0], k, k, cu, cu)),
            ("must be \\[tokens, heads", lambda: prompt_attention(q, k[..., :32], k[..., :32], cu, cu)),
            ("head_dim must be", lambda: prompt_attention(q[..., :32], k[..., :32], k[..., :32], cu, cu)),
            ("not a multiple", lambda: prompt_attention(q[:, :3], k, k, cu, cu)),
            ("offsets of their own", lambda: prompt_attention(q, k, k, cu)),
            ("cu_q must be int32", lambda: prompt_attention(q, k, k, cu.long(), cu)),
            ("cu_k must be int32 \\[2\\]", lambda: prompt_attention(q, k, k, cu, torch.zeros(3, dtype=torch.int32))),
            ("k_lens must be int32 \\[1\\]", lambda: prompt_attention(q, k, k, cu, cu, cu)),
            ("at least one offset", lambda: prompt_attention(q, k, k, cu[:0], cu)),
            ("scale must be", lambda: prompt_attention(q, k, k, cu, cu, scale=0.0)),
            ("scale must be", lambda: prompt_attention(q, k, k, cu, cu, scale=float("inf")))):
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError, match="no CPU path"):
        prompt_attention(q, k, k, cu, cu)


def test_no_backward_pass():
    """Inputs that ask for a gradient are refused before anything runs, unless gradients are off."""
    from embodied_efficiency_b200 import _lib
    x = torch.zeros(2, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward pass"):
        _lib.no_grad_through("op", None, x)
    with torch.no_grad():
        _lib.no_grad_through("op", x)
    _lib.no_grad_through("op", x.detach())


def test_abi_codes(lib):
    from embodied_efficiency_b200 import _lib
    # ee_quantize_tokens(x, ldx, xq, x_scales, m, k, act, stream)
    qt = [16, 64, 16, 16, 3, 64, _lib.EE_BF16, None]
    for i, v, rc in ((0, 0, 1), (2, 0, 1), (3, 0, 1), (0, 8, 3), (1, 63, 2), (1, 68, 2), (5, 40, 2), (4, -1, 2),
                     (6, 7, 4)):
        assert lib.ee_quantize_tokens(*(qt[:i] + [v] + qt[i + 1:])) == rc, (i, v)
    assert lib.ee_quantize_tokens(*(qt[:4] + [0] + qt[5:])) == 0  # nothing to do
    # ee_int8_gemm(xq, sx, weight, sw, bias, residual, y, m, n, k, scale_dtype, act, epilogue, stream)
    mm = [16, 16, 16, 16, 0, 0, 16, 3, 8, 64, _lib.EE_F32, _lib.EE_BF16, 0, None]
    for i, v, rc in ((0, 0, 1), (1, 0, 1), (2, 0, 1), (3, 0, 1), (6, 0, 1), (0, 8, 3), (2, 8, 3), (9, 24, 2),
                     (9, 131072, 2), (7, -1, 2), (7, 1 << 31, 2), (8, 1 << 31, 2), (10, _lib.EE_BF16, 4), (11, 2, 4),
                     (12, 8, 1), (12, _lib.EE_EPI_BIAS, 1), (12, _lib.EE_EPI_RESIDUAL, 1), (12, 6, 1), (4, 8, 3)):
        assert lib.ee_int8_gemm(*(mm[:i] + [v] + mm[i + 1:])) == rc, (i, v)
    # ee_int8_linear(x, ldx, weight, sw, bias, residual, y, ws, ws_bytes, m, n, k, scale_dtype, act, epilogue, stream)
    need = lib.ee_int8_linear_workspace_bytes(3, 64)
    assert need == 3 * 64 + 12 and lib.ee_int8_linear_workspace_bytes(-1, 64) == 0
    li = [16, 64, 16, 16, 0, 0, 16, 16, need, 3, 8, 64, _lib.EE_F32, _lib.EE_BF16, 0, None]
    for i, v, rc in ((7, 0, 5), (8, need - 1, 5), (7, 8, 3), (0, 0, 1), (1, 56, 2), (11, 24, 2), (13, 2, 4)):
        assert lib.ee_int8_linear(*(li[:i] + [v] + li[i + 1:])) == rc, (i, v)
    # ee_rotary(q, tok, head, q_out, tok, head, k, ..., k_out, ..., pos, pos_axis, pos_bits, freqs, tokens, n_q, n_kv,
    #           head_dim, sections, n_axes, interleaved, act, stream)
    sec = (ctypes.c_int32 * 2)(16, 16)
    ro = [16, 256, 64, 16, 256, 64, 16, 128, 64, 16, 128, 64, 16, 5, 32, 16, 5, 4, 2, 64, sec, 2, 0, _lib.EE_BF16, None]
    for i, v, rc in ((0, 0, 1), (3, 0, 1), (6, 0, 1), (9, 0, 1), (12, 0, 1), (15, 0, 1), (0, 8, 3), (9, 8, 3), (1, 4, 3),
                     (11, 4, 3), (12, 2, 3), (14, 16, 1), (16, -1, 1), (19, 96, 9), (19, 128, 2), (20, None, 1),
                     (21, 0, 1), (21, 5, 1), (23, 2, 4)):
        assert lib.ee_rotary(*(ro[:i] + [v] + ro[i + 1:])) == rc, (i, v)
    assert lib.ee_rotary(*(ro[:16] + [0] + ro[17:])) == 0
    # ee_prompt_attention(q, tok, head, k, .., v, .., out, .., cu_q, cu_k, k_lens, tq, tk, n_seq, n_q, n_kv, head_dim,
    #                     causal, scale, act, workspace, bytes, stream)
    pa = [16, 256, 64, 16, 128, 64, 16, 128, 64, 16, 256, 64, 16, 16, 0, 5, 9, 1, 4, 2, 64, 1, 0.125, _lib.EE_BF16, 0,
          0, None]
    for i, v, rc in ((0, 0, 1), (3, 0, 1), (6, 0, 1), (9, 0, 1), (12, 0, 1), (13, 0, 1), (3, 8, 3), (10, 4, 3),
                     (14, 2, 3), (15, -1, 2), (16, 1 << 31, 2), (17, -1, 2), (19, 3, 2), (18, 0, 2), (20, 256, 9),
                     (22, 0.0, 1), (22, float("nan"), 1), (23, 2, 4)):
        assert lib.ee_prompt_attention(*(pa[:i] + [v] + pa[i + 1:])) == rc, (i, v)
    assert lib.ee_prompt_attention(*(pa[:15] + [0] + pa[16:])) == 0
