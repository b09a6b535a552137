"""The 8-bit forward as a whole, heads of 96, the fp32 residual stream, strided scales: on a real MI355X."""
import copy

import pytest
import torch

from test_gpu_fp8 import check_matmul
from test_gpu_fp8_f32 import check
from test_gpu_fp8_model import CFG, batch, make

pytestmark = pytest.mark.gpu


@torch.no_grad()
@pytest.mark.parametrize("fp32_residual", [False, True])
@pytest.mark.parametrize("fp8_head", [False, True])
def test_forward_is_within_the_rounding_of_its_products(dev, fp32_residual, fp8_head):
    """Against the bf16 forward: each product carries the rounding of two operands, each uniform within 2^-4, so 2^-4 / sqrt(3)
    in the 2-norm, independent of each other; the products' shares add up as squares.  A forward without one of its
    sublayers (its last projection set to zero) is further off than that."""
    tr = make(dev, fp32_residual=fp32_residual, fp8_head=fp8_head).eval().transformer
    ids, att = batch(dev)
    live = att.bool()
    y8 = tr(ids, att).double()
    tr.fp8_inference = False

    def off(t):
        y = t(ids, att).double()
        return float((y8 - y)[live].norm() / y[live].norm())
    products = 4 * CFG["L"] + (1 if fp8_head else 0)
    bound = (products * 2 / 3) ** 0.5 * 2.0 ** -4
    assert off(tr) < bound
    for layer in range(CFG["L"]):
        for name in ("self_attn.out_proj", "swiglu.w3"):
            other = copy.deepcopy(tr)
            last = other.layers[layer].get_submodule(name)
            last.weight.zero_()
            last.bias.zero_()
            assert off(other) > 2 * bound


@torch.no_grad()
@pytest.mark.parametrize("H", [2, 3, 6])            # heads of 96, 64, 32
@pytest.mark.parametrize("fp32_residual", [False, True])
def test_forward_is_the_composition_of_the_operators(dev, H, fp32_residual):
    """The path written out with ops.* and freshly quantised weights gives the same bits: head widths, both residual streams."""
    from src import ops
    from src.transformer import DiffusionTransformer, DiffusionTransformerConfig
    torch.manual_seed(H)
    tr = DiffusionTransformer(DiffusionTransformerConfig(vocab_size=300, d_model=192, nhead=H, num_layers=2, dim_feedforward=200,
                                                         dropout=0.0)).to(dev).set_compute_dtype(torch.bfloat16).eval()
    tr.fp8_inference, tr.fp8_head, tr.fp32_residual = True, True, fp32_residual
    ids, att = batch(dev)
    ids = ids % 300

    def lin(x, *mods):
        wq, ws = ops.quantize_fp8_weight(torch.cat([k.weight for k in mods]))
        return ops.fp8_matmul(*x, wq, ws, bias=torch.cat([k.bias for k in mods]))
    branch, stream = ops.embedding(ids, tr.embedding.weight, torch.float32 if fp32_residual else torch.bfloat16), None
    key_valid = (att != 0).to(torch.uint8)
    for layer in tr.layers:
        q, s, stream = ops.rms_norm_fp8(branch, layer.norm1.weight, layer.norm1.eps, residual=stream)
        at = layer.self_attn
        cos, sin = at.rotary_emb.half_tables(q, ids.shape[1])
        qkv = lin((q, s), at.q_proj, at.k_proj, at.v_proj)
        o = ops.rope_attention(qkv, key_valid, *ids.shape, at.nhead, at.head_dim, cos, sin)
        branch = lin(ops.quantize_fp8(o), at.out_proj)
        q, s, stream = ops.rms_norm_fp8(branch, layer.norm2.weight, layer.norm2.eps, residual=stream)
        branch = lin(ops.quantize_fp8(lin((q, s), layer.swiglu.w1, layer.swiglu.w2), "swiglu"), layer.swiglu.w3)
    q, s, stream = ops.rms_norm_fp8(branch, tr.norm.weight, tr.norm.eps, residual=stream)
    assert stream.dtype == (torch.float32 if fp32_residual else torch.bfloat16)
    assert torch.equal(tr(ids, att), lin((q, s), tr.output_layer))


@pytest.mark.parametrize("M,N,K", [(20, 300, 400), (300, 700, 400), (4096, 4096, 512)])
def test_strided_scales(dev, M, N, K):
    """Scales as columns of a wider tensor, transposed, and with other memory behind every row."""
    from src import ops
    g = torch.Generator(device=dev).manual_seed(M)
    xq, xs = ops.quantize_fp8(torch.randn(M, K, generator=g, device=dev) * torch.exp(2 * torch.randn(M, 1, generator=g, device=dev)))
    wq, ws = ops.quantize_fp8_weight(torch.randn(N, K, generator=g, device=dev) * torch.exp(torch.randn(N, 1, generator=g, device=dev)))

    def wider(s):
        buf = torch.full((s.shape[0], s.shape[1] + 5), 255, dtype=torch.uint8, device=dev)
        buf[:, 3:3 + s.shape[1]] = s.view(torch.uint8)
        return buf.view(torch.float8_e8m0fnu)[:, 3:3 + s.shape[1]]

    def transposed(s):
        return s.view(torch.uint8).t().contiguous().t().view(torch.float8_e8m0fnu)
    want, want32 = ops.fp8_matmul(xq, xs, wq, ws), ops.fp8_matmul(xq, xs, wq, ws, out_dtype=torch.float32)
    if M < 1000:
        check_matmul(want, xq, xs, wq, ws, None, K)
        check(want32, xq, xs, wq, ws, None)
    for form in (wider, transposed):
        a, b = form(xs), form(ws)
        assert not a.is_contiguous()
        assert torch.equal(ops.fp8_matmul(xq, a, wq, b), want)
        assert torch.equal(ops.fp8_matmul(xq, a, wq, b, out_dtype=torch.float32), want32)
