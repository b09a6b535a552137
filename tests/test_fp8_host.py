"""Refusals of the 8-bit inference operators and of the filtered token choice (CPU only: every one is decided before a launch)."""
import math

import pytest
import torch


def test_wrappers_refuse_bad_arguments():
    from src import ops
    x = torch.zeros(4, 8)
    w = torch.ones(8)
    with pytest.raises(ValueError, match="activation"):
        ops.quantize_fp8(x, "gelu")
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        ops.quantize_fp8(x.half())
    with pytest.raises(ValueError, match="last dimension"):
        ops.quantize_fp8(torch.zeros(4, 0))
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.quantize_fp8(x)
    with pytest.raises(ValueError, match="weight"):
        ops.rms_norm_fp8(x, torch.ones(7), 1e-6)
    with pytest.raises(ValueError, match="weight"):
        ops.rms_norm_fp8(x, w.bfloat16(), 1e-6)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.rms_norm_fp8(x, w, 1e-6)
    q = torch.zeros(4, 16).to(torch.float8_e4m3fn)
    s = torch.zeros(4, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        ops.fp8_matmul(x, s, q, s[:1])
    with pytest.raises(TypeError, match="float8_e8m0fnu"):
        ops.fp8_matmul(q, torch.zeros(4, 1), q, s[:1])
    with pytest.raises(ValueError, match="scales of shape"):
        ops.fp8_matmul(q, s[:3], q, s[:1])
    with pytest.raises(ValueError, match="scales of shape"):
        ops.fp8_matmul(q, s, q, s)
    with pytest.raises(ValueError, match="columns"):
        ops.fp8_matmul(q, s, q[:, :8], s[:1])
    with pytest.raises(ValueError, match="bias"):
        ops.fp8_matmul(q, s, q, s[:1], bias=torch.zeros(5))
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.fp8_matmul(q, s, q, s[:1])
    with pytest.raises(ValueError, match="float32 matrix"):
        ops.quantize_fp8_weight(torch.zeros(3))
    u = torch.zeros(4)
    for bad in (dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf), dict(temperature=1e-40), dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.5),
                dict(top_p=math.nan), dict(min_p=-0.1), dict(min_p=1.1)):
        with pytest.raises(ValueError):
            ops.sample_tokens(x, u, **bad)
    with pytest.raises(ValueError, match="u must be"):
        ops.sample_tokens(x, torch.zeros(3))
    with pytest.raises(ValueError, match="u must be"):
        ops.sample_tokens(x, u.double())
    with pytest.raises(ValueError, match="ids must be"):
        ops.sample_tokens(x, u, ids=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.sample_tokens(x, u)


BADARG, ALIGN, SHAPE, DTYPE = -1, -2, -3, -4


def test_c_entry_points_refuse_before_launching():
    from src import _native as N
    lib = N.lib()
    P = 4096      # an address that is never read: each call below is refused on the host

    def quant(x=P, dtype=0, ld_x=256, T=4, d=256, sw=0, q=P, ld_q=256, s=P, ld_s=2):
        return lib.ldm_quant_fp8(x, dtype, ld_x, T, d, sw, q, ld_q, s, ld_s, None)
    assert quant(T=0) == 0
    assert quant(T=-1) == BADARG and quant(d=0) == BADARG and quant(x=None) == BADARG and quant(ld_x=255) == BADARG
    assert quant(sw=1, ld_x=511) == BADARG and quant(ld_s=1) == BADARG and quant(s=None) == BADARG
    assert quant(dtype=7) == DTYPE and quant(ld_q=255) == ALIGN and quant(q=P + 4) == ALIGN
    assert quant(T=1 << 40) == SHAPE

    def norm(x=P, xd=1, ld_x=256, r=P, sd=1, ld_r=256, w=P, T=4, d=256, out=P, q=P, ld_q=256, s=P, ld_s=2):
        return lib.ldm_rmsnorm_fp8(x, xd, ld_x, r, sd, ld_r, w, T, d, 1e-6, out, q, ld_q, s, ld_s, None)
    assert norm(T=0) == 0
    assert norm(x=None) == BADARG and norm(w=None) == BADARG and norm(out=None) == BADARG and norm(ld_r=128) == BADARG
    assert norm(xd=0, sd=1) == DTYPE and norm(xd=3) == DTYPE and norm(sd=5) == DTYPE
    assert norm(d=16385, ld_x=20000, ld_r=20000, ld_q=20000, ld_s=200) == SHAPE and norm(ld_q=260) == ALIGN

    def gemm(M=4, n=8, K=256, A=P, lda=256, sA=P, lsa=2, B=P, ldb=256, sB=P, lsb=2, bias=None, C=P, ldc=8):
        return lib.ldm_gemm_fp8(M, n, K, A, lda, sA, lsa, B, ldb, sB, lsb, bias, C, ldc, None)
    assert gemm(M=0) == 0 and gemm(n=0) == 0
    assert gemm(K=0) == BADARG and gemm(A=None) == BADARG and gemm(sB=None) == BADARG and gemm(lda=240) == BADARG
    assert gemm(ldc=7) == BADARG and gemm(lsa=1) == BADARG and gemm(lsb=1) == BADARG
    assert gemm(lda=264) == ALIGN and gemm(A=P + 8) == ALIGN and gemm(C=P + 1) == ALIGN and gemm(bias=P + 2) == ALIGN

    assert lib.ldm_quant_fp8_block(P, 200, 8, 256, P, 256, P, 2, None) == BADARG
    assert lib.ldm_quant_fp8_block(P, 256, 8, 256, P, 250, P, 2, None) == ALIGN
    assert lib.ldm_quant_fp8_block(P, 256, 0, 256, P, 256, P, 2, None) == 0

    def samp(l=P, dt=0, T=4, V=100, ld=100, u=P, ids=None, t=1.0, k=0, p=1.0, m=0.0, out=P):
        return lib.ldm_sample_filtered(l, dt, T, V, ld, u, ids, 103, t, k, p, m, out, None)
    assert samp(T=0) == 0
    assert samp(l=None) == BADARG and samp(u=None) == BADARG and samp(out=None) == BADARG and samp(ld=99) == BADARG
    assert samp(V=0) == BADARG and samp(k=-1) == BADARG and samp(p=0.0) == BADARG and samp(m=1.5) == BADARG
    assert samp(t=1e-40) == BADARG and samp(t=math.inf) == BADARG and samp(t=-0.5) == BADARG and samp(t=math.nan) == BADARG and samp(p=math.nan) == BADARG
    assert samp(dt=4) == DTYPE and samp(V=262145, ld=262145) == SHAPE


def test_weight_copies_refuse_a_pair_of_another_layout():
    from src import ops
    e4m3, e8m0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    w = torch.zeros(300, 200)

    def values(n=300, ld=208, k=200):
        return torch.zeros(n, ld, dtype=torch.uint8).view(e4m3)[:, :k]

    def scales(n=3, k=2):
        return torch.zeros(n, k, dtype=torch.uint8).view(e8m0)

    bad = [(values(), scales(2, 2)), (values(), scales(3, 1)), (values(), scales().view(torch.uint8)),
           (values(), scales(2, 3).t()), (values(n=299), scales()), (values(ld=200), scales()), (values(ld=224), scales()),
           (values().view(torch.uint8), scales()), (values().t(), scales()),
           (values(), scales(1, 2).expand(3, 2)),
           (torch.zeros(300 * 208 + 16, dtype=torch.uint8).view(e4m3)[8:8 + 300 * 208].view(300, 208)[:, :200], scales())]
    for pair in bad:
        with pytest.raises((ValueError, TypeError), match="out must be"):
            ops.quantize_fp8_weight(w, out=pair)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.quantize_fp8_weight(w, out=(values(), scales()))


def test_filters_of_the_draw_are_checked_at_every_temperature(monkeypatch):
    """generate / sample with a filter: a bad value is refused at temperature 0 too, and a bad temperature with any filter."""
    import types

    from src import _native
    from src.model import DiffusionLanguageModel
    monkeypatch.setattr(_native, "require_device", lambda t: None)
    m = types.SimpleNamespace(tokenizer=types.SimpleNamespace(mask_token_id=1))
    seq, logits = torch.zeros(1, 4, dtype=torch.int64), torch.zeros(1, 4, 8)
    for temperature, kw in ((-1.0, dict(top_k=5)), (math.nan, dict(top_p=0.9)), (0.0, dict(top_k=-1)),
                            (0.0, dict(top_p=1.5)), (0.0, dict(min_p=-0.5)), (1.0, dict(top_p=0.0))):
        with pytest.raises(ValueError):
            DiffusionLanguageModel._pick_tokens(m, seq, logits, temperature, **kw)


def test_fp32_product_refusals():
    from src import _native as N
    from src import ops
    q = torch.zeros(4, 16).to(torch.float8_e4m3fn)
    s = torch.zeros(4, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    for dt in (torch.float16, torch.float64, torch.int32, None):
        with pytest.raises(TypeError, match="out_dtype"):
            ops.fp8_matmul(q, s, q, s[:1], out_dtype=dt)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.fp8_matmul(q, s, q, s[:1], out_dtype=torch.float32)
    P = 4096      # an address that is never read

    def gemm(M=4, n=8, K=256, A=P, lda=256, sA=P, lsa=2, B=P, ldb=256, sB=P, lsb=2, bias=None, C=P, ldc=8):
        return N.lib().ldm_gemm_fp8_f32(M, n, K, A, lda, sA, lsa, B, ldb, sB, lsb, bias, C, ldc, None)
    assert gemm(M=0) == 0 and gemm(n=0) == 0
    assert gemm(K=0) == BADARG and gemm(M=-1) == BADARG and gemm(C=None) == BADARG and gemm(lda=240) == BADARG
    assert gemm(ldc=7) == BADARG and gemm(lsa=1) == BADARG and gemm(lsb=1) == BADARG
    assert gemm(lda=264) == ALIGN and gemm(B=P + 8) == ALIGN and gemm(C=P + 2) == ALIGN and gemm(bias=P + 2) == ALIGN
    assert gemm(K=(1 << 28) + 1, lda=1 << 29, ldb=1 << 29, lsa=1 << 22, lsb=1 << 22) == SHAPE


def test_copies_of_weights_are_written_by_one_thread(monkeypatch):
    """Threads that find the copies stale together: one writes, the others wait for it and see values, scales, bias and event whole."""
    import copy
    import threading
    import time
    import types

    from src import ops
    writes = []

    def quantize(w, out=None):
        writes.append(threading.get_ident())
        time.sleep(0.02)
        return out or (torch.zeros(3, 4), torch.zeros(1, 1))

    def event():
        time.sleep(0.02)
        return types.SimpleNamespace(record=lambda s: None)

    def wait(self, device):
        assert self._written is not None and self.b is not None and self._stream == 7

    monkeypatch.setattr(ops, "quantize_fp8_weight", quantize)
    monkeypatch.setattr(ops.Fp8Weights, "_wait", wait)
    monkeypatch.setattr(torch.cuda, "Event", event)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: types.SimpleNamespace(cuda_stream=7))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    w, b = torch.nn.Parameter(torch.zeros(3, 4)), torch.nn.Parameter(torch.zeros(3))
    pack = ops.Fp8Weights([w], [b])
    for step in range(3):
        got, failed = [], []

        def call():
            try:
                got.append(pack.get())
            except BaseException as e:
                failed.append(e)
        threads = [threading.Thread(target=call) for _ in range(8)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not failed and len(got) == 8 and len(writes) == step + 1, (failed, len(writes))
        assert all(g[0] is got[0][0] and g[2] is not None for g in got)
        with torch.no_grad():
            w.add_(1.0)
    twin = copy.deepcopy(pack)
    assert twin.q is None and twin.get()[0] is not pack.get()[0]


def test_copies_are_of_the_parameters_that_the_modules_hold_now():
    from src.transformer import DiffusionTransformer, DiffusionTransformerConfig
    cfg = DiffusionTransformerConfig(vocab_size=40, d_model=32, nhead=2, num_layers=1, dim_feedforward=24)
    tr, other = DiffusionTransformer(cfg), DiffusionTransformer(cfg)
    layer = tr.layers[0]

    def packs():
        return [layer.self_attn._fp8_pack("qkv"), layer.self_attn._fp8_pack("out"), layer.swiglu._fp8_pack("in"),
                layer.swiglu._fp8_pack("out"), tr._fp8_head_pack()]
    before = packs()
    assert all(a is b for a, b in zip(before, packs()))
    tr.load_state_dict(other.state_dict(), assign=True)
    assert all(a is not b for a, b in zip(before, packs()))
    held = {id(p) for p in tr.parameters()}
    assert all(id(p) in held for pack in packs() for p in pack.weights + pack.biases)
    layer.swiglu.w3.bias = torch.nn.Parameter(torch.ones(32))
    now = packs()
    assert now[3].biases[0] is layer.swiglu.w3.bias and now[2] is packs()[2]


def test_tangents_are_refused():
    """Forward-mode differentiation: a tensor with a tangent would lose it without a word."""
    from torch.autograd import forward_ad

    from src import ops
    x, w = torch.ones(4, 8), torch.ones(8)
    q = torch.zeros(4, 16).to(torch.float8_e4m3fn)
    s = torch.zeros(4, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    with forward_ad.dual_level():
        dual, dw = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: ops.quantize_fp8(dual), lambda: ops.quantize_fp8(dual, "swiglu"),
                     lambda: ops.rms_norm_fp8(dual, w, 1e-6), lambda: ops.rms_norm_fp8(x, dw, 1e-6),
                     lambda: ops.rms_norm_fp8(x, w, 1e-6, residual=dual),
                     lambda: ops.fp8_matmul(q[:, :8], s, q[:, :8], s[:1], bias=forward_ad.make_dual(torch.ones(4), torch.ones(4)))):
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent|ROCm device") as e:
                call()
            assert "tangent" in str(e.value)
        with pytest.raises(RuntimeError, match="ROCm device"):      # tensors without one: as ever
            ops.quantize_fp8(x)


def test_products_beyond_the_largest_grid_are_refused():
    from src import _native as N
    P = 4096      # an address that is never read
    for entry in (N.lib().ldm_gemm_fp8, N.lib().ldm_gemm_fp8_f32):
        for M, n in ((1, 1 << 29), (1 << 31, 1)):
            assert entry(M, n, 16, P, 16, P, 1, P, 16, P, 1, None, P, n, None) == SHAPE


def test_models_pickled_before_the_8_bit_path():
    """Their objects have none of its attributes: off by default, and usable."""
    import pickle

    from src.transformer import DiffusionTransformer, DiffusionTransformerConfig
    tr = DiffusionTransformer(DiffusionTransformerConfig(vocab_size=40, d_model=32, nhead=2, num_layers=1, dim_feedforward=24))
    for m in tr.modules():
        for name in ("_fp8_packs", "fp8_inference", "fp8_head"):
            m.__dict__.pop(name, None)
    tr = pickle.loads(pickle.dumps(tr))
    with torch.no_grad():
        assert tr._fp8_now() is False and tr.fp8_head is False
    layer = tr.layers[0]
    assert tr._fp8_head_pack() is tr._fp8_head_pack()
    assert layer.self_attn._fp8_pack("qkv") is layer.self_attn._fp8_pack("qkv") is not layer.self_attn._fp8_pack("out")
    assert layer.swiglu._fp8_pack("in").weights[1] is layer.swiglu.w2.weight
    other = DiffusionTransformer(DiffusionTransformerConfig(vocab_size=40, d_model=32, nhead=2, num_layers=1, dim_feedforward=24))
    other.fp8_inference = True
    assert tr.fp8_inference is False and other.layers[0].swiglu._fp8_pack("in") is not layer.swiglu._fp8_pack("in")
