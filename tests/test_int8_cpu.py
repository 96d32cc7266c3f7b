"""8-bit rows, the int8 product and the int8 DiT on CPU: the restatements against the definitions in fp64."""
import pytest
import torch

from harp_b200.inference import batch_image_inference
from harp_b200.models.dit import DiT, DiTConfig
from harp_b200.models.dit_int8 import DiTInt8
from harp_b200.ops import functional as Fn
from harp_b200.ops.modules import Int8Linear, kpLinear

CFG = DiTConfig(in_channels=4, hidden=96, depth=3, heads=2, mlp_ratio=4.0, text_dim=64, axes_dims=(16, 16, 16))


def _model(dtype=torch.bfloat16, cfg=CFG):
    torch.manual_seed(0)
    m = DiT(cfg)
    with torch.no_grad():
        for n, p in m.named_parameters():
            p.normal_(0, 0.02 if "adaLN" in n else 0.08)
            if "norm" in n:
                p.add_(1.0)
    return m.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (2, 1001)])
def test_rows(rows, cols, dtype):
    x = torch.randn(rows, cols, generator=torch.Generator().manual_seed(0)).to(dtype)
    q, s = Fn.quant_rows(x)
    y = x.double()
    s64 = y.abs().amax(1) / 127
    assert q.dtype == torch.int8 and s.dtype == torch.float32
    assert ((s.double() - s64).abs() <= 2.0 ** -23 * s64).all()
    assert ((q.double() * s64[:, None] - y).abs() <= s64[:, None] * (0.5 + 127 * 2.0 ** -22)).all()
    assert torch.equal(Fn.dequant_rows(q, s, torch.float32), q.float() * s[:, None])


def test_rows_special_values():
    x = torch.ones(5, 4)
    x[0] = 0
    x[1, 2] = float("nan")
    x[2, 0] = float("-inf")
    x[3] = 1e-44
    q, s = Fn.quant_rows(x)
    assert (q[0] == 0).all() and s[0] == 2.0 ** -126 and (q[3] == 0).all()
    assert torch.isnan(s[1:3]).all() and (q[1:3] == 0).all()
    assert (q[4] == 127).all()


def test_swiglu_and_norm():
    g = torch.Generator().manual_seed(1)
    gu = torch.randn(6, 40, generator=g)
    q, s = Fn.swiglu_quant(gu, 20)
    y = torch.nn.functional.silu(gu[:, :20].double()) * gu[:, 20:].double()
    assert ((q.double() * s.double()[:, None] - y).abs() <= 0.501 * s.double()[:, None]).all()
    x, r = torch.randn(6, 20, generator=g), torch.randn(6, 20, generator=g)
    w, mod = torch.randn(20, generator=g), torch.randn(2, 60, generator=g)
    q, s, h = Fn.rmsnorm_mod_quant(x, w, mod[:, :20], mod[:, 20:40], 3, 1e-6, residual=r, gate=mod[:, 40:])
    up = mod.double().repeat_interleave(3, 0)
    h64 = r.double() + up[:, 40:] * x.double()
    assert (h.double() - h64).abs().max() < 1e-6
    y = h64 / (h64.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * w.double() * (1 + up[:, :20]) + up[:, 20:40]
    assert ((q.double() * s.double()[:, None] - y).abs() <= 0.501 * s.double()[:, None]).all()
    assert Fn.rmsnorm_mod_quant(x, None, None, None, 0, 1e-6)[2] is x


def test_gemm_s8():
    g = torch.Generator().manual_seed(2)
    a = torch.randint(-128, 128, (5, 300), generator=g, dtype=torch.int8)
    b = torch.randint(-128, 128, (7, 300), generator=g, dtype=torch.int8)
    sa, sb, bias = torch.rand(5, generator=g), torch.rand(7, generator=g), torch.randn(7, generator=g)
    ref = (a.long() @ b.long().t()).double() * sa.double()[:, None] * sb.double() + bias.double()
    c = Fn.gemm_s8(a, sa, b, sb, bias=bias, out_dtype=torch.float32)
    assert ((c.double() - ref).abs() <= 4 * 2.0 ** -24 * ((ref - bias.double()).abs() + bias.double().abs())).all()
    out = torch.empty(5, 7, dtype=torch.bfloat16)
    assert Fn.gemm_s8(a, sa, b, sb, bias=bias, out=out) is out
    assert torch.equal(out, c.bfloat16())
    for bad in (lambda: Fn.gemm_s8(a.float(), sa, b, sb), lambda: Fn.gemm_s8(a, sa, b[:, :299], sb),
                lambda: Fn.gemm_s8(a, sa, b, sb, out_dtype=torch.half), lambda: Fn.quant_rows(a.float()[0]),
                lambda: Fn.quant_rows(a.half()), lambda: Fn.swiglu_quant(a.float(), 200),
                lambda: Fn.rmsnorm_mod_quant(a.float(), None, None, None, 0, 1e-6, gate=a.float()),
                lambda: Fn.dequant_rows(a, sa, torch.half), lambda: Fn.dequant_rows(a, sa[:4]),
                lambda: Fn.gemm_s8(a, sa[:1], b, sb), lambda: Fn.gemm_s8(a, sa, b, sb, bias=bias[:1]),
                lambda: Fn.rmsnorm_mod_quant(a.float(), None, a[:1].float(), None, 3, 1e-6),
                lambda: Fn.rmsnorm_mod_quant(a.float(), sa, None, None, 0, 1e-6),
                lambda: Fn.rmsnorm_mod_quant(a.float(), None, None, None, 0, 1e-6, residual=b.float())):
        with pytest.raises(RuntimeError):
            bad()


def test_int8_linear():
    torch.manual_seed(3)
    lin = kpLinear(64, 48, dtype=torch.float32)
    q = Int8Linear.from_linear(lin)
    x = torch.randn(2, 5, 64)
    y, ref = q(x), torch.nn.functional.linear(x.double(), lin.weight.double(), lin.bias.double())
    assert y.shape == (2, 5, 48) and y.dtype == torch.float32
    # each factor is within half a step: |dy| <= sum |x||dw| + |w||dx|
    sx, sw = x.abs().amax(-1, keepdim=True) / 127, lin.weight.abs().amax(1) / 127
    bound = 0.5 * (x.abs().sum(-1, keepdim=True) * sw + lin.weight.abs().sum(1) * sx) + 0.25 * 64 * sx * sw + 1e-5
    assert ((y.double() - ref).abs() <= 1.01 * bound).all()
    assert (q.dequantized(torch.float32) - lin.weight).abs().max() <= 0.501 * sw.max()
    m = Int8Linear(64, 48)
    m.load_state_dict(q.state_dict())
    assert torch.equal(m(x), y)


def test_dit_int8_follows_the_dit():
    """Rounding weights and activations to 8 bits moves each product by about 1 % (a step of
    amax / 127 is uniform noise of 0.3 steps; amax is 2 to 4 sigma), ten products deep by a few."""
    m = _model()
    g = torch.Generator().manual_seed(4)
    lat = torch.randn(2, 4, 8, 8, generator=g).bfloat16()
    text = torch.randn(2, 16, 64, generator=g).bfloat16()
    t = torch.tensor([0.3, 0.8])
    q = m.int8()
    assert isinstance(q, DiTInt8) and q.int8() is q
    with torch.no_grad():
        ref = m(lat, text, t).float()
    out = q(lat, text, t)
    assert out.dtype == torch.bfloat16 and not out.requires_grad
    rel = ((out.float() - ref).norm() / ref.norm()).item()
    assert rel < 0.06, rel
    # the blocks' matrices are held in one byte a weight
    held = sum(b.numel() for n, b in q.blocks.named_buffers() if b.dtype == torch.int8)
    assert held == sum(p.numel() for n, p in m.blocks.named_parameters() if p.dim() == 2)
    assert not list(q.blocks.parameters())
    with pytest.raises(ValueError):
        _model(torch.float32).int8()


def test_sampling_with_the_int8_dit():
    m = _model()
    g = torch.Generator().manual_seed(5)
    emb = [torch.randn(16, 64, generator=g).bfloat16() for _ in range(2)]
    neg = [torch.randn(16, 64, generator=g).bfloat16() for _ in range(2)]
    lat = torch.randn(2, 4, 8, 8, generator=g)
    kw = dict(prompt_embeds=emb, negative_prompt_embeds=neg, height=64, width=64, num_inference_steps=4,
              guidance_scale=2.0, initial_latents=lat)
    ref = batch_image_inference(m, **kw)["images"].float()
    out = batch_image_inference(m.int8(), **kw)["images"].float()
    assert out.shape == ref.shape and torch.isfinite(out).all()
    assert ((out - ref).norm() / ref.norm()).item() < 0.06
