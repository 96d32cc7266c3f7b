"""No gradient passes a rounding to 8 bits: results carry none, on the CPU as on CUDA, whatever the inputs carry."""
import pytest
import torch

from harp_b200.ops import functional as Fn
from harp_b200.ops.modules import Int8Linear

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _p(*shape, device, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(0)).to(device, dtype).requires_grad_()


@pytest.mark.parametrize("device", DEVICES)
def test_results_carry_no_gradient(device):
    x, gu, mod, w = _p(6, 32, device=device), _p(6, 64, device=device), _p(2, 32, device=device), _p(32, device=device)
    q, s = Fn.quant_rows(x)
    outs = [q, s, *Fn.swiglu_quant(gu, 32), *Fn.rmsnorm_mod_quant(x, w, mod, mod, 3, 1e-6, residual=x, gate=mod),
            *Fn.rmsnorm_mod_quant(x, w, mod, mod, 3, 1e-6)[:2]]
    sp = s.clone().requires_grad_()
    outs += [Fn.dequant_rows(q, sp, torch.float32), Fn.gemm_s8(q, sp, q, sp, bias=_p(6, device=device))]
    out = torch.zeros(6, 6, device=device)
    outs.append(Fn.gemm_s8(q, sp, q, sp, bias=_p(6, device=device), out=out))
    layer = Int8Linear.from_weight(_p(5, 32, device=device), _p(5, device=device))
    outs += [layer(x), layer.rows(q, sp), layer.dequantized()]
    for i, t in enumerate(outs):
        assert not t.requires_grad and t.grad_fn is None, i
    # without a residual h is x itself, not a copy
    assert Fn.rmsnorm_mod_quant(x, w, None, None, 0, 1e-6)[2] is x
