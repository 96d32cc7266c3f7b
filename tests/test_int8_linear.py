"""Int8Linear as a module: conversions, moves and inputs that any linear layer takes."""
import pytest
import torch

from harp_b200.ops import functional as Fn
from harp_b200.ops.modules import Int8Linear, kpLinear

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _layer(i=100, o=40, bias=True, device="cpu"):
    torch.manual_seed(0)
    return Int8Linear.from_linear(kpLinear(i, o, bias=bias, dtype=torch.float32).to(device))


def _x(*shape, dtype=torch.float32, device="cpu"):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(1)).to(device, dtype)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("how", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(),
                                 lambda m: m.bfloat16().float(), lambda m: torch.nn.Sequential(m).half()[0]])
@pytest.mark.parametrize("bias", [True, False])
def test_dtype_conversions_keep_the_scales(device, how, bias):
    m, x = _layer(bias=bias, device=device), _x(7, 100, device=device)
    scale, y = m.weight_scale.clone(), m(x)
    m = how(m)
    assert m.weight_q.dtype == torch.int8 and m.weight_scale.dtype == torch.float32
    assert torch.equal(m.weight_scale, scale) and m.weight_scale.device == x.device
    assert not bias or m.bias.dtype in (torch.bfloat16, torch.float32)
    # at most the bias is rounded, once, to bf16's 8 bits
    b = m.bias.float() if bias else torch.zeros(())
    assert ((m(x) - y).abs() <= 2.0 ** -8 * b.abs().to(x.device) + 2.0 ** -22 * y.abs()).all()


def _padded(q):
    return q.stride(1) == 1 and q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("i", [1, 100, 1155, 64])
def test_rows_stay_on_16_byte_boundaries(device, i):
    """What the int8 product reads in place: a layer that is built on the CPU, moved or copied keeps its rows there."""
    import copy

    m, x = _layer(i), _x(3, i)
    y = m(x)
    assert _padded(m.weight_q)
    w = m.weight_q.clone()
    for move in (lambda m: m.to(device), lambda m: m.cpu().to(device), copy.deepcopy, lambda m: m.to(torch.bfloat16)):
        m = move(m)
        assert m.weight_q.shape == (40, i) and _padded(m.weight_q) and torch.equal(m.weight_q.cpu(), w)
    m = m.to("meta").to_empty(device=device)
    assert m.weight_q.shape == (40, i) and _padded(m.weight_q)
    m = Int8Linear(i, 40)
    m.load_state_dict(_layer(i).state_dict())
    assert _padded(m.weight_q) and torch.equal(m(x), y)
    assert _padded(m.to(device).weight_q)


@pytest.mark.parametrize("device", DEVICES)
def test_inputs_and_weights_of_any_stride(device):
    """A transposed view as input (one sample of [B, C, L] seen as [B, L, C], a transposed matrix) or as weight."""
    m = _layer(100, 40, device=device)
    for x in (_x(1, 100, 6, device=device).transpose(1, 2), _x(100, 6, device=device).t(),
              _x(2, 100, 6, device=device).transpose(1, 2), _x(5, 200, device=device)[:, ::2],
              _x(6, 1, device=device).expand(6, 100)):
        assert torch.equal(m(x), m(x.contiguous()))
    w = _x(100, 40, device=device)
    n = Int8Linear.from_weight(w.t())
    ref = Int8Linear.from_weight(w.t().contiguous())
    assert torch.equal(n.weight_q, ref.weight_q) and torch.equal(n.weight_scale, ref.weight_scale)
