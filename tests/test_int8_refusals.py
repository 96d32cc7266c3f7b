"""The CPU statements of the int8 operators take and refuse what the kernels take and refuse."""
import pytest
import torch

from harp_b200.ops import functional as Fn

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _args(dev):
    x = torch.ones(4, 32, device=dev)
    return dict(x=x, i8=torch.ones(4, 32, dtype=torch.int8, device=dev), s=torch.ones(4, device=dev),
                v=torch.ones(1, 32, device=dev), w=torch.ones(32, device=dev),
                wide=torch.ones(4, 64, device=dev), i8w=torch.ones(4, 64, dtype=torch.int8, device=dev),
                s8=torch.ones(8, device=dev))


REFUSED = {
    # rows: type, dimensions, columns, inner stride
    "rows fp16": lambda x, **k: Fn.quant_rows(x.half()),
    "rows fp64": lambda x, **k: Fn.quant_rows(x.double()),
    "rows 1-D": lambda x, **k: Fn.quant_rows(x[0]),
    "rows 3-D": lambda x, **k: Fn.quant_rows(x[None]),
    "rows no columns": lambda x, **k: Fn.quant_rows(x[:, :0]),
    "rows transposed": lambda x, **k: Fn.quant_rows(x.t()),
    "rows every second": lambda wide, **k: Fn.quant_rows(wide[:, ::2]),
    "swiglu transposed": lambda x, **k: Fn.swiglu_quant(x.t(), 2),
    "swiglu width": lambda x, **k: Fn.swiglu_quant(x, 15),
    "dequant fp32 rows": lambda x, s, **k: Fn.dequant_rows(x, s),
    "dequant transposed": lambda i8, s, **k: Fn.dequant_rows(i8.t(), torch.ones(32, device=i8.device)),
    "dequant bf16 scale": lambda i8, s, **k: Fn.dequant_rows(i8, s.bfloat16()),
    "dequant 2-D scale": lambda i8, s, **k: Fn.dequant_rows(i8, s[:, None]),
    "dequant strided scale": lambda i8, s8, **k: Fn.dequant_rows(i8, s8[::2]),
    "dequant output type": lambda i8, s, **k: Fn.dequant_rows(i8, s, torch.half),
    # norm
    "norm transposed": lambda x, **k: Fn.rmsnorm_mod_quant(x.t(), None, None, None, 0, 1e-6),
    "norm strided w": lambda x, wide, **k: Fn.rmsnorm_mod_quant(x, wide[0, ::2], None, None, 0, 1e-6),
    "norm 2-D w": lambda x, v, **k: Fn.rmsnorm_mod_quant(x, v, None, None, 0, 1e-6),
    "norm w type": lambda x, w, **k: Fn.rmsnorm_mod_quant(x, w.bfloat16(), None, None, 0, 1e-6),
    "norm strided scale": lambda x, wide, **k: Fn.rmsnorm_mod_quant(x, None, wide[:1, ::2], None, 4, 1e-6),
    "norm strided shift": lambda x, wide, **k: Fn.rmsnorm_mod_quant(x, None, None, wide[:1, ::2], 4, 1e-6),
    "norm 1-D shift": lambda x, w, **k: Fn.rmsnorm_mod_quant(x, None, None, w, 4, 1e-6),
    "norm scale type": lambda x, v, **k: Fn.rmsnorm_mod_quant(x, None, v.bfloat16(), None, 4, 1e-6),
    "norm batch": lambda x, v, **k: Fn.rmsnorm_mod_quant(x, None, v, None, 3, 1e-6),
    "norm no rows a sample": lambda x, v, **k: Fn.rmsnorm_mod_quant(x, None, v, None, 0, 1e-6),
    "norm strided residual": lambda x, wide, **k: Fn.rmsnorm_mod_quant(x, None, None, None, 0, 1e-6, residual=wide[:, ::2]),
    "norm residual type": lambda x, **k: Fn.rmsnorm_mod_quant(x, None, None, None, 0, 1e-6, residual=x.bfloat16()),
    "norm residual shape": lambda x, **k: Fn.rmsnorm_mod_quant(x, None, None, None, 0, 1e-6, residual=x[:3]),
    "norm gate alone": lambda x, v, **k: Fn.rmsnorm_mod_quant(x, None, None, None, 4, 1e-6, gate=v),
    "norm strided gate": lambda x, wide, **k: Fn.rmsnorm_mod_quant(x, None, None, None, 4, 1e-6, residual=x,
                                                                   gate=wide[:1, ::2]),
    # product
    "gemm a type": lambda x, i8, s, **k: Fn.gemm_s8(x, s, i8, s),
    "gemm b type": lambda x, i8, s, **k: Fn.gemm_s8(i8, s, x, s),
    "gemm 1-D a": lambda i8, s, **k: Fn.gemm_s8(i8[0], s[:1], i8, s),
    "gemm 3-D a": lambda i8, s, **k: Fn.gemm_s8(i8[None], s, i8, s),
    "gemm 1-D b": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8[0], s),
    "gemm K": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8[:, :31], s),
    "gemm long K": lambda i8, s, **k: Fn.gemm_s8(i8[:1, :1].expand(1, 131072).contiguous(), s[:1],
                                                 i8[:1, :1].expand(1, 131072).contiguous(), s[:1]),
    "gemm transposed a": lambda i8, s, **k: Fn.gemm_s8(i8.t(), torch.ones(32, device=i8.device), i8[:, :4], s),
    "gemm strided b": lambda i8, i8w, s, **k: Fn.gemm_s8(i8, s, i8w[:, ::2], s),
    "gemm bf16 a_scale": lambda i8, s, **k: Fn.gemm_s8(i8, s.bfloat16(), i8, s),
    "gemm fp64 a_scale": lambda i8, s, **k: Fn.gemm_s8(i8, s.double(), i8, s),
    "gemm bf16 b_scale": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8, s.bfloat16()),
    "gemm fp64 b_scale": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8, s.double()),
    "gemm 2-D scale": lambda i8, s, **k: Fn.gemm_s8(i8, s[:, None], i8, s),
    "gemm strided scale": lambda i8, s8, s, **k: Fn.gemm_s8(i8, s8[::2], i8, s),
    "gemm short scale": lambda i8, s, **k: Fn.gemm_s8(i8, s[:1], i8, s),
    "gemm fp16 bias": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8, s, bias=s.half()),
    "gemm fp64 bias": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8, s, bias=s.double()),
    "gemm int8 bias": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8, s, bias=i8[0, :4]),
    "gemm 2-D bias": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8, s, bias=s[None]),
    "gemm strided bias": lambda i8, s, s8, **k: Fn.gemm_s8(i8, s, i8, s, bias=s8[::2]),
    "gemm short bias": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8, s, bias=s[:1]),
    "gemm out_dtype": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8, s, out_dtype=torch.half),
    "gemm out type": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8, s, out=torch.empty(4, 4, device=i8.device).half()),
    "gemm out rows": lambda i8, s, **k: Fn.gemm_s8(i8[:1], s[:1], i8, s, out=torch.empty(4, 4, device=i8.device)),
    "gemm out columns": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8[:1], s[:1], out=torch.empty(4, 4, device=i8.device)),
    "gemm out transposed": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8[:3], s[:3], out=torch.empty(3, 4, device=i8.device).t()),
    "gemm out of one row repeated": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8, s, out=torch.empty(1, 4, device=i8.device).expand(4, 4)),
    "gemm out with overlapping rows": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8, s, out=torch.empty(16, device=i8.device).as_strided(
        (4, 4), (3, 1))),
    "gemm out of one column repeated": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8[:1], s[:1], out=torch.empty(
        1, device=i8.device).as_strided((4, 1), (0, 1))),
    "gemm 1-D out": lambda i8, s, **k: Fn.gemm_s8(i8[:1], s[:1], i8, s, out=torch.empty(4, device=i8.device)),
}

TAKEN = {
    "rows in a wider matrix": lambda wide, **k: Fn.quant_rows(wide[:, 3:20]),
    "rows repeated": lambda v, **k: Fn.quant_rows(v.expand(5, 32)),
    "one column of many": lambda wide, **k: Fn.quant_rows(wide[:, 7:8]),
    "vectors of one product": lambda x, wide, **k: Fn.rmsnorm_mod_quant(x, None, wide[:2, :32], wide[:2, 32:], 2, 1e-6),
    "one scale of many": lambda i8, s8, s, **k: Fn.gemm_s8(i8[:1], s8[::2][:1], i8, s),
    "bf16 bias, fp32 output": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8, s, bias=s.bfloat16(), out_dtype=torch.float32),
    "fp32 bias, bf16 output": lambda i8, s, **k: Fn.gemm_s8(i8, s, i8, s, bias=s),
    "output in a wider matrix": lambda i8, s, wide, **k: Fn.gemm_s8(i8, s, i8, s, out=wide[:, 9:13]),
    "output of one row": lambda i8, s, **k: Fn.gemm_s8(i8[:1], s[:1], i8, s, out=torch.empty(1, 4, device=i8.device).as_strided((1, 4), (2, 1))),
    "output of every second row": lambda i8, s, wide, **k: Fn.gemm_s8(i8[:2], s[:2], i8, s, out=wide[::2, :4]),
    "K of zero": lambda i8, s, **k: Fn.gemm_s8(i8[:, :0], s, i8[:, :0], s, bias=s),
}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("what", REFUSED)
def test_refused(what, device):
    with pytest.raises(RuntimeError):
        REFUSED[what](**_args(device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("what", TAKEN)
def test_taken(what, device):
    out = TAKEN[what](**_args(device))
    out = out if isinstance(out, tuple) else (out,)
    assert all(torch.isfinite(t.float()).all() for t in out)
