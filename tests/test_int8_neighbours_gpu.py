"""Rows and vectors that lie between NaNs: the quantisers read nothing beside them, bit for bit."""
import pytest
import torch

from harp_b200.ops import functional as Fn

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
WIDTHS = [1, 7, 8, 56, 64, 72, 128, 130, 333, 512, 1001, 1152, 1154, 1155, 1160, 1288, 1536, 2056, 2304, 2560, 2568, 4100,
          4608, 6144, 8193, 12000]


def _between_nans(t):
    """The same values with NaN beside every row, rows on the same alignment."""
    t2 = t if t.dim() == 2 else t[None]
    R, D = t2.shape
    buf = torch.full((R + 2, -(-D // 16) * 16 + 32), float("nan"), device="cuda", dtype=t.dtype)
    v = buf[1:1 + R, 16:16 + D]
    v.copy_(t2)
    return v if t.dim() == 2 else v[0]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("cols", WIDTHS)
def test_quantisers_read_their_rows_alone(cols, dt):
    t = DT[dt]
    g = torch.Generator(device="cuda").manual_seed(cols)

    def r(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)

    for batch, rpb in ((1, 1), (3, 2), (2, 9), (3, 417), (1, 2500)):
        R = batch * rpb
        x, res, w = r(R, cols), r(R, cols), r(cols)
        scale, shift, gate = (r(batch, cols, scale=0.1) for _ in range(3))
        xs, ress, ws, scales, shifts, gates = map(_between_nans, (x, res, w, scale, shift, gate))
        gu = torch.cat([x, res], 1)
        for a, b in ((Fn.quant_rows(x), Fn.quant_rows(xs)),
                     (Fn.swiglu_quant(gu, cols), Fn.swiglu_quant(_between_nans(gu), cols)),
                     (Fn.rmsnorm_mod_quant(x, w, None, None, rpb, 1e-6)[:2], Fn.rmsnorm_mod_quant(xs, ws, None, None, rpb, 1e-6)[:2]),
                     (Fn.rmsnorm_mod_quant(x, w, scale, shift, rpb, 1e-6, residual=res, gate=gate),
                      Fn.rmsnorm_mod_quant(xs, ws, scales, shifts, rpb, 1e-6, residual=ress, gate=gates))):
            for p, q in zip(a, b):
                assert torch.isfinite(p.float()).all() and torch.equal(p, q), (batch, rpb)
        q, s = Fn.quant_rows(x)
        wide = torch.full((R + 2, q.stride(0) + 16), 99, dtype=torch.int8, device="cuda")
        qs = wide[1:1 + R, :cols].copy_(q)
        for odt in DT.values():
            assert torch.equal(Fn.dequant_rows(q, s, odt), Fn.dequant_rows(qs, s, odt))
