"""8-bit rows and the int8 GEMM on the GPU against plain fp64 statements.

Tolerances:
  * int8 rows.  The kernels work in fp32 on the same inputs, so y / s is off by
    at most 2^-18 relative (the norm's statistics, modulation, exp and the scale's
    reciprocal are 2^-24 to 2^-20 each); a value can then round to the other
    neighbour, one unit away, only within 127 * 2^-18 of a boundary.  quant_rows
    repeats the CPU statement's fp32 steps and has to match it bit for bit.
  * scales: the fp64 scale to 2^-20 relative (norm statistics over <= 2^15 values).
  * GEMM: exact integer sums, then at most 4 fp32 roundings of the terms and one
    rounding to the output's type.
"""
import math

import pytest
import torch

from harp_b200.ops import functional as Fn
from harp_b200.runtime import errors

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(scope="module", autouse=True)
def _lib():
    import harp_b200

    assert harp_b200.load_native(build_if_needed=True), "CUDA library must load on a GPU box"


def _x(rows, cols, dt, seed=0, ld=None, off=0):
    """[rows, cols] with row stride ld, starting `off` elements into its storage."""
    g = torch.Generator().manual_seed(seed)
    ld = ld or cols
    buf = (torch.randn(rows * ld + off, generator=g) * torch.exp(torch.randn(1, generator=g))).to(dt).cuda()
    return buf[off:off + rows * ld].view(rows, ld)[:, :cols] if rows else torch.empty(0, cols, dtype=dt, device="cuda")


def _rows64(y):
    s = (y.abs().amax(1) / 127).clamp_min(2.0 ** -126)
    return y / s[:, None], s


def _check_rows(q, s, y64):
    v, s64 = _rows64(y64)
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and q.shape == y64.shape
    assert q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0
    if y64.numel() == 0:
        return
    assert ((s.double() - s64).abs() <= 2.0 ** -20 * s64).all()
    d = (q.double() - torch.round(v)).abs()
    assert d.max() <= 1, d.max()
    wrong = d > 0
    # only where the exact quotient is next to a boundary (half of a bf16 row's maximum lies on one: 63.5)
    frac = (v - torch.floor(v) - 0.5).abs()
    assert (frac[wrong] <= 127 * 2.0 ** -18).all(), frac[wrong].max()


SHAPES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 255), (33, 256), (7, 1001), (64, 1152), (129, 1155), (4, 2304),
          (3, 4608), (2, 6145), (2, 8200), (3, 20480), (2, 20488), (300, 384)]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quant_rows(rows, cols, dt):
    x = _x(rows, cols, DT[dt])
    q, s = Fn.quant_rows(x)
    _check_rows(q, s, x.double())
    qc, sc = Fn.quant_rows(x.cpu())  # the same fp32 steps
    assert torch.equal(q.cpu(), qc) and torch.equal(s.cpu(), sc)
    for odt in DT.values():
        v = Fn.dequant_rows(q, s, odt)
        assert torch.equal(v, (q.float() * s[:, None]).to(odt))
    assert ((Fn.dequant_rows(q, s, torch.float32).double() - x.double()).abs()
            <= s.double()[:, None] * (0.5 + 127 * 2.0 ** -22)).all()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("ld,off", [(1160, 0), (1153, 0), (1152, 1), (1155, 3), (1160, 8)])
def test_quant_rows_strided(ld, off, dt):
    x = _x(37, 1152, DT[dt], ld=ld, off=off)
    q, s = Fn.quant_rows(x)
    qc, sc = Fn.quant_rows(x.contiguous().cpu())
    assert torch.equal(q.cpu(), qc) and torch.equal(s.cpu(), sc)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_swiglu_quant(rows, cols, dt):
    gu = _x(rows, 2 * cols, DT[dt], seed=1)
    q, s = Fn.swiglu_quant(gu, cols)
    g, u = gu[:, :cols].double(), gu[:, cols:].double()
    _check_rows(q, s, g * torch.sigmoid(g) * u)


NORM_FORMS = [dict(), dict(w=1), dict(scale=1, shift=1), dict(w=1, scale=1), dict(shift=1),
              dict(res=1), dict(res=1, gate=1), dict(res=1, gate=1, scale=1, shift=1), dict(res=1, w=1, gate=1, scale=1, shift=1)]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("form", range(len(NORM_FORMS)))
@pytest.mark.parametrize("batch,rpb,cols", [(1, 1, 1), (2, 3, 8), (1, 5, 77), (3, 11, 1152), (2, 17, 1155), (1, 2, 6144),
                                            (2, 2, 8201), (1, 2, 20488), (4, 1, 2304)])
def test_rmsnorm_mod_quant(batch, rpb, cols, form, dt):
    f, t = NORM_FORMS[form], DT[dt]
    R, eps = batch * rpb, 1e-6
    x = _x(R, cols, t, seed=2)
    mod = _x(batch, 3 * cols, t, seed=3) * 0.1
    scale = mod[:, :cols] if f.get("scale") else None
    shift = mod[:, cols:2 * cols] if f.get("shift") else None
    gate = mod[:, 2 * cols:] if f.get("gate") else None
    w = _x(1, cols, t, seed=4)[0] if f.get("w") else None
    res = _x(R, cols, t, seed=5) if f.get("res") else None
    q, s, h = Fn.rmsnorm_mod_quant(x, w, scale, shift, rpb, eps, residual=res, gate=gate)
    up = lambda v: v.double().repeat_interleave(rpb, 0)  # noqa: E731
    h64 = x.double()
    if gate is not None:
        h64 = h64 * up(gate)
    if res is not None:
        h64 = h64 + res.double()
        # one fp32 product and sum, one rounding to the type
        u = 2.0 ** -8 if t == torch.bfloat16 else 2.0 ** -23
        big = res.double().abs() + (h64 - res.double()).abs()
        assert h.dtype == t and ((h.double() - h64).abs() <= u * h64.abs() + 2.0 ** -22 * big).all()
    else:
        assert h is x
    y = h64 / torch.sqrt(h64.pow(2).mean(1, keepdim=True) + eps)
    if w is not None:
        y = y * w.double()
    if scale is not None:
        y = y * (1 + up(scale))
    if shift is not None:
        y = y + up(shift)
    _check_rows(q, s, y)


WIDTHS = [1, 8, 56, 64, 72, 128, 130, 333, 334, 512, 1000, 1152, 1155, 1160, 1536, 1792, 2048, 2304, 2306, 2560, 2568,
          3001, 4100, 4101, 4608, 6144, 7000, 8193, 12000]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("cols", WIDTHS)
def test_many_rows(cols, dt):
    """Enough rows for the kernels that take few warps a row and go over several rows."""
    t, rpb, batch = DT[dt], 417, 3
    R = rpb * batch
    x, res = _x(R, cols, t, seed=6), _x(R, cols, t, seed=7)
    q, s = Fn.quant_rows(x)
    qc, sc = Fn.quant_rows(x.cpu())
    assert torch.equal(q.cpu(), qc) and torch.equal(s.cpu(), sc)
    gu = torch.cat([x, res], 1)
    g, u = x.double(), res.double()
    _check_rows(*Fn.swiglu_quant(gu, cols), g * torch.sigmoid(g) * u)
    mod = _x(batch, 6 * cols, t, seed=8) * 0.1
    scale, shift, gate = (mod[:, i * cols:(i + 1) * cols] for i in range(3))
    w = _x(1, cols, t, seed=9)[0]
    up = lambda v: v.double().repeat_interleave(rpb, 0)  # noqa: E731

    def norm(h):
        return h / torch.sqrt(h.pow(2).mean(1, keepdim=True) + 1e-6)

    q, s, _ = Fn.rmsnorm_mod_quant(x, w, None, None, 0, 1e-6)
    _check_rows(q, s, norm(x.double()) * w.double())
    h64 = res.double() + up(gate) * x.double()
    q, s, h = Fn.rmsnorm_mod_quant(x, w, scale, shift, rpb, 1e-6, residual=res, gate=gate)
    _check_rows(q, s, norm(h64) * w.double() * (1 + up(scale)) + up(shift))
    eps = 2.0 ** -8 if t == torch.bfloat16 else 2.0 ** -23
    assert ((h.double() - h64).abs() <= eps * h64.abs() + 2.0 ** -22 * (res.double().abs() + (h64 - res.double()).abs())).all()
    # samples of a few rows each
    few = mod[:1].expand(R // 3, -1)[:, :cols]
    q, s, h = Fn.rmsnorm_mod_quant(x, None, None, few, 3, 1e-6, residual=res)
    _check_rows(q, s, norm(x.double() + res.double()) + mod[:1, :cols].double())


def test_rows_special_values():
    """Zero rows, tiny rows, NaN and infinities: each row by itself."""
    x = torch.randn(8, 1152, generator=torch.Generator().manual_seed(0))
    x[1] = 0.0
    x[2] = 1e-42 * x[2].sign()
    x[3, 5] = float("nan")
    x[4, 7] = float("inf")
    x[5, 9] = -float("inf")
    x[6] = torch.finfo(torch.float32).max * x[6].sign()
    x[7, :] = 0.0
    x[7, 1151] = -3.0
    for cols in (1152, 1151, 8):
        xc = x[:, 1152 - cols:].cuda() if cols != 8 else x[:, :8].cuda()
        q, s = Fn.quant_rows(xc)
        qc, sc = Fn.quant_rows(xc.cpu().contiguous())
        assert torch.equal(q.cpu(), qc)
        assert torch.equal(torch.isnan(s.cpu()), torch.isnan(sc))
        assert torch.equal(torch.nan_to_num(s.cpu(), 0.0), torch.nan_to_num(sc, 0.0))
    q, s = Fn.quant_rows(x.cuda())
    assert (q[1] == 0).all() and s[1] == 2.0 ** -126
    for r in (3, 4, 5):
        assert torch.isnan(s[r]) and (q[r] == 0).all()
        assert torch.isnan(Fn.dequant_rows(q, s)[r]).all()
    assert (q[6].abs() == 127).all() and torch.isfinite(s[6])
    assert q[7, 1151] == -127 and (q[7, :1151] == 0).all()
    # many rows, a NaN in the modulation of one sample and in one row: nothing else is touched
    y, m = torch.randn(1200, 1155, device="cuda"), torch.zeros(2, 1155, device="cuda")
    m[1, 1154], y[5, 1154] = float("nan"), float("inf")
    q, s, _ = Fn.rmsnorm_mod_quant(y, None, m, None, 600, 1e-6, residual=y, gate=m)
    bad = torch.isnan(s)
    assert bad[600:].all() and bad[5] and bad[:600].sum() == 1 and (q[bad] == 0).all()
    # norm: a zero row gives its shift; a NaN row stays its own
    z = torch.zeros(3, 64, device="cuda")
    z[1, 3] = float("nan")
    shift = torch.linspace(-1, 1, 64, device="cuda")[None]
    q, s, _ = Fn.rmsnorm_mod_quant(z, None, None, shift, 3, 1e-6)
    ref_q, ref_s = Fn.quant_rows(shift)
    for r in (0, 2):
        assert torch.equal(q[r], ref_q[0]) and torch.equal(s[r], ref_s[0])
    assert torch.isnan(s[1]) and (q[1] == 0).all()
    # swiglu: gates far from zero on both sides
    gu = torch.tensor([[-200.0, 200.0, -50.0, 0.0, 3.0, -3.0, 2.0, 1.0]], device="cuda")
    q, s = Fn.swiglu_quant(gu, 4)
    v = torch.nn.functional.silu(gu[:, :4].double()) * gu[:, 4:].double()
    assert (q.double() * s[:, None].double() - v).abs().max() <= 0.51 * s.item()


def test_empty_rows():
    for dt in DT.values():
        x = torch.empty(0, 96, dtype=dt, device="cuda")
        q, s = Fn.quant_rows(x)
        assert q.shape == (0, 96) and s.shape == (0,)
        q, s, h = Fn.rmsnorm_mod_quant(x, None, None, None, 0, 1e-6, residual=x)
        assert q.shape == (0, 96) and h.shape == (0, 96)
        assert Fn.swiglu_quant(x, 48)[0].shape == (0, 48)
    assert Fn.dequant_rows(q, s).shape == (0, 96)


# ---------------------------------------------------------------------------
# GEMM
# ---------------------------------------------------------------------------
def _i8(rows, cols, seed, ld=None, off=0):
    g = torch.Generator().manual_seed(seed)
    ld = ld or -(-cols // 16) * 16
    buf = torch.randint(-128, 128, (rows * ld + off,), generator=g, dtype=torch.int8).cuda()
    return buf[off:].view(rows, ld)[:, :cols]


def _gemm_check(a, b, bias_dt, out_dt, seed=0, out=None):
    M, N = a.shape[0], b.shape[0]
    g = torch.Generator().manual_seed(seed)
    sa = (torch.rand(M, generator=g) + 0.01).cuda()
    sb = (torch.rand(N, generator=g) * 1e-2 + 1e-4).cuda()
    bias = torch.randn(N, generator=g).to(bias_dt).cuda() if bias_dt is not None else None
    c = Fn.gemm_s8(a, sa, b, sb, bias=bias, out_dtype=out_dt, out=out)
    torch.cuda.synchronize()
    errors.check(a.device)
    acc = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()[None, :]
    ref = acc + bias.double() if bias is not None else acc
    big = acc.abs() + (bias.double().abs() if bias is not None else 0)
    tol = 4 * 2.0 ** -24 * big
    if out_dt == torch.bfloat16:
        tol = tol + 2.0 ** -8 * ref.abs()
    assert c.dtype == out_dt and c.shape == (M, N)
    d = (c.double() - ref).abs()
    assert (d <= tol + 1e-38).all(), ((d - tol).max(), torch.nonzero(d > tol)[:4])
    return c


GEMM_SHAPES = [(1, 1, 1), (1, 24, 16), (2, 128, 128), (3, 130, 48), (4, 6912, 1152), (5, 333, 1155), (8, 1152, 4608),
               (16, 512, 256), (17, 40, 24), (31, 257, 640), (33, 1000, 1152), (64, 3456, 1152), (65, 200, 2304),
               (100, 9216, 1152), (127, 128, 6144), (128, 256, 64), (129, 384, 129), (255, 1152, 1152),
               (288, 3456, 1152), (300, 200, 136), (511, 255, 127), (512, 256, 64), (600, 300, 200),
               (1000, 1152, 1152), (1061, 1003, 1155), (2176, 4608, 1152), (4352, 1152, 4608), (768, 640, 72),
               (3000, 24, 32), (513, 9216, 512)]


@pytest.mark.parametrize("out_dt", ["bf16", "fp32"])
@pytest.mark.parametrize("M,N,K", GEMM_SHAPES)
def test_gemm_s8(M, N, K, out_dt):
    a, b = _i8(M, K, 1), _i8(N, K, 2)
    _gemm_check(a, b, None, DT[out_dt])
    _gemm_check(a, b, torch.bfloat16 if out_dt == "bf16" else torch.float32, DT[out_dt], seed=3)


@pytest.mark.parametrize("M,N,K", [(3, 200, 144), (70, 200, 144), (600, 300, 208)])
@pytest.mark.parametrize("lda,offa,ldb,offb", [(145, 0, 160, 0), (208, 0, 209, 0), (208, 1, 208, 0), (208, 16, 224, 32),
                                               (400, 0, 416, 48)])
def test_gemm_s8_strides(M, N, K, lda, offa, ldb, offb):
    lda, ldb = max(lda, K), max(ldb, K)
    a, b = _i8(M, K, 1, lda, offa), _i8(N, K, 2, ldb, offb)
    _gemm_check(a, b, torch.bfloat16, torch.bfloat16)
    # a strided output, odd offset: nothing outside of it is written
    buf = torch.full((M, N + 13), 7.0, device="cuda", dtype=torch.bfloat16)
    _gemm_check(a, b, None, torch.bfloat16, out=buf[:, 5:5 + N])
    assert (buf[:, :5] == 7).all() and (buf[:, 5 + N:] == 7).all()


@pytest.mark.parametrize("M,N", [(1, 40), (40, 200), (200, 150), (600, 260)])
def test_gemm_s8_zero_k_and_extremes(M, N):
    _gemm_check(_i8(M, 0, 1, 16), _i8(N, 0, 2, 16), torch.bfloat16, torch.float32)
    K = 8192  # all -128: the largest sums
    a = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    b = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
    b[::2] = 127
    _gemm_check(a, b, None, torch.float32)


def test_gemm_s8_empty_and_longest_k():
    one = torch.ones(1, device="cuda")
    a = torch.zeros(0, 64, dtype=torch.int8, device="cuda")
    b = torch.zeros(3, 64, dtype=torch.int8, device="cuda")
    assert Fn.gemm_s8(a, one[:0], b, torch.ones(3, device="cuda")).shape == (0, 3)
    assert Fn.gemm_s8(b, torch.ones(3, device="cuda"), a, one[:0]).shape == (3, 0)
    K = 131071
    a = torch.full((1, K), -128, dtype=torch.int8, device="cuda")
    c = Fn.gemm_s8(a, one, a, one, out_dtype=torch.float32)
    assert c.item() == float(torch.tensor(16384.0 * K))


def test_gemm_s8_nan_scale_stays_in_its_row():
    a, b = _i8(300, 256, 1), _i8(260, 256, 2)
    sa, sb = torch.ones(300, device="cuda"), torch.ones(260, device="cuda")
    sa[7] = float("nan")
    c = Fn.gemm_s8(a, sa, b, sb)
    assert torch.isnan(c[7]).all() and torch.isfinite(c[:7]).all() and torch.isfinite(c[8:]).all()


def test_gemm_s8_bit_identical_and_streams():
    a, b = _i8(200, 4608, 1), _i8(1152, 4608, 2)
    sa, sb = torch.rand(200, device="cuda"), torch.rand(1152, device="cuda")
    c = [Fn.gemm_s8(a[:m], sa[:m], b, sb) for m in (1, 4, 40, 200) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c2 = Fn.gemm_s8(a, sa, b, sb)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(c[-1], c2)
    for i in range(0, 8, 2):
        assert torch.equal(c[i], c[i + 1])
        assert torch.equal(c[i], c2[: c[i].shape[0]])  # exact sums: no dependence on the kernel chosen


def test_refusals():
    x = torch.zeros(4, 32, device="cuda")
    i8 = torch.zeros(4, 32, dtype=torch.int8, device="cuda")
    s4 = torch.ones(4, device="cuda")
    bad = [
        lambda: Fn.quant_rows(x.half()), lambda: Fn.quant_rows(x[0]), lambda: Fn.quant_rows(x[:, :0]),
        lambda: Fn.quant_rows(x.t()),
        lambda: Fn.swiglu_quant(x, 15), lambda: Fn.swiglu_quant(x.double(), 16),
        lambda: Fn.rmsnorm_mod_quant(x, torch.ones(31, device="cuda"), None, None, 4, 1e-6),
        lambda: Fn.rmsnorm_mod_quant(x, torch.ones(32, device="cuda").bfloat16(), None, None, 4, 1e-6),
        lambda: Fn.rmsnorm_mod_quant(x, None, x[:1], None, 3, 1e-6),
        lambda: Fn.rmsnorm_mod_quant(x, None, x[:1], None, 0, 1e-6),
        lambda: Fn.rmsnorm_mod_quant(x, None, x[:2], None, 4, 1e-6),
        lambda: Fn.rmsnorm_mod_quant(x, None, None, None, 4, 1e-6, gate=x[:1]),
        lambda: Fn.rmsnorm_mod_quant(x, None, None, None, 4, 1e-6, residual=x.bfloat16()),
        lambda: Fn.rmsnorm_mod_quant(x, None, None, None, 4, 1e-6, residual=x[:3]),
        lambda: Fn.rmsnorm_mod_quant(x, None, x[:1].cpu(), None, 4, 1e-6),
        lambda: Fn.dequant_rows(x, s4), lambda: Fn.dequant_rows(i8, s4[:3]), lambda: Fn.dequant_rows(i8, s4, torch.half),
        lambda: Fn.gemm_s8(x, s4, i8, s4), lambda: Fn.gemm_s8(i8, s4[:3], i8, s4), lambda: Fn.gemm_s8(i8, s4, i8, s4.double()),
        lambda: Fn.gemm_s8(i8, s4, i8[:, :31], s4), lambda: Fn.gemm_s8(i8, s4, i8, s4, bias=s4[:3]),
        lambda: Fn.gemm_s8(i8, s4, i8, s4, bias=s4.half()), lambda: Fn.gemm_s8(i8, s4, i8, s4, out_dtype=torch.half),
        lambda: Fn.gemm_s8(i8, s4, i8, s4, out=torch.zeros(4, 5, device="cuda")),
        lambda: Fn.gemm_s8(i8.t(), s4, i8.t(), s4), lambda: Fn.gemm_s8(i8, s4, i8, s4.cpu()),
        lambda: Fn.gemm_s8(torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), s4[:1],
                           torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), s4[:1]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            raise AssertionError(f"case {i} was taken")
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------
# the layer and the model that use them
# ---------------------------------------------------------------------------
def test_int8_linear_cuda_matches_cpu():
    """Same bits in, exact products: outputs differ by the fp32 rounding of the last step only."""
    from harp_b200.ops.modules import Int8Linear, kpLinear

    torch.manual_seed(0)
    lin = kpLinear(200, 136, dtype=torch.float32)
    x = torch.randn(3, 50, 200)
    ref = Int8Linear.from_linear(lin)(x)
    out = Int8Linear.from_linear(lin.cuda())(x.cuda())
    assert out.shape == ref.shape and ((out.cpu() - ref).abs() <= 2.0 ** -21 * (ref.abs() + 1)).all()
    xs = x.cuda().transpose(0, 1)  # not contiguous
    assert torch.equal(Int8Linear.from_linear(lin)(xs), out.transpose(0, 1))


def _dit(seed=0):
    from harp_b200.models import dit as D

    torch.manual_seed(seed)
    m = D.DiT(D.PRESETS["small"])
    with torch.no_grad():
        for n, p in m.named_parameters():
            p.normal_(0, 0.02 if "adaLN" in n else 0.05)
            if "norm" in n:
                p.add_(1.0)
    return m.bfloat16()


@pytest.mark.parametrize("B,L,T", [(2, 16, 32), (1, 8, 5), (3, 34, 77)])
def test_dit_int8_cuda_matches_cpu(B, L, T):
    """The same model run through the CPU restatements; bf16 activations, as in the other models' test."""
    import copy

    m = _dit()
    g = torch.Generator().manual_seed(1)
    lat = torch.randn(B, 16, L, L, generator=g).bfloat16()
    text = torch.randn(B, T, 384, generator=g).bfloat16()
    t = torch.rand(B, generator=g)
    ref = m.int8()(lat, text, t).float()
    q = copy.deepcopy(m).cuda().int8()
    out = q(lat.cuda(), text.cuda(), t.cuda())
    torch.cuda.synchronize()
    errors.check(out.device)
    assert ((out.float().cpu() - ref).norm() / ref.norm()).item() < 3e-2
    # and it follows the bf16 model (about 1 % a product)
    with torch.no_grad():
        full = m.cuda()(lat.cuda(), text.cuda(), t.cuda())
    assert ((out - full).float().norm() / full.float().norm()).item() < 6e-2


def test_sampling_with_the_int8_dit():
    from harp_b200.inference import batch_image_inference

    m = _dit().cuda()
    g = torch.Generator().manual_seed(2)
    emb = [torch.randn(32, 384, generator=g).bfloat16().cuda() for _ in range(2)]
    lat = torch.randn(2, 16, 16, 16, generator=g).cuda()
    kw = dict(prompt_embeds=emb, height=128, width=128, num_inference_steps=4, initial_latents=lat)
    ref = batch_image_inference(m, **kw)["images"].float()
    out = batch_image_inference(m.int8(), **kw)["images"].float()
    assert torch.isfinite(out).all() and ((out - ref).norm() / ref.norm()).item() < 6e-2


def test_dependent_launches_are_ordered():
    """The kernels may start before the one ahead of them on the stream has finished; what they read and
    write has to be as if they had not: a chain through the same buffers, against one with a wait after
    every step.  Exact integer sums make both bit-identical."""
    g = torch.Generator().manual_seed(7)
    for M, N in ((3, 1152), (288, 1152), (1100, 1152), (5000, 1152)):
        x0 = torch.randn(M, N, generator=g).bfloat16().cuda()
        w = [Fn.quant_rows(torch.randn(N, N, generator=g).cuda() * N ** -0.5) for _ in range(3)]

        def chain(wait):
            x, h = x0.clone(), x0.clone()
            out = torch.empty_like(x)
            for i in range(30):
                q, s, h = Fn.rmsnorm_mod_quant(x, None, None, None, M, 1e-6, residual=h)
                wait()
                Fn.gemm_s8(q, s, *w[i % 3], out=out)
                wait()
                q, s = Fn.quant_rows(out)
                wait()
                Fn.gemm_s8(q, s, *w[(i + 1) % 3], out=out)  # over the rows just quantised
                wait()
                x = out if i % 2 else out.clone()  # now and then a kernel launched in the ordinary way
                wait()
            return x.clone(), h

        a = chain(torch.cuda.synchronize)
        b = chain(lambda: None)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c = chain(lambda: None)
        for t in c:
            t.zero_()
        graph.replay()
        graph.replay()
        assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])
    errors.check(x0.device)


def test_offsets_past_32_bits():
    """Rows whose element offsets pass 2^31: the last ones against the same rows by themselves."""
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB")
    R, D = 2_097_400, 1032  # 2.16e9 values
    x = torch.empty(R, D, dtype=torch.bfloat16, device="cuda")
    tail = slice(R - 7, R)
    x[: R - 7] = 1.0
    x[tail] = _x(7, D, torch.bfloat16, seed=3)
    q, s = Fn.quant_rows(x)
    qt, st = Fn.quant_rows(x[tail])
    assert torch.equal(q[tail], qt) and torch.equal(s[tail], st) and (q[:7] == 127).all() and (q[R // 2] == 127).all()
    assert torch.equal(Fn.dequant_rows(q, s)[tail], Fn.dequant_rows(qt, st))
    w = _x(1, D, torch.bfloat16, seed=4)[0]
    q, s, h = Fn.rmsnorm_mod_quant(x, w, None, None, 0, 1e-6, residual=x)
    y = x[tail].double() * 2
    _check_rows(q[tail], s[tail], y / torch.sqrt(y.pow(2).mean(1, keepdim=True) + 1e-6) * w.double())
    assert torch.equal(h[tail], (x[tail].float() * 2).bfloat16())
    q, s = Fn.swiglu_quant(x, D // 2)
    qt, st = Fn.swiglu_quant(x[tail], D // 2)
    assert torch.equal(q[tail], qt) and torch.equal(s[tail], st)
    del x, q, s, h
    M, N = 240_000, 9216  # 2.2e9 results
    a, b = _i8(M, 32, 1), _i8(N, 32, 2)
    sa, sb = torch.rand(M, device="cuda"), torch.rand(N, device="cuda")
    c = Fn.gemm_s8(a, sa, b, sb)
    assert torch.equal(c[-9:], Fn.gemm_s8(a[-9:], sa[-9:], b, sb)) and torch.equal(c[:9], Fn.gemm_s8(a[:9], sa[:9], b, sb))
    c = Fn.gemm_s8(a, sa, b[:1], sb[:1])  # one channel: the rows kernel or narrow pairs
    ref = (a.double() @ b[:1].double().t()) * sa.double()[:, None] * sb[:1].double()
    assert ((c.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-30).all()
    errors.check(a.device)


def test_results_can_be_saved(tmp_path):
    """What the quantisers return are tensors of their own: saved, loaded and copied like any."""
    import copy

    from harp_b200.ops.modules import Int8Linear, kpLinear

    q, s = Fn.quant_rows(_x(5, 1155, torch.bfloat16))
    torch.save({"q": q, "s": s}, tmp_path / "rows.pt")
    d = torch.load(tmp_path / "rows.pt")
    assert torch.equal(d["q"], q) and torch.equal(d["s"], s)
    m = Int8Linear.from_linear(kpLinear(72, 40, dtype=torch.float32).cuda())
    torch.save(m.state_dict(), tmp_path / "linear.pt")
    n = Int8Linear(72, 40, device="cuda")
    n.load_state_dict(torch.load(tmp_path / "linear.pt"))
    x = _x(9, 72, torch.float32, seed=1)
    assert torch.equal(m(x), n(x)) and torch.equal(m(x), copy.deepcopy(m)(x))
