"""What gemm_s8 does for operands that TMA cannot address and for an empty sum, it does in kernels of its own
(each adds to the launch count)."""
import pytest
import torch

from harp_b200.ops import functional as Fn
from harp_b200.runtime import errors

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _lib():
    import harp_b200

    assert harp_b200.load_native(build_if_needed=True), "CUDA library must load on a GPU box"


def _count(f):
    torch.ops.harp.reset_launch_count()
    out = f()
    torch.cuda.synchronize()
    return int(torch.ops.harp.launch_count()), out


def _i8(rows, cols, ld, off, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.randint(-128, 128, (rows * ld + off,), generator=g, dtype=torch.int8, device="cuda")
    return buf[off:].view(rows, ld)[:, :cols]


@pytest.mark.parametrize("K", [1, 3, 16, 20, 129, 385, 1152])
@pytest.mark.parametrize("pad,off", [(0, 1), (1, 0), (4, 0), (8, 4), (3, 16), (12, 2)])
@pytest.mark.parametrize("M,N", [(1, 40), (5, 1), (70, 200), (700, 300)])
def test_unaddressable_operands(M, N, K, pad, off):
    a, b = _i8(M, K, K + pad, off, 1), _i8(N, K, K + pad, off, 2)
    sa, sb = torch.rand(M, device="cuda") + 0.1, torch.rand(N, device="cuda") + 0.1

    def copies(t):
        return int(t.data_ptr() % 16 != 0 or (t.shape[0] > 1 and t.stride(0) % 16 != 0))

    n, c = _count(lambda: Fn.gemm_s8(a, sa, b, sb, out_dtype=torch.float32))
    assert n == 1 + copies(a) + copies(b)
    acc = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()
    assert ((c.double() - acc).abs() <= 4 * 2.0 ** -24 * acc.abs()).all()
    errors.check(a.device)


def test_repeated_rows():
    a, b = _i8(1, 100, 100, 0, 1).expand(33, 100), _i8(40, 100, 112, 0, 2)
    one, sb = torch.ones(33, device="cuda"), torch.ones(40, device="cuda")
    n, c = _count(lambda: Fn.gemm_s8(a, one, b, sb, out_dtype=torch.float32))
    assert n == 2 and torch.equal(c, (a.double() @ b.double().t()).float())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bias_dt", [None, torch.bfloat16, torch.float32])
def test_empty_sum(dt, bias_dt):
    """Of no terms the sum is zero, so the output is the bias; a row or channel whose scale is NaN is NaN, and large
    scales do not make one."""
    M, N = 300, 77
    a, b = torch.empty(M, 0, dtype=torch.int8, device="cuda"), torch.empty(N, 0, dtype=torch.int8, device="cuda")
    sa, sb = torch.full((M,), 1e30, device="cuda"), torch.full((N,), 1e30, device="cuda")
    sa[7] = sb[9] = float("nan")
    bias = torch.randn(N, device="cuda").to(bias_dt) if bias_dt is not None else None
    buf = torch.full((M, N + 5), 7.0, device="cuda", dtype=dt)
    n, c = _count(lambda: Fn.gemm_s8(a, sa, b, sb, bias=bias, out=buf[:, 2:2 + N]))
    assert n == 1
    ref = torch.zeros(M, N, device="cuda") if bias is None else bias.float().expand(M, N).clone()
    ref[7] = ref[:, 9] = float("nan")
    torch.testing.assert_close(c, ref.to(dt), rtol=0, atol=0, equal_nan=True)
    assert (buf[:, :2] == 7).all() and (buf[:, 2 + N:] == 7).all()
    cpu = Fn.gemm_s8(a.cpu(), sa.cpu(), b.cpu(), sb.cpu(), bias=None if bias is None else bias.cpu(), out_dtype=dt)
    torch.testing.assert_close(c.cpu(), cpu, rtol=0, atol=0, equal_nan=True)
