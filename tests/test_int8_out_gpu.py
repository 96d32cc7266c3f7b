"""gemm_s8 into a part of a larger matrix: nothing beside the part is written, whatever its width."""
import pytest
import torch

from harp_b200.ops import functional as Fn
from harp_b200.runtime import errors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(40, 64), (700, 385), (8704, 385), (12001, 1155)])
@pytest.mark.parametrize("N", [120, 121, 122, 124, 127, 129, 193, 513, 1003])
def test_what_lies_beside_the_output_stays(M, N, K, dt):
    g = torch.Generator(device="cuda").manual_seed(0)
    a, b = (torch.randint(-128, 128, (r, K), generator=g, dtype=torch.int8, device="cuda") for r in (M, N))
    sa, sb = torch.rand(M, generator=g, device="cuda"), torch.rand(N, generator=g, device="cuda")
    ref = Fn.gemm_s8(a, sa, b, sb, out_dtype=dt)
    for at in (16, 5):  # rows on 16-byte boundaries, and not
        buf = torch.full((M + 2, -(-N // 16) * 16 + 32 + (at == 5)), 7.0, device="cuda", dtype=dt)
        c = Fn.gemm_s8(a, sa, b, sb, out=buf[1:1 + M, at:at + N])
        assert torch.equal(c, ref)
        assert (buf[0] == 7).all() and (buf[1 + M:] == 7).all()
        assert (buf[:, :at] == 7).all() and (buf[:, at + N:] == 7).all()
    errors.check(a.device)
