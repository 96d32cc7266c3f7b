"""The int8 kernels back to back: what each reads was written by the kernel just ahead of it."""
import pytest
import torch

from harp_b200.ops import functional as Fn
from harp_b200.runtime import errors

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("B,S", [(1, 3), (2, 144), (4, 275), (2, 2500)])
def test_modulation_gate_weight_and_bias_of_the_kernel_just_before(B, S, dt):
    """A block's chain in which the modulation, the gate, the norm's weight, the product's bias and every scale are
    results of the launch ahead of their reader, in buffers that hold the last round's values until then: with no
    wait in between, from a graph, and with a wait after every step, bit for bit the same (exact integer sums)."""
    t, N, R = DT[dt], 1152, B * S
    g = torch.Generator().manual_seed(11)
    a0 = torch.randn(R, N, generator=g).to(t).cuda()
    wada = Fn.quant_rows(torch.randn(6 * N, N, generator=g).cuda() * (0.1 * N ** -0.5))
    wvec = Fn.quant_rows(torch.randn(N, N, generator=g).cuda() * N ** -0.5)
    w = [Fn.quant_rows(torch.randn(N, N, generator=g).cuda() * N ** -0.5) for _ in range(2)]

    def chain(wait):
        a, x = a0.clone(), a0.clone()
        mod = torch.zeros(B, 6 * N, device="cuda", dtype=t)
        vec = torch.zeros(1, N, device="cuda", dtype=t)
        kept = []
        for i in range(12):
            c8 = Fn.quant_rows(a.view(B, S, N)[:, 0])
            wait()
            Fn.gemm_s8(*c8, *wada, out=mod)
            wait()
            sh, sc, gate = (mod[:, k * N:(k + 1) * N] for k in range(3))
            q, s, x = Fn.rmsnorm_mod_quant(a, None, sc, sh, S, 1e-6, residual=x, gate=gate)
            wait()
            kept.append(Fn.dequant_rows(q, s, t))
            wait()
            Fn.gemm_s8(q[:1], s[:1], *wvec, out=vec)
            wait()
            Fn.gemm_s8(q, s, *w[i % 2], bias=vec[0], out=a)
            wait()
            Fn.gemm_s8(q[-1:], s[-1:], *wvec, out=vec)
            wait()
            q, s, _ = Fn.rmsnorm_mod_quant(a, vec[0], None, None, S, 1e-6)
            wait()
            Fn.gemm_s8(q, s, *w[1 - i % 2], out=a)
            wait()
        return a, x, torch.stack(kept)

    ref = chain(torch.cuda.synchronize)
    out = chain(lambda: None)
    assert all(torch.isfinite(r.float()).all() for r in ref)
    assert all(torch.equal(p, q) for p, q in zip(ref, out))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(lambda: None)
    for p in out:
        p.zero_()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(ref, out))
    errors.check(a0.device)
