"""What the int8 DiT holds of the model it was built from, and its sequence-parallel forward."""
import pytest
import torch

from harp_b200.models.dit import DiT, DiTConfig

CFG = DiTConfig(in_channels=4, hidden=96, depth=2, heads=2, mlp_ratio=4.0, text_dim=64, axes_dims=(16, 16, 16))


def _model():
    torch.manual_seed(0)
    m = DiT(CFG)
    with torch.no_grad():
        for n, p in m.named_parameters():
            p.normal_(0, 0.02 if "adaLN" in n else 0.08)
            if "norm" in n:
                p.add_(1.0)
    return m.bfloat16()


def _inputs():
    g = torch.Generator().manual_seed(1)
    return (torch.randn(2, 4, 8, 8, generator=g).bfloat16(), torch.randn(2, 16, 64, generator=g).bfloat16(),
            torch.tensor([0.3, 0.8]))


def test_the_blocks_hold_nothing_of_the_model_they_were_built_from():
    """A step that changes the model's blocks afterwards changes nothing in the int8 ones."""
    m = _model()
    q = m.int8()
    theirs = {p.untyped_storage().data_ptr() for p in m.blocks.parameters()}
    assert not [n for n, b in q.blocks.named_buffers() if b.untyped_storage().data_ptr() in theirs]
    before = q(*_inputs())
    with torch.no_grad():
        for p in m.blocks.parameters():
            p.mul_(-3.0).add_(0.5)
    assert torch.equal(q(*_inputs()), before)


@pytest.mark.timeout(600)
@pytest.mark.parametrize("world,mode", [(2, "ring"), (2, "ulysses"), (4, "ring")])
def test_sequence_parallel_forward(world, mode, tmp_path):
    """Rows are quantised each by itself, so ranks differ from one process only by the attention's order of sums,
    bf16's 8 bits and the 8-bit values that this moves to a neighbour (as the CUDA form from the CPU one)."""
    from test_dist_gloo import _run

    from harp_b200.parallel.sequence import SPContext

    q = _model().int8()
    lat, text, t = _inputs()
    n = lat.shape[-1] // q.cfg.patch_size
    ref = q.forward_local(q.patchify(lat), text, t, n, n, SPContext.single())[0].float()
    res = _run("dit_int8_sp", world, tmp_path, {"mode": mode})[0]
    seen = 0
    for r in range(world):
        lo, hi, pred = res[r]["lo"], res[r]["hi"], res[r]["pred"].float()
        assert lo == min(seen, ref.shape[1]) and pred.shape[1] == hi - lo and not res[r]["pred"].requires_grad
        seen = hi
        if hi > lo:
            assert ((pred - ref[:, lo:hi]).norm() / ref[:, lo:hi].norm()).item() < 3e-2
    assert seen == ref.shape[1]


@pytest.mark.gpu
def test_a_model_quantised_on_the_cpu_and_moved():
    """The quantisers give the same bits on both sides, so where the weights were quantised makes no difference."""
    import copy

    from harp_b200.models import dit as D

    torch.manual_seed(0)
    m = D.DiT(D.PRESETS["small"])
    with torch.no_grad():
        for n, p in m.named_parameters():
            p.normal_(0, 0.02 if "adaLN" in n else 0.05)
    m = m.bfloat16()
    a, b = m.int8().cuda().to(torch.bfloat16), copy.deepcopy(m).cuda().int8()
    for (n, p), (_, q) in zip(a.named_buffers(), b.named_buffers()):
        assert torch.equal(p, q) and p.stride() == q.stride() and p.dtype == q.dtype, n
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(2, 16, 16, 16, generator=g).bfloat16().cuda(), torch.randn(2, 32, 384, generator=g).bfloat16().cuda(),
         torch.rand(2, generator=g).cuda())
    assert torch.equal(a(*x), b(*x))
