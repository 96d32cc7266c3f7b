"""Every kernel form of gemm_s8 on ragged sizes.

The kernel, its tile and its split of K come from an estimate of the time, so which sizes run
which form is asked (``torch.ops.harp.gemm_s8_plan``), and sizes are taken from a wide grid until each form has
met every kind of edge that its code tells apart.  Each product is compared in full with exact integer sums
(fp64), in both output types, with and without a bias, into an output that TMA can address and into one that
it cannot, with what lies around the output checked too.

Tolerance as for the other products: the sum is exact; at most 4 fp32 roundings of the terms follow, and one
to the output's type (half of bf16's last of 8 bits).
"""
import itertools

import pytest
import torch

from harp_b200.ops import functional as Fn
from harp_b200.runtime import errors

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(900)]

MS = [1, 2, 3, 5, 8, 16, 17, 31, 33, 64, 65, 127, 129, 200, 255, 257, 300, 384, 385, 511, 513, 640, 700, 1000, 1061, 1500,
      2047, 2176, 3000, 3500, 4352, 4357, 6001, 8704, 12001, 17408, 17409, 17560]
NS = sorted({1, 24, 64, 65, 127, 128, 129, 200, 223, 1003, 1152, 2304, 3456, 4608, 6912, 9216}
            | {k * bn + r for bn in (128, 192, 256) for k in (0, 1, 2, 3, 4, 6, 8) for r in (0, 1, 31, 33, bn // 2, bn - 1)
               if k * bn + r > 0})
KS = [1, 15, 16, 32, 127, 128, 129, 255, 256, 257, 384, 385, 640, 1000, 1152, 1155, 1500, 2304, 4608, 6144]


@pytest.fixture(scope="module")
def grid():
    """Sizes by the form that runs them, smallest products first."""
    import harp_b200

    assert harp_b200.load_native(build_if_needed=True), "CUDA library must load on a GPU box"
    torch.zeros(1, device="cuda")
    by = {}
    for M, N, K in itertools.product(MS, NS, KS):
        bn, nt, sp = torch.ops.harp.gemm_s8_plan(M, N, K)
        by.setdefault(("pair", bn) if bn else ("rows", nt), []).append((M * N * max(K, 256), M, N, K, sp))
    return {k: sorted(v) for k, v in by.items()}


def _band(n, bn):
    """Kinds of a last column band: whole, the narrowest MMA, less than half, half, more, all but one."""
    r = n % bn
    return ("whole" if r == 0 else "narrowest" if r <= 32 else "under half" if r < bn // 2 else "half" if r == bn // 2
            else "all but one" if r == bn - 1 else "over half")


def _pair_edges(bn, M, N, K, _):
    atoms = -(-K // 128)
    depth = "one atom" if atoms == 1 else "one stage" if atoms == 2 else "odd" if atoms % 2 else "even"
    long = "pipeline full" if atoms > 8 else ""
    rows = "whole" if M % 256 == 0 else "one CTA" if M % 256 <= 128 else "both CTAs"
    tiles = -(-M // 256) * -(-N // bn)
    turns = min(3, -(-tiles // (torch.cuda.get_device_properties(0).multi_processor_count // 2)))
    band = _band(N, bn)
    return {(band, depth), (band, long), (band, rows), (band, turns), (depth, K % 128 == 0), (rows, K % 128 == 0), (turns, long)}


def _rows_edges(nt, M, N, K, sp):
    atoms = -(-K // 128)
    toks = "whole" if M % nt == 0 else "one" if M % nt == 1 else "some"
    chans = "whole" if N % 128 == 0 else "one" if N % 128 == 1 else "by fours" if N % 4 == 0 else "some"
    return {(sp, toks), (sp, chans), (toks, chans), (sp, atoms % sp == 0), (sp, K % 128 == 0), (atoms > 8, sp)}


def _cover(form, sizes, limit):
    """Sizes, small ones first, each of which meets an edge that the ones before it did not, and some more over the range."""
    kind, width = form
    sizes = [s for s in sizes if s[0] <= limit]
    seen, out = set(), []
    for _, *size in sizes:
        e = (_pair_edges if kind == "pair" else _rows_edges)(width, *size)
        if e - seen:
            seen |= e
            out.append(tuple(size[:3]))
    return out + [s[1:4] for s in sizes[::max(1, len(sizes) // 25)]], seen


def _i8(rows, cols, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = -(-cols // 16) * 16
    return torch.randint(-128, 128, (rows, ld), generator=g, dtype=torch.int8, device="cuda")[:, :cols]


def _check(M, N, K):
    a, b = _i8(M, K, 1), _i8(N, K, 2)
    g = torch.Generator(device="cuda").manual_seed(3)
    sa = torch.rand(M, generator=g, device="cuda") + 0.01
    sb = torch.rand(N, generator=g, device="cuda") * 1e-2 + 1e-4
    bias = torch.randn(N, generator=g, device="cuda")
    acc = (a.double() @ b.double().t()).mul_(sa.double()[:, None]).mul_(sb.double())
    for dt, bt, tma in itertools.product((torch.bfloat16, torch.float32), (None, torch.bfloat16, torch.float32), (True, False)):
        bv = None if bt is None else bias.to(bt)
        at, ld = (16, -(-N // 16) * 16 + 32) if tma else (5, N + 13 + N % 2)
        buf = torch.full((M + 3, ld), 7.0, device="cuda", dtype=dt)
        c = Fn.gemm_s8(a, sa, b, sb, bias=bv, out=buf[1:1 + M, at:at + N])
        ref = acc if bv is None else acc + bv.double()
        tol = acc.abs() if bv is None else acc.abs() + bv.double().abs()
        tol = tol.mul(4 * 2.0 ** -24).add_(1e-38)
        if dt == torch.bfloat16:
            tol += 2.0 ** -8 * ref.abs()
        what = (M, N, K, dt, bt, tma)
        assert ((c.double() - ref).abs() <= tol).all(), what
        del ref, tol
        assert (buf[0] == 7).all() and (buf[1 + M:] == 7).all(), what
        assert (buf[:, :at] == 7).all() and (buf[:, at + N:] == 7).all(), what
    errors.check(a.device)


@pytest.mark.parametrize("bn", [128, 192, 256])
def test_pairs(grid, bn):
    sizes, seen = _cover(("pair", bn), grid[("pair", bn)], 17408 * 2304 * 1152)
    bands = {"whole", "narrowest", "under half", "half", "over half", "all but one"}
    assert {b for b, _ in seen if b in bands} >= bands - {"under half" if bn == 128 else "", "over half" if bn == 128 else ""}
    for band in ("whole", "narrowest", "half", "all but one"):  # with long sums, and over both accumulators
        assert (band, "pipeline full") in seen and (band, 3) in seen, (band, sorted(map(str, seen)))
    for s in sizes:
        _check(*s)


@pytest.mark.parametrize("nt", [16, 32, 64, 128, 256])
def test_rows(grid, nt):
    sizes, seen = _cover(("rows", nt), grid[("rows", nt)], 17408 * 2304 * 1152)
    assert len(sizes) >= 3
    if nt == 16:
        assert {s for s, _ in seen if isinstance(s, int) and not isinstance(s, bool)} >= {1, 2, 4, 8}
    for s in sizes:
        _check(*s)


def test_the_largest_products():
    """What a DiT-XL/2 block at 1024 px and batch 4 multiplies, in full."""
    for M, N, K in ((17408, 3456, 1152), (17408, 1152, 1152), (17408, 1152, 4608), (17408, 9216, 1152)):
        assert torch.ops.harp.gemm_s8_plan(M, N, K)[0] > 0
        _check(M, N, K)


def test_plan_refuses_sizes_without_one():
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 131072), (1 << 31, 1, 1), (1, 1 << 31, 1)):
        with pytest.raises(RuntimeError):
            torch.ops.harp.gemm_s8_plan(*bad)
