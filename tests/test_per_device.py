"""What the int8 launchers set up once, they set up once for each device
(harp_b200/csrc/per_device.h)."""
import os
import re
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "harp_b200", "csrc")

_SRC = r"""
#include "per_device.h"

#include <stdexcept>
#include <thread>
#include <vector>

static harp::PerDevice<long> value;

int main() {
  int made = 0;
  auto of = [&](int device) { return value.get(device, [&] { ++made; return 100L + device; }); };
  for (int again = 0; again < 3; ++again)
    for (int d : {0, 1, 7, 63})
      if (of(d) != 100 + d) return 1;
  if (made != 4) return 2;
  for (int d : {-1, 64, 1000})  // beyond its places: made anew, as right
    if (of(d) != 100 + d || of(d) != 100 + d) return 3;
  if (made != 10) return 4;
  // a failure is passed on and not kept
  bool thrown = false;
  try {
    value.get(2, []() -> long { throw std::runtime_error("no"); });
  } catch (const std::runtime_error&) {
    thrown = true;
  }
  if (!thrown || value.get(2, [] { return 5L; }) != 5 || value.get(2, [] { return 6L; }) != 5) return 5;
  // many threads at once: one of them makes it, all see it
  harp::PerDevice<int> shared;
  std::atomic<int> calls{0}, wrong{0};
  std::vector<std::thread> ts;
  for (int t = 0; t < 16; ++t)
    ts.emplace_back([&] {
      for (int d = 0; d < 8; ++d)
        if (shared.get(d, [&] { ++calls; return d + 1; }) != d + 1) ++wrong;
    });
  for (auto& t : ts) t.join();
  return calls == 8 && wrong == 0 ? 0 : 6;
}
"""


def test_made_once_for_each_device(tmp_path):
    gxx = os.environ.get("CXX") or shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    src, exe = tmp_path / "per_device.cpp", str(tmp_path / "per_device")
    src.write_text(_SRC)
    build = subprocess.run([gxx, "-std=c++17", "-O1", "-pthread", "-I" + CSRC, str(src), "-o", exe],
                           capture_output=True, text=True, timeout=300)
    assert build.returncode == 0, build.stderr[-3000:]
    run = subprocess.run([exe], timeout=120)
    assert run.returncode == 0


@pytest.mark.parametrize("name", ["gemm_s8_sm100.cu", "quant.cu"])
def test_launchers_keep_nothing_for_the_first_device_only(name):
    code = re.sub(r"//[^\n]*", " ", open(os.path.join(CSRC, name)).read())
    kept = re.findall(r"\bstatic\s+(?!constexpr\b|thread_local\b)[^;]*;", code)
    assert kept and all(k.startswith("static PerDevice<") for k in kept), kept
    known = re.search(r"struct Known \{(.*?)\};", code, re.S)
    assert known is None or "device" in known.group(1)


@pytest.mark.gpu
@pytest.mark.multigpu
def test_second_device_of_a_process():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")
    import harp_b200
    from harp_b200.ops import functional as Fn
    from harp_b200.runtime import errors

    assert harp_b200.load_native(build_if_needed=True)
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(3000, 1152, generator=g).bfloat16(), torch.randn(1152, 1152, generator=g).bfloat16()
    outs = []
    for dev in ("cuda:0", "cuda:1"):
        xd, wd = x.to(dev), w.to(dev)
        for rows in (3, 300, 3000):
            q, s, h = Fn.rmsnorm_mod_quant(xd[:rows], wd[0], None, None, rows, 1e-6, residual=xd[:rows])
            outs.append((Fn.gemm_s8(q, s, *Fn.quant_rows(wd)).cpu(), h.cpu()))
        torch.cuda.synchronize(dev)
        errors.check(torch.device(dev))
    for a, b in zip(outs[:3], outs[3:]):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
