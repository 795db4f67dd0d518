"""Every line that compiles GPU code turns the packed 32-bit float instructions off (the engine's arithmetic is 64-bit) and keeps the
separately rounded multiply and add."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(not shutil.which("make"), reason="no make on this machine")
@pytest.mark.parametrize("target", ["all", "tuning", "asan", "ubsan"])
def test_make_lines(target):
  out = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "audiolazy_amd", "csrc"), target], capture_output=True, text=True,
                       check=True, timeout=60).stdout
  lines = [l for l in out.splitlines() if "--offload-arch" in l and " -c " in l]
  assert lines
  for l in lines:
    assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in l and "-ffp-contract=off" in l, l


def test_the_other_builds():
  for name in ("__graft_entry__.py", os.path.join("tools", "build_variant.sh"), os.path.join("tools", "build_fir_variants.sh")):
    with open(os.path.join(ROOT, name)) as f:
      assert "-packed-fp32-ops" in f.read(), name
