"""Hand-written loads that are waited for later (k_cdot3, csrc/alz_scan.hip: rows of the input and pairs of responses): on every path
of the listing the destination registers are left alone until the wait.  No other kernel loads vector registers that way."""
import importlib.util
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "audiolazy_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def checker():
  spec = importlib.util.spec_from_file_location("check_asm_paths", os.path.join(ROOT, "tools", "check_asm_paths.py"))
  mod = importlib.util.module_from_spec(spec)
  spec.loader.exec_module(mod)
  return mod.check


def listing(*body):
  return ["\t;;#ASMSTART", "\tglobal_load_dwordx2 v[2:3], v[8:9], off", "\t;;#ASMEND"] + ["\t" + l if not l.endswith(":") else l for l in body]


def test_the_checker_follows_branches():
  check = checker()
  wait, end = "s_waitcnt vmcnt(0)", "s_endpgm"
  assert check(listing(wait, "v_add_f64 v[2:3], v[2:3], v[4:5]", end)) == (1, [], 0)
  assert check(listing("v_mov_b32_e32 v4, v5", wait, end)) == (1, [], 0)
  assert len(check(listing("v_mov_b32_e32 v4, v3", wait, end))[1]) == 1                    # read too early
  assert len(check(listing("v_mov_b64_e32 v[0:2], 0", wait, end))[1]) == 1                 # written over
  assert len(check(listing("s_cbranch_vccz .L1", wait, end, ".L1:", "v_mov_b32_e32 v3, 0", end))[1]) == 1
  assert len(check([".L0:", "\tv_mov_b32_e32 v2, 0"] + listing("s_cbranch_vccz .L0", wait, end))[1]) == 1
  assert len(check(listing("s_waitcnt lgkmcnt(0)", "v_mov_b32_e32 v2, 0", end))[1]) == 1    # a wait for something else
  assert check(listing("s_setpc_b64 s[2:3]"))[2] == 1
  together = ["\t;;#ASMSTART", "\ts_load_dwordx2 s[4:5], s[0:1], 0x0", "\ts_waitcnt lgkmcnt(0)", "\t;;#ASMEND", "\ts_mov_b32 s4, 0"]
  assert check(together) == (0, [], 0)


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc on this machine")
@pytest.mark.parametrize("opt", ["-O3", "-O1"])
def test_k_cdot3(tmp_path, opt):
  out = tmp_path / "listing.s"
  subprocess.run([HIPCC, "--offload-arch=gfx950", opt, "-std=c++17", "-ffp-contract=off", "-fPIC", "-Xclang", "-target-feature", "-Xclang",
                  "-packed-fp32-ops", "-fno-fast-math", "-S", "--cuda-device-only", os.path.join(CSRC, "alz_scan.hip"), "-o", str(out)],
                 check=True, capture_output=True, timeout=600)
  requests, reports, left = checker()(out.read_text().split("\n"))
  assert requests > 30 and not reports and not left, reports


def test_no_other_kernel_loads_registers_by_hand():
  found = []
  for name in sorted(os.listdir(CSRC)):
    if name.endswith((".hip", ".h")) and name != "alz_scan.hip":
      with open(os.path.join(CSRC, name)) as f:
        found += ["%s: %s" % (name, l.strip()) for l in f if re.search(r"(global|buffer|flat)_load_(?!lds)\w+ %\d", l)]
  assert not found, found
