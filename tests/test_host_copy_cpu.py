"""The host-block entry point's copies: the caller's arrays reach the device through page-locked buffers that the library allocates
itself (csrc/alz_host.h cuts the block into pieces and copies them with a few threads); no caller's memory is page-locked."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "audiolazy_amd", "csrc")


def test_no_source_page_locks_memory_it_does_not_own():
  found = []
  for name in sorted(os.listdir(CSRC)):
    if name.endswith((".hip", ".h")):
      with open(os.path.join(CSRC, name)) as f:
        found += ["%s:%d" % (name, i) for i, line in enumerate(f, 1) if re.search(r"(hip|cuda)Host(Un)?[Rr]egister", line)]
  assert not found, found


@pytest.mark.skipif(not shutil.which("g++"), reason="no host compiler on this machine")
def test_pieces_and_crew_copy_every_rectangle(tmp_path):
  exe = str(tmp_path / "host_copy_check")
  subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", os.path.join(ROOT, "tests", "helpers", "host_copy_check.cpp"), "-o", exe],
                 check=True, capture_output=True, timeout=300)
  out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
  assert out.returncode == 0 and out.stdout == "ok 1400\n", out.stdout + out.stderr
