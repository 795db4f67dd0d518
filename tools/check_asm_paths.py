#!/usr/bin/env python3
"""Hand-written loads whose wait comes later: the compiler takes the outputs of such a statement as written at once, so nothing but the
listing shows whether it lets their registers alone until the wait.  This script reads a device assembly listing (hipcc -S
--cuda-device-only), follows every branch behind each such request, and reports any instruction that touches its destination registers
on a path without a wait for all loads of its kind (scalar: lgkmcnt(0), vector: vmcnt(0)).  Paths are not checked for being possible:
no report is a proof, a report has to be read.   usage: tools/check_asm_paths.py file.s"""
import re
import sys


def registers(text, kind):
  out = [(int(a), int(b)) for a, b in re.findall(r"\b%s\[(\d+):(\d+)\]" % kind, text)]
  return out + [(int(r), int(r)) for r in re.findall(r"\b%s(\d+)\b" % kind, text)]


def check(lines):
  """(requests, reports, scans that left the listing) of one listing"""
  label = {m.group(1): i for i, l in enumerate(lines) for m in [re.match(r"^([.\w$]+):", l)] if m}
  requests, reports, left, i = 0, [], 0, 0
  while i < len(lines):
    if ";;#ASMSTART" not in lines[i]:
      i += 1
      continue
    j, dst = i + 1, []
    while ";;#ASMEND" not in lines[j]:
      m = re.match(r"\s+s_load_dword\w*\s+(s\[\d+:\d+\]|s\d+),", lines[j])
      if m:
        dst.append(("s",) + registers(m.group(1), "s")[0])
      m = re.match(r"\s+(?:global|buffer|flat)_load_(?!lds)\w+\s+(v\[\d+:\d+\]|v\d+),", lines[j])
      if m:
        dst.append(("v",) + registers(m.group(1), "v")[0])
      if re.match(r"\s+s_waitcnt\b", lines[j]):
        dst = [d for d in dst if ("lgkmcnt(0)" if d[0] == "s" else "vmcnt(0)") not in lines[j]]
      j += 1
    i = j + 1
    if not dst:
      continue
    requests += 1
    kinds, seen, todo, hits = {d[0] for d in dst}, set(), [j + 1], set()
    while todo:
      k = todo.pop()
      while k < len(lines) and k not in seen:
        seen.add(k)
        text = lines[k]
        if not text.startswith("\t") or text.strip().startswith((";", ".")):
          k += 1
          continue
        text = text.split(";")[0]
        op = text.split()[0]
        if op == "s_waitcnt":
          if ("s" not in kinds or "lgkmcnt(0)" in text) and ("v" not in kinds or "vmcnt(0)" in text):
            break
          k += 1
          continue
        if op == "s_endpgm":
          break
        if op in ("s_setpc_b64", "s_swappc_b64"):
          left += 1
          break
        if any(not (b < lo or a > hi) for kind, lo, hi in dst for a, b in registers(text, kind)):
          hits.add(k)
          break
        if op == "s_branch":
          k = label[text.split()[1]]
          continue
        if op.startswith("s_cbranch"):
          todo.append(label[text.split()[1]])
        k += 1
    if hits:
      reports.append((j, dst, [(h + 1, lines[h].strip()) for h in sorted(hits)[:3]]))
  return requests, reports, left


if __name__ == "__main__":
  with open(sys.argv[1]) as f:
    requests, reports, left = check(f.read().split("\n"))
  for r in reports:
    print("line %d %s: touched before a wait at %s" % r)
  print("hand-written requests: %d, reports: %d, scans that left the listing: %d" % (requests, len(reports), left))
  sys.exit(1 if reports or left or not requests else 0)
