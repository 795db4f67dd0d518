"""No GPU source of the package writes through the scalar data cache (scalar stores and atomics, that cache's write-back and
discard): such a write is not ordered with the vector memory path the kernels use everywhere else.  The check reads the sources
and the scripts that build them, inactive branches of the preprocessor and comments included."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WRITES = re.compile(r"\bs_(?:(?:buffer_|scratch_)?(?:store|atomic)|dcache_(?:wb|discard))")
SOURCES = (".hip", ".h", ".inc", ".c", ".cpp", ".s", ".sh", ".py")


def scalar_writes(text):
  return [(text.count("\n", 0, m.start()) + 1, m.group()) for m in WRITES.finditer(text)]


def test_pattern_finds_the_instructions():
  for parts in (("s", "store", "dword"), ("s", "buffer", "store", "dwordx2"), ("s", "scratch", "store", "dword"),
                ("s", "atomic", "add"), ("s", "buffer", "atomic", "umax"), ("s", "dcache", "wb"), ("s", "dcache", "discard")):
    assert scalar_writes("x\n  asm(\"" + "_".join(parts) + " %0\")")[0][0] == 2
  for text in ("s_load_dwordx8", "s_dcache_inv", "ds_store_b64", "global_atomic_add", "buffer_store_dword", "s_waitcnt"):
    assert not scalar_writes(text)


def test_no_source_writes_through_the_scalar_cache():
  found = []
  for top in ("audiolazy_amd", "include", "oracle", "tests", "tools"):
    for folder, dirs, files in os.walk(os.path.join(ROOT, top)):
      for name in files:
        if name.endswith(SOURCES) or name == "Makefile":
          path = os.path.join(folder, name)
          with open(path, errors="replace") as f:
            found += ["%s:%d: %s" % (os.path.relpath(path, ROOT), n, t) for n, t in scalar_writes(f.read())]
  assert not found, "\n".join(found)
