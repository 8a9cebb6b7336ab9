"""In-tree build of liblewi_moe.so for sm_100a (explicit nvcc; the .so lands next to this file)."""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
UNITS = ("lewi_moe.cu", "mixers.cu")   # compiled side by side, then linked
OUT = os.path.join(HERE, "liblewi_moe.so")
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC"]


def _sources():
  csrc = os.path.join(HERE, "csrc")
  inc = os.path.join(os.path.dirname(HERE), "include")
  files = [os.path.join(csrc, f) for f in sorted(os.listdir(csrc))]
  files += [os.path.join(inc, f) for f in sorted(os.listdir(inc))]
  return files


def is_stale():
  if not os.path.exists(OUT):
    return True
  t = os.path.getmtime(OUT)
  return any(os.path.getmtime(f) > t for f in _sources())


def build(force=False, verbose=False):
  """Compile the CUDA library if it is missing or older than its sources.  Returns the .so path."""
  if not force and not is_stale():
    return OUT
  nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
  extra = ["-Xptxas", "-v"] if verbose else []
  with tempfile.TemporaryDirectory() as tmp:
    objects = [os.path.join(tmp, u + ".o") for u in UNITS]
    runs = [subprocess.Popen([nvcc, *extra, *NVCC_FLAGS, "-c", "-o", o, os.path.join(HERE, "csrc", u)], stdout=subprocess.PIPE,
                             stderr=subprocess.STDOUT, text=True) for u, o in zip(UNITS, objects)]
    said = [r.communicate()[0] for r in runs]
    if any(r.returncode != 0 for r in runs):
      raise RuntimeError("nvcc failed:\n" + "\n".join(said))
    linked = os.path.join(tmp, "lib.so")   # (moved into place whole: a process that loads it meanwhile has the old one)
    res = subprocess.run([nvcc, *NVCC_FLAGS, "-shared", "-o", linked, *objects], capture_output=True, text=True)
    if res.returncode != 0:
      raise RuntimeError("linking failed:\n" + res.stdout + res.stderr)
    shutil.copy(linked, OUT + ".new")
    os.replace(OUT + ".new", OUT)
  if verbose:
    print("\n".join(said))
  return OUT


if __name__ == "__main__":
  print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
