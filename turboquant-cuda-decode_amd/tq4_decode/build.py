"""Compile the gfx950 HIP library ``libtq4_decode.so`` in place (``hipcc``).

Run as ``python -m tq4_decode.build`` from ``turboquant-cuda-decode_amd/`` or call
``build()``; the library lands next to this file and is what ``tq4_decode._lib``
loads.  Every call recompiles.
"""
from __future__ import annotations

import os
import pathlib
import shutil
import subprocess
import tempfile

PKG = pathlib.Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = ROOT / "csrc"
LIB = PKG / "libtq4_decode.so"
SOURCES = ("tq4_decode.hip", "span_decode.hip", "prefix_decode.hip", "rope_store.hip", "chunk_attention.hip",
           "cache_load.hip")
ARCH = os.environ.get("TQ4_OFFLOAD_ARCH", "gfx950")

HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # keep hipcc from emitting packed-fp32 VALU ops
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMA accumulators in VGPRs: no AGPR<->VGPR copies around the softmax rescale
    "-mllvm", "-amdgpu-mfma-vgpr-form",
    "-Wall",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and pathlib.Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm)")


def build(verbose: bool = False) -> pathlib.Path:
    """Every source to an object of its own, at once, then the link."""
    with tempfile.TemporaryDirectory(dir=PKG, prefix="_build_") as tmp:
        objs = [pathlib.Path(tmp) / (pathlib.Path(src).stem + ".o") for src in SOURCES]
        cmds = [[hipcc(), *HIPCC_FLAGS, "-c", "-o", str(o), str(CSRC / src)] for src, o in zip(SOURCES, objs)]
        procs = [subprocess.Popen(c, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for c in cmds]
        said = [p.communicate()[0] for p in procs]
        for cmd, p, text in zip(cmds, procs, said):
            if p.returncode != 0:
                raise RuntimeError("hipcc failed:\n" + " ".join(cmd) + "\n" + text[-4000:])
            if verbose and text:
                print(text)
        out = LIB.with_suffix(".so.tmp")
        cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-o", str(out), *map(str, objs)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("hipcc failed:\n" + " ".join(cmd) + "\n" + res.stderr[-4000:])
    os.replace(out, LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))
