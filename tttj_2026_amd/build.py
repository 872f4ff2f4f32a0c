"""Build the gfx950 C-ABI library ``libtttj_amd.so`` in-tree with hipcc.

``python -m tttj_2026_amd.build`` (or ``__graft_entry__.build()``) compiles every ``csrc/*.hip``
to an object in ``_build/`` (in parallel) and links them into ``tttj_2026_amd/libtttj_amd.so``.
Only hipcc is needed; no GPU is needed to build.
"""

from __future__ import annotations

import concurrent.futures as cf
import os
import pathlib
import shutil
import subprocess
import sys

PKG = pathlib.Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
BUILD = ROOT / "_build"
LIB = PKG / "libtttj_amd.so"
ARCH = os.environ.get("TTTJ_OFFLOAD_ARCH", "gfx950")

HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # Packed fp32 VALU forms are kept out of the generated code on purpose.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    f"-I{INCLUDE}",
    f"-I{CSRC}",
]


# Per-source flags.  The attention kernel reads its MFMA accumulators element-wise (softmax,
# rescaling); keeping them in architectural VGPRs (instead of AGPRs) removes an AGPR <-> VGPR copy
# per element per tile.
SOURCE_FLAGS = {
    "attention.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
    "attention_small.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
    "rowchain.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
    "seq_attention.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
    "seq_attention_wide.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
    "seq_attention8.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
    "seq_attention8_wide.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
    "megakernel.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
}


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and pathlib.Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm)")


def _compile(src: pathlib.Path, extra) -> pathlib.Path:
    obj = BUILD / (src.stem + ".o")
    cmd = [hipcc(), *HIPCC_FLAGS, *SOURCE_FLAGS.get(src.name, []), *extra, "-c", str(src), "-o",
           str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{proc.stderr}")
    return obj


def build(verbose: bool = False, extra_flags=()) -> pathlib.Path:
    BUILD.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip"))
    if not sources:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    jobs = min(len(sources), max(1, min(8, os.cpu_count() or 1)))
    with cf.ThreadPoolExecutor(jobs) as pool:
        objs = list(pool.map(lambda s: _compile(s, list(extra_flags)), sources))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stderr}")
    os.replace(tmp, LIB)
    if verbose:
        print(f"built {LIB} from {len(sources)} sources")
    return LIB


if __name__ == "__main__":
    build(verbose=True, extra_flags=sys.argv[1:])
