"""Build the gfx950 HIP library ``tilert_amd/libtilert_amd.so`` in-tree with hipcc.

``python -m tilert_amd.build`` (or ``__graft_entry__.build()``) compiles every
``tilert_amd/csrc/*.hip`` for gfx950 and links one shared library exporting the C ABI
declared in ``include/tilert_amd.h``.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OUT = PKG / "libtilert_amd.so"
OBJ = PKG / "_build"
ARCH = "gfx950"

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # packed fp32 VALU ops are kept out of the device code (see the package docs)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    f"-I{ROOT / 'include'}",
    "-Wall",
    "-Wno-unused-function",
]


# Per-source extra flags.  indexer: MFMA results in VGPRs (its epilogue reads every result
# with VALU ops; in AGPRs each element would first need a v_accvgpr_read).  paged_mla, paged_gqa: the
# same; and with two waves a SIMD the registers are not halved into VGPRs and AGPRs.
EXTRA = {
    "indexer": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
    "paged_mla": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
    "paged_gqa": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
}


def _compile(src: Path) -> Path:
    obj = OBJ / (src.stem + ".o")
    cmd = [HIPCC, *FLAGS, *EXTRA.get(src.stem, []), "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    return obj


def build(verbose: bool = False) -> Path:
    OBJ.mkdir(exist_ok=True)
    srcs = sorted(CSRC.glob("*.hip"))
    with ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(_compile, srcs))
    tmp = OUT.with_suffix(".so.tmp")
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(tmp), *map(str, objs)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, OUT)
    if verbose:
        print(f"built {OUT}")
    return OUT


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
