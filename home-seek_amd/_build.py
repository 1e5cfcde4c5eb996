"""Builds libhsmoe.so (hipcc, gfx950) from csrc/ into this package directory."""
from __future__ import annotations

import concurrent.futures
import os
import subprocess
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
OBJ_DIR = PKG_DIR / "_build"
LIB_PATH = PKG_DIR / "libhsmoe.so"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

HIP_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wall",
    "-Wno-unused-function",
    # every float expression rounds once per operation (HIP's __fadd_rn and
    # __fmul_rn are plain operators, which clang would otherwise fuse into FMA)
    "-ffp-contract=off",
    # packed fp32 VALU ops stay off (hipcc's host pass warns it does not know
    # the feature; that warning is harmless)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    f"-I{REPO_DIR / 'include'}",
    f"-I{CSRC}",
]

# Flags of one source.  hsmoe_linear: matrix sums in ordinary registers; left to
# itself the compiler keeps them in the accumulation file and, in kernels of one
# wave per SIMD, moves 64 of them back and forth in every pass of the loop.
SOURCE_FLAGS = {"hsmoe_linear": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"]}


def _compile(src: Path) -> Path:
    obj = OBJ_DIR / (src.stem + ".o")
    cmd = [HIPCC, *HIP_FLAGS, *SOURCE_FLAGS.get(src.stem, []), "-c", str(src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{res.stderr}")
    return obj


def build_library(verbose: bool = False) -> Path:
    """Compiles every csrc/*.hip for gfx950 and links libhsmoe.so."""
    OBJ_DIR.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip"))
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(sources))) as ex:
        objs = list(ex.map(_compile, sources))
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link of libhsmoe.so failed:\n{res.stderr}")
    os.replace(tmp, LIB_PATH)
    if verbose:
        print(f"built {LIB_PATH} from {len(sources)} sources")
    return LIB_PATH
