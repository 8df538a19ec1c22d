"""Build the gfx950 HIP library ``lib/libmec.so`` in-tree with hipcc.

Usage: ``python -m memoryefficientclip_amd.build`` (or ``build()`` from
``__graft_entry__``).  hipcc cross-compiles for gfx950 without a GPU.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIB_DIR = PKG / "lib"
LIB = LIB_DIR / "libmec.so"
INCLUDE = PKG.parent / "include"

ARCH = os.environ.get("MEC_OFFLOAD_ARCH", "gfx950")

# Packed fp32 VALU forms are kept out of the device code (see the flag below);
# -munsafe-fp-atomics is not needed: scoped fp32 atomics already lower to
# global_atomic_add_f32 on gfx950.
HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-result",
]


def hipcc() -> str:
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    cand = Path(rocm) / "bin" / "hipcc"
    if cand.exists():
        return str(cand)
    found = shutil.which("hipcc")
    if not found:
        raise RuntimeError("hipcc not found (set ROCM_PATH)")
    return found


def sources() -> list[Path]:
    return [CSRC / "mec_abi.hip", CSRC / "mec_vocab.hip"]


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    # hipcc's host pass warns that it does not know the packed-fp32 feature; drop that noise.
    noise = "'-packed-fp32-ops' is not a recognized feature"
    err = "\n".join(l for l in res.stderr.splitlines() if noise not in l)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed ({res.returncode}):\n{err}")
    if verbose and err.strip():
        print(err, file=sys.stderr)


def build(verbose: bool = False) -> Path:
    """Compile the library (always recompiles, its sources side by side) and return its path."""
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    tmp = LIB.with_suffix(".so.tmp")
    objects = [LIB_DIR / f"{src.stem}.o" for src in sources()]
    with ThreadPoolExecutor() as pool:
        list(pool.map(lambda so: _run([hipcc(), *HIPCC_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", "-c", str(so[0]), "-o",
                                       str(so[1])], verbose), zip(sources(), objects)))
    _run([hipcc(), f"--offload-arch={ARCH}", "-fPIC", "-shared", *map(str, objects), "-o", str(tmp)], verbose)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))
