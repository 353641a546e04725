"""Build recipe for libgqa.so (hipcc, gfx950 only).

``python -m lara_amd.build`` compiles every HIP translation unit under ``lara_amd/csrc``
into ``lara_amd/libgqa.so`` in-tree.  Object files go to ``_build/`` at the repository
root.  The flags pin the target to gfx950 and turn off packed-fp32 code generation.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_ROOT = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
BUILD_DIR = REPO_ROOT / "_build"
LIB_PATH = PKG_DIR / "libgqa.so"
SOURCES = ("gqa_api.hip", "decode.hip", "decode_kv8.hip", "heads.hip", "kv8.hip", "kv_cache.hip", "layer.hip", "prefill.hip",
           "probe.hip", "rtl_exact.hip", "w4.hip")
DATA = PKG_DIR / "data"

HIP_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wall",
    "-Wno-unused-function",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    f"-I{REPO_ROOT / 'include'}",
    f"-I{BUILD_DIR}",
]


def hipcc() -> str:
    path = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(path).exists():
        raise RuntimeError("hipcc not found; the ROCm toolchain is required to build libgqa.so")
    return path


def _compile(src: Path, obj: Path) -> None:
    cmd = [hipcc(), *HIP_FLAGS, "-c", str(src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    # hipcc's host pass warns that it does not know the packed-fp32 feature; drop that line.
    noise = "'-packed-fp32-ops' is not a recognized feature"
    err = "\n".join(line for line in proc.stderr.splitlines() if noise not in line)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{err}")
    if err.strip():
        print(err, file=sys.stderr)


def write_rom_tables() -> Path:
    """Emit the board's ROM images (lara_amd/data/*.hex) as device constant tables."""
    out = BUILD_DIR / "rtl_luts.inc"
    lines = ["// generated by lara_amd/build.py from lara_amd/data/exp_lut.hex and recip_lut.hex", "#pragma once"]
    for name, sym, n in (("exp_lut.hex", "kRtlExpLut", 1024), ("recip_lut.hex", "kRtlRecipLut", 256)):
        words = [int(x, 16) for x in (DATA / name).read_text().split()]
        if len(words) != n:
            raise RuntimeError(f"{name}: expected {n} words, found {len(words)}")
        body = ",".join(f"0x{w:08x}u" for w in words)
        lines.append(f"__constant__ const uint32_t {sym}[{n}] = {{{body}}};")
    text = "\n".join(lines) + "\n"
    if not out.is_file() or out.read_text() != text:
        out.write_text(text)
    return out


def build(verbose: bool = True) -> Path:
    """Compile all sources and link lara_amd/libgqa.so; returns the library path."""
    BUILD_DIR.mkdir(exist_ok=True)
    write_rom_tables()
    objs = [BUILD_DIR / (name.rsplit(".", 1)[0] + ".o") for name in SOURCES]
    jobs = min(len(SOURCES), int(os.environ.get("MAX_JOBS", "8")))
    with ThreadPoolExecutor(max_workers=jobs) as pool:
        list(pool.map(lambda so: _compile(CSRC / so[0], so[1]), zip(SOURCES, objs)))
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", *map(str, objs), "-lhipblaslt", "-o", str(tmp)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stderr}")
    os.replace(tmp, LIB_PATH)
    if verbose:
        print(f"built {LIB_PATH}")
    return LIB_PATH


if __name__ == "__main__":
    build()
