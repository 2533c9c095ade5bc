"""Build libq6b200.so (the C-ABI library) in-tree with nvcc for sm_100a.

    python -m qwen_image_shardedit_mlx_b200.build [--force] [--verbose]

Each .cu under csrc/ is compiled to an object under csrc/_build/ (skipped when
up to date) and the objects are linked into qwen_image_shardedit_mlx_b200/libq6b200.so
with a static CUDA runtime, so the library carries no dependency on a
particular libcudart next to it.  The torch surface of the dense operators
(csrc/q6_torch.cpp) becomes the extension module _q6torch next to it, linked
against that library.
"""

from __future__ import annotations

import argparse
import importlib.metadata
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
BUILD = CSRC / "_build"
LIB = PKG / "libq6b200.so"
EXT = PKG / "_q6torch.so"
EXT_SOURCE = CSRC / "q6_torch.cpp"
INCLUDE = ROOT / "include"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3",
    "-std=c++17",
    "-lineinfo",
    "--expt-relaxed-constexpr",
    "-Xcompiler",
    "-fPIC",
    "-Xcompiler",
    "-fvisibility=hidden",
]


def nvcc() -> str:
    found = shutil.which("nvcc")
    if found:
        return found
    cand = Path("/usr/local/cuda/bin/nvcc")
    if cand.exists():
        return str(cand)
    raise RuntimeError("nvcc not found")


def _headers() -> list[Path]:
    return sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + sorted(INCLUDE.glob("*.h"))


def _needs(out: Path, deps: list[Path]) -> bool:
    if not out.exists():
        return True
    t = out.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def build(force: bool = False, verbose: bool = False, extra_flags: list[str] | None = None) -> Path:
    BUILD.mkdir(parents=True, exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    headers = _headers()
    flags = NVCC_FLAGS + (extra_flags or [])
    cmds: list[list[str]] = []
    objs: list[Path] = []
    for src in sources:
        obj = BUILD / (src.stem + ".o")
        objs.append(obj)
        if force or _needs(obj, [src, *headers]):
            cmds.append([nvcc(), *ARCH, *flags, "-I", str(INCLUDE), "-I", str(CSRC), "-c", str(src), "-o", str(obj)])

    def run(cmd: list[str]) -> None:
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or res.returncode != 0:
            sys.stdout.write(res.stdout)
            sys.stderr.write(res.stderr)
        if res.returncode != 0:
            raise RuntimeError(f"{Path(cmd[0]).name} failed for {cmd[-3]}")

    if cmds:
        with ThreadPoolExecutor(max_workers=min(len(cmds), os.cpu_count() or 4)) as pool:
            list(pool.map(run, cmds))
    if force or cmds or _needs(LIB, objs):
        link = [nvcc(), *ARCH, "-shared", "-cudart", "static", *[str(o) for o in objs], "-o", str(LIB)]
        run(link)
    if force or _extension_stale():
        run(_torch_extension_command(EXT_SOURCE))
        _stamp().write_text(_torch_abi())
    return LIB


def _stamp() -> Path:
    return BUILD / (EXT.stem + ".abi")


def _torch_abi() -> str:
    """What the extension module is bound to besides its sources."""

    return f"torch {importlib.metadata.version('torch')}, {sysconfig.get_config_var('SOABI')}"


def _extension_stale() -> bool:
    """Older than its sources, or built against another torch or Python: it would
    not load, whatever the file times say."""

    if _needs(EXT, [EXT_SOURCE, INCLUDE / "q6_b200.h", LIB]):
        return True
    return not _stamp().exists() or _stamp().read_text() != _torch_abi()


def _torch_extension_command(src: Path) -> list[str]:
    import torch
    from torch.utils import cpp_extension

    includes = [*cpp_extension.include_paths("cuda"), sysconfig.get_paths()["include"], str(INCLUDE)]
    libs = cpp_extension.library_paths("cuda")
    return [
        shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
        "-DTORCH_EXTENSION_NAME=_q6torch", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        *[f"-I{p}" for p in includes], str(src), *[f"-L{p}" for p in [*libs, str(PKG)]],
        "-l:libq6b200.so", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python",
        "-Wl,-rpath,$ORIGIN", "-o", str(EXT),
    ]


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", "-v", action="store_true")
    ap.add_argument("--ptxas-info", action="store_true", help="print register / smem use per kernel")
    args = ap.parse_args()
    extra = ["-Xptxas", "-v"] if args.ptxas_info else None
    print(build(force=args.force or args.ptxas_info, verbose=args.verbose or args.ptxas_info, extra_flags=extra))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
