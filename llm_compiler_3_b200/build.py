"""Build libnpu_b200.so (sm_100a) in-tree with nvcc.

Objects go to ``_build/`` at the repository root and the shared library to
``llm_compiler_3_b200/lib/libnpu_b200.so``; both are git-ignored but travel with
the source tree, so a machine with a GPU and no compiler can load the prebuilt
library.  Only sources newer than their object are recompiled.

    python -m llm_compiler_3_b200.build [--force] [-j N]
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
ROOT = PACKAGE.parent
CSRC = PACKAGE / "csrc"
INCLUDE = ROOT / "include"
BUILD = ROOT / "_build"
LIBDIR = PACKAGE / "lib"
LIBRARY = LIBDIR / "libnpu_b200.so"
BINDINGS = PACKAGE / "_bindings.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + [
    "-O3", "-lineinfo", "-std=c++17", "-rdc=true", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC,-O3,-fvisibility=hidden", "-I", str(INCLUDE), "-I", str(CSRC),
    "-DNPU_B200_BUILD",
]


def nvcc() -> str:
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(found).exists():
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build libnpu_b200")
    return found


def _headers_mtime() -> float:
    files = list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.hpp")) + list(INCLUDE.glob("*.h"))
    return max((f.stat().st_mtime for f in files), default=0.0)


def _compile(src: Path, force: bool, hdr_mtime: float, extra: list[str]) -> Path:
    obj = BUILD / (src.stem + ".o")
    if (not force and obj.exists() and obj.stat().st_mtime >= src.stat().st_mtime
            and obj.stat().st_mtime >= hdr_mtime):
        return obj
    cmd = [nvcc(), *NVCC_FLAGS, *extra, "-c", str(src), "-o", str(obj)]
    done = subprocess.run(cmd, capture_output=True, text=True)
    if done.returncode:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{done.stdout}\n{done.stderr}")
    return obj


def _build_bindings(force: bool, hdr_mtime: float) -> None:
    """The Python binding of the paged-cache and beam operators (csrc/bindings.cpp): C++ against
    torch's headers, calling the library next to it; built for one torch and one Python.  Without
    torch there is none, and the library serves its C ABI alone."""
    import sysconfig

    try:
        import torch
        from torch.utils.cpp_extension import include_paths, library_paths
    except ImportError as exc:
        print(f"no Python binding of the paged-cache and beam operators without torch ({exc})", file=sys.stderr)
        return
    src = CSRC / "bindings.cpp"
    stamp = BUILD / "bindings.stamp"
    built_for = f"torch {torch.__version__}, Python {sys.version_info.major}.{sys.version_info.minor}"
    if (not force and BINDINGS.exists() and stamp.exists() and stamp.read_text() == built_for
            and BINDINGS.stat().st_mtime >= max(src.stat().st_mtime, hdr_mtime)):
        return
    cuda = Path(nvcc()).resolve().parent.parent
    tmp = BINDINGS.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DNPU_B200_BUILT_FOR="{torch.__version__}"',
           "-I", str(INCLUDE), "-isystem", str(cuda / "include"),
           *[x for p in include_paths() for x in ("-isystem", p)],
           "-isystem", sysconfig.get_path("include"), str(src), "-o", str(tmp),
           *[f"-L{p}" for p in library_paths()], "-lc10", "-ltorch_cpu", "-ltorch", "-lc10_cuda",
           "-ltorch_cuda", "-ltorch_python", f"-L{LIBDIR}", "-lnpu_b200",
           "-Wl,-rpath,$ORIGIN/lib", *[f"-Wl,-rpath,{p}" for p in library_paths()]]
    done = subprocess.run(cmd, capture_output=True, text=True)
    if done.returncode:
        raise RuntimeError(f"g++ failed on {src.name}:\n{done.stdout}\n{done.stderr}")
    os.replace(tmp, BINDINGS)
    stamp.write_text(built_for)


def build(force: bool = False, jobs: int | None = None, verbose_ptxas: bool = False) -> Path:
    """Compile every csrc/*.cu for sm_100a, link libnpu_b200.so, build the Python binding that
    calls it (where there is torch); return the library's path."""
    BUILD.mkdir(exist_ok=True)
    LIBDIR.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    hdr = _headers_mtime()
    extra = ["-Xptxas", "-v"] if verbose_ptxas else []
    with ThreadPoolExecutor(max_workers=jobs or min(8, os.cpu_count() or 4)) as pool:
        objects = list(pool.map(lambda s: _compile(s, force, hdr, extra), sources))
    newest = max(o.stat().st_mtime for o in objects)
    if force or not LIBRARY.exists() or LIBRARY.stat().st_mtime < newest:
        tmp = LIBRARY.with_suffix(".so.tmp")
        cmd = [nvcc(), *ARCH, "-shared", "-rdc=true", *[str(o) for o in objects],
               "-o", str(tmp), "-ldl", "-lpthread"]
        done = subprocess.run(cmd, capture_output=True, text=True)
        if done.returncode:
            raise RuntimeError(f"link of libnpu_b200.so failed:\n{done.stdout}\n{done.stderr}")
        os.replace(tmp, LIBRARY)
    _build_bindings(force, hdr)
    return LIBRARY


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-j", "--jobs", type=int, default=None)
    ap.add_argument("--ptxas-verbose", action="store_true",
                    help="print registers/spills/shared memory per kernel")
    a = ap.parse_args(argv)
    path = build(force=a.force or a.ptxas_verbose, jobs=a.jobs, verbose_ptxas=a.ptxas_verbose)
    print(path)
    return 0


if __name__ == "__main__":
    sys.exit(main())
