"""Build librns8.so (the rns8 C ABI on sm_100a kernels) in-tree.

Every translation unit under rns8_b200/csrc is compiled by nvcc for
sm_100a only (-gencode arch=compute_100a,code=sm_100a) and linked into
rns8_b200/_build/librns8.so, which is what the Python bindings, the tests and
bench.py load. Object files are rebuilt when a source or header is newer.

Where torch with CUDA is installed, the torch binding of the 8-bit operators
(csrc/torch/quant_torch.cpp) is compiled against it by the host compiler into
rns8_b200/_build/_quant_torch.so; the library itself knows no torch, and its
build succeeds where the binding's does not.

    python -m rns8_b200.build [--force] [--ptxas-verbose]
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = BUILD / "librns8.so"
TORCH_SRC = CSRC / "torch" / "quant_torch.cpp"
TORCH_LIB = BUILD / "_quant_torch.so"
INCLUDE = ROOT / "include"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = [
    "-std=c++17",
    "-O3",
    "-lineinfo",
    "-Xcompiler",
    "-fPIC,-fvisibility=hidden",
    "--expt-relaxed-constexpr",
    "-DRNS8_BUILDING_LIBRARY",
    f"-I{INCLUDE}",
    f"-I{CSRC}",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build librns8.so")


def host_compiler() -> list[str]:
    # The system g++ is the toolchain nvcc 12.9 is validated against here.
    return ["-ccbin", "/usr/bin/g++"] if Path("/usr/bin/g++").exists() else []


def sources() -> list[Path]:
    return sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cpp")])


def headers() -> list[Path]:
    return [*CSRC.glob("*.hpp"), *CSRC.glob("*.cuh"), *INCLUDE.glob("rns8/*.h")]


def _compile(src: Path, obj: Path, extra: list[str]) -> tuple[Path, str]:
    cmd = [nvcc(), *host_compiler(), *COMMON, *ARCH_FLAGS, *extra, "-c", str(src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    return src, res.stdout + res.stderr


def build(force: bool = False, ptxas_verbose: bool = False, jobs: int | None = None) -> Path:
    BUILD.mkdir(exist_ok=True)
    hdr_time = max((h.stat().st_mtime for h in headers()), default=0.0)
    extra = ["-Xptxas", "-v"] if ptxas_verbose else []
    todo = []
    objs = []
    for src in sources():
        obj = BUILD / (src.name + ".o")
        objs.append(obj)
        if force or ptxas_verbose or not obj.exists() or obj.stat().st_mtime < max(src.stat().st_mtime, hdr_time):
            todo.append((src, obj))
    logs = []
    if todo:
        workers = jobs or min(len(todo), os.cpu_count() or 4)
        with cf.ThreadPoolExecutor(max_workers=workers) as pool:
            for src, log in pool.map(lambda t: _compile(t[0], t[1], extra), todo):
                if log.strip():
                    logs.append(f"--- {src.name}\n{log}")
    if todo or not LIB.exists():
        cmd = [nvcc(), *host_compiler(), *ARCH_FLAGS, "-shared", "-o", str(LIB), *map(str, objs), "-lcudart"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    if ptxas_verbose:
        print("\n".join(logs))
    try:
        build_torch_binding(force)
    except RuntimeError as e:  # the library is whole without it
        print(f"rns8_b200.quant is not available: {e}", file=sys.stderr)
    return LIB


def build_torch_binding(force: bool = False) -> Path | None:
    """Compile the torch binding; None where there is nothing to compile it
    against: no torch, one without CUDA, or no Python headers. It is built again
    when its sources, its command, torch or the Python it was built for change. A
    binding that does not compile raises, and leaves none of an earlier build."""
    if importlib.util.find_spec("torch") is None:
        return None
    import torch

    if torch.version.cuda is None or not (Path(sysconfig.get_paths()["include"]) / "Python.h").exists():
        return None
    root = Path(torch.__file__).resolve().parent
    compiler = "/usr/bin/g++" if Path("/usr/bin/g++").exists() else "g++"
    cuda = Path(nvcc()).resolve().parents[1]
    # System headers: their warnings are not ours.
    system = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
              sysconfig.get_paths()["include"], cuda / "include"]
    cmd = [compiler, "-std=c++17", "-O2", "-fPIC", "-shared", "-fvisibility=hidden", "-Wall", "-Wextra",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}",
           *(a for i in system for a in ("-isystem", str(i))),
           str(TORCH_SRC), "-o", str(TORCH_LIB), f"-L{root / 'lib'}", f"-Wl,-rpath,{root / 'lib'}", "-ltorch_python",
           "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda"]
    stamp = BUILD / "_quant_torch.stamp"
    built_for = "\n".join([torch.__version__, sys.version, *cmd])
    # The ABI version and the status codes are compiled in from the other headers.
    newest = max(p.stat().st_mtime for p in (TORCH_SRC, *INCLUDE.glob("rns8/*.h")))
    if (not force and TORCH_LIB.exists() and stamp.exists() and stamp.read_text() == built_for
            and TORCH_LIB.stat().st_mtime >= newest):
        return TORCH_LIB
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        TORCH_LIB.unlink(missing_ok=True)
        raise RuntimeError(f"torch binding failed:\n{' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    if res.stderr.strip():
        print(res.stderr, file=sys.stderr)
    stamp.write_text(built_for)
    return TORCH_LIB


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--ptxas-verbose", action="store_true")
    args = ap.parse_args()
    lib = build(force=args.force, ptxas_verbose=args.ptxas_verbose)
    print(lib)
    return 0


if __name__ == "__main__":
    sys.exit(main())
