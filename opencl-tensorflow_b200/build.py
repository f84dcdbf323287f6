"""Build the B200 backend library in-tree.

Compiles every ``csrc/*.cu`` for sm_100a with nvcc (in parallel, each object
rebuilt only when its source or a header changed) and links them into
``opencl_tf/libb2ocl.so``, the C-ABI library declared in
``include/b2_opencl_tf.h``; and compiles ``torch_binding/*.cpp``, torch's side
of some of its entries, into extension modules of the package with g++.  Usage::

    python opencl-tensorflow_b200/build.py [--force] [--verbose-ptxas]
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
OBJ = PKG / "_build"
LIB = PKG / "opencl_tf" / "libb2ocl.so"
BINDING = PKG / "torch_binding"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
         "-Xcompiler", "-Wall", "-I", str(INCLUDE), "-I", str(CSRC)]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _newest_header() -> float:
    hs = list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    return max((h.stat().st_mtime for h in hs), default=0.0)


def _compile(src: Path, force: bool, ptxas_v: bool) -> tuple[Path, str]:
    obj = OBJ / (src.stem + ".o")
    if not force and obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, _newest_header()):
        return obj, ""
    cmd = [nvcc(), *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
    if ptxas_v:
        cmd += ["-Xptxas", "-v"]
    out = subprocess.run(cmd, capture_output=True, text=True)
    if out.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{out.stdout}\n{out.stderr}")
    return obj, out.stderr if ptxas_v else ""


def _compile_binding(src: Path, force: bool) -> Path:
    """``opencl_tf/_<stem>.so`` from ``torch_binding/<stem>.cpp``, by the system's compiler: another one (from
    ``CXX``, say) may link parts of a libstdc++ beside the one that torch has loaded.  Built again when its sources
    are newer, or with another Python, torch or command than ``_build/_<stem>.stamp`` names."""
    import torch
    from torch.utils import cpp_extension
    out, stamp = PKG / "opencl_tf" / f"_{src.stem}.so", OBJ / f"_{src.stem}.stamp"
    cuda = Path(nvcc()).resolve().parent.parent
    includes = [a for p in cpp_extension.include_paths() for a in ("-isystem", p)]
    libs = [a for p in cpp_extension.library_paths() for a in ("-L", p)]
    system = "/usr/bin/g++"
    cmd = [system if os.path.exists(system) else "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
           f"-DTORCH_EXTENSION_NAME=_{src.stem}", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *includes, "-isystem", str(cuda / "include"), "-isystem", sysconfig.get_paths()["include"],
           "-I", str(INCLUDE), str(src), *libs, "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python"]
    built_with = "\n".join([sys.version, torch.__version__, *cmd])
    newest = max(p.stat().st_mtime for p in (src, INCLUDE / "b2_opencl_tf.h"))
    if (not force and out.exists() and out.stat().st_mtime >= newest and stamp.exists()
            and stamp.read_text() == built_with):
        return out
    part = out.with_suffix(f".{os.getpid()}.part")  # a process that has the old one loaded keeps it
    res = subprocess.run([*cmd, "-o", str(part)], capture_output=True, text=True)
    if res.returncode != 0:
        part.unlink(missing_ok=True)
        raise RuntimeError(f"g++ failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    os.replace(part, out)
    stamp.write_text(built_with)
    return out


def build(force: bool = False, ptxas_v: bool = False, quiet: bool = True) -> Path:
    OBJ.mkdir(exist_ok=True)
    srcs = sorted(CSRC.glob("*.cu"))
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        bindings = [ex.submit(_compile_binding, s, force) for s in sorted(BINDING.glob("*.cpp"))]
        results = list(ex.map(lambda s: _compile(s, force, ptxas_v), srcs))
    objs = [r[0] for r in results]
    if ptxas_v and not quiet:
        for _, log in results:
            sys.stdout.write(log)
    newest_obj = max(o.stat().st_mtime for o in objs)
    if force or not LIB.exists() or LIB.stat().st_mtime < newest_obj:
        cmd = [nvcc(), *ARCH, "-shared", "-o", str(LIB), *map(str, objs), "-lcudart"]
        out = subprocess.run(cmd, capture_output=True, text=True)
        if out.returncode != 0:
            raise RuntimeError(f"link failed:\n{out.stdout}\n{out.stderr}")
    for b in bindings:  # what fails here leaves the library, which needs no torch, built
        b.result()
    if not quiet:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose-ptxas", action="store_true")
    a = ap.parse_args()
    build(force=a.force, ptxas_v=a.verbose_ptxas, quiet=False)
