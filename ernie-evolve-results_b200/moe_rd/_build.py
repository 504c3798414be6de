"""Builds libmoe_rd.so in-tree with nvcc for sm_100a and _fastcall.so with the host compiler (no GPU needed to compile)."""
from __future__ import annotations

import os
import subprocess
import sys
import warnings
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent.parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
LIB = PKG / "moe_rd" / "libmoe_rd.so"
FASTCALL = PKG / "moe_rd" / "_fastcall.so"  # Python module: the ordinary call without Python in between

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    # keep every multiply and add a separate IEEE operation unless fmaf() is written
    "-fmad=false", "-Xcompiler", "-fPIC", "-Xptxas", "-v",
]


def _nvcc() -> str:
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if c and (os.path.sep not in c or os.path.exists(c)):
            return c
    raise RuntimeError("nvcc not found")


def fastcall_stamp() -> str:
    """What _fastcall.so is compiled for: it reads torch's and Python's objects in place, as their headers lay them out."""
    import sysconfig
    import torch
    return f"moe_rd fastcall for torch {torch.__version__} {torch.version.git_version}, {sysconfig.get_config_var('SOABI')}"


def fastcall_fits() -> bool:
    """Whether the _fastcall.so that is there was compiled for the torch and Python that run (seen without loading it)."""
    return fastcall_stamp().encode() + b"\0" in FASTCALL.read_bytes()


def build_fastcall(force: bool = False) -> Path:
    """csrc/fastcall.cpp against the headers of the installed torch and Python.  Written beside the module and moved in its
    place; a module that is out of date does not stay where the new one fails."""
    src = CSRC / "fastcall.cpp"
    if (not force and FASTCALL.exists() and all(FASTCALL.stat().st_mtime >= d.stat().st_mtime for d in (src, INCLUDE / "moe_rd.h"))
            and fastcall_fits()):
        return FASTCALL
    import sysconfig
    import torch
    root = Path(torch.__file__).resolve().parent
    FASTCALL.unlink(missing_ok=True)
    made = FASTCALL.with_name(f"{FASTCALL.name}.{os.getpid()}.tmp")
    cxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"
    include = [INCLUDE, sysconfig.get_paths()["include"], root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
               Path(_nvcc()).resolve().parent.parent / "include"]
    cmd = [cxx, "-O2", "-Wall", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DMOE_RD_BUILT_FOR="{fastcall_stamp()}"',
           *[f"-I{i}" for i in include], str(src), "-o", str(made), f"-L{root / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        made.unlink(missing_ok=True)
        raise RuntimeError(f"g++ failed on {src.name}:\n{r.stdout}\n{r.stderr}")
    os.replace(made, FASTCALL)
    return FASTCALL


def build(force: bool = False, verbose: bool = False) -> Path:
    with ThreadPoolExecutor(max_workers=1) as ex:  # beside nvcc
        fastcall = ex.submit(build_fastcall, force)
        lib = build_library(force, verbose)
        try:
            fastcall.result()
        except Exception as e:  # no torch headers, no g++: the library is whole and every call runs without the module
            warnings.warn(f"moe_rd: _fastcall.so is not built, the calls go through Python: {e}")
    return lib


def build_library(force: bool = False, verbose: bool = False) -> Path:
    srcs = sorted(CSRC.glob("*.cu"))
    deps = srcs + sorted(CSRC.glob("*.cuh")) + [INCLUDE / "moe_rd.h"]
    if not force and LIB.exists() and all(LIB.stat().st_mtime >= d.stat().st_mtime for d in deps):
        return LIB
    objdir = PKG / "build"
    objdir.mkdir(exist_ok=True)
    # the host compiler must be the system one (an environment CC may lack its specs)
    ccbin = ["-ccbin", "/usr/bin/g++"] if os.path.exists("/usr/bin/g++") else []

    def compile_one(src: Path):
        obj = objdir / (src.stem + ".o")
        cmd = [_nvcc(), *ccbin, *NVCC_FLAGS, "-I", str(INCLUDE), "-I", str(CSRC), "-c", str(src), "-o", str(obj)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        return src, obj, r

    with ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        results = list(ex.map(compile_one, srcs))
    log = []
    for src, obj, r in results:
        log.append(f"== {src.name}\n{r.stderr}")
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
    (objdir / "ptxas.log").write_text("\n".join(log))
    if verbose:
        print("\n".join(log))
    cmd = [_nvcc(), *ccbin, "-shared", "-o", str(LIB), *[str(o) for _, o, _ in results], "-lcudart"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
