"""Build the sm_100a shared library ``libpkv.so`` in-tree with nvcc.

    python mini_inference_b200/build.py        # runs without importing the package (which loads the library)

Every ``csrc/*.cu`` and ``csrc/*.cpp`` is compiled for
``-gencode arch=compute_100a,code=sm_100a`` into ``_build/`` (in parallel; a file
is rebuilt only when it or a header changed) and linked with the static CUDA
runtime into ``mini_inference_b200/libpkv.so``. nvcc cross-compiles, so no GPU
is needed to build. ``csrc/bindings/speculative.cpp`` (tensors to the C ABI for the calls
of a speculative decoding step) becomes ``mini_inference_b200/_speculative.<python tag>.so``,
compiled by g++ against the installed torch's headers and linked to ``libpkv.so``.
"""

from __future__ import annotations

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
INCLUDE = ROOT / "include"
BUILD = ROOT / "_build"
LIB = PKG / "libpkv.so"
SUFFIX = sysconfig.get_config_var("EXT_SUFFIX")  # of this Python
BINDING = PKG / ("_speculative" + SUFFIX)
BINDING_SRC = CSRC / "bindings" / "speculative.cpp"
BINDINGS = [(BINDING, BINDING_SRC), (PKG / ("_layer" + SUFFIX), CSRC / "bindings" / "layer.cpp")]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
         "--expt-relaxed-constexpr", "-I", str(INCLUDE)]


def nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(exe).exists():
        raise RuntimeError("nvcc not found: the CUDA toolkit is needed to build libpkv.so")
    return exe


def _headers() -> list[Path]:
    return list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h"))


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _compile(src: Path, verbose_ptxas: bool) -> Path:
    obj = BUILD / (src.name + ".o")
    if not _stale(obj, [src] + _headers()) and not verbose_ptxas:
        return obj
    cmd = [nvcc(), *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
    if verbose_ptxas and src.suffix == ".cu":
        cmd.insert(1, "-Xptxas=-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{res.stdout}\n{res.stderr}")
    if verbose_ptxas:
        sys.stderr.write(res.stderr)
    return obj


def _bind(binding: Path, source: Path) -> Path:
    """A compiled binding: rebuilt when its source, the C ABI or the torch it was built against changed."""
    spec = importlib.util.find_spec("torch")  # found, not imported: that takes seconds
    if spec is None or not spec.submodule_search_locations:
        raise RuntimeError("torch not found: its headers are needed to build the binding")
    torch_dir = Path(spec.submodule_search_locations[0])
    include = torch_dir / "include"
    # By torch's version and place: its files may be older than the binding of another torch.
    against = f"{torch_dir}\n{(torch_dir / 'version.py').read_text()}"
    stamp = BUILD / (binding.name + ".torch")
    deps = [source, source.with_name("common.h"), INCLUDE / "pkv.h"]
    if not _stale(binding, deps) and stamp.exists() and stamp.read_text() == against:
        return binding
    cuda = Path(nvcc()).resolve().parent.parent / "include"
    tmp = binding.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-I", sysconfig.get_paths()["include"]]
    for path in (include, include / "torch" / "csrc" / "api" / "include", cuda):
        cmd += ["-isystem", str(path)]
    cmd += [str(source), "-o", str(tmp), "-L", str(PKG), "-l:libpkv.so", "-Wl,-rpath,$ORIGIN", "-L",
            str(torch_dir / "lib"), "-ltorch_python", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on {source.name}:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, binding)
    stamp.write_text(against)
    return binding


def build(verbose_ptxas: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cpp"))
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose_ptxas), sources))
    if _stale(LIB, objs) or verbose_ptxas:
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *map(str, objs)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
        os.replace(tmp, LIB)
    with cf.ThreadPoolExecutor(max_workers=len(BINDINGS)) as ex:
        list(ex.map(lambda b: _bind(*b), BINDINGS))
    return LIB


if __name__ == "__main__":
    print(build(verbose_ptxas="-v" in sys.argv))
