"""Builds libntc_b200.so (the CUDA kernels, the host engine, the C ABI and the ntc_cuda::Trainer
class) in-tree with nvcc for sm_100a, and, where torch is installed, libntc_b200_torch.so (the host side of the operators on
torch tensors) with the C++ compiler. Run `python -m neural_block_textures_b200.build`."""
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
OUT_DIR = PKG / "_lib"
BUILD_DIR = PKG / "_build"
LIB = OUT_DIR / "libntc_b200.so"
TORCH_LIB = OUT_DIR / "libntc_b200_torch.so"
TORCH_SOURCE = "torch_host.cpp"
SOURCES = ["kernels_mlp.cu", "kernels_tc.cu", "kernels_latent.cu", "kernels_snap.cu", "kernels_stats.cu", "engine.cu",
           "ntcb_format.cpp", "ntcb_decoder.cu",
           "static_scratch.cu", "nccl_link.cpp", "p2p_exchange.cu", "device_cache.cu", "symbol_logprob.cu",
           "symbol_logprob_f32.cu", "symbol_logprob_f16.cu", "symbol_logprob_bf16.cu", "adamw.cu"]
GENCODE = ["-gencode", "arch=compute_100a,code=sm_100a"]
# No fast-math: the noise (logf / cosf / sqrtf), the sigmoid (expf) and every division must be CUDA's
# IEEE / accurate versions for parity with the reference backend.
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills"]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand


def _deps(src: Path) -> list[Path]:
    return [src, *sorted(CSRC.glob("*.cuh")), *sorted(CSRC.glob("*.h")), *sorted((ROOT / "include").glob("*.h"))]


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _compile(src: str, verbose: bool) -> Path:
    s = CSRC / src
    obj = BUILD_DIR / (src + ".o")
    if not _stale(obj, _deps(s)):
        return obj
    cmd = [nvcc(), *GENCODE, *NVCC_FLAGS, "-c", str(s), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    if verbose:
        sys.stderr.write(r.stderr)
    return obj


def _torch_host_lacks() -> str | None:
    """What keeps the torch library from being built here, if something does. The rest of the package needs neither."""
    if importlib.util.find_spec("torch") is None:
        return "torch is not installed"
    if not (Path(sysconfig.get_paths()["include"]) / "Python.h").exists():
        return "Python's headers are not installed"
    return None


def _torch_built_for(torch: Path) -> str:
    """What the torch library's code depends on beside its sources: torch's C++ classes and the interpreter's ABI."""
    return "\n".join([str(torch), (torch / "version.py").read_text(), sys.implementation.cache_tag, str(sysconfig.get_config_var("SOABI"))])


def _compile_torch_host() -> Path:
    """torch_host.cpp against the installed torch's headers."""
    s = CSRC / TORCH_SOURCE
    obj = BUILD_DIR / (TORCH_SOURCE + ".o")
    stamp = BUILD_DIR / (TORCH_SOURCE + ".torch")   # the torch that the object is for
    torch = Path(importlib.util.find_spec("torch").submodule_search_locations[0])
    if not _stale(obj, _deps(s)) and stamp.exists() and stamp.read_text() == _torch_built_for(torch):
        return obj
    cuda = Path(nvcc()).resolve().parent.parent
    inc = [torch / "include", torch / "include" / "torch" / "csrc" / "api" / "include", cuda / "include", sysconfig.get_paths()["include"]]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", *[f"-I{d}" for d in inc], "-c", str(s), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed for {TORCH_SOURCE}:\n{r.stdout}\n{r.stderr}")
    stamp.write_text(_torch_built_for(torch))
    return obj


def _link_torch_host(obj: Path) -> None:
    if not _stale(TORCH_LIB, [obj, LIB]):
        return
    torch = Path(importlib.util.find_spec("torch").submodule_search_locations[0])
    cmd = [os.environ.get("CXX", "g++"), "-shared", "-o", str(TORCH_LIB), str(obj), f"-L{OUT_DIR}", "-l:" + LIB.name, "-Wl,-rpath,$ORIGIN",
           f"-L{torch / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10_cuda", "-lc10"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")


def build(verbose: bool = False) -> Path:
    OUT_DIR.mkdir(exist_ok=True)
    BUILD_DIR.mkdir(exist_ok=True)
    lacks = _torch_host_lacks()
    with cf.ThreadPoolExecutor(max_workers=len(SOURCES) + 1) as ex:
        host = None if lacks else ex.submit(_compile_torch_host)
        objs = list(ex.map(lambda s: _compile(s, verbose), SOURCES))
    if _stale(LIB, objs):
        cmd = [nvcc(), *GENCODE, "-shared", "-Xcompiler", "-fPIC", "-o", str(LIB), *map(str, objs), "-cudart", "static"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    if lacks:
        sys.stderr.write(f"{TORCH_LIB.name} is left out: {lacks}\n")
    else:
        _link_torch_host(host.result())   # LIB is there whatever becomes of this
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
