"""Build the native libraries in-tree with nvcc for sm_100a.

    python -m soap_tp_b200.build_ext            # incremental (skips a library whose sources are older than it)
    python -m soap_tp_b200.build_ext --force

``soap_tp_b200/_C*.so`` (``csrc``) is a plain pybind11 module (no ATen): the optimizer.  ``soap_tp_b200/_decoder*.so``
(``csrc/decoder``) holds the operators of a decoder's training step as torch operators and is compiled against the installed torch.
``.cu`` files are compiled with ``nvcc -gencode arch=compute_100a,code=sm_100a -lineinfo`` and linked into one shared object
per library next to this file, so a source checkout plus this command is all a GPU box needs.  nvcc cross-compiles
without a GPU.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
BUILD = HERE / "csrc" / "build"
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


LIBRARIES = {"_C": CSRC, "_decoder": CSRC / "decoder"}


def target_path(library: str = "_C") -> Path:
    return HERE / (library + sysconfig.get_config_var("EXT_SUFFIX"))


def sources(library: str = "_C") -> list[Path]:
    folder = LIBRARIES[library]
    return sorted(list(folder.glob("*.cu")) + list(folder.glob("*.cpp")))


def _includes() -> list[str]:
    import pybind11

    return [f"-I{pybind11.get_include()}", f"-I{sysconfig.get_paths()['include']}", f"-I{CSRC}"]


def _nvcc() -> str:
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    candidate = Path(cuda_home) / "bin" / "nvcc"
    return str(candidate) if candidate.exists() else "nvcc"


def _torch_flags(library: str) -> tuple[list[str], list[str]]:
    """Flags that compile and link against torch, for the host sources of the library that uses it."""
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parents[1] if Path(_nvcc()).is_absolute() else Path("/usr/local/cuda")
    include = root / "include"
    compile_flags = [f"-I{include}", f"-I{include / 'torch' / 'csrc' / 'api' / 'include'}", f"-I{cuda / 'include'}",
                     f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f"-DTORCH_EXTENSION_NAME={library}"]
    link_flags = [f"-L{root / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"]
    return compile_flags, link_flags


def needs_build(library: str = "_C") -> bool:
    target = target_path(library)
    if not target.exists():
        return True
    headers = [p for folder in {CSRC, LIBRARIES[library]} for pattern in ("*.h", "*.cuh") for p in folder.glob(pattern)]
    newest = max(p.stat().st_mtime for p in sources(library) + headers)
    return newest > target.stat().st_mtime


def build(force: bool = False, verbose: bool = False) -> Path:
    """Builds what is out of date (``force``: everything) and returns the optimizer's library."""
    libraries = [name for name in LIBRARIES if force or needs_build(name)]
    common = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
              "--expt-relaxed-constexpr", *ARCH_FLAGS, *_includes()]
    if os.environ.get("SOAP_GEMM_TERMS"):
        common += [f"-DSOAP_GEMM_TERMS={int(os.environ['SOAP_GEMM_TERMS'])}"]     # timing experiments (see gemm_tf32x3.cu)
    if os.environ.get("SOAP_QR_TRACE", "0") == "1":
        common += ["-DSOAP_QR_TRACE"]     # clock64 stamps in the one-column QR panel kernel (kernel_cases --trace)
    if verbose:
        common += ["-Xptxas", "-v"]
    torch_compile, torch_link = _torch_flags("_decoder") if "_decoder" in libraries else ([], [])

    def run(cmd: list[str], what: str) -> None:
        result = subprocess.run(cmd, capture_output=True, text=True)
        if result.returncode != 0:
            raise RuntimeError(f"{what} failed:\n{result.stdout}\n{result.stderr}")
        if verbose and result.stderr:
            print(result.stderr, file=sys.stderr)

    def compile_one(job: tuple[str, Path]) -> Path:
        library, src = job
        folder = BUILD / library
        folder.mkdir(parents=True, exist_ok=True)
        obj = folder / (src.stem + ".o")
        if library == "_decoder" and src.suffix == ".cpp":      # torch's headers go to the host compiler alone
            run(["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", *torch_compile, *_includes(), "-c", str(src), "-o", str(obj)],
                f"g++ for {src.name}")
            return obj
        run([_nvcc(), *common, "-x", "cu" if src.suffix == ".cu" else "c++", "-c", str(src), "-o", str(obj)], f"nvcc for {src.name}")
        return obj

    jobs = [(library, src) for library in libraries for src in sources(library)]
    jobs.sort(key=lambda job: job[1].name != "decoder.cpp")      # the longest first
    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        objects = list(zip(jobs, pool.map(compile_one, jobs)))
    for library in libraries:
        mine = [str(obj) for (name, _), obj in objects if name == library]
        target = target_path(library)
        fresh = target.with_name(target.name + ".new")      # (a process that has the old one loaded keeps it)
        run([_nvcc(), "-shared", *ARCH_FLAGS, "-o", str(fresh), *mine, *(torch_link if library == "_decoder" else []), "-lcudart"],
            f"link of {library}")
        os.replace(fresh, target)
    return target_path()


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(path)
