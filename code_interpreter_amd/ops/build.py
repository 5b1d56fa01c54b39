"""In-tree build of the gfx950 extensions (_hipops, _hipgemm, _hiplm).

hipcc cross-compiles without a GPU, and the resulting .so lives next to
this file (in-tree, so it travels to GPU boxes with the repo snapshot).

Usage: python -m code_interpreter_amd.ops.build [--force]
"""

import importlib.util
import os
import subprocess
import sys
import sysconfig
import tempfile
from pathlib import Path

OPS_DIR = Path(__file__).resolve().parent
HIP_DIR = OPS_DIR / "hip"
OUTPUT = OPS_DIR / "_hipops.so"

GEMM_SOURCES = [
    HIP_DIR / "gemm_f32.hip",
    HIP_DIR / "gemm_f64.hip",
    HIP_DIR / "gemm_bf16.hip",
    HIP_DIR / "gemm_bf16_256.hip",
]
SOURCES = [
    HIP_DIR / "hipops.cpp",
    HIP_DIR / "kernels_ew.hip",
    HIP_DIR / "sort.hip",
    *GEMM_SOURCES,
]
# _hipgemm: the torch-interop module. Built SEPARATELY because zygote
# children fork with _hipops pre-imported, and a fat-binary registered
# pre-fork cannot be launched after the child re-initializes HIP (torch
# init) -- the torch routing layer dlopens this fresh per child.
GEMM_OUTPUT = OPS_DIR / "_hipgemm.so"
GEMM_MODULE_SOURCES = [HIP_DIR / "hipgemm.cpp", *GEMM_SOURCES]

# _hiplm: the language-model kernels, for torch tensors too.
LM_OUTPUT = OPS_DIR / "_hiplm.so"
LM_MODULE_SOURCES = [
    HIP_DIR / "hiplm.cpp",
    HIP_DIR / "mxfp4_quant.hip",
    HIP_DIR / "mxfp4_gemm.hip",
    HIP_DIR / "scoring.hip",
]
# host code against torch's headers
TORCH_SOURCES = {HIP_DIR / "hiplm.cpp"}
MODULES = [
    (OUTPUT, SOURCES),
    (GEMM_OUTPUT, GEMM_MODULE_SOURCES),
    (LM_OUTPUT, LM_MODULE_SOURCES),
]

ARCH = os.environ.get("PYTORCH_ROCM_ARCH", "gfx950")


def _needs(output: Path, sources) -> bool:
    if not output.exists():
        return True
    out_mtime = output.stat().st_mtime
    deps = [*sources, *HIP_DIR.glob("*.h"), Path(__file__)]
    return any(p.stat().st_mtime > out_mtime for p in deps)


def _torch_dir() -> Path | None:
    """Where torch for ROCm is, if it is here."""
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.submodule_search_locations:
        return None
    path = Path(spec.submodule_search_locations[0])
    return path if (path / "lib" / "libtorch_hip.so").exists() else None


def _buildable(sources) -> bool:
    """What takes torch's tensors is of use, and built, only next to it."""
    return TORCH_SOURCES.isdisjoint(sources) or _torch_dir() is not None


def needs_build() -> bool:
    return any(_needs(out, sources) for out, sources in MODULES
               if _buildable(sources))


def _run(cmd, verbose: bool) -> None:
    if verbose:
        print("+", " ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)


def _compile_torch(source: Path, output: Path, verbose: bool) -> None:
    include = _torch_dir() / "include"
    _run([
        os.environ.get("CXX", "g++"),
        "-O2", "-std=c++17", "-fPIC", "-c", str(source), "-o", str(output),
        "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-DHIPBLAS_V2",
        f"-I{include}", f"-I{include}/torch/csrc/api/include",
        f"-I{os.environ.get('ROCM_PATH', '/opt/rocm')}/include",
        f"-I{sysconfig.get_paths()['include']}", f"-I{HIP_DIR}",
    ], verbose)


def _compile(output: Path, sources, verbose: bool) -> None:
    hipcc = os.environ.get("HIPCC", "hipcc")
    py_include = sysconfig.get_paths()["include"]
    with tempfile.TemporaryDirectory() as scratch:
        cmd = [
            hipcc,
            f"--offload-arch={ARCH}",
            "-O3",
            # packed fp32 arithmetic, which the compiler makes of ordinary
            # float code, has given wrong results in some of its forms
            "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
            "-std=c++17",
            "-fPIC",
            "-shared",
            "-x", "hip",
            *[str(s) for s in sources if s not in TORCH_SOURCES],
            f"-I{py_include}",
            f"-I{HIP_DIR}",
            "-o",
            str(output),
        ]
        with_torch = [s for s in sources if s in TORCH_SOURCES]
        for source in with_torch:
            obj = Path(scratch) / (source.stem + ".o")
            _compile_torch(source, obj, verbose)
            cmd += ["-x", "none", str(obj)]
        if with_torch:
            # loaded after torch, which has them in the process already
            cmd += [f"-L{_torch_dir() / 'lib'}", "-ltorch_python",
                    "-ltorch_hip", "-ltorch_cpu", "-lc10_hip", "-lc10"]
        _run(cmd, verbose)


def build(force: bool = False, verbose: bool = True) -> Path:
    for out, sources in MODULES:
        if not _buildable(sources):
            print(f"{out.name} is not built: there is no torch for ROCm here",
                  flush=True)
        elif force or _needs(out, sources):
            _compile(out, sources, verbose)
    return OUTPUT


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(f"built {OUTPUT}")
