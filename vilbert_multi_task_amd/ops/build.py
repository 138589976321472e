"""In-tree build of the gfx950 HIP extension.

Drives hipcc directly (no hipify, no CUDA shims — the sources are native
HIP/CDNA4) and links against the installed PyTorch-ROCm. The resulting
ops/_C/vilbert_hip.so is committed-adjacent (git-ignored) and travels with
the repo snapshot to GPU boxes.

Usage: python -m vilbert_multi_task_amd.ops.build [--force]
"""

from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from typing import List

import torch
import torch.utils.cpp_extension as ce

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "_C")
OUT_SO = os.path.join(OUT_DIR, "vilbert_hip.so")

SOURCES = ["block_fp8.hip", "block_fp8_gemm.hip", "elementwise.hip", "attention.hip", "gemm_mfma.hip", "optim.hip", "attn_bwd.hip", "nms.hip", "roialign.hip", "linear_gelu.hip", "fp8_quant.hip",
    "train_bwd.hip", "bindings.cpp", "block_fp8_bindings.cpp"]
ARCH = os.environ.get("PYTORCH_ROCM_ARCH", "gfx950")


OBJ_DIR = os.path.join(OUT_DIR, "obj")
HEADERS = ["common.h", "block_fp8.h"]


def _mtime(path: str) -> float:
    return os.path.getmtime(path) if os.path.exists(path) else 0.0


def _src_mtime(source: str) -> float:
    return max(os.path.getmtime(os.path.join(CSRC, s)) for s in [source] + HEADERS)


def _object(source: str) -> str:
    return os.path.join(OBJ_DIR, source + ".o")


def _sanitize(asan: bool, ubsan: bool) -> List[str]:
    if ubsan:
        # UndefinedBehaviorSanitizer, host side: no allocator interception,
        # coexists with the HIP runtime (ASan's interceptors do not)
        return ["-Xarch_host", "-fsanitize=undefined",
                "-Xarch_host", "-fno-sanitize=vptr,function",
                "-Xarch_host", "-fno-sanitize-recover=undefined",
                "-shared-libsan", "-g1"]
    if asan:
        # host-side AddressSanitizer (scripts/sanitize.sh); device code is
        # not instrumented
        return ["-Xarch_host", "-fsanitize=address", "-shared-libsan", "-g1"]
    return []


def _compile_command(source: str, sanitize: List[str]) -> List[str]:
    return [
        os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"),
        f"--offload-arch={ARCH}",
        "-O3",
        "-std=c++17",
        "-fPIC",
        "-fno-gpu-rdc",
        # some forms of the packed f32 instructions have given wrong results
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
        "-DUSE_ROCM",
        "-D__HIP_PLATFORM_AMD__",
        "-DTORCH_EXTENSION_NAME=vilbert_hip",
        *sanitize,
        *(f"-I{inc}" for inc in ce.include_paths()),
        "-c", os.path.join(CSRC, source),
    ]


def _link_command(sanitize: List[str]) -> List[str]:
    torch_lib = ce.library_paths()[0]
    return [
        os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"),
        f"--offload-arch={ARCH}", "-shared", "-fPIC", *sanitize,
        *(_object(s) for s in SOURCES),
        f"-L{torch_lib}",
        f"-Wl,-rpath,{torch_lib}",
        "-ltorch",
        "-ltorch_hip",
        "-ltorch_cpu",
        "-lc10",
        "-lc10_hip",
        "-lamdhip64",
        "-lhipblaslt",
    ]


# Beside what is built lies how it was: a file is used again only where it is newer than
# its sources and would be made by the same commands, under the same torch.
def _made_by(*commands: List[str]) -> str:
    return "\n".join([torch.__version__, *(" ".join(c) for c in commands)])


def _is_made_by(path: str, made_by: str) -> bool:
    try:
        with open(path + ".made_by") as f:
            return os.path.exists(path) and f.read() == made_by
    except OSError:
        return False


def _make(path: str, command: List[str], made_by: str, verbose: bool) -> None:
    """Whole or not at all: the file is put in its place when it is done."""
    part = f"{path}.{os.getpid()}.part"
    if verbose:
        print("[vilbert_amd.ops.build]", " ".join(command), "-o", path, flush=True)
    try:
        subprocess.run([*command, "-o", part], check=True)
        if os.path.exists(path + ".made_by"):
            os.remove(path + ".made_by")
        os.replace(part, path)
    finally:
        if os.path.exists(part):
            os.remove(part)
    with open(path + ".made_by", "w") as f:
        f.write(made_by)


def needs_build(asan: bool = False, ubsan: bool = False) -> bool:
    sanitize = _sanitize(asan, ubsan)
    made_by = _made_by(*(_compile_command(s, sanitize) for s in SOURCES), _link_command(sanitize))
    return not _is_made_by(OUT_SO, made_by) or _mtime(OUT_SO) < max(_src_mtime(s) for s in SOURCES)


def build(force: bool = False, verbose: bool = True, asan: bool = False,
          ubsan: bool = False) -> str:
    """Compile what is older than its source or was compiled in another way
    (``force``: everything), one object per source and several at a time, and link."""
    if not force and not needs_build(asan, ubsan):
        return OUT_SO
    os.makedirs(OBJ_DIR, exist_ok=True)
    sanitize = _sanitize(asan, ubsan)

    def compile_one(source: str) -> List[str]:
        obj, command = _object(source), _compile_command(source, sanitize)
        made_by = _made_by(command)
        if force or not _is_made_by(obj, made_by) or _mtime(obj) < _src_mtime(source):
            _make(obj, command, made_by, verbose)
        return command

    jobs = max(1, min(int(os.environ.get("MAX_JOBS") or 8), os.cpu_count() or 1, 16))
    with ThreadPoolExecutor(max_workers=jobs) as pool:
        commands = list(pool.map(compile_one, SOURCES))
    link = _link_command(sanitize)
    _make(OUT_SO, link, _made_by(*commands, link), verbose)
    return OUT_SO


if __name__ == "__main__":
    build(force="--force" in sys.argv, asan="--asan" in sys.argv,
          ubsan="--ubsan" in sys.argv)
    print(f"built {OUT_SO}")
