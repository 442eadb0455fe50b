"""Builds libbzpf.so (the gfx950 HIP kernels behind the C ABI in include/bzpf.h) in-tree with hipcc, and _train.so (the
torch binding of its training operators, host code only).

Each source under csrc/ is compiled to an object in parallel, then linked into boltz_mlx_amd/libbzpf.so and _train.so.
Packed-FP32 instruction selection is disabled for the device code.
"""

from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libbzpf.so")
TRAIN = os.path.join(HERE, "_train.so")
ARCH = os.environ.get("BZPF_ARCH", "gfx950")

HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
CFLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-fPIC", "-std=c++17", "-Wall", "-Wno-unused-function",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMA accumulators in VGPRs: the kernels read every accumulator back with VALU ops (softmax, epilogues),
    # which the AGPR form would route through v_accvgpr moves
    "-mllvm", "-amdgpu-mfma-vgpr-form",
    "-munsafe-fp-atomics", f"-I{INCLUDE}", f"-I{CSRC}",
]


def torch_lib_dir() -> str:
    import importlib.util

    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.submodule_search_locations:
        raise RuntimeError("torch (ROCm build) is required to link against its HIP runtime")
    d = os.path.join(list(spec.submodule_search_locations)[0], "lib")
    if not os.path.exists(os.path.join(d, "libamdhip64.so")):
        raise RuntimeError(f"{d}/libamdhip64.so not found (torch must be a ROCm build)")
    return d


def sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))


# Per-source additions. The fp16 attention core is VALU-bound; without NaN semantics its fmaxf reductions over MFMA
# results need no canonicalising v_max_f32 per logit (its inputs are finite or -inf by construction).
FILE_FLAGS = {"bzpf_triattn_mfma.hip": ["-fno-honor-nans"]}


def torch_flags() -> list[str]:
    """g++ flags of a source that includes torch's extension header and the HIP runtime's (host code only): the compiler
    and settings of torch's own build, whose types and exceptions the binding shares."""
    import torch

    inc = os.path.join(os.path.dirname(torch_lib_dir()), "include")
    rocm = os.path.dirname(os.path.dirname(os.path.realpath(HIPCC)))
    dirs = (inc, os.path.join(inc, "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"],
            os.path.join(rocm, "include"))
    return ["-O2", "-fPIC", "-std=c++17", "-Wall", "-DUSE_ROCM", "-D__HIP_PLATFORM_AMD__=1",
            "-DTORCH_API_INCLUDE_EXTENSION_H", "-DTORCH_EXTENSION_NAME=_train", f'-DBZPF_TORCH="{torch.__version__}"',
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}",
            *(x for d in dirs for x in ("-isystem", d))]


def _compile(src: str) -> str:
    name, ext = os.path.splitext(os.path.basename(src))
    obj = os.path.join(BUILD, name + ".o")
    cmd = ["g++", *torch_flags()] if ext == ".cpp" else [HIPCC, *CFLAGS, *FILE_FLAGS.get(os.path.basename(src), [])]
    cmd += ["-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    err = "\n".join(line for line in (r.stderr or "").splitlines() if noise not in line)
    if r.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed on {os.path.basename(src)}:\n{err}")
    if err.strip():
        print(err, file=sys.stderr)
    return obj


def _link(out: str, objs: list[str], *libs: str) -> None:
    """A shared object at `out`, against torch's libraries, which it finds where they are now."""
    tlib = torch_lib_dir()
    r = subprocess.run(["g++", "-shared", "-fPIC", *objs, "-o", out + ".tmp", f"-L{tlib}", f"-Wl,-rpath,{tlib}",
                        *(f"-l:{lib}" for lib in libs)], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link of {os.path.basename(out)} failed:\n{r.stderr}")
    os.replace(out + ".tmp", out)


def build(verbose: bool = True) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sources()
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs) + 1)) as ex:
        binding = ex.submit(_compile, os.path.join(CSRC, "bzpf_torch.cpp"))  # first: torch's headers take the longest
        objs = list(ex.map(_compile, srcs))
    # Link against the HIP runtime that torch loads (torch/lib/libamdhip64.so), so that the library and torch
    # share one runtime instance (and one device context) in the process.
    _link(LIB, objs, "libamdhip64.so")
    # The library stands before the binding's result is asked for: inference needs it alone. A binding of earlier sources
    # goes where there is no new one.
    if binding.exception() is not None and os.path.exists(TRAIN):
        os.remove(TRAIN)
    _link(TRAIN, [binding.result()], "libtorch_python.so", "libtorch.so", "libtorch_cpu.so", "libc10_hip.so", "libc10.so",
          "libamdhip64.so")
    if verbose:
        print(f"built {LIB} and {os.path.basename(TRAIN)} from {len(srcs) + 1} sources")
    return LIB


if __name__ == "__main__":
    build()
