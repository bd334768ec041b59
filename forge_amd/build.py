"""Build the gfx950 shared library in-tree with hipcc.

    python -m forge_amd.build          # -> forge_amd/libforge_q.so, forge_amd/_step.so

The library is compiled for gfx950 only.  Packed-FP32 instruction selection
is disabled (-packed-fp32-ops) for every HIP translation unit.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libforge_q.so")
STEP = os.path.join(HERE, "_step.so")
OBJDIR = os.path.join(HERE, "_build")

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"

SOURCES = ["fq_dequant.hip", "fq_gemv1.hip", "fq_gemvp.hip", "fq_gemvt.hip", "fq_pack.hip", "fq_mmq.hip",
           "fq_mmqi.hip", "fq_mmqs.hip", "fq_mmqp.hip", "fq_mmqk.hip", "fq_mmqt.hip",
           "fq_plan.hip", "fq_rope.hip", "fq_attn.hip", "fq_logp.hip", "fq_step_capi.cpp",
           "fq_capi.cpp"]

COMMON = [
    "-O3", "-std=c++17", "-fPIC", f"--offload-arch={ARCH}",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument", "-I", os.path.join(ROOT, "include"),
]


# Per-file flags.  The prefill kernel adds one FMA per block to each of its 64
# MFMA results per lane: with the results in AGPRs (the compiler's default
# under that register pressure) every FMA needs a v_accvgpr_read first, so
# the MFMA results are kept in VGPRs.
EXTRA = {f: ["-mllvm", "-amdgpu-mfma-vgpr-form"] for f in ("fq_mmqp.hip", "fq_mmqk.hip", "fq_mmqt.hip")}


def _compile(src: str) -> str:
    obj = os.path.join(OBJDIR, os.path.basename(src) + ".o")
    lang = [] if src.endswith(".hip") else ["-x", "hip"]
    cmd = [HIPCC, *COMMON, *EXTRA.get(src, []), *lang, "-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stderr}")
    return obj


def _binding() -> None:
    """forge_amd/_step.so: the step operators' host side over torch tensors, a plain
    CPython extension that calls the library's C ABI.  Without torch, its or Python's
    headers or g++ it is left out (and one of an earlier library removed):
    forge_amd.step is not there then, the library is."""
    import sysconfig

    try:
        import torch
        from torch.utils import cpp_extension
        include = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"]]
        missing = next((h for h in ("torch/csrc/autograd/python_variable.h", "Python.h")
                        if not any(os.path.exists(os.path.join(p, h)) for p in include)),
                       None if shutil.which("g++") else "g++")
    except ImportError:
        missing = "torch"
    if missing:
        if os.path.exists(STEP):
            os.remove(STEP)
        print(f"no {missing}: {os.path.basename(STEP)} (forge_amd.step) is not built")
        return
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    tmp = STEP + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-isystem{p}" for p in include), os.path.join(CSRC, "fq_step_py.cpp"),
           "-o", tmp, f"-L{HERE}", "-l:libforge_q.so", "-Wl,-rpath,$ORIGIN", f"-L{lib}", "-lc10",
           "-ltorch_cpu", "-ltorch_python", f"-Wl,-rpath,{lib}"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for fq_step_py.cpp:\n{r.stderr}")
    os.replace(tmp, STEP)


def build(verbose: bool = True) -> str:
    os.makedirs(OBJDIR, exist_ok=True)
    srcs = [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    with ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(_compile, srcs))
    tmp = OUT + ".tmp"
    cmd = [HIPCC, "-shared", "-fPIC", f"--offload-arch={ARCH}", *objs, "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, OUT)
    _binding()
    if verbose:
        print(f"built {OUT}")
    return OUT


if __name__ == "__main__":
    build()
    sys.exit(0)
