"""In-tree build of ``libe4b_amd.so`` for gfx950 with ``hipcc`` (no cmake, no JIT cache).

``python -m experts4bit_qlora_amd._build`` (or ``__graft_entry__.build()``) compiles
``csrc/e4b_amd.hip`` (entry points and the routing / dequant / GEMV / LoRA / training kernels),
``csrc/mx_gemm.hip`` (the products of microscaled operands), ``csrc/gate.hip`` (the router's kernels), ``csrc/losses.hip`` (the losses over the vocabulary), and ``csrc/decode_inst.hip`` and ``csrc/gemm_inst.hip`` once per (activation dtype, weight format)
pair, all in parallel, then links them into ``experts4bit_qlora_amd/libe4b_amd.so``. The output is written to a temporary
name and renamed, so a failed build never leaves a half-written library behind. ``csrc/torch_losses.cpp``, host code that calls
the library from torch's autograd, becomes ``experts4bit_qlora_amd/libe4b_torch.so`` the same way, with the host compiler and
torch's headers; the library is built without it where that fails or is not asked for (``build(binding=False)``).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor

_HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_HERE, "csrc")
SRC = os.path.join(CSRC, "e4b_amd.hip")
DECODE_SRC = os.path.join(CSRC, "decode_inst.hip")
GEMM_SRC = os.path.join(CSRC, "gemm_inst.hip")
MX_SRC = os.path.join(CSRC, "mx_gemm.hip")
GATE_SRC = os.path.join(CSRC, "gate.hip")
LOSSES_SRC = os.path.join(CSRC, "losses.hip")
TORCH_SRC = os.path.join(CSRC, "torch_losses.cpp")
INCLUDE = os.path.join(os.path.dirname(_HERE), "include")
# (E4B_INST_DT, E4B_INST_FMT): bf16/fp16 x NF4/NF4_DQ/MXFP4
DECODE_PAIRS = [(dt, fmt) for dt in (0, 1) for fmt in (0, 1, 2)]
OUT = os.path.join(_HERE, "libe4b_amd.so")
TORCH_OUT = os.path.join(_HERE, "libe4b_torch.so")
ARCH = os.environ.get("E4B_OFFLOAD_ARCH", "gfx950")

FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # no silent a*b+c contraction: FMAs are written explicitly where they are wanted, and the
    # dequant / combine products must round exactly once
    "-ffp-contract=off",
    # packed fp32 (v_pk_*_f32) is not generated
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm)")


def _run_all(cmds):
    procs = [(cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)) for cmd in cmds]
    noise = "is not a recognized feature for this target"
    msgs, failed = [], []
    for cmd, p in procs:
        _, err = p.communicate()
        err = "\n".join(l for l in err.splitlines() if noise not in l)
        if p.returncode != 0:
            failed.append(f"{os.path.basename(cmd[0])} failed ({p.returncode}):\n{' '.join(cmd)}\n{err}")
        elif err.strip():
            msgs.append(err)
    if failed:
        raise RuntimeError("\n\n".join(failed))
    return msgs


def _torch_commands(obj: str, out: str):
    """(compile, link) of the extension that binds the library to torch's autograd."""
    from torch.utils import cpp_extension

    cxx = os.environ.get("CXX") or shutil.which("g++") or "c++"
    inc = [f"-I{p}" for p in (INCLUDE, *cpp_extension.include_paths("cuda"), sysconfig.get_paths()["include"])]
    libs = [f"-L{p}" for p in cpp_extension.library_paths("cuda")] + [
        "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-ltorch_python", "-lc10", "-lc10_hip"]
    compile_ = [cxx, "-O2", "-std=c++17", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM", *inc, "-c", "-o", obj, TORCH_SRC]
    link = [cxx, "-shared", "-o", out, obj, *libs, f"-L{_HERE}", "-l:libe4b_amd.so", "-Wl,-rpath,$ORIGIN"]
    return compile_, link


def _library(tmpdir: str) -> list[str]:
    """libe4b_amd.so: the messages of its compilation. A binding of an older library goes with that library."""
    cc = hipcc()
    inc = [f"-I{CSRC}", f"-I{INCLUDE}"]
    objs, cmds = [], []
    for name, src in (("e4b_amd.o", SRC), ("mx_gemm.o", MX_SRC), ("gate.o", GATE_SRC),
                      ("losses.o", LOSSES_SRC)):
        obj = os.path.join(tmpdir, name)
        cmds.append([cc, *FLAGS, *inc, "-c", "-o", obj, src])
        objs.append(obj)
    for dt, fmt in DECODE_PAIRS:
        obj = os.path.join(tmpdir, f"decode_{dt}_{fmt}.o")
        cmds.append([cc, *FLAGS, *inc, f"-DE4B_INST_DT={dt}", f"-DE4B_INST_FMT={fmt}", "-c", "-o", obj,
                     DECODE_SRC])
        objs.append(obj)
        obj = os.path.join(tmpdir, f"gemm_{dt}_{fmt}.o")
        cmds.append([cc, *FLAGS, *inc, f"-DE4B_INST_DT={dt}", f"-DE4B_INST_FMT={fmt}", "-c", "-o", obj,
                     GEMM_SRC])
        objs.append(obj)
    msgs = _run_all(cmds)
    tmp = OUT + ".tmp"
    msgs += _run_all([[cc, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]])
    if os.path.exists(TORCH_OUT):
        os.remove(TORCH_OUT)
    os.replace(tmp, OUT)
    return msgs


def _binding_object(tmpdir: str):
    """(link command of libe4b_torch.so, the messages of its compilation)"""
    compile_, link = _torch_commands(os.path.join(tmpdir, "torch_losses.o"), TORCH_OUT + ".tmp")
    return link, _run_all([compile_])


def build(verbose: bool = False, binding: bool = True) -> str:
    """The library and, with ``binding``, what binds it to torch's autograd. The library needs hipcc alone: where the binding
    fails it is in place all the same, without the binding, and the error is raised then."""
    with tempfile.TemporaryDirectory(prefix="e4b_build_") as tmpdir, ThreadPoolExecutor(1) as beside:
        compiled = beside.submit(_binding_object, tmpdir) if binding else None
        msgs = _library(tmpdir)
        if binding:
            try:
                link, more = compiled.result()
                msgs += more + _run_all([link])
            except Exception as e:
                raise RuntimeError(f"{OUT} is built, its binding to torch is not: {e}") from e
            os.replace(TORCH_OUT + ".tmp", TORCH_OUT)
    if verbose and msgs:
        print("\n".join(msgs), file=sys.stderr)
    return OUT


if __name__ == "__main__":
    print(build(verbose=True))
