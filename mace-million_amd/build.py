"""Build step of the MI355X library: generate the architecture-specific kernels and compile everything for gfx950.

    python mace-million_amd/build.py            (also called by __graft_entry__.build())

Output: mace-million_amd/lib/libmace_million_amd.so (git-ignored; it travels with the tree to the GPU box),
lib/mm_torch_ops.so: the PyTorch functions of the operators with autograd nodes (host C++ against the installed torch),
lib/kernel_ops.json: the fp32 operations per thread that the straight-line generated symmetric-contraction kernels
execute, counted from their gfx950 assembly (bench.py reports their FLOP rates from it), and lib/jit/: the
channelwise TP kernels of the path tables in o3.PREBUILT_JIT_TP_TABLES (mace_onegpu/tp_jit.py).
Every HIP source is compiled with -Xclang -target-feature -Xclang -packed-fp32-ops (no packed-FP32 instructions)
and -munsafe-fp-atomics (hardware float atomics instead of compare-and-swap loops).
"""
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
GEN = os.path.join(CSRC, "gen")
OBJ = os.path.join(HERE, "_build")
LIB_DIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIB_DIR, "libmace_million_amd.so")

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
FLAGS = ["-O3", "-std=c++17", "-fPIC", f"--offload-arch={ARCH}", "-Xclang", "-target-feature", "-Xclang",
         "-packed-fp32-ops", "-munsafe-fp-atomics", "-Wno-unused-command-line-argument"]


def generate():
    sys.path.insert(0, HERE)
    from mace_onegpu import codegen, model

    return codegen.generate(GEN, model.Tables(model.MaceSpec()))


def sources():
    out = []
    for d in (CSRC, GEN):
        for f in sorted(os.listdir(d)):
            if f.endswith((".hip", ".cpp")):
                out.append(os.path.join(d, f))
    return out


# files whose fp64 results must be bit-identical to the reference's separately rounded CPU arithmetic; and the
# files whose kernels run faster under the memory-clause scheduling strategy (same-box A/B at configuration 5:
# conv2_fwd 10.13 -> 9.88 ms and conv2_bwd 19.16 -> 19.00 ms per launch; the linears 35.8 -> 34.7 and 34.8 -> 34.4
# ms per step on two boxes).  The other kernels keep the default: the ACE kernels gained nothing reproducible, the
# same option made mm_symc1_fwd 11 % slower, and the max-ilp strategy made mm_symc1_bwd twice as slow.
MEMORY_CLAUSE = ["-mllvm", "-amdgpu-sched-strategy=max-memory-clause"]
EXTRA = {"nlist.hip": ["-ffp-contract=off"], "conv_l2.hip": MEMORY_CLAUSE, "linear.hip": MEMORY_CLAUSE}


def _compile(src):
    obj = os.path.join(OBJ, os.path.relpath(src, CSRC).replace(os.sep, "__") + ".o")
    cmd = [HIPCC] + FLAGS + EXTRA.get(os.path.basename(src), []) + ["-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return obj


# straight-line generated kernels whose executed fp32 operations are counted from their gfx950 assembly
COUNTED = {"symc_l1.hip": ("mm_symc1_fwd_kernel", "mm_symc1_bwd_kernel"),
           "symc_l2.hip": ("mm_symc2_fwd_kernel", "mm_symc2_bwd_kernel")}
OPS_JSON = os.path.join(LIB_DIR, "kernel_ops.json")


def _count_ops(name):
    """fp32 VALU operations per thread of the kernels of generated source `name`, from its device assembly."""
    sys.path.insert(0, HERE)
    from mace_onegpu import codegen

    src = os.path.join(GEN, name)
    asm = os.path.join(OBJ, name + ".s")
    cmd = [HIPCC] + FLAGS + ["--cuda-device-only", "-S", src, "-o", asm]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"assembly failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    text = open(asm).read()
    return {k: codegen.asm_valu_flops(text, k) for k in COUNTED[name]}


TORCH_OPS = os.path.join(LIB_DIR, "mm_torch_ops.so")
TORCH_SOURCES = ("ops", "train")


def _build_torch_ops():
    """lib/mm_torch_ops.so: csrc/torch/*.cpp, host C++ against the installed torch (linked by _link_torch_ops)."""
    import sysconfig

    import torch

    root = os.path.dirname(torch.__file__)
    base = ["g++", "-O2", "-std=c++17", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I" + os.path.join(root, "include"),
           "-I" + os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-I" + os.path.join(os.path.dirname(os.path.dirname(HIPCC)), "include"),
           "-I" + sysconfig.get_paths()["include"]]

    def one(name):
        obj = os.path.join(OBJ, f"torch__{name}.o")
        cmd = base + ["-c", os.path.join(CSRC, "torch", name + ".cpp"), "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
        return obj

    with ThreadPoolExecutor(len(TORCH_SOURCES)) as ex:
        return list(ex.map(one, TORCH_SOURCES)), os.path.join(root, "lib")


def _link_torch_ops(objs, torch_lib):
    tmp = TORCH_OPS + ".tmp"
    cmd = ["g++", "-shared", "-o", tmp] + objs + ["-L" + LIB_DIR, "-l:" + os.path.basename(LIB), "-L" + torch_lib,
           "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python", "-ltorch", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, TORCH_OPS)


def build(jobs=None, verbose=True):
    generate()
    os.makedirs(OBJ, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    srcs = sources()
    jobs = jobs or min(8, os.cpu_count() or 4)
    sys.path.insert(0, HERE)
    from mace_onegpu import o3, tp_jit

    with ThreadPoolExecutor(jobs) as ex:
        counts = [ex.submit(_count_ops, n) for n in COUNTED]
        # the kernels of the tables that FusedConvTP builds on first use, made ahead for the listed tables
        jit = [ex.submit(tp_jit.build, o3.tp_table(list(a), b, c), True) for a, b, c in o3.PREBUILT_JIT_TP_TABLES]
        torch_ops = ex.submit(_build_torch_ops)
        objs = list(ex.map(_compile, srcs))
        ops = {}
        for c in counts:
            ops.update(c.result())
        for j in jit:
            j.result()
        torch_ops = torch_ops.result()
    import json
    with open(OPS_JSON, "w") as fh:
        json.dump(ops, fh, indent=1)
    tmp = LIB + ".tmp"
    cmd = [HIPCC, "-shared", "-fPIC", f"--offload-arch={ARCH}", "-o", tmp] + objs
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    _link_torch_ops(*torch_ops)
    shutil.rmtree(OBJ, ignore_errors=True)
    if verbose:
        print(f"built {LIB} from {len(srcs)} sources")
    return LIB


if __name__ == "__main__":
    build()
