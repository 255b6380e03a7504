"""Build libbcjr_b200.so in-tree with nvcc for sm_100a.

    python -m quant_2bit_b200.build          # or quant_2bit_b200.build.build()

The library is a plain C-ABI shared object (include/bcjr_b200.h); it links
the CUDA runtime statically and has no torch dependency.
"""
import concurrent.futures
import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libbcjr_b200.so")
SOURCES = ["bcjr_capi.cu", "bcjr_generic.cu", "bcjr_l16.cu", "bcjr_b4.cu", "bcjr_noalloc.cu", "bcjr_rht.cu",
           "bcjr_viterbi.cu", "bcjr_vit_b4.cu", "bcjr_vit_b2.cu", "bcjr_codes.cu", "bcjr_l16_cl4.cu", "bcjr_probe.cu",
           "bcjr_mm.cu", "bcjr_grouped.cu", "bcjr_fp8.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
              "-Xcompiler", "-fvisibility=hidden"]

# Kernels that share their registers out among warpgroups are launched with the
# number that the source is written for, or not at all (another one would leave
# a share waiting for registers for good): {source: (kernel, its constant there)}.
LAUNCH_REGISTERS = {"bcjr_fp8.cu": ("fp8_rows_kernel", "kLaunchRegs")}


def _nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.sep not in cand or os.path.exists(cand)):
            return cand
    return "nvcc"


def _stale():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    deps.append(os.path.join(HERE, "..", "include", "bcjr_b200.h"))
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def registers(ptxas, kernel):
    """Registers of every instance of `kernel` in ptxas -v output."""
    return [int(n) for name, n in re.findall(r"Compiling entry function '(\w+)'.*?Used (\d+) registers", ptxas, re.S)
            if kernel in name]


def _compile(cmd, src, ptxas_info):
    run = subprocess.run(cmd + ["-Xptxas", "-v"] if ptxas_info or src in LAUNCH_REGISTERS else cmd,
                         stderr=subprocess.PIPE, text=True)
    for line in run.stderr.splitlines():
        if ptxas_info or run.returncode or not line.startswith("ptxas info") and " bytes stack frame" not in line:
            print(line, file=sys.stderr)
    run.check_returncode()
    if src in LAUNCH_REGISTERS:
        kernel, constant = LAUNCH_REGISTERS[src]
        with open(os.path.join(CSRC, src)) as f:
            want = int(re.search(constant + r" = (\d+)", f.read()).group(1))
        got = registers(run.stderr, kernel)
        if not got or set(got) != {want}:
            raise RuntimeError(f"{src}: {kernel} was compiled for {got} registers, its shares add up to {want}")


def build(force=False, verbose=False, ptxas_info=False):
    """Compile every source into one shared library (skipped when up to date)."""
    if not force and not _stale():
        return LIB
    srcs = [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    cmds, objs = [], []
    for s in srcs:
        obj = os.path.join(CSRC, s.replace(".cu", ".o"))
        cmd = [_nvcc(), *ARCH, *NVCC_FLAGS, "-c", os.path.join(CSRC, s), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        cmds.append(cmd)
        objs.append(obj)
    # the translation units are independent: compile them side by side
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(len(cmds), os.cpu_count() or 1)) as ex:
        for f in [ex.submit(_compile, c, s, ptxas_info) for c, s in zip(cmds, srcs)]:
            f.result()
    cmd = [_nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", *objs, "-o", LIB]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    for o in objs:
        os.remove(o)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True, ptxas_info="--ptxas" in sys.argv)
