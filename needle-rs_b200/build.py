"""Build libneedle3.so: the sm_100a CUDA engine plus its C ABI.

Kernels are compiled for sm_100a only, with -fmad=false (a product and an add
stay two roundings unless the source writes __fmaf_rn) and IEEE division and
square root; host code with -ffp-contract=off for the same reason.
"""

import os
import re
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
OUT_DIR = os.path.join(HERE, "needle_b200")
LIB = os.path.join(OUT_DIR, "libneedle3.so")
BUILD = os.path.join(HERE, "_build")

CU = ["kernels.cu", "tc_prefill.cu", "engine.cu", "ops.cu", "noalloc.cu", "kv4.cu", "kv4_attend.cu", "kv4_prefill.cu", "pages.cu", "verify.cu"]
CPP = ["cact.cpp"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nvcc():
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _stale(target, sources):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(s) > t for s in sources)


def check_registers(source: str, log: str) -> None:
    """The prompt kernel shares its registers out anew among its warpgroups; a
    share beyond what the block was launched with would wait for ever. So the
    build ends here should the compiler (its -v log) give a thread fewer than
    the PRE_REGS_LAUNCH that the source counts on (registers come in eights)."""
    need = int(re.search(r"PRE_REGS_LAUNCH = (\d+)", source).group(1))
    got = [int(n) for name, n in re.findall(r"Compiling entry function '(\S+)'.*?Used (\d+) registers", log, re.S)
           if "kv4_prefill_kernel" in name]
    if not got:
        raise RuntimeError("no register counts of kv4_prefill_kernel in the compiler's log")
    if any((n + 7) // 8 * 8 < need for n in got):
        raise RuntimeError(f"kv4_prefill_kernel has {min(got)} registers a thread; its warpgroups share out {need}")


def build(force: bool = False, verbose: bool = False) -> str:
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [
        os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)
    ]
    if not force and not _stale(LIB, deps):
        return LIB
    os.makedirs(BUILD, exist_ok=True)
    nvcc = _nvcc()
    objs = []
    common = ["-O3", "-std=c++17", "-I", CSRC, "-I", INCLUDE]
    for f in CPP:
        o = os.path.join(BUILD, f + ".o")
        cmd = ["g++", *common, "-fPIC", "-ffp-contract=off", "-fno-fast-math", "-pthread", "-c",
               os.path.join(CSRC, f), "-o", o]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.check_call(cmd)
        objs.append(o)
    procs = []
    for f in CU:
        o = os.path.join(BUILD, f + ".o")
        cmd = [nvcc, *ARCH, *common, "-lineinfo", "-fmad=false", "-prec-div=true", "-prec-sqrt=true",
               "-Xcompiler", "-fPIC,-ffp-contract=off", "-c", os.path.join(CSRC, f), "-o", o]
        shares = f == "kv4_prefill.cu"
        if shares:
            cmd += ["-Xptxas", "-v"]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        procs.append((cmd, shares, subprocess.Popen(cmd, stderr=subprocess.PIPE if shares else None, text=True)))
        objs.append(o)
    for cmd, shares, proc in procs:
        _, log = proc.communicate()
        if proc.returncode:
            print(log or "", file=sys.stderr)
            raise subprocess.CalledProcessError(proc.returncode, cmd)
        if shares:
            with open(os.path.join(CSRC, "kv4_prefill.cu")) as src:
                check_registers(src.read(), log)
    tmp = LIB + ".tmp"
    cmd = [nvcc, *ARCH, "-shared", "-o", tmp, *objs, "-lpthread"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.check_call(cmd)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
