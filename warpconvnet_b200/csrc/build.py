"""Build libwcn_b200.so in this folder with nvcc for sm_100a (no other architecture), and where they can be built the _fastcall.so
extension through which Python calls it (ctypes makes the calls elsewhere) and the _autograd.so extension whose graph nodes call it
(autograd functions in Python do elsewhere).

Usage: ``python -m warpconvnet_b200.csrc.build [--force] [--verbose]``
"""
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
SOURCES = ["api.cu", "hash_kmap.cu", "brick_kmap.cu", "cell_kmap.cu", "morton_sort.cu", "level_maps.cu", "net_run.cu", "conv_explicit.cu", "row_reduce.cu", "batch_norm.cu", "column_sums.cu", "conv_simt.cu", "conv_fp32.cu", "conv_split_tcgen05.cu", "conv_tcgen05.cu",
           "conv_wgrad_tcgen05.cu", "conv_wgrad_split_tcgen05.cu", "conv_wgrad_pairs.cu", "conv_rows_tcgen05.cu",
           "adamw.cu", "group_norm.cu", "linear_ce.cu", "linear_ce_tcgen05.cu",
           "rms_norm.cu", "dropout.cu", "linear.cu", "linear_tcgen05.cu", "linear_backward_tcgen05.cu", "linear_split_tcgen05.cu"]
HEADERS = ["wcn_common.cuh", "tile_order.cuh", "tcgen05_common.cuh", "split_bf16.cuh", "tma_common.cuh", "linear_ce.cuh", "philox.cuh", "linear.cuh", "linear_16bit.cuh", "linear_fp32.cuh", os.path.join("..", "..", "include", "wcn_b200.h")]
LIB = os.path.join(HERE, "libwcn_b200.so")
FASTCALL_SOURCE, FASTCALL = os.path.join(HERE, "fastcall.c"), os.path.join(HERE, "_fastcall.so")
AUTOGRAD_SOURCE, AUTOGRAD = os.path.join(HERE, "autograd.cpp"), os.path.join(HERE, "_autograd.so")
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", "--use_fast_math=false"]


def _nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isfile(cand) or cand == "nvcc"):
            return cand
    return "nvcc"


def needs_build():
    if not os.path.isfile(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(HERE, s) for s in SOURCES + HEADERS] + [os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > t for d in deps)


def build_fastcall(force=False):
    if force or not os.path.isfile(FASTCALL) or os.path.getmtime(FASTCALL_SOURCE) > os.path.getmtime(FASTCALL):
        cmd = [os.environ.get("CC", "gcc"), "-O2", "-shared", "-fPIC", "-I" + sysconfig.get_paths()["include"],
               FASTCALL_SOURCE, "-o", FASTCALL]
        try:
            subprocess.check_call(cmd)
        except (OSError, subprocess.CalledProcessError) as e:  # another machine, an older Python, no headers
            if os.path.isfile(FASTCALL):
                os.remove(FASTCALL)  # (of an earlier source)
            print(f"_fastcall.so was not built ({e}): calls go through ctypes")


def _autograd_is_built(version):
    """Whether the extension is there, of this source and of this torch."""
    header = os.path.join(HERE, "..", "..", "include", "wcn_b200.h")
    if not os.path.isfile(AUTOGRAD) or os.path.getmtime(AUTOGRAD) <= max(os.path.getmtime(AUTOGRAD_SOURCE), os.path.getmtime(header)):
        return False
    with open(AUTOGRAD, "rb") as f:
        return f"built with torch {version}, not ".encode() in f.read()


def build_autograd(force=False):
    try:
        import torch
        if not force and _autograd_is_built(torch.__version__):
            return
        root = os.path.dirname(torch.__file__)
        cuda = os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")
        cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
               f'-DWCN_BUILT_WITH="{torch.__version__}"',
               *("-I" + i for i in (os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), cuda,
                                    sysconfig.get_paths()["include"])),
               AUTOGRAD_SOURCE, "-o", AUTOGRAD, "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python",
               "-l:libstdc++.so.6"]  # (torch's own: some compilers would link theirs statically, and a process with two of them ends at the first error's text)
        subprocess.check_call(cmd)
    except (ImportError, OSError, subprocess.CalledProcessError) as e:  # no compiler, no headers
        if os.path.isfile(AUTOGRAD):
            os.remove(AUTOGRAD)  # (of an earlier source)
        print(f"_autograd.so was not built ({e}): gradients go through Python")


def build(force=False, verbose=False, ptxas_info=False):
    build_fastcall(force)
    build_autograd(force)
    if not force and not needs_build():
        return LIB
    flags = [f for f in NVCC_FLAGS if not f.startswith("--use_fast_math")]
    if ptxas_info:
        flags += ["-Xptxas", "-v"]
    objs = []
    procs = []
    for s in SOURCES:
        obj = os.path.join(HERE, s.replace(".cu", ".o"))
        cmd = [_nvcc(), *flags, "-c", os.path.join(HERE, s), "-o", obj]
        if verbose:
            print(" ".join(cmd))
        procs.append((s, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
        objs.append(obj)
    failed = False
    for s, pr in procs:
        out, _ = pr.communicate()
        if out.strip() and (verbose or ptxas_info or pr.returncode != 0):
            print(out)
        if pr.returncode != 0:
            failed = True
    if failed:
        raise RuntimeError("nvcc failed")
    cmd = [_nvcc(), "-shared", "-o", LIB, *objs, "-lcudart", "-Xlinker", "-rpath=/usr/local/cuda/lib64"]
    if verbose:
        print(" ".join(cmd))
    subprocess.check_call(cmd)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv, ptxas_info="--ptxas" in sys.argv))
