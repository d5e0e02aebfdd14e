"""Build recipe of libb200ops.so: every CUDA source under csrc/ compiled for sm_100a with nvcc; and of torch_calls.so, the
direct way from Python tensors into it (g++, against the installed torch's headers).

Both are built in-tree (next to this file) so that they travel with the source checkout;
nvcc cross-compiles for sm_100a on machines without a GPU.
"""
import glob
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB_PATH = os.path.join(HERE, "libb200ops.so")
CALLS_PATH = os.path.join(HERE, "torch_calls.so")
STAMP_PATH = os.path.join(HERE, "build", "torch_calls.stamp")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
]


def sources():
    return sorted(glob.glob(os.path.join(HERE, "csrc", "*.cu")))


def _torch_stamp():
    """What torch_calls.so is compiled against: the torch and the Python that load it must be these."""
    from importlib import metadata
    return "torch %s, python %d.%d" % (metadata.version("torch"), *sys.version_info[:2])


def _stale():
    if not os.path.exists(LIB_PATH) or not os.path.exists(CALLS_PATH):
        return True
    try:
        with open(STAMP_PATH) as f:
            if f.read() != _torch_stamp():
                return True
    except FileNotFoundError:
        return True
    t = min(os.path.getmtime(LIB_PATH), os.path.getmtime(CALLS_PATH))
    deps = sources() + glob.glob(os.path.join(HERE, "csrc", "*.cpp")) + glob.glob(os.path.join(HERE, "csrc", "*.cuh")) + \
        glob.glob(os.path.join(ROOT, "include", "*.h")) + [os.path.abspath(__file__)]
    return any(os.path.getmtime(p) > t for p in deps)


def build(force=False, verbose=False):
    """Compile csrc/*.cu into libb200ops.so and csrc/torch_calls.cpp into torch_calls.so (skipped when both are newer than
    their sources and the torch is the one they were built for)."""
    if not force and not _stale():
        return LIB_PATH
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    objs = []
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    procs = []
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + \
            ["-I", os.path.join(ROOT, "include"), "-c", src, "-o", obj]
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    procs.append((os.path.join(HERE, "csrc", "torch_calls.cpp"), subprocess.Popen(
        _calls_command(os.path.join(objdir, "torch_calls.o")), stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    for src, proc in procs:
        out, _ = proc.communicate()
        if verbose or proc.returncode != 0:
            sys.stderr.write(out)
        if proc.returncode != 0:
            raise RuntimeError("the compiler failed on %s" % src)
    link = [nvcc, "-shared", "-o", LIB_PATH] + objs + ["-lcudart"]
    subprocess.check_call(link)
    import torch
    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    subprocess.check_call(
        ["g++", "-shared", "-o", CALLS_PATH, os.path.join(objdir, "torch_calls.o"), "-L" + torch_lib, "-lc10", "-lc10_cuda",
         "-ltorch_cpu", "-ltorch_python", "-L" + HERE, "-l:libb200ops.so", "-Wl,-rpath,$ORIGIN"])
    with open(STAMP_PATH, "w") as f:
        f.write(_torch_stamp())
    return LIB_PATH


def _calls_command(obj):
    import sysconfig

    import torch
    base = os.path.join(os.path.dirname(torch.__file__), "include")
    includes = [os.path.join(ROOT, "include"), base, os.path.join(base, "torch", "csrc", "api", "include"),
                os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include"), sysconfig.get_paths()["include"]]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden",
            "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI] + [f for d in includes for f in ("-I", d)] + [
                "-c", os.path.join(HERE, "csrc", "torch_calls.cpp"), "-o", obj]


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
