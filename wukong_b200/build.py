"""Build step: compile every CUDA source under csrc/ for sm_100a into one C-ABI shared library,
in-tree (wukong_b200/libwukong_b200.so), and csrc/host/torch_calls.cpp -- calls on torch tensors that skip the Python level
-- into an extension module beside it (wukong_b200/_torch_calls.so).  nvcc cross-compiles without a GPU.  The library needs
nothing else; where torch or g++ is missing the module is left out, and the calls that go through it say so."""
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libwukong_b200.so")
OBJ = os.path.join(HERE, "build")
CALLS = os.path.join(CSRC, "host", "torch_calls.cpp")
CALLS_OUT = os.path.join(HERE, "_torch_calls.so")
CALLS_FOR = os.path.join(OBJ, "torch_calls.torch")      # the torch version that it was built against

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-fmad=false",  # every fused multiply-add in the sources is explicit
    "--expt-relaxed-constexpr",
]


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cpp")))


def needs_build():
    if not os.path.exists(OUT):
        return True
    t = os.path.getmtime(OUT)
    deps = sources() + glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh")) + \
        [os.path.join(HERE, "..", "include", "wukong_b200.h"), os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > t for d in deps)


def run_host_compiler(cmd, verbose):
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0 or verbose:
        sys.stderr.write("== torch_calls.cpp\n%s\n" % r.stdout)
    if r.returncode != 0:
        raise RuntimeError("g++ failed")


def build_calls(force=False, verbose=False):
    """The extension module of csrc/host: linked against torch and, beside it, the C-ABI library."""
    try:
        import torch
    except ImportError:
        sys.stderr.write("_torch_calls is left out: torch is not installed\n")
        return None
    header, version = os.path.join(HERE, "..", "include", "wukong_b200.h"), str(torch.__version__)
    built_for = open(CALLS_FOR).read() if os.path.exists(CALLS_FOR) else None
    if not force and built_for == version and os.path.exists(CALLS_OUT) and \
            os.path.getmtime(CALLS_OUT) > max(os.path.getmtime(p) for p in (CALLS, header, os.path.abspath(__file__))):
        return CALLS_OUT
    if not shutil.which("g++"):
        sys.stderr.write("_torch_calls is left out: there is no g++\n")
        return None
    root = os.path.dirname(os.path.abspath(torch.__file__))
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch._C._GLIBCXX_USE_CXX11_ABI), '-DWKB_TORCH_VERSION="%s"' % version,
           "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(root, "include"), "-I" + os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-I" + os.path.join(cuda, "include"), CALLS, "-o", CALLS_OUT, "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", "-L" + HERE,
           "-l:libwukong_b200.so", "-Wl,-rpath,$ORIGIN:" + os.path.join(root, "lib")]
    run_host_compiler(cmd, verbose)
    os.makedirs(OBJ, exist_ok=True)
    with open(CALLS_FOR, "w") as fh:
        fh.write(version)
    return CALLS_OUT


def build(force=False, verbose=False):
    build_library(force, verbose)
    build_calls(force, verbose)
    return OUT


def build_library(force=False, verbose=False):
    if not force and not needs_build():
        return OUT
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    os.makedirs(OBJ, exist_ok=True)
    objs, procs = [], []
    hdr_time = max(os.path.getmtime(p) for p in glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh")) +
                   [os.path.join(HERE, "..", "include", "wukong_b200.h")])
    for src in sources():
        obj = os.path.join(OBJ, os.path.basename(src) + ".o")
        objs.append(obj)
        if not force and os.path.exists(obj) and os.path.getmtime(obj) > max(os.path.getmtime(src), hdr_time):
            continue
        cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", src, "-o", obj]
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failed = False
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0 or verbose:
            sys.stderr.write("== %s\n%s\n" % (os.path.basename(src), out))
        failed |= p.returncode != 0
    if failed:
        raise RuntimeError("nvcc failed")
    subprocess.check_call([nvcc, "-shared", "-o", OUT] + objs)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
