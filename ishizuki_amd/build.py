"""Builds libishizuki_hip.so (the C-ABI HIP library) in-tree for gfx950 with hipcc.

Every .hip file under csrc/ is compiled with hipcc (and every .cpp, host-only, with g++) to an
object in parallel, then linked; csrc/python/bind.cpp, Python's way into the attention calls, becomes
_bind.so beside it, where torch is there (its headers; the C library needs none). hipcc flags:
  --offload-arch=gfx950                         CDNA4 only
  -Xclang -target-feature -Xclang -packed-fp32-ops   no packed fp32 instructions
  -O3 -fPIC -std=c++20 (g++ -std=c++17 for the host-only GGUF reader)
"""
import concurrent.futures
import glob
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libishizuki_hip.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = ["--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++20",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-Wno-unused-command-line-argument", "-I", os.path.join(HERE, "..", "include")]


HOST_FLAGS = ["-O2", "-fPIC", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I", "/opt/rocm/include",
              "-I", os.path.join(HERE, "..", "include")]


BIND = os.path.join(HERE, "_bind.so")


def _compile_bind():
    """The object of the Python binding of the attention calls (csrc/python): host code over torch's headers."""
    from torch.utils import cpp_extension
    obj = os.path.join(OBJ, "python", "bind.o")
    os.makedirs(os.path.dirname(obj), exist_ok=True)
    flags = [f"-I{p}" for p in [*cpp_extension.include_paths(), sysconfig.get_paths()["include"]]]
    cmd = ["g++", *HOST_FLAGS, "-DUSE_ROCM", "-fvisibility=hidden", *flags, "-c", os.path.join(CSRC, "python", "bind.cpp"), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("g++ failed on bind.cpp")
    return obj


def _link_bind(obj):
    from torch.utils import cpp_extension
    tmp = BIND + ".tmp"
    libs = [x for p in cpp_extension.library_paths() for x in ("-L" + p, "-Wl,-rpath," + p)]
    subprocess.run(["g++", "-shared", "-o", tmp, obj, "-L" + HERE, "-lishizuki_hip", "-Wl,-rpath,$ORIGIN", *libs, "-lc10", "-lc10_hip", "-ltorch_cpu",
                    "-ltorch_python"], check=True)
    os.replace(tmp, BIND)


def _compile(src):
    obj = os.path.join(OBJ, os.path.basename(src) + ".o")
    if src.endswith(".cpp"):  # host-only code (the GGUF reader)
        cmd = ["g++", *HOST_FLAGS, "-c", src, "-o", obj]
    else:
        cmd = [HIPCC, *FLAGS, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f"hipcc failed on {src}")
    return obj


def build(verbose=True):
    os.makedirs(OBJ, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.cpp")))
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        bind = ex.submit(_compile_bind) if importlib.util.find_spec("torch") else None
        objs = list(ex.map(_compile, srcs))
    tmp = LIB + ".tmp"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-shared", "-o", tmp, *objs], check=True)
    os.replace(tmp, LIB)
    if bind:
        _link_bind(bind.result())
    if verbose:
        print("built", LIB, "" if bind else "alone: no torch to build _bind.so with")
    return LIB


if __name__ == "__main__":
    build()
