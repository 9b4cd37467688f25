"""Builds the extension modules in this folder with the host compiler.

``pyCAHEL`` (binding.cpp) is what lancelot-main-GPU imports (``import pyCAHEL as cahel``): put this folder on PYTHONPATH.
It links ``../liblancelot_b200.so`` (found at run time relative to the module) and the CUDA runtime.
``_updates8`` (updates8.cpp) holds the 8-bit update calls of ``cabi.Context``; it links torch's C++ libraries as well, and is left out, with a
note, where torch or its CUDA part is not installed."""
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
ROOT = os.path.dirname(PKG)


def target(module="pyCAHEL"):
    return os.path.join(HERE, module + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))


def _compile(module, deps, flags, force, against=""):
    """against: what a module was linked to that its sources do not show; it is built anew when that changes"""
    out = target(module)
    record = os.path.join(PKG, "build", module + ".against")
    built = ""
    if os.path.exists(record):
        with open(record) as f:
            built = f.read()
    if not force and built == against and os.path.exists(out) and all(os.path.getmtime(d) <= os.path.getmtime(out) for d in deps):
        return out
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cxx = os.environ.get("CXX", "g++")
    cmd = [cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(ROOT, "include"),
           "-I" + os.path.join(cuda, "include"), deps[0], "-o", out + ".tmp",
           "-L" + PKG, "-llancelot_b200", "-L" + os.path.join(cuda, "lib64"), "-lcudart",
           "-Wl,-rpath,$ORIGIN/..", "-Wl,-rpath," + os.path.join(cuda, "lib64")] + flags
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("building %s failed: %s\n%s" % (module, " ".join(cmd), r.stderr))
    os.replace(out + ".tmp", out)
    os.makedirs(os.path.dirname(record), exist_ok=True)
    with open(record, "w") as f:
        f.write(against)
    return out


def build(force=False):
    """Returns the path of ``pyCAHEL``, which needs no torch."""
    import pybind11

    header = os.path.join(ROOT, "include", "lancelot_b200.h")
    out = _compile("pyCAHEL", [os.path.join(HERE, "binding.cpp"), os.path.join(ROOT, "include", "cahel_b200.hpp"), header],
                   ["-I" + pybind11.get_include()], force)
    try:
        import torch
    except ImportError:
        torch = None
    site = os.path.dirname(torch.__file__) if torch else ""
    lib = os.path.join(site, "lib")
    if not torch or not os.path.exists(os.path.join(lib, "libc10_cuda.so")):
        sys.stderr.write("no torch with CUDA: _updates8 is not built, the 8-bit update calls of cabi.Context will not import\n")
        return out
    _compile("_updates8", [os.path.join(HERE, "updates8.cpp"), header],
             ["-I" + os.path.join(site, "include"), "-I" + os.path.join(site, "include", "torch", "csrc", "api", "include"),
              "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch._C._GLIBCXX_USE_CXX11_ABI), "-L" + lib, "-lc10", "-lc10_cuda", "-ltorch_cpu",
              "-ltorch_python", "-Wl,-rpath," + lib], force, "torch %s %s in %s" % (torch.__version__, torch.version.git_version, site))
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv))
