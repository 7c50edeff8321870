"""Build libvla_b200.so in place with nvcc for sm_100a (cross-compiles without a GPU), and _vla_ops.so, the Python binding of the
operators that take torch tensors, with g++ (where torch is installed; --library leaves it out)."""
import os
import subprocess
import sys
import sysconfig
from importlib import metadata
from importlib.util import find_spec

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(HERE, "libvla_b200.so")
BINDING, BINDING_SRC = os.path.join(HERE, "_vla_ops.so"), "csrc/binding.cpp"
BINDING_FOR = os.path.join(HERE, "build", "_vla_ops.for")        # see _made_for
SOURCES = ["csrc/model.cu", "csrc/cache_ops.cu"]
# headers that only one of the sources includes; the others (common.cuh, host.cuh, the C header) belong to both
ONLY = {"csrc/cache_ops.cu": {"csrc/attention_paged.cuh", "csrc/attention_prompt.cuh", "csrc/cache_pages.cuh"}}
SHARED = {"csrc/common.cuh", "csrc/host.cuh", "../include/vla_b200.h"}
HEADERS = sorted("csrc/" + f for f in os.listdir(os.path.join(HERE, "csrc")) if f.endswith(".cuh")) + ["../include/vla_b200.h"]


def _object(src):
    return os.path.join(HERE, "build", os.path.basename(src) + ".o")


def _inputs(src):
    own = ONLY.get(src) or set(HEADERS) - set().union(*ONLY.values())
    return [os.path.join(HERE, f) for f in {src} | own | SHARED]


def _stale(target, inputs):
    return not os.path.exists(target) or any(os.path.getmtime(f) > os.path.getmtime(target) for f in inputs)


def needs_build(binding=True):
    return _stale(LIB, [os.path.join(HERE, f) for f in SOURCES + HEADERS]) or binding and _has_torch() and _binding_stale()


def _has_torch():
    return find_spec("torch") is not None


def _made_for():
    """What the binding is linked against: it loads with no other torch or Python."""
    try:
        version = metadata.version("torch")
    except metadata.PackageNotFoundError:      # a torch that runs from its source tree
        version = "unknown"
    return "torch %s in %s, %s" % (version, _torch_home(), sys.implementation.cache_tag)


def _torch_home():
    return os.path.dirname(find_spec("torch").origin)


def _read(path):
    if not os.path.exists(path):
        return None
    with open(path) as f:
        return f.read()


def _binding_stale():
    return _stale(BINDING, [os.path.join(HERE, f) for f in (BINDING_SRC, "../include/vla_b200.h")]) or _read(BINDING_FOR) != _made_for()


def _binding_command(nvcc):
    home = _torch_home()
    include = [os.path.join(home, "include"), os.path.join(home, "include/torch/csrc/api/include"), sysconfig.get_paths()["include"],
               os.path.join(os.path.dirname(os.path.dirname(nvcc)), "include")]
    libs = ["torch_python", "torch_cpu", "torch", "c10", "c10_cuda", "vla_b200"]
    # g++ as nvcc finds it: a compiler that links its own libstdc++ does not get on with torch's
    return (["g++", "-O2", "-std=c++17", "-fPIC", "-shared", BINDING_SRC, "-o", BINDING] + ["-I" + d for d in include] +
            ["-L" + os.path.join(home, "lib"), "-L" + HERE] + ["-l" + x for x in libs] + ["-Wl,-rpath,$ORIGIN"])


def build(force=False, verbose=False, binding=True):
    """The C library needs nvcc alone; `binding`: the Python binding too, where torch is installed."""
    if not force and not needs_build(binding):
        return LIB
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    flags = ["-O3", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-Xcompiler", "-fPIC"]
    if verbose:
        flags.insert(0, "-Xptxas=-v")
    os.makedirs(os.path.join(HERE, "build"), exist_ok=True)
    todo = [s for s in SOURCES if force or _stale(_object(s), _inputs(s))]
    running = [subprocess.Popen([nvcc] + flags + ["-c", s, "-o", _object(s)], cwd=HERE) for s in todo]
    failed = [s for s, p in zip(todo, running) if p.wait() != 0]
    if failed:
        raise RuntimeError("nvcc failed on " + ", ".join(failed))
    if force or _stale(LIB, [_object(s) for s in SOURCES]):
        subprocess.run([nvcc] + flags + ["-shared", "-o", LIB] + [_object(s) for s in SOURCES], cwd=HERE, check=True)
    if binding and not _has_torch():
        print("build.py: no torch here, so no _vla_ops.so; libvla_b200.so is complete", file=sys.stderr)
    elif binding and (force or _binding_stale()):
        try:
            subprocess.run(_binding_command(nvcc), cwd=HERE, check=True)
        except (OSError, subprocess.CalledProcessError) as e:
            raise RuntimeError("libvla_b200.so is complete, _vla_ops.so could not be built (--library leaves it out): %s" % e) from e
        with open(BINDING_FOR, "w") as f:
            f.write(_made_for())
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv, binding="--library" not in sys.argv))
