"""Build libvla_b200.so in place with nvcc for sm_100a (cross-compiles without a GPU)."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(HERE, "libvla_b200.so")
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


def needs_build():
    return _stale(LIB, [os.path.join(HERE, f) for f in SOURCES + HEADERS])


def build(force=False, verbose=False):
    if not force and not needs_build():
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
    subprocess.run([nvcc] + flags + ["-shared", "-o", LIB] + [_object(s) for s in SOURCES], cwd=HERE, check=True)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
