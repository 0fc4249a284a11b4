"""Builds the in-tree shared library ``dlf_b200/libdlf_b200.so`` with nvcc for sm_100a.

Run as ``python -m dlf_b200.build`` (add ``--force`` to rebuild, ``--verbose`` to see the
ptxas resource report). The library is the product: nothing in the package works without it.
"""
import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libdlf_b200.so")
OBJECTS = os.path.join(HERE, "objects")
SOURCES = ["api.cu", "quantized.cu", "attention.cu"]


def _headers(source):
    """The files of this tree that a source includes, directly or through another one."""
    found, todo = set(), [os.path.join(CSRC, source)]
    while todo:
        at = todo.pop()
        with open(at) as f:
            names = re.findall(r'^#include "([^"]+)"', f.read(), re.M)
        for name in names:
            h = os.path.normpath(os.path.join(os.path.dirname(at), name))
            if h not in found and os.path.exists(h):
                found.add(h)
                todo.append(h)
    return found


def _object(source):
    return os.path.join(OBJECTS, os.path.splitext(source)[0] + ".o")


def _object_stale(source):
    obj = _object(source)
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    return any(os.path.getmtime(d) > t for d in _headers(source) | {os.path.join(CSRC, source)})


def _stale():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(d) > t for s in SOURCES for d in _headers(s) | {os.path.join(CSRC, s)})


def _run(cmds):
    """Runs the commands side by side; their output, in order."""
    ps = [subprocess.Popen(c, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for c in cmds]
    outs = [p.communicate()[0] for p in ps]
    if any(p.returncode != 0 for p in ps):
        raise RuntimeError("nvcc failed:\n" + "".join(o for o, p in zip(outs, ps) if p.returncode != 0))
    return "".join(outs)


def build(force=False, verbose=False):
    """Compile the CUDA sources (one process each) and link libdlf_b200.so; returns the library path."""
    if not force and not _stale():
        return LIB
    os.makedirs(OBJECTS, exist_ok=True)
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    arch = ["-gencode", "arch=compute_100a,code=sm_100a"]
    flags = ["-std=c++17", "-O3", "-lineinfo", "-Xcompiler", "-fPIC"] + arch + (["-Xptxas", "-v"] if verbose else [])
    said = _run([[nvcc] + flags + ["-c", "-o", _object(s), os.path.join(CSRC, s)] for s in SOURCES if force or _object_stale(s)])
    if verbose:
        sys.stderr.write(said)
    _run([[nvcc, "-shared"] + arch + ["-o", LIB] + [_object(s) for s in SOURCES]])
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
