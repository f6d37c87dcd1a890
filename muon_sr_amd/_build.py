"""Builds libmuon_sr_amd.so (the gfx950 HIP kernels + C ABI) and _nodes.so (autograd nodes that call it) in-tree.

The library depends only on the HIP runtime; it is loaded with ctypes.  _nodes.so is host code against torch's C++
headers, a Python module; it finds the library beside itself.  The library is built whether or not they can be.
"""
from __future__ import annotations

import glob
import os
import subprocess
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmuon_sr_amd.so")
NODES = os.path.join(HERE, "_nodes.so")
ARCH = os.environ.get("MSR_OFFLOAD_ARCH", "gfx950")

# IEEE fp32 without contraction (the kernels restate the reference's expression
# order), no packed-fp32 instructions, correctly rounded / and sqrt (HIP default).
HIPCC_FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-shared",
    "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")))


def hipcc() -> str:
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    cand = os.path.join(rocm, "bin", "hipcc")
    return cand if os.path.exists(cand) else "hipcc"


# Per-source extra flags (none at present; kept so a source can get its own).
EXTRA_FLAGS = {}

_NOISE = "is not a recognized feature for this target"  # hipcc host pass; harmless


def _finish(cmd, res, verbose):
    err = "\n".join(line for line in res.stderr.splitlines() if _NOISE not in line)
    if res.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({res.returncode}): {' '.join(cmd)}\n{err}")
    if verbose and err.strip():
        print(err)


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    _finish(cmd, subprocess.run(cmd, capture_output=True, text=True), verbose)


def nodes_commands(obj: str, out: str):
    """Of the autograd nodes: compile, and link (after the library, which they are linked with)."""
    import torch
    from torch.utils.cpp_extension import include_paths
    includes = [*include_paths("cuda"), sysconfig.get_paths()["include"]]
    compile_ = ["g++", "-O2", "-std=c++17", "-fPIC", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-DTORCH_API_INCLUDE_EXTENSION_H",
                "-DTORCH_EXTENSION_NAME=_nodes", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                *(f for i in includes for f in ("-isystem", i)), "-c", "-o", obj, os.path.join(CSRC, "nodes.cpp")]
    link = ["g++", "-shared", "-o", out, obj, f"-L{HERE}", "-lmuon_sr_amd", "-Wl,-rpath,$ORIGIN",
            f"-L{os.path.join(os.path.dirname(torch.__file__), 'lib')}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_hip"]
    return compile_, link


def build(verbose: bool = False) -> str:
    """Compile every HIP source (each with its own flags, all at once) and link one
    shared library, then the autograd nodes.  Always recompiles; objects go to muon_sr_amd/_build/.  Where the nodes cannot be built (no g++, no
    headers of Python or torch) the library is there all the same when the error is raised."""
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    objs, jobs = [], []

    def start(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        return cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)

    def end(cmd, proc):
        out, err = proc.communicate()
        _finish(cmd, subprocess.CompletedProcess(cmd, proc.returncode, out, err), verbose)

    nodes = failed = None
    try:
        nodes_compile, nodes_link = nodes_commands(os.path.join(objdir, "nodes.cpp.o"), NODES + ".tmp")
        nodes = start(nodes_compile)
    except (ImportError, OSError) as e:
        failed = e
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src) + ".o")
        flags = [f for f in HIPCC_FLAGS if f != "-shared"]
        jobs.append(start([hipcc(), *flags, *EXTRA_FLAGS.get(os.path.basename(src), []), "-c", "-o", obj, src]))
        objs.append(obj)
    for job in jobs:
        end(*job)
    tmp = LIB + ".tmp"
    _run([hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs], verbose)
    # (nodes of an earlier build know that build's library)
    if os.path.exists(NODES):
        os.remove(NODES)
    os.replace(tmp, LIB)
    try:
        if failed is not None:
            raise failed
        end(*nodes)
        _run(nodes_link, verbose)
    except (ImportError, OSError, RuntimeError) as e:
        raise RuntimeError(f"{LIB} is built, but not the autograd nodes of layer_norm, embedding, linear_cross_entropy and balance_loss, "
                           f"which need g++ and the headers of Python and torch: {e}") from e
    os.replace(NODES + ".tmp", NODES)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))
