"""Builds libpsgdk.so (the HIP engine behind include/psgdk.h) in-tree with hipcc for gfx950.

hipcc cross-compiles without a GPU, so this runs in the build container; the built .so travels with the source
tree to the GPU box (it is git-ignored, not gpurun-ignored).
"""
import os
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
# translation units, compiled side by side: the preconditioner engine, the microscaled (MX) operators, their products
SRCS = [os.path.join(HERE, "csrc", f) for f in ("psgdk.hip", "psgdk_mx.hip", "psgdk_mx_gemm.hip")]
OUT = os.path.join(HERE, "libpsgdk.so")
# the measurement probes (matrix-core / HBM ceilings of the chip for bench.py's peak_measured) are a library of their own:
# the product library carries no probe kernels
PROBE_SRC = os.path.join(HERE, "csrc", "psgdk_probe.hip")
PROBE_OUT = os.path.join(HERE, "libpsgdk_probe.so")


def _sources():
    d = os.path.join(HERE, "csrc")
    return [os.path.join(d, f) for f in sorted(os.listdir(d)) if f.endswith((".hip", ".hiph"))] + [
        os.path.join(os.path.dirname(HERE), "include", "psgdk.h")]


def needs_build() -> bool:
    if not os.path.exists(OUT) or not os.path.exists(PROBE_OUT):
        return True
    t = min(os.path.getmtime(OUT), os.path.getmtime(PROBE_OUT))
    return any(os.path.getmtime(s) > t for s in _sources())


# (packed fp32 off: some forms of the packed instructions hipcc makes from plain float code have returned wrong results now and then; the GPT-2-small
# step takes 1.574 ms without them and 1.581 with, the LRA update 10.86 and 10.84)
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wno-unused-result", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def object_command(hipcc, src, obj):
    """Compiles one unit.  Its id is its name: hipcc would make one of the whole command line, so that objects of the same source in another temporary
    folder, and with them the library, would differ from build to build (profiles carry the hash of the library that they measured)."""
    return [hipcc, *FLAGS, "-cuid=" + os.path.splitext(os.path.basename(src))[0], "-c", src, "-o", obj]


def _run(cmds, verbose):
    """Runs the commands side by side; the first that fails raises with its output."""
    procs = []
    for cmd in cmds:
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        procs.append(subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True))
    outs = [p.communicate()[0] for p in procs]
    for p, out in zip(procs, outs):
        if p.returncode != 0:
            raise RuntimeError("hipcc failed:\n" + out)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return OUT
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    with tempfile.TemporaryDirectory() as tmp:
        objs = [os.path.join(tmp, os.path.basename(s) + ".o") for s in SRCS]
        _run([object_command(hipcc, s, o) for s, o in zip(SRCS, objs)]
             + [[hipcc, *FLAGS, "-shared", PROBE_SRC, "-o", PROBE_OUT]], verbose)
        _run([[hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", *objs, "-o", OUT]], verbose)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
