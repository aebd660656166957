"""Builds cutie_amd/libcutie_hip.so (gfx950) in-tree with hipcc.

    python -m cutie_amd.build [--force]

The .so is git-ignored but travels to the GPU box with the tree; nothing is built there.
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libcutie_hip.so")
SOURCES = ["core.hip", "grid_build.hip", "embed.hip", "embed_sorted.hip", "norm.hip", "group_norm.hip", "loss.hip", "optim.hip", "muon.hip", "conv_mfma.hip", "conv_wide.hip"]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-Wall", "-Wno-unused-function",
         # f32 arithmetic in scalar instructions alone, by choice (no v_pk_add_f32 and the like): the train step has the same rate per
         # clock with and without them (3952 docs/s at 1985 MHz held, 4181 at 2134)
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _stale(out, deps):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=True):
    hdrs = [os.path.join(CSRC, "common.h"), os.path.join(CSRC, "conv_common.h"),
            os.path.join(HERE, "..", "include", "cutie_hip.h")]
    objs = []
    procs = []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(CSRC, src.replace(".hip", ".o"))
        objs.append(o)
        if force or _stale(o, [s] + hdrs):
            cmd = [HIPCC] + FLAGS + ["-c", s, "-o", o]
            if verbose:
                print(" ".join(cmd), flush=True)
            procs.append((src, subprocess.Popen(cmd)))
    failed = [src for src, p in procs if p.wait() != 0]
    if failed:
        raise RuntimeError("hipcc failed for: %s" % ", ".join(failed))
    if force or procs or _stale(LIB, objs):
        cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print("built", LIB)
