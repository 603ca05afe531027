"""Ahead-of-time build of libaas_hip.so (hipcc, gfx950 only) and of nothing else.

    python -m aas_enhancement_amd.build        # incremental, parallel

The library is built IN-TREE at aas_enhancement_amd/lib/libaas_hip.so so that it travels to the GPU
box with the repo snapshot (git-ignored, not gpurun-ignored).
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "lib", "obj")
LIB = os.path.join(HERE, "lib", "libaas_hip.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# No packed fp32 instructions in the code objects: some of their forms have given wrong results now and then on this hardware.
# (The host pass of hipcc does not know the feature and says so; that is harmless.)
FLAGS = ["--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++17", "-Wall", "-Wno-unused-function",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _newer(a, b):
    return (not os.path.exists(b)) or os.path.getmtime(a) > os.path.getmtime(b)


def build(force=False, verbose=True):
    os.makedirs(OBJ, exist_ok=True)
    srcs = sorted(f for f in os.listdir(SRC) if f.endswith(".hip"))
    hdrs = [os.path.join(SRC, f) for f in os.listdir(SRC) if f.endswith(".h")]
    hdrs.append(os.path.join(os.path.dirname(HERE), "include", "aas_hip.h"))
    hdrs.append(os.path.join(os.path.dirname(HERE), "include", "aas_warpctc.h"))
    # what the objects were compiled with lies beside them: another compiler or other flags compile everything again
    command, record = " ".join([HIPCC] + FLAGS), os.path.join(OBJ, "command.txt")
    if not os.path.exists(record) or open(record).read() != command:
        force = True
        if os.path.exists(record):
            os.unlink(record)         # (a build that fails on the way leaves objects of both)
    jobs = []
    for f in srcs:
        src, obj = os.path.join(SRC, f), os.path.join(OBJ, f[:-4] + ".o")
        if force or _newer(src, obj) or any(_newer(h, obj) for h in hdrs):
            jobs.append((src, obj))

    def cc(job):
        src, obj = job
        r = subprocess.run([HIPCC] + FLAGS + ["-c", src, "-o", obj], capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("hipcc failed for %s:\n%s" % (src, r.stderr[-4000:]))
        return src

    if jobs:
        with ThreadPoolExecutor(max_workers=min(8, len(jobs))) as ex:
            for s in ex.map(cc, jobs):
                if verbose:
                    print("[build] compiled", os.path.basename(s), flush=True)
    if jobs:
        with open(record, "w") as f:
            f.write(command)
    objs = [os.path.join(OBJ, f[:-4] + ".o") for f in srcs]
    if jobs or not os.path.exists(LIB):
        r = subprocess.run([HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs,
                           capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("link failed:\n%s" % r.stderr[-4000:])
        if verbose:
            print("[build] linked", LIB, flush=True)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
