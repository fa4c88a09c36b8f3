"""Builds libmoe_hip.so in-tree with hipcc for gfx950: one object per source, compiled
side by side, then linked."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
SRCS = [os.path.join(HERE, "csrc", n) for n in ("moe_api.hip", "ops_api.hip", "router_api.hip", "mx_api.hip")]
OUT = os.path.join(HERE, "libmoe_hip.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
    # keep the compiler from forming packed-FP32 VALU ops (v_pk_*_f32)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def _run(cmds, verbose):
    """Runs the commands side by side; raises on the first that failed."""
    procs = []
    for cmd in cmds:
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append(subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                                      text=True))
    failed = None
    for cmd, p in zip(cmds, procs):
        text = p.communicate()[0]
        if p.returncode != 0:
            sys.stderr.write("\n".join(l for l in text.splitlines()
                                       if "packed-fp32-ops' is not a recognized feature" not in l) + "\n")
            failed = failed or (p.returncode, cmd[-1])
    if failed:
        raise RuntimeError(f"hipcc failed ({failed[0]}) on {failed[1]} building {OUT}")


def build(verbose=False):
    objs = [os.path.join(HERE, "csrc", os.path.basename(s).replace(".hip", ".o")) for s in SRCS]
    _run([[HIPCC, *FLAGS, "-c", "-o", o, s] for s, o in zip(SRCS, objs)], verbose)
    tmp = OUT + ".tmp"
    _run([[HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp, *objs]], verbose)
    for o in objs:
        os.remove(o)
    os.replace(tmp, OUT)
    return OUT


if __name__ == "__main__":
    print(build(verbose=True))
