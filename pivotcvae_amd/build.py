"""Build recipe for libpcvae_hip.so (gfx950 only; hipcc cross-compiles without a GPU).

    python -m pivotcvae_amd.build [--force] [--verbose]

The library is built IN-TREE (pivotcvae_amd/lib/) so it travels with the repo snapshot to the GPU box.
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "lib", "libpcvae_hip.so")
SOURCES = ["error.cpp", "elementwise.hip", "gemm_f32.hip", "catalog_f32.hip", "catalog_bf16.hip", "catalog_sparse.hip", "candidate_ce.hip", "catalog_sample.hip",
           "layer_norm.hip", "act8.hip", "catalog_api.cpp"]
HEADERS = ["common.h", "act8.h", "catalog_plan.h", "catalog_x3.h", os.path.join("..", "..", "include", "pcvae.h")]
# -packed-fp32-ops: hipcc forms v_pk_add / mul / fma_f32 out of ordinary float code by itself, and some of their operand forms have been
# seen to give wrong results on this chip; without the feature every one of them is two scalar instructions of the same rounding.
# (The host pass does not know the feature and says so: harmless.)
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function", "-Wno-inline-asm",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _stale(out, deps, recipe):
    """out is missing, older than a file it is made of, or was not made (to the end) by this recipe, which lies in <out>.cmd"""
    try:
        with open(out + ".cmd") as f:
            made_by = f.read()
        t = os.path.getmtime(out)
    except OSError:
        return True
    return made_by != recipe or any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def _begin(out):
    if os.path.exists(out + ".cmd"):
        os.remove(out + ".cmd")


def _done(out, recipe):
    with open(out + ".cmd", "w") as f:
        f.write(recipe)


def build(force=False, verbose=False):
    """Compile every translation unit to an object, then link the shared library."""
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    objdir = os.path.join(HERE, "lib", "obj")
    os.makedirs(objdir, exist_ok=True)
    hdrs = [os.path.join(CSRC, h) for h in HEADERS]
    objs, procs = [], []
    for s in SOURCES:
        src = os.path.join(CSRC, s)
        if not os.path.exists(src):
            continue
        obj = os.path.join(objdir, os.path.splitext(s)[0] + ".o")
        objs.append(obj)
        recipe = " ".join([hipcc] + FLAGS + [s])   # (no paths: the tree may be built in one place and used in another)
        if force or _stale(obj, [src] + hdrs, recipe):
            cmd = [hipcc] + FLAGS + ["-x", "hip", "-c", src, "-o", obj]
            if verbose:
                print(" ".join(cmd), flush=True)
            _begin(obj)
            procs.append((s, obj, recipe, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    failed = False
    for s, obj, recipe, p in procs:
        out = p.communicate()[0].decode()
        if p.returncode != 0:
            failed = True
            sys.stderr.write(f"--- {s} ---\n{out}\n")
            continue
        _done(obj, recipe)
        if verbose and out.strip():
            print(f"--- {s} ---\n{out}")
    if failed:
        raise RuntimeError("hipcc failed")
    link = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC"]
    recipe = " ".join(link + [os.path.basename(o) for o in objs])
    if force or procs or _stale(LIB, objs, recipe):
        cmd = link + ["-o", LIB] + objs
        if verbose:
            print(" ".join(cmd), flush=True)
        _begin(LIB)
        subprocess.check_call(cmd)
        _done(LIB, recipe)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv or "-v" in sys.argv))
