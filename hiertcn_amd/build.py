"""Builds libhiertcn_gfx950.so in-tree with hipcc (gfx950 only).  Used by __graft_entry__.build()
and by `python -m hiertcn_amd.build`.  hipcc cross-compiles without a GPU."""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libhiertcn_gfx950.so")
SOURCES = ["api.hip", "prep.hip", "pool_gru.hip", "gru_persist.hip", "tcn.hip", "tcn_layers.hip", "score.hip", "score_bwd.hip", "metrics.hip", "train.hip", "gmm.hip", "gmm_train.hip", "gmm_gram.hip", "exact.hip", "gemm.hip", "gru_x3.hip", "score_x3.hip", "score_x3w.hip", "lgru_tile.hip", "lgru_pipe.hip", "lgru_wide.hip",
           "ops.hip", "glr.hip", "seq_loss.hip", "adamw.hip"]
OPS_SOURCES = ("ops.hip", "glr.hip", "seq_loss.hip", "adamw.hip")   # the sequence operators (include/hiertcn_ops.h)
FLAGS = ["--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++17", "-Wall", "-Wno-unused-function", "-Wno-pass-failed", "-Wno-shift-negative-value",
         "-fno-gpu-rdc", "-D__HIP_PLATFORM_AMD__",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]   # no packed fp32 arithmetic: some of its forms have given wrong results on this hardware now and then


def _hipcc():
    for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if c and (os.path.isabs(c) and os.path.exists(c) or not os.path.isabs(c)):
            return c
    raise RuntimeError("hipcc not found")


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


NO_NAN_SOURCES = ("score.hip", "score_x3.hip", "score_x3w.hip")


def _flags_of(src: str, extra=()):
    # score.hip: logits are finite or -inf by construction; without NaN-honouring fmaxf needs no
    # canonicalising v_max on MFMA results (cdna_hip_programming.md, attention 'Pitfalls')
    return [*FLAGS, *(["-fno-honor-nans"] if src in NO_NAN_SOURCES else []), *extra]


def _compile(sources, obj_dir: str, extra=(), force: bool = False, verbose: bool = False):
    """Objects of `sources` in obj_dir -> (their paths, whether any was compiled).  An object is stale when its source or a header is newer, and ALL of a
    directory are when the flags they were compiled with (its objects.flags) are not today's: a changed flag leaves no old object behind."""
    os.makedirs(obj_dir, exist_ok=True)
    hipcc, headers = _hipcc(), _headers()
    stamp, flagset = os.path.join(obj_dir, "objects.flags"), "\n".join(" ".join([src, *_flags_of(src, extra)]) for src in sources)
    try:
        with open(stamp) as f:
            same = f.read() == flagset
    except OSError:
        same = False
    jobs, objs = [], []
    for src in sources:
        s, o = os.path.join(CSRC, src), os.path.join(obj_dir, src.replace(".hip", ".o"))
        objs.append(o)
        if force or not same or _stale(o, [s] + headers + _ops_headers(src)):
            jobs.append((src, s, o))
    if not same and os.path.exists(stamp):
        os.remove(stamp)                      # (until all of them are: a run that fails or is stopped half-way starts over)

    def cc(job):
        src, s, o = job
        cmd = [hipcc, *_flags_of(src, extra), "-c", s, "-o", o]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("hipcc failed: %s\n%s\n%s" % (" ".join(cmd), r.stdout, r.stderr))
        if verbose and r.stderr.strip():
            print(r.stderr, file=sys.stderr)

    if jobs:
        with ThreadPoolExecutor(max_workers=min(6, len(jobs))) as ex:
            list(ex.map(cc, jobs))
    if not same:
        with open(stamp, "w") as f:
            f.write(flagset)
    return objs, bool(jobs)


def _link(lib: str, objs):
    # nothing but the HIP runtime: every kernel of the library, the plain GEMMs of the backward pass included (csrc/gemm.hip), is its own
    r = subprocess.run([_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", "-o", lib, *objs], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("link failed: %s\n%s" % (r.stdout, r.stderr))


LIB_F16 = os.path.join(HERE, "libhiertcn_gfx950_f16.so")


LIB_TESTHOOKS = os.path.join(HERE, "libhiertcn_gfx950_testhooks.so")
TESTHOOK_SOURCES = ("gru_persist.hip", "lgru_pipe.hip", "api.hip", "glr.hip", "adamw.hip")   # the sources that hold a fault-injection switch / a test probe


# libhiertcn_gfx950_ablation.so: the bfloat16 library PLUS every superseded kernel and A/B switch (-DHIERTCN_ABLATION=1): the previous forms of the
# scoring / top-k / TCN-layer kernels, the legacy scoring backward (score_grad.hip), the timing flavours.  Only there are the old HIERTCN_* environment
# switches of those alternatives looked up.  Loaded through HIERTCN_LIB / Engine(lib_variant="ablation") by the A/B tests and scripts/reproduce.sh;
# the shipped libraries hold one kernel per job.
LIB_ABLATION = os.path.join(HERE, "libhiertcn_gfx950_ablation.so")
ABLATION_EXTRA_SOURCES = ["score_grad.hip"]


def _mentions_ablation(src: str) -> bool:
    with open(os.path.join(CSRC, src)) as f:
        t = f.read()
    return "HIERTCN_ABLATION" in t or "ABL_ENV" in t


def build_ablation(force: bool = False) -> str:
    build_lib(False)
    # a source without ablation content: the shipped library's object
    own = [src for src in SOURCES + ABLATION_EXTRA_SOURCES if src in ABLATION_EXTRA_SOURCES or _mentions_ablation(src)]
    objs, built = _compile(own, os.path.join(OBJ, "ablation"), ["-DHIERTCN_ABLATION=1"], force)
    objs += [os.path.join(OBJ, src.replace(".hip", ".o")) for src in SOURCES if src not in own]
    if force or built or _stale(LIB_ABLATION, objs):
        _link(LIB_ABLATION, objs)
    return LIB_ABLATION


def _headers():
    return [os.path.join(CSRC, h) for h in ("common.h", "train.h", "exact.h", "gemm.h", "gmm.h", "score_geom.h", "score_lists.h", "score_x3.h")] + [
        os.path.join(HERE, "..", "include", "hiertcn.h")]


def _ops_headers(src: str):
    return [os.path.join(CSRC, "ops.h"), os.path.join(HERE, "..", "include", "hiertcn_ops.h")] if src in OPS_SOURCES or src == "api.hip" else []


LIB_PACKER = os.path.join(HERE, "libhiertcn_packer.so")   # host-side batch packer (csrc/packer.c: plain C, gcc)


def build_packer(force: bool = False) -> str:
    src = os.path.join(CSRC, "packer.c")
    if force or _stale(LIB_PACKER, [src]):
        r = subprocess.run(["gcc", "-O2", "-fPIC", "-shared", "-std=c99", "-Wall", "-o", LIB_PACKER, src], capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("gcc failed: %s\n%s" % (src, r.stderr))
    return LIB_PACKER


def build_all(force: bool = False, verbose: bool = False):
    """Both storage variants: bfloat16 (default, training + inference) and IEEE half (-DHIERTCN_F16, inference)."""
    libs = build_lib(force, verbose), build_lib(force, verbose, f16=True)
    build_testhooks(force)
    build_ablation(force)
    build_packer(force)
    return libs


def build_testhooks(force: bool = False) -> str:
    """libhiertcn_gfx950_testhooks.so: the bfloat16 library with the fault-injection switches of the tests compiled IN (-DHIERTCN_TEST_HOOKS; the
    shipped libraries have none).  Same objects as the shipped library except the few sources that hold a switch.  Loaded only by
    tests/tools/persist_timeout_probe.py through HIERTCN_LIB."""
    build_lib(False)
    objs, built = _compile(TESTHOOK_SOURCES, os.path.join(OBJ, "testhooks"), ["-DHIERTCN_TEST_HOOKS=1"], force)
    objs += [os.path.join(OBJ, src.replace(".hip", ".o")) for src in SOURCES if src not in TESTHOOK_SOURCES]
    if force or built or _stale(LIB_TESTHOOKS, objs):
        _link(LIB_TESTHOOKS, objs)
    return LIB_TESTHOOKS


def build_lib(force: bool = False, verbose: bool = False, extra_flags=(), f16: bool = False) -> str:
    lib = LIB_F16 if f16 else LIB
    if f16:
        extra_flags = tuple(extra_flags) + ("-DHIERTCN_F16=1",)
    # flags of the caller's have an object directory of their own, and the library remembers which flags it was linked from: an
    # experiment can never leave objects (or a library) behind that a later plain build would ship as fresh
    import hashlib
    user_flags = [f for f in extra_flags if f != "-DHIERTCN_F16=1"]
    obj_dir = os.path.join(OBJ, *(["f16"] if f16 else []), *(["x" + hashlib.sha1(" ".join(user_flags).encode()).hexdigest()[:8]] if user_flags else []))
    flagset = " ".join([*FLAGS, *extra_flags])
    stamp = lib + ".flags"
    try:
        with open(stamp) as f:
            relink = f.read() != flagset
    except OSError:
        relink = True
    objs, built = _compile(SOURCES, obj_dir, extra_flags, force, verbose)
    if force or built or relink or _stale(lib, objs):
        _link(lib, objs)
        with open(stamp, "w") as f:
            f.write(flagset)
    return lib


if __name__ == "__main__":
    print(*build_all(force="--force" in sys.argv, verbose=True))
