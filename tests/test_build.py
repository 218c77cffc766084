"""When hiertcn_amd/build.py compiles again, with a compiler that only writes its output file and notes its command line."""
import os
import shutil
import subprocess
import types

import pytest

from hiertcn_amd import build as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def calls(tmp_path, monkeypatch):
    """The build in a tree of its own (sources where they are) -> the command lines it has run."""
    here = tmp_path / "hiertcn_amd"
    here.mkdir()
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    monkeypatch.setattr(B, "HERE", str(here))
    monkeypatch.setattr(B, "OBJ", str(here / "build"))
    for name in ("LIB", "LIB_F16", "LIB_TESTHOOKS", "LIB_ABLATION"):
        monkeypatch.setattr(B, name, str(here / (name.lower() + ".so")))
    monkeypatch.setattr(B, "FLAGS", ["--offload-arch=gfx950", "-O3"])
    monkeypatch.setattr(B, "_hipcc", lambda: "hipcc")
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("built")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(subprocess, "run", run)
    return ran


def compiled(ran):
    """Names of the sources compiled since the last look, and the number of links"""
    out = sorted(os.path.basename(c[c.index("-c") + 1]) for c in ran if "-c" in c), sum("-shared" in c for c in ran)
    ran.clear()
    return out


BUILDS = {
    "bf16": (lambda: B.build_lib(), lambda: B.SOURCES, 1),
    "f16": (lambda: B.build_lib(f16=True), lambda: B.SOURCES, 1),
    "testhooks": (lambda: B.build_testhooks(), lambda: [*B.SOURCES, *B.TESTHOOK_SOURCES], 2),
    "ablation": (lambda: B.build_ablation(), lambda: [*B.SOURCES, *B.ABLATION_EXTRA_SOURCES, *(s for s in B.SOURCES if B._mentions_ablation(s))], 2),
}


@pytest.mark.parametrize("which", BUILDS)
def test_a_changed_flag_compiles_everything(calls, monkeypatch, which):
    build, sources, links = BUILDS[which]
    everything = sorted(sources()), links
    build()
    assert compiled(calls) == everything
    build()
    assert compiled(calls) == ([], 0)
    monkeypatch.setattr(B, "FLAGS", [*B.FLAGS, "-mllvm-something"])
    build()
    assert all("-mllvm-something" in c for c in calls if "-c" in c)
    assert compiled(calls) == everything
    build()
    assert compiled(calls) == ([], 0)


def test_a_run_that_fails_half_way_starts_over(calls, monkeypatch):
    B.build_lib()
    compiled(calls)
    good = subprocess.run
    monkeypatch.setattr(B, "FLAGS", [*B.FLAGS, "-DNEW"])

    def fails(cmd, **kw):
        if cmd[-1].endswith("train.o"):
            return types.SimpleNamespace(returncode=1, stdout="", stderr="no")
        return good(cmd, **kw)

    monkeypatch.setattr(subprocess, "run", fails)
    with pytest.raises(RuntimeError, match="train.hip"):
        B.build_lib()
    monkeypatch.setattr(subprocess, "run", good)
    compiled(calls)
    monkeypatch.setattr(B, "FLAGS", B.FLAGS[:-1])          # back to the first flags: some objects have the others
    B.build_lib()
    assert compiled(calls) == (sorted(B.SOURCES), 1)


@pytest.mark.parametrize("which", ["bf16", "testhooks", "ablation"])
def test_the_operators_header_is_a_dependency_of_what_includes_it(calls, which):
    build, _, _ = BUILDS[which]
    build()
    compiled(calls)
    header = os.path.join(B.HERE, "..", "include", "hiertcn_ops.h")
    later = max(os.path.getmtime(os.path.join(d, f)) for d, _, fs in os.walk(B.HERE) for f in fs) + 10
    os.utime(header, (later, later))
    build()
    names, _ = compiled(calls)
    want = [s for s in B.SOURCES if s in B.OPS_SOURCES or s == "api.hip"]
    extra = [s for s in want if (s in B.TESTHOOK_SOURCES if which == "testhooks" else which == "ablation" and B._mentions_ablation(s))]
    assert names == sorted(want + extra)
