"""csrc/build.py compiles again whatever its flags, sources or headers changed for - without a compiler: its commands are recorded, not run."""
import importlib.util
import os
import subprocess

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "speechmix_amd", "csrc", "build.py")


@pytest.fixture
def make(tmp_path, monkeypatch):
    """make(**env) -> the sources that a build, as a new process with this environment would run it, compiles; and whether it links."""
    here = tmp_path / "pkg" / "csrc"
    here.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    (tmp_path / "include" / "speechmix_hip.h").write_text("// header\n")
    for n in ("gemm.hip", "verify.hip", "common.h"):
        (here / n).write_text("// " + n + "\n")
    ran = []

    def run(cmd, **kw):
        out = cmd[cmd.index("-o") + 1]
        with open(out, "w") as f:
            f.write("built")
        ran.append(cmd)
        return subprocess.CompletedProcess(cmd, 0, "", "")

    def go(change=None, force=False, **env):
        for k in ("SMX_DEFS", "SMX_PP_LAB"):
            monkeypatch.delenv(k, raising=False)
        for k, v in env.items():
            monkeypatch.setenv(k, v)
        spec = importlib.util.spec_from_file_location("smx_build_under_test", SRC)
        m = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(m)
        m.HERE, m.OBJ, m.OUT = str(here), str(here / "_obj"), str(tmp_path / "pkg" / "lib.so")
        monkeypatch.setattr(m.subprocess, "run", run)
        if change:
            change(m)
        ran.clear()
        m.build(force=force, verbose=False)
        return sorted(os.path.basename(c[c.index("-c") + 1]) for c in ran if "-c" in c), any("-shared" in c for c in ran)
    go.here, go.ran = here, ran
    return go


def test_nothing_changed_nothing_compiled(make):
    assert make() == (["gemm.hip", "verify.hip"], True)
    assert make() == ([], False)
    assert make(force=True) == (["gemm.hip", "verify.hip"], True)


def test_another_command_compiles_again(make):
    make()

    def more_flags(m):
        m.FLAGS = m.FLAGS + ["-DX=1"]
    assert make(more_flags) == (["gemm.hip", "verify.hip"], True)
    assert make(more_flags) == ([], False)
    assert make() == (["gemm.hip", "verify.hip"], True)          # and back
    assert make(SMX_DEFS="A=1,B=2") == (["gemm.hip", "verify.hip"], True)
    assert any("-DB=2" in c for c in make.ran)
    assert make(SMX_DEFS="A=1,B=2") == ([], False)
    assert make() == (["gemm.hip", "verify.hip"], True)


def test_an_object_that_is_newer_than_the_library_is_linked(make):
    """A build that ended between compiling and linking: the next one links, though it has nothing to compile."""
    make()
    lib = make.here.parent / "lib.so"
    t = os.path.getmtime(lib)
    os.utime(lib, (t - 100, t - 100))
    assert make() == ([], True)


def test_a_newer_source_or_header_compiles_again(make):
    make()
    obj = make.here / "_obj" / "verify.o"
    t = os.path.getmtime(obj) + 10
    os.utime(make.here / "verify.hip", (t, t))
    assert make()[0] == ["verify.hip"]
    for f in make.here.glob("_obj/*.o"):
        os.utime(f, (t + 10, t + 10))
    os.utime(make.here / "common.h", (t + 20, t + 20))
    assert make()[0] == ["gemm.hip", "verify.hip"]


def test_every_file_is_compiled_without_packed_fp32(make):
    """Some forms of the packed fp32 instructions give wrong results now and then: no file is compiled with them, and none writes them out."""
    make()
    for cmd in make.ran:
        if "-c" in cmd:
            at = cmd.index("-packed-fp32-ops")
            assert cmd[at - 3:at] == ["-Xclang", "-target-feature", "-Xclang"]
    here = os.path.dirname(SRC)
    for f in os.listdir(here):
        if f.endswith((".hip", ".h")):
            with open(os.path.join(here, f)) as s:
                assert not any(w in s.read() for w in ("v_pk_fma_f32", "v_pk_mul_f32", "v_pk_add_f32")), f
