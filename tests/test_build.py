"""__graft_entry__.build(): compiles on every call and puts the library in place whole (a stub stands for the compiler)"""
import os
import stat
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STUB = r"""#!%s
import os, sys
out = sys.argv[sys.argv.index("-o") + 1]
with open(out, "w") as f:
    f.write("half ")
    f.flush()
    if os.environ.get("STUB_FAILS") == ("link" if "-shared" in sys.argv else "compile"):
        sys.exit(1)
    f.write("whole")
with open(os.environ["STUB_LOG"], "a") as f:
    f.write(("link " if "-shared" in sys.argv else "compile ") + out + "\n")
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    import __graft_entry__ as G
    from fudanocr_amd import _lib
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    for name in ("a.hip", "b.hip"):
        (csrc / name).write_text("")
    stub = tmp_path / "hipcc"
    stub.write_text(STUB % sys.executable)
    stub.chmod(stub.stat().st_mode | stat.S_IXUSR)
    lib = tmp_path / "lib.so"
    lib.write_text("the last one")
    monkeypatch.setattr(G, "CSRC", str(csrc))
    monkeypatch.setattr(G, "LIB", str(lib))
    monkeypatch.setattr(_lib, "load", lambda: None)
    monkeypatch.setenv("HIPCC", str(stub))
    monkeypatch.setenv("STUB_LOG", str(tmp_path / "log"))
    return G, tmp_path, lib


def test_a_build_that_fails_leaves_the_library_alone(tree, monkeypatch):
    G, path, lib = tree
    for step in ("compile", "link"):
        monkeypatch.setenv("STUB_FAILS", step)
        with pytest.raises((RuntimeError, subprocess.CalledProcessError)):
            G.build()
        assert lib.read_text() == "the last one", step
    assert sorted(p.name for p in path.iterdir() if p.name.startswith("lib")) == ["lib.so"]


def test_every_build_compiles_into_files_of_its_own(tree):
    """the library appears under its name in one step, and two builds at once share no object file"""
    G, path, lib = tree
    G.build()
    first = (path / "log").read_text().split("\n")
    G.build(force=True)                                               # what earlier callers passed
    assert lib.read_text() == "half whole"
    lines = (path / "log").read_text().split()
    outs = lines[1::2]
    assert lines[0::2].count("compile") == 4 and lines[0::2].count("link") == 2 and len(first) == 4
    assert len(set(o for o, k in zip(outs, lines[0::2]) if k == "compile")) == 4
    assert str(lib) not in outs and not any(os.path.exists(o) for o in outs)


def test_the_command_names_what_it_does_not_know():
    res = subprocess.run([sys.executable, os.path.join(ROOT, "__graft_entry__.py"), "--fast"], capture_output=True, text=True)
    assert res.returncode != 0 and "--fast" in res.stderr
