"""What the library's build compiles again (no compiler runs here)."""

import os

import pytest

import __graft_entry__ as G


@pytest.fixture
def compiled(tmp_path, monkeypatch):
    """Builds into a folder of its own with a compiler that writes empty files; a call's sources and whether it linked."""
    monkeypatch.setattr(G, "ROOT", str(tmp_path))
    monkeypatch.setattr(G, "HIP_LIB", str(tmp_path / "appfl_amd" / "lib" / "lib.so"))
    done = []

    def check_call(command, cwd=None):
        out = command[command.index("-o") + 1]
        with open(out, "w"):
            pass
        done.append("link" if "-c" not in command else os.path.basename(command[command.index("-c") + 1]))
    monkeypatch.setattr(G.subprocess, "check_call", check_call)

    def build(**kw):
        done.clear()
        G.build_hip(lib=G.HIP_LIB, **kw)
        return sorted(done)
    return build


EVERYTHING = sorted([os.path.basename(s) for s in G.HIP_SOURCES] + ["link"])


def test_what_is_up_to_date_stays(compiled):
    assert compiled() == EVERYTHING and compiled() == []
    assert compiled(force=True) == EVERYTHING


def test_changed_flags_compile_everything_again(compiled, monkeypatch):
    compiled()
    monkeypatch.setattr(G, "HIPCC_FLAGS", G.HIPCC_FLAGS + ["-DSOMETHING"])
    assert compiled() == EVERYTHING and compiled() == []
    assert compiled(extra_flags=("-DMORE",)) == EVERYTHING


def test_objects_of_an_unknown_command_are_compiled_again(compiled):
    compiled()
    objects = os.path.join(G.ROOT, "appfl_amd", "lib", "obj")
    os.remove(os.path.join(objects, "token_ops.o.cmd"))
    assert compiled() == ["link", "token_ops.hip"]


def test_a_failed_compilation_is_taken_up_again(compiled, monkeypatch):
    compiled()
    works = G.subprocess.check_call

    def fails(command, cwd=None):
        if "-c" in command:
            raise G.subprocess.CalledProcessError(1, command)
        works(command, cwd)
    with monkeypatch.context() as m:
        m.setattr(G.subprocess, "check_call", fails)
        with pytest.raises(G.subprocess.CalledProcessError):
            compiled(force=True)
    assert "link" in compiled()
    assert compiled() == []
