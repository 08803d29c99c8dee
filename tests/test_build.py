"""The library is built by hipcc alone: the torch module beside it neither stops it nor makes it count as not built."""
import os

import pytest

from recommend_amd import build as rbuild


@pytest.fixture
def elsewhere(tmp_path, monkeypatch):
    """Built in a folder of its own, from the host's source only, by a compiler that writes its output file."""
    compiler = tmp_path / "cc"
    compiler.write_text('#!/bin/sh\nwhile [ "$1" != "-o" ]; do shift; done\necho built > "$2"\n')
    compiler.chmod(0o755)
    monkeypatch.setenv("HIPCC", str(compiler))
    monkeypatch.setattr(rbuild, "LIB_DIR", str(tmp_path))
    monkeypatch.setattr(rbuild, "LIB_PATH", str(tmp_path / "library.so"))
    monkeypatch.setattr(rbuild, "TORCH_OPS_PATH", str(tmp_path / "module.so"))
    monkeypatch.setattr(rbuild, "SOURCES", ["host.cpp"])
    return monkeypatch, str(compiler)


@pytest.mark.parametrize("command", [["false"], ["no-such-compiler"]])
def test_the_library_is_complete_where_the_module_fails(elsewhere, command):
    patch, _ = elsewhere
    patch.setattr(rbuild, "torch_ops_command", lambda out: command)
    open(rbuild.TORCH_OPS_PATH, "w").close()              # of other sources: gone afterwards
    with pytest.raises(RuntimeError, match="library is complete"):
        rbuild.build(force=True, verbose=False)
    assert os.path.exists(rbuild.LIB_PATH) and not os.path.exists(rbuild.TORCH_OPS_PATH)
    assert not rbuild.needs_library() and rbuild.needs_build()


def test_only_what_is_missing_is_built(elsewhere):
    patch, compiler = elsewhere
    patch.setattr(rbuild, "torch_ops_command", lambda out: [compiler, "-o", out])
    rbuild.build(verbose=False)
    assert not rbuild.needs_build()
    os.remove(rbuild.TORCH_OPS_PATH)
    patch.setenv("HIPCC", "false")                        # (the library is not built again)
    rbuild.build(verbose=False)
    assert not rbuild.needs_build()
    os.remove(rbuild.LIB_PATH)
    with pytest.raises(RuntimeError, match="host.cpp"):
        rbuild.build(verbose=False)
