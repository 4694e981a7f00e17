"""The build's steps with stand-in compilers: what fails, and what is left on the disk then."""
import os
import stat

import pytest

from geneface_amd.csrc import build


def _compiler(path, body):
    """A program that finds the file behind -o as $out."""
    path.write_text('#!/bin/sh\nwhile [ $# -gt 0 ]; do [ "$1" = -o ] && out=$2; shift; done\n' + body + "\n")
    path.chmod(path.stat().st_mode | stat.S_IXUSR)
    return str(path)


@pytest.fixture
def places(tmp_path, monkeypatch):
    """Everything that is built goes to a folder of the test's own, compilers come from there."""
    monkeypatch.setattr(build, "OUT", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build, "HOST_OUT", str(tmp_path / "host.so"))
    monkeypatch.setattr(build, "OBJ_DIR", str(tmp_path / "obj"))
    monkeypatch.setattr(build, "HIPCC", _compiler(tmp_path / "hipcc", 'echo made > "$out"'))
    monkeypatch.setenv("PATH", str(tmp_path) + os.pathsep + os.environ["PATH"])
    return tmp_path


def test_the_library_needs_no_host_compiler(places, capsys):
    _compiler(places / "g++", "echo no such header >&2; exit 1")
    assert build.build() == str(places / "lib.so") and (places / "lib.so").read_text() == "made\n"
    assert "no such header" in capsys.readouterr().err
    with pytest.raises(RuntimeError, match="no such header"):
        build.build_host()


def test_a_failing_device_compiler_is_an_error(places):
    _compiler(places / "g++", 'echo made > "$out"')
    _compiler(places / "hipcc", "echo wrong >&2; exit 1")
    with pytest.raises(RuntimeError, match="wrong"):
        build.build()
    assert not (places / "lib.so").exists()


def test_nothing_half_written_is_left_where_others_look(places):
    """A compiler that dies while it writes: what was there before is still there, whole, and no piece of a file beside it."""
    good, half = 'echo made > "$out"', 'echo half > "$out"; exit 1'
    _compiler(places / "g++", good)
    build.build()
    before = {f: f.read_text() for f in places.rglob("*") if f.suffix in (".so", ".o")}
    assert len(before) > 10 and set(before.values()) == {"made\n"}
    _compiler(places / "g++", half)
    with pytest.raises(RuntimeError):
        build.build_host(force=True)
    _compiler(places / "hipcc", half)
    with pytest.raises(RuntimeError):
        build.build(force=True)
    _compiler(places / "hipcc", f'case "$out" in *lib.so*) {half};; *) {good};; esac')
    with pytest.raises(RuntimeError):
        build.build(force=True)
    assert {f: f.read_text() for f in places.rglob("*") if f.suffix in (".so", ".o")} == before
    assert not [f for f in places.rglob("*") if "half" in f.name or f.name.endswith(".part")]


def test_a_file_appears_when_it_is_whole(places):
    """While the compiler writes, nothing is there to be loaded."""
    _compiler(places / "g++", f'echo half > "$out"; [ -e {places / "host.so"} ] && echo early >&2 && exit 1; echo whole >> "$out"')
    assert build.build_host() == str(places / "host.so") and (places / "host.so").read_text() == "half\nwhole\n"


def test_a_module_of_older_sources_is_not_kept_beside_a_new_library(places, capsys):
    _compiler(places / "g++", 'echo made > "$out"')
    build.build()
    assert (places / "host.so").exists()
    _compiler(places / "g++", "echo broken >&2; exit 1")
    build.build(force=True)
    assert "broken" in capsys.readouterr().err and (places / "lib.so").exists() and not (places / "host.so").exists()
