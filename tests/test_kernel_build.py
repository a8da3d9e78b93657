"""What the kernel library's build compiles again (ops/build.py), with a stand-in for the compiler."""
import os
import time

import pytest

from determined_1_amd.ops import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Two sources, an output and a compiler that writes what it is asked for and notes it."""
    src = [tmp_path / "one.hip", tmp_path / "two.hip"]
    for s in src:
        s.write_text("x")
    log = tmp_path / "log"
    cc = tmp_path / "cc"
    cc.write_text(f"""#!/bin/sh
echo "$@" >> {log}
while [ $# -gt 0 ]; do [ "$1" = -o ] && echo x > "$2"; shift; done
""")
    cc.chmod(0o755)
    monkeypatch.setattr(build, "HERE", tmp_path)
    monkeypatch.setattr(build, "SOURCES", src)
    monkeypatch.setattr(build, "OUT", tmp_path / "lib.so")
    monkeypatch.setattr(build, "hipcc", lambda: str(cc))

    def compiled(**kw):
        log.write_text("")
        build.build(**kw)
        return sorted(s.stem for s in src if f"-c {s}" in log.read_text())

    return compiled, src, tmp_path


def _newer(path):
    later = time.time() + 5
    os.utime(path, (later, later))


def test_only_what_changed_is_compiled_again(tree):
    compiled, src, _ = tree
    assert compiled() == ["one", "two"]
    assert compiled() == []
    _newer(src[1])
    assert compiled() == ["two"]
    assert compiled(force=True) == ["one", "two"]


def test_other_flags_compile_everything_again(tree, monkeypatch):
    compiled, src, tmp = tree
    compiled()
    monkeypatch.setattr(build, "ARCH", "gfx000")
    assert compiled() == ["one", "two"]
    assert compiled() == []
    # objects of flags that nobody wrote down
    (tmp / "build" / "flags").unlink()
    assert compiled() == ["one", "two"]
    # a build that breaks off leaves the old flags' note behind, so the next one starts over
    monkeypatch.setattr(build, "ARCH", "gfx001")
    good = build.hipcc()
    monkeypatch.setattr(build, "hipcc", lambda: "/bin/false")
    with pytest.raises(Exception):
        build.build()
    monkeypatch.setattr(build, "hipcc", lambda: good)
    assert compiled() == ["one", "two"]


def test_a_library_without_objects_is_taken_as_it_is(tree):
    """As on a machine that only got the library."""
    import shutil

    compiled, src, tmp = tree
    compiled()
    shutil.rmtree(tmp / "build")
    assert compiled() == []
    _newer(src[0])
    assert compiled() == ["one", "two"]
