"""CPU (-m "not gpu"): which objects the incremental build compiles again (with a compiler that only writes down that it was called)."""
import os

import pytest

from aas_enhancement_amd import build as b


@pytest.fixture
def tree(tmp_path, monkeypatch):
    src = tmp_path / "csrc"
    src.mkdir()
    for f in ("one.hip", "two.hip"):
        (src / f).write_text("")
    log = tmp_path / "log"
    cc = tmp_path / "cc"
    cc.write_text('#!/bin/sh\nfor a; do last="$out"; out="$a"; [ "$last" = -o ] && o="$a"; done\necho "$@" >> %s\n[ -e %s/broken ] && exit 1\n: > "$o"\n'
                  % (log, tmp_path))
    cc.chmod(0o755)
    monkeypatch.setattr(b, "SRC", str(src))
    monkeypatch.setattr(b, "OBJ", str(tmp_path / "lib" / "obj"))
    monkeypatch.setattr(b, "LIB", str(tmp_path / "lib" / "lib.so"))
    monkeypatch.setattr(b, "HIPCC", str(cc))

    def compiled():
        lines = log.read_text().split("\n") if log.exists() else []
        if log.exists():
            log.unlink()
        return sorted(os.path.basename(w) for line in lines if " -c " in line for w in line.split() if w.endswith(".hip"))
    return tmp_path, src, compiled


def test_changed_sources_only(tree):
    _, src, compiled = tree
    b.build(verbose=False)
    assert compiled() == ["one.hip", "two.hip"]
    b.build(verbose=False)
    assert compiled() == []
    later = os.path.getmtime(b.OBJ + "/one.o") + 10
    os.utime(str(src / "one.hip"), (later, later))
    b.build(verbose=False)
    assert compiled() == ["one.hip"]


def test_another_command_compiles_all_again(tree, monkeypatch):
    """Objects of other flags are not linked in beside new ones - nor objects that no record of their flags lies beside."""
    tmp, _, compiled = tree
    b.build(verbose=False)
    compiled()
    monkeypatch.setattr(b, "FLAGS", b.FLAGS + ["-DOTHER"])
    (tmp / "broken").write_text("")
    with pytest.raises(RuntimeError):
        b.build(verbose=False)
    compiled()
    (tmp / "broken").unlink()
    before = b.FLAGS[:-1]
    with monkeypatch.context() as m:                      # a build that failed on the way may have left objects of either
        m.setattr(b, "FLAGS", before)
        b.build(verbose=False)
        assert compiled() == ["one.hip", "two.hip"]
    b.build(verbose=False)
    assert compiled() == ["one.hip", "two.hip"]
    b.build(verbose=False)
    assert compiled() == []
    for f in os.listdir(b.OBJ):
        if not f.endswith(".o"):
            os.unlink(os.path.join(b.OBJ, f))
    b.build(verbose=False)
    assert compiled() == ["one.hip", "two.hip"]
