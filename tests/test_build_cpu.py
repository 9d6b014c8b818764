"""CPU: the build compiles what an edit, other flags or an unfinished build left behind (with a stand-in for the compiler)."""
import os
import stat

import pytest

from gan_amd import build as B


@pytest.fixture
def tree(tmp_path, monkeypatch):
    csrc = tmp_path / "gan_amd" / "csrc"
    csrc.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    for f in ("common.h", "swin_common.h", "seq_common.h", "a.hip", "b.hip"):
        (csrc / f).write_text("")
    (tmp_path / "include" / "gan_amd.h").write_text("")
    log = tmp_path / "log"
    cc = tmp_path / "cc"
    cc.write_text(f"""#!/bin/bash
[ -e {tmp_path}/broken ] && [[ "$*" == *"$(cat {tmp_path}/broken)"* ]] && exit 1
echo "$@" >> {log}
while [ $# -gt 0 ]; do [ "$1" = -o ] && echo built > "$2"; shift; done
""")
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("HIPCC", str(cc))
    monkeypatch.setattr(B, "HERE", tmp_path / "gan_amd")
    monkeypatch.setattr(B, "CSRC", csrc)
    monkeypatch.setattr(B, "LIB", tmp_path / "gan_amd" / "lib.so")
    monkeypatch.setattr(B, "SOURCES", ["a.hip", "b.hip"])

    def run():
        """What a build compiled and linked."""
        log.write_text("")
        for f in tmp_path.rglob("*"):  # everything so far is a second older than what comes now
            if f.is_file():
                t = f.stat().st_mtime - 1
                os.utime(f, (t, t))
        B.build()
        return ["link" if "-shared" in line else line.split("-c ")[1].split()[0].rsplit("/", 1)[1] for line in log.read_text().splitlines()]

    run.path = tmp_path
    return run


def test_only_what_changed_is_compiled(tree):
    assert sorted(tree()) == ["a.hip", "b.hip", "link"]
    assert tree() == []
    src = B.CSRC / "b.hip"
    later = src.stat().st_mtime + 3  # (a build ages every file by a second first)
    os.utime(src, (later, later))
    assert tree() == ["b.hip", "link"]
    assert tree.path.joinpath("log").read_text().count("-c ") == 1


def test_other_flags_or_another_compiler_compile_everything(tree, monkeypatch):
    tree()
    monkeypatch.setattr(B, "FLAGS", B.FLAGS + ["-DOTHER"])
    assert sorted(tree()) == ["a.hip", "b.hip", "link"]
    assert tree() == []
    other = tree.path / "cc2"
    other.write_text((tree.path / "cc").read_text())
    other.chmod(0o755)
    monkeypatch.setenv("HIPCC", str(other))
    assert sorted(tree()) == ["a.hip", "b.hip", "link"]


def test_objects_of_an_unknown_build_are_compiled_again(tree):
    tree()
    for f in (B.CSRC / "build").glob("*"):
        if f.suffix != ".o":
            f.unlink()
    assert sorted(tree()) == ["a.hip", "b.hip", "link"]


@pytest.mark.parametrize("fails", ["a.hip.o", "-shared"])
def test_after_a_failed_build_the_rest_is_made_up_for(tree, monkeypatch, fails):
    """New flags, and a build that ends after one object or before the link: the next one leaves nothing of the old flags."""
    tree()
    monkeypatch.setattr(B, "FLAGS", B.FLAGS + ["-DOTHER"])
    (tree.path / "broken").write_text(fails)
    with pytest.raises(RuntimeError):
        tree()
    (tree.path / "broken").unlink()
    assert "link" in tree()
    assert tree() == []


def test_back_to_the_old_flags_after_a_failed_build(tree, monkeypatch):
    tree()
    old = B.FLAGS
    monkeypatch.setattr(B, "FLAGS", old + ["-DOTHER"])
    (tree.path / "broken").write_text("b.hip.o")
    with pytest.raises(RuntimeError):
        tree()
    (tree.path / "broken").unlink()
    monkeypatch.setattr(B, "FLAGS", old)
    assert sorted(tree()) == ["a.hip", "b.hip", "link"]
