"""The compile flags belong to a kernel's identity: profiles are quoted, and objects reused, only for the flags they were made with."""
import os

import pytest

from yolo_master_amd import build

OTHER = {"NO_PACKED_FP32": [], "NO_CONTRACT": set(), "ARCH": "gfx942"}


@pytest.mark.parametrize("name", OTHER)
def test_the_source_hash_holds_the_flags(monkeypatch, name):
    before = build.source_hash(), build.source_hash(tokens=True)
    monkeypatch.setattr(build, name, OTHER[name])
    assert build.source_hash() != before[0]
    assert (build.source_hash(tokens=True) != before[1]) == (name != "NO_CONTRACT")   # none of the token sources is in it


def test_the_two_hashes_hold_their_own_sources(monkeypatch, tmp_path):
    for f in build.CSRC.iterdir():
        if f.suffix in (".hip", ".h"):
            (tmp_path / f.name).write_bytes(f.read_bytes())
    before = build.source_hash(), build.source_hash(tokens=True)
    monkeypatch.setattr(build, "CSRC", tmp_path)
    assert (build.source_hash(), build.source_hash(tokens=True)) == before
    for f, detector, tokens in (("expert.hip", False, True), ("rows.h", False, True), ("dwconv.hip", True, False), ("glds.h", True, True)):
        (tmp_path / f).write_text((tmp_path / f).read_text() + "\nint one_more;   // and a comment\n")
        now = build.source_hash(), build.source_hash(tokens=True)
        assert (now[0] != before[0], now[1] != before[1]) == (detector, tokens), f
        before = now
        (tmp_path / f).write_text("// 12 us\n" + (tmp_path / f).read_text().replace("and a comment", "another") + "/* two\nlines */\n")
        assert (build.source_hash(), build.source_hash(tokens=True)) == before   # comments are not the kernel


def test_objects_of_other_flags_are_stale(monkeypatch, tmp_path):
    monkeypatch.setattr(build, "CSRC", tmp_path)
    src, obj, flags = tmp_path / "k.hip", tmp_path / "k.o", ["-O3", "-a"]
    src.write_text("")
    assert build._stale("k.hip", obj, flags, 0.0)
    obj.write_text("")
    assert build._stale("k.hip", obj, flags, 0.0)          # nothing says how it was compiled
    obj.with_suffix(".flags").write_text("-O3 -a")
    assert not build._stale("k.hip", obj, flags, 0.0)
    assert build._stale("k.hip", obj, ["-O3"], 0.0) and build._stale("k.hip", obj, flags, obj.stat().st_mtime + 1)
    os.utime(src, (obj.stat().st_mtime + 5,) * 2)
    assert build._stale("k.hip", obj, flags, 0.0)
