"""Building the fused-ops extension (devspace_amd.ops.build), with a compiler that notes what it is given: what is linked
is always what the sources, flags and target now are, and carries their hash."""
import os
import threading
import time

import pytest

from devspace_amd.ops import build, fused

COMPILER = """#!/bin/sh
# --version | -c: "object of <arch>: <source>" | -shared: everything it links, joined
[ "$1" = --version ] && { cat "$HERE/compiler"; exit; }
src= out= arch= objs= compile= prev=
for a in "$@"; do
  [ "$prev" = -o ] && out="$a"
  [ "$prev" = -c ] && src="$a"
  case "$a" in --offload-arch=*) arch="${a#*=}";; -c) compile=1;; *.o|*.cpp) [ "$prev" = -o ] || objs="$objs $a";; esac
  prev="$a"
done
if [ -n "$compile" ]; then
  echo "${src##*/} $arch" >> "$HERE/log"
  sleep "$(cat "$HERE/delay")"
  { echo "object of $arch: $(cat "$src")"; grep -q broken "$src" && exit 1; } > "$out"
  [ ! -e "$HERE/edit" ] || { cat "$HERE/edit" >> "$HERE/rotary.hip"; rm "$HERE/edit"; }
else
  echo link >> "$HERE/log"
  cat $objs > "$out"
fi
"""


class Tree:
    def __init__(self, at):
        self.at = at
        for n in build.FUSED_SOURCES + build.FUSED_HEADERS:
            self.write(n, f"text of {n}\n")
        self.write("delay", "0")
        self.write("compiler", "one")

    def write(self, name, text, age=0):
        p = os.path.join(self.at, name)
        with open(p, "w") as f:
            f.write(text)
        os.utime(p, (time.time() - age, time.time() - age))

    def build(self, **kw):
        """Builds; returns what was compiled, in order of names, and the library's text."""
        log = os.path.join(self.at, "log")
        if os.path.exists(log):
            os.remove(log)
        out = build.build_fused(**kw)
        lines = open(log).read().split("\n")[:-1] if os.path.exists(log) else []
        text = open(out).read()
        assert build.source_sha() in text
        return sorted(x.split()[0] for x in lines if x != "link"), text


ALL = sorted(build.FUSED_SOURCES)


@pytest.fixture
def tree(tmp_path, monkeypatch):
    cc = tmp_path / "hipcc"
    cc.write_text(COMPILER)
    cc.chmod(0o755)
    at = tmp_path / "ops"
    at.mkdir()
    monkeypatch.setenv("HERE", str(at))
    monkeypatch.setattr(build, "HERE", str(at))
    monkeypatch.setattr(build, "hipcc", lambda: str(cc))
    t = Tree(str(at))
    assert t.build()[0] == ALL
    return t


def test_nothing_changed_nothing_done(tree):
    before = os.stat(build.fused_path()).st_mtime_ns
    assert tree.build()[0] == []
    assert os.stat(build.fused_path()).st_mtime_ns == before
    assert tree.build(force=True)[0] == ALL


def test_an_edit_with_an_old_time_is_compiled(tree):
    """A copy or a sync that keeps times brings a source that is older than its object."""
    tree.write("rotary.hip", "edited rotary\n", age=86400)
    assert tree.build()[0] == ["rotary.hip"]
    tree.write("rotary.hip", "again\n", age=86400)
    tree.write("dropout.hip", "edited dropout\n")
    done, text = tree.build()
    assert done == ["dropout.hip", "rotary.hip"]
    assert "again" in text and "edited dropout" in text and "edited rotary" not in text and "text of rotary" not in text


def test_a_header_another_target_compiler_or_torch_compiles_all(tree, monkeypatch):
    tree.write("fused_common.h", "other\n", age=86400)
    assert tree.build()[0] == ALL
    monkeypatch.setattr(build, "ARCH", "gfx942")
    tree.write("dropout.hip", "edited\n")
    done, text = tree.build()
    assert done == ALL and text.count("object of gfx942") == len(ALL) and "gfx950" not in text
    tree.write("compiler", "two")
    assert tree.build()[0] == ALL
    import torch

    monkeypatch.setattr(torch, "__version__", torch.__version__ + "x")
    assert tree.build()[0] == ALL
    sha = build.source_sha()
    monkeypatch.setattr(build, "FUSED_FLAGS", build.FUSED_FLAGS + ["-g"])
    assert build.source_sha() != sha and tree.build()[0] == ALL
    assert sorted(n.split(".hip")[0] + ".hip" for n in os.listdir(os.path.join(tree.at, "_obj")) if n.endswith(".o")) == ALL


def test_an_edit_during_the_build_is_an_error_and_not_kept(tree):
    old = open(build.fused_path()).read()
    tree.write("fused_ops.hip", "first edit\n")
    tree.write("edit", "second edit\n")
    with pytest.raises(RuntimeError, match="changed while"):
        build.build_fused()
    assert open(build.fused_path()).read() == old
    done, text = tree.build()
    assert done == ["fused_ops.hip", "rotary.hip"] and "first edit" in text and "second edit" in text


def test_a_failed_build_leaves_the_library_and_is_tried_again(tree):
    old = open(build.fused_path()).read()
    tree.write("dropout.hip", "broken\n")
    with pytest.raises(Exception, match="returned non-zero"):
        build.build_fused()
    assert open(build.fused_path()).read() == old
    tree.write("dropout.hip", "mended\n")
    done, text = tree.build()
    assert done == ["dropout.hip"] and "mended" in text


def test_a_library_from_elsewhere_is_linked_again(tree):
    want = open(build.fused_path()).read()
    with open(build.fused_path(), "w") as f:
        f.write("another state's")
    done, text = tree.build()
    assert done == [] and text.split("\n", 2)[2] == want.split("\n", 2)[2]
    os.remove(build.fused_path())
    assert tree.build()[0] == []


def test_two_builds_at_once(tree):
    """One waits for the other and finds its objects."""
    for n in build.FUSED_SOURCES:
        tree.write(n, f"new {n}\n")
    tree.write("delay", "0.3")
    os.remove(os.path.join(tree.at, "log"))
    errors = []

    def go():
        try:
            build.build_fused()
        except Exception as e:  # noqa: BLE001 - shown below
            errors.append(e)

    threads = [threading.Thread(target=go) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    lines = open(os.path.join(tree.at, "log")).read().split("\n")[:-1]
    assert sorted(x.split()[0] for x in lines) == sorted(ALL + ["link"])


@pytest.mark.parametrize("name", build.FUSED_SOURCES + build.FUSED_HEADERS)
def test_an_edit_of_any_source_makes_the_extension_stale(tree, name):
    class Loaded:
        source_sha = build.source_sha()

    fused._check_source(Loaded)
    tree.write(name, "edited\n", age=86400)
    with pytest.raises(RuntimeError, match="stale"):
        fused._check_source(Loaded)
    assert tree.build()[0] == (ALL if name in build.FUSED_HEADERS else [name])


def test_the_cached_build_of_a_vendored_copy(tree, tmp_path, monkeypatch):
    monkeypatch.setenv("DEVSPACE_OPS_CACHE", str(tmp_path / "cache"))
    out = build.ensure_fused_cached(verbose=False)
    assert build.source_sha() in open(out).read() and build.ensure_fused_cached(verbose=False) == out
    monkeypatch.setattr(build, "FUSED_FLAGS", build.FUSED_FLAGS + ["-g"])
    assert build.ensure_fused_cached(verbose=False) != out
    assert os.listdir(os.path.dirname(out)) == [os.path.basename(out)]
