"""When `fluidnet_amd.build` compiles again, with compilers that only touch their outputs."""
import os
import subprocess

import pytest

from fluidnet_amd import build as b


@pytest.fixture
def compiled(tmp_path, monkeypatch):
    """Runs build() on empty sources in a folder of its own; the commands of each call."""
    src, lib = tmp_path / "csrc", tmp_path / "lib"
    src.mkdir()
    for name in b.SOURCES + ["torch_ops.cpp", "one.h", "abi.h"]:
        (src / name).write_text("")
        os.utime(src / name, (1000, 1000))
    script = tmp_path / "build.py"
    script.write_text("")
    os.utime(script, (1000, 1000))
    for name, value in dict(CSRC=str(src), LIBDIR=str(lib), LIB=str(lib / "lib.so"), HEADERS=[str(src / "one.h"), str(src / "abi.h")],
                            TORCH_OPS_SRC=str(src / "torch_ops.cpp"), TORCH_OPS=str(lib / "ops.so"), __file__=str(script)).items():
        monkeypatch.setattr(b, name, value)
    now = [2000]

    def run(cmd, **kw):
        out = cmd[cmd.index("-o") + 1]
        open(out, "w").close()
        os.utime(out, (now[0], now[0]))
        commands.append(cmd)
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(b.subprocess, "run", run)
    commands = []

    def call(touch=None, **kw):
        commands.clear()
        now[0] += 100
        if touch:
            at = script if touch == "build.py" else src / touch
            os.utime(at, (now[0] - 50, now[0] - 50))
        b.build(verbose=False, **kw)
        return [os.path.basename(c[c.index("-o") + 1]) for c in commands]
    call.everything = sorted([s.replace(".hip", ".o") for s in b.SOURCES] + ["torch_ops.o", "lib.so", "ops.so"])
    return call


def test_only_what_changed(compiled):
    assert sorted(compiled()) == compiled.everything
    assert compiled() == []
    assert sorted(compiled(touch="fnet_optim.hip")) == ["fnet_optim.o", "lib.so", "ops.so"]
    assert sorted(compiled(touch="torch_ops.cpp")) == ["lib.so", "ops.so", "torch_ops.o"]
    assert "torch_ops.o" not in compiled(touch="one.h")
    assert sorted(compiled(touch="abi.h")) == compiled.everything
    assert sorted(compiled(force=True)) == compiled.everything


def test_other_flags_are_a_change(compiled):
    """The flags stand in build.py: objects that an older one built are not linked with new ones (as those with packed fp32 instructions were,
    in a tree that had been built before the flag that forbids them)."""
    compiled()
    assert sorted(compiled(touch="build.py")) == compiled.everything
    assert compiled() == []


def test_the_entry_point_compiles_every_time(monkeypatch):
    import __graft_entry__ as entry
    asked = []

    def fake(force=False, verbose=True):
        asked.append(force)
        return b.LIB
    monkeypatch.setattr(b, "build", fake)
    entry.build()
    assert asked == [True]
