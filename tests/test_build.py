"""The build entry point: what it runs on every call, with the compiler replaced by a record of the commands (CPU)."""
import glob
import os

import pytest


@pytest.fixture
def commands(monkeypatch):
    import __graft_entry__ as g
    seen = []

    class Done:
        def __init__(self, cmd, **_):
            seen.append(cmd)

        def wait(self):
            return 0
    from infinite_texture_gans_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        g.build()
    monkeypatch.setattr(g.subprocess, "Popen", Done)
    monkeypatch.setattr(g.subprocess, "check_call", lambda cmd, **_: seen.append(cmd))
    return g, seen


@pytest.mark.parametrize("args", [{}, {"force": False}, {"force": True}])
def test_every_source_is_compiled_on_every_call(commands, args):
    """``force``, as callers have passed it, is still taken: every call compiles every file whatever it says"""
    g, seen = commands
    g.build(**args)
    sources = sorted(glob.glob(os.path.join(g.CSRC, "*.hip")))
    assert len(sources) >= 12 and sorted(c[c.index("-c") + 1] for c in seen[:-1]) == sources
    assert "-shared" in seen[-1] and g.LIB in seen[-1] and all(g._obj(s) in seen[-1] for s in sources)


def test_packed_fp32_instructions_stay_off(commands):
    g, seen = commands
    g.build()
    for cmd in seen[:-1]:
        at = cmd.index("-packed-fp32-ops")
        assert cmd[at - 3:at] == ["-Xclang", "-target-feature", "-Xclang"], cmd
