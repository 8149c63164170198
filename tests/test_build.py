"""The build's command line, without compiling."""
import os
import runpy
import subprocess
import sys

import pytest

from trips_amd import build


@pytest.mark.parametrize("torch_there", [True, False])
def test_the_library_is_built_without_torch(torch_there, monkeypatch, capsys):
    """A program of the C ABI needs hipcc alone; what links libtorch is left out where there is none."""
    calls = []
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, **kw: calls.append(cmd))

    class Done:
        def __init__(self, cmd, **kw):
            calls.append(cmd)

        def wait(self):
            return 0

        returncode = 0
    monkeypatch.setattr(subprocess, "Popen", Done)
    monkeypatch.setattr(sys, "argv", ["build.py"])
    if not torch_there:
        monkeypatch.setitem(sys.modules, "torch", None)  # (import torch raises)
    runpy.run_path(build.__file__, run_name="__main__")
    text = " ".join(" ".join(c) for c in calls)
    assert "libtrips_splat.so" in text and ("_trips_host.so" in text) == torch_there
    out = capsys.readouterr().out
    assert os.path.basename(build.LIB) in out and ("no torch" in out) != torch_there
