"""The binding without its extension module: every function through ctypes, and a build
that goes on where the module cannot be compiled. Needs no GPU."""
import importlib
import os
import subprocess
import sys
import sysconfig

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

WITHOUT = """
import importlib, sys
sys.modules["resonance-net_b200._calls"] = None  # as where it was not built
rnet = importlib.import_module("resonance-net_b200")
args = (4096, 0, 64, 8192, None, -1, 12288, 16384, 20480, None, 0, 4, 64, None)
rnet.call("rnet_beam_select", *args)  # no sequences: nothing to do
assert rnet._quick is None
try:
    rnet.call("rnet_beam_select", None, *args[1:])
except rnet.RnetError as e:
    assert "null pointer" in str(e)
else:
    raise SystemExit("not refused")
"""


def test_the_library_loads_without_the_module():
    r = subprocess.run([sys.executable, "-c", WITHOUT], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.fixture
def build(tmp_path, monkeypatch):
    b = importlib.import_module("resonance-net_b200.build")
    monkeypatch.setattr(b, "CALLS", str(tmp_path / os.path.basename(b.CALLS)))
    return b


def test_the_module_is_named_for_its_interpreter(build):
    assert os.path.basename(build.CALLS) == "_calls" + sysconfig.get_config_var("EXT_SUFFIX")


@pytest.mark.parametrize("missing", ["headers", "compiler"])
def test_a_build_goes_on_without_it(build, monkeypatch, capsys, missing):
    with open(build.CALLS, "w") as f:
        f.write("of other headers")
    os.utime(build.CALLS, (1, 1))

    def run(cmd, **kw):
        if missing == "compiler":
            raise FileNotFoundError("g++")
        return subprocess.CompletedProcess(cmd, 1, "", "Python.h: No such file or directory")

    monkeypatch.setattr(build.subprocess, "run", run)
    build._build_calls(2.0)
    assert not os.path.exists(build.CALLS)  # its calls may not fit the library any more
    assert "_calls" in capsys.readouterr().err
