"""Building on first use: processes that start together build a stale file once, one after another."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import os, sys, time
sys.path.insert(0, sys.argv[1])
import build as _build
from framework import loader
folder, what = sys.argv[2:]
done, log = os.path.join(folder, "done"), os.path.join(folder, "log")
_build.BUILD = folder

def stale(*a):
    return not os.path.exists(done)

def compile_slowly(*a, **k):
    with open(log, "a") as f:
        f.write("begin\\n")
    time.sleep(0.5)
    with open(log, "a") as f:
        f.write("end\\n")
    open(done, "w").close()

open(os.path.join(folder, "ready-%d" % os.getpid()), "w").close()
while sum(n.startswith("ready") for n in os.listdir(folder)) < 3:
    time.sleep(0.01)
_build.NVCC = os.environ["CXX"] = sys.executable  # a compiler that is there
if what == "library":
    _build.stale, _build.build = stale, compile_slowly
    loader.ctypes.CDLL = lambda path: path
    loader.load_kernel("nothing")
else:
    _build.binding_stale, _build.build_binding = stale, compile_slowly
    loader.load_kernel = lambda name: None
    try:
        loader.load_torch_binding()
    except ImportError:
        pass  # there is no module to import here
"""


@pytest.mark.parametrize("what", ["library", "binding"])
def test_processes_that_start_together_build_once(what, tmp_path):
    pkg = os.path.join(ROOT, "nl2cuda-kernel-agent_b200")
    script = tmp_path / "child.py"
    script.write_text(CHILD)
    folder = tmp_path / "build"
    folder.mkdir()
    runs = [subprocess.Popen([sys.executable, str(script), pkg, str(folder), what]) for _ in range(3)]
    assert [r.wait(timeout=300) for r in runs] == [0, 0, 0]
    assert (folder / "log").read_text().split() == ["begin", "end"]
