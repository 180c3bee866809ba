"""nsfps_init_device prepares what a sampling call needs, and no more: the
kernels it loads are those that a process's first sampling call loads.  The
library runs on stand-ins for the HIP runtime; a second one counts the kernels
that are asked for."""

import os
import subprocess
import sys

import pytest

from conftest import ROOT

COUNT = """
int loads;
int hipFuncGetAttributes(void *a, const void *f) { return ++loads, !a || !f; }
"""

PROBE = """
import ctypes, sys
import numpy as np
from ns_fps_amd.capi import Lib, NsfpsError
lib, loads = Lib(), ctypes.c_int.in_dll(ctypes.CDLL(None), "loads")
if sys.argv[1] == "sample":
    try:
        lib.fps(np.random.RandomState(1).uniform(-1, 1, (500, 3)).astype(np.float32), 60,
                (-1.0, 1.0, -1.0, 1.0, -1.0, 1.0, 8, 8, 8))
    except NsfpsError:
        pass  # no kernel has run
else:
    getattr(lib, sys.argv[1])()
print(loads.value)
"""


@pytest.fixture(scope="module")
def loaded(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("fake")
    (tmp / "count.c").write_text(COUNT)
    libs = []
    for src in (str(tmp / "count.c"), os.path.join(ROOT, "tests", "fake_hip.c")):
        libs.append(str(tmp / os.path.basename(src)) + ".so")
        subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-Wall", src, "-o", libs[-1]], check=True)
    env = dict(os.environ,
               LD_PRELOAD=":".join(filter(None, [*libs, os.environ.get("LD_PRELOAD")])))

    def run(what):
        p = subprocess.run([sys.executable, "-c", PROBE, what], cwd=ROOT, env=env, check=True,
                           stdout=subprocess.PIPE, text=True)
        return int(p.stdout)
    return run


def test_preparing_loads_what_the_first_sampling_call_loads(loaded):
    assert loaded("init_device") == loaded("sample") > 0


def test_the_sequence_operators_have_their_own(loaded):
    assert loaded("init_sequence_device") > 0
