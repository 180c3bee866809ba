"""Which sort the lookup gradient takes, counted in launches on stand-ins for
the HIP runtime: one for few tokens of a large table, as far as that is the
faster, three a pass beyond."""

import os
import subprocess
import sys

import pytest

from conftest import ROOT

COUNT = """
#include <stdint.h>
typedef struct { uint32_t x, y, z; } Dim;
int launches;
/* a launch starts here; what is not 0 says not to make it */
int __hipPushCallConfiguration(Dim g, Dim b, uint64_t l, void *s) {
  return ++launches, (void)l, (void)s, g.x && b.x ? 1 : 2;
}
"""

PROBE = """
import ctypes, sys
from ns_fps_amd import capi
lib, n = capi.Lib(), ctypes.c_int.in_dll(ctypes.CDLL(None), "launches")
tokens, rows = int(sys.argv[1]), int(sys.argv[2])
A = 0x10000
args = capi.EmbedArgs(tokens=tokens, rows=rows, width=8, scale=1.0, table_stride=8, out_stride=8,
                      d_table=A, d_tokens=A, d_out=A, workspace=A, workspace_bytes=1 << 40)
lib.embed_grad_device(args)
print(n.value)
"""


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("fake")
    (tmp / "count.c").write_text(COUNT)
    libs = []
    for src in (str(tmp / "count.c"), os.path.join(ROOT, "tests", "fake_hip.c")):
        libs.append(str(tmp / os.path.basename(src)) + ".so")
        subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-Wall", src, "-o", libs[-1]], check=True)
    env = dict(os.environ,
               LD_PRELOAD=":".join(filter(None, [*libs, os.environ.get("LD_PRELOAD")])))

    def run(tokens, rows):
        p = subprocess.run([sys.executable, "-c", PROBE, str(tokens), str(rows)], cwd=ROOT, env=env,
                           check=True, stdout=subprocess.PIPE, text=True)
        return int(p.stdout)
    return run


# and the starts, the rows, the crowded rows' pieces and sums
@pytest.mark.parametrize("tokens,rows,sorts", [
    (100, 40000, 1), (512, 40000, 1), (513, 40000, 6), (1024, 40000, 6), (512, 1 << 20, 1),
    (513, 1 << 20, 9)])
def test_launches_of_a_sort(launches, tokens, rows, sorts):
    assert launches(tokens, rows) == sorts + 4


def test_one_pass_over_whole_keys_gives_the_starts_too(launches):
    assert launches(1000, 8192) == 3 + 3
