"""What the attention over pages works out on the host as on the device: which blocks of a tile's keys a wave has to do with."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from conftest import ROOT
from test_kernel_waits import PKG

SOURCE = """
#include "kv_attn.h"
extern "C" void blocks(int has_rows, int last0, int last1, int *out) {
    const WaveBlocks b = wave_blocks(has_rows, last0, last1);
    out[0] = b.whole, out[1] = b.any;
}
"""


@pytest.fixture(scope="module")
def blocks(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    d = tmp_path_factory.mktemp("tiles")
    (d / "t.hip").write_text(SOURCE)
    subprocess.run([hipcc, "-O1", "-std=c++17", "-fPIC", "-shared", "--cuda-host-only", "--offload-arch=gfx950", "-w",
                    f"-I{ROOT}/include", f"-I{PKG}/csrc", str(d / "t.hip"), "-o", str(d / "t.so")], check=True, capture_output=True)
    fn = C.CDLL(str(d / "t.so")).blocks

    def of(*args):
        out = (C.c_int * 2)()
        fn(*args, out)
        return out[0], out[1]

    return of


@pytest.mark.parametrize("group", [1, 2, 3, 16])
@pytest.mark.parametrize("past,n", [(0, 20), (0, 200), (31, 17), (32, 48), (1000, 21), (5003, 50), (0, 1)])
def test_a_wave_has_the_blocks_that_its_rows_see(blocks, past, n, group):
    """of each wave of each wide tile (32 of its 128 rows, heads of a group next to each other), by the definition; a wave behind
    the read's last row has none, though the tile has blocks"""
    rows, without = n * group, 0
    for r0 in range(0, -(-rows // 128) * 128, 32):
        mine = range(r0, min(r0 + 32, rows))
        last = [past + r // group for r in mine]  # the last key that each row sees
        whole = min(((k + 1) // 32 for k in last), default=0)
        some = max((k // 32 + 1 for k in last), default=0)
        key = lambda r: past + min(r, rows - 1) // group  # noqa: E731  (as the kernel has it: of a row that is there)
        assert blocks(r0 < rows, key(r0), key(r0 + 31)) == (whole, some)
        without += not mine
    assert without == -rows % 128 // 32


def test_no_keys_and_the_last_that_are_counted(blocks):
    assert blocks(1, -1, -1) == (0, 0) and blocks(0, -1, -1) == (0, 0)
    top = 2 ** 31 - 17
    assert blocks(1, top, top) == ((top + 1) // 32, top // 32 + 1) and blocks(0, top, top) == (0, 0)
