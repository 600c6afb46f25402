"""The prompt kernel's order of workgroups (spindle_amd/csrc/kv4_order.h), compiled for the host: every
row tile meets every key head exactly once."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = """
#include "kv4_order.h"
extern "C" void places(int jobs, int n_kv, int *at) {
  for (int i = 0; i < jobs * n_kv; i++) {
    const spx::RowsPlace p = spx::rows_place(i, jobs * n_kv, n_kv);
    at[i] = p.job < 0 || p.job >= jobs || p.head < 0 || p.head >= n_kv ? -1 : p.job * n_kv + p.head;
  }
}
"""


@pytest.fixture(scope="module")
def places(tmp_path_factory):
    d = tmp_path_factory.mktemp("order")
    (d / "order.cpp").write_text(SOURCE)
    so = str(d / "order.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I", os.path.join(ROOT, "spindle_amd", "csrc"), str(d / "order.cpp"), "-o", so], check=True)
    f = C.CDLL(so).places

    def run(jobs, n_kv):
        at = np.empty(jobs * n_kv, np.int32)
        f(jobs, n_kv, at.ctypes.data_as(C.c_void_p))
        return at
    return run


@pytest.mark.parametrize("n_kv", list(range(1, 65)) + [96, 100, 255, 256, 257, 1000, 1024])
def test_every_tile_and_head_once(places, n_kv):
    for jobs in list(range(1, 400 if n_kv <= 64 else 40)) + [451, 577, 833, 999, 1000]:
        at = places(jobs, n_kv)
        assert at.min() >= 0 and (np.bincount(at, minlength=jobs * n_kv) == 1).all(), jobs


def test_heavy_tiles_first(places):
    """The last tiles, whose rows see the most, are the first workgroups'; the second turn rises."""
    at = places(129, 4) // 4
    assert (at[:256] == 128 - np.arange(256) // 4).all() and (at[256:512] == 1 + np.arange(256) // 4).all() and (at[512:] == 0).all()
    at = places(193, 3) // 3
    assert (at[:255] == 192 - np.arange(255) // 3).all() and (at[255:510] == 23 + np.arange(255) // 3).all()
