"""Host-side parts of the serving-step operators, compiled into small host programs: the keys
that pages are chosen by."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from conftest import PKG

CSRC = os.path.join(PKG, "csrc")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")
pytestmark = pytest.mark.skipif(
    shutil.which("g++") is None or not os.path.exists(os.path.join(CUDA, "include")),
    reason="needs g++ and the CUDA headers")


def host_library(tmp_path, source, *flags):
    src, out = tmp_path / "host.cpp", tmp_path / "host.so"
    src.write_text(source)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-shared", "-fPIC", "-pthread",
                    f"-I{CSRC}", f"-I{CUDA}/include", *flags, "-o", str(out), str(src)], check=True)
    return ctypes.CDLL(str(out))


# --------------------------------------------------------------------------- the pages' keys
@pytest.fixture
def page_key(tmp_path):
    lib = host_library(tmp_path, '''
        #include "page_key.h"
        extern "C" unsigned key(float best, float sc) { return fe::step::page_key(best, sc); }
        extern "C" unsigned forced() { return fe::step::kForced; }''')
    lib.key.argtypes, lib.key.restype = [ctypes.c_float] * 2, ctypes.c_uint
    lib.forced.restype = ctypes.c_uint
    return lib


def floats(*bits):
    return [float(x) for x in np.array(bits, np.uint32).view(np.float32)]


def test_no_score_has_the_key_of_an_always_chosen_page(page_key):
    """More always-chosen keys than pages are kept would be listed past the list's end."""
    inf = float("inf")
    scales = [0.0, -0.0, 1.0, -1.0, inf, -inf, 2.0 ** -120, 2.0 ** 122] + floats(
        0x7fffffff, 0xffffffff, 0x7fc00000, 0xffc00000, 0x7f800001, 0xff800001)  # NaN
    sums = [0.0, -0.0, 1.0, -1.0, 2.0 ** 24, -2.0 ** 24, inf, -inf, 3e38, -3e38]
    for sc in scales:
        for best in sums:
            k = page_key.key(best, sc)
            assert 0 < k < page_key.forced(), (best, sc, hex(k))


def test_keys_are_in_the_order_of_the_scores(page_key):
    inf, nan = float("inf"), float("nan")
    scores = [-inf, -3e38, -1.5, -1.0, -1e-45, 0.0, 1e-45, 1.0, 1.5, 3e38, inf]
    keys = [page_key.key(x, 1.0) for x in scores]
    assert keys == sorted(set(keys))
    assert page_key.key(-0.0, 1.0) == page_key.key(0.0, 1.0)
    for sc, best in ((inf, -5.0), (inf, 0.0), (nan, 1.0), (nan, -1.0), (-inf, 0.0), (0.0, inf)):
        assert page_key.key(best, sc) == keys[-1], (sc, best)
