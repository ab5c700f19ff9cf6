"""CTAs of differential prompts that share an SM, reckoned without a device: whoever holds tensor memory waits for a neighbour, so all that are there together have to find some."""
import ctypes as C
import itertools
import os
import shutil
import subprocess

import pytest

from onyxia_b200 import _ffi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = next((d for d in (os.environ.get("CUDA_HOME"), "/usr/local/cuda") if d and os.path.exists(os.path.join(d, "include", "cuda_runtime.h"))), None)
SM_BYTES, SYSTEM_BYTES, SM_COLUMNS = 228 * 1024, 1024, 512

PROGRAM = r"""
#include "kernels/kernels.hpp"
extern "C" int bytes_of(int kp, int vp) { return oxk::differential_prefill_smem(kp, vp); }
extern "C" int columns_of(int kp, int vp) { return oxk::differential_prefill_columns(kp, vp); }
"""


@pytest.fixture(scope="module")
def sizes(tmp_path_factory):
    if CUDA is None or shutil.which("g++") is None:
        pytest.skip("needs g++ and CUDA's headers")
    d = tmp_path_factory.mktemp("places")
    (d / "places.cpp").write_text(PROGRAM)
    _ffi.cuda_lib()
    pkg = os.path.dirname(_ffi.cuda_path())
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "onyxia_b200", "csrc"), "-I", os.path.join(ROOT, "include"), "-I", os.path.join(CUDA, "include"),
                    str(d / "places.cpp"), "-o", str(d / "places.so"), "-L" + pkg, "-lonyxia_cuda", "-lonyxia_ir", "-Wl,-rpath," + pkg], check=True)
    lib = C.CDLL(str(d / "places.so"))
    return {(kp, vp): (lib.bytes_of(kp, vp), lib.columns_of(kp, vp)) for kp in (1, 2) for vp in (1, 2, 3, 4)}


def test_any_that_fit_beside_each_other_have_tensor_memory(sizes):
    """Sizes of maps (up to 64 or 128 dimensions) and values (up to 64, 128, 192 or 256) of sessions of their own, two and three at a time."""
    assert all(cols in (256, 512) and b <= 227 * 1024 for b, cols in sizes.values())
    for n in (2, 3):
        for who in itertools.combinations_with_replacement(sizes, n):
            if sum(sizes[w][0] + SYSTEM_BYTES for w in who) <= SM_BYTES:
                assert sum(sizes[w][1] for w in who) <= SM_COLUMNS, who


def test_what_is_left_beside_two_holds_no_kernel_of_more_columns(sizes):
    """A kernel of single CTAs that waits for more columns than are left beside two CTAs of a pair's form would keep a third from its share: the smallest of them (a product's, with more than
    256 columns: two stages of 128 weight rows and 128 activation rows of 64 k in two planes) takes 64 KB."""
    least = min(b for b, cols in sizes.values() if cols <= 256)
    assert SM_BYTES - 2 * (least + SYSTEM_BYTES) - SYSTEM_BYTES < 64 * 1024


def test_the_memory_of_a_cta_holds_its_parts(sizes):
    """Queries in two parts (128 rows), tiles of keys and halves of values on their way, barriers, factors, and what threads of a row tell each other."""
    for (kp, vp), (b, cols) in sizes.items():
        keys, stages = (64, 3) if cols == 256 else (128, 2)
        assert (kp, vp) in ((1, 1), (1, 2)) or keys == 128
        assert b >= 1024 + 2 * kp * 128 * 128 + stages * (kp * keys * 128 + vp * 64 * 128) + 23 * 8 + 8 + 256 + 4 * 128 * 4
