"""Which forms of onyxia.DifferentialAttention the backend takes, asked of its registry without a device."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

import differential_util as util
from differential_util import Form
from onyxia_b200 import _ffi, ir

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = next((d for d in (os.environ.get("CUDA_HOME"), "/usr/local/cuda") if d and os.path.exists(os.path.join(d, "include", "cuda_runtime.h"))), None)

PROGRAM = r"""
#include "backend/runtime.hpp"
#include "ir/module_api.hpp"
extern "C" int takes(ox_module* h) {
    const ox::Module& m = h->b.module();
    for (auto& n : m.nodes)
        if (!n.is_prim) return oxrt::standard_kernels().get(n.composite.name)->accepts(m, n);
    return -1;
}
"""


@pytest.fixture(scope="module")
def takes(tmp_path_factory):
    if CUDA is None or shutil.which("g++") is None:
        pytest.skip("needs g++ and CUDA's headers")
    d = tmp_path_factory.mktemp("takes")
    (d / "takes.cpp").write_text(PROGRAM)
    _ffi.cuda_lib()
    pkg = os.path.dirname(_ffi.cuda_path())
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "onyxia_b200", "csrc"), "-I", os.path.join(ROOT, "include"), "-I", os.path.join(CUDA, "include"),
                    str(d / "takes.cpp"), "-o", str(d / "takes.so"), "-L" + pkg, "-lonyxia_cuda", "-lonyxia_ir", "-Wl,-rpath," + pkg], check=True)
    fn = C.CDLL(str(d / "takes.so")).takes
    fn.argtypes, fn.restype = [C.c_void_p], C.c_int

    def asked(f, dtype=ir.BF16, **changed):
        m = util.module(f, dtype, changed.pop("lam", np.zeros(f.heads)), changed.pop("gain", np.zeros(f.vdim)), **changed)
        return fn(m.handle)

    return asked


def test_forms_that_are_taken(takes):
    for f in (Form(4, 2, 64, 128, 64), Form(1, 1, 1, 1), Form(6, 3, 24, 40, 8, page=1, window=5, softcap=2.0, norm=1, sink=1), Form(4, 2, 64, 128, 64, head_norm=0)):
        for dtype in (ir.F32, ir.BF16):
            assert takes(f, dtype) == 1


F = Form(4, 2, 64, 128, 64)


@pytest.mark.parametrize("changed", [
    {"heads": 3}, {"heads": 0}, {"heads": -4}, {"kv_heads": 0}, {"kv_heads": 4}, {"dim": 32}, {"dim": 0}, {"vdim": 64}, {"rot_dims": 63}, {"rot_dims": 66}, {"rot_dims": -2},
    {"window": -1}, {"window": 2 ** 31}, {"q_offset": -1}, {"q_offset": 2 ** 62}, {"k_offset": 10 ** 6}, {"v_offset": 10 ** 6}, {"scale": float("nan")}, {"softcap": -1.0},
    {"softcap": float("nan")}, {"epsilon": -1e-6}, {"head_epsilon": float("inf")}, {"operands": 7}, {"lam": np.zeros(2)}, {"gain": np.zeros(64)}, {"turns": np.zeros((2, 16))},
    {"turns": np.zeros((1, 32))}, {"seq_info": (ir.I64, [3, 4])}, {"seq_info": (ir.I32, [3, 3])}, {"page_table": (ir.I64, [3, 4])}, {"page_table": (ir.I32, [5, 4])},
    {"page_table": (ir.I32, [3])}, {"proj": (ir.F16, [9, F.width])}, {"proj": (ir.F32, [9, F.width])}, {"proj": (ir.BF16, [9, F.width - 1])}, {"proj": (ir.BF16, [F.width])},
    {"pages.keys": (ir.BF16, [9, 2, 64, 64])}, {"pages.keys": (ir.F32, [9, 2, 64, 128])}, {"pages.keys": (ir.BF16, [9, 2, 48, 128])}, {"pages.keys": (ir.BF16, [9, 4, 64, 128])},
    {"pages.keys": (ir.BF16, [9, 2, 32, 128])}, {"pages.values": (ir.BF16, [9, 2, 64, 64])}, {"pages.values": (ir.BF16, [8, 2, 64])}, {"out": (ir.F32, [9, 512])},
    {"out": (ir.BF16, [9, 256])}], ids=lambda c: " ".join(f"{k}={v.shape if hasattr(v, 'shape') else v}" for k, v in c.items()))
def test_forms_that_are_refused(takes, changed):
    assert takes(F, **changed) == 0


def test_sizes_above_what_a_block_holds_are_refused(takes):
    assert takes(Form(1, 1, 8193, 8)) == 0 and takes(Form(1, 1, 8, 8200)) == 0 and takes(Form(65536, 1, 1, 1)) == 0


@pytest.mark.parametrize("changed", [{"scale": 1e31}, {"scale": -1e31}, {"softcap": 1e31}, {"softcap": 1e-31}, {"scale": float("inf")}], ids=str)
def test_factors_that_f32_cannot_hold_are_refused(takes, changed):
    assert takes(F, **changed) == 0
    assert takes(F, scale=1e-30, softcap=1e-30) == 1 and takes(F, scale=-1e30) == 1
