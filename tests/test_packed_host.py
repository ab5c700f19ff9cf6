"""Which forms of the composites over keys and values in 4 bits the backend takes, asked of its registry without a device, and the format as the tests write it out."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

import packed_util as util
from packed_util import Form
from onyxia_b200 import _ffi, ir

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = next((d for d in (os.environ.get("CUDA_HOME"), "/usr/local/cuda") if d and os.path.exists(os.path.join(d, "include", "cuda_runtime.h"))), None)

PROGRAM = r"""
#include "backend/runtime.hpp"
#include "ir/module_api.hpp"
extern "C" int taken(ox_module* h) {
    const ox::Module& m = h->b.module();
    int n = 0;
    for (auto& node : m.nodes)
        if (!node.is_prim) n += oxrt::standard_kernels().get(node.composite.name)->accepts(m, node);
    return n;
}
extern "C" int early(ox_module* h) {
    const ox::Module& m = h->b.module();
    int n = 0;
    for (auto& node : m.nodes)
        if (!node.is_prim) n += oxrt::may_begin_early(*oxrt::standard_kernels().get(node.composite.name), m, node);
    return n;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if CUDA is None or shutil.which("g++") is None:
        pytest.skip("needs g++ and CUDA's headers")
    d = tmp_path_factory.mktemp("takes")
    (d / "takes.cpp").write_text(PROGRAM)
    _ffi.cuda_lib()
    pkg = os.path.dirname(_ffi.cuda_path())
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "onyxia_b200", "csrc"), "-I", os.path.join(ROOT, "include"), "-I", os.path.join(CUDA, "include"),
                    str(d / "takes.cpp"), "-o", str(d / "takes.so"), "-L" + pkg, "-lonyxia_cuda", "-lonyxia_ir", "-Wl,-rpath," + pkg], check=True)
    lib = C.CDLL(str(d / "takes.so"))
    for fn in (lib.taken, lib.early):
        fn.argtypes, fn.restype = [C.c_void_p], C.c_int
    return lib


@pytest.fixture(scope="module")
def taken(lib):
    def asked(f, dtype=ir.BF16, kind="attend", **changed):
        m = util.module(f, dtype, kind, **changed)
        return lib.taken(m.handle)

    return asked


KINDS = {"attend": 1, "shared": 1, "write": 1, "read": 1, "chain": 3}


def test_forms_that_are_taken(taken):
    for f in (Form(4, 2, 64, 128, 64), Form(1, 1, 16, 16), Form(6, 3, 48, 80, 8, page=16, window=5, softcap=2.0, norm=1, sink=1, factors=1), Form(18, 2, 272, 512, 272, gap=5)):
        for dtype in (ir.F32, ir.BF16):
            for kind, nodes in KINDS.items():
                assert taken(f, dtype, kind) == nodes


def test_what_the_run_makes_is_waited_for(lib):
    """Pools that another node of the step updates are operands of the run; batch descriptions, tables and factors are there before it."""
    for kind, nodes in KINDS.items():
        m = util.module(Form(4, 2, 64, 128, 64, factors=1), ir.BF16, kind)
        assert lib.early(m.handle) == nodes


F = Form(4, 2, 64, 128, 64)
EVERY = [
    {"kv_heads": 0}, {"kv_heads": 4}, {"dim": 32}, {"dim": 0}, {"dim": -64}, {"vdim": 64}, {"factors": 1}, {"factors": 2}, {"page_table": (ir.I64, [3, 4])}, {"page_table": (ir.I32, [3])},
    {"pages.keys": (ir.U8, [9, 2, 64, 64])}, {"pages.keys": (ir.I8, [9, 2, 64, 36])}, {"pages.keys": (ir.BF16, [9, 2, 64, 36])}, {"pages.keys": (ir.U8, [9, 2, 48, 36])},
    {"pages.keys": (ir.U8, [9, 4, 64, 36])}, {"pages.keys": (ir.U8, [9, 2, 32, 36])}, {"pages.values": (ir.U8, [9, 2, 64, 36])}, {"pages.values": (ir.U8, [8, 2, 64, 72])},
    {"pages.values": (ir.U8, [8, 2, 64])}, {"out": (ir.F16, [9, 512])}, {"out": (ir.BF16, [9, 256])}, {"out": (ir.BF16, [9])}]
BATCHED = [
    {"rot_dims": 63}, {"rot_dims": 66}, {"rot_dims": -2}, {"k_offset": 10 ** 6}, {"k_offset": -1}, {"v_offset": 10 ** 6}, {"epsilon": -1e-6}, {"epsilon": float("nan")}, {"operands": 5},
    {"turns": np.zeros((2, 16))}, {"turns": np.zeros((1, 32))}, {"seq_info": (ir.I64, [3, 4])}, {"seq_info": (ir.I32, [3, 3])}, {"page_table": (ir.I32, [5, 4])},
    {"proj": (ir.F16, [9, F.width])}, {"proj": (ir.BF16, [9, F.width - 1])}, {"proj": (ir.BF16, [F.width])}, {"updated": (ir.U8, [9, 2, 64, 37])}]
ATTENDING = [
    {"heads": 3}, {"heads": 0}, {"heads": -4}, {"q_offset": -1}, {"q_offset": 2 ** 62}, {"window": -1}, {"window": 2 ** 31}, {"scale": float("nan")}, {"softcap": -1.0}, {"softcap": float("nan")},
    {"scale": 1e31}, {"softcap": 1e31}, {"softcap": 1e-31}, {"scale": float("inf")}, {"proj": (ir.F32, [9, F.width])}]


def label(c):
    return " ".join(f"{k}={v.shape if hasattr(v, 'shape') else v}" for k, v in c.items())


@pytest.mark.parametrize("kind,changed", [("read", c) for c in EVERY + [{"places": (ir.I64, [9, 2])}, {"places": (ir.I32, [9, 3])}, {"places": (ir.I32, [9])}, {"operands": 3}]] +
                         [("write", c) for c in EVERY[:-3] + BATCHED] + [("attend", c) for c in EVERY + BATCHED + ATTENDING], ids=lambda c: c if isinstance(c, str) else label(c))
def test_forms_that_are_refused(taken, kind, changed):
    assert taken(F, kind=kind, **changed) == 0


@pytest.mark.parametrize("kind", ["attend", "shared", "write", "read"])
def test_sizes_and_factors_that_are_refused(taken, kind):
    for f in (Form(1, 1, 24, 16), Form(1, 1, 16, 40), Form(1, 1, 8208, 16), Form(1, 1, 16, 8208), Form(512, 512, 4096, 4112), Form(4, 2, 64, 64, page=8), Form(1, 1, 16, 2048, page=1 << 20), Form(1, 1, 16, 16, page=1 << 21), Form(4, 2, 64, 64, page=1)):
        assert taken(f, kind=kind) == 0
    f = Form(4, 2, 64, 64, factors=1)
    for bad in (0.0, -1.0, np.inf, np.nan, 1e-31, 1e31):
        for pair in ([[1.0, bad], [1.0, 1.0]], [[1.0, 1.0], [bad, 1.0]]):
            assert taken(f, kind=kind, factor_values=pair) == 0
    assert taken(f, kind=kind, factor_values=[[1.0, 2.0, 3.0], [1.0, 1.0]]) == 0 and taken(f, kind=kind, factor_values=[[1e-30, 1e30], [1.0, 1.0]]) == 1


# ── the format as the tests have it ──
def test_the_nearest_code_and_of_two_the_even_one():
    one = lambda *x: util.packed(np.array([[list(x) + [0.0] * (16 - len(x))]], np.float32), [1.0])  # noqa: E731
    # a largest magnitude of 6 has the scale 1: halfway between two codes is the even one's
    codes, scales = one(6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0, 0.26, 4.99, 5.01, -0.0)
    assert util.scale_values(scales).tolist() == [[[1.0]]]
    assert codes[0, 0, :14].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 0, 14, 1, 6, 7, 0]
    # scales: the largest, the least, what is too small for one
    assert one(2688.0)[1].item() == one(1e30)[1].item() == one(np.inf)[1].item() == 126 and one(6 * 2.0 ** -9)[1].item() == 1
    codes, scales = one(6 * 2.0 ** -10, -1e-9)
    assert scales.item() == 0 and not codes.any()  # halfway to the least: even
    codes, scales = one(1.0, np.nan, 3.0)
    assert scales.item() == 127 and np.isnan(util.valued(codes, scales, [1.0])).all()


def test_values_come_back_within_half_a_step():
    x = np.random.default_rng(0).standard_normal((50, 3, 64)).astype(np.float32) * np.exp(np.random.default_rng(1).uniform(-2, 2, (50, 3, 1))).astype(np.float32)
    factor = np.array([0.5, 1.0, 3.0], np.float32)
    codes, scales = util.packed(x, factor)
    back = util.valued(codes, scales, factor)
    # a scale is off by 2^-4 of itself at most and the largest value by that and what saturates; codes by half of the widest step, 1 of 6
    top = np.abs(x.reshape(50, 3, 4, 16)).max(-1)
    assert (np.abs(back - x).reshape(50, 3, 4, 16).max(-1) <= top * (1 / 6 + 2 ** -4) * (1 + 2 ** -4)).all()
    pool = util.bytes_of(codes[None].transpose(0, 2, 1, 3)[:, :, :32], scales[None].transpose(0, 2, 1, 3)[:, :, :32])
    assert pool.shape == (1, 3, 32, 36)
    for a, b in zip(util.parts_of(pool), (codes, scales)):
        assert np.array_equal(a[0], b.transpose(1, 0, 2)[:, :32])
