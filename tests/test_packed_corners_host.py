"""What keys and values in 4 bits refuse beside what test_packed_host.py has, asked of the backend's registry without a device, and the quotients that their kernels take by a product."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

import packed_util as util
from packed_util import Form
from onyxia_b200 import ir
from onyxia_b200.ir import HostTensor
from test_packed_host import ROOT, lib  # noqa: F401  (a fixture)


@pytest.fixture
def with_attrs(monkeypatch):
    """Modules whose composites have more attributes."""
    def build(f, dtype, kind, **more):
        class Builder(ir.GraphBuilder):
            def composite(self, name, attrs, *rest):
                return super().composite(name, {**attrs, **(more if name != "onyxia.CacheRead" else {})}, *rest)

        with monkeypatch.context() as m:
            m.setattr(ir, "GraphBuilder", Builder)
            return util.module(f, dtype, kind)

    return build


@pytest.mark.parametrize("dtype", [ir.F32, ir.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", ["attend", "shared", "write"])
@pytest.mark.parametrize("name", ["interleaved", "gate", "sinks", "temps", "talk"])
def test_attributes_that_only_the_whole_cache_has(lib, with_attrs, name, kind, dtype):  # noqa: F811
    """Pairs side by side, gates, learned sinks, temperatures and mixed heads are not left out without a word."""
    f = Form(4, 2, 64, 128, 64)
    for value, nodes in ((0, 1), (1, 0), (2, 0)):
        m = with_attrs(f, dtype, kind, **{name: value, "gate_offset": 3})
        assert lib.taken(m.handle) == nodes


QUOTIENT = r"""
#include "kernels/quotient.hpp"
// 0 where there is none
extern "C" unsigned by_of(int64_t d, int64_t most) {
    try {
        return oxk::by_of(d, most);
    } catch (const std::exception&) {
        return 0;
    }
}
"""


def test_quotients_by_a_product(tmp_path):
    """Every divisor up to 2^18 (the blocks of 16 dimensions that a place may have) for as many as the kernels divide, and at the ends of what it serves."""
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    (tmp_path / "q.cpp").write_text(QUOTIENT)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "onyxia_b200", "csrc"), str(tmp_path / "q.cpp"), "-o", str(tmp_path / "q.so")], check=True)
    by_of = C.CDLL(str(tmp_path / "q.so")).by_of
    by_of.argtypes, by_of.restype = [C.c_int64, C.c_int64], C.c_uint
    assert by_of(1, 2 ** 31 - 1) == 0
    for d in [*range(2, 2 ** 18 + 1, 7), *range(65530, 65600), 80000, 131070, 153600, 2 ** 17, 2 ** 18]:
        for most in (d - 1, 2048, 2 ** 19):
            by = by_of(d, most)
            # the ends of the last multiples of the divisor, where the product is first too large, and of the first ones
            n = np.concatenate([np.arange(0, 3) * d + d - 1, (most + 1) // d * d - 1 - np.arange(0, 3) * d, [most]])
            n = n[(n >= 0) & (n <= most)].astype(np.uint64)
            right = bool(((n * np.uint64(-(-2 ** 32 // d))) >> np.uint64(32) == n // np.uint64(d)).all())
            assert by == (-(-2 ** 32 // d) if by else 0) and (right or not by), (d, most)
    # what every call of a kernel divides is served
    assert all(by_of(d, most) for d, most in ((512, 2 ** 18), (1024, 2 ** 19), (65535, 65535), (2048, 2048), (16, 1024)))
    # one place of this many blocks is not: the reading kernel has one place per block of threads there, and divides nothing
    assert by_of(65537, 65536) == by_of(80000, 79999) == by_of(153600, 153599) == 0


@pytest.mark.parametrize("kind,computed,early", [(k, c, e) for k in ("attend", "shared", "write") for c, e in (("", 1), ("reshaped", 1), ("seq_info", 0), ("page_table", 0), ("turns", 0))] +
                         [("read", "", 1), ("read", "reshaped", 1), ("read", "page_table", 0)])
def test_what_the_module_computes_is_waited_for(lib, monkeypatch, kind, computed, early):  # noqa: F811
    """Single tokens look at the batch description, the page table and the angles before the launches in front of theirs have ended: only where nothing of the run makes them."""
    class Builder(ir.GraphBuilder):
        def input(self, name, dtype, shape):
            if name == computed:
                return self.cast(super().input(name, ir.I64, shape), ir.I32)
            if name == "page_table" and computed == "reshaped":
                return self.reshape(super().input(name, dtype, [shape[0], 1, shape[1]]), shape)
            return super().input(name, dtype, shape)

        def constant(self, tensor):
            a = tensor.numpy()
            if computed != "turns" or a.shape != (2, 32):
                return super().constant(tensor)
            half = [super(Builder, self).constant(HostTensor.from_numpy(a / 2)) for _ in range(2)]
            return self.add(*half)

    with monkeypatch.context() as m:
        m.setattr(ir, "GraphBuilder", Builder)
        module = util.module(Form(4, 2, 64, 128, 64, factors=1), ir.BF16, kind)
    assert lib.taken(module.handle) == 1 and lib.early(module.handle) == early
