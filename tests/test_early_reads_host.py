"""Kernels that look at a batch before the launches in front of them have ended, asked of the backend's registry without a device: they do so only where nothing of what they look at is made by the run itself."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

import differential_model
import kipizen_util
import lovuzen_util
import mufevik_util
import zusitar_util
from differential_computed import module as computed_module
from differential_util import Form
from onyxia_b200 import _ffi, checkpoint, ir, kipizen, lovuzen, mufevik, zusitar

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = next((d for d in (os.environ.get("CUDA_HOME"), "/usr/local/cuda") if d and os.path.exists(os.path.join(d, "include", "cuda_runtime.h"))), None)

PROGRAM = r"""
#include "backend/runtime.hpp"
#include "ir/module_api.hpp"
// how many nodes of the name (null: of any kernel that looks at a batch) may begin early, or may not
extern "C" int count(ox_module* h, const char* name, int early) {
    const ox::Module& m = h->b.module();
    int found = 0;
    for (auto& n : m.nodes) {
        if (n.is_prim || (name && n.composite.name != name)) continue;
        const oxrt::FusedKernel* k = oxrt::standard_kernels().get(n.composite.name);
        if (k && !k->of_run.empty()) found += oxrt::may_begin_early(*k, m, n) == (early != 0);
    }
    return found;
}
"""


@pytest.fixture(scope="module")
def count(tmp_path_factory):
    if CUDA is None or shutil.which("g++") is None:
        pytest.skip("needs g++ and CUDA's headers")
    d = tmp_path_factory.mktemp("early")
    (d / "early.cpp").write_text(PROGRAM)
    _ffi.cuda_lib()
    pkg = os.path.dirname(_ffi.cuda_path())
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "onyxia_b200", "csrc"), "-I", os.path.join(ROOT, "include"), "-I", os.path.join(CUDA, "include"),
                    str(d / "early.cpp"), "-o", str(d / "early.so"), "-L" + pkg, "-lonyxia_cuda", "-lonyxia_ir", "-Wl,-rpath," + pkg], check=True)
    fn = C.CDLL(str(d / "early.so")).count
    fn.argtypes, fn.restype = [C.c_void_p, C.c_char_p, C.c_int], C.c_int
    return lambda m, early, name=None: fn(m.handle, name.encode() if name else None, early)


@pytest.mark.parametrize("maps,name", [(1, "onyxia.PagedKVAttention"), (2, "onyxia.DifferentialAttention")])
def test_what_the_module_computes_is_waited_for(count, maps, name):
    f = Form(4, 2, 64, 128, 64)
    for computed, early in (((), 1), (("reshaped",), 1), (("seq_info",), 0), (("page_table",), 0), (("turns",), 0), (("seq_info", "page_table"), 0)):
        m = computed_module(f, ir.BF16, np.zeros(4), np.zeros(128), computed, maps)
        assert count(m, early, name) == 1 and count(m, 1 - early, name) == 0, computed


def test_every_batched_kernel_of_every_design_begins_early(count):
    """Their batch descriptions, tables and weights are inputs and constants."""
    for design, util, config in ((kipizen, kipizen_util, kipizen.KipizenConfig), (lovuzen, lovuzen_util, lovuzen.LovuzenConfig), (mufevik, mufevik_util, mufevik.MufevikConfig),
                                 (zusitar, zusitar_util, zusitar.ZusitarConfig)):
        for name in util.CONFIGS:
            c, w = util.model(name)
            m = design.build(config.from_dict(c), checkpoint.Weights.from_f32(w))
            assert count(m, 0) == 0 and count(m, 1) >= len(c["layers"]) // 2, (design.__name__, name)
    c = differential_model.CONFIG
    m = kipizen.build(kipizen.KipizenConfig.from_dict(c), checkpoint.Weights.from_f32(differential_model.weights(c)))
    assert count(m, 0) == 0 and count(m, 1, "onyxia.DifferentialAttention") == 2
