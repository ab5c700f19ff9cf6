"""What ox_session_constrain_last refuses, asked without a device."""
import os
import shutil
import subprocess

import pytest

from onyxia_b200 import _ffi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = next((d for d in (os.environ.get("CUDA_HOME"), "/usr/local/cuda") if d and os.path.exists(os.path.join(d, "include", "cuda_runtime.h"))), None)

PROGRAM = r"""
#include "backend/rules.hpp"
#include <cstdio>
#include <functional>
using namespace oxrt;
struct Case { DTensor logits, history, lengths, penalties, bias_ids, bias, masks, mask_of; Rules r; };
static DTensor t(DType d, std::vector<int64_t> shape) {
    static BufferRef some(reinterpret_cast<DeviceBuffer*>(64), [](DeviceBuffer*) {});
    DTensor x;
    x.dtype = d, x.shape = std::move(shape), x.buf = some;
    return x;
}
static bool refused(std::function<void(Case&)> change) {
    Case c{t(DType::F32, {3, 100}), t(DType::I32, {3, 7}), t(DType::I32, {3, 2}), t(DType::F32, {3, 3}), t(DType::I32, {3, 5}), t(DType::F32, {3, 5}), t(DType::U32, {9, 4}), t(DType::I32, {3}), {}};
    c.r = Rules{&c.history, &c.lengths, &c.penalties, &c.bias_ids, &c.bias, &c.masks, &c.mask_of};
    change(c);
    try {
        check_rules(c.logits, c.r);
    } catch (const ox::Error&) {
        return true;
    }
    return false;
}
int main() {
    int at = 0, bad = 0;
    auto expect = [&](bool want, std::function<void(Case&)> change) {
        at++;
        if (refused(change) != want) std::printf("case %d\n", at), bad++;
    };
    expect(false, [](Case&) {});
    expect(false, [](Case& c) { c.logits.dtype = DType::F16; });
    expect(false, [](Case& c) { c.logits.shape = {3, 1, 100}; });
    expect(false, [](Case& c) { c.r = Rules{}; });
    expect(false, [](Case& c) { c.r.history = c.r.lengths = c.r.penalties = nullptr; });
    expect(false, [](Case& c) { c.r.bias_ids = c.r.bias = nullptr; });
    expect(false, [](Case& c) { c.r.masks = c.r.mask_of = nullptr; });
    expect(false, [](Case& c) { c.r.mask_of = nullptr, c.masks.shape = {3, 4}; });
    expect(false, [](Case& c) { c.history.shape = {3, 0}, c.bias_ids.shape = c.bias.shape = {3, 0}; });
    expect(false, [](Case& c) { c.logits.shape = {0, 100}, c.r = Rules{}; });
    expect(true, [](Case& c) { c.logits.dtype = DType::BF16; });
    expect(true, [](Case& c) { c.logits.dtype = DType::I32; });
    expect(true, [](Case& c) { c.logits.shape = {3, 0}; });
    expect(true, [](Case& c) { c.logits.shape = {}; });
    expect(true, [](Case& c) { c.logits.shape = {65536, 100}, c.r = Rules{}; });
    expect(true, [](Case& c) { c.logits.buf = nullptr; });
    expect(true, [](Case& c) { c.r.history = nullptr; });
    expect(true, [](Case& c) { c.r.lengths = nullptr; });
    expect(true, [](Case& c) { c.r.penalties = nullptr; });
    expect(true, [](Case& c) { c.r.bias = nullptr; });
    expect(true, [](Case& c) { c.r.bias_ids = nullptr; });
    expect(true, [](Case& c) { c.r.masks = nullptr; });
    expect(true, [](Case& c) { c.r.mask_of = nullptr; });  // nine masks for three rows
    expect(true, [](Case& c) { c.history.dtype = DType::I64; });
    expect(true, [](Case& c) { c.history.shape = {2, 7}; });
    expect(true, [](Case& c) { c.history.shape = {3}; });
    expect(true, [](Case& c) { c.lengths.shape = {3}; });
    expect(true, [](Case& c) { c.lengths.dtype = DType::U32; });
    expect(true, [](Case& c) { c.penalties.shape = {3, 2}; });
    expect(true, [](Case& c) { c.penalties.dtype = DType::F16; });
    expect(true, [](Case& c) { c.bias_ids.shape = {3, 4}; });
    expect(true, [](Case& c) { c.bias.shape = {3, 4}; });
    expect(true, [](Case& c) { c.bias.dtype = DType::F16; });
    expect(true, [](Case& c) { c.bias_ids.shape = c.bias.shape = {3, 4097}; });
    expect(true, [](Case& c) { c.masks.shape = {9, 3}; });
    expect(true, [](Case& c) { c.masks.dtype = DType::I32; });
    expect(true, [](Case& c) { c.mask_of.shape = {4}; });
    expect(true, [](Case& c) { c.mask_of.shape = {3, 1}; });
    expect(true, [](Case& c) { c.mask_of.buf = nullptr; });
    return bad;
}
"""


@pytest.mark.skipif(CUDA is None or shutil.which("g++") is None, reason="needs g++ and CUDA's headers")
def test_rules_that_do_not_fit_are_refused(tmp_path):
    source, program = tmp_path / "rules.cpp", tmp_path / "rules"
    source.write_text(PROGRAM)
    _ffi.cuda_lib()
    pkg = os.path.dirname(_ffi.cuda_path())
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "onyxia_b200", "csrc"), "-I", os.path.join(CUDA, "include"), str(source), "-o", str(program), "-L" + pkg, "-lonyxia_cuda",
                    "-lonyxia_ir", "-Wl,-rpath," + pkg], check=True)
    run = subprocess.run([str(program)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout
