"""Rules of requests and of rows where they meet other limits: tokens without a logit, biases that add up beyond f32, every place a number."""
import ctypes as C

import numpy as np
import pytest

import test_gpu_rules as plain
from gpu_util import cuda_backend
from onyxia_b200 import OnyxiaError, _ffi, ir
from onyxia_b200.engine import Engine
from onyxia_b200.ir import HostTensor

pytestmark = pytest.mark.gpu

VOCAB, MORE, WIDTH = 40, 9, 16


def engine(max_seqs=4):
    """Logits of `VOCAB` tokens, embeddings of `MORE` beyond them (places of a prompt that no answer has): each token's logits are those of its embedding alone."""
    r = np.random.default_rng(0)
    embed, head = r.standard_normal((VOCAB + MORE, WIDTH)).astype(np.float32), r.standard_normal((WIDTH, VOCAB)).astype(np.float32)
    b = ir.GraphBuilder()
    N, R, TW, W = b.sym("num_tokens"), b.sym("num_seqs"), b.sym("table_width"), b.sym("num_logits")
    ids = b.input("input_ids", ir.I64, [N])
    b.input("seq_info", ir.I32, [R, 4])
    b.input("page_table", ir.I32, [R, TW])
    rows = b.input("logit_rows", ir.I64, [W])
    const = lambda a: b.constant(HostTensor.from_numpy(a))  # noqa: E731
    b.output("logits", b.matmul(b.gather(b.gather(const(embed), ids, 0), rows, 0), const(head)))
    return Engine(cuda_backend().prepare(b.finish()), 256, max_seqs), (embed @ head).astype(np.float64)


def answer(e, request):
    out = []
    while e.stats()["waiting"] + e.stats()["running"]:
        out += [t for q, t, _ in e.step() if q == request]
    return out


def expected(logits, prompt, n, repetition=1.0, frequency=0.0, presence=0.0):
    said = []
    for _ in range(n):
        x = logits[(prompt + said)[-1]].copy()
        for t in set(prompt + said):
            if t < VOCAB:
                x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
        for t in set(said):
            x[t] -= said.count(t) * frequency + presence
        said.append(int(np.argmax(x)))
    return said


@pytest.mark.parametrize("rules", [dict(repetition=1.9), dict(frequency=3.0), dict(repetition=1.3, presence=2.0)], ids=str)
def test_tokens_of_a_prompt_that_have_no_logit_have_no_penalty(rules):
    e, logits = engine()
    prompt = [3, VOCAB, 7, VOCAB + MORE - 1, 7, VOCAB + 2]
    assert answer(e, e.submit(prompt, 8)) == expected(logits, prompt, 8)
    assert answer(e, e.submit(prompt, 8, **rules)) == expected(logits, prompt, 8, **rules) != expected(logits, prompt, 8)
    only = [VOCAB, VOCAB + 1]
    assert answer(e, e.submit(only, 8, **rules)) == expected(logits, only, 8, **rules)


def constrain(e, request, ids, values, n=None):
    ids, values = np.array(ids, np.int32), np.array(values, np.float32)
    at = lambda a, kind: a.ctypes.data_as(C.POINTER(kind)) if a.size else None  # noqa: E731
    _ffi.check(_ffi.cuda_lib().ox_engine_constrain(e._h, request, 1.0, 0.0, 0.0, at(ids, C.c_int32), at(values, C.c_float), len(ids) if n is None else n))


def test_biases_that_add_up():
    """A token may be listed more than once. What its biases add up to is a number, or minus infinity; minus infinity for all tokens is refused however it comes about."""
    e, logits = engine()
    big = float(np.finfo(np.float32).max)
    r = e.submit([3], 2)
    with pytest.raises(OnyxiaError, match="biases of token 5 add up"):
        constrain(e, r, [5, 7, 5], [big, 1.0, big])
    with pytest.raises(OnyxiaError, match="leave no token"):
        constrain(e, r, list(range(VOCAB)) * 2, [-big] * VOCAB * 2)
    constrain(e, r, list(range(VOCAB - 1)) * 2, [-big] * (VOCAB - 1) * 2)
    with pytest.raises(OnyxiaError, match="leave no token"):
        e.allow(r, [4, 5])
    assert answer(e, r) == [VOCAB - 1] * 2
    r = e.submit([3], 1)
    constrain(e, r, [5, 5, 5], [big, -big, 100.0])
    assert answer(e, r) == [5]


def test_biases_without_tokens_or_values_are_refused_at_the_c_entry():
    e, _ = engine()
    r = e.submit([3], 1)
    for ids, values, n in (([], [], 3), ([], [], -1), ([4], [], 1), ([], [1.0], 1)):
        with pytest.raises(OnyxiaError, match="without their tokens or values"):
            constrain(e, r, ids, values, n)
    constrain(e, r, [], [], 0)
    assert len(answer(e, r)) == 1


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 33), (5, 4097), (3, 50021), (64, 8192)])
def test_every_result_is_a_number_and_close(rows, vocab, dtype):
    """Every place where the plain implementation has a number, those under rules among them: no NaN hides there. Tolerance: that of test_gpu_rules.py."""
    r = np.random.default_rng(vocab)
    x = (4.0 * r.standard_normal((rows, vocab))).astype(dtype)
    b = ir.GraphBuilder()
    b.output("one", b.const_f32([1.0], [1]))
    session = cuda_backend().prepare(b.finish())
    for width, n_bias, n_masks in ((0, 0, 0), (40, 7, 0), (700, 300, 3), (30, 0, 2), (0, 20, 0)):
        more = plain.rules(rows, vocab, width, n_bias, n_masks, seed=rows)
        got = session.download(session.constrain_last(session.upload(HostTensor.from_numpy(x)), **{k: session.upload(HostTensor.from_numpy(v)) for k, v in more.items()})).numpy()
        want = plain.reference(x, **more)
        assert not np.isnan(got).any() and np.array_equal(np.isfinite(got), np.isfinite(want))
        there = np.isfinite(want)
        assert np.max(np.abs(got[there] - want[there]), initial=0.0) <= plain.TOL


def test_null_logits_and_rules_are_refused_at_the_c_entry():
    b = ir.GraphBuilder()
    b.output("one", b.const_f32([1.0], [1]))
    session, out = cuda_backend().prepare(b.finish()), C.c_void_p()
    x, rules = session.upload(HostTensor.from_numpy(np.ones((1, 8), np.float32))), _ffi.LogitRules()
    for logits, described in ((None, C.byref(rules)), (x.handle, None), (None, None)):
        with pytest.raises(OnyxiaError, match="rules need logits"):
            _ffi.check(_ffi.cuda_lib().ox_session_constrain_last(session._h, logits, described, C.byref(out)))
    assert (session.download(session.constrain_last(x)).numpy() == 1.0).all()


@pytest.mark.parametrize("rows,vocab,n_bias", [(3, 4096, 4096), (2, 50021, 4096), (1, 262144, 1000), (3, 33, 200), (2, 4100, 31), (2, 4100, 33)])
def test_biases_are_added_up_in_their_order(rows, vocab, n_bias):
    """Bit by bit as one after the other in f32, tokens listed many times, near each other and far apart among them, biases of very different sizes; a zero that has no bias keeps its sign."""
    r = np.random.default_rng(n_bias + vocab)
    x = np.where(r.random((rows, vocab)) < 0.2, np.float32(-0.0), r.standard_normal((rows, vocab))).astype(np.float32)
    few = r.integers(0, vocab, 5)
    ids = np.where(r.random((rows, n_bias)) < 0.4, few[r.integers(0, 5, (rows, n_bias))], r.integers(0, vocab, (rows, n_bias))).astype(np.int32)
    ids[r.random(ids.shape) < 0.1] = -1
    bias = (r.standard_normal(ids.shape) * 10.0 ** r.integers(-4, 5, ids.shape)).astype(np.float32)
    want = x.copy()
    for i in range(rows):
        sums = {}
        for t, b in zip(ids[i].tolist(), bias[i]):
            if t >= 0:
                sums[t] = np.float32(sums.get(t, np.float32(0.0)) + b)
        for t, s in sums.items():
            want[i, t] = np.float32(x[i, t] + s)
    b = ir.GraphBuilder()
    b.output("one", b.const_f32([1.0], [1]))
    session = cuda_backend().prepare(b.finish())
    up = lambda a: session.upload(HostTensor.from_numpy(a))  # noqa: E731
    got = session.download(session.constrain_last(up(x), bias_ids=up(ids), bias=up(bias))).numpy()
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32))
