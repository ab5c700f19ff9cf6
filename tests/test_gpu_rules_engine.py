"""A model with differential attention through the engine, and requests whose tokens are under rules: the whole against the plain implementation in 64 bits."""
import numpy as np
import pytest

import differential_model as model
import kipizen_ref as ref
import kipizen_util as util
from gpu_util import cuda_backend
from onyxia_b200 import OnyxiaError, checkpoint, ir, kipizen
from onyxia_b200.engine import Engine
from onyxia_b200.ir import HostTensor

pytestmark = pytest.mark.gpu

# as of the designs' own tests: f32 agrees to a few parts in a million, bf16 to the rounding of its activations
TOL = {ir.F32: 1e-5, ir.BF16: 3e-2}


def engine(dtype, max_tokens=2048, max_seqs=6):
    c, w = model.CONFIG, model.weights(model.CONFIG)
    stored = checkpoint.Weights.from_bf16({k: HostTensor.bf16(v).data.view(np.uint16).reshape(v.shape) for k, v in w.items()})
    return Engine(cuda_backend().prepare(kipizen.build(kipizen.KipizenConfig.from_dict(c), stored, dtype)), max_tokens, max_seqs), w


@pytest.fixture(autouse=True)
def plain_form(monkeypatch):
    monkeypatch.setattr(ref, "attention_mixer", model.mixer)


def tokens(n, seed):
    return np.random.default_rng(seed).integers(0, model.CONFIG["vocab"], n).tolist()


@pytest.mark.parametrize("dtype", [ir.F32, ir.BF16], ids=["f32", "bf16"])
def test_whole_prompts_portions_and_tokens(dtype):
    e, w = engine(dtype)
    a, b = tokens(150, 1), tokens(90, 2)
    want = [ref.forward(model.CONFIG, w, t) for t in (a, b)]

    def check(got, rows):
        assert np.sqrt(((got - rows) ** 2).mean()) <= TOL[dtype] * np.sqrt((rows ** 2).mean())

    got = e.forward([(0, a, list(range(150))), (1, b[:40], [39])])
    check(got[:150], want[0])
    check(got[150:], want[1][39:40])
    check(e.forward([(1, b[40:85], [0, 44])]), want[1][[40, 84]])
    e.release(0)
    e.forward([(2, a[:70], [])])
    for i in range(85, 90):  # single tokens beside a portion and beside each other
        check(e.forward([(1, b[i:i + 1], [0]), (2, a[i - 15:i - 14], [0])] if i > 85 else [(1, b[i:i + 1], [0]), (2, a[70:71], [0])]), np.stack([want[1][i], want[0][i - 15]]))


def under(logits, prompt, answer, repetition=1.0, frequency=0.0, presence=0.0, bias=None, allowed=None):
    x = logits.astype(np.float64).copy()
    for t in set(prompt + answer):
        x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
    for t in set(answer):
        x[t] -= answer.count(t) * frequency + presence
    for t, v in (bias or {}).items():
        x[t] += v
    if allowed is not None:
        x[[t for t in range(len(x)) if t not in allowed]] = -np.inf
    return x


def test_greedy_answers_under_rules():
    """Each request of a batch has rules of its own; a grammar changes with every token. The engine's tokens are those of the plain implementation, as long as its first two candidates are
    further apart than f32 is off (1e-3 of logits of a few units: never closer here)."""
    e, w = engine(ir.F32)
    prompts = [tokens(n, 10 + n) for n in (20, 70, 5, 33)]
    rules = [dict(repetition=1.8), dict(frequency=0.7, presence=0.4), dict(bias={7: 3.0, 8: 2.9, 100: -float("inf")}), dict(repetition=1.3, frequency=0.2, bias={3: 1.0})]
    grammar = lambda n: set(range(n % 5, 131, 5))  # noqa: E731
    ids = [e.submit(p, 12, **r) for p, r in zip(prompts, rules)]
    free = e.submit(prompts[0], 12)
    answers, plain = {i: [] for i in ids + [free]}, []
    while e.stats()["waiting"] + e.stats()["running"]:
        if len(answers[ids[3]]) < 12:
            e.allow(ids[3], sorted(grammar(len(answers[ids[3]]))))
        for request, token, _ in e.step(4096):
            answers[request].append(token)
    for k, (p, r) in enumerate(zip(prompts + [prompts[0]], rules + [{}])):
        got, said = answers[(ids + [free])[k]], []
        for n in range(12):
            x = under(ref.forward(model.CONFIG, w, p + said)[-1], p, said, allowed=grammar(n) if k == 3 else None, **r)
            first, second = np.argsort(-x, kind="stable")[:2]
            assert x[first] - x[second] > 1e-3
            said.append(int(first))
        assert got == said, k
        plain.append(said)
    assert plain[0] != plain[4]  # the rules did something


def test_sampled_answers_stay_in_the_grammar():
    e, _ = engine(ir.BF16)
    allowed = {2, 30, 64, 65, 130}
    ids = [e.submit(tokens(9, s), 20, temperature=1.5, seed=s) for s in range(4)]
    for i in ids[:3]:
        e.allow(i, sorted(allowed))
    mask = np.zeros(131, bool)
    mask[[130]] = True
    e.allow(ids[2], mask)
    e.allow(ids[1], [5])
    e.allow(ids[1], None)
    answers = {i: [] for i in ids}
    while e.stats()["waiting"] + e.stats()["running"]:
        for request, token, _ in e.step():
            answers[request].append(token)
    assert set(answers[ids[0]]) <= allowed and len(set(answers[ids[0]])) > 1
    assert set(answers[ids[2]]) == {130}
    assert not set(answers[ids[1]]) <= allowed and not set(answers[ids[3]]) <= allowed


def test_rules_that_mean_nothing_change_no_token():
    e, _ = engine(ir.BF16)
    prompts = [tokens(n, n) for n in (40, 3, 77)]
    plain = e.generate(prompts, 10)
    assert e.generate(prompts, 10, bias={5: 0.0}) == plain
    sampled = e.generate(prompts, 10, temperature=0.9, top_k=20, seed=3)
    assert e.generate(prompts, 10, temperature=0.9, top_k=20, seed=3, bias={5: 0.0}) == sampled


def test_rules_that_are_refused():
    e, _ = engine(ir.BF16)
    r = e.submit(tokens(5, 0), 3)
    for bad in (dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=float("nan")), dict(frequency=float("inf")), dict(presence=float("nan")), dict(bias={131: 1.0}),
                dict(bias={3: float("nan")}), dict(bias={3: float("inf")})):
        with pytest.raises(OnyxiaError):
            e.constrain(r, **bad)
        waiting = e.stats()["waiting"]
        with pytest.raises(OnyxiaError):
            e.submit(tokens(5, 0), 3, **bad)
        assert e.stats()["waiting"] == waiting
    with pytest.raises(ValueError):
        e.constrain(r, bias={-1: 1.0})
    for bad in ([], [131], [-1], np.zeros(131, bool), np.ones(130, bool)):
        with pytest.raises((OnyxiaError, ValueError)):
            e.allow(r, bad)
    with pytest.raises(OnyxiaError, match="no unfinished request"):
        e.allow(r + 1, [3])
    # biases and a mask that together leave nothing
    bar = {t: -float("inf") for t in range(131)}
    with pytest.raises(OnyxiaError, match="leave no token"):
        e.constrain(r, bias=bar)
    e.constrain(r, bias={t: -float("inf") for t in range(130)})
    for bad in ([5], [5, 129]):
        with pytest.raises(OnyxiaError, match="leave no token"):
            e.allow(r, bad)
    e.allow(r, [5, 130])
    with pytest.raises(OnyxiaError, match="leave no token"):
        e.constrain(r, bias={5: -float("inf"), 130: -float("inf")})
    word = np.ones(5, np.uint32)
    from onyxia_b200 import _ffi
    import ctypes
    assert _ffi.cuda_lib().ox_engine_allow(e._h, r, word.ctypes.data_as(ctypes.POINTER(ctypes.c_uint32)), 0) != 0
    answer = []
    while len(answer) < 3:
        answer += [t for q, t, _ in e.step() if q == r]
    assert answer == [130] * 3
    assert len(e.generate([tokens(4, 1)], 3)[0]) == 3  # and the engine goes on
    with pytest.raises(OnyxiaError, match="no unfinished request"):
        e.constrain(r, repetition=1.1)
