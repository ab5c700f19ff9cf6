"""A model whose keys and values are held in 4 bits through the engine, the single-sequence loop and the command line: the whole against the plain implementation in 64 bits.

Tolerances. What is stored depends on which side of a border a value lies. In f32 keys and values are off the plain ones by some 1e-6 of themselves, so that of about 100 000 stored ones less than one is
expected on the other side; rows that see it are off by what an element in 32 that changes by a third does to them (5e-2 at most), all others by 1e-5. In bf16 they are off by 2^-9 for each of a few
roundings, some hundredth part: about three in a hundred change by a quarter, 4 % of the root mean square, which moves scores of a spread of 1.1 by 0.05 and results by as much, in each of three layers: 0.15.
"""
import functools
import json
import os
import subprocess
import sys

import numpy as np
import pytest

import kipizen_ref as ref
import packed_model as model
from gpu_util import cuda_backend
from kipizen_util import to_bf16
from onyxia_b200 import checkpoint, ir, kipizen, llm
from onyxia_b200.engine import Engine
from onyxia_b200.ir import HostTensor

pytestmark = pytest.mark.gpu


def stored():
    return checkpoint.Weights.from_bf16({k: HostTensor.bf16(v).data.view(np.uint16).reshape(v.shape) for k, v in model.weights(model.CONFIG).items()})


def engine(dtype, max_tokens=2048, max_seqs=6):
    return Engine(cuda_backend().prepare(kipizen.build(kipizen.KipizenConfig.from_dict(model.CONFIG), stored(), dtype)), max_tokens, max_seqs)


@pytest.fixture
def plain(monkeypatch):
    def forward(dtype, tokens):
        round_to = to_bf16 if dtype == ir.BF16 else lambda a: np.asarray(a, np.float32)
        monkeypatch.setattr(ref, "attention_mixer", functools.partial(model.mixer, round_to=round_to))
        return ref.forward(model.CONFIG, model.weights(model.CONFIG), tokens)

    return forward


def tokens(n, seed):
    return np.random.default_rng(seed).integers(0, model.CONFIG["vocab"], n).tolist()


def compare(dtype, got, want):
    off = np.sqrt(((got - want) ** 2).mean(1) / (want ** 2).mean())
    if dtype == ir.F32:
        assert np.quantile(off, 0.9) <= 1e-5 and off.max() <= 5e-2
    else:
        assert np.sqrt((off ** 2).mean()) <= 0.15


@pytest.mark.parametrize("dtype", [ir.F32, ir.BF16], ids=["f32", "bf16"])
def test_whole_prompts_portions_and_tokens(dtype, plain):
    e = engine(dtype)
    a, b = tokens(150, 1), tokens(90, 2)
    want = [plain(dtype, t) for t in (a, b)]
    got = e.forward([(0, a, list(range(150))), (1, b[:40], [39])])
    compare(dtype, got[:150], want[0])
    compare(dtype, got[150:], want[1][39:40])
    compare(dtype, e.forward([(1, b[40:85], [0, 44])]), want[1][[40, 84]])
    e.release(0)
    e.forward([(2, a[:70], [])])
    rows, plain_rows = [], []
    for i in range(85, 90):  # single tokens beside a portion and beside each other
        rows.append(e.forward([(1, b[i:i + 1], [0]), (2, a[i - 15:i - 14], [0])]))
        plain_rows.append(np.stack([want[1][i], want[0][i - 15]]))
    compare(dtype, np.concatenate(rows), np.concatenate(plain_rows))


def test_greedy_answers(plain):
    """The engine's tokens are those of the plain implementation as long as its first two candidates are further apart than a changed code moves them (5e-2 of logits of a few units)."""
    e = engine(ir.F32)
    prompts = [tokens(n, 10 + n) for n in (20, 70, 5)]
    ids = [e.submit(p, 8) for p in prompts]
    answers = {i: [] for i in ids}
    while e.stats()["waiting"] + e.stats()["running"]:
        for request, token, _ in e.step(4096):
            answers[request].append(token)
    for i, p in zip(ids, prompts):
        logits = plain(ir.F32, p + answers[i])
        for t, token in enumerate(answers[i]):
            row = logits[len(p) - 1 + t]
            assert row[token] >= row.max() - 0.05 * np.sqrt((row ** 2).mean())
        assert len(answers[i]) == 8


def test_pools_are_a_third_of_what_they_were():
    """4.5 bits a value instead of 16, for the layers that have keys of their own."""
    def held(c):
        m = kipizen.build(kipizen.KipizenConfig.from_dict(c), checkpoint.Weights.from_bf16({k: HostTensor.bf16(v).data.view(np.uint16).reshape(v.shape) for k, v in model.weights(c).items()}), ir.BF16)
        session = cuda_backend().prepare(m)
        before = session.resident_bytes()
        e = Engine(session, 65536, 1)
        return session.resident_bytes() - before, e

    c = json.loads(json.dumps(model.CONFIG))
    packed = held(c)[0]
    for l in c["layers"]:
        l["mixer"].pop("cache", None)
    whole = held(c)[0]
    values = 65536 * (2 * (32 + 64) + 1 * (64 + 128))
    assert whole - packed == values * 16 // 8 - values * 9 // 16


def test_single_sequence_loop_and_command_line(tmp_path):
    """Both give the engine's tokens."""
    prompt = tokens(30, 4)
    want = engine(ir.F32).generate([prompt], 6)[0]
    loop = llm.NativeLlmSession(cuda_backend(), kipizen.build(kipizen.KipizenConfig.from_dict(model.CONFIG), stored(), ir.F32), 256)
    assert loop.generate(prompt, 6) == want
    with open(tmp_path / "config.json", "w") as f:
        json.dump(model.CONFIG, f)
    checkpoint.write_safetensors(str(tmp_path / "model.safetensors"), stored())
    r = subprocess.run([sys.executable, "-m", "onyxia_b200", "generate", "--model", str(tmp_path), "--dtype", "float32", "--prompt", " ".join(map(str, prompt)), "-n", "6"],
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert [int(t) for t in r.stdout.split()] == want
