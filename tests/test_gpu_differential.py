"""Differential attention on the device against the formulas in 64 bits (differential_util.py): prompts, single tokens and both beside each other, head layouts,
page sizes, windows, capped scores, sinks, odd sizes, rows of no sequence, bad pages.

Tolerances. f32: a score is a sum of `dim` products, each rounded to 2^-24 relative to sums of the order of the score's spread (some units), its exponential to a few 2^-24; a difference of
two maps with λ ≤ 0.8 loses at most a factor of ten of that: 1e-5 in the root mean square of a row. bf16: queries, keys, weights and results are each rounded once to 2^-9 relative (root
mean square 2^-9 / sqrt 3 = 1.1e-3). Queries and keys: scores are off by 1.1e-3 · sqrt 2 · their spread (1.5 here), weights by as much, which a difference of maps amplifies by
sqrt(1 + λ²) / sqrt(1 + λ²) where they are independent and up to (1 + λ) / (1 − λ) = 9 where a row sees a few keys: rows 3e-2, all rows together 1e-2. With a factor of the scores other than dim^-1/2 their
spread is 1.5 · factor · dim^1/2 and what the rounding of queries and keys does to the weights grows with it: both bounds are times the ratio of the factors (16 for a factor of 2 over
64 dimensions: scores of a spread of 24 are off by 1.1e-3 · sqrt 2 · 24 = 3.7e-2).
"""
import dataclasses

import numpy as np
import pytest

import differential_util as util
from differential_util import Form
from gpu_util import cuda_backend
from kipizen_util import to_bf16
from onyxia_b200 import OnyxiaError, ir
from onyxia_b200 import backend as be
from onyxia_b200.ir import HostTensor

pytestmark = pytest.mark.gpu

DTYPES = {"f32": ir.F32, "bf16": ir.BF16}
ROW = {"f32": 1e-5, "bf16": 3e-2}
ALL = {"f32": 3e-6, "bf16": 1e-2}


def act(kind):
    return HostTensor.bf16 if kind == "bf16" else lambda a: HostTensor.from_numpy(np.asarray(a, np.float32))


def stored(kind):
    return to_bf16 if kind == "bf16" else lambda a: np.asarray(a, np.float32)


def rows_of(s):
    return np.concatenate([np.arange(r, r + n) for r, n, _, _ in s.seqs] + [np.zeros(0, np.int64)]).astype(np.int64)


def compare(got, want, kind, s, spread=1.0):
    live = rows_of(s)
    got, want = got[live].astype(np.float64), want[live]
    assert np.isfinite(got).all()
    scale, more = np.sqrt((want ** 2).mean()), max(1.0, spread) if kind == "bf16" else 1.0
    err = np.sqrt(((got - want) ** 2).mean(1)) / scale
    whole, worst = float(np.sqrt((err ** 2).mean())), float(err.max())
    assert whole <= ALL[kind] * more and worst <= ROW[kind] * more


def run(f, s, kind, backend=None):
    session = (backend or cuda_backend()).prepare(util.module(f, DTYPES[kind], s.lam, s.gain))
    dev = {k: session.upload(v) for k, v in util.feed(s, act(kind)).items()}
    return session, dev, {n: t for n, t in session.run(dev)}


def check(f, lengths, kind, seed=0, **more):
    s = util.step(f, lengths, seed, round_to=stored(kind), **more)
    session, _, outs = run(f, s, kind)
    got = {n: session.download(t).numpy() for n, t in outs.items()}
    want, keys, values = util.reference(f, s, stored(kind))
    compare(got["out"], want, kind, s, f.scale * f.dim ** 0.5)
    # what is no new key or value is as it was, NaN too; new keys are off by a rounding of the stored type (f32 angles: 1e-6)
    assert np.array_equal(got["updated.pages.values"], values.astype(np.float32), equal_nan=True)
    k = got["updated.pages.keys"].astype(np.float64)
    assert np.array_equal(np.isnan(k), np.isnan(keys))
    assert np.nanmax(np.abs(k - keys) / np.maximum(np.abs(keys), 0.1)) <= (2 ** -7 if kind == "bf16" else 1e-5)
    return s, got


LAYOUTS = [Form(4, 1, 128, 256, 128), Form(16, 4, 64, 128, 64), Form(6, 2, 32, 64, 16), Form(5, 5, 48, 48, 48), Form(3, 1, 80, 160, 40), Form(20, 2, 64, 64, 0),
           Form(2, 1, 24, 40, 8), Form(3, 3, 20, 36, 6), Form(9, 1, 16, 32, 16), Form(1, 1, 7, 5, 4), Form(2, 2, 136, 264, 8), Form(8, 8, 112, 224, 112, gap=8), Form(4, 2, 64, 128, 32, gap=3)]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("f", LAYOUTS, ids=lambda f: f"{f.heads}x{f.kv_heads}x{f.dim}x{f.vdim}")
def test_layouts(f, kind):
    check(f, [(70, 0)], kind)
    check(f, [(1, 90), (1, 0), (1, 63), (1, 64)], kind, seed=1)
    check(f, [(3, 40), (1, 129), (66, 0), (1, 5), (65, 62)], kind, seed=2)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("page", [1, 4, 8, 16, 32, 128, 256])
def test_page_sizes(page, kind):
    f = Form(4, 2, 32, 64, 32, page=page)
    check(f, [(1, 70), (37, 3), (1, 300), (130, 65)], kind)
    check(f, [(1, 70), (1, 255), (1, 0)], kind, seed=1)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("more", [dict(window=1), dict(window=17), dict(window=64), dict(window=100, sink=1), dict(softcap=5.0), dict(sink=1), dict(norm=1), dict(head_norm=0),
                                  dict(softcap=20.0, sink=1, norm=1, window=90, head_norm=0), dict(scale=2.0)], ids=str)
def test_scores(more, kind):
    f = Form(4, 2, 64, 128, 64, **more)
    check(f, [(150, 0), (1, 200), (20, 130), (1, 0), (1, 64)], kind)
    check(f, [(1, 200), (1, 1), (1, 500)], kind, seed=1)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_long_ranges(kind):
    f = Form(8, 2, 64, 128, 64)
    check(f, [(1, 3000), (1, 1), (1, 4095)], kind)
    check(f, [(300, 900), (1, 2000)], kind, seed=1)
    check(Form(4, 1, 128, 256, 128), [(1, 2500)], kind, seed=2)
    check(Form(4, 1, 128, 256, 128, window=200), [(70, 1000), (1, 1500)], kind, seed=3)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_and_sequences_of_a_padded_batch(kind):
    """Rows behind the last sequence are left alone, and sequences without new tokens (behind all others) do nothing, to the pools neither."""
    f = Form(4, 2, 64, 128, 64)
    for lengths, tail in (([(5, 3), (1, 70), (0, 10)], 9), ([(1, 3), (1, 70), (0, 10), (0, 0)], 1), ([(80, 0)], 70), ([(0, 5)], 3), ([(1, 70)], 4)):
        s, got = check(f, lengths, kind, tail=tail) if any(n for n, _ in lengths) else (None, None)
        s = s or util.step(f, lengths, tail=tail, round_to=stored(kind))
        session = cuda_backend().prepare(util.module(f, DTYPES[kind], s.lam, s.gain))
        dev = {k: session.upload(v) for k, v in util.feed(s, act(kind)).items()}
        for name, t in session.run(dev):
            session.download(t)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_keys_that_stand_out_and_keys_that_are_far_away(kind):
    """One key takes nearly all weight of a map; scores of hundreds; scores that are all equal."""
    f = Form(4, 2, 64, 128, 0, scale=1.0)
    s = util.step(f, [(70, 20), (1, 130)], 5, round_to=stored(kind), spread=8.0)
    session, _, outs = run(f, s, kind)
    got = session.download(outs["out"]).numpy()
    want = util.reference(f, s, stored(kind))[0]
    # scores of hundreds in bf16: the stored operands are exact here (no rotation), so the products are, but for their sums
    live = rows_of(s)
    err = np.sqrt(((got[live] - want[live]) ** 2).mean(1)) / np.sqrt((want[live] ** 2).mean())
    assert np.isfinite(got[live]).all() and np.median(err) <= ALL[kind] and err.max() <= (2e-4 if kind == "f32" else 3e-2)
    s.proj[:, :f.offsets[1]] = 0.0  # every visible key weighs the same in both maps
    session, _, outs = run(f, s, kind)
    compare(session.download(outs["out"]).numpy(), util.reference(f, s, stored(kind))[0], kind, s)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_the_same_bits_again_and_from_captured_steps(kind):
    """Runs of one plan (the second and later ones replay a graph), and of a backend that launches one by one, are the same bits."""
    f = Form(8, 2, 64, 128, 64)
    for lengths in ([(1, 3000), (1, 100)], [(200, 700), (1, 900), (33, 0)]):
        s = util.step(f, lengths, 3, round_to=stored(kind))
        session, dev, outs = run(f, s, kind)
        first = session.download(outs["out"]).numpy()[rows_of(s)]
        for _ in range(4):
            assert np.array_equal(session.download(session.run(dev)[0][1]).numpy()[rows_of(s)], first)
        plain = be.CudaBackend((0,), disable_graphs=True)
        session, _, outs = run(f, s, kind, plain)
        assert np.array_equal(session.download(outs["out"]).numpy()[rows_of(s)], first)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [-1, 99, 2 ** 31 - 1])
@pytest.mark.parametrize("lengths", [[(1, 200)], [(90, 60)], [(1, 200), (70, 3)]], ids=str)
def test_a_page_that_is_none_is_reported(lengths, bad, kind):
    f = Form(4, 2, 64, 128, 64)
    s = util.step(f, lengths, round_to=stored(kind))
    s.table[0, 1] = bad
    s.keys[np.isnan(s.keys)] = 0.0
    s.values[np.isnan(s.values)] = 0.0
    session = cuda_backend().prepare(util.module(f, DTYPES[kind], s.lam, s.gain))
    dev = {k: session.upload(v) for k, v in util.feed(s, act(kind)).items()}
    outs = session.run(dev)
    with pytest.raises(OnyxiaError, match="out of range"):
        session.download(outs[0][1])
    # the session goes on with a good table
    s.table[0, 1] = s.table[0, 0]
    dev["page_table"] = session.upload(HostTensor.from_numpy(s.table))
    session.download(session.run(dev)[0][1])


def test_a_prompt_in_a_batch_of_no_more_rows_than_sequences_is_reported():
    f = Form(4, 2, 64, 128, 64)
    s = util.step(f, [(1, 3), (3, 5), (0, 0), (0, 0)])
    session, _, outs = run(f, s, "bf16")
    with pytest.raises(OnyxiaError, match="sequence 1 has 3 new tokens"):
        session.download(outs["out"])


def test_nothing_to_do_and_nowhere_to_put_it():
    f = Form(4, 2, 64, 128, 64)
    s = util.step(f, [(2, 3)])
    session = cuda_backend().prepare(util.module(f, ir.BF16, s.lam, s.gain))
    dev = {k: session.upload(v) for k, v in util.feed(s, act("bf16")).items()}
    none = dict(dev, proj=session.upload(HostTensor.bf16(s.proj[:0])))
    assert session.run(none)[0][1].shape == (0, f.heads * f.vdim)
    none = dict(dev, seq_info=session.upload(HostTensor.from_numpy(s.seqs[:0])), page_table=session.upload(HostTensor.from_numpy(s.table[:0])))
    assert session.run(none)[0][1].shape == (2, f.heads * f.vdim)
    none = {**dev, "pages.keys": session.upload(HostTensor.bf16(s.keys[:0])), "pages.values": session.upload(HostTensor.bf16(s.values[:0]))}
    with pytest.raises(OnyxiaError, match="without a page"):
        session.run(none)
    want = util.reference(f, s)[0]
    compare(session.download(session.run(dev)[0][1]).numpy(), want, "bf16", s)


def test_views_and_uploads_of_device_memory():
    torch = pytest.importorskip("torch")
    f = Form(4, 2, 64, 128, 64)
    s = util.step(f, [(1, 90), (40, 20)])
    session, dev, outs = run(f, s, "bf16")
    want = session.download(outs["out"]).numpy()
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            x = torch.from_numpy(s.proj).cuda().bfloat16()
            dev["proj"] = session.upload_device(ir.BF16, x.shape, x.data_ptr(), stream.cuda_stream)
            x.zero_()  # behind the copy
            out = session.run(dev)[0][1]
            got = torch.as_tensor(session.view(out, stream.cuda_stream), device="cuda").view(torch.bfloat16)
            assert got.data_ptr() == torch.as_tensor(session.view(out), device="cuda").data_ptr()
            del out  # the view holds the memory
            again = session.run(dev)[0][1]
            assert np.array_equal(got.float().cpu().numpy(), want) and np.array_equal(session.download(again).numpy(), want)
            got.zero_()
            del got
            assert np.array_equal(session.download(session.run(dev)[0][1]).numpy(), want)  # whatever buffer it got
    host = np.zeros(16, np.float32)
    with pytest.raises(OnyxiaError, match="not memory of the session's device"):
        session.upload_device(ir.F32, (16,), host.ctypes.data)
    empty = session.upload_device(ir.F32, (0, 3), 0)
    assert empty.shape == (0, 3) and torch.as_tensor(session.view(empty), device="cuda").shape == (0, 3)
    with pytest.raises(ValueError, match="4-bit"):
        session.view(session.upload(HostTensor.packed_u4(np.arange(8) % 16, (8,))))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("lengths,row", [([(1, 200), (1, 3)], (1, 1, 2 ** 30, 1)), ([(1, 200), (1, 3)], (2, 1, 3, 1)), ([(40, 60), (7, 3)], (-1, 7, 3, 1)), ([(40, 60), (7, 3)], (40, 8, 3, 1)),
                                         ([(40, 60), (7, 3)], (40, 7, -1, 1)), ([(40, 60), (7, 3)], (40, -7, 3, 1)), ([(40, 60), (7, 3)], (40, 7, 2 ** 31 - 1, 1))], ids=str)
def test_a_sequence_that_does_not_lie_in_the_batch_is_reported(lengths, row, kind):
    f = Form(4, 2, 64, 128, 64)
    s = util.step(f, lengths, round_to=stored(kind))
    good = dataclasses.replace(s, seqs=s.seqs.copy())
    s.seqs[1] = row
    session = cuda_backend().prepare(util.module(f, DTYPES[kind], s.lam, s.gain))
    dev = {k: session.upload(v) for k, v in util.feed(s, act(kind)).items()}
    outs = session.run(dev)
    with pytest.raises(OnyxiaError, match="sequence 1 does not lie in"):
        session.download(outs[0][1])
    dev = {k: session.upload(v) for k, v in util.feed(good, act(kind)).items()}
    compare(session.download(session.run(dev)[0][1]).numpy(), util.reference(f, good, stored(kind))[0], kind, good)


def test_streams_that_are_captured_are_refused():
    torch = pytest.importorskip("torch")
    session = cuda_backend().prepare(util.module(Form(4, 2, 64, 128, 64), ir.BF16, np.ones(4, np.float32), np.ones(128, np.float32)))
    t, x, side = session.upload(HostTensor.from_numpy(np.arange(6, dtype=np.float32))), torch.ones(6, device="cuda"), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):
        y = x + 1
        for call in (lambda: session.upload_device(ir.F32, (6,), x.data_ptr(), side.cuda_stream), lambda: session.view(t, side.cuda_stream)):
            with pytest.raises(OnyxiaError, match="captured"):
                call()
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(y.cpu().numpy(), np.full(6, 2.0)) and np.array_equal(session.download(t).numpy(), np.arange(6))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_more_sequences_and_heads_than_places(kind):
    """More CTAs than run at a time: the last round's are cut into pieces."""
    lengths = [(1, 40 + 67 * i % 500) for i in range(40)]
    check(Form(16, 16, 32, 64, 16), lengths, kind)
    check(Form(16, 16, 64, 128, 64, window=300), lengths[:30], kind, seed=1)
    check(Form(9, 9, 128, 256, 32), lengths[:20], kind, seed=2)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("cap", [1.0, 4.0, 9.0, 100.0])
def test_caps(cap, kind):
    """Scores far above the cap, near it, at half of it and far below."""
    for f in (Form(4, 2, 64, 128, 64, softcap=cap), Form(4, 1, 128, 256, 128, softcap=cap)):
        check(f, [(100, 150), (1, 90)], kind)
