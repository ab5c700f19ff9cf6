"""Keys and values in 4 bits on the device against the format and the formulas in 64 bits (packed_util.py).

Stored bytes are those of the format, all of them: rotations, norms and quotients next to a border between two codes are taken so that no rounding of theirs shows.

Tolerances of results. f32: a score is a sum of `dim` products, each rounded to 2^-24 relative to sums of the order of the score's spread (some units), its exponential to a few 2^-24: 1e-5 of a
row's length, 3e-6 over all rows. bf16: a result is rounded to 2^-8 of itself at most (2^-8 / sqrt 3 in the root mean square), what is stored not at all. Queries may be rounded to 2^-11 of themselves, which
moves a score by 2^-11 / sqrt 3 of its spread S (1.5 · scale · sqrt dim) and its weight by as much, weights to 2^-11, both for each key alone. In the root mean square of a row that is
2^-11 · (S + 1/2) at most; single rows, of few keys, get three times that.
"""
import dataclasses

import numpy as np
import pytest

import packed_util as util
from gpu_util import cuda_backend
from kipizen_util import to_bf16
from onyxia_b200 import OnyxiaError, ir
from onyxia_b200 import backend as be
from onyxia_b200.ir import HostTensor
from packed_util import Form

pytestmark = pytest.mark.gpu

DTYPES = {"f32": ir.F32, "bf16": ir.BF16}
BOTH = pytest.mark.parametrize("kind", ["f32", "bf16"])


def act(kind):
    return HostTensor.bf16 if kind == "bf16" else lambda a: HostTensor.from_numpy(np.asarray(a, np.float32))


def rounded(kind):
    return to_bf16 if kind == "bf16" else lambda a: np.asarray(a, np.float32)


def rows_of(s):
    return np.concatenate([np.arange(r, r + n) for r, n, _, _ in s.seqs] + [np.zeros(0, np.int64)]).astype(np.int64)


def compare(got, want, kind, s, spread=1.5):
    live = rows_of(s)
    got, want = got[live].astype(np.float64), want[live]
    assert np.isfinite(got).all()
    off, size = np.sqrt(((got - want) ** 2).sum(1)), np.sqrt((want ** 2).sum(1))
    more = 2 ** -11 * (spread + 0.5)
    whole, row = (2 ** -8 / 3 ** 0.5 + more, 2 ** -8 + 3 * more) if kind == "bf16" else (3e-6, 1e-5)
    assert np.sqrt((off ** 2).sum()) <= whole * np.sqrt((size ** 2).sum()) and (off / size).max() <= row


def run(f, s, kind, form="attend", places=None, backend=None):
    session = (backend or cuda_backend()).prepare(util.module(f, DTYPES[kind], form))
    dev = {k: session.upload(v) for k, v in util.feed(s, act(kind)).items()}
    if form == "read":
        dev = {k: v for k, v in dev.items() if k not in ("proj", "seq_info")}
    if places is not None:
        dev["places"] = session.upload(HostTensor.from_numpy(np.asarray(places, np.int32).reshape(-1, 2)))
    return session, dev, {n: t for n, t in session.run(dev)}


def check(f, lengths, kind, seed=0, form="attend", **more):
    s = util.step(f, lengths, seed, round_to=rounded(kind), **more)
    session, _, outs = run(f, s, kind, form)
    got = {n: session.download(t).numpy() for n, t in outs.items()}
    pools = [s.keys, s.values] if f.shared else util.written(f, s, rounded(kind))
    for name, want in zip(("updated.pages.keys", "updated.pages.values"), pools):
        assert name not in got or np.array_equal(got[name], want)
    if "out" in got:
        compare(got["out"], util.reference(f, s, pools), kind, s, 1.5 * abs(f.scale) * f.dim ** 0.5)
    return s, got


LAYOUTS = [Form(4, 1, 128, 256, 128), Form(16, 4, 64, 128, 64), Form(6, 2, 32, 64, 16), Form(5, 5, 48, 48, 48), Form(3, 1, 80, 160, 40), Form(20, 2, 64, 64, 0), Form(2, 1, 16, 32, 8),
           Form(3, 3, 16, 16, 6), Form(9, 1, 16, 32, 16), Form(1, 1, 256, 256, 256), Form(2, 2, 272, 144, 8), Form(8, 8, 112, 96, 112, gap=8), Form(4, 2, 64, 128, 32, gap=3), Form(34, 2, 96, 80, 96),
           Form(4, 4, 128, 128, 128, factors=1), Form(12, 1, 192, 64, 64, factors=1), Form(130, 1, 16, 32, 16)]


@BOTH
@pytest.mark.parametrize("f", LAYOUTS, ids=lambda f: f"{f.heads}x{f.kv_heads}x{f.dim}x{f.vdim}")
def test_layouts(f, kind):
    check(f, [(70, 0)], kind)
    check(f, [(1, 90), (1, 0), (1, 63), (1, 64)], kind, seed=1)
    check(f, [(3, 40), (1, 129), (66, 0), (1, 5), (65, 62)], kind, seed=2)


@BOTH
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
def test_page_sizes(page, kind):
    f = Form(4, 2, 32, 64, 32, page=page)
    check(f, [(1, 70), (37, 3), (1, 300), (130, 65)], kind)
    check(f, [(1, 70), (1, 255), (1, 0)], kind, seed=1)
    check(dataclasses.replace(f, dim=128, vdim=128, scale=0.1), [(150, 85), (1, 1100)], kind, seed=2)


@BOTH
@pytest.mark.parametrize("more", [dict(window=1), dict(window=17), dict(window=64), dict(window=100, sink=1), dict(softcap=5.0), dict(sink=1), dict(norm=1), dict(factors=1),
                                  dict(softcap=20.0, sink=1, norm=1, window=90, factors=1), dict(scale=0.25), dict(scale=-0.125),
                                  dict(scale=-0.125, softcap=3.0), dict(scale=1e-30, window=70)], ids=str)
def test_scores(more, kind):
    f = Form(4, 2, 64, 128, 64, **more)
    check(f, [(150, 0), (1, 200), (20, 130), (1, 0), (1, 64)], kind)
    check(f, [(1, 200), (1, 1), (1, 500)], kind, seed=1)


@BOTH
def test_long_ranges(kind):
    f = Form(8, 2, 64, 128, 64)
    check(f, [(1, 3000), (1, 1), (1, 4095)], kind)
    check(f, [(300, 900), (1, 2000)], kind, seed=1)
    check(Form(4, 1, 256, 256, 128), [(1, 2500)], kind, seed=2)
    check(Form(4, 1, 256, 256, 128, window=200), [(70, 1000), (1, 1500)], kind, seed=3)


@BOTH
def test_rows_and_sequences_of_a_padded_batch(kind):
    """Rows behind the last sequence are left alone, and sequences without new tokens (behind all others) do nothing, to the pools neither."""
    f = Form(4, 2, 64, 128, 64)
    for lengths, tail in (([(5, 3), (1, 70), (0, 10)], 9), ([(1, 3), (1, 70), (0, 10), (0, 0)], 1), ([(1, 3), (1, 70), (0, 10), (0, 0)], 2), ([(80, 0)], 70), ([(0, 5)], 3), ([(1, 70)], 4),
                          ([(3, 70), (0, 5), (0, 5), (0, 1), (0, 2)], 0), ([(2, 70), (1, 5), (0, 5), (0, 1), (0, 2)], 0)):
        if any(n for n, _ in lengths):
            check(f, lengths, kind, tail=tail)
        else:
            s = util.step(f, lengths, tail=tail, round_to=rounded(kind))
            session, _, outs = run(f, s, kind)
            assert np.array_equal(session.download(outs["updated.pages.keys"]).numpy(), s.keys)


@BOTH
def test_keys_that_stand_out_and_keys_that_weigh_the_same(kind):
    f = Form(4, 2, 64, 128, 0, scale=1.0)
    s = util.step(f, [(70, 20), (1, 130)], 5, round_to=rounded(kind), spread=8.0)
    session, _, outs = run(f, s, kind)
    got, pools = session.download(outs["out"]).numpy(), util.written(f, s, rounded(kind))
    want, live = util.reference(f, s, pools), rows_of(s)
    # scores of a spread of 64: where two keys are near each other both errors grow with it, else one key has all weight
    off = np.sqrt(((got[live] - want[live]) ** 2).sum(1)) / np.sqrt((want[live] ** 2).sum(1))
    assert np.isfinite(got[live]).all() and np.median(off) <= (2 ** -8 if kind == "bf16" else 1e-5) and off.max() <= (3 * 64 * 2 ** -11 if kind == "bf16" else 3 * 64 * 2 ** -20)
    s.proj[:, :f.offsets[1]] = 0.0  # every visible key weighs the same
    session, _, outs = run(f, s, kind)
    compare(session.download(outs["out"]).numpy(), util.reference(f, s, util.written(f, s, rounded(kind))), kind, s)


@BOTH
@pytest.mark.parametrize("size", [1e-6, 1e-3, 0.02, 300.0, 1e6])
def test_sizes_of_what_is_stored(size, kind):
    """Below the least scale all is 0, above the largest all is cut off; in between queries of the other size keep the scores where they are."""
    f = Form(4, 2, 64, 64, 64)
    s = util.step(f, [(70, 20), (1, 130), (1, 0)], 5, round_to=rounded(kind), size=size, spread=1.5 / size if 1e-5 < size < 1e4 else 1.0)
    session, _, outs = run(f, s, kind)
    pools = util.written(f, s, rounded(kind))
    assert np.array_equal(session.download(outs["updated.pages.keys"]).numpy(), pools[0])
    got, want = session.download(outs["out"]).numpy()[rows_of(s)], util.reference(f, s, pools)[rows_of(s)]
    if size < 6 * 2 ** -10 / 4:  # no value is four spreads from 0
        assert not got.any() and not want.any()
    elif size < 1e4:
        compare(session.download(outs["out"]).numpy(), util.reference(f, s, pools), kind, s)
    else:
        assert np.isfinite(got).all()


@BOTH
def test_values_that_are_no_numbers_are_stored_as_such(kind):
    """A value that is no number takes its sixteen with it, an infinite one is the largest there is; nothing else changes."""
    f = Form(4, 2, 64, 96, 32, factors=1)
    s = util.step(f, [(6, 3), (1, 20)], 1, round_to=rounded(kind))
    _, k0, v0 = f.offsets
    s.proj[1, k0 + 40] = np.nan
    s.proj[2, v0 + 96 + 17] = np.inf
    s.proj[3, v0 + 3:v0 + 5] = -np.inf, np.nan
    s.proj[4, v0:v0 + 192] = 0.0
    s.proj[5, v0:v0 + 192] = -0.0
    s.proj[6, v0] = 3e38
    session, _, outs = run(f, s, kind, "write")
    for name, want in zip(("updated.pages.keys", "updated.pages.values"), util.written(f, s, rounded(kind))):
        assert np.array_equal(session.download(outs[name]).numpy(), want)
    places = [(0, j) for j in range(9)] + [(1, 20)]
    want = util.read(f, util.written(f, s, rounded(kind)), s.table, places)
    s.keys, s.values = util.written(f, s, rounded(kind))
    session, _, outs = run(f, s, kind, "read", places)
    got = session.download(outs["stored"]).numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(want).sum() == 32
    assert np.array_equal(got[~np.isnan(got)], rounded(kind)(want.astype(np.float32))[~np.isnan(got)])


@BOTH
@pytest.mark.parametrize("f", [Form(4, 2, 64, 96, 32), Form(8, 8, 128, 128, 128, window=40), Form(40, 8, 128, 64, 0, page=16), Form(2, 1, 256, 256, 256)], ids=lambda f: f"{f.heads}x{f.kv_heads}x{f.dim}x{f.vdim}")
def test_what_is_no_number_reaches_the_rows_that_see_it(f, kind):
    """A key that is none: the rows of its head that see it. Sixteen dimensions of a value: these of the same rows. Rows before them, behind the window, and other heads are as without."""
    lengths = [(150, 20), (1, 130), (70, 0), (1, 20)]
    s = util.step(f, lengths, 3, round_to=rounded(kind))
    _, k0, v0 = f.offsets
    g = f.kv_heads - 1
    s.proj[60, v0 + g * f.vdim + 17] = np.nan    # token 60 of the first sequence: position 80
    s.proj[131, k0 + g * f.dim + 3] = np.nan     # token 131: position 151
    session, _, outs = run(f, s, kind)
    pools = util.written(f, s, rounded(kind))
    assert np.array_equal(session.download(outs["updated.pages.values"]).numpy(), pools[1])
    got, live = session.download(outs["out"]).numpy().reshape(len(s.proj), f.heads, f.vdim), rows_of(s)
    want = np.zeros(got.shape, bool)
    rep, w = f.heads // f.kv_heads, f.window or 10 ** 6
    want[60:min(150, 60 + w), g * rep:(g + 1) * rep, 16:32] = True
    want[131:min(150, 131 + w), g * rep:(g + 1) * rep] = True
    assert np.array_equal(np.isnan(got[live]), want[live])
    s.proj[60, v0 + g * f.vdim + 17] = s.proj[131, k0 + g * f.dim + 3] = 0.0
    other = util.reference(f, s, util.written(f, s, rounded(kind))).reshape(got.shape)
    seen = want.any(2)[live]
    off = np.sqrt(((got[live] - other[live]) ** 2).sum(2)) / np.sqrt((other[live] ** 2).sum(2))
    assert off[~seen].max() <= (2 ** -8 + 3 * 2 ** -10 if kind == "bf16" else 1e-5)


@BOTH
@pytest.mark.parametrize("f", LAYOUTS[::3] + [Form(2, 2, 16, 400, 16, page=16, factors=1, norm=1), Form(8, 8, 128, 128, 128, page=256, norm=1)], ids=lambda f: f"{f.kv_heads}x{f.dim}x{f.vdim}x{f.page}")
def test_written_and_read_back(f, kind):
    """What one call stores another reads, in any order, places twice too."""
    for lengths in ([(1, 0)], [(70, 3), (1, 200), (33, 31)], [(1, 30), (1, 64)]):
        s, got = check(f, lengths, kind, 3, "write", tail=2)
        s.keys, s.values = got["updated.pages.keys"], got["updated.pages.values"]
        places = [(i, j) for i, (_, n, past, _) in enumerate(s.seqs) for j in range(past + n)]
        places = np.array(places)[np.random.default_rng(1).permutation(len(places))]
        places = np.concatenate([places, places[:3]])
        session, _, outs = run(f, s, kind, "read", places)
        want = util.read(f, [s.keys, s.values], s.table, places).astype(np.float32)
        assert np.array_equal(session.download(outs["stored"]).numpy(), rounded(kind)(want))


@BOTH
@pytest.mark.parametrize("lengths", [[(150, 0), (1, 200), (20, 130)], [(1, 200), (1, 1), (1, 500)]], ids=str)
def test_a_run_of_them_together(lengths, kind):
    """Written, attended to by another node, and read back, in one step: as the one node that does both, and again from a captured step."""
    f = Form(8, 2, 64, 128, 32, norm=1, factors=1, sink=1)
    s = util.step(f, lengths, 2, round_to=rounded(kind))
    places = [(i, past + t) for i, (_, n, past, _) in enumerate(s.seqs) for t in range(n)] + [(0, 0)]
    session, dev, outs = run(f, s, kind, "chain", places)
    first = {n: session.download(t).numpy() for n, t in outs.items()}
    pools = util.written(f, s, rounded(kind))
    assert np.array_equal(first["updated.pages.keys"], pools[0]) and np.array_equal(first["updated.pages.values"], pools[1])
    assert np.array_equal(first["stored"], rounded(kind)(util.read(f, pools, s.table, places).astype(np.float32)))
    compare(first["out"], util.reference(f, s, pools), kind, s)
    one, _, whole = run(f, s, kind)
    assert np.array_equal(one.download(whole["out"]).numpy()[rows_of(s)], first["out"][rows_of(s)])
    for _ in range(3):
        for n, t in session.run(dev):
            assert np.array_equal(session.download(t).numpy(), first[n]) or n == "out" and np.array_equal(session.download(t).numpy()[rows_of(s)], first[n][rows_of(s)])


@BOTH
def test_queries_alone(kind):
    """Pools that hold the batch's keys and values already."""
    for more in ({}, dict(window=40, sink=1, factors=1)):
        check(Form(8, 2, 64, 128, 64, shared=True, **more), [(150, 0), (1, 200), (20, 130), (1, 0)], kind, 1, "shared")
        check(Form(4, 1, 128, 64, 64, shared=True, **more), [(1, 200), (1, 1000)], kind, 1, "shared")


@BOTH
def test_the_same_bits_again_and_from_captured_steps(kind):
    """Runs of one plan (the second and later ones replay a graph), and of a backend that launches one by one, are the same bits."""
    f = Form(8, 2, 64, 128, 64)
    for lengths in ([(1, 3000), (1, 100)], [(200, 700), (1, 900), (33, 0)]):
        s = util.step(f, lengths, 3, round_to=rounded(kind))
        session, dev, outs = run(f, s, kind)
        first = session.download(outs["out"]).numpy()[rows_of(s)]
        for _ in range(4):
            assert np.array_equal(session.download(session.run(dev)[0][1]).numpy()[rows_of(s)], first)
        session, _, outs = run(f, s, kind, backend=be.CudaBackend((0,), disable_graphs=True))
        assert np.array_equal(session.download(outs["out"]).numpy()[rows_of(s)], first)


@BOTH
@pytest.mark.parametrize("bad", [-1, 99, 2 ** 31 - 1])
@pytest.mark.parametrize("lengths", [[(1, 200)], [(90, 60)], [(1, 200), (70, 3)]], ids=str)
def test_a_page_that_is_none_is_reported(lengths, bad, kind):
    f = Form(4, 2, 64, 128, 64)
    s = util.step(f, lengths, round_to=rounded(kind))
    s.table[0, 1] = bad
    session, dev, outs = run(f, s, kind)
    with pytest.raises(OnyxiaError, match="out of range"):
        session.download(outs["out"])
    # the session goes on with a good table
    s.table[0, 1] = s.table[0, 0]
    dev["page_table"] = session.upload(HostTensor.from_numpy(s.table))
    session.download(session.run(dev)[0][1])


@BOTH
@pytest.mark.parametrize("bad", [(-1, 3), (2, 3), (0, -1), (0, 64), (1, 2 ** 31 - 1), (-2 ** 31, -2 ** 31), (1, 130)], ids=str)
def test_a_place_that_is_none_is_reported_and_reads_as_zeros(bad, kind):
    f = Form(4, 2, 64, 128, 64)
    s = util.step(dataclasses.replace(f, shared=True), [(1, 2), (1, 100)], round_to=rounded(kind), spare=0)  # the table is two pages wide, the first row has one
    session, dev, outs = run(f, s, kind, "read", [(0, 1), bad, (1, 100)])
    with pytest.raises(OnyxiaError, match="out of range"):
        session.download(outs["stored"])
    got = session.download(outs["stored"]).numpy()
    want = rounded(kind)(util.read(f, [s.keys, s.values], s.table, [(0, 1), (1, 100)]).astype(np.float32))
    assert np.array_equal(got[[0, 2]], want) and not got[1].any()


def test_a_prompt_in_a_batch_of_as_many_rows_as_sequences():
    """Taken in f32; in bf16 such a batch is one of single tokens, and a sequence of more is reported."""
    f = Form(4, 2, 64, 128, 64)
    check(f, [(3, 3), (1, 5), (0, 0), (0, 0)], "f32")
    s = util.step(f, [(3, 3), (1, 5), (0, 0), (0, 0)])
    session, _, outs = run(f, s, "bf16")
    with pytest.raises(OnyxiaError, match="sequence 0 has 3 new tokens"):
        session.download(outs["out"])


@BOTH
@pytest.mark.parametrize("form", ["attend", "write", "read"])
def test_nothing_to_do_and_nowhere_to_put_it(form, kind):
    f = Form(4, 2, 64, 128, 64)
    s = util.step(dataclasses.replace(f, shared=True), [(2, 3)], round_to=rounded(kind))
    session, dev, outs = run(f, s, kind, form, [(0, 1)] if form == "read" else None)
    first = session.download(next(iter(outs.values()))).numpy()
    up = lambda a: session.upload(HostTensor.from_numpy(a))  # noqa: E731
    if form == "read":
        assert session.run(dict(dev, places=up(np.zeros((0, 2), np.int32))))[0][1].shape == (0, 2 * 192)
    else:
        session.run(dict(dev, proj=session.upload(act(kind)(s.proj[:0]))))
        session.run(dict(dev, seq_info=up(s.seqs[:0]), page_table=up(s.table[:0])))
        with pytest.raises(OnyxiaError, match="without a page"):
            session.run({**dev, "pages.keys": up(s.keys[:0]), "pages.values": up(s.values[:0])})
    session.wait_idle()
    if form != "write":
        assert np.array_equal(session.download(session.run(dev)[0][1]).numpy(), first)


@BOTH
@pytest.mark.parametrize("lengths,row", [([(1, 200), (1, 3)], (1, 1, 2 ** 30, 1)), ([(1, 200), (1, 3)], (2, 1, 3, 1)), ([(40, 60), (7, 3)], (-1, 7, 3, 1)), ([(40, 60), (7, 3)], (40, 8, 3, 1)),
                                         ([(40, 60), (7, 3)], (40, 7, -1, 1)), ([(40, 60), (7, 3)], (40, -7, 3, 1)), ([(40, 60), (7, 3)], (40, 7, 2 ** 31 - 1, 1))], ids=str)
def test_a_sequence_that_does_not_lie_in_the_batch_is_reported(lengths, row, kind):
    f = Form(4, 2, 64, 128, 64)
    s = util.step(f, lengths, round_to=rounded(kind))
    good = dataclasses.replace(s, seqs=s.seqs.copy())
    s.seqs[1] = row
    session, dev, outs = run(f, s, kind)
    with pytest.raises(OnyxiaError, match="sequence 1 does not lie in"):
        session.download(outs["out"])
    dev = {k: session.upload(v) for k, v in util.feed(good, act(kind)).items()}
    compare(session.download(session.run(dev)[0][1]).numpy(), util.reference(f, good, util.written(f, good, rounded(kind))), kind, good)


@BOTH
def test_more_sequences_and_heads_than_places(kind):
    lengths = [(1, 40 + 67 * i % 500) for i in range(40)]
    check(Form(16, 16, 32, 64, 16), lengths, kind)
    check(Form(16, 16, 64, 128, 64, window=300), lengths[:30], kind, seed=1)
    check(Form(9, 9, 128, 256, 32), lengths[:20], kind, seed=2)


@BOTH
@pytest.mark.parametrize("cap", [1.0, 4.0, 9.0, 100.0])
def test_caps(cap, kind):
    """Scores far above the cap, near it, at half of it and far below."""
    for f in (Form(4, 2, 64, 128, 64, softcap=cap), Form(4, 1, 128, 256, 128, softcap=cap)):
        check(f, [(100, 150), (1, 90)], kind)


@BOTH
@pytest.mark.parametrize("new", [1, 70])
def test_pools_of_more_bytes_than_32_bits_count(new, kind):
    torch = pytest.importorskip("torch")
    f = Form(2, 1, 256, 16, 256, page=256)
    s = util.step(f, [(new, 300)], round_to=rounded(kind), spare=0)
    pages, want = 120_000, util.written(f, s, rounded(kind))
    session = cuda_backend().prepare(util.module(f, DTYPES[kind]))
    dev = {k: session.upload(v) for k, v in util.feed(s, act(kind)).items()}
    at = torch.tensor([pages - 1, pages // 2])[:len(s.keys)]
    for name, small in (("pages.keys", s.keys), ("pages.values", s.values)):
        x = torch.zeros(pages, *small.shape[1:], dtype=torch.uint8, device="cuda")
        x[at] = torch.from_numpy(small).cuda()
        dev[name] = session.upload_device(ir.U8, tuple(x.shape), x.data_ptr(), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        del x
    dev["page_table"] = session.upload(HostTensor.from_numpy(at.numpy()[s.table].astype(np.int32)))
    outs = dict(session.run(dev))
    compare(session.download(outs["out"]).numpy(), util.reference(f, s, want), kind, s)
    for name, pool in zip(("updated.pages.keys", "updated.pages.values"), want):
        got = torch.as_tensor(session.view(outs[name], torch.cuda.current_stream().cuda_stream), device="cuda")
        assert np.array_equal(got[at].cpu().numpy(), pool) and not got[:pages // 2].any()
        del got
    torch.cuda.empty_cache()
