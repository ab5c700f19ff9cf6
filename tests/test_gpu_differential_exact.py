"""bf16 kernels of differential attention against what their roundings may cost (differential_exact.py).

All results together are off by what they are due, give or take a tenth: over the thousands of (row, head) of each case the mean of squares is known to 2 %, and mantissas of exponentials of
scores that spread over octaves, and of results, are spread as logarithms to a few percent. A query rounded once more would add 1.5 · 1.66e-3 to every score (a spread of 1.5), and with it
sqrt((2 + 1.5²) / 2) = 1.46 times what is due at D = 1. Sums that miss a scaling, or the values of half a tile, are off by the order of the results.
"""
import numpy as np
import pytest

import differential_computed
import differential_exact as exact
import differential_util as util
from differential_util import Form
from gpu_util import cuda_backend
from kipizen_util import to_bf16
from onyxia_b200 import ir
from onyxia_b200.ir import HostTensor

pytestmark = pytest.mark.gpu

DUE = 1.1
# A few rows that see a few keys: one (row, head) of nearly equal maps over five keys may be most of the sum, and the mean of five squares is above four in one of a thousand.
DUE_FEW = 2.0
# the second form's products are made by halves of a tile: maps above 64 or values above 128 dimensions
NARROW, WIDE, WIDE_VALUES = Form(8, 2, 64, 128, 64), Form(4, 1, 128, 256, 128), Form(4, 2, 64, 192, 64)


def results(f, s, runs=1):
    session = cuda_backend().prepare(util.module(f, ir.BF16, s.lam, s.gain))
    dev = {k: session.upload(v) for k, v in util.feed(s, HostTensor.bf16).items()}
    return [session.download(session.run(dev)[0][1]).numpy() for _ in range(runs)]


def rising(f, s, by):
    """Keys grow along their sequences: every tile of keys brings rows a new maximum. Queries see them from their own side: all first dimensions are positive."""
    q0, k0, _ = f.offsets
    for i, (row, n, past, _) in enumerate(s.seqs):
        for pos in range(past):
            pg, off = s.table[i, pos // f.page], pos % f.page
            for m in (0, 1):
                s.keys[pg, :, off, m * f.dim] = by * pos / 64
        for t in range(n):
            for g in range(2 * f.kv_heads):
                s.proj[row + t, k0 + g * f.dim] = by * (past + t) / 64
    s.proj[:, q0:q0 + f.heads * 2 * f.dim:f.dim] = 1.0 / f.scale
    s.keys, s.proj = to_bf16(s.keys), to_bf16(s.proj)


@pytest.mark.parametrize("f", [NARROW, WIDE, WIDE_VALUES], ids=["narrow", "wide", "wide values"])
@pytest.mark.parametrize("by", [0.05, 0.5, 3.0])
def test_maxima_that_rise_with_every_tile(f, by):
    """Sums are scaled again and again, by threads that share a row, in front of the products of either half of a tile."""
    f = Form(f.heads, f.kv_heads, f.dim, f.vdim, 0)
    s = util.step(f, [(700, 900), (130, 60)], 7)
    rising(f, s, by)
    first, *more = results(f, s, 6)
    assert exact.share(f, s, first, to_bf16) <= DUE
    live = np.concatenate([np.arange(r, r + n) for r, n, _, _ in s.seqs])
    for again in more:
        assert np.array_equal(again[live], first[live])


@pytest.mark.parametrize("f", [NARROW, WIDE, WIDE_VALUES], ids=["narrow", "wide", "wide values"])
@pytest.mark.parametrize("window", [0, 100])
def test_a_tile_that_begins_and_ends_within_a_page_of_no_numbers(f, window):
    """Prompts end in every part of a tile, and windows begin there; what lies behind the last key, and in front of the first, is NaN. Maxima stand still, so that nothing waits for products."""
    f = Form(f.heads, f.kv_heads, f.dim, f.vdim, 0, window=window)
    s = util.step(f, [(33, 128 * 3 + 1 + 13 * i) for i in range(12)] + [(200, 7), (90, 1200)], 11, spread=0.0)
    if window:
        for i, (_, _, past, _) in enumerate(s.seqs):
            for pos in range(max(0, past - window + 1)):
                s.keys[s.table[i, pos // f.page], :, pos % f.page] = s.values[s.table[i, pos // f.page], :, pos % f.page] = np.nan
    first, *more = results(f, s, 6)
    live = np.concatenate([np.arange(r, r + n) for r, n, _, _ in s.seqs])
    assert np.isfinite(first[live]).all()
    for again in more:
        assert np.array_equal(again[live], first[live])
    known = util.Step(s.proj, np.nan_to_num(s.keys), np.nan_to_num(s.values), s.seqs, s.table, s.lam, s.gain)  # (nothing times NaN is no number in the formulas)
    assert exact.share(f, known, first, to_bf16) <= DUE


def test_as_many_heads_as_fill_a_blocks_memory_with_factors():
    """Normed queries and keys of 4096 heads and as many key heads: 64 KB of factors."""
    f = Form(4096, 4096, 16, 16, 16, page=8, norm=1)
    s = util.step(f, [(3, 9), (2, 0)], 3, spare=0)
    assert exact.share(f, s, results(f, s)[0], to_bf16) <= DUE


@pytest.mark.parametrize("lengths", [[(2, 5), (0, 9), (0, 0)], [(2, 70), (1, 3), (0, 0), (0, 4)], [(1, 80), (3, 0)] + [(0, 1)] * 4, [(1, 64), (1, 0), (0, 7)], [(1, 130), (0, 0), (0, 0)], [(70, 60)] + [(0, 0)] * 90], ids=str)
@pytest.mark.parametrize("f", [NARROW, WIDE, Form(20, 2, 24, 40, 8, page=4, window=50, sink=1, softcap=5.0, norm=1, gap=3)], ids=["narrow", "wide", "odd"])
def test_batches_padded_with_sequences_without_new_tokens(f, lengths):
    """Fewer rows than sequences: sequences may have any number of new tokens. (As many rows as sequences say that each has one at most.)"""
    s = util.step(f, lengths, 5)
    assert exact.share(f, s, results(f, s)[0], to_bf16) <= DUE_FEW


@pytest.mark.parametrize("maps", [2, 1], ids=["differential", "plain"])
@pytest.mark.parametrize("computed", [("seq_info",), ("page_table",), ("turns",), ("reshaped",), ("seq_info", "page_table", "turns")], ids="+".join)
def test_batches_and_angles_that_the_module_computes(computed, maps):
    """The same bits as where they are inputs and constants, whether a run is launched one by one or replayed. The batch changes between runs."""
    f = Form(16, 4, 64, 128, 64)
    for lengths in ([(1, 700 + 50 * i) for i in range(20)], [(130, 40), (1, 900), (3, 60)]):
        s = util.step(f, lengths, 3)
        keys, values = s.keys[..., :maps * f.dim], s.values
        want, got = [], []
        for how, into in (((), want), (computed, got)):
            session = cuda_backend().prepare(differential_computed.module(f, ir.BF16, s.lam, s.gain, how, maps))
            feed = {"proj": session.upload(HostTensor.bf16(s.proj)), "pages.keys": session.upload(HostTensor.bf16(keys)), "pages.values": session.upload(HostTensor.bf16(values))}
            for back in (0, 1, 5, 0, 2):
                seqs = s.seqs.copy()
                seqs[:, 2] = np.maximum(seqs[:, 2] - back, 0)
                table = s.table[:, None] if "reshaped" in how else s.table
                feed["seq_info"] = session.upload(HostTensor.from_numpy(seqs.astype(np.int64 if "seq_info" in how else np.int32)))
                feed["page_table"] = session.upload(HostTensor.from_numpy(table.astype(np.int64 if "page_table" in how else np.int32)))
                outs = dict(session.run(feed))
                into.append([session.download(outs[n]).numpy() for n in ("out", "updated.pages.keys")])
                feed["pages.keys"], feed["pages.values"] = outs["updated.pages.keys"], outs["updated.pages.values"]
        for (a, k), (b, l) in zip(want, got):
            assert np.array_equal(a, b) and np.array_equal(k, l, equal_nan=True)


@pytest.mark.parametrize("f", [NARROW, WIDE], ids=["narrow", "wide"])
def test_what_lies_behind_the_last_key_changes_no_bit(f):
    """Caps are a polynomial or an exponential by what a warp's scores are: those of keys that a row sees."""
    f = Form(f.heads, f.kv_heads, f.dim, f.vdim, 0, softcap=4.0, window=150)
    s = util.step(f, [(20, 40), (130, 100), (1, 70), (40, 300)], 13, spread=0.5)
    outs = []
    for behind in (0.0, 1.0, -300.0, 3e38, np.inf, np.nan):
        keys = s.keys.copy()
        keys[np.isnan(keys)] = behind
        outs += results(f, util.Step(s.proj, to_bf16(keys), np.nan_to_num(s.values), s.seqs, s.table, s.lam, s.gain), 2)
    assert exact.share(f, s, outs[0], to_bf16) <= DUE
    live = np.concatenate([np.arange(r, r + n) for r, n, _, _ in s.seqs])
    for other in outs[1:]:
        assert np.array_equal(other[live], outs[0][live])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("lengths,tail", [([(0, 5)], 3), ([(0, 5), (0, 70), (0, 0)], 3), ([(0, 5), (0, 70), (0, 0)], 9), ([(2, 3), (0, 70), (0, 0)], 0), ([(2, 3), (0, 70), (0, 0)], 9)], ids=str)
def test_sequences_without_new_tokens_leave_the_pools_alone(lengths, tail, kind):
    """Rows of nobody behind them or not; the first run, and replayed ones."""
    f = Form(4, 2, 64, 128, 64)
    act = HostTensor.bf16 if kind == "bf16" else lambda a: HostTensor.from_numpy(np.asarray(a, np.float32))
    s = util.step(f, lengths, tail=tail)
    session = cuda_backend().prepare(util.module(f, ir.BF16 if kind == "bf16" else ir.F32, s.lam, s.gain))
    dev = {k: session.upload(v) for k, v in util.feed(s, act).items()}
    keys, values = util.reference(f, s, to_bf16 if kind == "bf16" else lambda a: np.asarray(a, np.float32))[1:]
    for _ in range(3):
        outs = dict(session.run(dev))
        dev["pages.keys"], dev["pages.values"] = outs["updated.pages.keys"], outs["updated.pages.values"]
        assert np.array_equal(session.download(dev["pages.values"]).numpy(), values.astype(np.float32), equal_nan=True)
        got = session.download(dev["pages.keys"]).numpy()
        old = ~np.isnan(s.keys)
        assert np.array_equal(got[old], s.keys[old]) and np.array_equal(np.isnan(got), np.isnan(keys))


@pytest.mark.parametrize("f", [NARROW, WIDE, WIDE_VALUES, Form(20, 2, 48, 96, 48)], ids=["narrow", "wide", "wide values", "many heads"])
@pytest.mark.parametrize("more", [dict(norm=1), dict(norm=1, sink=1, softcap=30.0, window=700), dict(softcap=1.0), dict(softcap=3.0, sink=1)], ids=str)
@pytest.mark.parametrize("lengths", [[(700, 900), (130, 60), (1, 400)], [(1, 1000 + 37 * i) for i in range(40)]], ids=["prompts", "tokens"])
def test_scores_that_do_not_spread_cost_no_precision(f, more, lengths):
    """Normed queries and keys, and tight caps: where maps of nearly equal weights are taken from each other, D is 1.2 and more, and results are off by their own rounding all the same."""
    f = Form(f.heads, f.kv_heads, f.dim, f.vdim, f.rot_dims, **more)
    s = util.step(f, lengths, 17)
    assert exact.share(f, s, results(f, s)[0], to_bf16, two_parts=True) <= DUE


@pytest.mark.parametrize("f", [NARROW, WIDE], ids=["narrow", "wide"])
@pytest.mark.parametrize("by", [0.05, 3.0])
def test_maxima_that_rise_with_weights_in_two_parts(f, by):
    """The weights of a tile are written behind the products of the tile before it, the sums scaled in front of them."""
    f = Form(f.heads, f.kv_heads, f.dim, f.vdim, 0, softcap=3.0)
    s = util.step(f, [(700, 900), (130, 60)], 7)
    rising(f, s, by)
    first, *more = results(f, s, 6)
    assert exact.share(f, s, first, to_bf16, two_parts=True) <= DUE
    live = np.concatenate([np.arange(r, r + n) for r, n, _, _ in s.seqs])
    for again in more:
        assert np.array_equal(again[live], first[live])
