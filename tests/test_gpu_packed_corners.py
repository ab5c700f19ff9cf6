"""Keys and values in 4 bits where the kernels' number ranges end: keys that have nearly all weight, wide caps, positions next to 2^31, norms of many heads, places of very many values. The formulas in 64 bits and the tolerances are those of test_gpu_packed.py; what these do not
cover stands at each test."""
import dataclasses

import numpy as np
import pytest

import packed_util as util
import test_gpu_packed as base
from kipizen_util import to_bf16
from onyxia_b200 import OnyxiaError
from packed_util import Form
from test_gpu_packed import BOTH, compare, rounded, rows_of, run

pytestmark = pytest.mark.gpu


STEPS_MADE = {}


def fresh(f, lengths, kind):
    """util.step, made once for all that begin with the same."""
    key = repr(f), str(lengths), kind
    if key not in STEPS_MADE:
        STEPS_MADE[key] = util.step(f, lengths, 3, round_to=rounded(kind))
    return dataclasses.replace(STEPS_MADE[key], proj=STEPS_MADE[key].proj.copy())


def with_block(f, s, score, value):
    """Keys whose first sixteen dimensions are `score(sequence, position)` times those of a query, and keys whose value is `value(position)` times what it was: the score of a key is that, and a normal number of
    spread 1 from its other dimensions. Queries are neither turned nor normed: f16 holds them."""
    assert f.rot_dims == 0 and not f.norm and f.dim > 16 and not f.factors
    r, (q0, k0, v0) = np.random.default_rng(7), f.offsets
    q = r.standard_normal((len(s.proj), f.heads, f.dim)) / (f.scale * (f.dim - 16) ** 0.5)
    q[..., :16] = 1.0 / (16 * f.scale)
    s.proj[:, q0:q0 + f.heads * f.dim] = to_bf16(q.reshape(len(q), -1).astype(np.float32))
    pools = [[x.copy() for x in util.parts_of(pool)] for pool in (s.keys, s.values)]
    for i, (row, n, past, _) in enumerate(s.seqs):
        j = np.arange(past + n)
        for part, d, of in ((pools[0], f.dim, "key"), (pools[1], f.vdim, "value")):
            x = np.zeros((len(j), f.kv_heads, d), np.float32)
            old = j[:past]
            at = s.table[i, old // f.page], slice(None), old % f.page
            new = s.proj[row:row + n, (k0 if of == "key" else v0):][:, :f.kv_heads * d].reshape(n, f.kv_heads, d)
            assert np.shares_memory(new, s.proj)
            x[:past], x[past:] = util.valued(part[0][at], part[1][at], np.ones(f.kv_heads)), new
            if of == "key":
                x[..., :16] = np.array([score(p) for p in j])[:, None, None]
                x[..., 16:][np.array([score(p) for p in j]) != 0] *= 0.25
            else:
                x *= np.array([value(p) for p in j])[:, None, None]
            x = to_bf16(x)
            part[0][at], part[1][at] = util.packed(x[:past], np.ones(f.kv_heads))
            new[:] = x[past:]
    s.keys, s.values = util.bytes_of(*pools[0]), util.bytes_of(*pools[1])


def check(f, s, kind, gap):
    """bf16: the tolerances of `compare` at a spread of 1; a weight that is `gap` and a few units below the largest may be off by 2^-33 of that, which over a few thousand keys is 2^-33 / sqrt 3 · e^gap of the result, 6e-4
    at 17. f32: a product's sum reaches gap / scale in its first sixteen terms, each rounded to 2^-24, the exponential's argument and its value once more."""
    session, _, outs = run(f, s, kind)
    got, pools = session.download(outs["out"]).numpy(), util.written(f, s, rounded(kind))
    want, live = util.reference(f, s, pools), rows_of(s)
    empty = ~want[live].any(1)  # rows that see nothing but a value of 0
    assert not got[live][empty].any()
    if kind == "bf16":
        got[live[empty]] = want[live[empty]] = 1.0
        compare(got, want, kind, s, 1.0)
    else:
        off = np.sqrt(((got[live] - want[live]) ** 2).sum(1))[~empty] / np.sqrt((want[live] ** 2).sum(1))[~empty]
        assert off.max() <= 2.0 ** -24 * (18 * gap + 20)


FORMS = [Form(8, 2, 64, 128), Form(4, 4, 128, 64), Form(20, 1, 256, 256)]
STEPS = [[(150, 3000), (1, 4000), (1, 3500)], [(1, 8000), (1, 3000)], [(70, 4000)]]


@BOTH
@pytest.mark.parametrize("gap", [12, 14, 17])
@pytest.mark.parametrize("lengths", STEPS, ids=str)
@pytest.mark.parametrize("f", FORMS, ids=lambda f: f"{f.heads}x{f.kv_heads}x{f.dim}x{f.vdim}")
def test_a_first_key_that_has_nearly_all_weight(f, lengths, gap, kind):
    """As in trained models: its value adds little, so that a row's result is that of all the others."""
    s = fresh(f, lengths, kind)
    with_block(f, s, lambda p: gap * (p == 0), lambda p: float(p != 0))
    check(f, s, kind, gap)


@BOTH
def test_a_long_prompt_behind_such_a_key(kind):
    """Its own first key: two tiles of rows in a CTA, and rows of few keys."""
    f = Form(16, 16, 64, 64)
    s = util.step(f, [(4800 if kind == "bf16" else 300, 0)], 3, round_to=rounded(kind))
    with_block(f, s, lambda p: 12 * (p == 0), lambda p: float(p != 0))
    check(f, s, kind, 12)


@BOTH
@pytest.mark.parametrize("lengths", STEPS, ids=str)
def test_scores_that_rise_and_a_key_far_above_the_ones_before(lengths, kind):
    """What weights are taken against moves many times, by little and by much."""
    f = Form(8, 2, 64, 128)
    for score in (lambda p: 30.0 * p / 4000, lambda p: 9.0 * (p // 700), lambda p: 60.0 * (p == 1234), lambda p: -20.0 * (p < 2500)):
        s = fresh(f, lengths, kind)
        with_block(f, s, score, lambda p: 1.0)
        check(f, s, kind, 60)


@BOTH
@pytest.mark.parametrize("f", [Form(1, 5000, 128, 128, page=16), Form(1, 65535, 16, 16, page=16), Form(1, 150, 8192, 8192, page=16), Form(1, 520, 2048, 2032, page=16)], ids=lambda f: f"{f.kv_heads}x{f.dim}x{f.vdim}")
def test_places_of_very_many_values(f, kind):
    """More blocks of 16 dimensions than a quotient by a product serves: written, and read back."""
    s, got = base.check(f, [(2, 0), (1, 17)], kind, 3, "write")
    s.keys, s.values = got["updated.pages.keys"], got["updated.pages.values"]
    places = [(1, 17), (0, 1), (0, 0), (1, 3)]
    session, _, outs = run(f, s, kind, "read", places)
    assert np.array_equal(session.download(outs["stored"]).numpy(), rounded(kind)(util.read(f, [s.keys, s.values], s.table, places).astype(np.float32)))


@BOTH
@pytest.mark.parametrize("cap", [1e3, 1e4, 1e6, 1e9, 1e30])
def test_wide_caps(cap, kind):
    """A cap far above all scores changes none of them, in prompts and single tokens, whole tiles and those with hidden keys."""
    for f in (Form(4, 2, 64, 128, 64, softcap=cap), Form(4, 1, 128, 256, 128, softcap=cap, window=90), Form(16, 16, 64, 64, 64, softcap=cap)):
        base.check(f, [(100, 150), (1, 90)], kind)
        base.check(f, [(1, 700), (1, 3)], kind, seed=1)


@BOTH
@pytest.mark.parametrize("cap", [1e-30, 1e-38, 1e-40, 1e-46])
def test_caps_next_to_nothing(cap, kind):
    """Every key weighs the same, also where f32 does not hold the cap."""
    f = Form(4, 2, 64, 128, 64, softcap=cap, scale=cap * 1e25)
    base.check(f, [(100, 150), (1, 90)], kind)
    base.check(f, [(1, 700), (1, 3)], kind, seed=1)


@BOTH
@pytest.mark.parametrize("cap", [300.0, 4e3, 1e4, 1e6])
@pytest.mark.parametrize("lengths", STEPS, ids=str)
def test_scores_on_both_sides_of_a_quarter_of_a_wide_cap(lengths, cap, kind):
    """A few keys far below the others, which have all weight."""
    f = Form(8, 2, 64, 128, softcap=cap)
    s = fresh(f, lengths, kind)
    with_block(f, s, lambda p: -2600.0 * (p % 97 == 5), lambda p: 1.0)
    check(f, s, kind, 10)


@BOTH
@pytest.mark.parametrize("scale", [3e5, -3e6, 3e7, -3e8, 3e9, -3e10, 1e29, -1e29, 1e30, -1e30])
def test_scores_of_any_size_that_f32_has(scale, kind):
    """A row that sees one key has its value, whatever the score, far below 0 too."""
    f = Form(4, 2, 64, 128, 64, window=1, scale=scale)
    for lengths in ([(150, 20), (1, 200), (20, 130), (1, 0)], [(1, 200), (1, 0), (1, 63)]):
        s = util.step(f, lengths, 1, round_to=rounded(kind))
        session, _, outs = run(f, s, kind)
        want = util.reference(f, s, util.written(f, s, rounded(kind)))[rows_of(s)]
        assert np.array_equal(session.download(outs["out"]).numpy()[rows_of(s)], rounded(kind)(want.astype(np.float32)))


@BOTH
@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("form", ["attend", "write"])
def test_the_last_positions(form, new, kind):
    """Keys are counted in 32 bits, 128 at a time. Up to 2^31 - 128 a window's keys are those of the same page at its first place; a sequence that ends behind that is reported."""
    f = Form(2, 1, 16, 16, page=1 << 20, window=100)
    s = util.step(f, [(new, 500)], 3, round_to=rounded(kind), spare=0)
    place = f.page - 128 - new  # where the new tokens go; the window's keys come from where the step has some
    pools = [[x.copy() for x in util.parts_of(p)] for p in (s.keys, s.values)]
    for codes, scales in pools:
        codes[:, :, place - 500:place], scales[:, :, place - 500:place] = codes[:, :, :500].copy(), scales[:, :, :500].copy()
    s.keys, s.values = (util.bytes_of(*p) for p in pools)
    s.seqs[0, 2] = place
    session, _, outs = run(f, s, kind, form)
    want = {n: session.download(t).numpy() for n, t in outs.items()}
    s.table = np.full((1, 2048), -1, np.int32)
    s.table[0, -1] = 0
    s.seqs[0, 2] = 2 ** 31 - 128 - new
    session, dev, outs = run(f, s, kind, form)
    assert all(np.array_equal(session.download(t).numpy(), want[n]) for n, t in outs.items()) and len(want) == (3 if form == "attend" else 2)
    s.seqs[0, 2] += 1
    session, _, outs = run(f, s, kind, form)
    with pytest.raises(OnyxiaError, match="sequence 0 does not lie in"):
        session.download(next(iter(outs.values())))


@BOTH
@pytest.mark.parametrize("heads,kv", [(95, 1), (126, 1), (127, 1), (128, 1), (120, 40), (96, 32), (192, 96)], ids=str)
def test_norms_of_many_heads(heads, kv, kind):
    """A block of threads sums the squares of up to 128 heads at a time: as many, one fewer, one more, and a second and third time; queries and keys in one turn."""
    f = Form(heads, kv, 32, 32, 32, norm=1)
    base.check(f, [(40, 30), (1, 70), (3, 0)], kind)
    base.check(dataclasses.replace(f, rot_dims=0), [(5, 30)], kind, form="write")
    base.check(f, [(1, 30), (1, 70)], kind, seed=1)


@BOTH
@pytest.mark.parametrize("more", [dict(), dict(softcap=5.0), dict(softcap=1e4, window=200), dict(window=90), dict(sink=1, norm=1, factors=1), dict(scale=-0.125), dict(softcap=20.0, sink=1, norm=1, window=70, factors=1)], ids=str)
def test_two_tiles_of_rows(more, kind):
    """As many heads as give a block of threads two tiles of rows; tiles of one sequence, of its end, and of others."""
    f = Form(40, 40, 96, 64, 32, **more)
    base.check(f, [(280, 50), (30, 0), (1, 200)], kind)
    base.check(dataclasses.replace(f, heads=80, page=16), [(129, 300), (128, 0), (3, 63)], kind, seed=1)


@BOTH
def test_what_is_no_number_in_two_tiles_of_rows(kind):
    base.test_what_is_no_number_reaches_the_rows_that_see_it(Form(80, 80, 96, 64, 32), kind)
