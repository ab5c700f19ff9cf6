"""Rules on logits on the device against a plain implementation in 64 bits.

Tolerance: a logit is multiplied or divided once, n · frequency and presence are taken from it and a few biases added, each rounded to 2^-24 of terms up to 40 here: at most
eight roundings of values below 64, 8 · 64 · 2^-24 = 3.1e-5. What no rule touches, and what is not allowed, is exact.
"""
import numpy as np
import pytest

from gpu_util import cuda_backend
from onyxia_b200 import OnyxiaError, ir
from onyxia_b200.ir import HostTensor

pytestmark = pytest.mark.gpu

TOL = 8 * 64 * 2.0 ** -24


@pytest.fixture(scope="module")
def session():
    b = ir.GraphBuilder()
    b.output("one", b.const_f32([1.0], [1]))
    return cuda_backend().prepare(b.finish())


def up(session, a, dtype=None):
    return None if a is None else session.upload(HostTensor.from_numpy(a))


def rules(rows, vocab, width, n_bias, n_masks, seed=0):
    r = np.random.default_rng(seed)
    few = r.integers(0, vocab, 9)
    history = np.where(r.random((rows, width)) < 0.5, few[r.integers(0, 9, (rows, width))], r.integers(0, vocab, (rows, width))).astype(np.int32)
    total = r.integers(0, width + 1, rows)
    total[0] = width
    lengths = np.stack([r.integers(0, total + 1), total], 1).astype(np.int32)
    if width:
        history[np.arange(width) >= total[:, None]] = 2 ** 31 - 1  # nobody reads there
    out = {"history": history, "lengths": lengths,
           "penalties": np.stack([r.uniform(0.7, 1.5, rows), r.uniform(-0.2, 0.5, rows), r.uniform(-0.5, 0.7, rows)], 1).astype(np.float32)}
    if n_bias:
        ids = r.integers(0, vocab, (rows, n_bias)).astype(np.int32)
        ids[r.random(ids.shape) < 0.2] = -1
        ids[:, n_bias // 2:] = np.where(r.random((rows, n_bias - n_bias // 2)) < 0.3, ids[:, :n_bias - n_bias // 2], ids[:, n_bias // 2:])  # listed again
        out.update(bias_ids=ids, bias=(3.0 * r.standard_normal(ids.shape)).astype(np.float32))
    if n_masks:
        out["masks"] = r.integers(0, 2 ** 32, (n_masks, -(-vocab // 32)), dtype=np.uint32)
        out["masks"][0] = 0 if n_masks > 1 else out["masks"][0]
        out["mask_of"] = r.integers(-1, n_masks, rows).astype(np.int32)
    return out


def reference(x, history=None, lengths=None, penalties=None, bias_ids=None, bias=None, masks=None, mask_of=None):
    y = x.astype(np.float64)
    for r in range(len(y)):
        if history is not None:
            prompt, total = lengths[r]
            rep, freq, pres = penalties[r].astype(np.float64)
            for t in set(history[r, :total].tolist()):
                y[r, t] = y[r, t] / rep if y[r, t] > 0 else y[r, t] * rep
            said = history[r, prompt:total].tolist()
            for t in set(said):
                y[r, t] -= said.count(t) * freq + pres
        if bias_ids is not None:
            for t, b in zip(bias_ids[r], bias[r]):
                if t >= 0:
                    y[r, t] += float(b)
        if masks is not None:
            m = r if mask_of is None else mask_of[r]
            if m >= 0:
                bits = np.unpackbits(masks[m].view(np.uint8), bitorder="little")[:y.shape[1]]
                y[r, bits == 0] = -np.inf
    return y


def check(session, x, more):
    got = session.download(session.constrain_last(up(session, x), **{k: up(session, v) for k, v in more.items()}))
    assert got.dtype == ir.F32 and got.shape == x.shape
    got, want = got.numpy().reshape(-1, x.shape[-1]), reference(x.reshape(-1, x.shape[-1]), **more)
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    with np.errstate(invalid="ignore"):
        assert np.nanmax(np.where(np.isneginf(want), 0.0, np.abs(got - want)), initial=0.0) <= TOL
    same = want == x.reshape(want.shape)
    assert np.array_equal(got[same], x.reshape(want.shape).astype(np.float32)[same])


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 3), (2, 31), (3, 32), (2, 33), (1, 4095), (3, 4096), (5, 4097), (2, 12288 + 4), (1, 32000), (70, 517), (3, 50021), (2, 262144), (300, 1000)])
def test_sizes(session, rows, vocab, dtype):
    r = np.random.default_rng(vocab)
    x = (4.0 * r.standard_normal((rows, vocab))).astype(dtype)
    for width, n_bias, n_masks in ((0, 0, 0), (1, 0, 1), (40, 7, 0), (700, 300, 3)):
        check(session, x, rules(rows, vocab, width, n_bias, n_masks, seed=rows))


def test_each_rule_alone_and_no_rule(session):
    r = np.random.default_rng(1)
    for dtype in (np.float32, np.float16):
        x = (4.0 * r.standard_normal((4, 2, 1000))).astype(dtype)
        every = rules(8, 1000, 50, 20, 4)
        check(session, x, {})
        check(session, x, {k: every[k] for k in ("history", "lengths", "penalties")})
        check(session, x, {k: every[k] for k in ("bias_ids", "bias")})
        check(session, x, {k: every[k] for k in ("masks", "mask_of")})
        check(session, x, {"masks": r.integers(0, 2 ** 32, (8, 32), dtype=np.uint32)})


def test_one_token_many_times(session):
    x = np.full((2, 100), 2.0, np.float32)
    history = np.full((2, 3000), 7, np.int32)
    more = {"history": history, "lengths": np.array([[0, 3000], [3000, 3000]], np.int32), "penalties": np.array([[2.0, 0.01, 0.5]] * 2, np.float32),
            "bias_ids": np.full((2, 4096), 7, np.int32), "bias": np.full((2, 4096), 0.001, np.float32)}
    got = session.download(session.constrain_last(up(session, x), **{k: up(session, v) for k, v in more.items()})).numpy()
    # 4096 biases are added one after the other: each sum, up to 4.1, is rounded to 2^-22 · 1/2; 4096 · 2^-23 = 5e-4
    assert abs(got[0, 7] - (1.0 - 30.0 - 0.5 + 4.096)) <= 6e-4 and abs(got[1, 7] - (1.0 + 4.096)) <= 6e-4
    assert (np.delete(got, 7, 1) == 2.0).all()


def test_infinities_and_nan(session):
    """They are what the arithmetic makes of them, and nothing where they are not allowed."""
    x = np.zeros((1, 64), np.float32)
    x[0, :6] = np.inf, -np.inf, np.nan, np.inf, np.nan, -np.finfo(np.float32).max
    masks = np.full((1, 2), 0xFFFFFFFF, np.uint32)
    masks[0, 0] &= ~np.uint32(0b11000)
    more = {"history": np.arange(6, dtype=np.int32)[None], "lengths": np.array([[3, 6]], np.int32), "penalties": np.array([[1.5, 0.1, 0.1]], np.float32), "masks": masks}
    got = session.download(session.constrain_last(up(session, x), **{k: up(session, v) for k, v in more.items()})).numpy()[0]
    assert got[0] == np.inf and got[1] == -np.inf and np.isnan(got[2]) and got[3] == got[4] == -np.inf and got[5] == -np.inf and (got[6:] == 0).all()


def test_a_mask_that_allows_nothing(session):
    x = up(session, np.zeros((2, 40), np.float32))
    y = session.constrain_last(x, masks=up(session, np.array([[0, 0], [4, 0]], np.uint32)))
    assert np.isneginf(session.download(y).numpy()[0]).all()
    assert session.download(session.argmax_last(y)).numpy().tolist() == [39, 2]
    with pytest.raises(OnyxiaError, match="row 0"):
        session.download(session.sample_last(y, 1.0, 0, 1.0, [0.5, 0.5]))
    y = session.constrain_last(x, masks=up(session, np.array([[4, 0]], np.uint32)), mask_of=up(session, np.array([0, 0], np.int32)))
    assert session.download(session.sample_last(y, 1.0, 0, 1.0, [0.0001, 1.0])).numpy().tolist() == [2, 2]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("change,message", [
    (lambda m: m["history"].__setitem__((1, 2), 1000), "token 1000 is not one of 1000"), (lambda m: m["history"].__setitem__((1, 2), -1), "token -1 is not one of 1000"),
    (lambda m: m["lengths"].__setitem__(1, [3, 51]), "lengths of row 1"), (lambda m: m["lengths"].__setitem__(1, [8, 7]), "lengths of row 1"),
    (lambda m: m["lengths"].__setitem__(1, [-1, 7]), "lengths of row 1"), (lambda m: m["bias_ids"].__setitem__((1, 3), 2 ** 31 - 1), "token 2147483647"),
    (lambda m: m["mask_of"].__setitem__(1, 4), "mask 4 is not one of 4")], ids=range(7))
def test_contents_that_are_wrong_are_reported(session, change, message, dtype):
    more = rules(2, 1000, 50, 20, 4)
    more["lengths"][:] = 10, 50
    more["history"][:] = 5
    good = {k: v.copy() for k, v in more.items()}
    change(more)
    x = up(session, np.zeros((2, 1000), dtype))
    y = session.constrain_last(x, **{k: up(session, v) for k, v in more.items()})
    with pytest.raises(OnyxiaError, match=message):
        session.download(y)
    check(session, np.zeros((2, 1000), dtype), good)  # the session goes on


def test_shapes_and_types_that_do_not_fit_are_refused(session):
    x = up(session, np.zeros((2, 100), np.float32))
    more = {k: up(session, v) for k, v in rules(2, 100, 5, 3, 2).items()}
    for gone in ("history", "lengths", "penalties", "bias_ids", "bias", "masks"):
        with pytest.raises(OnyxiaError, match="rules"):
            session.constrain_last(x, **{k: v for k, v in more.items() if k != gone})
    with pytest.raises(OnyxiaError, match="rules"):
        session.constrain_last(up(session, np.zeros((3, 100), np.float32)), **more)
    with pytest.raises(OnyxiaError, match="f32 or f16"):
        session.constrain_last(up(session, np.zeros((2, 100), np.int32)))


def test_logits_that_are_part_of_a_buffer_and_the_same_bits_again(session):
    """Rows whose first logit lies on no boundary of four, and runs that follow one another."""
    r = np.random.default_rng(3)
    for vocab in (1001, 1002, 4099):
        x = (4.0 * r.standard_normal((5, vocab))).astype(np.float16)
        more = rules(5, vocab, 60, 200, 2)
        dev = {k: up(session, v) for k, v in more.items()}
        check(session, x, more)
        first = session.download(session.constrain_last(up(session, x), **dev)).numpy()
        for _ in range(3):
            assert np.array_equal(session.download(session.constrain_last(up(session, x), **dev)).numpy(), first, equal_nan=True)
