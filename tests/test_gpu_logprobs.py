"""Log probabilities of tokens, entropy and best alternatives (wdc_token_logprobs) against the definitions in 64 bits.

Tolerances, from the formula: a log probability is (x - max) - log(sum): the sum of n positive float32 terms, each off by a few
2^-24, is off by less than 2^-18 of itself in any order of n < 2^20 / 16 chained additions a thread, the logarithm's error is
that sum's relative one, and the differences round to 2^-23 of their size: |error| <= 2^-18 + 2^-22 * |value|.  The entropy is a
difference of log(sum) and a weighted mean of (x - max), both of which are off by at most 2^-18 of themselves.
"""
from ctypes import byref, c_void_p

import numpy as np
import pytest

from webdnn_b200.backend import CPUTensor
from webdnn_b200.lib import CudaBackendError, LogprobsDesc

pytestmark = pytest.mark.gpu
f32 = np.float32


def dev(ctx, a):
    return ctx.move_tensor(CPUTensor.from_array(np.ascontiguousarray(a)))


def reference(x, tokens, top):
    x = x.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = x.max(1, keepdims=True)
        e = np.exp(x - m)
        logs = x - m - np.log(e.sum(1, keepdims=True))
        p = e / e.sum(1, keepdims=True)
        entropy = -np.where(p > 0, p * logs, np.where(np.isnan(p), np.nan, 0)).sum(1)
    bad = ~np.isfinite(m[:, 0])
    logs[bad] = entropy[bad] = np.nan
    order = np.lexsort((np.broadcast_to(np.arange(x.shape[1]), x.shape), -np.where(np.isnan(x), np.inf, x), ~np.isnan(x)), axis=1)
    ids = order[:, :top]
    inside = (tokens >= 0) & (tokens < x.shape[1])
    logprob = np.where(inside, logs[np.arange(len(x)), np.where(inside, tokens, 0)], np.nan)
    return logprob, entropy, ids, np.take_along_axis(logs, ids, 1), m[:, 0]


def near(got, want, slack):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isinf(got), np.isinf(want)) and np.array_equal(got[np.isinf(got)], want[np.isinf(want)])
    fine = np.isfinite(want)
    assert (np.abs(got - want)[fine] <= (2.0 ** -18 * slack + 2.0 ** -22 * np.abs(want))[fine]).all(), np.abs(got - want)[fine].max()


def check(ctx, x, tokens, top, vocab=None):
    vocab = x.shape[1] if vocab is None else vocab
    ts = [dev(ctx, x), dev(ctx, tokens.astype(np.int32))]
    got = ctx.token_logprobs(*ts, top, vocab=vocab)
    logprob, entropy, ids, best, _ = reference(x[:, :vocab], tokens, top)
    near(got[0].get_data(), logprob, 1)
    near(got[1].get_data(), entropy, 1 + np.log(vocab) + np.nan_to_num(np.abs(entropy)))
    if top:
        assert np.array_equal(got[2].get_data().reshape(ids.shape), ids)
        near(got[3].get_data().reshape(ids.shape), best, 1)
    for t in ts + [t for t in got if t is not None]:
        t.dispose()


@pytest.mark.parametrize("rows,vocab,pad,top", [
    (1, 1, 0, 1), (3, 2, 1, 2), (2, 31, 0, 5), (5, 33, 3, 32), (1, 255, 0, 0), (4, 1000, 1, 8), (300, 257, 2, 3),
    (1, 32000, 0, 20), (7, 4099, 1, 32), (2, 100003, 0, 32), (40, 20001, 3, 1), (1, 200001, 0, 5), (150, 9000, 0, 32),
    (1000, 1025, 0, 1), (3, 65536, 0, 16), (37, 50021, 0, 10), (1, 1025, 3, 32), (296, 2048, 1, 7)])
def test_rows(cuda_context, rows, vocab, pad, top):
    rng = np.random.default_rng(rows + vocab)
    x = (rng.standard_normal((rows, vocab + pad)) * 4).astype(f32)
    check(cuda_context, x, rng.integers(0, vocab, rows), top, vocab)


@pytest.mark.parametrize("rows,vocab", [(1, 50000), (9, 3000), (200, 700)])
def test_orders_and_ties(cuda_context, rows, vocab):
    """Rising and falling rows, equal logits, few different ones, both zeros: the lower index stands first."""
    rng = np.random.default_rng(vocab)
    rising = np.broadcast_to(np.linspace(-20, 20, vocab, dtype=f32), (rows, vocab))
    tokens = rng.integers(0, vocab, rows)
    for x in (rising, rising[:, ::-1], np.zeros((rows, vocab), f32), rng.integers(-3, 3, (rows, vocab)).astype(f32),
              np.where(rng.random((rows, vocab)) < 0.5, f32(0.0), f32(-0.0)), np.full((rows, vocab), -np.inf, f32)):
        x = np.array(x)
        if np.isneginf(x).all():
            x[:, vocab // 3] = 2.0                    # one token is left, and probability 1 is its
        check(cuda_context, x, tokens, 32)


@pytest.mark.parametrize("vocab", [40, 5000, 70001])
def test_masked_and_special_logits(cuda_context, vocab):
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((12, vocab)).astype(f32)
    x[0] = -np.inf                                   # nothing is left
    x[1, rng.random(vocab) < 0.9] = -np.inf
    x[2, :] = -np.inf
    x[2, -1] = 5                                     # less than `top` are left
    x[3, vocab // 2] = np.nan
    x[4, 7] = np.inf
    x[5, [3, 9]] = np.nan
    x[6] = np.finfo(f32).min                         # masks of the type's lowest value
    x[7, 1:] = np.finfo(f32).min
    x[8] *= 1e30
    x[9, ::2] = -np.inf
    x[10] = 1e-40
    x[11] = np.finfo(f32).max
    tokens = np.array([0, 1, vocab - 1, 3, 7, 9, 2, 0, 5, 2, 4, vocab - 2])
    check(cuda_context, x, tokens, 10)


def test_tokens_out_of_range_have_no_probability(cuda_context):
    x = np.random.default_rng(0).standard_normal((5, 300)).astype(f32)
    check(cuda_context, x, np.array([-1, 300, 299, 2 ** 31 - 1, -2 ** 31]), 2)


def test_entropy_of_peaked_and_flat_rows(cuda_context):
    """Nearly all probability on one token: the entropy is small and so is its error (a sum just above 1 is rounded to 2^-24, and
    1 itself is exact)."""
    n = 1000
    x = np.zeros((3, n), f32)
    x[0, 5], x[1, 5] = 40, 15
    ts = dev(cuda_context, x)
    _, entropy, _, _ = cuda_context.token_logprobs(ts)
    want = reference(x, np.zeros(3, int), 0)[1]
    assert (np.abs(entropy.get_data() - want) <= np.array([1e-14, 2.0 ** -22, 2.0 ** -18 * 8])).all()


def test_parts_are_optional_and_rows_may_be_none(cuda_context):
    ctx = cuda_context
    x = dev(ctx, np.random.default_rng(1).standard_normal((2, 3, 50)).astype(f32))
    out = ctx.token_logprobs(x)
    assert out[0] is None and out[1].dims == [2, 3] and out[2] is None and out[3] is None
    t = dev(ctx, np.zeros((2, 3), np.int32))
    full = ctx.token_logprobs(x, t, 4)
    assert [o.dims for o in full] == [[2, 3], [2, 3], [2, 3, 4], [2, 3, 4]]
    only = ctx.token_logprobs(x, t, 4, out=(None, None, full[2], full[3]))
    assert only[0] is None
    none = ctx.token_logprobs(ctx.empty_tensor([0, 50]), ctx.empty_tensor([0], "int32"), 2)
    assert [o.dims for o in none] == [[0], [0], [0, 2], [0, 2]]
    ctx.sync()


def test_refusals(cuda_context):
    ctx = cuda_context
    x, t = ctx.empty_tensor([2, 64]), ctx.empty_tensor([2], "int32")
    for bad in (dict(top=33), dict(top=-1), dict(vocab=65), dict(vocab=0)):
        with pytest.raises(ValueError):
            ctx.token_logprobs(x, t, **bad)
    with pytest.raises(TypeError):
        ctx.token_logprobs(t, t)
    with pytest.raises(TypeError):
        ctx.token_logprobs(x, x)
    with pytest.raises(ValueError):
        ctx.token_logprobs(x, t, 1, out=(t, t, t, t))
    p = lambda a: c_void_p(a.ptr)  # noqa: E731
    for d, args in ((LogprobsDesc(2, 64, 64, 33), [p(x), p(t), p(x), p(x), p(t), p(x)]),
                    (LogprobsDesc(2, 0, 64, 0), [p(x), p(t), p(x), None, None, None]),
                    (LogprobsDesc(-1, 64, 64, 0), [p(x), p(t), p(x), None, None, None]),
                    (LogprobsDesc(2, 64, -64, 0), [p(x), p(t), p(x), None, None, None]),
                    (LogprobsDesc(2, 64, 64, 0), [None, p(t), p(x), None, None, None]),
                    (LogprobsDesc(2, 64, 64, 0), [p(x), None, p(x), None, None, None]),
                    (LogprobsDesc(2, 64, 64, 1), [p(x), p(t), p(x), None, p(t), None])):
        with pytest.raises(CudaBackendError) as e:
            ctx._call("wdc_token_logprobs", byref(d), *args)
        assert e.value.status == 1
    ctx.sync()


@pytest.mark.parametrize("vocab,top", [(1, 1), (5, 5), (32, 32), (40, 10), (5000, 32), (70001, 7)])
def test_nan_at_the_first_logit(cuda_context, vocab, top):
    """The first logit can be the one that is no number, alone or among others; every place of the order is somebody's."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((6, vocab)).astype(f32)
    x[:5, 0] = np.nan
    x[1] = np.nan
    x[2, -1] = np.nan
    x[3, 1:2] = np.inf
    x[4, 1:] = -np.inf
    x[5, 0] = -np.float32(np.nan)
    check(cuda_context, x, rng.integers(0, vocab, 6), top)


@pytest.mark.parametrize("top", [0, 5, 32])
@pytest.mark.parametrize("rows", [300, 450, 900, 1800])
def test_long_rows_of_one_cta_each(cuda_context, rows, top):
    """Rows of many rounds with eight, four, two and one warp: rising (every logit is a candidate), falling, random, mostly masked,
    and with few different logits."""
    rng = np.random.default_rng(rows)
    vocab = 20001                                    # (rows begin at every place between two 16-byte boundaries)
    x = rng.standard_normal((10, vocab)).astype(f32) * 3
    x[0] = np.linspace(-20, 20, vocab, dtype=f32)
    x[1] = x[0, ::-1]
    x[2] = np.arange(vocab) // 7 * f32(1e-3)
    x[3, rng.random(vocab) < 0.999] = -np.inf
    x[4, 100:] = -np.inf
    x[5] = rng.integers(-3, 3, vocab)
    x[6, :vocab // 2] -= 50                          # the best are behind all that the first rounds kept
    of = np.arange(rows) % len(x)
    tokens = rng.integers(0, vocab, len(x))
    logprob, entropy, ids, best, _ = reference(x, tokens, top)
    ts = [dev(cuda_context, x[of]), dev(cuda_context, tokens[of].astype(np.int32))]
    got = cuda_context.token_logprobs(*ts, top)
    near(got[0].get_data(), logprob[of], 1)
    near(got[1].get_data(), entropy[of], (1 + np.log(vocab) + entropy)[of])
    if top:
        assert np.array_equal(got[2].get_data().reshape(rows, top), ids[of])
        near(got[3].get_data().reshape(rows, top), best[of], 1)
    for t in ts + [t for t in got if t is not None]:
        t.dispose()
