"""Sampling on the GPU against a plain implementation in 64 bits.

Weights differ from the plain ones by 2^-43 of each and sums in their order: a
choice differs where a uniform value lies that near a token's border, which no
case here does (a border is hit with probability about 2^-25 at 300001 tokens and
2^-19 at 2^24).
"""
from __future__ import annotations

import math
from fractions import Fraction

import numpy as np
import pytest

from runtime_amd import hiptime
from runtime_amd.backend import ExecutorError, HipBackend

pytestmark = pytest.mark.gpu


def say(*words):
    print(*words, flush=True)


def token(logits, u, temperature, top_k, top_p, min_p, admitted=None):
    x = logits.astype(np.float64)
    if admitted is not None:
        x = np.where(admitted, x, -np.inf)
    if np.any(np.isnan(x)) or np.any(x == np.inf) or np.all(x == -np.inf):
        return np.nan
    if temperature == 0.0:
        return float(np.argmax(x))
    with np.errstate(over="ignore"):
        weight = np.exp((x - x.max()) / temperature)
    order = np.argsort(-x, kind="stable")
    if top_k:
        order = order[:int(top_k)]
    reached = np.cumsum(weight[order])
    order = order[:1 + np.searchsorted(reached[:-1], top_p * reached[-1], side="left")]
    order = np.sort(order[weight[order] >= min_p])
    reached = np.cumsum(weight[order])
    return float(order[np.searchsorted(reached, u * reached[-1], side="right")])


def run(backend, logits, uniforms, params, mask=None):
    logits = np.asarray(logits, np.float32)
    out = backend.allocate_f32((len(logits),))
    backend.sample_rows(out, backend.upload_f32(logits.shape, logits),
                        backend.upload_f32((len(logits),), uniforms),
                        backend.upload_f32(np.shape(params), params),
                        None if mask is None else
                        backend.upload_u8_classified(mask.shape, mask))
    return backend.read(out)


def check(backend, logits, uniforms, params, admitted=None):
    logits = np.asarray(logits, np.float32)
    uniforms = np.asarray(uniforms, np.float32)
    params = np.asarray(params, np.float32)
    mask = None
    if admitted is not None:
        mask = np.packbits(admitted, axis=1, bitorder="little")
    got = run(backend, logits, uniforms, params, mask)
    rows = len(logits)
    each = np.broadcast_to(params.astype(np.float64), (rows, 4))
    allowed = [None] * rows if admitted is None else np.broadcast_to(admitted, logits.shape)
    want = [token(l, float(u), *p, a) for l, u, p, a in zip(logits, uniforms, each, allowed)]
    assert np.array_equal(got, np.array(want, np.float32), equal_nan=True), (
        [(i, g, w) for i, (g, w) in enumerate(zip(got, want)) if not (g == w)][:5])


SETTINGS = {"all": (1.0, 0, 1.0, 0.0), "greedy": (0.0, 5, 0.5, 0.1), "hot": (1.7, 0, 1.0, 0.0),
            "k1": (0.8, 1, 1.0, 0.0), "k50": (0.8, 50, 1.0, 0.0), "k900": (1.2, 900, 1.0, 0.0),
            "p": (0.9, 0, 0.9, 0.0), "p0": (0.9, 0, 0.0, 0.0), "p-low": (1.3, 0, 0.05, 0.0),
            "p-high": (2.0, 0, 0.999, 0.0), "min": (1.1, 0, 1.0, 0.05),
            "min1": (1.1, 0, 1.0, 1.0), "kp": (0.7, 64, 0.95, 0.0),
            "everything": (0.9, 300, 0.97, 0.002), "cold": (0.01, 40, 0.9, 0.0),
            "k-wide": (1.0, 10 ** 6, 0.8, 0.0), "k5000": (3.0, 5000, 0.9, 0.0)}


@pytest.mark.parametrize("rounded", [False, True], ids=["", "ties"])
@pytest.mark.parametrize("width", [1, 2, 63, 64, 65, 1000, 4096, 65536, 65537, 130003])
@pytest.mark.parametrize("name", list(SETTINGS))
def test_settings(backend, name, width, rounded):
    say("sample", name, width, rounded)
    rng = np.random.default_rng(width + 7 * len(name))
    rows = 6 if width < 5000 else 3
    logits = 2.5 * rng.standard_normal((rows, width))
    logits[:, ::max(1, width // 20)] += 5
    if rounded:
        logits = np.round(logits * 4) / 4
    uniforms = rng.random(rows).astype(np.float32)
    uniforms[0] = 0.0
    uniforms[-1] = np.float32(1 - 2.0 ** -24)
    check(backend, logits, uniforms, [SETTINGS[name]])


@pytest.mark.parametrize("rounded", [False, True], ids=["", "ties"])
@pytest.mark.parametrize("width", [131072, 131073, 300001])
@pytest.mark.parametrize("name", list(SETTINGS))
def test_wide_rows(backend, name, width, rounded):
    """Rows that are coded in several pieces; with half of the tokens admitted too."""
    say("wide", name, width, rounded)
    rng = np.random.default_rng(width + 5 * len(name))
    logits = 2.5 * rng.standard_normal((2, width))
    logits[:, ::width // 20] += 5
    if rounded:
        logits = np.round(logits * 4) / 4
    uniforms = rng.random(2).astype(np.float32)
    check(backend, logits, uniforms, [SETTINGS[name]])
    check(backend, logits, uniforms, [SETTINGS[name]], rng.random((2, width)) < 0.5)


@pytest.mark.parametrize("name", ["all", "greedy", "k50", "p", "min"])
def test_the_widest_row(backend, name):
    say("widest", name)
    rng = np.random.default_rng(41)
    logits = rng.standard_normal((1, 1 << 24), dtype=np.float32) * 2
    check(backend, logits, [0.73], [SETTINGS[name]])


def test_rows_have_their_own_settings(backend):
    rng = np.random.default_rng(1)
    params = np.array(list(SETTINGS.values()) * 9, np.float32)
    check(backend, 3 * rng.standard_normal((len(params), 2047)), rng.random(len(params)), params)


@pytest.mark.parametrize("name", list(SETTINGS))
@pytest.mark.parametrize("value", [0.0, -3.4028235e38, 3.4028235e38, -0.0, 1e-40])
def test_equal_logits(backend, value, name):
    """Every token ties: the first ones by index are kept."""
    rng = np.random.default_rng(2)
    logits = np.full((4, 3001), value, np.float32)
    check(backend, logits, rng.random(4), [SETTINGS[name]])


@pytest.mark.parametrize("name", list(SETTINGS))
def test_zeros_of_both_signs_tie(backend, name):
    rng = np.random.default_rng(3)
    logits = np.where(rng.random((8, 777)) < 0.5, 0.0, -0.0)
    check(backend, logits, rng.random(8), [SETTINGS[name]])


@pytest.mark.parametrize("name", list(SETTINGS))
def test_masked_tokens(backend, name):
    """Logits of -infinity and of the lowest value, and a mask; what the mask
    leaves out may hold anything."""
    say("masked", name)
    rng = np.random.default_rng(4)
    logits = 2 * rng.standard_normal((6, 1501))
    logits[rng.random(logits.shape) < 0.3] = -np.inf
    logits[rng.random(logits.shape) < 0.3] = -3.4028235e38
    uniforms = rng.random(6)
    check(backend, logits, uniforms, [SETTINGS[name]])
    for rows in (1, 6):
        admitted = rng.random((rows, 1501)) < 0.2
        admitted[:, 3] = True
        wild = logits.copy()
        wild[:, 3] = 1.0
        wild[:, ~admitted.any(axis=0)] = np.nan
        check(backend, wild, uniforms, [SETTINGS[name]], admitted)
    only = np.zeros((1, 1501), bool)
    only[0, 1500] = True
    logits[:, 1500] = -3.0
    check(backend, logits, uniforms, [SETTINGS[name]], only)


def test_logits_far_apart(backend):
    logits = np.full((3, 300), -3.4028235e38, np.float32)
    logits[0, 7], logits[1, 9], logits[2, 11] = 3.4028235e38, 1e-38, -3.4e38
    for name in ("all", "p", "kp", "cold", "hot"):
        check(backend, logits, [0.0, 0.5, 0.999], [SETTINGS[name]])


def test_bad_rows_give_nan(backend):
    rng = np.random.default_rng(5)
    logits = rng.standard_normal((14, 100)).astype(np.float32)
    logits[0, 50], logits[1, 99], logits[2] = np.nan, np.inf, -np.inf
    uniforms = np.full(14, 0.5, np.float32)
    uniforms[3], uniforms[4], uniforms[5] = 1.0, -0.1, np.nan
    params = np.tile(np.array([1.0, 10, 0.9, 0.1], np.float32), (14, 1))
    params[6, 0], params[7, 0], params[8, 1], params[9, 1] = -1, np.inf, 1.5, -1
    params[10, 2], params[11, 3], params[12, 1] = 1.5, np.nan, np.nan
    got = run(backend, logits, uniforms, params)
    assert np.all(np.isnan(got[:13])) and got[13] == token(logits[13], 0.5, 1.0, 10,
                                                           float(np.float32(0.9)),
                                                           float(np.float32(0.1)))
    nothing = np.zeros((1, 13), np.uint8)
    assert np.all(np.isnan(run(backend, logits, uniforms, params, nothing)))


def test_the_whole_range_of_uniforms(backend):
    """Every token is chosen by the uniforms of its weight."""
    logits = np.log(np.array([[1, 2, 3, 4, 0.5, 5.5]], np.float64)).repeat(256, axis=0)
    uniforms = (np.arange(256) + 0.5) / 256
    check(backend, logits, uniforms, [(1.0, 0, 1.0, 0.0)])
    check(backend, logits, uniforms, [(1.0, 4, 0.9, 0.0)])


def test_no_rows(backend):
    assert run(backend, np.zeros((0, 5)), np.zeros(0), np.ones((1, 4))).shape == (0,)


def test_refusals(backend):
    f = backend.allocate_f32

    def refused(variant, out, logits, uniforms, params, mask=None):
        with pytest.raises(ExecutorError) as error:
            backend.sample_rows(out, logits, uniforms, params, mask)
        assert error.value.variant == variant, error.value

    ok = f((3,)), f((3, 10)), f((3,)), f((1, 4))
    refused("InvalidShape", f((2,)), *ok[1:])
    refused("InvalidShape", ok[0], f((30,)), *ok[2:])
    refused("Unsupported", ok[0], f((3, 0)), *ok[2:])
    refused("InvalidShape", *ok[:2], f((1,)), ok[3])
    refused("InvalidShape", *ok[:3], f((2, 4)))
    refused("InvalidShape", *ok[:3], f((3, 3)))
    refused("InvalidShape", *ok, backend.upload_u8_classified((1, 3), [1, 2, 3]))
    refused("InvalidShape", *ok, backend.upload_u8_classified((2,), [1, 2]))
    refused("InvalidDType", *ok, f((1, 2)))
    refused("InvalidArgument", ok[2], *ok[1:])
    other = HipBackend(0, owner=9)
    refused("WrongBackend", *ok[:3], other.allocate_f32((1, 4)))
    other.close()


def test_a_model_generates_sampled_tokens(backend):
    """The device loop against its steps one by one, each token checked against
    the logits it was drawn from."""
    from runtime_amd.lfm2 import ATTENTION, CONV, Lfm2Config, Lfm2Model, synthetic_weights

    cfg = Lfm2Config(hidden=256, intermediate=512, attention_heads=4, key_value_heads=2,
                     vocab=1000, layers=[CONV, ATTENTION], max_tokens=64,
                     formats={"embedding": "int8", "conv": "nf4", "attention": "nf4",
                              "ffn": "ternary"})
    model = Lfm2Model(backend, cfg)
    synthetic_weights(model)
    model.append([1, 2, 3, 4, 5])
    prefix = model.snapshot()
    rng = np.random.default_rng(12)
    steps, settings = 9, (0.9, 40, 0.95, 0.01)
    uniforms = rng.random(steps).astype(np.float32)
    params = backend.upload_f32((1, 4), settings)
    for admitted in (None, rng.random(1000) < 0.5):
        mask = None
        if admitted is not None:
            bits = np.packbits(admitted[None], axis=1, bitorder="little")
            mask = backend.upload_u8_classified(bits.shape, bits)
        model.restore(prefix)
        ids = backend.read(model.generate_sampled(steps, backend.upload_f32((steps,), uniforms),
                                                  params, mask))
        assert model.length == 5 + steps
        model.restore(prefix)
        for i in range(steps):
            logits = backend.read(model.logits)[0]
            model.sample_with(backend.upload_f32((1,), uniforms[i:i + 1]), params, mask)
            want = token(logits, float(uniforms[i]), *(float(np.float32(p)) for p in settings),
                         admitted)
            assert backend.read(model.sampled)[0] == ids[i] == want
            model.append(model.sampled)
    model.restore(prefix)
    bad = backend.upload_f32((1, 4), (-1.0, 40, 0.95, 0.01))
    halves = backend.upload_f32((3,), [0.5] * 3)
    assert np.isnan(backend.read(model.generate_sampled(3, halves, bad))).all()
    one = backend.upload_f32((1,), [0.5])
    for variant, call in [
            ("InvalidShape", lambda: model.generate_sampled(3, one, params)),
            ("InvalidShape", lambda: model.generate_sampled(1, one, one)),
            ("InvalidShape", lambda: model.generate_sampled(1, one, params, ids=params)),
            ("InvalidArgument", lambda: model.generate_sampled(1, one, params, ids=one)),
            ("InvalidShape", lambda: model.sample_with(params, params)),
            ("OutOfBounds", lambda: model.generate_sampled(
                60, backend.allocate_f32((60,)), params))]:
        with pytest.raises(ExecutorError) as error:
            call()
        assert error.value.variant == variant, error.value
    model.close()


@pytest.mark.parametrize("k", [0, 10 ** 7], ids=["", "k"])
@pytest.mark.parametrize("exponent,kept", [(-0.6, 0.6), (0.5, 0.75)])
@pytest.mark.parametrize("width", [1 << 20, 1 << 22, 1 << 24])
def test_flat_tails(backend, width, exponent, kept, k):
    """One token and a wide flat tail of tokens of 2^-41 to 2^-37 of its weight, of which
    top-p keeps a part: none is lost for being small.

    The share is found to within e = 2^-41 (2^-38 past 2^20) of the sum, so the tail's
    kept part, a number of equal weights w, to within e / w tokens; the last uniform
    value below one chooses near its end, 2^-24 of the sum before.  A token each for
    the rounding of that number, of the choice and of its sums.
    """
    say("flat", width, exponent, k)
    logits = np.full((1, width), (exponent - 61 + math.log2(width)) * math.log(2), np.float32)
    logits[0, 5] = 0.0
    w = Fraction(math.exp(float(logits[0, 0])))  # within 2^-52 of itself
    tail = (min(width, k) if k else width) - 1
    total = 1 + tail * w
    p = np.float32(float((1 + Fraction(kept) * tail * w) / total))
    u = np.float32(1 - 2.0 ** -24)
    assert p < 1
    goal = Fraction(float(p)) * total
    ties = min(tail, math.ceil((goal - 1) / w))
    want = math.floor((Fraction(float(u)) * (1 + ties * w) - 1) / w) + 1
    assert 1000 < want < ties < tail
    got = run(backend, logits, [u], [(1.0, k, p, 0.0)])[0]
    error = 2.0 ** (-41 if width <= 1 << 20 else -38)
    say("want", want, "got", got)
    assert abs(got - want) <= error / float(w) + 3


@pytest.mark.parametrize("k", [2, 50, 3000])
@pytest.mark.parametrize("temperature", [0.1, 0.05, 0.01, 1e-4, 1e-30])
@pytest.mark.parametrize("width", [2048, 2049, 4097, 65536, 130003])
def test_top_k_keeps_what_weighs_little(backend, width, temperature, k):
    """A uniform value of zero takes the first token of the k, however small its weight:
    what is too small for 64 bits is zero.  (token() would lose tokens that add nothing
    to a sum at top_p = 1, where all are kept.)"""
    say("cold", width, temperature, k)
    rng = np.random.default_rng(width + k)
    logits = 2.5 * rng.standard_normal((6, width))
    logits[1:3] = np.round(logits[1:3] * 4) / 4
    logits[2:4, 100] = 13.0
    logits[3, 37] = 11.9  # e^-11 to e^-110 of the largest at the first three temperatures
    logits[4] = -logits[4] ** 2
    logits = logits.astype(np.float32)
    uniforms = np.float32([0, 0, 0, 0, 0, 1e-30])
    t = float(np.float32(temperature))
    for share in (None, 0.5, 30 / width):
        admitted = np.ones((6, width), bool) if share is None else rng.random((6, width)) < share
        want = []
        for row, u, allowed in zip(logits, uniforms, admitted):
            x = np.where(allowed, row.astype(np.float64), -np.inf)
            kept = np.sort(np.argsort(-x, kind="stable")[:k])
            reached = np.cumsum(np.exp((x[kept] - x.max()) / t))
            want.append(kept[np.searchsorted(reached, float(u) * reached[-1], side="right")])
        got = run(backend, logits, uniforms, [(temperature, k, 1.0, 0.0)],
                  None if share is None else np.packbits(admitted, axis=1, bitorder="little"))
        assert np.array_equal(got, np.float32(want)), (share, got, want)


def test_a_failed_draw_ends_the_loop_before_the_step(backend):
    """An error of a draw's launch (here one that an earlier HIP call of the thread left)
    is the draw's: no step is queued behind it, and the model is where it was."""
    from runtime_amd.lfm2 import ATTENTION, CONV, Lfm2Config, Lfm2Model, synthetic_weights

    cfg = Lfm2Config(hidden=256, intermediate=512, attention_heads=4, key_value_heads=2,
                     vocab=1000, layers=[CONV, ATTENTION], max_tokens=64,
                     formats={"embedding": "int8", "conv": "nf4", "attention": "nf4",
                              "ffn": "ternary"})
    model = Lfm2Model(backend, cfg)
    synthetic_weights(model)
    model.append([1, 2, 3, 4, 5])
    prefix = model.snapshot()
    uniforms = backend.upload_f32((9,), np.random.default_rng(13).random(9).astype(np.float32))
    params = backend.upload_f32((1, 4), (0.9, 40, 0.95, 0.01))
    want = backend.read(model.generate_sampled(9, uniforms, params))
    model.restore(prefix)
    logits = backend.read(model.logits)
    assert hiptime.hip().hipSetDevice(9999) != 0
    with pytest.raises(ExecutorError) as error:
        model.generate_sampled(9, uniforms, params)
    assert error.value.variant == "BackendFailure" and "sampling" in str(error.value)
    assert model.length == 5
    assert np.array_equal(backend.read(model.logits), logits)
    assert np.array_equal(backend.read(model.generate_sampled(9, uniforms, params)), want)
    model.close()
