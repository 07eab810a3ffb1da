"""Paged caches on the GPU: rotation tables, the entry of new tokens, attention
of single tokens, page copies, and a decode loop of all of them, against plain
implementations in 64 bits.

Tolerances count roundings: half a step of f32 is 2^-24 of a value, of binary16
2^-11.
"""
from __future__ import annotations

import ctypes
import math
import time

import numpy as np
import pytest

from runtime_amd import hiptime
from runtime_amd.backend import (CACHE, ExecutorError, CacheLength, GqaSpec, HipBackend, Limits,
                                 PackedHeadSpec, PagedRopeSpec, RopeScaling, RotarySpec)

pytestmark = pytest.mark.gpu

EPSILON = 1.0e-5
F32, F16 = 2.0 ** -24, 2.0 ** -11


def say(*words):
    print(*words, flush=True)


def upload(backend, array):
    array = np.asarray(array)
    if array.dtype == np.float16:
        shape = array.shape[:-1] + (2 * array.shape[-1],)
        return backend.upload_u8_classified(shape, np.ascontiguousarray(array).view(np.uint8),
                                            CACHE)
    return backend.upload_f32(array.shape, array)


def read_pages(backend, buffer):
    """A page buffer's values as f32."""
    if buffer.dtype == 0:
        return backend.read(buffer)
    pages, heads, size, width = buffer.shape
    wide = backend.alloc_pages(pages, heads, size, width // 2)
    backend.copy_pages([wide], [buffer], range(pages), range(pages))
    return backend.read(wide)


def random_pages(rng, pages, heads, size, dim, half):
    values = rng.standard_normal((pages, heads, size, dim)).astype(np.float32)
    return values.astype(np.float16) if half else values


def tables_for(rng, lengths, size, columns=None, spare=1):
    """(page count, table): distinct pages in random order, others name none."""
    need = [-(-int(n) // size) for n in lengths]
    columns = columns if columns is not None else max(1, max(need, default=1))
    order = rng.permutation(sum(need) + spare)
    table = np.full((len(lengths), columns), -7.0, np.float32)
    at = 0
    for row, n in zip(table, need):
        row[:n] = order[at:at + n]
        at += n
    return sum(need) + spare, table


# ---- rotation tables --------------------------------------------------------------

def frequencies(dim, theta, s):
    f = theta ** (-2.0 * np.arange(dim // 2) / dim)
    if s is None or s.kind == "none":
        return f
    if s.kind == "linear":
        return f / s.factor
    if s.kind == "ntk":
        return (theta * s.factor ** (dim / (dim - 2))) ** (-2.0 * np.arange(dim // 2) / dim)
    if s.kind == "wavelength":
        turns = s.original_positions * f / (2 * math.pi)
        blend = np.clip((turns - s.low) / (s.high - s.low), 0, 1)
        return blend * f + (1 - blend) * f / s.factor
    at = lambda n: dim * math.log(s.original_positions / (2 * math.pi * n)) / (  # noqa: E731
        2 * math.log(theta))
    first, last = max(math.floor(at(s.high)), 0), min(math.ceil(at(s.low)), dim - 1)
    ramp = np.clip((np.arange(dim // 2) - first) / (last - first if last > first else 0.001), 0, 1)
    return f * (1 - ramp) + f / s.factor * ramp


SCALINGS = [None, RopeScaling("none", magnitude=0.75), RopeScaling("linear", 4.0),
            RopeScaling("ntk", 8.0),
            RopeScaling("wavelength", 8.0, 8192.0, 1.0, 4.0),
            RopeScaling("yarn", 16.0, 4096.0, 1.0, 32.0, magnitude=1.25)]


@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: s.kind if s else "null")
@pytest.mark.parametrize("positions,dim", [(1, 2), (7, 64), (1000, 36), (131075, 14),
                                           (3, 130)])
def test_rotation_table(backend, positions, dim, scaling):
    say("rotation", positions, dim, scaling)
    if scaling is not None and scaling.kind == "ntk" and dim == 2:
        dim = 4
    theta = float(np.float32(1.0e6 / 3))
    out = backend.allocate_f32((positions, dim))
    backend.rotation_table(out, theta, scaling)
    got = backend.read(out)
    angle = np.arange(positions, dtype=np.float64)[:, None] * frequencies(dim, theta, scaling)
    magnitude = scaling.magnitude if scaling else 1.0
    want = magnitude * np.concatenate([np.cos(angle), np.sin(angle)], axis=1)
    # One rounding of a value, and 64-bit angles of up to 2^17 (2^-53 each).
    assert np.all(np.abs(got - want) <= F32 * np.abs(want) + 1e-9 * magnitude)


def test_rotation_table_of_no_positions(backend):
    out = backend.allocate_f32((0, 8))
    backend.rotation_table(out, 1.0e4)
    assert backend.read(out).shape == (0, 8)


# ---- new tokens into the caches ------------------------------------------------------

def head_turn(x, weight, turn, pairs, interleaved):
    """[tokens, heads, d] in 64 bits; turn [tokens, 2 * pairs]."""
    x = x.astype(np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(EPSILON))) * weight
    first = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    second = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    cosine, sine = turn[:, None, :pairs], turn[:, None, pairs:]
    a, b = x[..., first].copy(), x[..., second].copy()
    x[..., first], x[..., second] = a * cosine - b * sine, b * cosine + a * sine
    return x


def near(got, want, x, half):
    """Elementwise: a pair's products of normed values (each about 4 + d / 64
    roundings of sums, root and products off, bounded by 16), and the store."""
    scale = np.abs(want) + np.abs(x).max(-1, keepdims=True)
    bound = 16 * F32 * scale + (F16 * np.abs(want) + 2.0 ** -25 if half else 0.0)
    assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) / bound)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary,size,norm", [
    (1, 32, 8, 64, 64, 16, True), (5, 16, 8, 64, 32, 8, True), (37, 6, 3, 80, 80, 32, True),
    (3, 4, 1, 128, 64, 16, False), (9, 2, 2, 2, 2, 8, True), (2, 3, 1, 250, 126, 64, True),
    (130, 8, 4, 128, 128, 256, True), (4, 4, 4, 96, 0, 16, True), (6, 5, 5, 7, 4, 8, False),
    (2, 8, 1, 1024, 256, 8, True)])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
def test_tokens_enter_the_caches(backend, tokens, heads, kv_heads, dim, rotary, size, norm,
                                 interleaved, half):
    say("append", tokens, heads, kv_heads, dim, rotary, size, norm, interleaved, half)
    rng = np.random.default_rng(tokens * 1000 + dim + half)
    # Three sequences; the last third of the tokens is padding or has bad ids.
    sequences = rng.integers(0, 3, tokens)
    positions = np.zeros(tokens, np.float32)
    count = [0, 0, 0]
    for t, s in enumerate(sequences):
        positions[t] = count[s] + 5 * s
        count[s] += 1
    limit = int(positions.max()) + 2
    pages, table = tables_for(rng, [limit] * 3, size)
    bad = {}
    if tokens > 4:
        bad = {tokens - 1: (-1.0, None), tokens - 2: (float("nan"), None),
               tokens - 3: (float(limit), None), tokens - 4: (0.5, 2.0)}
    ids = sequences.astype(np.float32)
    for t, (position, sequence) in bad.items():
        positions[t] = position
        if sequence is not None:
            ids[t] = sequence
    x = {n: rng.standard_normal((tokens, h * dim)).astype(np.float32) * 3
         for n, h in (("q", heads), ("k", kv_heads), ("v", kv_heads))}
    w = {n: (1 + 0.1 * rng.standard_normal(dim)).astype(np.float32) if norm else None
         for n in "qk"}
    turn = rng.standard_normal((limit, rotary)).astype(np.float32)
    old = {n: random_pages(rng, pages, kv_heads, size, dim, half) for n in "kv"}
    cache = {n: upload(backend, old[n]) for n in "kv"}
    out = backend.allocate_f32((tokens, heads * dim))
    backend.paged_qk_norm_rope(
        out, cache["k"], cache["v"], *(upload(backend, x[n]) for n in "qkv"),
        *(None if w[n] is None else upload(backend, w[n]) for n in "qk"),
        upload(backend, turn), upload(backend, table), upload(backend, ids),
        upload(backend, positions), PagedRopeSpec(heads, kv_heads, dim, interleaved), EPSILON)
    good = np.array([t not in bad for t in range(tokens)])
    at = np.where(good, positions, 0).astype(int)
    split = {n: v.reshape(tokens, -1, dim) for n, v in x.items()}
    want = {n: head_turn(split[n], w[n], turn[at], rotary // 2, interleaved) for n in "qk"}
    got = backend.read(out).reshape(tokens, heads, dim)
    assert np.all(np.isnan(got[~good]))
    size_of = lambda n: (head_turn(split[n], w[n], turn[at][:, :0], 0, False)  # noqa: E731
                         * max(1.0, np.abs(turn).max(initial=0.0)) * 2)
    near(got[good], want["q"][good], size_of("q")[good], False)
    touched = np.zeros((pages, size), bool)
    for n in "kv":
        now = read_pages(backend, cache[n])
        for t in np.flatnonzero(good):
            page, slot = int(table[sequences[t], at[t] // size]), at[t] % size
            touched[page, slot] = True
            if n == "v":
                assert np.array_equal(now[page, :, slot], split["v"][t].astype(old["v"].dtype))
            else:
                near(now[page, :, slot], want["k"][t], size_of("k")[t], half)
        untouched = np.broadcast_to(~touched[:, None, :, None], now.shape)
        assert np.array_equal(now[untouched], old[n].astype(np.float32)[untouched])


def test_token_rows_are_sequences_without_ids(backend):
    rng = np.random.default_rng(3)
    q, k, v = (rng.standard_normal((4, 2 * 16)).astype(np.float32) for _ in range(3))
    keys, values = (backend.alloc_pages(9, 2, 8, 16) for _ in range(2))
    table = np.array([[1, 5], [8, 2], [3, 9], [float("inf"), 4]], np.float32)
    positions = np.array([0, 15, 8, 3], np.float32)  # page 9 and infinity are none
    out = backend.allocate_f32((4, 32))
    turn = np.concatenate([np.ones((16, 8)), np.zeros((16, 8))], axis=1).astype(np.float32)
    backend.paged_qk_norm_rope(out, keys, values, *(upload(backend, a) for a in (q, k, v)), None,
                               None, upload(backend, turn), upload(backend, table), None,
                               upload(backend, positions), PagedRopeSpec(2, 2, 16), EPSILON)
    got = backend.read(out)
    assert np.array_equal(got[:2], q[:2]) and np.all(np.isnan(got[2:]))
    want = np.zeros((9, 2, 8, 16), np.float32)
    want[1, :, 0], want[2, :, 7] = k[0].reshape(2, 16), k[1].reshape(2, 16)
    assert np.array_equal(backend.read(keys), want)


def test_binary16_caches_saturate(backend):
    value = np.array([1e30, -1e30, 65504.0, 65519.0, 65520.0, 2.0 ** -24, 2.0 ** -25 * 1.01, 0.1,
                      float("inf"), -float("inf"), float("nan"), 1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11,
                      -0.0, 1e-30, 3.0], np.float32)
    keys, values = (backend.alloc_pages(1, 1, 8, 16, half=True) for _ in range(2))
    out = backend.allocate_f32((1, 16))
    ones = upload(backend, np.ones((1, 16), np.float32))
    backend.paged_qk_norm_rope(out, keys, values, ones, ones, upload(backend, value[None]), None,
                               None, backend.allocate_f32((1, 0)),
                               upload(backend, np.zeros((1, 1), np.float32)), None,
                               upload(backend, np.zeros(1, np.float32)), PagedRopeSpec(1, 1, 16),
                               EPSILON)
    got = read_pages(backend, values)[0, 0, 0]
    with np.errstate(over="ignore"):
        want = value.astype(np.float16).astype(np.float32)
    want[[0, 4]], want[1] = 65504.0, -65504.0
    assert np.array_equal(got, want, equal_nan=True)


# ---- attention over pages -------------------------------------------------------------

def attend(query, keys, values, table, lengths, heads):
    """In 64 bits: (outputs, the bound of their error)."""
    n = len(lengths)
    _, kv_heads, size, dim = keys.shape
    group = heads // kv_heads
    out, bound = np.zeros((n, heads, dim)), np.zeros((n, heads, dim))
    query = query.reshape(n, heads, dim).astype(np.float64)
    for i, length in enumerate(lengths):
        length = int(length)
        if not length:
            continue
        ids = table[i, :-(-length // size)].astype(int)
        for h in range(kv_heads):
            key = keys[ids, h].reshape(-1, dim)[:length].astype(np.float64)
            value = values[ids, h].reshape(-1, dim)[:length].astype(np.float64)
            for g in range(h * group, (h + 1) * group):
                score = key @ query[i, g] / math.sqrt(dim)
                p = np.exp(score - score.max())
                p /= p.sum()
                out[i, g] = p @ value
                # A score's error: dim products and sums, scale and exponent
                # (8 more); it moves numerator and denominator.  Then the
                # weighted sums: the keys of a tile and the tiles of a part.
                size_of = (np.abs(key) @ np.abs(query[i, g])).max() / math.sqrt(dim)
                relative = 2 * (dim + 8) * F32 * size_of + (64 + length / 64 + 32) * F32
                bound[i, g] = relative * (p @ np.abs(value)) + 2.0 ** -40
    return out.reshape(n, -1), bound.reshape(n, -1)


def run_attention(backend, query, keys, values, table, lengths, heads, kv_heads, dim):
    out = upload(backend, np.full(query.shape, 7.0, np.float32))
    backend.paged_gqa(out, upload(backend, query), upload(backend, keys), upload(backend, values),
                      upload(backend, table), upload(backend, np.asarray(lengths, np.float32)),
                      GqaSpec(heads, kv_heads, dim))
    return backend.read(out)


LENGTHS = {"one": [1], "none": [0], "mixed": [0, 1, 15, 16, 17, 31, 32, 33, 0, 63, 64, 65, 127,
                                              128, 129, 300],
           "long": [4099], "ragged": [1, 2500, 7, 0, 130, 1025], "ones": [1] * 70}


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim,size", [
    (32, 8, 64, 16), (32, 8, 128, 32), (4, 4, 64, 8), (16, 1, 128, 64), (40, 2, 64, 16),
    (6, 2, 80, 16), (8, 2, 96, 8), (3, 1, 256, 128), (8, 4, 32, 256), (5, 5, 16, 16),
    (6, 3, 20, 8), (2, 1, 7, 16), (2, 2, 1, 8), (2, 1, 1000, 16), (34, 1, 130, 32),
    (9, 3, 112, 64), (2, 2, 144, 16)])
@pytest.mark.parametrize("which", list(LENGTHS))
def test_attention_over_pages(backend, which, heads, kv_heads, dim, size, half):
    lengths = LENGTHS[which]
    say("attend", which, heads, kv_heads, dim, size, half)
    rng = np.random.default_rng(dim * 31 + size + len(lengths) + half)
    pages, table = tables_for(rng, lengths, size)
    keys, values = (random_pages(rng, pages, kv_heads, size, dim, half) for _ in range(2))
    # Pages end behind the lengths in values that must not matter.
    for i, length in enumerate(lengths):
        if length % size:
            page, row = int(table[i, length // size]), length % size
            keys[page, :, row:], values[page, :, row:] = np.nan, np.inf
    query = rng.standard_normal((len(lengths), heads * dim)).astype(np.float32) * 2
    got = run_attention(backend, query, keys, values, table, lengths, heads, kv_heads, dim)
    want, bound = attend(query, keys, values, table, lengths, heads)
    assert np.all(np.abs(got - want) <= bound), np.nanmax(np.abs(got - want) / (bound + 1e-30))
    again = run_attention(backend, query, keys, values, table, lengths, heads, kv_heads, dim)
    assert np.array_equal(got, again)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 20])
def test_many_ragged_sequences(backend, dim, half):
    """More sequences than a block has threads, and more units than blocks."""
    say("many", dim, half)
    rng = np.random.default_rng(dim + half)
    lengths = rng.integers(0, 90, 700)
    lengths[[5, 333]] = 6000, 2222
    pages, table = tables_for(rng, lengths, 16)
    keys, values = (random_pages(rng, pages, 2, 16, dim, half) for _ in range(2))
    query = rng.standard_normal((700, 6 * dim)).astype(np.float32)
    got = run_attention(backend, query, keys, values, table, lengths, 6, 2, dim)
    want, bound = attend(query, keys, values, table, lengths, 6)
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("dim", [64, 20])
@pytest.mark.parametrize("count", [3, 64, 65, 203, 255, 256, 257])
def test_any_count_of_sequences(backend, count, dim):
    """Some without a key, some with an invalid length, the last and first long."""
    say("count", count, dim)
    rng = np.random.default_rng(count + dim)
    lengths = rng.integers(0, 40, count)
    lengths[[0, -1]] = 333, 555
    lengths[rng.random(count) < 0.3] = 0
    pages, table = tables_for(rng, lengths, 16)
    keys, values = (random_pages(rng, pages, 2, 16, dim, True) for _ in range(2))
    query = rng.standard_normal((count, 6 * dim)).astype(np.float32)
    want, bound = attend(query, keys, values, table, lengths, 6)
    given = lengths.astype(np.float32)
    bad = np.arange(1, count, 7)
    given[bad] = np.resize(np.array([-1, 0.5, np.nan, np.inf, 16 * table.shape[1] + 1, 2e7],
                                    np.float32), len(bad))
    got = run_attention(backend, query, keys, values, table, given, 6, 2, dim)
    good = np.setdiff1d(np.arange(count), bad)
    assert np.isnan(got[bad]).all()
    assert np.all(np.abs(got - want)[good] <= bound[good])


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 36])
def test_small_weights_keep_their_precision(backend, dim, half):
    """One key has nearly all the weight and a zero value: the others, at e^-14
    of it, make up the output."""
    say("small", dim, half)
    rng = np.random.default_rng(dim)
    n = 777
    keys, values = (random_pages(rng, 49, 1, 16, dim, half) for _ in range(2))
    table = np.arange(49, dtype=np.float32)[None]
    keys *= 0.01 if not half else np.float16(0.01)
    query = rng.standard_normal((1, dim)).astype(np.float32)
    q = query[0].astype(np.float64)
    keys[20, 0, 3] = (q * 14 * math.sqrt(dim) / (q @ q)).astype(keys.dtype)
    values[20, 0, 3] = 0
    got = run_attention(backend, query, keys, values, table, [n], 1, 1, dim)
    want, bound = attend(query, keys, values, table, [n], 1)
    assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) / bound)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 20])
@pytest.mark.parametrize("scale", [1e-30, 1e-6, 300.0])
def test_queries_and_values_of_any_size(backend, scale, dim, half):
    say("scale", scale, dim, half)
    rng = np.random.default_rng(8)
    keys, values = (random_pages(rng, 20, 2, 16, dim, half) for _ in range(2))
    table = np.arange(20, dtype=np.float32)[None]
    if half:
        keys[3, 0, 5] = 2.0 ** -20  # subnormal there
        values[3, 0, 5] = 3 * 2.0 ** -24
    else:
        values *= np.float32(1 / scale)
    query = (scale * rng.standard_normal((1, 4 * dim))).astype(np.float32)
    query[0, 1] *= 1e-4
    got = run_attention(backend, query, keys, values, table, [319], 4, 2, dim)
    want, bound = attend(query, keys, values, table, [319], 4)
    assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) / bound)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 10])
def test_bad_lengths_and_pages_give_nan_rows(backend, dim, half):
    say("bad", dim, half)
    rng = np.random.default_rng(dim)
    size, columns = 8, 40
    lengths = np.full(12, 200, np.float32)
    lengths[[0, 1, 2, 3, 4, 5]] = -1, 0.5, np.nan, np.inf, 8 * columns + 1, 2.0 ** 25
    lengths[11] = 8 * columns
    pages, table = tables_for(rng, [columns * size] * 12, size)
    bad = {6: (3, -1.0), 7: (24, float(pages)), 8: (0, np.nan), 9: (11, 1.5)}
    for row, (at, value) in bad.items():
        table[row, at] = value
    table[10, 25:] = np.nan  # behind the length: not read
    keys, values = (random_pages(rng, pages, 2, size, dim, half) for _ in range(2))
    query = rng.standard_normal((12, 4 * dim)).astype(np.float32)
    got = run_attention(backend, query, keys, values, table, lengths, 4, 2, dim)
    assert np.all(np.isnan(got[:10]))
    want, bound = attend(query[10:], keys, values, table[10:], lengths[10:], 4)
    assert np.all(np.abs(got[10:] - want) <= bound)


def test_sequences_share_pages(backend):
    rng = np.random.default_rng(4)
    keys, values = (random_pages(rng, 12, 2, 16, 64, False) for _ in range(2))
    table = np.array([[3, 4, 5, 6], [3, 4, 5, 7], [3, 3, 3, 3]], np.float32)
    lengths = [50, 64, 33]
    query = rng.standard_normal((3, 4 * 64)).astype(np.float32)
    got = run_attention(backend, query, keys, values, table, lengths, 4, 2, 64)
    want, bound = attend(query, keys, values, table, lengths, 4)
    assert np.all(np.abs(got - want) <= bound)


def test_no_sequences(backend):
    pages = backend.alloc_pages(1, 1, 8, 64)
    other = backend.alloc_pages(1, 1, 8, 64)
    out, query = backend.allocate_f32((0, 64)), backend.allocate_f32((0, 64))
    backend.paged_gqa(out, query, pages, other, backend.allocate_f32((0, 3)),
                      backend.allocate_f32((0,)), GqaSpec(1, 1, 64))
    out = upload(backend, np.full((2, 64), 7.0, np.float32))
    backend.paged_gqa(out, backend.allocate_f32((2, 64)), pages, other,
                      backend.allocate_f32((2, 0)),
                      upload(backend, np.array([0, 1], np.float32)), GqaSpec(1, 1, 64))
    got = backend.read(out)
    assert np.all(got[0] == 0) and np.all(np.isnan(got[1]))


def test_offsets_past_32_bits(backend):
    """Pages whose elements lie past 2^32, written and read."""
    size, heads, dim = 4096, 8, 128  # 16 MB a page in f32
    pages = 1100                     # 4.6e9 elements
    rng = np.random.default_rng(5)
    keys, values = (backend.alloc_pages(pages, heads, size, dim) for _ in range(2))
    far = [1099, 1030, 2]
    table = np.array([[far[0]], [far[1]], [far[2]]], np.float32)
    new = {n: rng.standard_normal((3, heads * dim)).astype(np.float32) for n in "qkv"}
    out = backend.allocate_f32((3, heads * dim))
    position = np.array([0, 0, 0], np.float32)
    backend.paged_qk_norm_rope(out, keys, values, *(upload(backend, new[n]) for n in "qkv"), None,
                               None, backend.allocate_f32((1, 0)), upload(backend, table), None,
                               upload(backend, position), PagedRopeSpec(heads, heads, dim),
                               EPSILON)
    backend.copy_pages([keys, values], [keys, values], [1099], [1098])
    table[0, 0] = 1098
    result = backend.allocate_f32((3, heads * dim))
    backend.paged_gqa(result, out, keys, values, upload(backend, table),
                      upload(backend, np.ones(3, np.float32)), GqaSpec(heads, heads, dim))
    assert np.array_equal(backend.read(result), new["v"])
    del keys, values


# ---- page copies ------------------------------------------------------------------------

@pytest.mark.parametrize("from_half,to_half", [(False, False), (True, True), (True, False),
                                               (False, True)])
@pytest.mark.parametrize("heads,size,dim", [(8, 16, 64), (3, 8, 7), (1, 128, 130)])
@pytest.mark.parametrize("count,buffers", [(1, 1), (5, 40), (300, 2), (0, 3)])
def test_copy_pages(backend, count, buffers, heads, size, dim, from_half, to_half):
    say("copy", count, buffers, heads, size, dim, from_half, to_half)
    rng = np.random.default_rng(count + dim)
    pages = 2 * count + 3
    source = [random_pages(rng, pages, heads, size, dim, from_half) for _ in range(buffers)]
    target = [random_pages(rng, pages + 1, heads, size, dim, to_half) for _ in range(buffers)]
    froms, tos = rng.integers(0, pages, count), rng.permutation(pages + 1)[:count]
    to = [upload(backend, t) for t in target]
    backend.copy_pages(to, [upload(backend, s) for s in source], froms, tos)
    for i in range(buffers):
        want = target[i].copy()
        want[tos] = source[i][froms].astype(want.dtype)
        assert np.array_equal(read_pages(backend, to[i]), want.astype(np.float32))


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_copy_pages_in_place(backend, half):
    rng = np.random.default_rng(2)
    old = [random_pages(rng, 600, 2, 16, 32, half) for _ in range(2)]
    order = rng.permutation(600)
    froms, tos = order[:290], order[290:580]
    froms[7] = froms[8]  # one page forked twice
    buffers = [upload(backend, o) for o in old]
    backend.copy_pages(buffers, buffers, froms, tos)
    for o, b in zip(old, buffers):
        want = o.copy()
        want[tos] = o[froms]
        assert np.array_equal(read_pages(backend, b), want.astype(np.float32))


# ---- all of them, as a server uses them ---------------------------------------------------

@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_decode_loop_with_a_fork(backend, half):
    """Two prompts, a fork of the first, and six steps of the three sequences,
    captured once and replayed with new positions, against contiguous caches."""
    say("loop", half)
    rng = np.random.default_rng(17 + half)
    heads, kv_heads, dim, size, steps = 8, 2, 64, 16, 6
    spec = PagedRopeSpec(heads, kv_heads, dim)
    w = [upload(backend, (1 + 0.1 * rng.standard_normal(dim)).astype(np.float32))
         for _ in range(2)]
    turn = backend.allocate_f32((128, dim))
    backend.rotation_table(turn, 1.0e6)
    keys, values = (backend.alloc_pages(30, kv_heads, size, dim, half) for _ in range(2))
    order = iter(rng.permutation(30))
    prompts = [37, 50]
    table = np.full((3, 8), -1.0, np.float32)
    for s, n in enumerate(prompts):
        for c in range(-(-(n + steps) // size)):
            table[s, c] = next(order)
    history = [[], [], []]

    def rows(n):
        return [rng.standard_normal((n, h * dim)).astype(np.float32)
                for h in (heads, kv_heads, kv_heads)]

    for s, n in enumerate(prompts):
        new = rows(n)
        out = backend.allocate_f32((n, heads * dim))
        backend.paged_qk_norm_rope(out, keys, values, *(upload(backend, a) for a in new), *w, turn,
                                   upload(backend, table),
                                   upload(backend, np.full(n, s, np.float32)),
                                   upload(backend, np.arange(n, dtype=np.float32)), spec, EPSILON)
        history[s].append(new)
    # The fork shares the whole pages and gets a copy of the page it will write.
    shared = prompts[0] // size
    table[2, :shared] = table[0, :shared]
    table[2, shared] = next(order)
    backend.copy_pages([keys, values], [keys, values], [int(table[0, shared])],
                       [int(table[2, shared])])
    history[2] = [tuple(a.copy() for a in history[0][0])]
    lengths = np.array([prompts[0], prompts[1], prompts[0]], np.float32)

    # One step over fixed buffers; its inputs change between replays.
    buffers = [backend.allocate_f32((3, h * dim)) for h in (heads, kv_heads, kv_heads)]
    positions, one = upload(backend, lengths - 1), upload(backend, np.ones(3, np.float32))
    now = backend.allocate_f32((3,))
    query, out = (backend.allocate_f32((3, heads * dim)) for _ in range(2))
    tables = upload(backend, table)

    def step():
        backend.add(now, positions, one)  # the new token's position
        backend.copy(positions, now)
        backend.paged_qk_norm_rope(query, keys, values, *buffers, *w, turn, tables, None,
                                   positions, spec, EPSILON)
        backend.add(now, positions, one)  # the length with it
        backend.paged_gqa(out, query, keys, values, tables, now, GqaSpec(heads, kv_heads, dim))

    hip, stream = hiptime.hip(), ctypes.c_void_p(backend.stream())
    program, graph = ctypes.c_void_p(), ctypes.c_void_p()
    scratch = backend.allocate_f32((3, heads * dim))  # eager, so that the workspace is there
    backend.paged_gqa(scratch, query, keys, values, tables, now, GqaSpec(heads, kv_heads, dim))
    backend.synchronize()
    hiptime.check(hip.hipStreamBeginCapture(stream, 0), "begin capture")
    try:
        step()
    finally:
        hiptime.check(hip.hipStreamEndCapture(stream, ctypes.byref(graph)), "end capture")
    hiptime.check(hip.hipGraphInstantiate(ctypes.byref(program), graph, None, None,
                                          ctypes.c_size_t(0)), "instantiate")
    for i in range(steps):
        new = rows(3)
        for buffer, a in zip(buffers, new):
            backend.copy(buffer, upload(backend, a))
        hiptime.check(hip.hipGraphLaunch(program, stream), "launch")
        got = backend.read(out)
        for s in range(3):
            history[s].append(tuple(a[s:s + 1] for a in new))
            got_row = got[s]
            # The same sequence over contiguous f32 caches.
            q, k, v = (np.concatenate([h[j] for h in history[s]]) for j in range(3))
            n = len(q)
            turned = [backend.allocate_f32(a.shape) for a in (q, k)]
            backend.qk_norm_rope(*turned, upload(backend, q), upload(backend, k), *w, range(n),
                                 RotarySpec(PackedHeadSpec(heads, dim), 1.0e6),
                                 PackedHeadSpec(kv_heads, dim), EPSILON)
            full = backend.allocate_f32(q.shape)
            caches = [backend.allocate_f32_classified((n, kv_heads * dim), CACHE)
                      for _ in range(2)]
            backend.causal_gqa(full, *turned, upload(backend, v), *caches, CacheLength(0),
                               GqaSpec(heads, kv_heads, dim))
            want = backend.read(full)[-1]
            # Binary16 caches: keys and values each off by 2^-11 of their size;
            # scores are up to |q| |k| / 8 <= 8 * 1.5.  f32: the angles' rounding
            # in the contiguous operation (2^-24 * 56 at most).
            bound = (2 * 12 * F16 + F16 if half else 2 * 12 * 64 * F32) * 4
            assert np.max(np.abs(got_row - want)) <= bound, (i, s, np.max(np.abs(got_row - want)))
    hiptime.check(hip.hipGraphExecDestroy(program), "destroy")
    hiptime.check(hip.hipGraphDestroy(graph), "destroy")


def test_a_captured_workspace_is_kept():
    """A later, larger call does not take the captured call's workspace away."""
    backend = HipBackend(0)
    rng = np.random.default_rng(6)
    keys, values = (random_pages(rng, 200, 2, 16, 64, False) for _ in range(2))
    k, v = upload(backend, keys), upload(backend, values)
    table = np.arange(200, dtype=np.float32)[None]
    query = rng.standard_normal((1, 256)).astype(np.float32)
    q, t = upload(backend, query), upload(backend, table)
    n = upload(backend, np.array([3200], np.float32))
    out = backend.allocate_f32((1, 256))
    spec = GqaSpec(4, 2, 64)
    hip, stream = hiptime.hip(), ctypes.c_void_p(backend.stream())
    graph, program = ctypes.c_void_p(), ctypes.c_void_p()
    hiptime.check(hip.hipStreamBeginCapture(stream, 0), "begin capture")
    with pytest.raises(ExecutorError) as refused:  # no workspace yet
        backend.paged_gqa(out, q, k, v, t, n, spec)
    assert refused.value.variant == "ResourceLimit"
    hiptime.check(hip.hipStreamEndCapture(stream, ctypes.byref(graph)), "end capture")
    hiptime.check(hip.hipGraphDestroy(graph), "destroy")
    backend.paged_gqa(out, q, k, v, t, n, spec)
    want = backend.read(out)
    hiptime.check(hip.hipStreamBeginCapture(stream, 0), "begin capture")
    backend.paged_gqa(out, q, k, v, t, n, spec)
    hiptime.check(hip.hipStreamEndCapture(stream, ctypes.byref(graph)), "end capture")
    hiptime.check(hip.hipGraphInstantiate(ctypes.byref(program), graph, None, None,
                                          ctypes.c_size_t(0)), "instantiate")
    # A call with a larger workspace, then buffers that would take the old one.
    many = 40000
    wide = backend.allocate_f32((many, 256))
    backend.paged_gqa(wide, backend.allocate_f32((many, 256)), k, v,
                      backend.allocate_f32((many, 200)), backend.allocate_f32((many,)), spec)
    taken = [upload(backend, np.full(1 << 18, 5.0, np.float32)) for _ in range(8)]
    for _ in range(3):
        hiptime.check(hip.hipGraphLaunch(program, stream), "launch")
        assert np.array_equal(backend.read(out), want)
        assert all(np.all(backend.read(b) == 5.0) for b in taken)
    hiptime.check(hip.hipGraphExecDestroy(program), "destroy")
    hiptime.check(hip.hipGraphDestroy(graph), "destroy")
    backend.close()


def test_a_workspace_past_the_limit_is_refused():
    """Nothing is written then, and with room the same call works."""
    for limit, variant in ((6 << 20, "ResourceLimit"), (64 << 20, None)):
        backend = HipBackend(0, limits=Limits(max_total_bytes=limit))
        k, v = (backend.alloc_pages(1, 1, 16, 256, half=True) for _ in range(2))
        query = backend.allocate_f32((64, 16 * 256))
        out = upload(backend, np.full((64, 16 * 256), 7.0, np.float32))
        # 64 items of 53 units each: 256 blocks of two records of 16 rows of 256.
        args = (out, query, k, v, backend.allocate_f32((64, 100)),
                upload(backend, np.full(64, 5.0, np.float32)), GqaSpec(16, 1, 256))
        if variant:
            with pytest.raises(ExecutorError) as error:
                backend.paged_gqa(*args)
            assert error.value.variant == variant
            assert np.all(backend.read(out) == 7.0)
        else:
            backend.paged_gqa(*args)
            assert np.all(backend.read(out) == 0.0)
        backend.close()


def captured(backend, call):
    """The call as a graph: (replay, end)."""
    hip, stream = hiptime.hip(), ctypes.c_void_p(backend.stream())
    graph, program = ctypes.c_void_p(), ctypes.c_void_p()
    hiptime.check(hip.hipStreamBeginCapture(stream, 0), "begin capture")
    try:
        call()
    finally:
        hiptime.check(hip.hipStreamEndCapture(stream, ctypes.byref(graph)), "end capture")
    hiptime.check(hip.hipGraphInstantiate(ctypes.byref(program), graph, None, None,
                                          ctypes.c_size_t(0)), "instantiate")

    def replay():
        hiptime.check(hip.hipGraphLaunch(program, stream), "launch")

    def end():
        hiptime.check(hip.hipGraphExecDestroy(program), "destroy")
        hiptime.check(hip.hipGraphDestroy(graph), "destroy")

    return replay, end


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim,size", [
    (16, 1, 256, 16), (17, 1, 256, 8), (66, 2, 64, 32), (20, 1, 80, 4096), (40, 2, 128, 64),
    (9, 1, 1000, 16), (8, 2, 48, 16), (6, 2, 112, 8), (8, 2, 160, 16), (12, 2, 192, 8),
    (12, 2, 192, 64), (18, 1, 16, 8)])
def test_wide_groups(backend, heads, kv_heads, dim, size, half):
    """Groups of query heads that fill a row tile, and pass it by one or more."""
    say("groups", heads, kv_heads, dim, size, half)
    rng = np.random.default_rng(heads + dim)
    lengths = [4097, 1, 0, 130]
    pages, table = tables_for(rng, lengths, size)
    keys, values = (random_pages(rng, pages, kv_heads, size, dim, half) for _ in range(2))
    query = rng.standard_normal((len(lengths), heads * dim)).astype(np.float32)
    got = run_attention(backend, query, keys, values, table, lengths, heads, kv_heads, dim)
    want, bound = attend(query, keys, values, table, lengths, heads)
    assert np.all(np.abs(got - want) <= bound), np.nanmax(np.abs(got - want) / (bound + 1e-30))


def test_a_padded_batch(backend):
    """Rows with position -1 and length 0 around two sequences: nothing enters the
    caches for them and their attention is zeros; a table may name a page twice."""
    rng = np.random.default_rng(23)
    heads, kv_heads, dim, size = 4, 2, 64, 16
    keys, values = (random_pages(rng, 9, kv_heads, size, dim, False) for _ in range(2))
    k, v = upload(backend, keys), upload(backend, values)
    table = np.array([[-1, -1, -1], [4, 7, 4], [0, 2, -1], [np.nan, 1e9, -1]], np.float32)
    positions = np.array([-1, 31, 16, -1], np.float32)
    lengths = np.array([0, 32, 17, 0], np.float32)
    rows = [rng.standard_normal((4, h * dim)).astype(np.float32) for h in (heads, kv_heads, kv_heads)]
    turn = backend.allocate_f32((64, 0))
    query, out = (backend.allocate_f32((4, heads * dim)) for _ in range(2))
    backend.paged_qk_norm_rope(query, k, v, *(upload(backend, a) for a in rows), None, None, turn,
                               upload(backend, table), None, upload(backend, positions),
                               PagedRopeSpec(heads, kv_heads, dim), EPSILON)
    for pages, new in ((keys, rows[1]), (values, rows[2])):
        pages[7, :, 15] = new[1].reshape(kv_heads, dim)
        pages[2, :, 0] = new[2].reshape(kv_heads, dim)
    assert np.array_equal(backend.read(k), keys) and np.array_equal(backend.read(v), values)
    got_query = backend.read(query)
    assert np.array_equal(got_query[1:3], rows[0][1:3]) and np.isnan(got_query[[0, 3]]).all()
    tables = upload(backend, table)
    backend.paged_gqa(out, query, k, v, tables, upload(backend, lengths),
                      GqaSpec(heads, kv_heads, dim))
    alone = backend.allocate_f32((1, heads * dim))
    got = backend.read(out)
    assert np.all(got[[0, 3]] == 0.0)
    for s in (1, 2):
        # As the sequence alone.  Scores are the same products; their distance from
        # the maximum, the exponent and sums of up to 32 terms, on both sides, are
        # under 64 roundings of a mean of values below 5.
        backend.paged_gqa(alone, upload(backend, got_query[s:s + 1]), k, v,
                          upload(backend, table[s:s + 1]), upload(backend, lengths[s:s + 1]),
                          GqaSpec(heads, kv_heads, dim))
        assert np.max(np.abs(backend.read(alone)[0] - got[s])) <= 64 * 5 * F32


def test_a_captured_step_of_everything(backend):
    """Append, attention, a page copy and sampling in one graph; replays with other
    inputs and eager calls between them equal eager calls."""
    rng = np.random.default_rng(29)
    heads, kv_heads, dim, size, rows = 8, 2, 64, 16, 3
    spec, rope = GqaSpec(heads, kv_heads, dim), PagedRopeSpec(heads, kv_heads, dim)
    first = [random_pages(rng, 24, kv_heads, size, dim, True) for _ in range(2)]
    table = rng.permutation(24)[:21].reshape(3, 7).astype(np.float32)
    spare = sorted(set(range(24)) - set(table.astype(int).reshape(-1)))[0]
    turn = backend.allocate_f32((112, dim))
    backend.rotation_table(turn, 1.0e4)
    tables = upload(backend, table)
    params = backend.upload_f32((1, 4), (0.8, 40, 0.9, 0.0))

    def world():
        return {"k": upload(backend, first[0]), "v": upload(backend, first[1]),
                "in": [backend.allocate_f32((rows, h * dim)) for h in (heads, kv_heads, kv_heads)],
                "position": backend.allocate_f32((rows,)), "length": backend.allocate_f32((rows,)),
                "u": backend.allocate_f32((rows,)), "ids": backend.allocate_f32((rows,)),
                "q": backend.allocate_f32((rows, heads * dim)),
                "out": backend.allocate_f32((rows, heads * dim))}

    def step(w):
        backend.paged_qk_norm_rope(w["q"], w["k"], w["v"], *w["in"], None, None, turn, tables,
                                   None, w["position"], rope, EPSILON)
        backend.paged_gqa(w["out"], w["q"], w["k"], w["v"], tables, w["length"], spec)
        backend.copy_pages([w["k"], w["v"]], [w["k"], w["v"]], [int(table[1, 2])], [spare])
        backend.sample_rows(w["ids"], w["out"], w["u"], params)

    eager, graphed = world(), world()
    step(graphed)  # the workspace
    for name, pages in zip("kv", first):
        graphed[name] = upload(backend, pages)
    replay, end = captured(backend, lambda: step(graphed))
    for i in range(5):
        new = [rng.standard_normal((rows, h * dim)).astype(np.float32)
               for h in (heads, kv_heads, kv_heads)]
        position = np.array([3 + i, 37 + i, 100 + i], np.float32)
        u = rng.random(rows).astype(np.float32)
        for w in (eager, graphed):
            for to, a in zip((*w["in"], w["position"], w["length"], w["u"]),
                             (*new, position, position + 1, u)):
                backend.copy(to, upload(backend, a))
        step(eager)
        replay()
        for name in ("out", "ids", "q"):
            assert np.array_equal(backend.read(eager[name]), backend.read(graphed[name])), (i, name)
    end()
    for name in "kv":
        wide = [backend.alloc_pages(24, kv_heads, size, dim) for _ in range(2)]
        backend.copy_pages(wide, [eager[name], graphed[name]], range(24), range(24))
        assert np.array_equal(backend.read(wide[0]), backend.read(wide[1])), name


def test_two_contexts_at_once():
    """Calls of two contexts, queued without waiting, equal each one's alone."""
    rng = np.random.default_rng(31)
    spec = GqaSpec(8, 2, 64)
    keys, values = (random_pages(rng, 300, 2, 16, 64, False) for _ in range(2))
    worlds = []
    for n in (4800, 3333):
        backend = HipBackend(0)
        query = rng.standard_normal((1, 512)).astype(np.float32)
        args = (upload(backend, query), upload(backend, keys), upload(backend, values),
                upload(backend, rng.permutation(300).astype(np.float32)[None]),
                upload(backend, np.array([n], np.float32)))
        alone = backend.allocate_f32((1, 512))
        backend.paged_gqa(alone, *args, spec)
        worlds.append((backend, args, backend.read(alone),
                       [backend.allocate_f32((1, 512)) for _ in range(20)]))
    for i in range(20):
        for backend, args, _, outs in worlds:
            backend.paged_gqa(outs[i], *args, spec)
    for backend, _, want, outs in worlds:
        assert all(np.array_equal(backend.read(out), want) for out in outs)
        backend.close()


# ---- refusals ---------------------------------------------------------------------------------

def refused(variant, call, *args):
    with pytest.raises(ExecutorError) as error:
        call(*args)
    assert error.value.variant == variant, error.value


def test_page_buffer_refusals(backend):
    refused("InvalidShape", backend.alloc_pages, 4, 2, 12, 64)
    refused("InvalidShape", backend.alloc_pages, 4, 2, 4, 64)
    refused("InvalidShape", backend.alloc_pages, 4, 2, 8192, 64)
    refused("InvalidShape", backend.alloc_pages, 0, 2, 16, 64)
    refused("InvalidShape", backend.alloc_pages, 4, 0, 16, 64, True)
    refused("InvalidShape", backend.alloc_pages, 4, 2, 16, 0)


def test_rotation_table_refusals(backend):
    out = backend.allocate_f32((4, 6))
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        refused("InvalidArgument", backend.rotation_table, out, bad)
        refused("InvalidArgument", backend.rotation_table, out, 1e4, RopeScaling("linear", bad))
        refused("InvalidArgument", backend.rotation_table, out, 1e4,
                RopeScaling("none", magnitude=bad))
    refused("InvalidArgument", backend.rotation_table, out, 1e4,
            RopeScaling("yarn", 2.0, 100.0, 4.0, 4.0))
    refused("InvalidArgument", backend.rotation_table, out, 1e4,
            RopeScaling("wavelength", 2.0, 0.0, 1.0, 4.0))
    refused("InvalidArgument", backend.rotation_table, out, 1.0,
            RopeScaling("yarn", 2.0, 100.0, 1.0, 4.0))
    refused("InvalidShape", backend.rotation_table, backend.allocate_f32((4, 5)), 1e4)
    refused("InvalidShape", backend.rotation_table, backend.allocate_f32((4, 0)), 1e4)
    refused("InvalidShape", backend.rotation_table, backend.allocate_f32((4,)), 1e4)
    refused("InvalidShape", backend.rotation_table, backend.allocate_f32((4, 2)), 1e4,
            RopeScaling("ntk", 2.0))


def test_append_refusals(backend):
    f = backend.allocate_f32
    spec = PagedRopeSpec(4, 2, 16)

    def call(**over):
        a = dict(out=f((3, 64)), k=backend.alloc_pages(5, 2, 8, 16),
                 v=backend.alloc_pages(5, 2, 8, 16), q=f((3, 64)), key=f((3, 32)),
                 value=f((3, 32)), qw=f((16,)), kw=f((16,)), rotation=f((9, 16)), tables=f((3, 2)),
                 ids=f((3,)), positions=f((3,)), spec=spec, epsilon=EPSILON)
        a.update(over)
        backend.paged_qk_norm_rope(*a.values())

    call()
    for variant, over in [
            ("InvalidArgument", {"epsilon": 0.0}), ("InvalidArgument", {"qw": None}),
            ("InvalidShape", {"spec": PagedRopeSpec(3, 2, 16)}),
            ("InvalidShape", {"spec": PagedRopeSpec(4, 0, 16)}),
            ("InvalidShape", {"spec": PagedRopeSpec(4, 2, 32)}),
            ("InvalidShape", {"q": f((3, 63))}), ("InvalidShape", {"key": f((2, 32))}),
            ("InvalidShape", {"value": f((3, 31))}), ("InvalidShape", {"qw": f((15,))}),
            ("InvalidShape", {"rotation": f((9, 18))}), ("InvalidShape", {"rotation": f((9, 7))}),
            ("InvalidShape", {"ids": f((2,))}), ("InvalidShape", {"ids": None, "tables": f((2, 2))}),
            ("InvalidShape", {"positions": f((4,))}), ("InvalidShape", {"tables": f((6,))}),
            ("InvalidShape", {"out": f((3, 32))}),
            ("InvalidShape", {"v": backend.alloc_pages(5, 2, 8, 16, True)}),
            ("InvalidShape", {"v": backend.alloc_pages(6, 2, 8, 16)}),
            ("InvalidShape", {"k": f((5, 2, 16))}),
            ("InvalidDType", {"positions": backend.upload_u8_classified((3,), [0, 0, 0])})]:
        say(variant, sorted(over))
        refused(variant, lambda: call(**over))
    same = backend.alloc_pages(5, 2, 8, 16)
    refused("InvalidArgument", lambda: call(k=same, v=same))
    rows = f((3, 64))
    refused("InvalidArgument", lambda: call(out=rows, q=rows))


def test_attention_refusals(backend):
    f = backend.allocate_f32

    def call(**over):
        a = dict(out=f((3, 64)), q=f((3, 64)), k=backend.alloc_pages(5, 2, 8, 16),
                 v=backend.alloc_pages(5, 2, 8, 16), tables=f((3, 2)), lengths=f((3,)),
                 spec=GqaSpec(4, 2, 16))
        a.update(over)
        backend.paged_gqa(*a.values())

    call()
    wide = [backend.alloc_pages(1, 1, 8, 1025) for _ in range(2)]
    for variant, over in [
            ("InvalidShape", {"q": f((2, 64))}), ("InvalidShape", {"lengths": f((2,))}),
            ("InvalidShape", {"tables": f((3,))}), ("InvalidShape", {"out": f((3, 65))}),
            ("InvalidShape", {"spec": GqaSpec(3, 2, 16)}),
            ("InvalidShape", {"spec": GqaSpec(4, 2, 8)}),
            ("InvalidShape", {"k": backend.alloc_pages(5, 2, 8, 16, True)}),
            ("Unsupported", {"k": wide[0], "v": wide[1], "spec": GqaSpec(1, 1, 1025),
                             "q": f((3, 1025)), "out": f((3, 1025))})]:
        say(variant, sorted(over))
        refused(variant, lambda: call(**over))
    rows = f((3, 64))
    refused("InvalidArgument", lambda: call(out=rows, q=rows))
    other = HipBackend(0, owner=2)
    refused("WrongBackend", lambda: call(q=other.allocate_f32((3, 64))))
    other.close()
    backend.request_cancel()
    try:
        refused("Cancelled", backend.paged_gqa, rows, rows, rows, rows, rows, rows,
                GqaSpec(4, 2, 16))
    finally:
        backend.clear_cancel()


def test_host_page_ids_are_not_converted(backend):
    a, b = (backend.alloc_pages(5, 2, 8, 32) for _ in range(2))
    for ids in ([-1], [2 ** 32 + 3], [1.5], np.array([-2]), np.array([2 ** 32], np.uint64)):
        with pytest.raises((ValueError, OverflowError)):
            backend.copy_pages([a], [b], ids, [2])
        with pytest.raises((ValueError, OverflowError)):
            backend.copy_pages([a], [b], [2], ids)
    backend.copy_pages([a], [b], np.array([1], np.int8), (2,))
    backend.copy_pages([a], [b], [], [])


def test_copy_refusals(backend):
    a, b = backend.alloc_pages(5, 2, 8, 16), backend.alloc_pages(7, 2, 8, 16)
    copy = backend.copy_pages
    refused("OutOfBounds", copy, [a], [b], [7], [0])
    refused("OutOfBounds", copy, [a], [b], [0], [5])
    refused("InvalidArgument", copy, [a], [b], [0, 1], [2, 2])
    refused("InvalidArgument", copy, [a], [a], [1], [1])
    refused("InvalidArgument", copy, [a], [a], [1, 2], [2, 3])
    refused("InvalidArgument", copy, [a, a], [b, b], [1], [2])
    refused("InvalidArgument", copy, [a, b], [b, a], [1], [2])
    refused("InvalidShape", copy, [a], [backend.alloc_pages(5, 2, 16, 16)], [1], [2])
    refused("InvalidShape", copy, [a], [backend.allocate_f32((5, 256))], [1], [2])
    copy([], [], [1, 1], [2, 2])
    copy([a], [b], [6, 6], [1, 2])


def test_page_shapes_are_checked_before_room():
    """A bad shape is one at any size, and costs no memory."""
    backend = HipBackend(0, limits=Limits(max_total_bytes=1 << 20))
    big = 1 << 24
    for half in (False, True):
        refused("InvalidShape", backend.alloc_pages, big, 64, 12, 256, half)
        refused("InvalidShape", backend.alloc_pages, big, 64, 8192, 256, half)
        refused("InvalidShape", backend.alloc_pages, big, 0, 8192, 256, half)
        refused("Unsupported", backend.alloc_pages, big + 1, 1, 16, 8, half)
        refused("Overflow", backend.alloc_pages, 1, 1 << 16, 8, 8, half)
        refused("Overflow", backend.alloc_pages, 1, 1, 8, 1 << 16, half)
        refused("ResourceLimit", backend.alloc_pages, big, 64, 16, 256, half)
    backend.close()


@pytest.mark.parametrize("count", [2, 16, 17, 300, 4999])
def test_copied_pages_are_compared_wherever_they_stand(backend, count):
    """A target named twice, or copied from as well, anywhere in lists of any length."""
    rng = np.random.default_rng(count)
    pages = 10000
    a, b = (backend.alloc_pages(pages, 1, 8, 2) for _ in range(2))
    order = rng.permutation(pages)
    source, target = order[:count], order[count:2 * count]
    whole = upload(backend, rng.standard_normal((pages, 16)).astype(np.float32))
    ramp = backend.read(whole)
    cache = backend.upload_f32((pages, 1, 8, 2), ramp.reshape(pages, 1, 8, 2))
    backend.copy_pages([cache], [cache], source, target)
    want = ramp.copy()
    want[target] = ramp[source]
    assert np.array_equal(backend.read(cache).reshape(pages, 16), want)
    for _ in range(4):
        i, j = rng.choice(count, 2, replace=False)
        twice = target.copy()
        twice[i] = twice[j]
        refused("InvalidArgument", backend.copy_pages, [a], [b], source, twice)
        both = target.copy()
        both[i] = source[j]
        refused("InvalidArgument", backend.copy_pages, [a], [a], source, both)
        backend.copy_pages([a], [b], source, both)
    refused("InvalidArgument", backend.copy_pages, [a], [b], np.zeros(pages + 1, np.uint32),
            np.arange(pages + 1) % pages)


def test_a_few_pages_cost_the_same_in_any_cache(backend):
    """The host's part of a two-page copy, in a cache of 8 pages and in one of 2^24, which
    took 13 times as long when the call went over all of its pages."""
    times = []
    for pages in (8, 1 << 24):
        cache = backend.alloc_pages(pages, 1, 8, 2, half=True)
        each = []
        for _ in range(31):
            backend.synchronize()
            begin = time.perf_counter()
            backend.copy_pages([cache], [cache], [0, 1], [pages - 1, pages - 2])
            each.append(time.perf_counter() - begin)
        times.append(sorted(each)[15])
    say("us a call", [1e6 * t for t in times])
    assert times[1] < 5 * times[0]


def test_a_graph_for_each_batch_size():
    """Every size's workspace is larger than the last one's; the ones that the graphs hold
    stay theirs, and together are no larger than the last."""
    backend = HipBackend(0)
    rng = np.random.default_rng(31)
    keys, values = (random_pages(rng, 7, 1, 16, 256, False) for _ in range(2))
    k, v = upload(backend, keys), upload(backend, values)
    spec, graphs = GqaSpec(16, 1, 256), []
    held = 0
    for count in range(24, 172, 8):
        query = rng.standard_normal((count, 16 * 256)).astype(np.float32)
        table = rng.integers(0, 7, (count, 1)).astype(np.float32)
        lengths = rng.integers(1, 17, count).astype(np.float32)
        args = (backend.allocate_f32((count, 16 * 256)), upload(backend, query), k, v,
                upload(backend, table), upload(backend, lengths), spec)
        before = backend.resource_report().scratch_bytes
        backend.paged_gqa(*args)  # outside of capture, so that there is room
        held += backend.resource_report().scratch_bytes - before
        graphs.append((args, backend.read(args[0]), *captured(backend,
                                                              lambda: backend.paged_gqa(*args))))
    # 256 blocks of two records of 16 rows of 256 and two statistics: the last one's.
    largest = 2 * 256 * 16 * 258 * 4 + 172 * 8
    say("held", held, "largest", largest)
    # Twice, for the last one's room, twice, for the ones replaced, an eighth for the pool's
    # steps.
    assert held <= 4 * largest * 9 / 8
    for _ in range(3):
        for args, want, replay, _end in graphs:
            backend.paged_gqa(*graphs[-1][0])
            replay()
            assert np.array_equal(backend.read(args[0]), want)
    for *_rest, end in graphs:
        end()
    backend.close()


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("dim", [64, 7, 300])
def test_prepared_keys_enter_as_they_are(backend, dim, interleaved, half):
    """Without weights and with no rotated column nothing is changed but by the pages'
    format: the keys of a prompt that ran over contiguous caches."""
    rng = np.random.default_rng(dim)
    tokens, heads, kv_heads, size = 21, 6, 3, 8
    q, k, v = (rng.standard_normal((tokens, h * dim)).astype(np.float32)
               for h in (heads, kv_heads, kv_heads))
    keys, values = (backend.alloc_pages(4, kv_heads, size, dim, half) for _ in range(2))
    table = np.array([[2, 0, 3]], np.float32)
    out = backend.allocate_f32((tokens, heads * dim))
    backend.paged_qk_norm_rope(out, keys, values, *(upload(backend, a) for a in (q, k, v)), None,
                               None, backend.allocate_f32((tokens, 0)), upload(backend, table),
                               upload(backend, np.zeros(tokens, np.float32)),
                               upload(backend, np.arange(tokens, dtype=np.float32)),
                               PagedRopeSpec(heads, kv_heads, dim, interleaved), EPSILON)
    assert np.array_equal(backend.read(out), q)
    for pages, rows in ((keys, k), (values, v)):
        got = read_pages(backend, pages)[[2, 0, 3]].transpose(0, 2, 1, 3).reshape(-1, kv_heads, dim)
        want = rows.reshape(tokens, kv_heads, dim).astype(np.float16 if half else np.float32)
        assert np.array_equal(got[:tokens], want)
        assert not got[tokens:].any()
