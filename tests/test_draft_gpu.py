"""Drafted trees and latent caches on the GPU: layout, entry at places, attention of runs,
settling, and a decode loop of all of them, against plain implementations in 64 bits.

Tolerances count roundings: half a step of f32 is 2^-24 of a value, of binary16
2^-11.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from runtime_amd import hiptime
from runtime_amd.backend import (CACHE, ExecutorError, GqaSpec, HipBackend, Limits, PagedRopeSpec,
                                 SCRATCH)

pytestmark = pytest.mark.gpu

EPSILON = 1.0e-5
F32, F16 = 2.0 ** -24, 2.0 ** -11
NAN = float("nan")


def say(*words):
    print(*words, flush=True)


def upload(backend, array):
    array = np.asarray(array)
    if array.dtype == np.float16:
        shape = array.shape[:-1] + (2 * array.shape[-1],)
        return backend.upload_u8_classified(shape, np.ascontiguousarray(array).view(np.uint8),
                                            CACHE)
    if array.dtype == np.uint8:
        return backend.upload_u8_classified(array.shape, array, SCRATCH)
    return backend.upload_f32(array.shape, array)


def f32(backend, values):
    return upload(backend, np.asarray(values, np.float32))


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


def starts_of(runs, before=0):
    return np.concatenate([[before], before + np.cumsum(runs)]).astype(np.float32)


def random_tree(rng, n):
    """Parents of one run."""
    return np.array([-1 if i == 0 else int(rng.integers(max(-1, i - 6), i)) for i in range(n)],
                    np.float32)


def ancestors(parents):
    """[n, n]: row i names itself and its ancestors."""
    n = len(parents)
    seen = np.zeros((n, n), bool)
    for i in range(n):
        j = i
        while j >= 0:
            seen[i, j] = True
            j = int(parents[j])
    return seen


def packed(seen, bytes_):
    wide = np.zeros((len(seen), 8 * bytes_), bool)
    count = min(seen.shape[1], 8 * bytes_)
    wide[:, :count] = seen[:, :count]
    return np.packbits(wide, axis=1, bitorder="little")


# ---- layout ----------------------------------------------------------------------

def run_layout(backend, starts, parents, lengths, tokens, bytes_):
    outs = [upload(backend, np.full(tokens, 9.0, np.float32)) for _ in range(3)]
    mask = (upload(backend, np.full((tokens, bytes_), 255, np.uint8)) if bytes_ else None)
    backend.draft_layout(*outs, mask, f32(backend, starts),
                         None if parents is None else f32(backend, parents), f32(backend, lengths))
    return [backend.read(o) for o in outs], backend.read_u8(mask) if bytes_ else None


@pytest.mark.parametrize("runs,bytes_", [
    ([1], 1), ([16], 2), ([64], 8), ([0, 5, 0, 17, 1], 3), ([65, 3], 9), ([63, 64, 65, 0], 16),
    ([300], 38), ([4200, 2], 525), ([7] * 300, 1), ([20, 9], 0)])
@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
def test_layout(backend, runs, bytes_, tree):
    say("layout", runs[:5], bytes_, tree)
    rng = np.random.default_rng(sum(runs) + bytes_)
    before, behind = 2, 3
    tokens = before + sum(runs) + behind
    starts, lengths = starts_of(runs, before), rng.integers(0, 5000, len(runs))
    parents = np.full(tokens, NAN, np.float32)
    for s, n in enumerate(runs):
        first = int(starts[s])
        parents[first:first + n] = random_tree(rng, n) if tree else np.arange(n) - 1
    got, mask = run_layout(backend, starts, parents if tree else None, lengths, tokens, bytes_)
    want = np.full((3, tokens), -1.0)
    bits = np.zeros((tokens, max(bytes_, 1)), np.uint8)
    for s, n in enumerate(runs):
        first = int(starts[s])
        seen = ancestors(parents[first:first + n])
        bits[first:first + n] = packed(seen, max(bytes_, 1))
        want[0, first:first + n] = s
        want[1, first:first + n] = lengths[s] + seen.sum(axis=1) - 1
        want[2, first:first + n] = lengths[s] + np.arange(n)
    assert np.array_equal(got, want)
    assert mask is None or np.array_equal(mask, bits)


def test_layout_of_bad_trees(backend):
    """Bad parents and what descends from them, masks too narrow, bad lengths."""
    parents = [-1, 0, 2, 2, 1, NAN, 0.5, 5, -2, -1, 9, 8] + [-1, 0, 1] + [-1, 0] + [0, -1] + [-1]
    starts, lengths = [0, 12, 15, 17, 19], [10, 0.5, 2 ** 24 - 1, 7]
    got, mask = run_layout(backend, starts, parents, lengths, 20, 2)
    good = {0: (0, 10, 10, 1), 1: (0, 11, 11, 3), 4: (0, 12, 14, 0b10011),
            9: (0, 10, 19, 1 << 9), 10: (0, 11, 20, 3 << 9), 18: (3, 7, 8, 2)}
    for t in range(20):
        want = good.get(t, (-1, -1, -1, 0))
        assert tuple(o[t] for o in got) == want[:3], t
        assert int(mask[t, 0]) | int(mask[t, 1]) << 8 == want[3], t
    # A token past the mask's last bit has no place; nor have tokens that follow it.
    got, mask = run_layout(backend, [0, 20], [-1] + list(range(19)), [3], 20, 2)
    assert np.array_equal(got[2], [3 + i if i < 16 else -1 for i in range(20)])
    assert mask[15].tolist() == [255, 255] and mask[16].tolist() == [0, 0]


@pytest.mark.parametrize("bad", [NAN, -1.0, 2.5, 3.0, 99.0, float("inf")])
@pytest.mark.parametrize("at", [0, 2, 3])
def test_a_bad_start_ends_the_list(backend, bad, at):
    starts, lengths = np.array([0, 4, 6, 8], np.float32), [1, 2, 3]
    starts[at] = bad
    got, _ = run_layout(backend, starts, None, lengths, 9, 1)
    want = np.full(9, -1.0)
    for s in range(3):
        ok = all(starts[i] == np.trunc(starts[i]) and 0 <= starts[i] <= starts[i + 1] <= 9
                 and starts[i + 1] == np.trunc(starts[i + 1]) for i in range(s + 1))
        if ok:
            want[int(starts[s]):int(starts[s + 1])] = s
    assert np.array_equal(got[0], want)


# ---- attention of runs ----------------------------------------------------------------

class Batch:
    """Runs over paged caches; `kind` is chain, tree, bits (any mask) or none (one token each,
    no starts)."""

    def __init__(self, seed, shapes, kind, size, before=0, behind=0, bytes_=None):
        self.rng, self.size, self.kind = np.random.default_rng(seed), size, kind
        self.lengths = np.array([length for length, _ in shapes], np.float32)
        self.runs = [n for _, n in shapes]
        self.starts = starts_of(self.runs, before)
        self.tokens = before + sum(self.runs) + behind
        self.pages, self.table = tables_for(self.rng, [a + b for a, b in shapes], size)
        self.seen, most = [], max(self.runs)
        self.bytes = bytes_ or -(-most // 8)
        self.mask = np.full((self.tokens, self.bytes), 255, np.uint8)
        for s, n in enumerate(self.runs):
            if kind == "tree":
                seen = ancestors(random_tree(self.rng, n))
            elif kind == "bits":
                seen = self.rng.random((n, n)) < 0.4
                seen[:, 8 * self.bytes:] = False
                seen[n // 2:n // 2 + 1] = False
                if n > 2:
                    seen[:, n - 2] = False  # a token that none attends
            else:
                seen = np.tril(np.ones((n, n), bool))
            self.seen.append(seen)
            self.mask[int(self.starts[s]):int(self.starts[s]) + n] = packed(seen, self.bytes)

    def args(self, backend):
        """tables, starts, lengths, mask."""
        return (upload(backend, self.table),
                None if self.kind == "none" else upload(backend, self.starts),
                upload(backend, self.lengths),
                upload(backend, self.mask) if self.kind in ("tree", "bits") else None)

    def spoil(self, *pages):
        """What no token attends holds NaN and infinities."""
        for s, n in enumerate(self.runs):
            end = int(self.lengths[s]) + n
            places = [end - n + i for i in range(n) if n and not self.seen[s][:, i].any()]
            if end % self.size:
                places += range(end, -(-end // self.size) * self.size)
            for place in places:
                for i, array in enumerate(pages):
                    array[int(self.table[s, place // self.size]), :, place % self.size] = (
                        np.inf if i else np.nan)

    def attend(self, query, keys, values, scale):
        """In 64 bits, query [tokens, heads, d]: (outputs, the bound of their error), NaN in
        rows of no run."""
        heads, kv_heads, dim, dv = query.shape[1], keys.shape[1], keys.shape[3], values.shape[3]
        group = heads // kv_heads
        out = np.full((self.tokens, heads, dv), np.nan)
        bound = np.zeros((self.tokens, heads, dv))
        for s, n in enumerate(self.runs):
            length, first = int(self.lengths[s]), int(self.starts[s])
            total = length + n
            ids = self.table[s, :-(-total // self.size)].astype(int)
            seen = np.ones((n, total), bool)
            seen[:, length:] = self.seen[s]
            for h in range(heads):
                key = keys[ids, h // group].reshape(-1, dim)[:total].astype(np.float64)
                value = values[ids, h // group].reshape(-1, dv)[:total].astype(np.float64)
                used = seen.any(axis=0)
                key, value = np.where(used[:, None], key, 0), np.where(used[:, None], value, 0)
                q = query[first:first + n, h].astype(np.float64)
                score = np.where(seen, q @ key.T * scale, -np.inf)
                top = np.maximum(score.max(axis=1, initial=-np.inf), -1e300)[:, None]
                p = np.exp(score - top)
                weight = p.sum(axis=1, keepdims=True)
                p = p / np.where(weight > 0, weight, 1)
                out[first:first + n, h] = p @ value
                # A score's error: dim products and sums, scale and exponent (8 more); it
                # moves numerator and denominator.  Then the weighted sums: the keys of a
                # tile and the tiles of a part.  Last, probabilities below 2^-40 of the
                # largest may be cut.
                size_of = np.where(seen, np.abs(q) @ np.abs(key).T, 0).max(
                    axis=1, initial=0)[:, None] * scale
                relative = 2 * (dim + 8) * F32 * size_of + (64 + total / 64 + 32) * F32
                bound[first:first + n, h] = (relative * (p @ np.abs(value)) + 2.0 ** -40 +
                                             total * 2.0 ** -41 * np.abs(value).max(initial=0))
        return out, bound


def check(got, want, bound, untouched):
    """Rows of a run against the bound, others as they were."""
    mine = ~np.isnan(want).any(axis=tuple(range(1, want.ndim)))
    assert np.all(got[~mine] == untouched)
    off = np.abs(got[mine] - want[mine])
    assert np.all(off <= bound[mine]), np.nanmax(off / (bound[mine] + 1e-30))


SHAPES = {"one": [(0, 1)], "first": [(0, 40)], "single": [(1, 1), (33, 1), (64, 1), (500, 1)],
          "mixed": [(0, 3), (5, 1), (16, 0), (31, 17), (64, 8), (100, 33), (0, 0), (129, 2)],
          "long": [(4090, 9)], "wide": [(70, 130)], "many": [(3, 2)] * 70 + [(90, 5)],
          "few": [(0, 2), (0, 0), (7, 0), (40, 3), (5, 0), (0, 1), (3, 0), (0, 0)]}


def run_tree(backend, batch, query, keys, values, heads, kv_heads, dim):
    out = upload(backend, np.full(query.shape, 7.0, np.float32))
    table, starts, lengths, mask = batch.args(backend)
    backend.paged_tree_gqa(out, upload(backend, query), upload(backend, keys),
                           upload(backend, values), table, starts, lengths, mask,
                           GqaSpec(heads, kv_heads, dim))
    return backend.read(out)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim,size", [
    (8, 2, 64, 16), (4, 4, 128, 32), (12, 4, 64, 8), (16, 1, 128, 64), (6, 2, 80, 16),
    (8, 2, 96, 8), (3, 1, 256, 128), (8, 4, 32, 256), (40, 2, 64, 16), (5, 5, 16, 16),
    (6, 3, 20, 8), (2, 1, 7, 16), (2, 2, 1, 8), (2, 1, 1000, 16), (9, 3, 112, 64),
    (2, 1, 160, 16), (5, 1, 192, 8)])
@pytest.mark.parametrize("kind", ["chain", "tree", "bits"])
@pytest.mark.parametrize("which", list(SHAPES))
def test_attention_of_runs(backend, which, kind, heads, kv_heads, dim, size, half):
    say("tree", which, kind, heads, kv_heads, dim, size, half)
    batch = Batch(dim * 31 + size + half, SHAPES[which], kind, size, 1, 2)
    keys, values = (random_pages(batch.rng, batch.pages, kv_heads, size, dim, half)
                    for _ in range(2))
    batch.spoil(keys, values)
    query = batch.rng.standard_normal((batch.tokens, heads * dim)).astype(np.float32) * 2
    got = run_tree(backend, batch, query, keys, values, heads, kv_heads, dim)
    want, bound = batch.attend(query.reshape(batch.tokens, heads, dim), keys, values,
                               1 / math.sqrt(dim))
    check(got.reshape(want.shape), want, bound, 7.0)
    assert np.array_equal(got, run_tree(backend, batch, query, keys, values, heads, kv_heads, dim))


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 20])
def test_a_token_each_without_starts(backend, dim, half):
    shapes = [(0, 1), (1, 1), (63, 1), (64, 1), (300, 1), (15, 1)] * 9
    batch = Batch(dim, shapes, "none", 16)
    keys, values = (random_pages(batch.rng, batch.pages, 2, 16, dim, half) for _ in range(2))
    batch.spoil(keys, values)
    query = batch.rng.standard_normal((batch.tokens, 6 * dim)).astype(np.float32)
    got = run_tree(backend, batch, query, keys, values, 6, 2, dim)
    want, bound = batch.attend(query.reshape(-1, 6, dim), keys, values, 1 / math.sqrt(dim))
    check(got.reshape(want.shape), want, bound, 7.0)
    # The same as one token's attention, within both's roundings.
    out = backend.allocate_f32(query.shape)
    backend.paged_gqa(out, upload(backend, query), upload(backend, keys), upload(backend, values),
                      upload(backend, batch.table), f32(backend, batch.lengths + 1),
                      GqaSpec(6, 2, dim))
    assert np.all(np.abs(backend.read(out).reshape(want.shape) - got.reshape(want.shape))
                  <= 2 * bound)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 20])
@pytest.mark.parametrize("scale", [1e-30, 1e-6, 300.0])
def test_queries_and_values_of_any_size(backend, scale, dim, half):
    say("scale", scale, dim, half)
    batch = Batch(8, [(300, 19)], "tree", 16)
    keys, values = (random_pages(batch.rng, batch.pages, 2, 16, dim, half) for _ in range(2))
    if half:
        keys[3, 0, 5] = 2.0 ** -20  # subnormal there
        values[3, 0, 5] = 3 * 2.0 ** -24
    else:
        values *= np.float32(1 / scale)
    query = (scale * batch.rng.standard_normal((19, 4 * dim))).astype(np.float32)
    query[0, 1] *= 1e-4
    got = run_tree(backend, batch, query, keys, values, 4, 2, dim)
    want, bound = batch.attend(query.reshape(-1, 4, dim), keys, values, 1 / math.sqrt(dim))
    check(got.reshape(want.shape), want, bound, 7.0)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 20])
def test_one_large_value(backend, dim, half):
    """A value far above the others at a key without weight, keys of very different sizes."""
    batch = Batch(9, [(200, 6)], "chain", 16)
    keys, values = (random_pages(batch.rng, batch.pages, 1, 16, dim, half) for _ in range(2))
    query = batch.rng.standard_normal((6, dim)).astype(np.float32)
    place = (int(batch.table[0, 2]), 0, 5)
    keys[place] = -40 * np.sign(query[0]) / math.sqrt(dim)
    values[place] = 6e4 if half else 1e8
    query[1:] = query[0] * (1 + 0.01 * batch.rng.standard_normal((5, 1))).astype(np.float32)
    got = run_tree(backend, batch, query, keys, values, 1, 1, dim)
    want, bound = batch.attend(query.reshape(-1, 1, dim), keys, values, 1 / math.sqrt(dim))
    check(got.reshape(want.shape), want, bound, 7.0)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 10])
def test_bad_lengths_and_pages_of_runs(backend, dim, half):
    shapes = [(200, 4)] * 10 + [(316, 4), (317, 3)]
    batch = Batch(dim, shapes, "chain", 8)
    good = batch.lengths.copy()
    batch.lengths[:6] = -1, 0.5, np.nan, np.inf, 317, 2.0 ** 24
    batch.table[6, 3], batch.table[7, 24], batch.table[8, 0] = -1.0, batch.pages, np.nan
    # Places 200 to 203 lie in page 25; only tokens there attend it.
    batch.table[9, 25] = 1.5
    keys, values = (random_pages(batch.rng, batch.pages, 2, 8, dim, half) for _ in range(2))
    query = batch.rng.standard_normal((batch.tokens, 4 * dim)).astype(np.float32)
    got = run_tree(backend, batch, query, keys, values, 4, 2, dim)
    assert np.all(np.isnan(got[:40]))
    batch.lengths = good
    batch.table[:10] = 0
    want, bound = batch.attend(query.reshape(-1, 4, dim), keys, values, 1 / math.sqrt(dim))
    check(got[40:].reshape(want[40:].shape), want[40:], bound[40:], 7.0)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 20])
@pytest.mark.parametrize("kind", ["chain", "tree"])
def test_a_bad_page_reaches_those_that_attend_it(backend, kind, dim, half):
    """A run over several pages, the third of them bad: rows that attend none of it are as
    without it."""
    batch = Batch(dim + 5, [(20, 60)], kind, 8)
    keys, values = (random_pages(batch.rng, batch.pages, 2, 8, dim, half) for _ in range(2))
    query = batch.rng.standard_normal((60, 8 * dim)).astype(np.float32)
    want, bound = batch.attend(query.reshape(-1, 8, dim), keys, values, 1 / math.sqrt(dim))
    batch.table[0, 5] = 1e9  # places 40 to 47: tokens 20 to 27
    got = run_tree(backend, batch, query, keys, values, 8, 2, dim).reshape(want.shape)
    reached = batch.seen[0][:, 20:28].any(axis=1)
    assert np.all(np.isnan(got[reached]))
    assert np.all(np.abs(got[~reached] - want[~reached]) <= bound[~reached])


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 20])
@pytest.mark.parametrize("kind", ["chain", "tree"])
@pytest.mark.parametrize("what", [np.nan, np.inf])
def test_values_that_are_not_finite_reach_those_that_attend_them(backend, kind, dim, half, what):
    batch = Batch(dim + 6, [(37, 50)], kind, 16)
    keys, values = (random_pages(batch.rng, batch.pages, 2, 16, dim, half) for _ in range(2))
    query = batch.rng.standard_normal((50, 8 * dim)).astype(np.float32)
    want, bound = batch.attend(query.reshape(-1, 8, dim), keys, values, 1 / math.sqrt(dim))
    for token, pages in ((21, keys), (30, values)):
        place = 37 + token
        pages[int(batch.table[0, place // 16]), 1, place % 16] = what
    got = run_tree(backend, batch, query, keys, values, 8, 2, dim).reshape(want.shape)
    reached = np.zeros((50, 8), bool)
    reached[:, 4:] = batch.seen[0][:, [21, 30]].any(axis=1)[:, None]
    assert not np.any(np.isfinite(got[reached]).all(axis=-1))
    assert np.all(np.abs(got[~reached] - want[~reached]) <= bound[~reached])


@pytest.mark.parametrize("dim", [32, 64, 128, 20])
@pytest.mark.parametrize("kind", ["chain", "tree"])
def test_the_largest_finite_values_stay_with_those_that_attend_them(backend, kind, dim):
    batch = Batch(dim + 8, [(37, 50)], kind, 16)
    keys, values = (random_pages(batch.rng, batch.pages, 2, 16, dim, False) for _ in range(2))
    query = batch.rng.standard_normal((50, 8 * dim)).astype(np.float32)
    want, bound = batch.attend(query.reshape(-1, 8, dim), keys, values, 1 / math.sqrt(dim))
    for token, pages in ((21, keys), (30, values)):
        place = 37 + token
        pages[int(batch.table[0, place // 16]), 1, place % 16] = np.finfo(np.float32).max
    got = run_tree(backend, batch, query, keys, values, 8, 2, dim).reshape(want.shape)
    reached = np.zeros((50, 8), bool)
    reached[:, 4:] = batch.seen[0][:, [21, 30]].any(axis=1)[:, None]
    assert np.all(np.abs(got[~reached] - want[~reached]) <= bound[~reached])


@pytest.mark.parametrize("count", [1, 3, 64, 65, 255, 256, 257, 300])
@pytest.mark.parametrize("dim", [64, 20])
def test_any_count_of_runs(backend, count, dim):
    rng = np.random.default_rng(count)
    shapes = [(int(rng.integers(0, 90)), int(rng.integers(0, 6))) for _ in range(count)]
    batch = Batch(count, shapes, "tree", 8, bytes_=1)
    keys, values = (random_pages(batch.rng, batch.pages, 2, 8, dim, False) for _ in range(2))
    query = batch.rng.standard_normal((batch.tokens, 4 * dim)).astype(np.float32)
    bad = rng.random(count) < 0.1
    want, bound = batch.attend(query.reshape(-1, 4, dim), keys, values, 1 / math.sqrt(dim))
    batch.lengths[bad] = -3
    got = run_tree(backend, batch, query, keys, values, 4, 2, dim).reshape(want.shape)
    for s in range(count):
        rows = slice(int(batch.starts[s]), int(batch.starts[s + 1]))
        if bad[s]:
            assert np.all(np.isnan(got[rows]))
        else:
            assert np.all(np.abs(got[rows] - want[rows]) <= bound[rows])


def test_batches_of_nothing(backend):
    pages, other = (backend.alloc_pages(1, 1, 8, 64) for _ in range(2))
    none = backend.allocate_f32((0, 64))
    backend.paged_tree_gqa(none, backend.allocate_f32((0, 64)), pages, other,
                           backend.allocate_f32((0, 3)), None, backend.allocate_f32((0,)), None,
                           GqaSpec(1, 1, 64))
    out = upload(backend, np.full((3, 64), 7.0, np.float32))
    query = backend.allocate_f32((3, 64))
    # No sequences; sequences without runs; a table without columns.
    backend.paged_tree_gqa(out, query, pages, other, backend.allocate_f32((0, 3)),
                           f32(backend, [0]), backend.allocate_f32((0,)), None, GqaSpec(1, 1, 64))
    backend.paged_tree_gqa(out, query, pages, other, backend.allocate_f32((2, 3)),
                           f32(backend, [1, 1, 1]), f32(backend, [5, 0]), None, GqaSpec(1, 1, 64))
    assert np.all(backend.read(out) == 7.0)
    backend.paged_tree_gqa(out, query, pages, other, backend.allocate_f32((1, 0)),
                           f32(backend, [0, 2]), f32(backend, [0]), None, GqaSpec(1, 1, 64))
    got = backend.read(out)
    assert np.all(np.isnan(got[:2])) and np.all(got[2] == 7.0)
    # A mask that leaves a row nothing.
    backend.paged_tree_gqa(out, query, pages, other, backend.allocate_f32((1, 1)),
                           f32(backend, [0, 3]), f32(backend, [0]),
                           upload(backend, np.array([[1], [0], [6]], np.uint8)), GqaSpec(1, 1, 64))
    assert np.all(backend.read(out) == 0.0)


# ---- latents ----------------------------------------------------------------------------

def run_latent(backend, batch, latent_query, rotary_query, pages, heads, scale):
    out = upload(backend, np.full(latent_query.shape, 7.0, np.float32))
    table, starts, lengths, mask = batch.args(backend)
    backend.paged_latent_attention(out, upload(backend, latent_query),
                                   upload(backend, rotary_query), upload(backend, pages), table,
                                   starts, lengths, mask, heads, scale)
    return backend.read(out)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("heads,rank,rope,size", [
    (16, 512, 64, 16), (5, 512, 32, 64), (128, 512, 64, 8), (20, 256, 64, 16), (64, 256, 32, 8),
    (3, 128, 64, 128), (33, 128, 32, 16), (4, 96, 32, 16), (7, 30, 6, 8), (1, 1, 2, 8),
    (2, 960, 64, 8), (6, 64, 0, 16)])
@pytest.mark.parametrize("which,kind", [("one", "none"), ("single", "none")] + [
    (which, kind) for which in ("one", "single", "mixed", "long", "wide", "few")
    for kind in ("chain", "tree", "bits")])
def test_latent_attention(backend, which, kind, heads, rank, rope, size, half):
    shapes = SHAPES[which]
    if heads * sum(n for _, n in shapes) > 5000:
        shapes = [(a, min(n, 40)) for a, n in shapes]
    say("latent", which, kind, heads, rank, rope, size, half)
    pad = (0, 0) if kind == "none" else (2, 1)
    batch = Batch(rank + size + half, shapes, kind, size, *pad)
    pages = random_pages(batch.rng, batch.pages, 1, size, rank + rope, half)
    batch.spoil(pages)
    latent, rotary = (batch.rng.standard_normal((batch.tokens, heads * w)).astype(np.float32)
                      for w in (rank, rope))
    scale = float(np.float32(1.5 / math.sqrt(rank + rope)))
    got = run_latent(backend, batch, latent, rotary, pages, heads, scale)
    query = np.concatenate([x.reshape(batch.tokens, heads, -1 if x.size else 0)
                            for x in (latent, rotary)], axis=2)
    want, bound = batch.attend(query, pages, pages[..., :rank], scale)
    check(got.reshape(want.shape), want, bound, 7.0)
    assert np.array_equal(got, run_latent(backend, batch, latent, rotary, pages, heads, scale))


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("rank", [512, 30])
def test_bad_pages_of_latents(backend, rank, half):
    batch = Batch(rank, [(20, 60), (30, 2), (9, 3)], "chain", 8)
    pages = random_pages(batch.rng, batch.pages, 1, 8, rank + 64, half)
    latent, rotary = (batch.rng.standard_normal((65, 4 * w)).astype(np.float32)
                      for w in (rank, 64))
    scale = float(np.float32(1 / math.sqrt(rank)))
    query = np.concatenate([latent.reshape(65, 4, -1), rotary.reshape(65, 4, -1)], axis=2)
    want, bound = batch.attend(query, pages, pages[..., :rank], scale)
    batch.table[0, 5], batch.lengths[1] = -2.0, NAN
    got = run_latent(backend, batch, latent, rotary, pages, 4, scale).reshape(want.shape)
    reached = np.zeros(65, bool)
    reached[20:62] = True
    assert np.all(np.isnan(got[reached]))
    assert np.all(np.abs(got[~reached] - want[~reached]) <= bound[~reached])


# ---- entry ------------------------------------------------------------------------------

def turned(x, turn, interleaved):
    """[tokens, heads, rope] in 64 bits; turn [tokens, rope]."""
    x, pairs = x.astype(np.float64), x.shape[-1] // 2
    first = slice(0, None, 2) if interleaved else slice(0, pairs)
    second = slice(1, None, 2) if interleaved else slice(pairs, None)
    out, cosine, sine = x.copy(), turn[:, None, :pairs], turn[:, None, pairs:]
    out[..., first] = x[..., first] * cosine - x[..., second] * sine
    out[..., second] = x[..., second] * cosine + x[..., first] * sine
    return out


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("tokens,heads,rank,rope,size,norm,places", [
    (1, 16, 512, 64, 16, True, False), (37, 32, 512, 64, 64, True, True), (6, 5, 256, 32, 8, True, False),
    (9, 3, 30, 6, 8, True, True), (5, 7, 33, 2, 16, False, False), (4, 1, 1, 0, 8, True, True),
    (3, 128, 512, 64, 16, False, True), (2, 2, 960, 64, 8, True, False),
    (4, 3, 1500, 100, 8, True, False)])
def test_tokens_enter_latent_caches(backend, tokens, heads, rank, rope, size, norm, places,
                                    interleaved, half):
    say("enter", tokens, heads, rank, rope, size, norm, places, interleaved, half)
    rng = np.random.default_rng(tokens * 100 + rank + half)
    sequences = np.arange(tokens) % 3
    position = (rng.permutation(40)[:tokens] if tokens <= 40 else np.arange(tokens)).astype(np.float32)
    place = rng.permutation(60)[:tokens].astype(np.float32) if places else position.copy()
    bad = np.zeros(tokens, bool)
    if tokens > 4:
        position[-1], position[-2], place[-2], sequences = -1, 50, 3, sequences.astype(np.float32)
        sequences[-3] = 3 if tokens > 5 else sequences[-3]
        bad[[-1, -2]] = True
        bad[-3] = tokens > 5
        place = np.where(position == -1, -1, place).astype(np.float32) if not places else place
        if places:
            place[-4], bad[-4] = 64, True
    if not places:
        place = position
    pages, table = tables_for(rng, [60] * 3, size)
    old = random_pages(rng, pages, 1, size, rank + rope, half)
    cache = upload(backend, old)
    x = {n: rng.standard_normal((tokens, w)).astype(np.float32) * 3
         for n, w in (("q", heads * rope), ("c", rank), ("k", rope))}
    weight = (1 + 0.1 * rng.standard_normal(rank)).astype(np.float32) if norm else None
    turn = rng.standard_normal((50, rope)).astype(np.float32)
    out = backend.allocate_f32((tokens, heads * rope))
    backend.paged_latent_append(
        out, cache, upload(backend, x["q"]), upload(backend, x["c"]), upload(backend, x["k"]),
        None if weight is None else upload(backend, weight), upload(backend, turn),
        upload(backend, table), f32(backend, sequences), f32(backend, position),
        f32(backend, place) if places else None, heads, interleaved, EPSILON)
    good = ~bad
    coefficients = turn[np.where(good, position, 0).astype(int)]
    got, now = backend.read(out).reshape(tokens, heads, rope), read_pages(backend, cache)
    assert np.all(np.isnan(got[bad]))
    queries = turned(x["q"].reshape(tokens, heads, rope), coefficients, interleaved)
    keys = turned(x["k"].reshape(tokens, 1, rope), coefficients, interleaved)[:, 0]
    # Two products and a sum of values below 8 times 4; the norm: rank / 64 + 10 roundings.
    largest = 8 * np.abs(turn).max(initial=0) * 3
    assert np.all(np.abs(got[good] - queries[good]) <= 3 * F32 * largest)
    latent = x["c"].astype(np.float64)
    if norm:
        latent = latent / np.sqrt((latent ** 2).mean(axis=1, keepdims=True) +
                                  float(np.float32(EPSILON))) * weight
    store = lambda v: F16 * np.abs(v) + 2.0 ** -25 if half else 0.0  # noqa: E731
    untouched = np.ones((pages, size), bool)
    for t in np.flatnonzero(good):
        page, slot = int(table[int(sequences[t]), int(place[t]) // size]), int(place[t]) % size
        row = now[page, 0, slot]
        untouched[page, slot] = False
        assert np.all(np.abs(row[rank:] - keys[t]) <= 3 * F32 * largest + store(keys[t]))
        if norm:
            assert np.all(np.abs(row[:rank] - latent[t]) <=
                          (rank / 64 + 10) * F32 * np.abs(latent[t]) + store(latent[t]))
        else:
            assert np.array_equal(row[:rank], x["c"][t].astype(old.dtype))
    assert np.array_equal(now[:, 0][untouched], old.astype(np.float32)[:, 0][untouched])


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 7])
def test_siblings_share_a_position(backend, dim, half):
    """Tokens at places of their own turn by their positions; bad places enter nothing."""
    rng = np.random.default_rng(dim)
    positions = np.array([5, 6, 6, 7, 6, 6, 6], np.float32)
    places = np.array([5, 6, 7, 8, -1, 24, NAN], np.float32)
    q, k, v = (rng.standard_normal((7, 2 * dim)).astype(np.float32) for _ in range(3))
    turn = rng.standard_normal((9, dim // 2 * 2)).astype(np.float32)
    table = f32(backend, [[2, 0, 3]])
    spec = PagedRopeSpec(2, 2, dim)

    def enter(at, where, rows):
        cache = [backend.alloc_pages(4, 2, 8, dim, half=half) for _ in range(2)]
        out = backend.allocate_f32((len(rows), 2 * dim))
        arguments = [out, *cache, *(upload(backend, a[rows]) for a in (q, k, v)), None, None,
                     upload(backend, turn), table, f32(backend, np.zeros(len(rows))),
                     f32(backend, at)]
        if where is None:
            backend.paged_qk_norm_rope(*arguments, spec, EPSILON)
        else:
            backend.paged_qk_norm_rope_at(*arguments, f32(backend, where), spec, EPSILON)
        return backend.read(out), [read_pages(backend, c) for c in cache]

    out, cache = enter(positions, places, np.arange(7))
    assert np.all(np.isnan(out[4:])) and np.all(np.isfinite(out[:4]))
    want = [np.zeros_like(c) for c in cache]
    for t in range(4):
        alone, at_position = enter(positions[[t]], None, np.array([t]))
        assert np.array_equal(alone[0], out[t])
        for w, c in zip(want, at_position):
            a, b = int(positions[t]), int(places[t])
            w[[2, 0, 3][b // 8], :, b % 8] = c[[2, 0, 3][a // 8], :, a % 8]
    assert all(np.array_equal(w, c) for w, c in zip(want, cache))


# ---- settling ------------------------------------------------------------------------------

def settled(starts, parents, tokens, choices, lengths, table, size, columns, caches):
    """(emitted, counts, next), caches changed in place."""
    n = len(lengths)
    emitted = np.full((n, columns), -1.0)
    counts, last = np.zeros(n), np.full(n, -1.0)
    for s in range(n):
        first, count = int(starts[s]), int(starts[s + 1] - starts[s])
        if not count:
            continue
        path = [0]
        while len(path) < columns:
            at = path[-1]
            child = [i for i in range(at + 1, count)
                     if (parents[first + i] if parents is not None else i - 1) == at
                     and tokens[first + i] == choices[first + at]]
            if not child:
                break
            path.append(child[0])
        spots = []
        for k, i in enumerate(path):
            for place in (int(lengths[s]) + i, int(lengths[s]) + k):
                spots.append((int(table[s, place // size]), place % size))
        for array in caches:
            moved = [array[page, :, slot].copy() for page, slot in spots[0::2]]
            for row, (page, slot) in zip(moved, spots[1::2]):
                array[page, :, slot] = row
        emitted[s, :len(path)] = [choices[first + i] for i in path]
        counts[s], last[s] = len(path), emitted[s, len(path) - 1]
    return emitted, counts, last


def run_settle(backend, starts, parents, tokens, choices, lengths, table, columns, caches):
    n = len(lengths)
    outs = [upload(backend, np.full(shape, 9.0, np.float32)) for shape in ((n, columns), (n,), (n,))]
    backend.settle_drafts(*outs, caches, f32(backend, tokens), f32(backend, choices),
                          f32(backend, starts), None if parents is None else f32(backend, parents),
                          f32(backend, lengths), upload(backend, table))
    return [backend.read(o) for o in outs]


@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
@pytest.mark.parametrize("runs,columns,size,widths", [
    ([16], 16, 16, [(8, 64, False)] * 12), ([1, 0, 33, 7, 64, 65], 12, 8, [(2, 64, True), (1, 576, True)]),
    ([40] * 30, 40, 32, [(3, 7, False), (5, 9, True), (1, 36, False)]), ([300, 20], 1024, 8, [(1, 16, True)]),
    ([9, 9], 1, 8, [(1, 4, False)]), ([5, 12], 5, 8, []), ([6] * 3, 6, 8, [(1, 8, False)] * 70)])
def test_settling(backend, runs, columns, size, widths, tree):
    say("settle", runs[:6], columns, size, len(widths), tree)
    rng = np.random.default_rng(sum(runs) + columns)
    starts, lengths = starts_of(runs, 2), rng.integers(0, 100, len(runs))
    count = int(starts[-1]) + 3
    tokens = rng.integers(0, 6, count).astype(np.float32)
    choices = rng.integers(0, 6, count).astype(np.float32)
    parents = np.full(count, NAN, np.float32)
    for s, n in enumerate(runs):
        first = int(starts[s])
        parents[first:first + n] = random_tree(rng, n) if tree else np.arange(n) - 1
        for i in range(n):  # most go on
            child = [j for j in range(i + 1, n) if parents[first + j] == i]
            if child and rng.random() < 0.9:
                choices[first + i] = tokens[first + int(rng.choice(child))]
    pages, table = tables_for(rng, lengths + runs, size)
    caches = [random_pages(rng, pages, heads, size, dim, half) for heads, dim, half in widths]
    given = [upload(backend, c) for c in caches]
    got = run_settle(backend, starts, parents if tree else None, tokens, choices, lengths, table,
                     columns, given)
    want = settled(starts, parents, tokens, choices, lengths, table, size, columns, caches)
    for g, w in zip(got, want):
        assert np.array_equal(g, w)
    assert want[1].max() >= min(columns, 2)
    # Rows of a path's places, and all outside of the runs, are as expected.
    for g, w in zip(given, caches):
        assert np.array_equal(read_pages(backend, g), w.astype(np.float32))


def test_settling_of_bad_sequences(backend):
    """Bad lengths, places without a page, choices that are NaN, a bad list of starts."""
    rng = np.random.default_rng(2)
    runs = [4, 4, 4, 4, 4, 4]
    starts = starts_of(runs)
    tokens = np.arange(24, dtype=np.float32) % 4
    choices = np.roll(tokens, -1)
    choices[17] = NAN
    lengths = np.array([3, NAN, 2.5, 6, 5, 2], np.float32)
    pages, table = tables_for(rng, [16] * 6, 8)
    table[0, 0], table[3, 1] = -1, pages
    starts[6] = 23.5
    old = random_pages(rng, pages, 2, 8, 5, False)
    cache = upload(backend, old)
    emitted, counts, last = run_settle(backend, starts, None, tokens, choices, lengths, table, 4,
                                       [cache])
    assert np.all(np.isnan(counts[:4])) and np.all(np.isnan(last[:4])) and np.all(
        np.isnan(emitted[:4]))
    assert counts[4] == 2 and emitted[4, 0] == 1 and np.isnan(emitted[4, 1]) and np.isnan(last[4])
    assert emitted[4, 2:].tolist() == [-1, -1]
    assert counts[5] == 0 and last[5] == -1 and np.all(emitted[5] == -1)
    assert np.array_equal(backend.read(cache), old)


# ---- together ---------------------------------------------------------------------------------

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


class Model:
    """A layer of keys and values and one of latents over a vocabulary of projections; its
    choice of the next token is the largest of its logits."""

    heads, kv_heads, dim, rank, rope, vocab, size, sequences, columns = 4, 2, 64, 128, 32, 97, 8, 3, 6
    most = 64  # places of a sequence

    def __init__(self, backend, half, seed=3):
        rng = np.random.default_rng(seed)
        self.b = backend
        shape = {"q": self.heads * self.dim, "k": self.kv_heads * self.dim,
                 "v": self.kv_heads * self.dim, "lq": self.heads * self.rank,
                 "lr": self.heads * self.rope, "c": self.rank, "r": self.rope}
        self.by_token = {n: upload(backend, rng.standard_normal((self.vocab, w)).astype(np.float32))
                         for n, w in shape.items()}
        self.heads_out = {n: upload(backend, rng.standard_normal((self.vocab, w)).astype(np.float32))
                          for n, w in (("q", shape["q"]), ("lq", shape["lq"]))}
        self.weight = f32(backend, 1 + 0.1 * rng.standard_normal(self.rank))
        self.turn, self.latent_turn = (backend.allocate_f32((self.most, w))
                                       for w in (self.dim, self.rope))
        backend.rotation_table(self.turn, 1.0e4)
        backend.rotation_table(self.latent_turn, 1.0e4)
        pages = self.sequences * self.most // self.size
        self.table = f32(backend, rng.permutation(pages).reshape(self.sequences, -1))
        self.caches = [backend.alloc_pages(pages, self.kv_heads, self.size, self.dim, half)
                       for _ in range(2)]
        self.caches.append(backend.alloc_pages(pages, 1, self.size, self.rank + self.rope, half))

    def buffers(self, tokens):
        a = self.b.allocate_f32
        got = {n: a((tokens, w.shape[1])) for n, w in self.by_token.items()}
        got |= {n: a((tokens, self.by_token[of].shape[1]))
                for n, of in (("q'", "q"), ("lr'", "lr"), ("o", "q"), ("lo", "lq"))}
        got |= {n: a((tokens, self.vocab)) for n in ("first", "second", "logits")}
        return got | {n: a((tokens,)) for n in ("sequence", "position", "place", "choice")}

    def run(self, w, tokens, starts, parents, lengths, mask):
        """The choices after every token, whose keys, values and latents enter the caches."""
        b = self.b
        b.draft_layout(w["sequence"], w["position"], w["place"], mask, starts, parents, lengths)
        for n in self.by_token:
            b.gather_rows(w[n], self.by_token[n], tokens)
        b.paged_qk_norm_rope_at(w["q'"], *self.caches[:2], w["q"], w["k"], w["v"], None, None,
                                self.turn, self.table, w["sequence"], w["position"], w["place"],
                                PagedRopeSpec(self.heads, self.kv_heads, self.dim), EPSILON)
        b.paged_latent_append(w["lr'"], self.caches[2], w["lr"], w["c"], w["r"], self.weight,
                              self.latent_turn, self.table, w["sequence"], w["position"],
                              w["place"], self.heads, True, EPSILON)
        b.paged_tree_gqa(w["o"], w["q'"], *self.caches[:2], self.table, starts, lengths, mask,
                         GqaSpec(self.heads, self.kv_heads, self.dim))
        b.paged_latent_attention(w["lo"], w["lq"], w["lr'"], self.caches[2], self.table, starts,
                                 lengths, mask, self.heads, 0.08)
        b.linear(w["first"], w["o"], self.heads_out["q"])
        b.linear(w["second"], w["lo"], self.heads_out["lq"])
        b.add(w["logits"], w["first"], w["second"])
        b.argmax(w["choice"], w["logits"])


def plain_decode(backend, half, prompts, steps):
    """Token by token, each sequence's run of one."""
    model = Model(backend, half)
    lengths, last, said = np.zeros(3, np.float32), None, [[] for _ in prompts]
    for at in range(max(map(len, prompts)) + steps):
        tokens = np.array([p[at] if at < len(p) else s[-1] for p, s in zip(prompts, said)],
                          np.float32)
        w = model.buffers(3)
        model.run(w, f32(backend, tokens), f32(backend, [0, 1, 2, 3]), None,
                  f32(backend, lengths), None)
        last = backend.read(w["choice"])
        for i, p in enumerate(prompts):
            if at >= len(p) - 1:
                said[i].append(int(last[i]))
        lengths += 1
    return said


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_drafted_decoding_says_what_plain_decoding_says(backend, half, graph):
    """Prompts in one run, then trees whose branches hold some of the true tokens: the
    emitted tokens are those of decoding one at a time.  Largest logits stand apart by far
    more than the order of sums moves them."""
    rng = np.random.default_rng(17)
    prompts = [list(rng.integers(0, 97, n)) for n in (9, 1, 4)]
    truth = plain_decode(backend, half, prompts, 32)
    model, b = Model(backend, half), backend
    runs = [len(p) for p in prompts]
    w = model.buffers(sum(runs) + 2)  # two padded tokens
    tokens = f32(b, sum(prompts, []) + [5, 6])
    model.run(w, tokens, f32(b, starts_of(runs)), None, f32(b, [0, 0, 0]), None)
    choice = b.read(w["choice"])
    said = [[int(choice[int(e) - 1])] for e in starts_of(runs)[1:]]
    assert [s[0] for s in said] == [t[0] for t in truth]
    lengths, n = f32(b, runs), 8
    # Slots for runs of up to n tokens; the graph is captured once.
    slot = {"tokens": b.allocate_f32((3 * n,)), "parents": b.allocate_f32((3 * n,)),
            "starts": b.allocate_f32((4,)), "lengths": b.allocate_f32((3,)),
            "mask": upload(b, np.zeros((3 * n, 1), np.uint8)),
            "emitted": b.allocate_f32((3, model.columns)), "counts": b.allocate_f32((3,)),
            "next": b.allocate_f32((3,)), "grown": b.allocate_f32((3,))}
    w = model.buffers(3 * n)

    def step():
        model.run(w, slot["tokens"], slot["starts"], slot["parents"], slot["lengths"], slot["mask"])
        b.settle_drafts(slot["emitted"], slot["counts"], slot["next"], model.caches,
                        slot["tokens"], w["choice"], slot["starts"], slot["parents"],
                        slot["lengths"], model.table)
        b.add(slot["grown"], slot["lengths"], slot["counts"])

    b.copy(slot["lengths"], lengths)
    b.copy(slot["starts"], f32(b, [0, 0, 0, 0]))
    step()  # of no runs: the workspace
    assert np.all(b.read(slot["counts"]) == 0) and np.all(b.read(slot["next"]) == -1)
    replay, end = captured(b, step) if graph else (step, lambda: None)
    accepted = 0
    for turn in range(4):
        drafted, parents, sizes = [], [], [8, 5, 7] if turn % 2 else [3, 8, 1]
        for s, t, size in zip(said, truth, sizes):
            tree = random_tree(rng, size)
            tree[1:] = np.maximum(tree[1:], 0)
            depth = ancestors(tree).sum(axis=1) - 1
            at = len(s) - 1
            # The true token of a place on some branches, others elsewhere.
            drafted += [s[-1] if i == 0 else t[at + d] if rng.random() < 0.7
                        else (t[at + d] + 1) % 97 for i, d in enumerate(depth)]
            parents += list(tree)
        pad = 3 * n - len(drafted)
        b.copy(slot["tokens"], f32(b, drafted + [0] * pad))
        b.copy(slot["parents"], f32(b, parents + [-1] * pad))
        b.copy(slot["starts"], f32(b, starts_of(sizes)))
        replay()
        emitted, counts = b.read(slot["emitted"]), b.read(slot["counts"]).astype(int)
        last, grown = b.read(slot["next"]), b.read(slot["grown"])
        for i in range(3):
            assert 1 <= counts[i] <= model.columns
            said[i] += [int(v) for v in emitted[i, :counts[i]]]
            assert last[i] == said[i][-1] and np.all(emitted[i, counts[i]:] == -1)
            assert said[i] == truth[i][:len(said[i])], (turn, i)
            accepted += counts[i] - 1
        b.copy(slot["lengths"], f32(b, grown))
        assert np.all(grown == [len(p) + len(s) - 1 for p, s in zip(prompts, said)])
    end()
    assert accepted > 3


def test_two_contexts_at_once():
    """Calls of two contexts, queued without waiting, equal each one's alone."""
    worlds = []
    for seed, shapes in ((1, [(900, 12), (33, 4)]), (2, [(2000, 7)])):
        backend = HipBackend(0)
        batch = Batch(seed, shapes, "tree", 16)
        keys, values = (random_pages(batch.rng, batch.pages, 2, 16, 64, True) for _ in range(2))
        query = batch.rng.standard_normal((batch.tokens, 512)).astype(np.float32)
        args = (upload(backend, query), upload(backend, keys), upload(backend, values),
                *batch.args(backend), GqaSpec(8, 2, 64))
        alone = backend.allocate_f32(query.shape)
        backend.paged_tree_gqa(alone, *args)
        worlds.append((backend, args, backend.read(alone),
                       [backend.allocate_f32(query.shape) for _ in range(20)]))
    for i in range(20):
        for backend, args, _, outs in worlds:
            backend.paged_tree_gqa(outs[i], *args)
    for backend, _, want, outs in worlds:
        assert all(np.array_equal(backend.read(out), want) for out in outs)
        backend.close()


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("rank,rope", [(512, 64), (512, 32), (130, 32)])
def test_latents_past_32_bits(backend, rank, rope, half):
    """Pages whose elements, or bytes, lie past 2^32, entered, settled and attended."""
    pages, size = 2000, 4096
    assert 1990 * size * (rank + rope) > (2 ** 32 if rank == 512 else 2 ** 30)
    rng = np.random.default_rng(5)
    cache = backend.alloc_pages(pages, 1, size, rank + rope, half)
    table = f32(backend, [[1999], [1990]])
    latent, key, query = (rng.standard_normal((4, w)).astype(np.float32) for w in (rank, rope, rope))
    out = backend.allocate_f32((4, rope))
    turn = backend.allocate_f32((8, rope))
    backend.rotation_table(turn, 1.0e4)
    backend.paged_latent_append(out, cache, upload(backend, query), upload(backend, latent),
                                upload(backend, key), None, turn, table,
                                f32(backend, [0, 0, 0, 1]), f32(backend, [0, 1, 1, 0]),
                                f32(backend, [0, 1, 2, 0]), 1, False, EPSILON)
    emitted, counts, last = (backend.allocate_f32(s) for s in ((2, 4), (2,), (2,)))
    # The second child is accepted and moves to place 1.
    backend.settle_drafts(emitted, counts, last, [cache], f32(backend, [1, 2, 3, 1]),
                          f32(backend, [3, 9, 8, 7]), f32(backend, [0, 3, 4]),
                          f32(backend, [-1, 0, 0, -1]), f32(backend, [0, 0]), table)
    assert backend.read(counts).tolist() == [2, 1] and backend.read(last).tolist() == [8, 7]
    # A query that meets one row alone: the others' scores are far below.
    result = backend.allocate_f32((2, rank))
    want = latent.astype(np.float16).astype(np.float32) if half else latent
    big = np.stack([want[2], want[3]]) * 40
    backend.paged_latent_attention(result, upload(backend, big), backend.allocate_f32((2, rope)),
                                   cache, table, None, f32(backend, [1, 0]), None, 1, 1.0)
    assert np.all(np.abs(backend.read(result) - want[2:]) <= 4 * F32 * np.abs(want[2:]))
    del cache


# ---- refusals -----------------------------------------------------------------------------------

def refused(variant, call, *args):
    with pytest.raises(ExecutorError) as error:
        call(*args)
    assert error.value.variant == variant, error.value


def changed(arguments, **of):
    return [of.get(name, value) for name, value in arguments.items()]


def test_layout_refusals(backend):
    a = backend.allocate_f32
    good = dict(sequences=a((6,)), positions=a((6,)), places=a((6,)),
                mask=upload(backend, np.zeros((6, 1), np.uint8)), starts=a((3,)), parents=a((6,)),
                lengths=a((2,)))
    call = backend.draft_layout
    call(*good.values())
    call(*changed(good, parents=None, mask=None))
    for name, other, variant in (
            ("positions", a((5,)), "InvalidShape"), ("places", a((6, 1)), "InvalidShape"),
            ("starts", a((2,)), "InvalidShape"), ("parents", a((7,)), "InvalidShape"),
            ("lengths", a((2, 1)), "InvalidShape"), ("mask", a((6, 1)), "InvalidDType"),
            ("mask", upload(backend, np.zeros((6, 0), np.uint8)), "InvalidShape"),
            ("mask", upload(backend, np.zeros((5, 1), np.uint8)), "InvalidShape"),
            ("places", good["positions"], "InvalidArgument"),
            ("sequences", good["parents"], "InvalidArgument"),
            ("sequences", good["mask"], "InvalidDType")):
        refused(variant, call, *changed(good, **{name: other}))


def test_runs_beyond_the_longest_list(backend):
    a = backend.allocate_f32
    most = 65536
    for count in (most, most + 1):
        layout = [a((1,)), a((1,)), a((1,)), None, a((count + 1,)), None, a((count,))]
        attention = [a((1, 64)), a((1, 64)), backend.alloc_pages(1, 1, 8, 64),
                     backend.alloc_pages(1, 1, 8, 64), a((count, 1)), a((count + 1,)),
                     a((count,)), None, GqaSpec(1, 1, 64)]
        settle = [a((count, 1)), a((count,)), a((count,)), [], a((1,)), a((1,)), a((count + 1,)),
                  None, a((count,)), a((count, 1))]
        for call, arguments in ((backend.draft_layout, layout), (backend.paged_tree_gqa, attention),
                                (backend.settle_drafts, settle)):
            if count > most:
                refused("Overflow", call, *arguments)
            else:
                call(*arguments)
    backend.synchronize()


def test_many_sequences(backend):
    # The last of the longest list's runs has all three tokens.
    most = 65536
    starts = np.zeros(most + 1, np.float32)
    starts[-1] = 3
    outputs = [backend.allocate_f32((3,)) for _ in range(3)]
    backend.draft_layout(*outputs, None, f32(backend, starts), None,
                         f32(backend, np.full(most, 5, np.float32)))
    got = [backend.read(o) for o in outputs]
    assert np.array_equal(got, [[most - 1] * 3, [5, 6, 7], [5, 6, 7]])


def test_attention_refusals(backend):
    a = backend.allocate_f32
    pages = lambda *shape: backend.alloc_pages(*shape)  # noqa: E731
    good = dict(output=a((6, 256)), query=a((6, 256)), key_pages=pages(3, 2, 8, 64),
                value_pages=pages(3, 2, 8, 64), tables=a((2, 4)), starts=a((3,)), lengths=a((2,)),
                mask=upload(backend, np.zeros((6, 1), np.uint8)), spec=GqaSpec(4, 2, 64))
    call = backend.paged_tree_gqa
    call(*good.values())
    for name, other, variant in (
            ("output", a((6, 255)), "InvalidShape"), ("query", a((6, 128)), "InvalidShape"),
            ("output", good["query"], "InvalidArgument"), ("tables", a((3, 4)), "InvalidShape"),
            ("starts", a((4,)), "InvalidShape"), ("starts", None, "InvalidShape"),
            ("lengths", a((3,)), "InvalidShape"), ("value_pages", good["key_pages"], "InvalidArgument"),
            ("value_pages", pages(3, 2, 8, 32), "InvalidShape"),
            ("mask", a((6, 1)), "InvalidDType"),
            ("mask", upload(backend, np.zeros((5, 1), np.uint8)), "InvalidShape"),
            ("spec", GqaSpec(3, 2, 64), "InvalidShape"), ("spec", GqaSpec(4, 2, 32), "InvalidShape")):
        refused(variant, call, *changed(good, **{name: other}))
    refused("Unsupported", call, a((2, 1025)), a((2, 1025)), pages(1, 1, 8, 1025),
            pages(1, 1, 8, 1025), a((2, 1)), None, a((2,)), None, GqaSpec(1, 1, 1025))
    good = dict(output=a((6, 4 * 128)), latent_query=a((6, 4 * 128)), rotary_query=a((6, 4 * 32)),
                pages=pages(3, 1, 8, 160), tables=a((2, 4)), starts=a((3,)), lengths=a((2,)),
                mask=None, heads=4, scale=0.1)
    call = backend.paged_latent_attention
    call(*good.values())
    for name, other, variant in (
            ("output", a((6, 4 * 160)), "InvalidShape"), ("rotary_query", a((6, 100)), "InvalidShape"),
            ("rotary_query", a((5, 128)), "InvalidShape"), ("pages", pages(3, 2, 8, 160), "InvalidShape"),
            ("pages", pages(3, 1, 8, 192), "InvalidShape"), ("heads", 3, "InvalidShape"),
            ("heads", 0, "InvalidArgument"), ("scale", 0.0, "InvalidArgument"),
            ("scale", NAN, "InvalidArgument"), ("output", good["latent_query"], "InvalidArgument"),
            ("starts", None, "InvalidShape")):
        refused(variant, call, *changed(good, **{name: other}))


def test_entry_refusals(backend):
    a = backend.allocate_f32
    good = dict(query_out=a((2, 64)), pages=backend.alloc_pages(3, 1, 8, 48), query=a((2, 64)),
                latent=a((2, 32)), key=a((2, 16)), weight=a((32,)), rotation=a((5, 16)),
                tables=a((2, 2)), sequences=a((2,)), positions=a((2,)), places=a((2,)), heads=4,
                interleaved=False, epsilon=EPSILON)
    call = backend.paged_latent_append
    call(*good.values())
    call(*changed(good, sequences=None, places=None, weight=None))
    for name, other, variant in (
            ("query_out", a((2, 32)), "InvalidShape"), ("query", a((2, 60)), "InvalidShape"),
            ("latent", a((2, 31)), "InvalidShape"), ("latent", a((2, 49)), "InvalidShape"),
            ("key", a((2, 15)), "InvalidShape"), ("key", a((3, 16)), "InvalidShape"),
            ("weight", a((16,)), "InvalidShape"), ("rotation", a((5, 14)), "InvalidShape"),
            ("tables", a((2,)), "InvalidShape"), ("sequences", a((3,)), "InvalidShape"),
            ("places", a((3,)), "InvalidShape"), ("positions", a((1,)), "InvalidShape"),
            ("heads", 0, "InvalidArgument"), ("epsilon", 0.0, "InvalidArgument"),
            ("pages", backend.alloc_pages(3, 2, 8, 48), "InvalidShape"),
            ("query_out", good["query"], "InvalidArgument")):
        refused(variant, call, *changed(good, **{name: other}))
    pages = [backend.alloc_pages(2, 1, 8, 16) for _ in range(2)]
    call = lambda places: backend.paged_qk_norm_rope_at(  # noqa: E731
        a((2, 16)), *pages, a((2, 16)), a((2, 16)), a((2, 16)), None, None, a((4, 16)), a((2, 1)),
        None, a((2,)), places, PagedRopeSpec(1, 1, 16), EPSILON)
    call(f32(backend, [0, 1]))
    refused("InvalidShape", call, a((3,)))
    refused("InvalidDType", call, upload(backend, np.zeros(2, np.uint8)))


def test_settling_refusals(backend):
    a = backend.allocate_f32
    pages = backend.alloc_pages(3, 2, 8, 4)
    good = dict(emitted=a((2, 4)), counts=a((2,)), next=a((2,)), pages=[pages], tokens=a((6,)),
                choices=a((6,)), starts=a((3,)), parents=a((6,)), lengths=a((2,)), tables=a((2, 1)))
    call = backend.settle_drafts
    call(*good.values())
    for name, other, variant in (
            ("emitted", a((3, 4)), "InvalidShape"), ("emitted", a((2, 0)), "InvalidShape"),
            ("emitted", a((2, 1025)), "Unsupported"), ("counts", a((3,)), "InvalidShape"),
            ("next", a((1,)), "InvalidShape"), ("choices", a((5,)), "InvalidShape"),
            ("starts", a((2,)), "InvalidShape"), ("parents", a((5,)), "InvalidShape"),
            ("tables", a((3, 1)), "InvalidShape"), ("pages", [pages, pages], "InvalidArgument"),
            ("pages", [pages, backend.alloc_pages(3, 2, 16, 4)], "InvalidShape"),
            ("pages", [a((3, 4))], "InvalidShape"), ("next", good["counts"], "InvalidArgument"),
            ("counts", good["lengths"], "InvalidArgument")):
        refused(variant, call, *changed(good, **{name: other}))


def test_u8_readbacks(backend):
    values = np.arange(300, dtype=np.uint8).reshape(30, 10)
    buffer = upload(backend, values)
    assert np.array_equal(backend.read_u8(buffer), values)
    with pytest.raises(ExecutorError) as error:
        backend.read(buffer)
    assert error.value.variant == "InvalidDType"
    with pytest.raises(ExecutorError) as error:
        backend.read_u8(backend.allocate_f32((3,)))
    assert error.value.variant == "InvalidDType"
    limited = HipBackend(0, limits=Limits(max_total_bytes=64 << 20))
    small = limited.upload_u8_classified((1000,), values.reshape(-1)[:300].repeat(4)[:1000], SCRATCH)
    readback = limited.read_u8_async(small)
    assert limited.resource_report().pending_operation_bytes == 1000
    while readback.poll_step() is None:
        pass
    assert limited.resource_report().pending_operation_bytes == 0
    limited.close()
