"""Runs of tokens on the GPU, where the helpers of the drafted trees' tests serve: layout of
long runs, settling of runs that the layout refuses, and attention at the ends of its ranges,
against plain implementations in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

from runtime_amd.backend import GqaSpec
from test_draft_gpu import (F32, NAN, Batch, Model, captured, check, f32, plain_decode, random_pages,
                            read_pages, refused, run_latent, run_layout, say, settled, starts_of,
                            tables_for, upload)

pytestmark = pytest.mark.gpu


# ---- long lists --------------------------------------------------------------------------------

def attended_page(query, keys, values, page, count):
    """(outputs, bound) in 64 bits of tokens that attend the first `count` places of a page each."""
    want, bound = np.empty(query.shape), np.empty(query.shape)
    dim = query.shape[1]
    for first in range(0, len(query), 40000):
        rows = slice(first, first + 40000)
        key, value = (x[page[rows], 0].astype(np.float64) for x in (keys, values))
        seen = np.arange(8) < count[rows, None]
        terms = key * query[rows, None] / math.sqrt(dim)
        score = np.where(seen, terms.sum(axis=2), -np.inf)
        p = np.exp(score - score.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        want[rows] = (p[..., None] * value).sum(axis=1)
        # As Batch.attend bounds it, of one tile.
        size = np.where(seen, np.abs(terms).sum(axis=2), 0).max(axis=1)[:, None]
        relative = 2 * (dim + 8) * F32 * size + 97 * F32
        bound[rows] = relative * (p[..., None] * np.abs(value)).sum(axis=1) + 2.0 ** -37
    return want, bound


@pytest.mark.parametrize("dim", [32, 20])
@pytest.mark.parametrize("count", [65536, 65537, 400000])
def test_many_sequences_of_a_token_each(backend, count, dim):
    """Without starts there is no list to look through, and no limit to it."""
    say("many", count, dim)
    rng = np.random.default_rng(count + dim)
    keys, values = (random_pages(rng, 97, 1, 8, dim, False) for _ in range(2))
    table = rng.integers(0, 97, (count, 1)).astype(np.float32)
    lengths = rng.integers(0, 8, count).astype(np.float32)
    lengths[[0, count // 2, -1]] = 8, NAN, 7
    query = rng.standard_normal((count, dim)).astype(np.float32)
    out = backend.allocate_f32((count, dim))
    backend.paged_tree_gqa(out, upload(backend, query), upload(backend, keys),
                           upload(backend, values), upload(backend, table), None,
                           upload(backend, lengths), None, GqaSpec(1, 1, dim))
    got = backend.read(out)
    bad = np.isnan(lengths) | (lengths == 8)  # a ninth token has no page
    assert np.all(np.isnan(got[bad])) and bad.sum() == 2
    want, bound = attended_page(query, keys, values, table[:, 0].astype(int),
                                np.where(bad, 1, lengths + 1))
    assert np.all(np.abs(got - want)[~bad] <= bound[~bad])


@pytest.mark.parametrize("dim", [32, 20])
def test_the_longest_list_of_starts(backend, dim):
    """65536 runs of no, one and two tokens: attended, and settled."""
    say("starts", dim)
    count, rng = 65536, np.random.default_rng(dim)
    runs = rng.integers(0, 3, count)
    starts = starts_of(runs, 3)
    sequence = np.repeat(np.arange(count), runs)
    tokens, number = 3 + len(sequence) + 2, np.arange(len(sequence)) + 3 - starts[sequence]
    lengths = rng.integers(0, 7, count).astype(np.float32)
    # Each sequence has a page of its own, which settling changes.
    keys, values = (random_pages(rng, count, 1, 8, dim, False) for _ in range(2))
    table = rng.permutation(count).astype(np.float32)[:, None]
    query = rng.standard_normal((tokens, dim)).astype(np.float32)
    out = upload(backend, np.full(query.shape, 7.0, np.float32))
    caches = [upload(backend, keys), upload(backend, values)]
    given = [upload(backend, table), f32(backend, starts), upload(backend, lengths)]
    backend.paged_tree_gqa(out, upload(backend, query), *caches, *given, None, GqaSpec(1, 1, dim))
    got = backend.read(out)
    mine = slice(3, 3 + len(sequence))
    want, bound = attended_page(query[mine], keys, values, table[sequence, 0].astype(int),
                                lengths[sequence] + number + 1)
    assert np.all(np.abs(got[mine] - want) <= bound)
    assert np.all(got[:3] == 7) and np.all(got[-2:] == 7)
    drafted, choices = rng.integers(0, 2, (2, tokens)).astype(np.float32)
    got = settle_at(backend, starts, None, drafted, choices, lengths, table, 2, caches, None)
    want = settled(starts, None, drafted, choices, lengths.astype(int), table, 8, 2, [keys, values])
    for g, w in zip(got, want):
        assert np.array_equal(g, w)
    assert set(want[1]) == {0, 1, 2}
    for buffer, array in zip(caches, (keys, values)):
        assert np.array_equal(backend.read(buffer), array)


def test_extents_of_runs_past_the_index_range(backend):
    a = backend.allocate_f32
    # Rows: 2^25 at most.
    pages = [backend.alloc_pages(1, 1, 8, 1) for _ in range(2)]
    for tokens in (512, 513):
        given = [a((tokens, 65535)), a((tokens, 65535)), *pages, a((tokens, 1)), None, a((tokens,)),
                 None, GqaSpec(65535, 1, 1)]
        if tokens == 512:
            backend.paged_tree_gqa(*given)
        else:
            refused("Overflow", backend.paged_tree_gqa, *given)
    # Units: 64 heads of 2^24 places a row are 2^24 for each sequence, and some more.
    pages = [backend.alloc_pages(1, 64, 4096, 64) for _ in range(2)]
    for sequences in (126, 127):
        given = [a((sequences, 4096)), a((sequences, 4096)), *pages, a((sequences, 4096)), None,
                 a((sequences,)), None, GqaSpec(64, 64, 64)]
        if sequences == 126:
            backend.paged_tree_gqa(*given)
            assert np.all(backend.read(given[0]) == 0)
        else:
            refused("Overflow", backend.paged_tree_gqa, *given)


# ---- layout of long runs ------------------------------------------------------------------------

def laid_out(parents, length, bytes_):
    """(positions, places, bad) of one run, by one pass over it; mask rows where bytes_ > 0."""
    n = len(parents)
    depth, rows = np.full(n, -1), np.zeros((n, bytes_), np.uint8)
    for i, parent in enumerate(parents):
        if bytes_ and i >= 8 * bytes_:
            continue
        if parent == -1:
            depth[i] = 0
        elif 0 <= parent < i and parent == int(parent) and depth[int(parent)] >= 0:
            depth[i] = depth[int(parent)] + 1
            rows[i] = rows[int(parent)]
        else:
            continue
        if bytes_:
            rows[i, i // 8] |= 1 << i % 8
    good = depth >= 0
    return (np.where(good, length + depth, -1), np.where(good, length + np.arange(n), -1), good, rows)


@pytest.mark.parametrize("runs,bytes_", [
    ([65], 9), ([64, 66, 127, 128, 129], 17), ([1000], 125), ([700, 3, 2048], 200), ([500], 0),
    ([300], 1)])
@pytest.mark.parametrize("kind", ["chain", "tree", "star", "far", "bad"])
def test_layout_of_long_runs(backend, kind, runs, bytes_):
    say("layout", kind, runs, bytes_)
    rng = np.random.default_rng(sum(runs) + bytes_)
    parents = []
    for n in runs:
        i = np.arange(n)
        each = {"chain": i - 1, "star": np.where(i, 0, -1), "far": np.floor(rng.random(n) * i),
                }.get(kind, i - 1 - np.floor(rng.random(n) * np.minimum(i, 9))).astype(np.float32)
        each[0] = -1
        if kind == "bad":
            each[rng.integers(0, n, 2)] = NAN, 0.5
            each[rng.integers(1, n, 3)] = n, -2, -1
        parents.append(each)
    lengths, starts = rng.integers(0, 9000, len(runs)), starts_of(runs, 1)
    tokens = int(starts[-1]) + 1
    flat = np.concatenate([[0], *parents, [0]])
    got, mask = run_layout(backend, starts, flat, lengths, tokens, bytes_)
    for s, n in enumerate(runs):
        at = slice(int(starts[s]), int(starts[s]) + n)
        positions, places, good, rows = laid_out(parents[s], lengths[s], bytes_)
        assert np.array_equal(got[0][at], np.where(good, s, -1))
        assert np.array_equal(got[1][at], positions)
        assert np.array_equal(got[2][at], places)
        assert mask is None or np.array_equal(mask[at], rows)
    assert all(out[0] == out[-1] == -1 for out in got)


def test_layout_of_the_longest_runs(backend):
    """Time grows as the run, not as its square: a chain of 300000 takes some 4 ms."""
    n = 300000
    rng = np.random.default_rng(1)
    i = np.arange(n)
    for parents in (i - 1, np.where(i, i - 1 - np.floor(rng.random(n) * np.minimum(i, 99)), -1)):
        say("layout", parents[-1])
        got, _ = run_layout(backend, [0, n], parents, [5], n, 0)
        positions, places, _, _ = laid_out(parents, 5, 0)
        assert np.array_equal(got, [np.zeros(n), positions, places])
    # A length that leaves no places.
    got, _ = run_layout(backend, [0, n], i - 1, [2 ** 24 - n + 1], n, 0)
    assert np.all(np.array(got) == -1)


# ---- scales of latents ------------------------------------------------------------------------

@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("rank,rope", [(64, 0), (128, 0), (256, 0), (128, 64), (512, 64), (30, 6)])
@pytest.mark.parametrize("scale,size", [(1e-20, 1e-27), (1e-44, 1.0), (1e-30, 1e30)])
def test_scales_and_queries_whose_product_vanishes(backend, scale, size, rank, rope, half):
    """Scores of about 0: each row is the mean of the values that it attends."""
    say("scale", scale, size, rank, rope, half)
    batch = Batch(rank + half, [(70, 9), (0, 5)], "tree", 16)
    pages = random_pages(batch.rng, batch.pages, 1, 16, rank + rope, half)
    batch.spoil(pages)
    latent, rotary = ((size * batch.rng.standard_normal((14, 4 * w))).astype(np.float32)
                      for w in (rank, rope))
    scale = float(np.float32(scale))
    got = run_latent(backend, batch, latent, rotary, pages, 4, scale)
    query = np.concatenate([x.reshape(14, 4, -1 if x.size else 0) for x in (latent, rotary)], axis=2)
    want, bound = batch.attend(query, pages, pages[..., :rank], scale)
    check(got.reshape(want.shape), want, bound, 7.0)


def test_scales_beyond_f32(backend):
    """Scores are formed times log2 e: scales that pass f32 with it are refused."""
    a, pages = backend.allocate_f32, backend.alloc_pages(1, 1, 8, 64)
    given = [a((1, 64)), a((1, 64)), a((1, 0)), pages, a((1, 1)), None, a((1,)), None, 1]
    for scale in (2.35e38, 1e-45):
        backend.paged_latent_attention(*given, scale)
        assert np.all(backend.read(given[0]) == 0)  # one key of zeros
    for scale in (2.36e38, 3.4e38, np.inf, -1.0):
        refused("InvalidArgument", backend.paged_latent_attention, *given, scale)


# ---- settling ------------------------------------------------------------------------------

def settle_at(backend, starts, parents, tokens, choices, lengths, table, columns, caches, places):
    n = len(lengths)
    outs = [upload(backend, np.full(shape, 9.0, np.float32)) for shape in ((n, columns), (n,), (n,))]
    backend.settle_drafts(*outs, caches, f32(backend, tokens), f32(backend, choices),
                          f32(backend, starts), None if parents is None else f32(backend, parents),
                          f32(backend, lengths), upload(backend, table),
                          places=None if places is None else f32(backend, places))
    return [backend.read(o) for o in outs]


@pytest.mark.parametrize("given", [False, True], ids=["alone", "places"])
def test_settling_of_runs_whose_first_token_follows_another(backend, given):
    """The layout refuses them, so nothing was stored for them: no token is accepted."""
    rng = np.random.default_rng(4)
    firsts = [NAN, 0, 5, -2, -0.5, -1]
    starts, lengths = starts_of([4] * 6), [3, 0, 9, 2, 5, 7]
    tokens = np.arange(24, dtype=np.float32) % 4
    choices = np.roll(tokens, -1)
    parents = np.tile(np.array([0, 0, 0, 2], np.float32), 6)  # the first child never drafted
    parents[::4] = firsts
    choices[::4] = 2  # the second child, which moves
    pages, table = tables_for(rng, [16] * 6, 8)
    old = random_pages(rng, pages, 2, 8, 5, False)
    cache = upload(backend, old)
    (_, _, places), _ = run_layout(backend, starts, parents, lengths, 24, 1)
    assert np.array_equal(places, [-1] * 20 + [7, 8, 9, 10])
    emitted, counts, last = settle_at(backend, starts, parents, tokens, choices, lengths, table, 4,
                                      [cache], places if given else None)
    for got in (emitted[:5], counts[:5], last[:5]):
        assert np.all(np.isnan(got))
    want = settled(starts[5:], parents, tokens, choices, lengths[5:], table[5:], 8, 4, [old])
    for got, w in zip((emitted, counts, last), want):
        assert np.array_equal(got[5], w[0])
    assert counts[5] == 3
    assert np.array_equal(backend.read(cache), old)


@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
def test_settling_stops_where_tokens_have_no_place(backend, tree):
    """Tokens past the mask's last bit were not stored: the path ends before them."""
    rng = np.random.default_rng(5)
    runs, lengths = [12, 100, 3, 9], [4, 30, 0, 11]
    starts = starts_of(runs)
    # In the tree odd tokens are one branch, even ones another, which is accepted.
    parents = np.concatenate([np.maximum(np.arange(n) - 2, -1) if tree else np.arange(n) - 1
                              for n in runs])
    if tree:
        parents[starts[:-1].astype(int) + 1] = 0
    tokens = np.concatenate([np.arange(n) for n in runs])
    choices = tokens + (2 if tree else 1)
    pages, table = tables_for(rng, [160] * 4, 16)
    old = random_pages(rng, pages, 1, 16, 6, True)
    cache = upload(backend, old)
    (_, _, places), _ = run_layout(backend, starts, parents, lengths, sum(runs), 1)
    got = settle_at(backend, starts, parents if tree else None, tokens, choices, lengths, table, 64,
                    [cache], places)
    # As of runs of the tokens that have one.
    short = [min(n, 8) for n in runs]
    keep = np.concatenate([int(a) + np.arange(n) for a, n in zip(starts, short)])
    want = settled(starts_of(short), parents[keep], tokens[keep], choices[keep], lengths, table, 16,
                   64, [old])
    for g, w in zip(got, want):
        assert np.array_equal(g, w)
    assert got[1].tolist() == ([4, 4, 2, 4] if tree else [8, 8, 3, 8])
    assert np.array_equal(read_pages(backend, cache), old.astype(np.float32))
    # Places that are not the tokens' own are none; without the first one the sequence is bad.
    places[3] += 1
    places[12], places[113] = -1, NAN
    got = settle_at(backend, starts, parents if tree else None, tokens, choices, lengths, table, 64,
                    [cache], places)
    assert np.array_equal(got[1], [4, NAN, 2, 4] if tree else [3, NAN, 1, 8], equal_nan=True)


def test_settling_refusals_of_places(backend):
    a = backend.allocate_f32
    pages = backend.alloc_pages(3, 2, 8, 4)
    good = [a((2, 4)), a((2,)), a((2,)), [pages], a((6,)), a((6,)), a((3,)), a((6,)), a((2,)),
            a((2, 1))]
    backend.settle_drafts(*good, places=a((6,)))
    for places, variant in ((a((5,)), "InvalidShape"), (a((6, 1)), "InvalidShape"),
                            (good[0], "InvalidShape"), (pages, "InvalidShape"),
                            (upload(backend, np.zeros(6, np.uint8)), "InvalidDType")):
        refused(variant, backend.settle_drafts, *good, places)
    # Outputs of as many sequences as tokens.
    good = [a((2, 4)), a((2,)), a((2,)), [], a((2,)), a((2,)), a((3,)), None, a((2,)), a((2, 1))]
    for places in good[1:3]:
        refused("InvalidArgument", backend.settle_drafts, *good, places)


# ---- together -----------------------------------------------------------------------------------

@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
def test_drafts_longer_than_the_mask(backend, graph):
    """Drafts of 12 tokens, all of them true, where the mask has eight bits: eight are accepted a
    step, and decoding goes on as one token at a time does."""
    prompts = [[5, 80, 3], [11], [40, 41]]
    truth = plain_decode(backend, True, prompts, 30)
    model, b, n = Model(backend, True), backend, 12
    said = [[t[0]] for t in truth]
    w = model.buffers(6)
    model.run(w, f32(b, sum(prompts, [])), f32(b, starts_of([3, 1, 2])), None, f32(b, [0, 0, 0]), None)
    w = model.buffers(3 * n)
    tokens, starts, lengths = f32(b, np.zeros(3 * n)), f32(b, np.zeros(4)), f32(b, [3, 1, 2])
    mask = upload(b, np.zeros((3 * n, 1), np.uint8))
    parents = f32(b, np.tile(np.arange(n) - 1, 3))
    emitted, counts, last = b.allocate_f32((3, 16)), b.allocate_f32((3,)), b.allocate_f32((3,))
    grown = b.allocate_f32((3,))

    def step():
        model.run(w, tokens, starts, parents, lengths, mask)
        b.settle_drafts(emitted, counts, last, model.caches, tokens, w["choice"], starts, parents,
                        lengths, model.table, places=w["place"])
        b.add(grown, lengths, counts)

    step()  # of no runs: the workspace
    replay, end = captured(b, step) if graph else (step, lambda: None)
    b.copy(starts, f32(b, starts_of([n] * 3)))
    for _ in range(3):
        b.copy(tokens, f32(b, np.concatenate([t[len(x) - 1:len(x) - 1 + n]
                                              for t, x in zip(truth, said)])))
        replay()
        got, count = b.read(emitted), b.read(counts)
        assert count.tolist() == [8, 8, 8]
        for i in range(3):
            said[i] += [int(v) for v in got[i, :8]]
            assert said[i] == truth[i][:len(said[i])]
        b.copy(lengths, grown)
    end()
    assert [len(x) for x in said] == [25] * 3
