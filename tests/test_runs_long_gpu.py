"""Attention of runs where its blocks walk many tiles: prompts, and long caches of many sequences.

A kernel keeps up to four tiles on their way to LDS, in a ring of stages, and the places of 512
runs of eight keys, in a ring of two halves.  Each case's blocks walk at least twice the stages
and pass the end of a half, which the plan's arithmetic here says beforehand.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import numpy as np
import pytest

from runtime_amd.backend import GqaSpec
from test_draft_gpu import Batch, random_pages, say, upload

pytestmark = pytest.mark.gpu

CUS = 256


class Plan(NamedTuple):
    """Query rows of an item, keys of a tile, blocks on a CU, stages of tiles; whether tiles are
    copied to LDS, with the places of runs of eight keys in a ring."""
    rows: int
    keys: int
    resident: int
    stages: int
    copied: bool

    def walks(self, batch, group, kv_heads):
        """(first, last) tile of every part of an item that a block holds."""
        own = 8 if self.resident == 3 else 5  # units besides an item's tiles
        masked = batch.kind in ("tree", "bits")
        items = []  # (units, tiles)
        for length, n in zip(batch.lengths.astype(int), batch.runs):
            each = []
            for tile in range(-(-n * group // self.rows)):
                seen = n if masked else min(n, (self.rows * (tile + 1) - 1) // group + 1)
                if masked or n == 1:
                    units = own + -(-(length + n) // self.keys)
                else:
                    step = max(1, self.rows // self.keys)
                    every = max(1, self.keys // self.rows) * group
                    units = own + -(-length // self.keys) + step + tile // every * step
                each.append((units, -(-(length + seen) // self.keys)))
            items += each * kv_heads
        total = sum(units for units, _ in items)
        blocks = min(total, CUS * self.resident, 1024)
        starts = [b * total // blocks for b in range(blocks + 1)]
        found, at, block = [], 0, 0
        for units, tiles in items:
            while starts[block + 1] <= at:
                block += 1
            b = block
            while b < blocks and starts[b] < at + units:
                place = [min(max(u - at, 0), units) for u in (starts[b], starts[b + 1])]
                first, last = (tiles if u == units else min(max(u - own, 0), tiles) for u in place)
                found.append((first, last))
                b += 1
            at += units
        return found

    def check(self, batch, group, kv_heads):
        walks = self.walks(batch, group, kv_heads)
        half = 2048 // self.keys  # tiles of a half of the ring
        longest = max(last - first for first, last in walks)
        # Refills inside of the loop, where the tile stages - 1 ahead starts a half.
        refills = sum(any(tile % half == 0 for tile in range(first + self.stages - 1, last))
                      for first, last in walks)
        say("walks of up to", longest, "tiles,", self.stages, "stages,", refills, "refills")
        assert longest >= 2 * self.stages
        assert refills > 0 or not self.copied


# By (width, format, whether sequences have more than 64 rows on average), as the kernels' shapes
# give them.
HEADS = {
    (64, True, True): Plan(128, 64, 2, 4, True), (64, True, False): Plan(64, 64, 2, 4, True),
    (128, True, True): Plan(64, 32, 3, 3, True), (128, True, False): Plan(64, 64, 2, 2, True),
    (192, True, False): Plan(64, 32, 1, 4, True), (256, True, False): Plan(64, 32, 1, 4, True),
    (96, True, True): Plan(128, 32, 2, 2, False), (96, True, False): Plan(64, 64, 2, 2, False),
    (64, False, False): Plan(64, 64, 2, 1, False), (128, False, False): Plan(64, 32, 1, 1, False),
}
# By (rank, rope, format, whether more than 32 rows); f32 of rank 512 up to 16 rows: 16 an item.
LATENTS = {
    (512, 64, True, False): Plan(32, 32, 1, 3, True), (512, 64, True, True): Plan(64, 32, 1, 3, True),
    (256, 64, True, False): Plan(32, 32, 1, 4, True), (128, 64, True, False): Plan(32, 32, 1, 4, True),
    (128, 64, True, True): Plan(64, 32, 1, 4, True), (512, 32, True, False): Plan(32, 32, 1, 2, False),
    (512, 64, False, False): Plan(16, 32, 1, 1, False),
    (512, 64, False, True): Plan(32, 32, 1, 1, False),
}


class Long(Batch):
    """Runs over long caches, all of whose pages are of a small pool, some more than once."""

    def __init__(self, seed, shapes, kind, size, pool=40):
        super().__init__(seed, shapes, kind, size)
        self.pages = pool
        self.table = self.rng.integers(0, pool, self.table.shape).astype(np.float32)


def near(batch, got, want, bound):
    """Within the worst case's bound, and the norm of all that f32's roundings make of it: 4e-7
    for 512 keys, as sqrt(n) from there, two and a half times."""
    got = got.reshape(want.shape)
    assert np.all(np.abs(got - want) <= bound)
    keys = max(batch.lengths + batch.runs)
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    say("off by", off)
    assert off < 1.0e-6 * max(1.0, math.sqrt(keys / 512))


def attend_heads(backend, batch, query, keys, values, heads, kv_heads, dim):
    out = upload(backend, np.full(query.shape, 7.0, np.float32))
    args = (upload(backend, query), upload(backend, keys), upload(backend, values),
            *batch.args(backend), GqaSpec(heads, kv_heads, dim))
    backend.paged_tree_gqa(out, *args)
    got = backend.read(out)
    for _ in range(3):  # the same each time
        backend.paged_tree_gqa(out, *args)
        assert np.array_equal(got, backend.read(out), equal_nan=True)
    return got


PROMPT = [(2048, 2048)]
MANY = [(2500, 32), (1900, 30), (2100, 18), (4000, 32)] * 12
FEW = [(2600, 4), (2100, 3), (2300, 1), (4100, 4)] * 16


@pytest.mark.parametrize("dim,half,shapes,kind", [
    (64, True, PROMPT, "chain"), (64, True, MANY, "tree"), (64, True, FEW, "chain"),
    (64, True, FEW, "bits"), (128, True, PROMPT, "chain"), (128, True, MANY, "tree"),
    (128, True, FEW, "tree"), (192, True, PROMPT, "chain"), (192, True, FEW, "tree"),
    (256, True, MANY, "bits"), (256, True, FEW, "chain"), (96, True, MANY, "tree"),
    (96, True, FEW, "chain"), (64, False, PROMPT, "chain"), (64, False, MANY, "tree"),
    (128, False, MANY, "chain"), (128, False, FEW, "tree")],
    ids=lambda v: "%dx%d" % (len(v), v[0][1]) if isinstance(v, list) else
    {True: "f16", False: "f32"}.get(v, str(v)) if isinstance(v, bool) else str(v))
def test_long_walks_of_heads(backend, dim, half, shapes, kind):
    say("long", dim, half, len(shapes), shapes[0], kind)
    heads, kv_heads = 8, 2
    batch = Long(dim + half, shapes, kind, 16)
    many = batch.tokens * 4 > 64 * len(shapes)
    plan = HEADS.get((dim, half, many)) or HEADS[dim, half, False]
    plan.check(batch, 4, kv_heads)
    keys, values = (random_pages(batch.rng, batch.pages, kv_heads, 16, dim, half) for _ in range(2))
    query = 2 * batch.rng.standard_normal((batch.tokens, heads * dim)).astype(np.float32)
    got = attend_heads(backend, batch, query, keys, values, heads, kv_heads, dim)
    near(batch, got, *batch.attend(query.reshape(-1, heads, dim), keys, values, 1 / math.sqrt(dim)))


@pytest.mark.parametrize("rank,rope,half,heads,shapes,kind", [
    (512, 64, True, 8, FEW, "chain"), (512, 64, True, 40, FEW[:20], "tree"),
    (512, 64, True, 6, PROMPT, "chain"), (256, 64, True, 6, FEW, "tree"),
    (128, 64, True, 8, FEW, "bits"), (128, 64, True, 40, FEW[:20], "chain"),
    (512, 32, True, 8, FEW, "tree"), (512, 64, False, 4, FEW, "tree"),
    (512, 64, False, 12, FEW[:20], "chain")])
def test_long_walks_of_latents(backend, rank, rope, half, heads, shapes, kind):
    say("long", rank, rope, half, heads, len(shapes), shapes[0], kind)
    batch = Long(rank + half, shapes, kind, 16)
    rows = batch.tokens * heads / len(shapes)
    LATENTS[rank, rope, half, rows > (32 if half else 16)].check(batch, heads, 1)
    pages = random_pages(batch.rng, batch.pages, 1, 16, rank + rope, half)
    latent, rotary = (2 * batch.rng.standard_normal((batch.tokens, heads * w)).astype(np.float32)
                      for w in (rank, rope))
    scale = float(np.float32(1 / math.sqrt(rank + rope)))
    out = upload(backend, np.full(latent.shape, 7.0, np.float32))
    table, starts, lengths, mask = batch.args(backend)
    args = (upload(backend, latent), upload(backend, rotary), upload(backend, pages), table, starts,
            lengths, mask, heads, scale)
    backend.paged_latent_attention(out, *args)
    got = backend.read(out)
    for _ in range(3):
        backend.paged_latent_attention(out, *args)
        assert np.array_equal(got, backend.read(out))
    query = np.concatenate([x.reshape(batch.tokens, heads, -1) for x in (latent, rotary)], axis=2)
    near(batch, got, *batch.attend(query, pages, pages[..., :rank], scale))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("what", ["page", "key"])
def test_what_is_bad_in_a_long_walk(backend, dim, what):
    """A page without an id, or a key that is not finite, among a prompt's own tokens: those before
    it are as without it.  One among the cached keys reaches every row of its sequence alone."""
    say("bad", dim, what)
    shapes = [(1900, 1400), (2100, 700), (2300, 3)]
    batch = Batch(dim, shapes, "chain", 16)
    many = batch.tokens * 4 > 64 * len(shapes)
    (HEADS.get((dim, True, many)) or HEADS[dim, True, False]).check(batch, 4, 2)
    keys, values = (random_pages(batch.rng, batch.pages, 2, 16, dim, True) for _ in range(2))
    query = batch.rng.standard_normal((batch.tokens, 8 * dim)).astype(np.float32)
    want, bound = batch.attend(query.reshape(-1, 8, dim), keys, values, 1 / math.sqrt(dim))
    reached = np.zeros((batch.tokens, 8), bool)
    if what == "page":
        # Places 2912 to 2927: tokens 1012 on of the first run; of the third, all.
        batch.table[0, 182], batch.table[2, 100] = -1, 1e6
        reached[1012:1400] = reached[2100:] = True
    else:
        place = 1900 + 1012
        keys[int(batch.table[0, place // 16]), 0, place % 16, 3] = np.nan
        values[int(batch.table[2, 100]), 1, 7, dim - 1] = np.inf
        reached[1012:1400, :4] = True
        reached[2100:, 4:] = True
    got = attend_heads(backend, batch, query, keys, values, 8, 2, dim).reshape(want.shape)
    assert not np.any(np.isfinite(got[reached]).all(axis=-1))
    assert np.all(np.abs(got[~reached] - want[~reached]) <= bound[~reached])
