"""How near attention of runs comes to 64 bits.

f32 caches are read as three bfloat16 parts, of whose nine products six are formed; queries and
probabilities over binary16 caches are two binary16 parts.  A part or product that is lost
moves outputs by 1e-6 of their norm and more (the CPU test forms each of these), f32's own
roundings by less:

- a score's sums, of 2 to 20 steps and values of a few units: 1e-7 to 3e-7;
- its place on the line of exponents, up to 16 units: 2^-21 / sqrt(3) log 2 = 1.9e-7;
- the exponential: 6e-8;
- a lane's sum of n / 4 weights and an output's of n / 32 products in two or three parts, each step
  within 2^-24 of sums that grow to their last value: 2^-24 / sqrt(3) sqrt(n / 12) and less,
  2.2e-7 for 512 keys.

Together 4e-7, which TOLERANCE is two and a half times.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

from test_draft_gpu import Batch, random_pages, run_latent, run_tree, say

TOLERANCE = 1.0e-6


def relative(got, want):
    """The error's norm by the outputs', over the rows of runs."""
    mine = ~np.isnan(want).any(axis=tuple(range(1, want.ndim)))
    got, want = got.reshape(want.shape)[mine], want[mine]
    return float(np.linalg.norm(got - want) / np.linalg.norm(want))


# ---- what a lost part would do, on the CPU --------------------------------------------------

def parts(x, bits, count):
    """x as `count` parts of `bits` significant bits, each the nearest to what is left."""
    out = []
    for _ in range(count):
        mantissa, exponent = np.frexp(x)
        part = np.ldexp(np.rint(np.ldexp(mantissa, bits)), exponent - bits)
        out.append(part)
        x = x - part
    return out


def attended(score_of, value_of, query, keys, values, scale):
    """Softmax attention with the two products formed by `score_of` and `value_of`."""
    score = score_of(query, keys.T) * scale
    p = np.exp(score - score.max(axis=1, keepdims=True))
    return value_of(p, values) / p.sum(axis=1, keepdims=True)


def products(bits, a_parts, b_parts, pairs):
    """A product of operands in parts, of the given pairs of them."""
    def form(a, b):
        x, y = parts(a, bits, a_parts), parts(b, bits, b_parts)
        return sum(x[i] @ y[j] for i, j in pairs)
    return form


SIX = [(0, 0), (0, 1), (1, 0), (0, 2), (1, 1), (2, 0)]


@pytest.mark.parametrize("dim,dv", [(32, 32), (64, 64), (80, 80), (128, 128), (256, 256), (192, 128),
                                    (576, 512)])
def test_lost_parts_pass_the_tolerance(dim, dv):
    rng = np.random.default_rng(dim)
    query = 2 * rng.standard_normal((40, dim)).astype(np.float32).astype(np.float64)
    keys = rng.standard_normal((480, dim)).astype(np.float32).astype(np.float64)
    values = rng.standard_normal((480, dv)).astype(np.float32).astype(np.float64)
    scale = 1 / math.sqrt(dim)
    f32 = products(8, 3, 3, SIX)
    want = attended(np.matmul, np.matmul, query, keys, values, scale)
    assert relative(attended(f32, f32, query, keys, values, scale), want) < 0.1 * TOLERANCE
    for pair in SIX:
        less = products(8, 3, 3, [other for other in SIX if other != pair])
        for score_of, value_of in ((less, f32), (f32, less)):
            off = relative(attended(score_of, value_of, query, keys, values, scale), want)
            assert off > 1.1 * TOLERANCE, (pair, off)
    # Binary16: 11 bits a part; keys and values are such already.
    keys, values = (parts(x, 11, 1)[0] for x in (keys, values))
    want = attended(np.matmul, np.matmul, query, keys, values, scale)
    two, one = products(11, 2, 1, [(0, 0), (1, 0)]), products(11, 1, 1, [(0, 0)])
    assert relative(attended(two, two, query, keys, values, scale), want) < 0.2 * TOLERANCE
    for score_of, value_of in ((one, two), (two, one)):
        assert relative(attended(score_of, value_of, query, keys, values, scale), want) > 50 * TOLERANCE


# ---- every kernel ---------------------------------------------------------------------------

# Rows to a sequence decide which kernel of a width runs: few and many, in items of every size.
RUNS = {"few": [(470, 4), (100, 3), (31, 1), (201, 6)], "many": [(300, 60), (100, 40), (0, 70)]}


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("dim", [32, 64, 80, 96, 112, 128, 160, 192, 256])
@pytest.mark.parametrize("which", list(RUNS))
@pytest.mark.parametrize("kind", ["chain", "tree"])
def test_heads_are_as_near_as_f32(backend, kind, which, dim, half):
    say("near", kind, which, dim, half)
    batch = Batch(dim + half, RUNS[which], kind, 16)
    keys, values = (random_pages(batch.rng, batch.pages, 2, 16, dim, half) for _ in range(2))
    query = 2 * batch.rng.standard_normal((batch.tokens, 6 * dim)).astype(np.float32)
    got = run_tree(backend, batch, query, keys, values, 6, 2, dim)
    want, _ = batch.attend(query.reshape(-1, 6, dim), keys, values, 1 / math.sqrt(dim))
    off = relative(got, want)
    say(off)
    assert off < TOLERANCE


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("rank,rope", [(512, 64), (512, 32), (256, 64), (256, 32), (128, 64),
                                       (128, 32), (64, 0), (256, 0)])
@pytest.mark.parametrize("heads,shapes", [
    (4, [(480, 1), (33, 4), (200, 3)]), (12, [(480, 1), (33, 4), (200, 3)]),
    (40, [(480, 1), (100, 3)]), (16, [(300, 30), (0, 45)])])
def test_latents_are_as_near_as_f32(backend, heads, shapes, rank, rope, half):
    say("near", heads, rank, rope, half)
    batch = Batch(rank + rope + half, shapes, "tree", 16)
    pages = random_pages(batch.rng, batch.pages, 1, 16, rank + rope, half)
    latent, rotary = (2 * batch.rng.standard_normal((batch.tokens, heads * w)).astype(np.float32)
                      for w in (rank, rope))
    scale = float(np.float32(1 / math.sqrt(rank + rope)))
    got = run_latent(backend, batch, latent, rotary, pages, heads, scale)
    query = np.concatenate([x.reshape(batch.tokens, heads, -1 if x.size else 0)
                            for x in (latent, rotary)], axis=2)
    want, _ = batch.attend(query, pages, pages[..., :rank], scale)
    off = relative(got, want)
    say(off)
    assert off < TOLERANCE
