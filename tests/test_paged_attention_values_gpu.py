"""Paged decode attention where single weights, values or pages are extreme: a
key far above long tails of others, infinite and NaN values, sequences without
any key in the cache.

Tolerance of the tails, with u = 2^-24, n keys and head size D: a weight is off
by the factor 2 (D + 6) u S_max (its score: D products, scaled; S_max the
largest sum of their sizes) and 2^-22 (ex2.approx), numerator and denominator
each, and their sums round by (n + 16) u each: with A = sum p_j |V_j|,
A (4 (D + 6) u S_max + 2 (n + 16) u + 2^-20).  16-bit kernels hold a weight as
two values of the type, 2^-16 relative.  In FP16 the second one's step ends at
2^-24, of weights that are scaled so that the largest is 2^15: half a step is
2^-40 of the largest weight, 2^-40 sum |V_j| / sum w with sum w >= 1.
"""
from __future__ import annotations

import math

import pytest
import torch

from test_paged_cache_gpu import (TYPES, U, Paged, clean_watchdog, close, gen,  # noqa: F401
                                  names, randn, watchdog)

pytestmark = pytest.mark.gpu
HALF_TYPES = [torch.float16, torch.bfloat16]


# ------------------------------------------------------------- long tails

def sink_inputs(dtype, heads, kv_heads, dim, batch, tail, gap, seed, sink):
    """`batch` sequences over the same pages: key `sink` scores `gap` above the
    `tail` others (all zero), and its value is 0."""
    g = gen(seed)
    page = 64
    n = tail + 1
    pages = -(-n // page)
    k = torch.zeros(pages, page, kv_heads, dim, dtype=dtype, device="cuda")
    v = (torch.rand(pages, page, kv_heads, dim, generator=g, device="cuda") + 0.5).to(dtype)
    k[sink // page, sink % page, :, 0] = gap
    v[sink // page, sink % page] = 0
    q = randn(g, batch, heads, dim, dtype=dtype)
    q[:, :, 0] = 1
    table = torch.arange(pages, device="cuda", dtype=torch.int32).repeat(batch, 1)
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    return q, k, v, table, lens


@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("gap", [12.0, 17.0, 17.25, 17.375, 18.0, 20.0, 22.0])
@pytest.mark.parametrize("heads,kv_heads,dim,batch,tail,sink", [
    (4, 4, 64, 450, 8192, 0), (4, 4, 64, 450, 8192, 4100), (16, 1, 128, 1200, 4096, 0),
    (6, 1, 80, 1, 131070, 7), (12, 1, 256, 3, 20000, 0), (4, 2, 71, 2, 5000, 60)])
def test_tail_far_below_one_key(ops, dtype, gap, heads, kv_heads, dim, batch, tail, sink):
    """Many keys far below one whose value is 0: the tail is the result.  With
    many sequences a warp holds a whole one, with few it is cut."""
    q, k, v, table, lens = sink_inputs(dtype, heads, kv_heads, dim, batch, tail, gap, dim, sink)
    got = ops.paged_attention(q, k, v, table, lens, 1.0)
    n = tail + 1
    values = v.reshape(-1, kv_heads, dim)[:n].double()
    weight = math.exp(-float(k[sink // 64, sink % 64, 0, 0]))
    total = 1 + tail * weight
    want = (values.sum(0) * weight / total).repeat_interleave(heads // kv_heads, 0)
    slack = want * (4 * (dim + 6) * U * gap + 2 * (n + 16) * U + 2.0 ** -20)
    if dtype != torch.float32:
        slack = slack + 2.0 ** -16 * want
    if dtype == torch.float16:
        slack = slack + 2.0 ** -40 * values.sum(0).repeat_interleave(heads // kv_heads, 0) / total
    close(got, want.expand_as(got), slack)


# ------------------------------------------------- infinite and NaN values

@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("heads", [2, 12, 16, 32])
@pytest.mark.parametrize("dim", [64, 80, 128, 192, 256, 71])
@pytest.mark.parametrize("lens", [[100, 40], [3000, 70], [100] * 900], ids=lambda x: f"{len(x)}x{x[0]}")
def test_infinite_values(ops, dtype, heads, dim, lens):
    """Column d of key-value head 1 reads an infinity from key d (weights of
    all sizes): infinite, with its sign; NaN where both signs or a NaN are
    read; and nothing else changes."""
    cache = Paged(lens, 2, dim, 16, dtype, 25)
    q = randn(gen(1), len(lens), heads, dim, dtype=dtype)
    clean = ops.paged_attention(q, cache.k, cache.v, cache.table, cache.seq_lens)
    v = cache.v.clone()

    def put(key, column, value):
        v[cache.table[0, key // 16].long(), key % 16, 1, column] = value

    want = clean.clone()
    for column in range(0, dim - 8, 2):
        sign = 1 if column % 4 else -1
        put(column % 100, column, sign * math.inf)
        want[0, heads // 2:, column] = sign * math.inf
    for column, values in ((dim - 1, (math.inf, -math.inf)), (dim - 3, (math.nan,)),
                           (dim - 5, (math.inf, math.nan)), (dim - 7, (-math.inf, -math.inf))):
        for key, value in zip((3, 90), values):
            put(key, column, value)
        want[0, heads // 2:, column] = math.nan if dim - column < 7 else -math.inf
    got = ops.paged_attention(q, cache.k, v, cache.table, cache.seq_lens)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("heads", [1, 8, 16])
@pytest.mark.parametrize("gap", [8.0, 16.0, 24.0, 40.0, 80.0])
def test_infinite_value_of_small_weight(ops, dtype, heads, gap):
    """An infinity counts as long as FP32 holds its weight (e^-87)."""
    q, k, v, table, lens = sink_inputs(dtype, heads, 1, 64, 3, 500, gap, 3, 200)
    v[1, 7, 0, 11] = math.inf
    v[5, 7, 0, 12] = -math.inf
    got = ops.paged_attention(q, k, v, table, lens, 1.0)
    assert (got[..., 11] == math.inf).all() and (got[..., 12] == -math.inf).all()
    got[..., 11:13] = 0
    assert got.isfinite().all()


# ------------------------------------------------------ no key in the cache

@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("heads", [2, 12, 32])
@pytest.mark.parametrize("dim", [64, 128, 256, 71])
@pytest.mark.parametrize("lens", [[40, 30], [6000, 70], [20] * 900], ids=lambda x: f"{len(x)}x{x[0]}")
def test_sequence_with_every_page_outside(ops, dtype, heads, dim, lens):
    """Its keys are left out, so it has none and gives zeros, whether one warp
    holds it or it is cut over many CTAs; the others keep their bits."""
    cache = Paged(lens, 2, dim, 16, dtype, 27)
    q = randn(gen(1), len(lens), heads, dim, dtype=dtype)
    clean = ops.paged_attention(q, cache.k, cache.v, cache.table, cache.seq_lens)
    table = cache.table.clone()
    table[0] = cache.k.shape[0]
    got = ops.paged_attention(q, cache.k, cache.v, table, cache.seq_lens)
    assert watchdog() == 0x6b02
    assert not got[0].any() and torch.equal(got[1:], clean[1:])


@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("heads", [2, 12, 32])
@pytest.mark.parametrize("dim", [64, 256, 71])
@pytest.mark.parametrize("n", [40, 6000])
def test_scores_all_minus_infinity(ops, dtype, heads, dim, n):
    """Keys that all score -inf are keys: 0 / 0, as the formula has it.  One
    finite score among them, or in another part of the sequence, is the
    result."""
    cache = Paged([n, 9], 2, dim, 16, dtype, 28)
    q = randn(gen(1), 2, heads, dim, dtype=dtype).abs()
    clean = ops.paged_attention(q, cache.k, cache.v, cache.table, cache.seq_lens)
    k = cache.k.clone()
    k[cache.table[0].long()] = -math.inf
    got = ops.paged_attention(q, k, cache.v, cache.table, cache.seq_lens)
    assert got[0].isnan().all() and torch.equal(got[1], clean[1])
    key = n - 3
    page = cache.table[0, key // 16].long()
    k[page, key % 16] = 0
    got = ops.paged_attention(q, k, cache.v, cache.table, cache.seq_lens)
    want = cache.v[page, key % 16].repeat_interleave(heads // 2, 0)
    assert torch.equal(got[0], want) and torch.equal(got[1], clean[1])


@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("heads", [2, 12, 32])
@pytest.mark.parametrize("dim", [64, 256, 71])
@pytest.mark.parametrize("n", [40, 6000])
def test_scores_all_nan(ops, dtype, heads, dim, n):
    """A query or keys that are no numbers: neither is the result, whole or cut."""
    cache = Paged([n, 9], 2, dim, 16, dtype, 29)
    q = randn(gen(1), 2, heads, dim, dtype=dtype)
    clean = ops.paged_attention(q, cache.k, cache.v, cache.table, cache.seq_lens)
    bad = q.clone()
    bad[0, 0] = math.nan
    got = ops.paged_attention(bad, cache.k, cache.v, cache.table, cache.seq_lens)
    assert got[0, 0].isnan().all()
    assert torch.equal(got[0, 1:], clean[0, 1:]) and torch.equal(got[1], clean[1])
    k = cache.k.clone()
    k[cache.table[0].long(), :, 1] = math.nan
    got = ops.paged_attention(q, k, cache.v, cache.table, cache.seq_lens)
    assert got[0, heads // 2:].isnan().all()
    assert torch.equal(got[0, :heads // 2], clean[0, :heads // 2])
    assert torch.equal(got[1], clean[1])
