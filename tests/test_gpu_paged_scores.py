"""Paged attention with scores far from zero: the powers' reference is then a
large number whose own rounding is of the order of the differences between
scores, or larger. Queries and keys are chosen so that every score is exact in
fp32 and the softmax of the exact scores is known to the last bits."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import paged_util as pu
from test_gpu_paged import DTYPES, i32, randh

pytestmark = pytest.mark.gpu


def cache_of(ops, rng, dtype, keys, scales, page, values=None):
    """A cache of one sequence: keys [n, d] (fp16 values, or codes with scales
    [n]) and values [n, d] (random ones by default) for every kv head. Returns
    it with the float64 values as cached [hkv, n, d]."""
    hkv = 2
    n, d = keys.shape
    table, n_pages = pu.page_table(rng, [n], page)
    cache, _, v = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    ids = torch.from_numpy(table[0].astype(np.int64))

    def put(to, rows):
        full = torch.ones(len(ids) * page, *rows.shape[1:], dtype=rows.dtype)
        full[:n] = rows
        to[ids.cuda()] = full.view(len(ids), 1, page, *rows.shape[1:]).expand(-1, hkv, page, *rows.shape[1:]).cuda()

    put(cache.k_pages, keys)
    if scales is not None:
        put(cache.k_scales, scales)
    if values is None:
        return cache, pu.rows_of(v, table, 0, n)
    if dtype == torch.int8:
        code, scale = pu.quantise(values)
        put(cache.v_pages, code)
        put(cache.v_scales, scale)
        values = code.double() * scale.double()[:, None]
    else:
        put(cache.v_pages, values.half())
        values = values.half().double()
    return cache, values.expand(hkv, n, d)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,d", [(6, 64), (4, 128), (32, 64)])
@pytest.mark.parametrize("sign", [1, -1])
def test_one_position_is_its_value(cuda, ops, dtype, hq, d, sign):
    """Scores of 2^7 to 2^35 in log2 units: with one position the output is its
    value, whatever the score (the probability's rounding to fp16 and the
    result's: E16 each)."""
    rng = np.random.default_rng(51)
    for a in (25.0, 400.0, 1000.0, 2000.0, 4000.0, 8000.0, 16000.0, 20000.0, 33333.0, 60000.0):
        if dtype == torch.int8:
            keys, scales = torch.full((1, d), 127, dtype=torch.int8), torch.tensor([a / 127])
        else:
            keys, scales = torch.full((1, d), a).half(), None
        cache, v = cache_of(ops, rng, dtype, keys, scales, 8)
        q = torch.full((1, hq, d), sign * a, device="cuda").half()
        got = ops.attention_paged(q, cache, i32([0]), i32([0]))[0].cpu().double()
        want = v[:, 0].repeat_interleave(hq // 2, 0)
        assert ((got - want).abs() <= 2.01 * pu.E16 * want.abs() + pu.TINY16).all(), a


SIZES = [40, 600, 5000, 70000]  # warps of a CTA, a cluster, and parts that a second kernel joins


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("sign", [1, -1])
def test_equal_largest_scores_share_the_output(cuda, ops, dtype, n, sign):
    """Positions whose score is the largest, all others below by thousands of
    log2 units: the output is the mean of those positions' values. Scores up to
    2^29 in log2 units, a step of fp32 there being 32. Equal scores have equal
    powers and equal references in every warp and part, so besides E16 of the
    probability and of the result there are only the sums' roundings (two per
    16 positions of a warp, n / 16 for one warp alone)."""
    rng = np.random.default_rng(n)
    hq, d = 14, 64
    top = rng.permutation(n)[:7]
    for a, b in ((1024.0, 8192.0), (4096.0, 16384.0), (16384.0, 16384.0), (32768.0, 32768.0), (60000.0, 60000.0)):
        level = 1 - rng.integers(1, 8, n) / 16.0 if sign == 1 else 1 + rng.integers(1, 8, n) / 16.0
        level[top] = 1.0
        if dtype == torch.int8:
            # the same score from two codes and scales that differ by a factor of two
            keys = torch.zeros(n, d, dtype=torch.int8)
            keys[:, 3] = torch.from_numpy(np.where(np.arange(n) % 2 == 0, 64, 32).astype(np.int8))
            scales = torch.from_numpy(level * b / 64 * np.where(np.arange(n) % 2 == 0, 1.0, 2.0)).float()
        else:
            keys, scales = torch.zeros(n, d, dtype=torch.float16), None
            keys[:, 3] = torch.from_numpy(level * b / 2).half()
        q = torch.zeros(1, hq, d, dtype=torch.float16, device="cuda")
        q[:, :, 3] = sign * a
        q[:, 5, 3] = 0.0  # one head of the group far from the others: the mean of all values
        cache, v = cache_of(ops, rng, dtype, keys, scales, 16)
        got = ops.attention_paged(q, cache, i32([n - 1]), i32([0]))[0].cpu().double()
        for h in range(hq):
            rows = v[h // 7] if h == 5 else v[h // 7, top]
            want, size = rows.mean(0), rows.abs().mean(0)
            bound = (2 * pu.E16 + 4 * (n / 16 + 32) * pu.E32) * size + pu.TINY16
            assert ((got[h] - want).abs() <= bound).all(), (a, b, h)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("sign", [1, -1])
def test_parts_with_unequal_maxima_are_weighed_right(cuda, ops, dtype, n, sign):
    """Scores near +-2^19 in log2 units that differ by up to 5.4, constant over
    stretches of the sequence as the values are, so that warps and parts join
    with unequal references and outputs: a reference off by its own rounding
    (2^-5 there) would misweigh them by two percent.

    The exact products enter the powers unrounded. A power's exponent is off by
    the FMA's rounding (at most 2^-19 below 64), ex2's 2 units in the last place,
    the same again in each of two joins, and the scale's rounding on a
    difference of at most 8 (2^-21): 2^-16 bounds their sum. The probability's
    rounding and the result's are E16 each; the sums' roundings as above."""
    rng = np.random.default_rng(n + 1)
    hq, d = 14, 64
    at = np.arange(n) * 64 // n
    level = rng.permutation(64)[at] % 16
    values = torch.from_numpy(rng.standard_normal((64, d)))[torch.from_numpy(at)]
    q = torch.zeros(1, hq, d, dtype=torch.float16, device="cuda")
    if dtype == torch.int8:
        # one code, scales in steps of 2^-21: every product but the scale's is the same
        keys, q[:, :, 3] = torch.zeros(n, d, dtype=torch.int8), sign * 1024.0
        keys[:, 3] = 64
        scales = torch.from_numpy(64.0 * (1 + sign * level * 2.0 ** -21)).float()
        score = 1024.0 * sign * 64 * scales.double()
    else:
        # a product of 2^22 and one of up to 30 in steps of 2: 22 bits
        keys, scales = torch.zeros(n, d, dtype=torch.float16), None
        keys[:, 3], keys[:, 40] = 1024.0, torch.from_numpy(level * 2.0).half()
        q[:, :, 3], q[:, :, 40] = sign * 4096.0, 1.0
        score = sign * 2.0 ** 22 + keys[:, 40].double()
    cache, v = cache_of(ops, rng, dtype, keys, scales, 16, values)
    got = ops.attention_paged(q, cache, i32([n - 1]), i32([0]))[0].cpu().double()
    p = torch.softmax(score / math.sqrt(d), 0)
    for h in range(hq):
        want, size = p @ v[h // 7], p @ v[h // 7].abs()
        bound = (2 * pu.E16 + 2 * 2.0 ** -16 + 4 * (n / 16 + 32) * pu.E32) * size + pu.TINY16
        assert ((got[h] - want).abs() <= bound).all(), h


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_that_climb(cuda, ops, dtype):
    """Scores that rise from -2^26 to 2^26 along the sequence, through zero:
    the last position alone counts, or the first for the opposite query."""
    rng = np.random.default_rng(52)
    n, hq, d = 3000, 4, 128
    ramp = torch.linspace(-1, 1, n, dtype=torch.float64)
    if dtype == torch.int8:
        keys, scales = torch.zeros(n, d, dtype=torch.int8), 16384.0 / 64 * ramp.abs().float()
        keys[:, 9] = (64 * ramp.sign()).to(torch.int8)
    else:
        keys, scales = torch.zeros(n, d, dtype=torch.float16), None
        keys[:, 9] = (16384.0 * ramp).half()
    q = torch.zeros(1, hq, d, dtype=torch.float16, device="cuda")
    q[0, :, 9] = torch.tensor([30000.0, -30000.0, -30000.0, 30000.0])
    cache, v = cache_of(ops, rng, dtype, keys, scales, 32)
    got = ops.attention_paged(q, cache, i32([n - 1]), i32([0]))[0].cpu().double()
    score = (keys[:, 9].double() * (1 if scales is None else scales.double()))
    for h, way in enumerate((1, -1, -1, 1)):
        best = (way * score) == (way * score).max()
        want = v[h // 2, best].mean(0)
        assert ((got[h] - want).abs() <= 2.01 * pu.E16 * v[h // 2, best].abs().mean(0) + pu.TINY16).all()
