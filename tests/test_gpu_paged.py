"""The paged KV cache on the GPU: norm + RoPE + append, read back, decode
attention, against plain forms in 64 bits (paged_util). Bounds follow from the
roundings counted there."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_util as pu
from gpu_util import canary_intact, dev

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.int8]


def i32(a):
    return dev(np.asarray(a, np.int32), torch.int32)


def randh(rng, *shape, scale=1.0):
    return torch.from_numpy(rng.standard_normal(shape) * scale).half()


def flags(device="cuda:0"):
    return torch.zeros(1, dtype=torch.int32, device=device)


def check_append(ops, rng, dtype, hq, hkv, d, page, positions, seqs, n_seqs, bias=None, norm=None, theta=1e4,
                 packed=False, in_place=False, eps=1e-6):
    """Runs one append and compares q, the written rows and everything else of
    the cache; returns the cache."""
    t = len(positions)
    q, k, v = randh(rng, t, hq, d), randh(rng, t, hkv, d), randh(rng, t, hkv, d)
    bq, bk, bv = ((randh(rng, n * d).to(bias) for n in (hq, hkv, hkv)) if bias else (None,) * 3)
    qn, kn = ((1 + randh(rng, d, scale=0.2)).to(norm) for _ in range(2)) if norm else (None, None)
    lengths = [1 + max([p for p, s in zip(positions, seqs) if s == b], default=0) for b in range(n_seqs)]
    table, n_pages = pu.page_table(rng, lengths, page)
    cache, k0, v0 = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    before = [x.clone() for x in (cache.k_pages, cache.v_pages)]
    scales0 = [None if x is None else x.clone() for x in (cache.k_scales, cache.v_scales)]
    if packed:
        whole = torch.cat([x.flatten(1) for x in (q, k, v)], 1).cuda()
        qd, kd, vd = (x.unflatten(1, (-1, d)) for x in whole.split((hq * d, hkv * d, hkv * d), 1))
    else:
        qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
    q_out = None if in_place else torch.full((t, hq, d), -3.0, dtype=torch.float16, device="cuda")
    err = flags()
    on = [None if x is None else x.cuda() for x in (bq, bk, bv, qn, kn)]
    got_q = ops.qkv_norm_rope_kv_append_paged(qd, kd, vd, cache, i32(positions), i32(seqs), theta, *on, eps=eps,
                                              q_out=q_out, err_flags=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    (wq, wk, wv), (sq, sk, sv) = pu.norm_rope(q, k, v, bq, bk, bv, qn, kn, eps, theta, positions)
    assert got_q.shape == (t, hq, d)
    bad = (got_q.cpu().double() - wq).abs() > pu.f16_bound(wq, sq)
    assert not bad.any(), f"q: {int(bad.sum())} of {bad.numel()}"
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)  # k and v are read only
    place = [(int(table[s, p // page]), p % page) for p, s in zip(positions, seqs)]
    pages = torch.tensor([x for x, _ in place])
    rows = torch.tensor([y for _, y in place])
    for name, tensor, scale, want, size, old, old_scale in (
            ("k", cache.k_pages, cache.k_scales, wk, sk, before[0], scales0[0]),
            ("v", cache.v_pages, cache.v_scales, wv, sv, before[1], scales0[1])):
        got = tensor.cpu()[pages, :, rows]
        if dtype == torch.float16:
            assert not ((got.double() - want).abs() > pu.f16_bound(want, size)).any(), name
        else:
            s = scale.cpu()[pages, :, rows].double()
            amax = want.abs().amax(-1)
            # scale: the maximum's error, the division's rounding
            assert ((s - amax / 127).abs() <= (pu.ROPE_ERR * size[..., 0] + 4 * pu.E32 * amax) / 127).all(), name
            # a code is the nearest whole number of x / scale, whose error is that of x and of the scale
            slack = 127 * (pu.ROPE_ERR * size / amax[..., None] * 2 + 8 * pu.E32)
            exact = want / (amax[..., None] / 127)
            assert ((got.double() - exact).abs() <= 0.5 + slack).all(), name
            assert int(got.abs().max()) == 127
        # every other row is as it was
        touched = torch.zeros(tensor.shape[0], tensor.shape[2], dtype=torch.bool)
        touched[pages, rows] = True
        keep = ~touched[:, None, :].expand(-1, hkv, -1)
        assert torch.equal(tensor.cpu()[keep], old.cpu()[keep]), name
        if scale is not None:
            assert torch.equal(scale.cpu()[keep], old_scale.cpu()[keep]), name
    return cache


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page,bias,norm", [
    (14, 2, 64, 16, torch.float16, None),            # Qwen2.5-0.5B heads, biases, no norm
    (32, 32, 128, 64, None, torch.float16),          # Llama-2-7B heads, norms
    (5, 1, 64, 8, torch.float32, torch.float32),     # odd head count, fp32 parameters
    (9, 3, 128, 256, torch.float16, torch.float32),
    (16, 1, 64, 32, None, None),                     # rotation only
])
def test_append(cuda, ops, dtype, hq, hkv, d, page, bias, norm):
    rng = np.random.default_rng(hq * 100 + page)
    # ragged: a chunk of 37 tokens continuing at 5, one token at 600, a chunk from 0, in mixed order
    positions = [600, *range(5, 42), *range(0, 20)]
    seqs = [2] + [0] * 37 + [1] * 20
    order = rng.permutation(len(positions))
    check_append(ops, rng, dtype, hq, hkv, d, page, [positions[i] for i in order], [seqs[i] for i in order], 3,
                 bias=bias, norm=norm)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("packed,in_place", [(True, False), (True, True), (False, True)])
def test_append_strided_and_in_place(cuda, ops, dtype, packed, in_place):
    rng = np.random.default_rng(3)
    check_append(ops, rng, dtype, 6, 2, 64, 16, list(range(33)), [0] * 33, 1, bias=torch.float16,
                 norm=torch.float16, packed=packed, in_place=in_place)
    check_append(ops, rng, dtype, 4, 4, 128, 16, [7], [1], 2, bias=torch.float16, packed=packed, in_place=in_place)


@pytest.mark.parametrize("hq,hkv,d,n", [
    (14, 2, 64, 301), (32, 8, 128, 301),
    (14, 2, 64, 4100),    # tokens that share a CTA
    (32, 8, 128, 1400),   # three sets of heads per warp
    (40, 8, 128, 1100),   # two
])
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_many_tokens(cuda, ops, dtype, hq, hkv, d, n):
    """A decode batch: one token per sequence at scattered positions."""
    rng = np.random.default_rng(8)
    check_append(ops, rng, dtype, hq, hkv, d, 16, rng.integers(0, 50, n).tolist(), rng.permutation(n).tolist(),
                 n, norm=torch.float16, bias=torch.float16, theta=1e6)


def test_append_far_positions_keep_their_phase(cuda, ops):
    """Position 10^6 at the fastest frequency: an fp32 angle would be 0.03 rad
    off, hundreds of times the bound."""
    rng = np.random.default_rng(5)
    hq, hkv, d, page = 2, 2, 64, 1 << 20
    table = np.zeros((1, 1), np.int32)
    cache = ops.PagedKVCache.allocate(1, page, hkv, d, 1, 1)
    cache.page_table.copy_(torch.from_numpy(table))
    positions = [999_983, (1 << 20) - 1, 524_287, 0]
    q, k, v = randh(rng, 4, hq, d), randh(rng, 4, hkv, d), randh(rng, 4, hkv, d)
    out = torch.empty(4, hq, d, dtype=torch.float16, device="cuda")
    ops.qkv_norm_rope_kv_append_paged(q.cuda(), k.cuda(), v.cuda(), cache, i32(positions), i32([0] * 4), 1e4,
                                      q_out=out)
    (wq, wk, _), (sq, sk, _) = pu.norm_rope(q, k, v, None, None, None, None, None, 0.0, 1e4, positions)
    assert not ((out.cpu().double() - wq).abs() > pu.f16_bound(wq, sq)).any()
    got = cache.k_pages[0, :, torch.tensor(positions, device="cuda")].permute(1, 0, 2).cpu().double()
    assert not ((got - wk).abs() > pu.f16_bound(wk, sk)).any()
    assert torch.equal(out[3].cpu(), q[3])  # position 0 turns nothing


def test_append_matches_the_head_major_operator(cuda, ops):
    """With page_size = max_seq and the slot as the only page, the paged
    operator fills the head-major cache that attention_head_major reads; both
    operators' rows differ by their roundings (the biased value's to fp16, E16,
    and that of the fp32 angle, at most position * E32) and no more."""
    rng = np.random.default_rng(12)
    hq, hkv, d, max_seq, n = 14, 2, 64, 512, 40
    q, k, v = randh(rng, n, hq, d), randh(rng, n, hkv, d), randh(rng, n, hkv, d)
    bq, bk, bv = randh(rng, hq * d), randh(rng, hkv * d), randh(rng, hkv * d)
    positions, slots = i32(np.tile(np.arange(20), 2) + 300), i32(np.repeat([2, 0], 20))
    head_major = [torch.zeros(3, hkv, max_seq, d, dtype=torch.float16, device="cuda") for _ in range(2)]
    q1 = q.cuda().clone()
    on = [x.cuda() for x in (bq, bk, bv)]
    ops.qkv_bias_rope_kv_append(q1, k.cuda(), v.cuda(), *on, positions, slots, 1e6, *head_major)
    cache = ops.PagedKVCache(*(torch.zeros_like(x) for x in head_major), i32([[0], [1], [2]]))
    q2 = ops.qkv_norm_rope_kv_append_paged(q.cuda().clone(), k.cuda(), v.cuda(), cache, positions, slots, 1e6, *on)
    for a, b in ((q1, q2), (head_major[0], cache.k_pages), (head_major[1], cache.v_pages)):
        size = b.double().abs().amax(-1, keepdim=True) * 2
        assert ((a.double() - b.double()).abs() <= (3 * pu.E16 + 320 * pu.E32) * size + 2 * pu.TINY16).all()
    assert torch.equal(head_major[1], cache.v_pages)  # the value rows take one rounding in both


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_padding_and_bad_tokens_leave_everything(cuda, ops, dtype):
    from littlellm_b200 import _capi
    rng = np.random.default_rng(9)
    hq, hkv, d, page = 4, 2, 64, 8
    table = np.array([[0, 1], [2, 77], [-5, 3]], np.int32)  # 4 pages: 77 and -5 are no pages
    cache, _, _ = pu.random_cache(rng, ops, dtype, 4, hkv, page, d, table)
    q, k, v = (randh(rng, 8, h, d).cuda() for h in (hq, hkv, hkv))
    cases = [((-1, 0), 0), ((-1, 99), 0), ((-2, 0), _capi.FLAG_BAD_POSITION), ((16, 1), _capi.FLAG_BAD_POSITION),
             ((3, 3), _capi.FLAG_BAD_SEQ), ((3, -1), _capi.FLAG_BAD_SEQ), ((9, 1), _capi.FLAG_BAD_PAGE),
             ((0, 2), _capi.FLAG_BAD_PAGE)]
    tensors = [x for x in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales) if x is not None]
    before = [x.clone() for x in tensors]
    everything = 0
    for i, ((p, s), flag) in enumerate(cases):
        err = flags()
        out = torch.full((1, hq, d), -7.0, dtype=torch.float16, device="cuda")
        ops.qkv_norm_rope_kv_append_paged(q[i:i + 1], k[i:i + 1], v[i:i + 1], cache, i32([p]), i32([s]), 1e4,
                                          q_out=out, err_flags=err)
        assert int(err.item()) == flag, (p, s)
        assert bool((out == -7.0).all())
        everything |= flag
    err = flags()
    out = torch.full((8, hq, d), -7.0, dtype=torch.float16, device="cuda")
    ops.qkv_norm_rope_kv_append_paged(q, k, v, cache, i32([c[0][0] for c in cases]), i32([c[0][1] for c in cases]),
                                      1e4, q_out=out, err_flags=err)
    assert int(err.item()) == everything and bool((out == -7.0).all())
    assert all(torch.equal(a, b) for a, b in zip(tensors, before))
    ops.qkv_norm_rope_kv_append_paged(q, k, v, cache, i32([c[0][0] for c in cases]), i32([c[0][1] for c in cases]),
                                      1e4)  # no flag word: nothing to set
    torch.cuda.synchronize()


def test_append_special_rows_int8(cuda, ops):
    """Rows of zeros, tiny rows, one large value, infinities and NaN."""
    rng = np.random.default_rng(10)
    d, page = 64, 8
    cache = ops.PagedKVCache.allocate(1, page, 1, d, 1, 1, dtype=torch.int8)
    cache.page_table.zero_()
    k = torch.zeros(6, 1, d, dtype=torch.float16)
    k[1] = 2.0 ** -24                  # fp16's smallest value
    k[2, 0, 5] = 60000.0
    k[3] = randh(rng, 1, d)
    k[3, 0, 7] = float("inf")
    k[4] = randh(rng, 1, d)
    k[4, 0, 60] = float("nan")
    k[5] = randh(rng, 1, d)
    positions, seqs = i32(np.zeros(6)), i32(np.zeros(6))
    q = torch.zeros(6, 1, d, dtype=torch.float16, device="cuda")
    for i in range(6):  # one row each, all at position 0 (no rotation), read back one by one
        ops.qkv_norm_rope_kv_append_paged(q[i:i + 1], k[i:i + 1].cuda(), k[i:i + 1].cuda(), cache, positions[:1],
                                          seqs[:1], 1e4)
        rk, rv = ops.kv_read_paged(cache, positions[:1], seqs[:1])
        assert torch.equal(rk.cpu().view(torch.int16), rv.cpu().view(torch.int16))
        got, scale = rk.cpu().double()[0, 0], float(cache.k_scales[0, 0, 0])
        if i in (3, 4):
            assert np.isnan(scale) and torch.isnan(got).all()
            assert int(cache.k_pages[0, 0, 0].abs().max()) == 0
        elif i == 0:
            assert scale == 0.0 and (got == 0).all()
        else:
            want = k[i, 0].double()
            assert ((got - want).abs() <= 0.5 * want.abs().max() / 127 * (1 + 64 * pu.E32) + pu.E16 * want.abs()
                    + pu.TINY16).all()


# ---- read back ------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,d,page", [(2, 64, 16), (32, 128, 64), (3, 64, 8), (1, 128, 256)])
def test_read_token_rows(cuda, ops, dtype, hkv, d, page):
    """fp16 rows come back bit for bit, int8 rows as fp16(code * scale)."""
    rng = np.random.default_rng(hkv + page)
    lengths = [70, 1, 33]
    table, n_pages = pu.page_table(rng, lengths, page)
    cache, _, _ = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    pairs = [(p, s) for s, n in enumerate(lengths) for p in range(n)] + [(5, 0), (5, 0)]
    pairs = [pairs[i] for i in rng.permutation(len(pairs))]
    positions, seqs = i32([p for p, _ in pairs]), i32([s for _, s in pairs])
    err = flags()
    k, v = ops.kv_read_paged(cache, positions, seqs, err_flags=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    ids = torch.tensor([int(table[s, p // page]) for p, s in pairs], device="cuda")
    off = torch.tensor([p % page for p, _ in pairs], device="cuda")
    for got, pages, scales in ((k, cache.k_pages, cache.k_scales), (v, cache.v_pages, cache.v_scales)):
        want = pages[ids, :, off]
        if scales is not None:
            want = (want.float() * scales[ids, :, off][..., None]).half()
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("dtype", DTYPES)
def test_read_into_head_major(cuda, ops, dtype):
    """Rows land at [slot, head, position]; every other row stays, padding and
    bad tokens write nothing and are flagged."""
    from littlellm_b200 import _capi
    rng = np.random.default_rng(21)
    hkv, d, page, max_seq, n_slots = 2, 64, 16, 40, 3
    table, n_pages = pu.page_table(rng, [64, 30], page)
    table[1, 1] = n_pages  # positions 16.. of sequence 1 have no page
    cache, kd, vd = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    tokens = [(p, 0, 2, 0) for p in range(40)] + [(p, 1, 0, 0) for p in range(16)]
    tokens += [(-1, 0, 1, 0), (-1, 9, 9, 0), (40, 0, 1, _capi.FLAG_BAD_POSITION), (64, 0, 1, _capi.FLAG_BAD_POSITION),
               (-3, 0, 1, _capi.FLAG_BAD_POSITION), (3, 2, 1, _capi.FLAG_BAD_SEQ), (3, 0, 3, _capi.FLAG_BAD_SLOT),
               (3, 0, -1, _capi.FLAG_BAD_SLOT), (17, 1, 1, _capi.FLAG_BAD_PAGE)]
    k_whole = torch.full((n_slots * hkv * max_seq * d + 64,), -9.0, dtype=torch.float16, device="cuda")
    v_whole = k_whole.clone()
    shape = (n_slots, hkv, max_seq, d)
    k_out, v_out = k_whole[:-64].view(shape), v_whole[:-64].view(shape)
    for part in [tokens] + [[t] for t in tokens[-9:]]:
        err = flags()
        ops.kv_read_paged(cache, i32([t[0] for t in part]), i32([t[1] for t in part]), k_out=k_out, v_out=v_out,
                          out_slots=i32([t[2] for t in part]), err_flags=err)
        assert int(err.item()) == int(np.bitwise_or.reduce([t[3] for t in part]))
    for out, dense in ((k_out, kd), (v_out, vd)):
        want = torch.full(shape, -9.0, dtype=torch.float64)
        want[2] = pu.rows_of(dense, table, 0, 40)
        table_ok = table.copy()
        want[0, :, :16] = pu.rows_of(dense, table_ok, 1, 16)
        got = out.cpu().double()
        assert ((got - want).abs() <= 2 * pu.E16 * want.abs() + pu.TINY16).all()
        assert (got[1] == -9.0).all() and (got[0, :, 16:] == -9.0).all()
    assert canary_intact(k_whole, k_whole.numel() - 64, -9.0) and canary_intact(v_whole, v_whole.numel() - 64, -9.0)


def test_offsets_past_32_bits(cuda, ops):
    """A cache of 2^32 + codes per tensor: the last page is reached by append,
    read back and attention, and its low 32 bits alone would name page 0."""
    rng = np.random.default_rng(31)
    hkv, d, page = 2, 128, 1 << 15
    n_pages = (1 << 32) // (hkv * d * page) + 2
    k_pages = torch.empty(n_pages, hkv, page, d, dtype=torch.int8, device="cuda")
    v_pages = torch.empty_like(k_pages)
    k_pages[0] = 99
    v_pages[0] = 99
    scales = [torch.ones(n_pages, hkv, page, device="cuda") for _ in range(2)]
    cache = ops.PagedKVCache(k_pages, v_pages, i32([[n_pages - 1], [n_pages - 2]]), *scales)
    n = 70
    q, k, v = randh(rng, n, 4, d), randh(rng, n, hkv, d), randh(rng, n, hkv, d)
    for seq in (0, 1):
        positions, seqs = i32(np.arange(n)), i32(np.full(n, seq))
        rq = ops.qkv_norm_rope_kv_append_paged(q.cuda(), k.cuda(), v.cuda(), cache, positions, seqs, 1e4)
        rk, rv = ops.kv_read_paged(cache, positions, seqs)
        # half a step of amax / 127, the rounding of the value read back to fp16, and the scale's own
        amax = v.double().abs().amax(-1, keepdim=True)
        assert ((rv.cpu().double() - v.double()).abs() <= amax / 254 + 1.01 * pu.E16 * amax + 8 * pu.E32 * amax).all()
        out = ops.attention_paged(rq, cache, positions, seqs).cpu().double()
        at = n_pages - 1 - seq
        dense = [(p[at, :, :n].cpu().double() * s[at, :, :n].cpu().double()[..., None])
                 for p, s in ((k_pages, scales[0]), (v_pages, scales[1]))]
        for t in (0, 1, 31, 32, 69):
            want, bound = pu.attention(rq[t].cpu().double(), dense[0][:, :t + 1], dense[1][:, :t + 1])
            assert ((out[t] - want).abs() <= bound).all()
    assert bool((k_pages[0] == 99).all()) and bool((v_pages[0] == 99).all())


# ---- attention ------------------------------------------------------------------


def check_attention(ops, q, cache, dense, table, positions, seqs, **kw):
    """Runs attention_paged and compares each token; returns the output."""
    err = flags()
    out = ops.attention_paged(q, cache, i32(positions), i32(seqs), err_flags=err, **kw)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    got = out.cpu().double()
    worst = 0.0
    for t, (p, s) in enumerate(zip(positions, seqs)):
        if p == -1:
            assert (got[t] == 0).all()
            continue
        want, bound = pu.attention(q[t].cpu().double(), pu.rows_of(dense[0], table, s, p + 1),
                                   pu.rows_of(dense[1], table, s, p + 1))
        worst = max(worst, float(((got[t] - want).abs() / bound).max()))
    assert worst <= 1.0, f"{worst} of the bound"
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page,lengths", [
    (14, 2, 64, 16, [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 1000]),  # Qwen2.5-0.5B heads
    (32, 32, 128, 64, [1, 64, 65, 300, 511]),                             # Llama-2-7B heads
    (16, 1, 64, 8, [5, 8, 9, 640]),                                       # the largest group, the smallest page
    (8, 1, 128, 256, [1, 255, 256, 257, 2049]),                           # a full tile of heads
    (9, 1, 128, 32, [3, 100, 333]),                                       # one head past a tile
    (6, 2, 128, 16, [4096]),                                              # one long sequence: split
    (10, 5, 64, 128, [700, 1, 64]),
])
def test_attention(cuda, ops, dtype, hq, hkv, d, page, lengths):
    rng = np.random.default_rng(hq * 10 + d + page)
    table, n_pages = pu.page_table(rng, lengths, page)
    cache, k, v = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    order = rng.permutation(len(lengths))
    positions = [lengths[i] - 1 for i in order] + [-1]
    seqs = [int(i) for i in order] + [-1]
    q = randh(rng, len(positions), hq, d, scale=1.5).cuda()
    check_attention(ops, q, cache, (k, v), table, positions, seqs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,n_tok", [(2, 1), (2, 40), (1, 300), (8, 100)])
def test_attention_batches(cuda, ops, dtype, hkv, n_tok):
    """From one token (many parts) to batches that need none."""
    rng = np.random.default_rng(n_tok)
    hq, d, page = hkv * 4, 64, 16
    lengths = rng.integers(1, 400, n_tok)
    lengths[0] = 1500
    table, n_pages = pu.page_table(rng, lengths, page)
    cache, k, v = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    q = randh(rng, n_tok, hq, d, scale=2.0).cuda()
    check_attention(ops, q, cache, (k, v), table, (lengths - 1).tolist(), list(range(n_tok)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_long(cuda, ops, dtype):
    """One token over 40,001 positions (the most parts), and again with others beside it."""
    rng = np.random.default_rng(77)
    hq, hkv, d, page = 14, 2, 64, 64
    lengths = [40001, 39000, 7]
    table, n_pages = pu.page_table(rng, lengths, page)
    cache, k, v = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    q = randh(rng, 3, hq, d, scale=3.0).cuda()
    check_attention(ops, q[:1], cache, (k, v), table, [40000], [0])
    check_attention(ops, q, cache, (k, v), table, [40000, 38999, 6], [0, 1, 2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_of_one_position_is_its_value(cuda, ops, dtype):
    rng = np.random.default_rng(4)
    table, n_pages = pu.page_table(rng, [1, 20], 8)
    cache, k, v = pu.random_cache(rng, ops, dtype, n_pages, 2, 8, 64, table)
    q = randh(rng, 1, 6, 64).cuda()
    out = ops.attention_paged(q, cache, i32([0]), i32([0]))
    want = pu.rows_of(v, table, 0, 1)[:, 0].repeat_interleave(3, 0)
    # the probability's factor cancels but for one rounding of p * scale (int8) and of the quotient
    assert ((out[0].cpu().double() - want).abs() <= 2 * pu.E16 * want.abs() + pu.TINY16).all()
    if dtype == torch.float16:
        assert torch.equal(out[0].cpu(), want.half())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,page", [(64, 8), (64, 64), (128, 32)])
def test_attention_never_uses_rows_past_the_position(cuda, ops, dtype, d, page):
    """NaN and infinities behind the position, in the rest of its page, in the
    sequence's later pages and in every page it does not own."""
    rng = np.random.default_rng(d + page)
    hq, hkv = 6, 2
    lengths = [1, 7, 30, 33, 64, 65, 200]
    table, n_pages = pu.page_table(rng, [n + 3 * page for n in lengths], page)
    cache, k, v = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    mine = torch.zeros(n_pages, page, dtype=torch.bool)
    for s, n in enumerate(lengths):
        for p in range(n):
            mine[int(table[s, p // page]), p % page] = True
    junk = (~mine)[:, None, :].expand(-1, hkv, -1).cuda()
    if dtype == torch.float16:
        cache.k_pages[junk] = float("nan")
        cache.v_pages[junk] = float("inf")
    else:
        cache.k_scales[junk] = float("inf")
        cache.v_scales[junk] = float("nan")
        cache.k_pages[junk] = 127
        cache.v_pages[junk] = -128
    q = randh(rng, len(lengths), hq, d).cuda()
    check_attention(ops, q, cache, (k, v), table, [n - 1 for n in lengths], list(range(len(lengths))))
    # and with the batch large enough that no sequence is split
    many = 200
    q = randh(rng, many, hq, d).cuda()
    which = rng.integers(0, len(lengths), many).tolist()
    check_attention(ops, q, cache, (k, v), table, [lengths[s] - 1 for s in which], which)


def test_attention_propagates_nan_rows(cuda, ops):
    """An int8 row marked NaN (an infinity was appended) makes the heads that
    attend to it NaN, and no others."""
    rng = np.random.default_rng(6)
    table, n_pages = pu.page_table(rng, [50, 50], 16)
    cache, _, _ = pu.random_cache(rng, ops, torch.int8, n_pages, 2, 16, 64, table)
    q = randh(rng, 2, 4, 64).cuda()
    cache.v_scales[int(table[0, 2]), 1, 5] = float("nan")
    out = ops.attention_paged(q, cache, i32([49, 49]), i32([0, 1])).cpu()
    assert torch.isnan(out[0, 2:]).all() and torch.isfinite(out[0, :2]).all() and torch.isfinite(out[1]).all()
    cache.k_scales[int(table[1, 0]), 0, 0] = float("nan")
    out = ops.attention_paged(q, cache, i32([49, 49]), i32([0, 1])).cpu()
    assert torch.isnan(out[1, :2]).all() and torch.isfinite(out[1, 2:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_sharp_scores(cuda, ops, dtype):
    """Scores spread over +-200 that keep rising along the sequence: the
    reference moves again and again."""
    rng = np.random.default_rng(13)
    hq, hkv, d, page, n = 4, 2, 64, 16, 900
    table, n_pages = pu.page_table(rng, [n] * 6, page)
    cache, k, v = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    q = randh(rng, 6, hq, d, scale=25.0)
    q[5] = 0.0  # equal scores: the mean of the values
    if dtype == torch.float16:  # keys of sequence 0 that point along the query ever more
        ramp = torch.linspace(-1, 1, n, dtype=torch.float64)
        ids = torch.from_numpy(table[0].astype(np.int64))
        for g in range(hkv):
            rows = (q[0, 2 * g].double()[None] * ramp[:, None] * 0.1).half()
            full = torch.zeros(len(ids) * page, d, dtype=torch.float16)
            full[:n] = rows
            k[ids, g] = full.view(len(ids), page, d).double()
            cache.k_pages[ids.cuda(), g] = full.view(len(ids), page, d).cuda()
    check_attention(ops, q.cuda(), cache, (k, v), table, [n - 1] * 6, list(range(6)))


def test_attention_value_scales_of_all_sizes(cuda, ops):
    """int8 value rows whose scales span ten orders of magnitude, rising and
    falling along the sequence."""
    rng = np.random.default_rng(14)
    hq, hkv, d, page, n = 8, 2, 64, 16, 500
    table, n_pages = pu.page_table(rng, [n, n, n], page)
    cache, k, v = pu.random_cache(rng, ops, torch.int8, n_pages, hkv, page, d, table)
    for s, power in ((0, torch.linspace(-6, 1, n)), (1, torch.linspace(1, -6, n)), (2, torch.full((n,), -8.0))):
        for p in range(n):
            at = int(table[s, p // page])
            cache.v_scales[at, :, p % page] = 10.0 ** float(power[p])
            v[at, :, p % page] = (cache.v_pages[at, :, p % page].cpu().double()
                                  * cache.v_scales[at, :, p % page].cpu().double()[:, None])
    q = randh(rng, 3, hq, d).cuda()
    check_attention(ops, q, cache, (k, v), table, [n - 1] * 3, [0, 1, 2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_several_tokens_of_one_sequence(cuda, ops, dtype):
    """Four draft tokens of each sequence, each at its own position."""
    rng = np.random.default_rng(15)
    hq, hkv, d, page = 14, 2, 64, 16
    table, n_pages = pu.page_table(rng, [130, 64], page)
    cache, k, v = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    positions = [126, 127, 128, 129, 60, 61, 62, 63]
    q = randh(rng, 8, hq, d).cuda()
    check_attention(ops, q, cache, (k, v), table, positions, [0] * 4 + [1] * 4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_workspace_and_strides(cuda, ops, dtype):
    """No workspace, small ones and the preferred one agree within the bound;
    q and out are views with gaps that stay as they were; calls repeat bit for bit."""
    rng = np.random.default_rng(16)
    hq, hkv, d, page, n = 6, 2, 128, 32, 4000
    table, n_pages = pu.page_table(rng, [n, n // 2], page)
    cache, k, v = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    packed = randh(rng, 2, (hq + 2 * hkv) * d).cuda()
    q = packed[:, :hq * d].unflatten(1, (hq, d))
    full = ops.attention_paged_workspace_bytes(2, hq, cache)
    assert ops.attention_paged_workspace_bytes(2000, hq, cache) == 0  # a batch that fills the device needs none
    for nbytes in {0, 16, full // 3 // 16 * 16, full}:
        ws = torch.full((max(nbytes, 16) + 64,), 0x7f, dtype=torch.uint8, device="cuda")
        whole = torch.full((2, hq * d + 40), -5.0, dtype=torch.float16, device="cuda")
        out = whole[:, :hq * d].unflatten(1, (hq, d))
        work = ws[:nbytes] if nbytes else ws[:0]
        check_attention(ops, q, cache, (k, v), table, [n - 1, n // 2 - 1], [0, 1], out=out, workspace=work)
        first = out.clone()
        ops.attention_paged(q, cache, i32([n - 1, n // 2 - 1]), i32([0, 1]), out=out, workspace=work)
        assert torch.equal(out, first)
        assert bool((whole[:, hq * d:] == -5.0).all()) and bool((ws[nbytes:] == 0x7f).all())


def test_attention_bad_tokens_are_zero_and_flagged(cuda, ops):
    from littlellm_b200 import _capi
    rng = np.random.default_rng(17)
    hq, hkv, d, page = 4, 2, 64, 8
    table, n_pages = pu.page_table(rng, [400, 90, 90], page)
    table[1, 4] = n_pages   # position 32.. of sequence 1
    table[2, 0] = -1
    cache, k, v = pu.random_cache(rng, ops, torch.float16, n_pages, hkv, page, d, table)
    capacity = table.shape[1] * page
    cases = [((399, 0), 0), ((31, 1), 0), ((32, 1), _capi.FLAG_BAD_PAGE), ((89, 1), _capi.FLAG_BAD_PAGE),
             ((0, 2), _capi.FLAG_BAD_PAGE), ((89, 2), _capi.FLAG_BAD_PAGE), ((-1, 0), 0),
             ((-2, 0), _capi.FLAG_BAD_POSITION), ((capacity, 0), _capi.FLAG_BAD_POSITION),
             ((5, 3), _capi.FLAG_BAD_SEQ), ((5, -1), _capi.FLAG_BAD_SEQ)]
    q = randh(rng, len(cases), hq, d).cuda()
    for rep in (1, 40):  # split and unsplit
        positions, seqs = [c[0][0] for c in cases] * rep, [c[0][1] for c in cases] * rep
        err = flags()
        out = ops.attention_paged(q.repeat(rep, 1, 1), cache, i32(positions), i32(seqs), err_flags=err).cpu()
        assert int(err.item()) == _capi.FLAG_BAD_PAGE | _capi.FLAG_BAD_POSITION | _capi.FLAG_BAD_SEQ
        for t, ((p, s), flag) in enumerate(cases * rep):
            if flag or p == -1:
                assert (out[t] == 0).all(), (p, s)
            else:
                want, bound = pu.attention(q[t % len(cases)].cpu().double(), pu.rows_of(k, table, s, p + 1),
                                           pu.rows_of(v, table, s, p + 1))
                assert ((out[t].double() - want).abs() <= bound).all()
    for i, ((p, s), flag) in enumerate(cases):
        err = flags()
        ops.attention_paged(q[i:i + 1], cache, i32([p]), i32([s]), err_flags=err)
        assert int(err.item()) == flag, (p, s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_infinite_and_nan_queries(cuda, ops, dtype):
    """A head whose query holds an infinity or NaN becomes NaN; the other heads
    of its group, computed in the same tiles, do not."""
    rng = np.random.default_rng(41)
    hq, hkv, d, page = 8, 2, 64, 16
    table, n_pages = pu.page_table(rng, [100, 100], page)
    cache, k, v = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    q = randh(rng, 2, hq, d)
    bad = q.clone()
    bad[0, 1, 3] = float("nan")
    bad[1, 6, 63] = float("inf")
    bad[1, 6, 0] = 1.0
    out = ops.attention_paged(bad.cuda(), cache, i32([99, 99]), i32([0, 1])).cpu()
    assert torch.isnan(out[0, 1]).all() and torch.isnan(out[1, 6]).all()
    for t, skip in ((0, 1), (1, 6)):
        want, bound = pu.attention(q[t].double(), pu.rows_of(k, table, t, 100), pu.rows_of(v, table, t, 100))
        for h in set(range(hq)) - {skip}:
            assert ((out[t, h].double() - want[h]).abs() <= bound[h]).all()


def test_attention_extreme_codes(cuda, ops):
    """Every code a byte can hold, -128 among them, and queries at the ends of fp16."""
    rng = np.random.default_rng(42)
    hq, hkv, d, page, n = 4, 2, 64, 8, 64
    table, n_pages = pu.page_table(rng, [n], page)
    cache, k, v = pu.random_cache(rng, ops, torch.int8, n_pages, hkv, page, d, table)
    codes = torch.from_numpy(rng.integers(-128, 128, k.shape, dtype=np.int8))
    cache.k_pages.copy_(codes)
    cache.v_pages.copy_(codes.flip(-1))
    cache.k_scales.fill_(1e-7)
    cache.v_scales.fill_(0.5)
    k, v = codes.double() * float(cache.k_scales[0, 0, 0]), codes.flip(-1).double() * 0.5
    q = torch.from_numpy(rng.choice([65504.0, -65504.0, 6e-8, 0.0, 1.0], (1, hq, d))).half()
    out = ops.attention_paged(q.cuda(), cache, i32([n - 1]), i32([0])).cpu().double()
    want, bound = pu.attention(q[0].double(), pu.rows_of(k, table, 0, n), pu.rows_of(v, table, 0, n))
    assert ((out[0] - want).abs() <= bound).all()


@pytest.mark.parametrize("pdl", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_split_in_a_graph(cuda, ops, dtype, pdl):
    """A long cache whose parts go through the workspace, captured once and
    replayed at positions that fill all parts, some, one, and none; the
    positions are written by a kernel of the same graph."""
    rng = np.random.default_rng(43)
    hq, hkv, d, page, n = 4, 1, 64, 64, 20000
    table, n_pages = pu.page_table(rng, [n], page)
    cache, k, v = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    q = randh(rng, 1, hq, d, scale=2.0).cuda()
    nbytes = ops.attention_paged_workspace_bytes(1, hq, cache)
    assert nbytes > 0
    ws = torch.full((nbytes,), 0xff, dtype=torch.uint8, device="cuda")  # NaN everywhere
    given, positions, seqs = i32([5]), i32([-1]), i32([0])
    out = torch.empty(1, hq, d, dtype=torch.float16, device="cuda")
    previous = ops.set_pdl(pdl)
    try:
        def step():
            torch.add(given, 0, out=positions)
            ops.attention_paged(q, cache, positions, seqs, out=out, workspace=ws)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    finally:
        ops.set_pdl(previous)
    for pos in (n - 1, 12345, 300, 0, -1, 31, n - 1):
        given.fill_(pos)
        graph.replay()
        torch.cuda.synchronize()
        if pos < 0:
            assert bool((out == 0).all())
        else:
            want, bound = pu.attention(q[0].cpu().double(), pu.rows_of(k, table, 0, pos + 1),
                                       pu.rows_of(v, table, 0, pos + 1))
            assert ((out[0].cpu().double() - want).abs() <= bound).all(), pos


def test_attention_two_streams_at_once(cuda, ops):
    """Calls that overlap on two streams, each with the workspace its call makes."""
    rng = np.random.default_rng(44)
    hq, hkv, d, page, n = 4, 1, 64, 64, 20000
    table, n_pages = pu.page_table(rng, [n, n], page)
    cache, _, _ = pu.random_cache(rng, ops, torch.float16, n_pages, hkv, page, d, table)
    q = [randh(rng, 1, hq, d).cuda() for _ in range(2)]
    at = [(i32([n - 1 - i]), i32([i])) for i in range(2)]
    want = [ops.attention_paged(q[i], cache, *at[i]).clone() for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, ops.attention_paged(q[i], cache, *at[i])))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i, x in got)


def test_no_tokens(cuda, ops):
    cache = ops.PagedKVCache.allocate(2, 16, 2, 64, 1, 2, dtype=torch.int8)
    none, q, kv = i32([]), torch.empty(0, 4, 64, dtype=torch.float16, device="cuda"), None
    kv = torch.empty(0, 2, 64, dtype=torch.float16, device="cuda")
    assert ops.qkv_norm_rope_kv_append_paged(q, kv, kv, cache, none, none, 1e4).shape == q.shape
    assert ops.attention_paged(q, cache, none, none).shape == q.shape
    assert all(x.shape == (0, 2, 64) for x in ops.kv_read_paged(cache, none, none))
    assert ops.token_logprobs(torch.empty(0, 50, dtype=torch.float16, device="cuda"), none, 3).top_ids.shape == (0, 3)
    torch.cuda.synchronize()


def test_wrapper_refusals(cuda, ops):
    """Shapes, dtypes and layouts that the C entry points cannot see."""
    from littlellm_b200 import _capi
    cache = ops.PagedKVCache.allocate(2, 16, 2, 64, 1, 2)
    q, kv, at = (torch.zeros(3, 4, 64, dtype=torch.float16, device="cuda"),
                 torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda"), i32([0, 1, 2]))
    codes = torch.zeros(2, 2, 16, 64, dtype=torch.int8, device="cuda")
    scales = torch.zeros(2, 2, 16, device="cuda")
    calls = [
        (_capi.ERR_DTYPE, lambda: ops.attention_paged(q.float(), cache, at, at)),
        (_capi.ERR_DTYPE, lambda: ops.attention_paged(q, cache, at.long(), at)),
        (_capi.ERR_SHAPE, lambda: ops.attention_paged(q, cache, at[:2], at)),
        (_capi.ERR_SHAPE, lambda: ops.attention_paged(q[:, :3], cache, at, at)),          # 3 heads over 2
        (_capi.ERR_SHAPE, lambda: ops.attention_paged(q.transpose(0, 1), cache, at, at)),
        (_capi.ERR_SHAPE, lambda: ops.attention_paged(q.expand(3, 4, 64)[..., :32], cache, at, at)),
        (_capi.ERR_SHAPE, lambda: ops.attention_paged(q[:1].expand(3, 4, 64), cache, at, at)),  # one row for all tokens
        (_capi.ERR_SHAPE, lambda: ops.attention_paged(q, cache, at, at, out=q[:2])),
        (_capi.ERR_SHAPE, lambda: ops.qkv_norm_rope_kv_append_paged(q, kv[:2], kv, cache, at, at, 1e4)),
        (_capi.ERR_SHAPE, lambda: ops.qkv_norm_rope_kv_append_paged(q, kv, kv, cache, at, at, 1e4, q_norm=q[0, 0, :32])),
        (_capi.ERR_SHAPE, lambda: ops.qkv_norm_rope_kv_append_paged(q, kv, kv, cache, at, at, 1e4, bq=q[0, 0])),
        (_capi.ERR_DTYPE, lambda: ops.qkv_norm_rope_kv_append_paged(q, kv, kv, cache, at, at, 1e4, q_norm=q[0, 0].int(),
                                                                    k_norm=q[0, 0].int())),
        (_capi.ERR_DTYPE, lambda: ops.qkv_norm_rope_kv_append_paged(q, kv, kv, cache, at, at, 1e4, q_norm=q[0, 0],
                                                                    k_norm=q[0, 0].float())),
        (_capi.ERR_INVALID_ARG, lambda: ops.attention_paged(q, cache, at.cpu(), at)),
        (_capi.ERR_SHAPE, lambda: ops.kv_read_paged(cache, at, at, out_slots=at)),
        (_capi.ERR_SHAPE, lambda: ops.kv_read_paged(cache, at, at, k_out=kv[:2], v_out=kv)),
        (_capi.ERR_DTYPE, lambda: ops.PagedKVCache(codes, codes, cache.page_table)),
        (_capi.ERR_SHAPE, lambda: ops.PagedKVCache(codes, codes, cache.page_table, scales[:1], scales)),
        (_capi.ERR_INVALID_ARG, lambda: ops.PagedKVCache(cache.k_pages, cache.v_pages, cache.page_table, scales, scales)),
        (_capi.ERR_DTYPE, lambda: ops.PagedKVCache(cache.k_pages, cache.v_pages, cache.page_table.long())),
        (_capi.ERR_DTYPE, lambda: ops.PagedKVCache(cache.k_pages.float(), cache.v_pages.float(), cache.page_table)),
        (_capi.ERR_SHAPE, lambda: ops.token_logprobs(q[0].t(), None, 1)),
        (_capi.ERR_SHAPE, lambda: ops.token_logprobs(q[0], None, 33)),
        (_capi.ERR_SHAPE, lambda: ops.token_logprobs(q[0], at)),
        (_capi.ERR_DTYPE, lambda: ops.token_logprobs(codes[0, 0])),
        (_capi.ERR_SHAPE, lambda: ops.token_logprobs(q[0], None, 3, out=ops.token_logprobs_buffers(q[0], 2))),
    ]
    for i, (status, call) in enumerate(calls):
        with pytest.raises(_capi.KllmError) as e:
            call()
        assert e.value.status == status, (i, e.value)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,d,n,longest", [
    (2, 64, 400, 4096),    # GQA heads
    (2, 64, 1025, 4095),   # one token past a thread's first
    (1, 64, 3001, 2600),
    (32, 128, 29, 4093),   # many heads, few tokens
    (3, 128, 513, 2048),   # just long enough to be put in order
    (3, 128, 513, 2047),   # and not
    (2, 64, 1024, 1),      # one position each
])
def test_attention_longest_first(cuda, ops, dtype, hkv, d, n, longest):
    """Batches of more items than run at once: the order in which they are
    taken changes no bit, with padding and bad tokens among them."""
    rng = np.random.default_rng(n + longest)
    page, n_pages, hq = 16, 40, 2 * hkv
    table = rng.integers(0, n_pages, (n, 256)).astype(np.int32)  # sequences share pages
    cache, k, v = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    positions = rng.integers(0, longest, n)
    positions[rng.integers(0, n, 2)] = longest - 1
    seqs = rng.permutation(n)
    q = randh(rng, n, hq, d, scale=1.5).cuda()
    nbytes = ops.attention_paged_workspace_bytes(n, hq, cache)
    # in order from one to eight waves of CTAs; fp16 rows of 128 leave room for
    # one CTA of 128 KB per SM, so 1539 items are ten waves of 148
    waves_past = dtype == torch.float16 and hkv * n > 8 * 148 and d == 128
    assert nbytes == (0 if waves_past else 16 * n)
    ws = torch.full((nbytes + 64,), 0x7f, dtype=torch.uint8, device="cuda")
    sample = rng.permutation(n)[:12].tolist() + [int(positions.argmax())]
    for bad in (False, True):
        want_flags = 0
        if bad:
            positions[:5], seqs[5] = [-1, -1, 4096, -2, 2 ** 31 - 1], n
            from littlellm_b200 import _capi
            want_flags = _capi.FLAG_BAD_POSITION | _capi.FLAG_BAD_SEQ
        outs = []
        for work in (ws[:0], ws[:nbytes], None):
            err = flags()
            out = torch.full((n, hq, d), -5.0, dtype=torch.float16, device="cuda")
            ops.attention_paged(q, cache, i32(positions), i32(seqs), out=out, workspace=work, err_flags=err)
            torch.cuda.synchronize()
            assert int(err.item()) == want_flags
            outs.append(out)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
        assert bool((ws[nbytes:] == 0x7f).all())
        if bad:
            assert bool((outs[0][:6] == 0).all())
            continue
        got = outs[0].cpu().double()
        for t in sample:
            p, at = int(positions[t]), int(seqs[t])
            want, bound = pu.attention(q[t].cpu().double(), pu.rows_of(k, table, at, p + 1), pu.rows_of(v, table, at, p + 1))
            assert ((got[t] - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,n", [(14, 2, 64, 60), (4, 4, 128, 36), (16, 1, 64, 90), (5, 1, 128, 9)])
def test_attention_long_and_padded(cuda, ops, dtype, hq, hkv, d, n):
    """Padded batches over a long cache, split into more parts than run at
    once; sequences share pages, lengths from one position to all."""
    rng = np.random.default_rng(hq + n)
    page, n_pages, capacity = 64, 96, 65536
    table = rng.integers(0, n_pages, (n, capacity // page)).astype(np.int32)
    cache, k, v = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    lengths = [1, 32, 33, 1023, 1024, 1025, 4097, 40_000, 65_536]
    positions = np.full(n, -1)
    at = rng.permutation(n)[:len(lengths)]
    positions[at] = np.array(lengths) - 1
    seqs = rng.permutation(n)
    q = randh(rng, n, hq, d, scale=1.5).cuda()
    nbytes = ops.attention_paged_workspace_bytes(n, hq, cache)
    assert nbytes > 0 and nbytes % (n * hq * (d + 2) * 4) == 0
    ws = torch.full((nbytes + 64,), 0x7f, dtype=torch.uint8, device="cuda")
    for work in (ws[:nbytes], ws[:nbytes // 2], ws[:0]):
        check = np.concatenate([at, np.flatnonzero(positions == -1)])
        out = check_attention(ops, q, cache, (k, v), table, positions.tolist(), seqs.tolist(), workspace=work) \
            if work.numel() == nbytes else ops.attention_paged(q, cache, i32(positions), i32(seqs), workspace=work)
        if work.numel() == nbytes:
            again = ops.attention_paged(q, cache, i32(positions), i32(seqs), workspace=work)
            assert torch.equal(out, again)
        else:  # two forms of one answer, each within the bound checked above of the same value
            want = [pu.attention(q[t].cpu().double(), pu.rows_of(k, table, int(seqs[t]), int(positions[t]) + 1),
                                 pu.rows_of(v, table, int(seqs[t]), int(positions[t]) + 1)) for t in at[:6]]
            for t, (w, bound) in zip(at[:6], want):
                assert ((out[t].cpu().double() - w).abs() <= bound).all()
            assert bool((out[check[len(at):]] == 0).all())
    assert bool((ws[nbytes:] == 0x7f).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,n,longest", [
    (14, 2, 64, 600, 128),     # Qwen2.5-0.5B heads
    (32, 32, 128, 40, 33),     # Llama-2-7B heads, one position past a tile
    (16, 1, 64, 1000, 64),     # two tiles of heads
    (32, 2, 128, 700, 100),
    (9, 3, 128, 500, 1),
    (4, 2, 64, 3001, 500),
])
def test_attention_many_short(cuda, ops, dtype, hq, hkv, d, n, longest):
    """Batches of many short items (a CTA of one warp each), ragged, with
    padding and a bad page; sequences share pages."""
    rng = np.random.default_rng(hq + n)
    page, n_pages = 8, 50
    max_pages = -(-longest // page)
    table = rng.integers(0, n_pages, (n, max_pages)).astype(np.int32)
    cache, k, v = pu.random_cache(rng, ops, dtype, n_pages, hkv, page, d, table)
    positions = rng.integers(0, longest, n)
    positions[rng.integers(0, n, 2)] = longest - 1
    seqs = rng.permutation(n)
    q = randh(rng, n, hq, d, scale=1.5).cuda()
    assert ops.attention_paged_workspace_bytes(n, hq, cache) == 0
    err = flags()
    out = ops.attention_paged(q, cache, i32(positions), i32(seqs), err_flags=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    got = out.cpu().double()
    for t in rng.permutation(n)[:20].tolist() + [int(positions.argmax()), int(positions.argmin())]:
        p, at = int(positions[t]), int(seqs[t])
        want, bound = pu.attention(q[t].cpu().double(), pu.rows_of(k, table, at, p + 1), pu.rows_of(v, table, at, p + 1))
        assert ((got[t] - want).abs() <= bound).all()
    # padding and a page out of range: zeros there, no bit elsewhere changes
    from littlellm_b200 import _capi
    positions[7] = -1
    bad = table.copy()
    bad[seqs[11], int(positions[11]) // page] = n_pages
    cache.page_table.copy_(torch.from_numpy(bad))
    again = ops.attention_paged(q, cache, i32(positions), i32(seqs), err_flags=err)
    torch.cuda.synchronize()
    assert int(err.item()) == _capi.FLAG_BAD_PAGE
    assert bool((again[[7, 11]] == 0).all())
    rest = [t for t in range(n) if t not in (7, 11)]
    assert torch.equal(again[rest], out[rest])


def test_attention_longest_first_in_a_graph(cuda, ops):
    """The order is made from the positions of each replay; lengths all equal,
    ragged, and all padding."""
    rng = np.random.default_rng(77)
    n, hq, hkv, d = 640, 4, 2, 64
    table = rng.integers(0, 40, (n, 256)).astype(np.int32)
    cache, _, _ = pu.random_cache(rng, ops, torch.int8, 40, hkv, 16, d, table)
    q, seqs = randh(rng, n, hq, d).cuda(), i32(rng.permutation(n))
    positions, out = i32(np.zeros(n)), torch.empty(n, hq, d, dtype=torch.float16, device="cuda")
    ws = torch.empty(ops.attention_paged_workspace_bytes(n, hq, cache), dtype=torch.uint8, device="cuda")
    assert ws.numel() == 16 * n
    ops.attention_paged(q, cache, positions, seqs, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_paged(q, cache, positions, seqs, out=out, workspace=ws)
    for p in (np.full(n, 4095), rng.integers(-1, 4096, n), np.full(n, -1), rng.integers(0, 4096, n)):
        positions.copy_(i32(p))
        out.fill_(-5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.attention_paged(q, cache, positions, seqs, workspace=ws[:0]))


def test_wrapper_refuses_flags_and_counts(cuda, ops):
    from littlellm_b200 import _capi
    cache = ops.PagedKVCache.allocate(2, 16, 2, 64, 1, 2)
    q, kv, at = (torch.zeros(3, 4, 64, dtype=torch.float16, device="cuda"),
                 torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda"), i32([0, 1, 2]))
    seqs = i32([0, 0, 0])
    for flags in (torch.zeros(1, dtype=torch.uint8, device="cuda"), torch.zeros(1, device="cuda")):
        for call in (lambda: ops.attention_paged(q, cache, at, seqs, err_flags=flags),
                     lambda: ops.kv_read_paged(cache, at, seqs, err_flags=flags),
                     lambda: ops.qkv_norm_rope_kv_append_paged(q, kv, kv, cache, at, seqs, 1e4, err_flags=flags),
                     lambda: ops.token_logprobs(q[0], err_flags=flags)):
            with pytest.raises(_capi.KllmError) as e:
                call()
            assert e.value.status == _capi.ERR_DTYPE
    for k in (-1, 33, 1 << 33):
        with pytest.raises(_capi.KllmError) as e:
            ops.token_logprobs(q[0], None, k)
        assert e.value.status == _capi.ERR_SHAPE
    with pytest.raises(_capi.KllmError) as e:
        ops.attention_paged(q, cache, at, seqs, out=q)
    assert e.value.status == _capi.ERR_INVALID_ARG
    torch.cuda.synchronize()


# ---- a step as it is used ---------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_then_decode(cuda, ops, dtype):
    """Two sequences: their prompts are appended in two chunks; the second
    chunk reads the prefix back into a head-major cache and attends with the
    prefill kernel; then three decode steps append and attend over the pages on
    another stream, captured in a CUDA graph and replayed."""
    rng = np.random.default_rng(18)
    hq, hkv, d, page, theta, eps = 8, 2, 64, 16, 1e4, 1e-6
    prompt, steps, n_seqs = 48, 3, 2
    max_pages = -(-(prompt + steps) // page)
    cache = ops.PagedKVCache.allocate(n_seqs * max_pages, page, hkv, d, n_seqs, max_pages, dtype=dtype)
    cache.page_table.copy_(i32(rng.permutation(n_seqs * max_pages).reshape(n_seqs, max_pages)))
    qn, kn = (1 + randh(rng, d, scale=0.2)).cuda(), (1 + randh(rng, d, scale=0.2)).cuda()
    total = prompt + steps
    q, k, v = (randh(rng, n_seqs, total, h, d) for h in (hq, hkv, hkv))

    def slice_(lo, hi):
        flat = [x[:, lo:hi].reshape(-1, x.shape[2], d).cuda() for x in (q, k, v)]
        return flat, i32(np.tile(np.arange(lo, hi), n_seqs)), i32(np.repeat(np.arange(n_seqs), hi - lo))

    def dense(name, n):
        pages = getattr(cache, name + "_pages").cpu().double()
        scales = getattr(cache, name + "_scales")
        if scales is not None:
            pages = pages * scales.cpu().double()[..., None]
        table = cache.page_table.cpu().numpy()
        return [pu.rows_of(pages, table, s, n) for s in range(n_seqs)]

    for lo, hi in ((0, 16), (16, prompt)):
        (cq, ck, cv), positions, seqs = slice_(lo, hi)
        ops.qkv_norm_rope_kv_append_paged(cq, ck, cv, cache, positions, seqs, theta, q_norm=qn, k_norm=kn, eps=eps)
        head_major = [torch.zeros(n_seqs, hkv, prompt, d, dtype=torch.float16, device="cuda") for _ in range(2)]
        every = slice_(0, hi)
        ops.kv_read_paged(cache, every[1], every[2], *head_major, out_slots=every[2])
        out = ops.attention_head_major(cq, *head_major, positions, seqs, seq_len=hi - lo)
        kk, vv = dense("k", hi), dense("v", hi)
        for t in range(0, 2 * (hi - lo), 7):
            s, p = int(seqs[t]), int(positions[t])
            want, bound = pu.attention(cq[t].cpu().double(), kk[s][:, :p + 1], vv[s][:, :p + 1])
            # the read back rounded the int8 rows to fp16 once more, and the
            # prefill kernel's probabilities are fp16 too
            more = 8 * pu.E16 * (1 + cq[t].abs().max().double().cpu() * 8) * vv[s].abs().max()
            assert ((out[t].cpu().double() - want).abs() <= bound + more).all()

    stream = torch.cuda.Stream()
    static = [torch.empty(n_seqs, h, d, dtype=torch.float16, device="cuda") for h in (hq, hkv, hkv)]
    q_rot = torch.empty_like(static[0])
    out = torch.empty_like(static[0])
    positions, seqs, err = i32([-1] * n_seqs), i32(range(n_seqs)), flags()
    ws = torch.empty(ops.attention_paged_workspace_bytes(n_seqs, hq, cache) + 16, dtype=torch.uint8, device="cuda")

    def step():
        ops.qkv_norm_rope_kv_append_paged(*static, cache, positions, seqs, theta, q_norm=qn, k_norm=kn, eps=eps,
                                          q_out=q_rot, err_flags=err)
        ops.attention_paged(q_rot, cache, positions, seqs, out=out, workspace=ws, err_flags=err)

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step()  # padding only: changes nothing
        stream.synchronize()
        assert bool((out == 0).all())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for i in range(steps):
            for buf, x in zip(static, (q, k, v)):
                buf.copy_(x[:, prompt + i])
            positions.fill_(prompt + i)
            graph.replay()
            stream.synchronize()
            n = prompt + i + 1
            (wq, wk, wv), (sq, sk, _) = pu.norm_rope(*(x[:, prompt + i] for x in (q, k, v)), None, None, None,
                                                     qn.cpu(), kn.cpu(), eps, theta, [prompt + i] * n_seqs)
            assert not ((q_rot.cpu().double() - wq).abs() > pu.f16_bound(wq, sq)).any()
            kk, vv = dense("k", n), dense("v", n)
            for s in range(n_seqs):
                step16 = wk[s].abs().amax(-1, keepdim=True) / 127 if dtype == torch.int8 else 0.0
                assert ((kk[s][:, -1] - wk[s]).abs() <= 0.51 * step16 + pu.f16_bound(wk[s], sk[s])).all()
                want, bound = pu.attention(q_rot[s].cpu().double(), kk[s], vv[s])
                assert ((out[s].cpu().double() - want).abs() <= bound).all()
    assert int(err.item()) == 0


def test_pdl_launch_mode(cuda, ops):
    """Back to back under programmatic dependent launch: each call reads what
    the one before it wrote."""
    rng = np.random.default_rng(19)
    hq, hkv, d, page, n = 14, 2, 64, 16, 200
    table, n_pages = pu.page_table(rng, [n] * 4, page)
    cache, _, _ = pu.random_cache(rng, ops, torch.int8, n_pages, hkv, page, d, table)
    q, k, v = randh(rng, 4, hq, d).cuda(), randh(rng, 4, hkv, d).cuda(), randh(rng, 4, hkv, d).cuda()
    positions, seqs = i32([n - 1] * 4), i32(range(4))

    def step():
        rq = ops.qkv_norm_rope_kv_append_paged(q, k, v, cache, positions, seqs, 1e4, q_out=torch.empty_like(q))
        out = ops.attention_paged(rq, cache, positions, seqs)
        rows = ops.kv_read_paged(cache, positions, seqs)
        return [rq, out, *rows]

    want = step()
    torch.cuda.synchronize()
    previous = ops.set_pdl(True)
    try:
        for _ in range(20):
            for p in (cache.k_pages, cache.v_pages):  # the rows the step writes
                p[torch.from_numpy(table[:, (n - 1) // page].astype(np.int64)).cuda(), :, (n - 1) % page] = 1
            got = step()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    finally:
        ops.set_pdl(previous)
