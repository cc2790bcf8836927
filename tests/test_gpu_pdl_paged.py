"""Paged attention's forms and the log probabilities under programmatic
dependent launch: calls back to back on one stream, each reading what the launch
directly before it wrote and overwriting what that one still reads (workspace,
positions, logits), give the bits of plain launches."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_util as pu
from test_gpu_paged import DTYPES, i32, randh

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,n,longest,ordered", [
    (4, 2, 64, 640, 4096, True),     # longest first: an ordering kernel before each call's attention
    (32, 32, 128, 29, 4096, True),
    (14, 2, 64, 3000, 128, False),   # one warp per CTA
    (4, 2, 64, 3, 16384, False),     # parts joined by a second kernel
])
def test_attention_forms(cuda, ops, dtype, hq, hkv, d, n, longest, ordered):
    rng = np.random.default_rng(n)
    page = 16
    table = rng.integers(0, 40, (n, longest // page)).astype(np.int32)
    cache, _, _ = pu.random_cache(rng, ops, dtype, 40, hkv, page, d, table)
    seqs = i32(rng.permutation(n))
    nbytes = ops.attention_paged_workspace_bytes(n, hq, cache)
    assert (nbytes == 16 * n) == ordered and (nbytes > 0) == (longest >= 4096 or ordered)
    ws = torch.full((max(nbytes, 16),), 0xff, dtype=torch.uint8, device="cuda")[:nbytes]
    kc, vc = (torch.zeros(n, hkv, 8, d, dtype=torch.float16, device="cuda") for _ in range(2))
    slots, places = i32(range(n)), i32(np.arange(n) % 8)
    at = [i32(rng.integers(-1, longest, n)) for _ in range(4)]
    given = [randh(rng, n, hq, d, scale=1.5).cuda() for _ in range(4)]
    kv = [randh(rng, n, hkv, d).cuda() for _ in range(2)]

    def calls():
        outs = []
        for i in range(12):
            q = given[i % 4].clone()
            out = torch.empty_like(q)
            # a library kernel writes the queries in the launch before; the workspace is used again at once
            ops.qkv_bias_rope_kv_append(q, *kv, None, None, None, places, slots, 1e4 + i, kc, vc)
            ops.attention_paged(q, cache, at[i % 4], seqs, out=out, workspace=ws)
            ops.attention_paged(q, cache, at[(i + 1) % 4], seqs, out=q_out[i], workspace=ws)
            outs += [out, q_out[i]]
        torch.cuda.synchronize()
        return outs

    q_out = [torch.empty_like(given[0]) for _ in range(12)]
    want = [x.clone() for x in calls()]
    previous = ops.set_pdl(True)
    try:
        for _ in range(3):
            for x in q_out:
                x.fill_(-5.0)
            assert all(torch.equal(a, b) for a, b in zip(calls(), want))
    finally:
        ops.set_pdl(previous)


@pytest.mark.parametrize("rows,vocab", [(1, 65536), (4, 40000), (70, 20000), (700, 5000), (600, 151936)])
def test_logprobs_of_logits_written_by_the_launch_before(cuda, ops, rows, vocab):
    """One CTA per row and clusters of two to eight, all of a row kept or not."""
    rng = np.random.default_rng(rows)
    w = (torch.randn(vocab, 128, device="cuda") / 8).half()
    x = [randh(rng, rows, 128).cuda() for _ in range(4)]
    tokens = i32(rng.integers(0, vocab, rows))
    logits = torch.empty(rows, vocab, dtype=torch.float16, device="cuda")

    def calls():
        got = []
        for i in range(12):
            ops.linear(x[i % 4], w, out=logits)
            got.append(ops.token_logprobs(logits, tokens, 5))
        torch.cuda.synchronize()
        return got

    want = calls()
    for i in range(4):
        ref = torch.log_softmax(ops.linear(x[i], w).double(), 1)
        # a term's exponent is off by 2^-20 (below 32), a thread's sum of at most 600 terms by as many halves of a
        # step: 2^-14 of the sum, and so of its log
        assert ((want[i].logprobs.double() - ref.gather(1, tokens.long()[:, None])[:, 0]).abs() <= 2.0 ** -12).all()
    previous = ops.set_pdl(True)
    try:
        for _ in range(3):
            for a, b in zip(calls(), want):
                assert all(torch.equal(u, v) for u, v in zip(a, b))
    finally:
        ops.set_pdl(previous)
