"""token_logprobs on the GPU against torch in float64.

Bounds. Sums of n exponentials are taken by at least 256 threads per 8192
values, each adding its share one by one, and joined in a tree: at most
n / 256 + 64 fp32 roundings on any path, one step (2 E32) each, with 4 E32 per
term for the exponential and its argument (whose rounding is E32 |t| for a term
e^t, at most e^-1 after weighting)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E32 = torch.finfo(torch.float32).eps / 2
INF = math.inf


def reference(x, tokens, k):
    """float64 answers on the CPU; a row of -inf has no distribution."""
    x = x.cpu().double()
    # shifted by the maximum first: at 1e38 a double cannot hold lse beside it
    top = torch.where(torch.isnan(x), torch.full_like(x, -INF), x).amax(1, keepdim=True)
    below = x - torch.where(torch.isfinite(top), top, 0.0)
    lse = torch.logsumexp(below, 1, keepdim=True)
    lp = torch.where(torch.isneginf(lse), torch.full_like(x, -INF), below - lse)
    p = lp.exp()
    terms = torch.where(torch.isneginf(lp), torch.zeros_like(lp), p * lp)
    broken = torch.isnan(x).any(1) | torch.isposinf(x).any(1)
    lp[broken] = math.nan
    entropy = torch.where(broken, torch.full((x.shape[0],), math.nan, dtype=torch.float64), -terms.sum(1))
    # largest first, NaN last, equal values in the order of their ids
    keyed = torch.where(torch.isnan(x), torch.full_like(x, -INF), x)
    order = np.lexsort((np.arange(x.shape[1])[None].repeat(x.shape[0], 0), torch.isnan(x).numpy(), -keyed.numpy()))
    ids = torch.from_numpy(order[:, :k].copy())
    got = {"ids": ids, "top": lp.gather(1, ids), "entropy": entropy, "lse": lse}
    if tokens is not None:
        t = tokens.cpu().long()[:, None]
        there = (t >= 0) & (t < x.shape[1])
        at = t.clamp(0, x.shape[1] - 1)
        got["logprob"] = torch.where(there, lp.gather(1, at), 0.0)[:, 0]
        got["rank"] = torch.where(there, 1 + (x > x.gather(1, at)).sum(1, keepdim=True), 0)[:, 0]
        got["given"] = x.gather(1, at)[:, 0]
    return got


def close(got, want, bound, what):
    # as fp32 holds it: a difference of -6e38 is past its range and is -inf there
    got, want = got.cpu().double(), want.float().double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    fine = torch.isfinite(got) & torch.isfinite(want) & ((got - want).abs() <= bound)
    assert bool((same | fine).all()), f"{what}: {float((got - want).abs().nan_to_num().max())}"


def check(ops, x, tokens, k, err=None, **kw):
    out = ops.token_logprobs(x, tokens, k, err_flags=err, **kw)
    torch.cuda.synchronize()
    want = reference(x, tokens, k)
    n = x.shape[1]
    rel = (2 * (n / 256 + 64) + 8) * E32  # of the sums
    lp_bound = lambda lp: rel + 4 * E32 * (1 + lp.abs().nan_to_num(posinf=0, neginf=0))  # noqa: E731
    if tokens is not None:
        close(out.logprobs, want["logprob"], lp_bound(want["logprob"]), "logprobs")
        assert torch.equal(out.ranks.cpu().long(), want["rank"].long())
    # entropy = log s - w / s, two terms of one sign: each takes the sums' error, and
    # log s is moved by it as a whole
    h = want["entropy"]
    close(out.entropies, h, (rel + 8 * E32) * (2 * h.abs().nan_to_num() + 2), "entropies")
    if k:
        assert torch.equal(out.top_ids.cpu().long(), want["ids"])
        close(out.top_logprobs, want["top"], lp_bound(want["top"]), "top_logprobs")
    return out


def logits(rng, rows, vocab, dtype, pad=0, lead=0):
    """Model-like logits, as a view with `pad` values between rows that starts
    `lead` values into its storage."""
    whole = torch.full((rows * (vocab + pad) + lead,), INF, dtype=dtype, device="cuda")  # gaps must not be read as logits
    x = whole[lead:].view(rows, vocab + pad)[:, :vocab]
    y = rng.standard_normal((rows, vocab)) * 2.5
    y[np.arange(rows), rng.integers(0, vocab, rows)] += 8.0
    x.copy_(torch.from_numpy(y).to(dtype))
    return x


def tokens_for(rng, rows, vocab):
    return torch.from_numpy(rng.integers(0, vocab, rows).astype(np.int32)).cuda()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,k", [
    (1, 151936, 20), (3, 32000, 5), (1, 1, 1), (2, 2, 2), (5, 7, 7), (4, 31, 8), (9, 256, 32), (3, 2047, 32),
    (2, 8193, 1), (17, 4099, 0), (700, 1000, 3), (150, 32003, 20), (1, 1000003, 32), (400, 50021, 32),
])
def test_against_float64(cuda, ops, dtype, rows, vocab, k):
    rng = np.random.default_rng(rows * 7 + vocab)
    check(ops, logits(rng, rows, vocab, dtype), tokens_for(rng, rows, vocab), k)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("vocab,pad,lead", [(1001, 0, 0), (1001, 0, 1), (1000, 1, 3), (997, 37, 5), (6, 1, 1),
                                            (32001, 7, 2)])
def test_strides_and_alignment(cuda, ops, dtype, vocab, pad, lead):
    rng = np.random.default_rng(vocab + pad)
    check(ops, logits(rng, 13, vocab, dtype, pad, lead), tokens_for(rng, 13, vocab), min(vocab, 10))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [40, 5000, 70001])
def test_ties_take_the_lowest_id(cuda, ops, dtype, vocab):
    rng = np.random.default_rng(vocab)
    rows = 6
    y = np.zeros((rows, vocab))
    y[1] = rng.integers(0, 3, vocab)                      # three values only
    y[2] = -5.0
    y[2, -3:] = 2.0                                        # the largest at the end
    y[3, ::2] = -0.0                                       # both zeros are one value
    y[4] = np.round(rng.standard_normal(vocab) * 2) / 2
    y[5] = np.arange(vocab) * (60000.0 / vocab)            # rising (fp16: long runs of equal values)
    x = torch.from_numpy(y).to(dtype).cuda()
    for k in (1, 5, 32):
        check(ops, x, tokens_for(rng, rows, vocab), k)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [33, 4097, 50000])
def test_masked_and_broken_rows(cuda, ops, dtype, vocab):
    """-inf in most places, in all but one, in all; the type's lowest value as a
    mask; infinities and NaN; each with fewer numbers than entries asked for."""
    rng = np.random.default_rng(vocab)
    lowest = torch.finfo(dtype).min
    x = torch.from_numpy(rng.standard_normal((12, vocab)) * 3).to(dtype)
    x[0] = -INF
    x[1, :] = -INF
    x[1, vocab // 2] = -4.0
    x[2, torch.from_numpy(rng.random(vocab) < 0.9)] = -INF
    x[3] = lowest
    x[4] = lowest
    x[4, vocab - 1] = 3.0
    x[5] = lowest
    x[5, ::2] = -INF
    x[6, 5] = INF
    x[7, 6] = math.nan
    x[8] = math.nan
    x[9, 3:] = math.nan
    x[10, :] = -INF
    x[10, 4] = math.nan
    x[11, 2] = INF
    x[11, 9] = INF
    x = x.cuda()
    for token in (0, 4, 5, vocab // 2, vocab - 1):
        check(ops, x, torch.full((12,), token, dtype=torch.int32, device="cuda"), 20)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 40, 5000, 151936])
def test_one_possible_token(cuda, ops, dtype, vocab):
    """A grammar that leaves one token: log probability and entropy are 0, not
    nearly 0; two tokens, one 12 above the other, keep the small one's share."""
    rng = np.random.default_rng(vocab)
    rows = 5
    x = torch.full((rows, vocab), -INF, dtype=dtype)
    at = torch.from_numpy(rng.integers(0, vocab, rows))
    x[torch.arange(rows), at] = torch.tensor([3.3, -7.7, 0.0, 11.1, -0.013], dtype=dtype)
    out = ops.token_logprobs(x.cuda(), at.int().cuda(), 1)
    assert bool((out.logprobs == 0).all()) and bool((out.entropies == 0).all()) and bool((out.ranks == 1).all())
    assert bool((out.top_logprobs == 0).all()) and torch.equal(out.top_ids[:, 0].cpu(), at.int())
    if vocab >= 2:
        x[torch.arange(rows), (at + vocab // 2) % vocab] = (x[torch.arange(rows), at].double() - 12).to(dtype)
        out = ops.token_logprobs(x.cuda(), at.int().cuda(), 2)
        want = reference(x, at.int(), 2)
        # 1 + e^-12 in fp32: one rounding of the sum, 1 / 6e-6 of its excess; log, product and e^-12 add a few E32
        close(out.logprobs, want["logprob"], 4 * E32, "logprobs")
        close(out.entropies, want["entropy"], 16 * E32, "entropies")


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_extreme_logits(cuda, ops, dtype):
    """Magnitudes at the ends of the type: differences, not values, set the answer."""
    rng = np.random.default_rng(2)
    big = 60000.0 if dtype == torch.float16 else 3e38
    x = torch.from_numpy(rng.standard_normal((5, 3000))).to(dtype)
    x[0] += big / 2
    x[1] = big
    x[1, 7] = -big
    x[2] = -big
    x[2, 2999] = big
    x[3] *= 1e-4
    x[4] = torch.linspace(-100, 100, 3000).to(dtype)
    check(ops, x.cuda(), tokens_for(rng, 5, 3000), 12)


def test_tokens_none_padding_and_bad(cuda, ops):
    from littlellm_b200 import _capi
    rng = np.random.default_rng(3)
    x = logits(rng, 6, 777, torch.float16)
    out = check(ops, x, None, 4)
    assert out.logprobs is None and out.ranks is None
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(ops, x, torch.tensor([3, -1, 776, -1, 0, 5], dtype=torch.int32, device="cuda"), 2, err)
    assert int(err.item()) == 0
    check(ops, x, torch.tensor([3, -2, 777, -1, 0, 1 << 30], dtype=torch.int32, device="cuda"), 2, err)
    assert int(err.item()) == _capi.FLAG_BAD_TOKEN


def test_outputs_given_and_nothing_else_written(cuda, ops):
    """Outputs inside larger buffers: the rest stays; repeated calls and calls
    in a captured graph give the same bits."""
    rng = np.random.default_rng(4)
    rows, vocab, k = 5, 20000, 6
    x, tokens = logits(rng, rows, vocab, torch.float16), tokens_for(rng, rows, vocab)
    whole = [torch.full((rows * n + 16,), -77, dtype=t, device="cuda")
             for t, n in ((torch.float32, 1), (torch.int32, 1), (torch.float32, 1), (torch.int32, k), (torch.float32, k))]
    views = [w[:-16].view(rows, -1) for w in whole]
    out = ops.TokenLogprobs(*(v.flatten() if v.shape[1] == 1 else v for v in views))
    check(ops, x, tokens, k, out=out)
    assert all(bool((w[-16:] == -77).all()) for w in whole)
    first = [v.clone() for v in out]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops.token_logprobs(x, tokens, k, out=out)
    for v in out:
        v.fill_(-1)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, first))
    x[:, 5] += 20.0
    graph.replay()
    torch.cuda.synchronize()
    assert bool((out.top_ids[:, 0] == 5).all())


def test_answers_of_a_forward_step(cuda, ops):
    """The lm_head product of a batch and the answers from its logits."""
    rng = np.random.default_rng(5)
    h = torch.from_numpy(rng.standard_normal((8, 896))).half().cuda()
    w = torch.from_numpy(rng.standard_normal((32000, 896)) / 30).half().cuda()
    x = ops.linear(h, w)
    out = check(ops, x, x.argmax(1).int(), 5)
    assert torch.equal(out.ranks, torch.ones_like(out.ranks))
    assert torch.equal(out.top_logprobs[:, 0], out.logprobs)


def test_many_rows_of_a_long_vocabulary(cuda, ops):
    """Row offsets past 2^31 elements."""
    rng = np.random.default_rng(6)
    rows, vocab = 15000, 151936
    x = torch.full((rows, vocab), -3.0, dtype=torch.float16, device="cuda")
    some = torch.tensor([0, 1, 7000, 14134, 14135, 14999], device="cuda")
    x[some] = logits(rng, 6, vocab, torch.float16)
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    out = ops.token_logprobs(x, tokens, 5)
    part = ops.TokenLogprobs(*(None if t is None else t[some] for t in out))
    want = reference(x[some], tokens[some], 5)
    assert torch.equal(part.top_ids.cpu().long(), want["ids"])
    assert torch.equal(part.ranks.cpu().long(), want["rank"].long())
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[some] = False
    flat = math.log(vocab)
    assert bool((out.logprobs[rest].double() + flat).abs().max() < 1300 * E32)
    assert bool((out.top_ids[rest] == torch.arange(5, device="cuda")).all())
