"""Cases of the paged-cache and log-probability operators, for timing and for checking.

Four operators, as one serving step uses them:

- ``append``: q/k/v of new tokens get their biases, q and k the per-head norms
  and the rotation of their positions; k and v are written to a paged cache
  (fp16, or int8 with a scale per token and head), and the rows just written
  are read back (so an 8-bit cache is seen as the values it stands for);
- ``read``: rows of a paged cache back as fp16, into a head-major cache;
- ``attention``: one new token per sequence over its pages;
- ``logprobs``: log probability and rank of a given token, entropy and the
  most likely alternatives of each row of logits.

``own`` false computes the plain form in elementary torch operations; ``own``
true makes the calls a user makes of ``littlellm_b200.ops``.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

# (query heads, kv heads, head_dim): the two benchmark models' layouts, then
# other group sizes the operators serve (one kv head, 16 and 3 queries a head).
LAYOUTS = ((14, 2, 64), (32, 32, 128), (8, 1, 128), (16, 4, 64), (16, 1, 64), (9, 3, 128), (6, 6, 64), (40, 8, 128))


def listed():
    return [
        # append: one token of one sequence (the latency of a single stream's step); biases, no norms
        {"name": "append one token f16", "op": "append", "cache": "f16", "heads": 14, "kv_heads": 2, "head_dim": 64,
         "page": 16, "tokens": 1, "seqs": 1, "start": 1000, "norm": False, "bias": True, "packed": False},
        # append: a decode batch of 2048 sequences into an int8 cache, q/k/v views of one packed projection
        {"name": "append decode 2048 i8", "op": "append", "cache": "i8", "heads": 14, "kv_heads": 2, "head_dim": 64,
         "page": 16, "tokens": 2048, "seqs": 2048, "start": 2047, "norm": True, "bias": True, "packed": True},
        # append: the 32 x 512 prefill batch, multi-head layout, int8 cache
        {"name": "append prefill 16384 i8", "op": "append", "cache": "i8", "heads": 32, "kv_heads": 32,
         "head_dim": 128, "page": 64, "tokens": 16384, "seqs": 32, "start": 0, "norm": True, "bias": False,
         "packed": False},
        # read: the 513-token prefix of one sequence, before a chunk of its prompt attends to it
        {"name": "read prefix 513 f16", "op": "read", "cache": "f16", "heads": 14, "kv_heads": 2, "head_dim": 64,
         "page": 16, "seqs": 1, "length": 513},
        # read: 32 sequences of 2048 tokens from int8 pages
        {"name": "read 32 x 2048 i8", "op": "read", "cache": "i8", "heads": 32, "kv_heads": 32, "head_dim": 128,
         "page": 64, "seqs": 32, "length": 2048},
        # attention: one sequence, the step of a single stream
        {"name": "attend one 1001 f16", "op": "attention", "cache": "f16", "heads": 14, "kv_heads": 2,
         "head_dim": 64, "page": 16, "seqs": 1, "shortest": 1001, "longest": 1001, "padded": 0},
        # attention: one sequence with a long document in front of it
        {"name": "attend one 131072 f16", "op": "attention", "cache": "f16", "heads": 14, "kv_heads": 2,
         "head_dim": 64, "page": 64, "seqs": 1, "shortest": 131072, "longest": 131072, "padded": 0},
        # attention: a small batch, multi-head layout, int8 pages, ragged lengths, three padded rows of a fixed batch
        {"name": "attend 29 ragged i8", "op": "attention", "cache": "i8", "heads": 32, "kv_heads": 32,
         "head_dim": 128, "page": 32, "seqs": 29, "shortest": 77, "longest": 4093, "padded": 3},
        # attention: the decode batch of 2048 sequences, fp16 pages
        {"name": "attend 2048 ragged f16", "op": "attention", "cache": "f16", "heads": 14, "kv_heads": 2,
         "head_dim": 64, "page": 16, "seqs": 2048, "shortest": 1, "longest": 4095, "padded": 0},
        # attention: the decode batch of 2048 sequences, int8 pages
        {"name": "attend 2048 ragged i8", "op": "attention", "cache": "i8", "heads": 14, "kv_heads": 2,
         "head_dim": 64, "page": 16, "seqs": 2048, "shortest": 1, "longest": 4095, "padded": 0},
        # logprobs: one row of logits with 20 alternatives (what a completion API answers with)
        {"name": "logprobs 1 x 151936 f16", "op": "logprobs", "dtype": "f16", "rows": 1, "vocab": 151936, "pad": 0,
         "top": 20, "masked": 0.0},
        # logprobs: the logits of the 2048-sequence decode batch
        {"name": "logprobs 2048 x 151936 f16", "op": "logprobs", "dtype": "f16", "rows": 2048, "vocab": 151936,
         "pad": 0, "top": 5, "masked": 0.0},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], its logarithm evenly spread."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("append", "read", "attention", "attention", "logprobs", "logprobs"))
    if op == "logprobs":
        vocab = _spread(rng, 2, 262144)
        rows = _spread(rng, 1, max(1, min(4096, 2048 * 151936 // (2 * vocab))))
        return {"op": op, "dtype": rng.choice(("f16", "f32")), "rows": rows, "vocab": vocab,
                "pad": rng.choice((0, 0, 1, 8, 37)), "top": min(vocab, rng.choice((0, 1, 5, 20, rng.randint(1, 32)))),
                "masked": rng.choice((0.0, 0.0, 0.5, 0.99))}
    heads, kv_heads, d = rng.choice(LAYOUTS)
    case = {"op": op, "cache": rng.choice(("f16", "i8")), "heads": heads, "kv_heads": kv_heads, "head_dim": d,
            "page": 2 ** rng.randint(3, 8)}
    if op == "append":
        tokens = _spread(rng, 1, max(1, 16384 * 96 * 128 // ((heads + 2 * kv_heads) * d) // 4))
        seqs = _spread(rng, 1, tokens)
        tokens = tokens // seqs * seqs
        # far positions too, as long as the page table stays a small part of the call
        return case | {"tokens": tokens, "seqs": seqs,
                       "start": _spread(rng, 1, min(200000, max(1, (case["page"] << 22) // seqs))) - 1,
                       "norm": rng.random() < 0.7, "bias": rng.random() < 0.5, "packed": rng.random() < 0.5}
    if op == "read":
        length = _spread(rng, 1, 32768)
        return case | {"seqs": _spread(rng, 1, max(1, min(512, 32 * 2048 * 32 * 128 // (length * kv_heads * d)))),
                       "length": length}
    longest = _spread(rng, 1, 131072)
    most = max(1, min(2048, 2048 * 4096 * 2 * 64 // (longest * kv_heads * d * 2)))
    seqs = _spread(rng, 1, most)
    return case | {"seqs": seqs, "shortest": rng.randint(1, longest) if seqs > 1 else longest, "longest": longest,
                   "padded": rng.choice((0, 0, 1, 5))}


def _lengths(case):
    """Sequence lengths of an attention case: evenly spread from the shortest to the longest."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    return np.array([hi]) if n == 1 else lo + (np.arange(n, dtype=np.int64) * (hi - lo)) // (n - 1)


def _table(rng, lengths, page):
    """A page table for these lengths: pages handed out in random order, -1 where a sequence has none."""
    need = -(-np.asarray(lengths) // page)
    ids = rng.permutation(int(need.sum())).astype(np.int32)
    table = np.full((len(need), int(need.max())), -1, np.int32)
    table[np.arange(table.shape[1])[None, :] < need[:, None]] = ids
    return table, len(ids)


def _quantise(x):
    """Codes and scales of rows (the last axis): scale = amax / 127."""
    amax = x.abs().amax(-1)
    scale = amax / 127
    code = torch.where(amax[..., None] > 0, torch.round(x / scale[..., None]), 0.0)
    return code.to(torch.int8), scale


def _pages(case, gen, n_pages, dev, filled):
    """Page tensors: keys and values of unit variance as cached, or empty pages to append to."""
    shape = (n_pages, case["kv_heads"], case["page"], case["head_dim"])
    got = {}
    for name in ("k", "v"):
        if case["cache"] == "f16":
            got[name] = (torch.randn(shape, device=dev, dtype=torch.float16, generator=gen) if filled
                         else torch.zeros(shape, device=dev, dtype=torch.float16))
            got[name + "_scale"] = None
        elif filled:
            x = torch.randn(shape, device=dev, dtype=torch.float16, generator=gen)
            got[name] = torch.empty(shape, device=dev, dtype=torch.int8)
            got[name + "_scale"] = torch.empty(shape[:-1], device=dev)
            for part in range(0, n_pages, 65536):
                at = slice(part, part + 65536)
                got[name][at], got[name + "_scale"][at] = _quantise(x[at].float())
        else:
            got[name] = torch.zeros(shape, device=dev, dtype=torch.int8)
            got[name + "_scale"] = torch.zeros(shape[:-1], device=dev)
    return got


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = {"case": case}
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        dtype = torch.float16 if case["dtype"] == "f16" else torch.float32
        # logits of a language model: a spread of a few units, some tokens far above the rest
        x = torch.randn(rows, vocab + case["pad"], device=dev, dtype=dtype, generator=gen) * 2.5
        peak = torch.randint(0, vocab, (rows, min(8, vocab)), device=dev, generator=gen)
        x.scatter_add_(1, peak, torch.rand(peak.shape, device=dev, generator=gen).to(dtype) * 10)
        if case["masked"]:
            # a grammar that allows some tokens only; token 0 is always among them
            part = max(1, (1 << 28) // x.shape[1])
            for r in range(0, rows, part):
                off = torch.rand(x[r:r + part].shape, device=dev, generator=gen) < case["masked"]
                off[:, 0] = False
                x[r:r + part].masked_fill_(off, -math.inf)
        s["logits"] = x[:, :vocab]
        any_token = torch.randint(0, vocab, (rows,), device=dev, generator=gen)
        s["tokens"] = torch.where(torch.rand(rows, device=dev, generator=gen) < 0.7, peak[:, 0], any_token).int()
        return s

    hq, hkv, d, page, n = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["seqs"]
    if case["op"] == "append":
        per = case["tokens"] // n
        end = case["start"] + per
        # the pages of the last positions only: a long sequence's earlier pages are not touched by an append
        first = case["start"] // page
        table, n_pages = _table(rng, [end - first * page] * n, page)
        table = np.concatenate([np.full((n, first), -1, np.int32), table], axis=1)
        positions, seqs = np.tile(np.arange(case["start"], end), n), np.repeat(rng.permutation(n), per)
        t = case["tokens"]
        widths = (hq * d, hkv * d, hkv * d)
        if case["packed"]:
            x = torch.randn(t, sum(widths), device=dev, dtype=torch.float16, generator=gen)
            x = torch.split(x, widths, dim=1)
        else:
            x = [torch.randn(t, w, device=dev, dtype=torch.float16, generator=gen) for w in widths]
        s["q"], s["k"], s["v"] = (y.unflatten(1, (-1, d)) for y in x)
        if case["bias"]:
            s["bias"] = [torch.randn(w, device=dev, dtype=torch.float16, generator=gen) * 0.3 for w in widths]
        if case["norm"]:
            s["norm"] = [1 + 0.2 * torch.randn(d, device=dev, dtype=torch.float16, generator=gen) for _ in range(2)]
        s["theta"], s["eps"] = 1e6, 1e-6
        s["q_out"] = torch.empty(t, hq, d, device=dev, dtype=torch.float16)
        s["k_out"], s["v_out"] = (torch.empty(t, hkv, d, device=dev, dtype=torch.float16) for _ in range(2))
    else:
        lengths = _lengths(case) if case["op"] == "attention" else np.full(n, case["length"])
        lengths = rng.permutation(lengths)
        table, n_pages = _table(rng, lengths, page)
        if case["op"] == "attention":
            # one new token per sequence, at its last position; padded rows of a fixed batch carry -1
            pad = np.full(case["padded"], -1)
            order = rng.permutation(n)
            positions, seqs = np.concatenate([lengths[order] - 1, pad]), np.concatenate([order, pad])
            s["q"] = torch.randn(len(seqs), hq, d, device=dev, dtype=torch.float16, generator=gen) * 1.5
            s["out"] = torch.empty_like(s["q"])
        else:
            positions, seqs = np.tile(np.arange(case["length"]), n), np.repeat(np.arange(n), case["length"])
            s["k_out"], s["v_out"] = (torch.zeros(n, hkv, case["length"], d, device=dev, dtype=torch.float16)
                                      for _ in range(2))
    s["table"] = torch.from_numpy(table).to(dev)
    s["positions"], s["seqs"] = (torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(dev)
                                 for a in (positions, seqs))
    s["pages"] = _pages(case, gen, n_pages, dev, case["op"] != "append")
    return s


def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    return {"append": _append, "read": _read, "attention": _attention, "logprobs": _logprobs}[op](s)


def _own(s, op):
    from littlellm_b200 import ops
    if op == "logprobs":
        if "answer" not in s:
            s["answer"] = ops.token_logprobs_buffers(s["logits"], s["case"]["top"])
        got = ops.token_logprobs(s["logits"], s["tokens"], s["case"]["top"], out=s["answer"])
        return [got.logprobs, got.ranks, got.entropies, got.top_ids, got.top_logprobs]
    if "cache" not in s:
        p = s["pages"]
        s["cache"] = ops.PagedKVCache(p["k"], p["v"], s["table"], p["k_scale"], p["v_scale"])
    cache, positions, seqs = s["cache"], s["positions"], s["seqs"]
    if op == "attention":
        return ops.attention_paged(s["q"], cache, positions, seqs, out=s["out"])
    if op == "read":
        return ops.kv_read_paged(cache, positions, seqs, k_out=s["k_out"], v_out=s["v_out"], out_slots=seqs)
    bq, bk, bv = s.get("bias", (None, None, None))
    q_norm, k_norm = s.get("norm", (None, None))
    q = ops.qkv_norm_rope_kv_append_paged(s["q"], s["k"], s["v"], cache, positions, seqs, s["theta"], bq=bq, bk=bk,
                                          bv=bv, q_norm=q_norm, k_norm=k_norm, eps=s["eps"], q_out=s["q_out"])
    k, v = ops.kv_read_paged(cache, positions, seqs, k_out=s["k_out"], v_out=s["v_out"])
    return [q, k, v]


# ---- plain forms ------------------------------------------------------------------------------------------------

def _place(s):
    """Page and row in the page of each token."""
    page = s["case"]["page"]
    pos, seq = s["positions"].long(), s["seqs"].long()
    return s["table"][seq, pos // page].long(), pos % page


def _rows(s, name):
    """Values of the tokens' cached rows, [tokens, kv heads, head_dim], in fp32."""
    at, row = _place(s)
    x = s["pages"][name][at, :, row].float()
    scale = s["pages"][name + "_scale"]
    return x if scale is None else x * scale[at, :, row][..., None]


def _append(s):
    case = s["case"]
    d = case["head_dim"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if case["bias"]:
        q, k, v = (x + b.float().view(-1, d) for x, b in zip((q, k, v), s["bias"]))
    if case["norm"]:
        q, k = (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * w.float()
                for x, w in zip((q, k), s["norm"]))
    freq = s["theta"] ** (-torch.arange(0, d, 2, device=q.device, dtype=torch.float64) / d)
    angle = s["positions"].double()[:, None] * freq
    c, sn = (f(angle).float()[:, None, :] for f in (torch.cos, torch.sin))

    def turn(x):
        a, b = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([a * c - b * sn, b * c + a * sn], dim=-1)

    s["q_out"].copy_(turn(q))
    at, row = _place(s)
    for name, x in (("k", turn(k)), ("v", v)):
        if case["cache"] == "f16":
            s["pages"][name][at, :, row] = x.half()
        else:
            code, scale = _quantise(x)
            s["pages"][name][at, :, row] = code
            s["pages"][name + "_scale"][at, :, row] = scale
    return [s["q_out"], _rows(s, "k").half(), _rows(s, "v").half()]


def _read(s):
    for name in ("k", "v"):
        s[name + "_out"][s["seqs"].long(), :, s["positions"].long()] = _rows(s, name).half()
    return s["k_out"], s["v_out"]


def _attention(s):
    case = s["case"]
    hq, hkv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    real = s["positions"] >= 0
    table = s["table"][s["seqs"].clamp(min=0).long()].clamp(min=0).long()
    t, n = table.shape

    def dense(name):
        x = s["pages"][name][table].float()  # [tokens, pages, kv heads, page, d]
        if s["pages"][name + "_scale"] is not None:
            x = x * s["pages"][name + "_scale"][table][..., None]
        return x.transpose(1, 2).reshape(t, hkv, n * page, d)

    q = s["q"].float().view(t, hkv, hq // hkv, d)
    score = torch.matmul(q, dense("k").transpose(2, 3)) / math.sqrt(d)
    seen = torch.arange(n * page, device=q.device)[None, :] <= s["positions"][:, None]
    score = score.masked_fill(~seen[:, None, None, :], -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    v = dense("v").masked_fill(~seen[:, None, :, None], 0.0)
    o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
    return torch.where(real[:, None, None], o.reshape(t, hq, d), 0.0).half()


def _order(x):
    """Whole numbers in the order of the values, 32 bits; the two zeros are one value."""
    bits = (x + 0.0).float().view(torch.int32)
    return torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)


def _logprobs(s):
    x, token, top = s["logits"].float(), s["tokens"].long(), s["case"]["top"]
    m = x.amax(-1, keepdim=True)
    below = x - m
    e = torch.exp(below)
    z = e.sum(-1, keepdim=True)
    logz = torch.log(z)
    logprob = (below.gather(1, token[:, None]) - logz)[:, 0]
    entropy = (logz - torch.where(e > 0, e * below, 0.0).sum(-1, keepdim=True) / z)[:, 0]
    rank = 1 + (x > x.gather(1, token[:, None])).sum(-1)
    place = torch.arange(x.shape[1], device=x.device)
    best = torch.topk((_order(x).long() << 32) - place, top, dim=-1).values  # equal values: the lower place first
    ids = (-best) & 0xFFFFFFFF
    return [logprob, rank.int(), entropy, ids.int(), below.gather(1, ids) - logz]


# ---- definitions in 64 bits -------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "read": _exact_read, "attention": _exact_attention,
            "logprobs": _exact_logprobs}[case["op"]](s, case)


def _exact_append(s, case):
    d = case["head_dim"]
    half = d // 2
    pos = s["positions"].double()
    got = []
    for i, x in enumerate((s["q"], s["k"], s["v"])):
        x = x.double()
        if case["bias"]:
            x = x + s["bias"][i].double().reshape(1, -1, d)
        if i < 2:
            if case["norm"]:
                size = torch.sqrt(torch.einsum("thd,thd->th", x, x) / d + s["eps"])
                x = x / size[..., None] * s["norm"][i].double()
            y = torch.empty_like(x)
            for j in range(half):
                w = pos * float(s["theta"]) ** (-2.0 * j / d)
                y[:, :, j] = torch.cos(w)[:, None] * x[:, :, j] - torch.sin(w)[:, None] * x[:, :, j + half]
                y[:, :, j + half] = torch.sin(w)[:, None] * x[:, :, j] + torch.cos(w)[:, None] * x[:, :, j + half]
            x = y
        if i > 0 and case["cache"] == "i8":
            step = x.abs().max(dim=-1, keepdim=True).values / 127
            x = torch.round(x / step) * step
        got.append(x)
    return got


def _exact_read(s, case):
    page = case["page"]
    got = []
    for name in ("k", "v"):
        x = s["pages"][name].double()
        if case["cache"] == "i8":
            x *= s["pages"][name + "_scale"].double().unsqueeze(-1)
        out = torch.empty(case["seqs"], case["kv_heads"], case["length"], case["head_dim"], dtype=torch.float64,
                          device=x.device)
        for b in range(case["seqs"]):
            for p in range(-(-case["length"] // page)):
                n = min(page, case["length"] - p * page)
                out[b, :, p * page:p * page + n] = x[s["table"][b, p], :, :n]
        got.append(out)
    return tuple(got)


def _exact_attention(s, case):
    page, group = case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    where = s["positions"].tolist()
    which = s["seqs"].tolist()
    for t, (pos, seq) in enumerate(zip(where, which)):
        if pos < 0:
            continue
        ids = s["table"][seq, :pos // page + 1].long()
        kv = []
        for name in ("k", "v"):
            x = s["pages"][name].index_select(0, ids).double()
            if case["cache"] == "i8":
                x = x * s["pages"][name + "_scale"].index_select(0, ids).double()[..., None]
            kv.append(x.permute(1, 0, 2, 3).flatten(1, 2)[:, :pos + 1].repeat_interleave(group, dim=0))
        w = torch.einsum("hd,hjd->hj", s["q"][t].double(), kv[0]) / case["head_dim"] ** 0.5
        out[t] = torch.einsum("hj,hjd->hd", torch.softmax(w, dim=-1), kv[1])
    return out


def _exact_logprobs(s, case):
    got = [[], [], [], [], []]
    part = max(1, (1 << 27) // case["vocab"])
    for r in range(0, case["rows"], part):
        x = s["logits"][r:r + part].double()
        token = s["tokens"][r:r + part].long().unsqueeze(1)
        lp = torch.log_softmax(x, dim=1)
        got[0].append(lp.gather(1, token).squeeze(1))
        got[1].append((x > x.gather(1, token)).sum(1).int() + 1)
        got[2].append(-torch.nansum(lp.exp() * lp, dim=1))
        # largest first, equal values in their order of place
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
        got[3].append(ids.int())
        got[4].append(lp.gather(1, ids))
    return [torch.cat(g) for g in got]


def work(case):
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "f16" else 4) + case["rows"] * (16 + 8 * case["top"]),
                "flops": 6 * n}
    hq, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    row = d * 2 if case["cache"] == "f16" else d + 4  # a cached row of one head
    if case["op"] == "append":
        t = case["tokens"]
        # the inputs, the rotated queries, the rows written, and the same rows read back as fp16
        return {"bytes": t * (2 * (hq + 2 * hkv) * d + 2 * hq * d + 4 * hkv * row + 4 * hkv * d + 8),
                "flops": t * (hq + 2 * hkv) * d * 10}
    if case["op"] == "read":
        t = case["seqs"] * case["length"]
        return {"bytes": t * (2 * hkv * row + 4 * hkv * d + 8), "flops": t * 2 * hkv * d}
    seen = int(_lengths(case).sum())
    return {"bytes": seen * 2 * hkv * row + 2 * (case["seqs"] + case["padded"]) * hq * d * 2,
            "flops": 4 * seen * hq * d}
