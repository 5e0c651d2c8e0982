"""The operators of serving with drafted tokens over a paged cache, measured one call at a time.

A case is a dict of plain values; its "op" names the operator:

  append    norms, rotation and the store of a batch's tokens into a paged cache (ops.paged_append)
  attn      attention of those tokens (single ones, chains, trees) over the paged cache (ops.paged_attn)
  logprobs  log probabilities of given tokens, entropy and the best alternatives of rows of logits (ops.token_logprobs)
  commit    the accepted drafted rows moved together in every layer's pools (ops.paged_commit)

Where `own` is false, run() computes them in plain torch operations, in 32 bits, rounded once at the end.

The operators' definitions, as far as a reader needs them to see what the plain forms do:

* Rotation angles are the f32 product f32(position) * inv_freq[i], as in every other prep of this library (its rows and
  a paged cache's rows are the same values); cos and sin of that angle are exact.
* Cached row r of a sequence is row r % page_size of page block_table[sequence][r // page_size]. Rows below ctx are
  committed (position r); row ctx + j belongs to the sequence's drafted token j.
* Top alternatives are ranked by the logit itself (softcap and temperature keep the order), ties by the lower index.

Inputs: raw projections N(0, 1); norm weights near 1 (q) and near 1/8 (k); cached K rows normalised and weighted the
same way, V rows of unit RMS: scores of a few nats, as trained models have them. Logits N(0, 4^2) with one likely token.
Lengths of a ragged batch follow from the case's own numbers; every value, page order and tree from the seed.
"""
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

EPS = 1e-6


def _ops():
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "gemma4-webgpu_amd"))
    from g4attn import ops

    return ops


# ---- the cases -----------------------------------------------------------------------

def listed():
    return [
        # One drafted-nothing token of one chat on a local layer (512-token window): the smallest call, all latency.
        dict(name="attn_local_1", op="attn", seqs=1, lo=512, hi=512, drafted=1, tree=False, head_dim=256, nqh=8, nkh=1,
             window=512, cap=0.0, kv="f16", page=64),
        # A tree of 26 drafted tokens verified at 8K context on a global layer of head_dim 512.
        dict(name="attn_tree_8k_512", op="attn", seqs=1, lo=8192, hi=8192, drafted=26, tree=True, head_dim=512, nqh=8,
             nkh=1, window=0, cap=0.0, kv="f16", page=64),
        # A serving batch: 64 sequences of 1K to 32K rows, each with a tree of 8 tokens.
        dict(name="attn_batch_64", op="attn", seqs=64, lo=1024, hi=32768, drafted=8, tree=True, head_dim=256, nqh=8,
             nkh=1, window=0, cap=0.0, kv="f16", page=64),
        # Three long documents in 8-bit caches, five chained drafts each, capped scores, four heads a kv head.
        dict(name="attn_long_e4m3", op="attn", seqs=3, lo=100001, hi=131072, drafted=5, tree=False, head_dim=256, nqh=8,
             nkh=2, window=0, cap=50.0, kv="e4m3", page=128),
        # A prompt's chunk of 1024 tokens after 7001 cached rows: long chains over pages.
        dict(name="attn_chunk_1024", op="attn", seqs=1, lo=7001, hi=7001, drafted=1024, tree=False, head_dim=256, nqh=8,
             nkh=1, window=0, cap=0.0, kv="f16", page=64),
        # The drafted trees' tokens of that serving batch, stored before their attention.
        dict(name="append_tree_64", op="append", seqs=64, lo=256, hi=2048, drafted=8, tree=True, head_dim=256, nqh=8,
             nkh=1, kv="f16", page=64, theta=1e4, divisor=False),
        # Four prompts' chunks, ragged around 1000 tokens, into an 8-bit cache of a global layer of head_dim 512.
        dict(name="append_prompts_e4m3", op="append", seqs=4, lo=0, hi=900, drafted=1000, tree=False, head_dim=512,
             nqh=8, nkh=1, kv="e4m3", page=64, theta=1e6, divisor=True),
        # One sampled token with its five best alternatives, softcapped logits: the end of every chat step.
        dict(name="logprobs_1", op="logprobs", rows=1, vocab=262144, dtype="f32", top=5, cap=30.0, temperature=1.0),
        # The drafted tokens of a batch scored with 20 alternatives.
        dict(name="logprobs_64", op="logprobs", rows=64, vocab=262144, dtype="f32", top=20, cap=30.0, temperature=0.7),
        # A prompt's tokens scored (no alternatives), bf16 logits.
        dict(name="logprobs_prompt", op="logprobs", rows=701, vocab=262144, dtype="bf16", top=0, cap=0.0,
             temperature=1.0),
        # One sequence's accepted path of a tree, over the 15 layers that own a cache.
        dict(name="commit_1", op="commit", seqs=1, lo=2048, hi=2048, drafted=26, path=6, locals=12, globals=3, nkh=1,
             kv="f16", page=64),
        # A batch of 64 with trees of 32, accepted paths of up to 9.
        dict(name="commit_64", op="commit", seqs=64, lo=100, hi=400, drafted=32, path=9, locals=8, globals=2, nkh=1,
             kv="f16", page=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "append", "append", "logprobs", "logprobs", "commit"])
    kv, page = rng.choice(["f16", "f16", "e4m3"]), rng.choice([16, 32, 64, 128])
    nqh, nkh = rng.choice([(8, 1), (8, 1), (4, 1), (8, 2), (8, 4), (6, 2), (4, 4)])
    head_dim = rng.choice([256, 256, 512])
    tree = rng.random() < 0.6
    if op == "attn":
        drafted = _log_int(rng, 1, 64) if tree else _log_int(rng, 1, 700)
        seqs = _log_int(rng, 1, 64)
        rows = min(131072, 2_000_000 * 256 // (seqs * nkh * head_dim), 1024 * 8025 * 8 * 256 // (seqs * drafted * nqh * head_dim))
        hi = _log_int(rng, 16, max(17, rows - drafted))
        return dict(op=op, seqs=seqs, lo=rng.randint(0, hi), hi=hi, drafted=drafted, tree=tree, head_dim=head_dim,
                    nqh=nqh, nkh=nkh, window=rng.choice([0, 0, 512, 1024]), cap=rng.choice([0.0, 0.0, 50.0]), kv=kv,
                    page=page)
    if op == "append":
        seqs = _log_int(rng, 1, 64)
        drafted = _log_int(rng, 1, 64) if tree else _log_int(rng, 1, max(2, 4000 // seqs))
        hi = _log_int(rng, 1, 2048)
        return dict(op=op, seqs=seqs, lo=rng.randint(0, hi), hi=hi, drafted=drafted, tree=tree, head_dim=head_dim,
                    nqh=nqh, nkh=nkh, kv=kv, page=page, theta=rng.choice([1e4, 1e6]), divisor=rng.random() < 0.4)
    if op == "logprobs":
        vocab = _log_int(rng, 1000, 262144)
        return dict(op=op, rows=_log_int(rng, 1, min(1024, 64 * 262144 // vocab)), vocab=vocab,
                    dtype=rng.choice(["f32", "f32", "f16", "bf16"]), top=rng.choice([0, 1, 5, 20, 32]),
                    cap=rng.choice([0.0, 30.0]), temperature=rng.choice([1.0, 1.0, 0.7]))
    hi = _log_int(rng, 16, 400)
    return dict(op="commit", seqs=_log_int(rng, 1, 64), lo=rng.randint(0, hi), hi=hi, drafted=rng.randint(9, 64),
                path=rng.randint(1, 9), locals=rng.randint(1, 8), globals=rng.randint(0, 2), nkh=rng.choice([1, 1, 2]),
                kv=kv, page=page)


def _lengths(c):
    """(committed rows, drafted tokens) of each sequence."""
    rng = random.Random(c["seqs"] * 7919 + c["hi"] * 31 + c["drafted"])
    ctx = [rng.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]
    ctx[0] = c["hi"]
    if c["op"] == "commit" or c["seqs"] == 1:
        return ctx, [c["drafted"]] * c["seqs"]
    return ctx, [c["drafted"] if c["tree"] else rng.randint((c["drafted"] + 1) // 2, c["drafted"]) for _ in ctx]


# ---- inputs --------------------------------------------------------------------------

def _pool(gen, dev, shape, kv, scale):
    x = torch.randn(*shape, generator=gen, device=dev)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * scale
    return x.to(torch.float8_e4m3fn if kv == "e4m3" else torch.float16)


def _batch(c, seed, gen, dev, extra=0):
    """Lengths, shuffled pages and the drafted tokens' trees."""
    ctx, drafted = _lengths(c)
    S, P = c["seqs"], c["page"]
    pages = [-(-(n + t + extra) // P) for n, t in zip(ctx, drafted)]
    width, total = max(pages), sum(pages) + 1
    host = np.random.default_rng(seed * 1_000_003 + 5)
    order = host.permutation(total)
    table = np.zeros((S, width), np.int32)
    at = 0
    for s, n in enumerate(pages):
        table[s, :n] = order[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum(drafted)]).astype(np.int32)
    b = dict(ctx=torch.tensor(ctx, dtype=torch.int32, device=dev), start=torch.from_numpy(start).to(dev),
             table=torch.from_numpy(table).to(dev), pages=total, tokens=int(start[-1]), longest=max(drafted),
             rows=max(n + t for n, t in zip(ctx, drafted)), positions=None, mask=None)
    if c.get("tree"):
        depth, bits = [], []
        for n, t in zip(ctx, drafted):
            d, m = [], []
            for j in range(t):
                p = int(host.integers(max(-1, j - 6), j)) if j else -1
                d.append(d[p] + 1 if p >= 0 else 0)
                m.append((m[p] if p >= 0 else 0) | (1 << j))
            depth += [n + x for x in d]
            bits += m
        b["positions"] = torch.tensor(depth, dtype=torch.int32, device=dev)
        b["mask"] = torch.from_numpy(np.array(bits, np.uint64).view(np.int64)).to(dev).view(-1, 1)
    return b


def _handles(st):
    """The cache and batch descriptions that a serving loop keeps over a step's layers."""
    ops = _ops()
    b = st["b"]
    st["ops"] = ops
    st["batch"] = ops.PagedBatch(b["table"], b["start"], b["ctx"], b["tokens"], max_tokens=b["longest"],
                                 positions=b["positions"], tree_mask=b["mask"])
    st["caches"] = [ops.PagedCache(k, v) for k, v in zip(st["k"], st["v"])]


def prepare(case, seed):
    c = case
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(1_000_003 * seed + 29)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=dev)  # noqa: E731
    st = dict(c=c)
    if c["op"] == "logprobs":
        x = normal(c["rows"], c["vocab"]) * 4
        st["tokens"] = torch.randint(c["vocab"], (c["rows"],), generator=gen, device=dev, dtype=torch.int32)
        hot = torch.randint(c["vocab"], (c["rows"], 1), generator=gen, device=dev)
        x.scatter_add_(1, hot, torch.full_like(hot, 14, dtype=x.dtype))
        st["logits"] = x.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[c["dtype"]])
        if own:
            ops = st["ops"] = _ops()
            st["ws"] = torch.empty(ops.token_logprobs_workspace_bytes(c["rows"], c["vocab"], c["top"]), dtype=torch.uint8,
                                   device=dev)
            st["out"] = [torch.empty(c["rows"], device=dev), torch.empty(c["rows"], device=dev),
                         torch.empty(c["rows"], c["top"], dtype=torch.int32, device=dev),
                         torch.empty(c["rows"], c["top"], device=dev)]
        return st
    if c["op"] == "commit":
        b = st["b"] = _batch(c, seed, gen, dev)
        dims = [256] * c["locals"] + [512] * c["globals"]
        st["k"] = [_pool(gen, dev, (b["pages"], c["page"], c["nkh"], d), c["kv"], 0.125) for d in dims]
        st["v"] = [_pool(gen, dev, (b["pages"], c["page"], c["nkh"], d), c["kv"], 1.0) for d in dims]
        host = np.random.default_rng(seed * 1_000_003 + 7)
        path = np.stack([np.sort(host.choice(c["drafted"], c["path"], replace=False)) for _ in range(c["seqs"])])
        st["path"] = torch.from_numpy(path.astype(np.int32)).to(dev)
        st["accepted"] = torch.from_numpy(host.integers(0, c["path"] + 1, c["seqs"]).astype(np.int32)).to(dev)
        st["accepted"][0] = c["path"]
        st["new"] = torch.zeros_like(b["ctx"])
        if own:
            _handles(st)
        return st
    hd, nqh, nkh = c["head_dim"], c["nqh"], c["nkh"]
    b = st["b"] = _batch(c, seed, gen, dev)
    st["k"] = [_pool(gen, dev, (b["pages"], c["page"], nkh, hd), c["kv"], 0.125)]
    st["v"] = [_pool(gen, dev, (b["pages"], c["page"], nkh, hd), c["kv"], 1.0)]
    if c["op"] == "attn":
        st["q"] = _pool(gen, dev, (b["tokens"], nqh, hd), "f16", 1.0)
        if own:
            _handles(st)
            st["out"] = torch.zeros(b["tokens"], nqh, hd, device=dev)
            st["ws"] = torch.empty(st["ops"].paged_attn_workspace_bytes(st["caches"][0], st["batch"], nqh), dtype=torch.uint8,
                                   device=dev)
        return st
    st["q"], st["kin"], st["vin"] = normal(b["tokens"], nqh, hd), normal(b["tokens"], nkh, hd), normal(b["tokens"], nkh, hd)
    st["wq"], st["wk"] = (1 + 0.1 * normal(hd)).half(), ((1 + 0.1 * normal(hd)) / 8).half()
    freq = torch.tensor([1.0 / c["theta"] ** (2 * i / hd) for i in range(hd // 2)], dtype=torch.float64)
    if c["divisor"]:  # the global layers' proportional rotation: a quarter of the pairs turn
        freq[hd // 8:] = 0
    st["inv"] = freq.float().to(dev)
    st["qout"] = torch.zeros(b["tokens"], nqh, hd, dtype=torch.float16, device=dev)
    if own:
        _handles(st)
    return st


# ---- the plain forms -----------------------------------------------------------------

def _raw(pool):
    """A pool as integers or halves that torch can index."""
    return pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool


def _token_rows(b):
    """(sequence, index in it, cache row) of every token."""
    t = torch.arange(b["tokens"], device=b["start"].device, dtype=torch.int32)
    seq = torch.searchsorted(b["start"][1:].contiguous(), t, right=True)
    j = t - b["start"][seq]
    return seq, j, b["ctx"][seq] + j


def _plain_append(st):
    c, b = st["c"], st["b"]
    seq, _, row = _token_rows(b)
    pos = row if b["positions"] is None else b["positions"]
    angle = (pos.float()[:, None] * st["inv"][None, :]).double()
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    half = c["head_dim"] // 2

    def norm(x, w):
        return x * w / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)

    def rope(x):
        a, d = x[..., :half], x[..., half:]
        return torch.cat([a * cos - d * sin, a * sin + d * cos], -1)

    q, k, v = rope(norm(st["q"], st["wq"].float())), rope(norm(st["kin"], st["wk"].float())), norm(st["vin"], 1.0)
    page, off = b["table"][seq, (row // c["page"]).long()].long(), (row % c["page"]).long()
    for pool, x in ((st["k"][0], k), (st["v"][0], v)):
        _raw(pool)[page, off] = _raw(x.to(pool.dtype))
    st["qout"].copy_(q.half())
    return st["qout"], st["k"][0], st["v"][0]


def _plain_attn(st):
    c, b = st["c"], st["b"]
    hd, nqh, nkh, P = c["head_dim"], c["nqh"], c["nkh"], c["page"]
    S, T, R = c["seqs"], b["longest"], b["rows"]
    dev = st["q"].device
    r = torch.arange(R, device=dev, dtype=torch.int32)
    page = b["table"][:, (r // P).long()].long()
    k, v = (_raw(p)[page, (r % P).long()[None, :]].view(p.dtype).float().permute(0, 2, 1, 3) for p in (st["k"][0], st["v"][0]))
    seq, j, row = _token_rows(b)
    q = torch.zeros(S, T, nqh, hd, device=dev)
    q[seq, j.long()] = st["q"].float()
    q = q.view(S, T, nkh, nqh // nkh, hd).permute(0, 2, 1, 3, 4).reshape(S, nkh, T * (nqh // nkh), hd)
    s = q @ k.transpose(-1, -2).contiguous()
    if c["cap"]:
        s = c["cap"] * torch.tanh(s / c["cap"])
    ctx, n = b["ctx"], b["start"][1:] - b["start"][:-1]
    jr = r[None, :] - ctx[:, None]  # the drafted index of each row, negative for committed ones
    live = (jr < n[:, None])[:, None, :]
    tok = (b["start"][:-1, None] + torch.arange(T, device=dev)[None, :]).clamp(max=b["tokens"] - 1).long()
    if b["mask"] is not None:
        bit = (b["mask"][tok, 0][:, :, None] >> jr.clamp(0, 63).long()[:, None, :]) & 1
        live = live & ((jr < 0)[:, None, :] | (bit == 1))
    else:
        live = live & (jr[:, None, :] <= torch.arange(T, device=dev)[None, :, None])
    if c["window"]:
        pos = row if b["positions"] is None else b["positions"]
        draft = pos[(b["start"][:-1, None] + jr.clamp(min=0)).clamp(max=b["tokens"] - 1).long()]
        rpos = torch.where(jr < 0, r[None, :].expand(S, R), draft)
        live = live & (rpos[:, None, :] > pos[tok][:, :, None] - c["window"])
    s = s.view(S, nkh, T, nqh // nkh, R).masked_fill(~live[:, None, :, None, :], -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(s - m)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = p.view(S, nkh, -1, R) @ v
    o = o.view(S, nkh, T, nqh // nkh, hd).permute(0, 2, 1, 3, 4).reshape(S, T, nqh, hd)
    return o[seq, j.long()]


def _plain_logprobs(st):
    c, x = st["c"], st["logits"]
    z = x.float()
    if c["cap"]:
        z = c["cap"] * torch.tanh(z / c["cap"])
    z = z / c["temperature"]
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    got = (z.gather(1, st["tokens"].long()[:, None]) - lse)[:, 0]
    entropy = (torch.log(total) - (e * (z - m)).sum(-1, keepdim=True) / total)[:, 0]
    if not c["top"]:
        return got, entropy
    ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :c["top"]]
    return got, entropy, ids.int(), z.gather(1, ids) - lse


def _plain_commit(st):
    c, b = st["c"], st["b"]
    d = torch.arange(c["path"], device=st["path"].device, dtype=torch.int32)[None, :]
    dst = b["ctx"][:, None] + d
    src = torch.where(d < st["accepted"][:, None], b["ctx"][:, None] + st["path"], dst)

    def flat(row):
        return (b["table"].gather(1, (row // c["page"]).long()).long() * c["page"] + row % c["page"]).reshape(-1)

    src, dst = flat(src), flat(dst)
    for pool in st["k"] + st["v"]:
        rows = _raw(pool).view(-1, c["nkh"] * pool.shape[-1])
        rows[dst] = rows[src]
    return (torch.add(b["ctx"], st["accepted"]), *st["k"], *st["v"])


def run(state):
    st, c = state, state["c"]
    if not own:
        return {"append": _plain_append, "attn": _plain_attn, "logprobs": _plain_logprobs, "commit": _plain_commit}[c["op"]](st)
    ops = st["ops"]
    if c["op"] == "append":
        ops.paged_append(st["caches"][0], st["batch"], st["q"], st["kin"], st["vin"], st["wq"], st["wk"], st["inv"], st["qout"],
                         eps=EPS)
        return st["qout"], st["k"][0], st["v"][0]
    if c["op"] == "attn":
        ops.paged_attn(st["caches"][0], st["batch"], st["q"], st["out"], st["ws"], scale=1.0, sliding_window=c["window"],
                       softcap=c["cap"])
        return st["out"]
    if c["op"] == "logprobs":
        got, entropy, ids, lp = st["out"]
        ops.token_logprobs(st["logits"], st["tokens"], got, entropy, st["ws"], top_ids=ids if c["top"] else None,
                           top_logprobs=lp if c["top"] else None, cap=c["cap"], temperature=c["temperature"])
        return (got, entropy, ids, lp) if c["top"] else (got, entropy)
    ops.paged_commit(st["caches"], st["batch"], st["path"], st["accepted"], st["new"])
    return (st["new"], *st["k"], *st["v"])


# ---- what a pass cannot do without ----------------------------------------------------

def work(case):
    c = case
    if c["op"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * (4 if c["dtype"] == "f32" else 2) + c["rows"] * (12 + 8 * c["top"]), "flops": 6 * n}
    width = 1 if c["kv"] == "e4m3" else 2
    ctx, drafted = _lengths(c)
    if c["op"] == "commit":
        elems = (c["locals"] * 256 + c["globals"] * 512) * c["nkh"]
        rows = c["path"] + (c["seqs"] - 1) * c["path"] / 2
        return {"bytes": rows * elems * 2 * 2 * width, "flops": 0}
    hd, nqh, nkh = c["head_dim"], c["nqh"], c["nkh"]
    tokens = sum(drafted)
    if c["op"] == "append":
        return {"bytes": tokens * hd * ((nqh + 2 * nkh) * 4 + nqh * 2 + 2 * nkh * width), "flops": tokens * (nqh + 2 * nkh) * hd * 8}
    w, rows, keys = c["window"], 0, 0
    for n, t in zip(ctx, drafted):
        rows += min(n, w - 1 if w else n) + t
        keys += sum(min(n + i + 1, w or n + i + 1) for i in range(t)) if not c["tree"] else t * (min(n, w or n) + 3)
    return {"bytes": rows * 2 * nkh * hd * width + tokens * nqh * hd * 6, "flops": 4.0 * hd * nqh * keys}


# ---- the definitions in 64 bits --------------------------------------------------------

def exact(case, seed):
    c = case
    st = prepare(case, seed)
    if c["op"] == "logprobs":
        ids, lp, h, tops = [], [], [], []
        for i in range(0, c["rows"], 64):
            x = st["logits"][i:i + 64]
            z = x.double()
            z = (c["cap"] * torch.tanh(z / c["cap"]) if c["cap"] else z) / c["temperature"]
            logp = torch.log_softmax(z, -1)
            lp.append(logp.gather(1, st["tokens"][i:i + 64].long()[:, None])[:, 0])
            h.append(-(logp.exp() * logp).sum(-1))
            if c["top"]:
                order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :c["top"]]
                ids.append(order.int())
                tops.append(logp.gather(1, order))
        out = (torch.cat(lp), torch.cat(h))
        return out + (torch.cat(ids), torch.cat(tops)) if c["top"] else out
    b = st["b"]
    ctx, drafted = _lengths(c)
    table, start = b["table"].cpu().numpy(), b["start"].tolist()

    def rows_of(s, first, last):
        r = np.arange(first, last)
        return (torch.from_numpy(table[s, r // c["page"]].astype(np.int64) * c["page"] + r % c["page"])).to(b["ctx"].device)

    if c["op"] == "commit":
        path, n = st["path"].tolist(), st["accepted"].tolist()
        got = []
        for pool in st["k"] + st["v"]:
            flat = _raw(pool).view(-1, c["nkh"] * pool.shape[-1])
            before = flat.clone()
            for s in range(c["seqs"]):
                if n[s]:
                    src = rows_of(s, ctx[s], ctx[s] + c["drafted"])[torch.tensor(path[s][:n[s]], device=flat.device)]
                    flat[rows_of(s, ctx[s], ctx[s] + n[s])] = before[src]
            got.append(pool.float())
        return (torch.tensor([a + m for a, m in zip(ctx, n)], dtype=torch.int32), *got)
    hd, nqh, nkh = c["head_dim"], c["nqh"], c["nkh"]
    if c["op"] == "append":
        k_new, v_new = st["k"][0].double().view(-1, nkh, hd), st["v"][0].double().view(-1, nkh, hd)
        pos = np.concatenate([np.arange(n, n + t) for n, t in zip(ctx, drafted)])
        at = torch.cat([rows_of(s, ctx[s], ctx[s] + drafted[s]) for s in range(c["seqs"])])
        if b["positions"] is not None:
            pos = b["positions"].cpu().numpy()
        # The angle's f32 product belongs to the definition; its turn is exact.
        ang = (pos.astype(np.float32)[:, None] * st["inv"].cpu().numpy()[None, :]).astype(np.float64)
        turn = torch.from_numpy(np.exp(1j * ang)).to(at.device)[:, None, :]

        def rotated(x, w):
            x = x.double()
            x = x * w.double() / (x.square().sum(-1, keepdim=True) / hd + EPS).sqrt()
            y = torch.complex(x[..., :hd // 2], x[..., hd // 2:]) * turn
            return torch.cat([y.real, y.imag], -1)

        v = st["vin"].double()
        k_new[at] = rotated(st["kin"], st["wk"])
        v_new[at] = v / (v.square().sum(-1, keepdim=True) / hd + EPS).sqrt()
        return rotated(st["q"], st["wq"]), k_new.view(st["k"][0].shape), v_new.view(st["v"][0].shape)
    out = torch.zeros(b["tokens"], nqh, hd, dtype=torch.float64, device=b["ctx"].device)
    for s in range(c["seqs"]):
        n, t = ctx[s], drafted[s]
        pos = np.arange(n, n + t) if b["positions"] is None else b["positions"][start[s]:start[s + 1]].cpu().numpy()
        see = np.ones((t, n + t), bool)
        see[:, n:] = np.tril(np.ones((t, t), bool))
        if b["mask"] is not None:
            bits = b["mask"][start[s]:start[s + 1], 0].cpu().numpy().view(np.uint64)
            see[:, n:] = (bits[:, None] >> np.arange(t, dtype=np.uint64)[None, :]) & np.uint64(1)
        if c["window"]:
            see &= np.concatenate([np.arange(n), pos])[None, :] > pos[:, None] - c["window"]
        hide = torch.from_numpy(~see).to(out.device)
        at = rows_of(s, 0, n + t)
        k, v = (_raw(p).view(-1, nkh, hd)[at].view(p.dtype).double() for p in (st["k"][0], st["v"][0]))
        for h in range(nqh):
            x = st["q"][start[s]:start[s + 1], h].double() @ k[:, h * nkh // nqh].T
            x = c["cap"] * torch.tanh(x / c["cap"]) if c["cap"] else x
            w = torch.softmax(x.masked_fill(hide, -math.inf), -1)
            out[start[s]:start[s + 1], h] = w @ v[:, h * nkh // nqh]
    return out
