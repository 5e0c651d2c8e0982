"""g4_paged_append against g4_attn_prompt_prep bit for bit and against the definition in 64 bits; g4_paged_commit against
plain copies; and a step of all the operators in turn."""
import numpy as np
import pytest
import torch

from conftest import announce
from g4attn import ops
from paged_helpers import EPS, Paged, normed, random_parents

pytestmark = pytest.mark.gpu


class Append:
    def __init__(self, dev, p, seed, theta=1e4, divisor=False):
        r = np.random.default_rng(seed)
        self.p, self.dev = p, dev
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
        n = p.tokens
        self.q, self.k, self.v = (r.standard_normal((n, h, p.hd)).astype(np.float32) * 3 for h in (p.nqh, p.nkh, p.nkh))
        self.wq = (1 + 0.1 * r.standard_normal(p.hd)).astype(np.float16)
        self.wk = ((1 + 0.1 * r.standard_normal(p.hd)) / 8).astype(np.float16)
        freqs = np.where(np.arange(p.hd // 2) < p.hd // 8, 1.0, np.inf).astype(np.float16)
        self.freqs = t(freqs.view(np.int16)) if divisor else None
        self.inv = ops.rope_inv_freq(theta, p.hd, divisor, self.freqs)
        self.theta, self.divisor = theta, divisor
        self.d = dict(q=t(self.q), k=t(self.k), v=t(self.v), q_weight=t(self.wq), k_weight=t(self.wk),
                      rope_inv_freq=self.inv)
        self.q_out = torch.full((n, p.nqh, p.hd), -9.0, dtype=torch.float16, device=dev)

    def run(self, **over):
        kw = dict(self.d, q_out=self.q_out)
        kw.update(over)
        ops.paged_append(self.p.cache, self.p.batch, **kw, eps=EPS)
        torch.cuda.synchronize()

    def positions(self):
        p = self.p
        pos = np.concatenate([[c + j for j in range(t)] for c, t in zip(p.ctx, p.new)] or [[]]).astype(np.int64)
        return pos if p.positions is None else p.positions[:len(pos)].astype(np.int64)

    def exact(self):
        pos = self.positions()
        n = len(pos)
        ang = (pos.astype(np.float32)[:, None] * self.inv.cpu().numpy()[None]).astype(np.float64)[:, None, :]
        c, s = np.cos(ang), np.sin(ang)
        half = self.p.hd // 2

        def rope(x):
            a, b = x[..., :half], x[..., half:]
            return np.concatenate([a * c - b * s, a * s + b * c], -1)

        q, k, v = (normed(x[:n].astype(np.float64)) for x in (self.q, self.k, self.v))
        return rope(q * self.wq.astype(np.float64)), rope(k * self.wk.astype(np.float64)), v


def near(got, want, kv):
    """Within half a step of the cache's type, and what the f32 arithmetic before the rounding adds: the sum of
    squares (HD half-steps at most of its value, halved by the root), the quotient and the rotation, whose two
    products may cancel: 2^-24 * 270 of the row's largest element covers them."""
    eps, tiny = (2.0 ** -4, 2.0 ** -10) if kv == "e4m3" else (2.0 ** -11, 2.0 ** -25)
    slack = 270 * 2.0 ** -24 * np.abs(want).max(-1, keepdims=True)
    return np.abs(got - want) <= np.abs(want) * eps + tiny + slack * (1 + eps)


@pytest.mark.parametrize("hd,nqh,nkh", [(256, 8, 1), (256, 6, 2), (512, 8, 1), (512, 4, 4)])
@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("tree", [False, True])
def test_append_matches_the_definition(dev, hd, nqh, nkh, kv, tree):
    r = np.random.default_rng(hd + nqh)
    new, ctx = [1, 0, 17, 5], [0, 3, 60, 15]
    far = [0] + [60 + j for j in range(17)] + [131000 + 3 * j for j in range(5)] + [0] * 3
    p = Paged(dev, 5 + hd, ctx, new, hd=hd, nqh=nqh, nkh=nkh, kv=kv, page=64, pad=3, max_tokens=17,
              parents=[random_parents(r, t) for t in new] if tree else None, positions=None if tree else far).upload()
    a = Append(dev, p, 9, divisor=hd == 512, theta=1e6 if hd == 512 else 1e4)
    announce(f"pagedAppend hd={hd} heads={nqh}/{nkh} kv={kv} tree={tree}")
    a.run()
    q, k, v = a.exact()
    got_q = a.q_out.cpu().double().numpy()
    assert near(got_q[:23], q, "f16").all()
    assert (got_q[23:] == -9.0).all()  # padding
    pools = {"k": (p.d_k.cpu(), p.k.clone()), "v": (p.d_v.cpu(), p.v.clone())}
    for name, want in (("k", k), ("v", v)):
        got, before = (x.float().double().numpy() for x in pools[name])
        tok = 0
        touched = np.zeros(got.shape[:2], bool)
        for s in range(4):
            for row in p.rows(s)[p.ctx[s]:]:
                assert near(got[row], want[tok], kv).all(), (name, tok)
                touched[row] = True
                tok += 1
        assert np.array_equal(got[~touched], before[~touched]), f"{name}: rows of others were written"


@pytest.mark.parametrize("hd", [256, 512])
def test_append_gives_the_prompt_preps_bits(dev, hd):
    p = Paged(dev, 12, [77, 0, 4000], [9, 40, 1], hd=hd, page=32).upload()
    a = Append(dev, p, 10)
    announce(f"pagedAppend against attnPromptPrep hd={hd}")
    a.run()
    for s in range(3):
        lo, n, c = int(p.start[s]), p.new[s], p.ctx[s]
        q_out = torch.zeros(n, 8, hd, dtype=torch.float16, device=dev)
        kc, vc = (torch.zeros(c + n, 1, hd, dtype=torch.float16, device=dev) for _ in range(2))
        ops.attn_prompt_prep(a.d["q"][lo:lo + n].contiguous(), a.d["q_weight"], q_out, n, c, 8, 1, hd, a.theta, False,
                             k=a.d["k"][lo:lo + n].contiguous(), v=a.d["v"][lo:lo + n].contiguous(),
                             k_weight=a.d["k_weight"], k_cache=kc, v_cache=vc, max_seq_len=c + n, rope_inv_freq=a.inv)
        torch.cuda.synchronize()
        assert torch.equal(q_out.view(torch.int16), a.q_out[lo:lo + n].view(torch.int16))
        at = p.rows(s)[c:]
        for pool, want in ((p.d_k, kc), (p.d_v, vc)):
            got = torch.stack([pool[r] for r in at])
            assert torch.equal(got.view(torch.int16), want[c:].view(torch.int16))


def test_append_of_parts_of_one_projection(dev):
    """q, k and v as slices of one [tokens, (NQH + 2 NKH) HD] output; then only q; then only the store."""
    p = Paged(dev, 13, [20, 7], [3, 6], nqh=4, nkh=2).upload()
    a = Append(dev, p, 11)
    announce("pagedAppend strided")
    a.run()
    want_q, want_k, want_v = a.q_out.clone(), p.d_k.clone(), p.d_v.clone()
    one = torch.cat([a.d["q"].reshape(9, -1), a.d["k"].reshape(9, -1), a.d["v"].reshape(9, -1)], 1).contiguous()
    parts = [x.view(9, -1, 256) for x in one.split([4 * 256, 2 * 256, 2 * 256], 1)]
    assert parts[0].stride(0) == 8 * 256
    p.d_k.copy_(p.k)
    p.d_v.copy_(p.v)
    a.q_out.zero_()
    a.run(q=parts[0], k=None, v=None, k_weight=None)
    assert torch.equal(a.q_out, want_q) and torch.equal(p.d_k.cpu(), p.k) and torch.equal(p.d_v.cpu(), p.v)
    a.q_out.zero_()
    a.run(q=None, q_weight=None, q_out=None, k=parts[1], v=parts[2])
    assert torch.equal(p.d_k, want_k) and torch.equal(p.d_v, want_v) and not a.q_out.any()


def test_append_without_pages_past_the_table_and_extremes(dev):
    """Rows whose page id is none, or past the table, are not stored (q is); e4m3 saturates and keeps NaN."""
    p = Paged(dev, 14, [30, 5], [6, 2], kv="e4m3", page=16).upload()
    before = p.d_k.clone()
    p.d_table[0, 1] = p.num_pages  # rows 16 .. 31 of sequence 0
    p.d_ctx[1] = p.table.shape[1] * 16 - 1  # its second new token is past the table
    p.d_table[1, -1] = int(p.table[1, 0])
    a = Append(dev, p, 15)
    a.d["k_weight"] = torch.full((256,), 2000.0, dtype=torch.float16, device=dev)
    a.d["k"][3, 0, 5] = float("nan")
    announce("pagedAppend rows without a page")
    a.run()
    got = p.d_k.float().cpu().numpy()
    assert np.isfinite(a.q_out.cpu().numpy()).all() and (a.q_out != -9.0).all()
    wrote = (p.d_k.view(torch.uint8) != before.view(torch.uint8)).flatten(1).view(p.num_pages, 16, -1).any(-1).cpu().numpy()
    page = int(p.table[0, 2])
    assert wrote[page, :4].all()  # rows 32 .. 35 (tokens 2 .. 5)
    assert wrote.sum() == 5 and wrote[int(p.table[1, 0]), 15]  # and sequence 1's first new token
    assert np.isnan(got[page, 1]).all()  # token 3: its mean square is NaN
    live = got[page, [0, 2, 3]]
    assert np.isfinite(live).all() and np.abs(live).max() == 448.0


def test_append_many_sequences_and_empty_ones(dev):
    r = np.random.default_rng(3)
    new = [int(x) for x in r.integers(0, 3, 150)]
    p = Paged(dev, 15, [int(x) for x in r.integers(0, 50, 150)], new, nqh=2, pad=1, max_tokens=2).upload()
    a = Append(dev, p, 16)
    announce("pagedAppend 150 sequences")
    a.run()
    q, k, _ = a.exact()
    got = p.d_k.double().cpu().numpy()
    tok = 0
    for s in range(150):
        for row in p.rows(s)[p.ctx[s]:]:
            assert near(got[row], k[tok], "f16").all()
            tok += 1
    assert near(a.q_out.double().cpu().numpy()[:tok], q, "f16").all()


@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("steps", [1, 9, 20])
def test_commit_moves_the_accepted_rows(dev, kv, steps):
    r = np.random.default_rng(steps)
    new = [24, 0, 30, 24, 26, 24]
    p = Paged(dev, 20, [100, 5, 0, 63, 17, 40], new, hd=256, kv=kv, page=16).upload()
    second = Paged(dev, 20, [100, 5, 0, 63, 17, 40], new, hd=512, nkh=2, kv="f16", page=16)
    second.table, second.num_pages = p.table, p.num_pages
    second.upload()
    path = np.stack([np.sort(r.choice(24, steps, replace=False)) for _ in new]).astype(np.int32)
    n = np.array([steps, steps, steps, 0, steps + 7, -3], np.int32)
    if steps > 4:
        path[4, 3] = path[4, 2]  # not ascending: the path ends after three
    new_ctx = torch.full((6,), -1, dtype=torch.int32, device=dev)
    announce(f"pagedCommit kv={kv} steps={steps}")
    ops.paged_commit([p.cache, second.cache], p.batch, torch.from_numpy(path).to(dev), torch.from_numpy(n).to(dev), new_ctx)
    torch.cuda.synchronize()
    length = [steps, 0, steps, 0, 3 if steps > 4 else steps, 0]  # sequence 1 has no new tokens
    assert new_ctx.tolist() == [c + m for c, m in zip(p.ctx, length)]
    for c, host, devs in ((p, (p.k, p.v), (p.d_k, p.d_v)), (second, (second.k, second.v), (second.d_k, second.d_v))):
        for h, d in zip(host, devs):
            bits = torch.uint8 if h.dtype == torch.float8_e4m3fn else torch.int16
            want, before = h.view(bits).clone(), h.view(bits)
            for s in range(6):
                rows = c.rows(s)
                for i in range(length[s]):
                    want[rows[c.ctx[s] + i]] = before[rows[c.ctx[s] + int(path[s, i])]]
            assert torch.equal(d.cpu().view(bits), want)


def test_commit_of_rows_without_pages(dev):
    p = Paged(dev, 22, [10], [20], page=16).upload()
    p.d_table[0, 1] = -1  # rows 16 .. 31 have no page: neither read nor written
    path = torch.tensor([[4, 7, 15]], dtype=torch.int32, device=dev)
    new_ctx = torch.zeros(1, dtype=torch.int32, device=dev)
    announce("pagedCommit rows without a page")
    ops.paged_commit([p.cache], p.batch, path, torch.tensor([3], dtype=torch.int32, device=dev), new_ctx)
    torch.cuda.synchronize()
    want = p.k.clone()
    rows = p.rows(0)
    want[rows[10]] = p.k[rows[14]]  # row 17 has no page; row 25 neither
    assert torch.equal(p.d_k.cpu().view(torch.int16), want.view(torch.int16)) and new_ctx.item() == 13


@pytest.mark.parametrize("hd", [256, 512])
def test_a_drafted_step_equals_the_tokens_one_by_one(dev, hd):
    """A tree of drafts: append, attention, log probabilities, commit; then the accepted path's rows and outputs equal
    those of a cache that took the same tokens one at a time, and the next token's attention agrees."""
    r = np.random.default_rng(hd)
    ctx, parents, path = 37, [-1, 0, 0, 1, 2, 2, 5], [0, 2, 5, 6]
    p = Paged(dev, 30, [ctx], [7], hd=hd, page=16, parents=[parents], spare_pages=2, extra_cols=1)
    one = Paged(dev, 30, [ctx], [7], hd=hd, page=16, spare_pages=2, extra_cols=1)
    for x in (p, one):
        x.upload()
    a = Append(dev, p, 31)
    announce(f"drafted step hd={hd}")
    a.run()
    p.k, p.v = p.d_k.cpu(), p.d_v.cpu()
    tree_out = torch.empty(7, 8, hd, device=dev)
    ws = torch.empty(ops.paged_attn_workspace_bytes(p.cache, p.batch, 8), dtype=torch.uint8, device=dev)
    ops.paged_attn(p.cache, p.batch, a.q_out, tree_out, ws)
    # the drafts' log probabilities under a head over the attention's outputs
    head = torch.from_numpy(r.standard_normal((8 * hd, 1000)).astype(np.float32)).to(dev) * 0.05
    logits = tree_out.reshape(7, -1) @ head
    tokens = torch.tensor([1, 5, 9, 100, 999, 0, 3], dtype=torch.int32, device=dev)
    lp, ent = torch.empty(7, device=dev), torch.empty(7, device=dev)
    ids, tops = torch.empty(7, 4, dtype=torch.int32, device=dev), torch.empty(7, 4, device=dev)
    lws = torch.empty(ops.token_logprobs_workspace_bytes(7, 1000, 4), dtype=torch.uint8, device=dev)
    ops.token_logprobs(logits, tokens, lp, ent, lws, ids, tops, cap=30.0)
    want_lp = torch.log_softmax(30 * torch.tanh(logits.double() / 30), -1)
    assert torch.allclose(lp.double(), want_lp.gather(1, tokens.long()[:, None])[:, 0], atol=2e-5, rtol=0)
    assert torch.equal(ids[:, 0].long(), logits.argmax(-1))
    new_ctx = torch.zeros(1, dtype=torch.int32, device=dev)
    ops.paged_commit([p.cache], p.batch, torch.tensor([path], dtype=torch.int32, device=dev),
                     torch.tensor([len(path)], dtype=torch.int32, device=dev), new_ctx)
    torch.cuda.synchronize()
    assert new_ctx.item() == ctx + 4
    # one by one
    outs = []
    for d, j in enumerate(path):
        c = torch.tensor([ctx + d], dtype=torch.int32, device=dev)
        b = ops.PagedBatch(one.d_table, torch.tensor([0, 1], dtype=torch.int32, device=dev), c, 1)
        qo = torch.empty(1, 8, hd, dtype=torch.float16, device=dev)
        out = torch.empty(1, 8, hd, device=dev)
        ops.paged_append(one.cache, b, a.d["q"][j:j + 1], a.d["k"][j:j + 1], a.d["v"][j:j + 1], a.d["q_weight"],
                         a.d["k_weight"], a.inv, qo, eps=EPS)
        w1 = torch.empty(ops.paged_attn_workspace_bytes(one.cache, b, 8), dtype=torch.uint8, device=dev)
        ops.paged_attn(one.cache, b, qo, out, w1)
        outs.append(out[0])
    torch.cuda.synchronize()
    for d, row in enumerate(p.rows(0)[ctx:ctx + 4]):
        assert torch.equal(p.d_k[row], one.d_k[row]) and torch.equal(p.d_v[row], one.d_v[row])
    # The same rows in another order and split: both sides are within their bound of the exact result.
    p.q = a.q_out.cpu().numpy()
    _, tol = p.expected()
    for d, j in enumerate(path):
        assert (tree_out[j] - outs[d]).abs().max().item() <= 2 * tol[j]


@pytest.mark.parametrize("hd,kv,seqs", [(256, "f16", 3), (512, "e4m3", 2), (256, "e4m3", 70)])
def test_a_captured_step_serves_later_steps(dev, hd, kv, seqs):
    """Append, attention, log probabilities and commit captured once, then replayed with other lengths, paths and inputs
    written in place: every replay gives the eager calls' bits, in the outputs and in the pools. 70 sequences of
    a query tile each are more than a wave's scan holds at once."""
    r = np.random.default_rng(seqs)
    longest = [int(x) for x in r.integers(40, 700, seqs)]
    parents = [random_parents(r, 5) for _ in range(seqs)]
    p = Paged(dev, 50, longest, [5] * seqs, hd=hd, page=16, kv=kv, parents=parents)
    p.upload()
    a = Append(dev, p, 51)
    n, vocab, top = p.tokens, 700, 3
    out = torch.zeros(n, p.nqh, hd, device=dev)
    ws = torch.empty(ops.paged_attn_workspace_bytes(p.cache, p.batch, p.nqh), dtype=torch.uint8, device=dev)
    logits = torch.zeros(n, vocab, device=dev)
    tokens = torch.arange(n, dtype=torch.int32, device=dev) % vocab
    lp, ent, tops = torch.zeros(n, device=dev), torch.zeros(n, device=dev), torch.zeros(n, top, device=dev)
    ids = torch.zeros(n, top, dtype=torch.int32, device=dev)
    lws = torch.empty(ops.token_logprobs_workspace_bytes(n, vocab, top), dtype=torch.uint8, device=dev)
    path = torch.zeros(seqs, 5, dtype=torch.int32, device=dev)
    accepted = torch.zeros(seqs, dtype=torch.int32, device=dev)
    new_ctx = torch.zeros(seqs, dtype=torch.int32, device=dev)
    caches = ops.PagedCaches([p.cache])
    results = (a.q_out, out, lp, ent, ids, tops, new_ctx, p.d_k, p.d_v)

    def step():
        ops.paged_append(p.cache, p.batch, **a.d, q_out=a.q_out, eps=EPS)
        ops.paged_attn(p.cache, p.batch, a.q_out, out, ws, sliding_window=256)
        ops.token_logprobs(logits, tokens, lp, ent, lws, ids, tops, cap=30.0)
        ops.paged_commit(caches, p.batch, path, accepted, new_ctx)

    announce(f"captured drafted step hd={hd} {kv} {seqs} sequences")
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    k0, v0 = p.d_k.clone(), p.d_v.clone()
    depth = p.batch.tensors[3] - p.d_ctx.repeat_interleave(5)
    for turn in range(4):
        ctx = torch.tensor([int(r.integers(0, x + 1)) for x in longest], dtype=torch.int32, device=dev)
        p.d_ctx.copy_(ctx)
        p.batch.tensors[3].copy_(ctx.repeat_interleave(5) + depth)
        for s in range(seqs):
            m = int(r.integers(0, 6))
            accepted[s] = m
            path[s, :m] = torch.tensor(sorted(r.choice(5, m, replace=False).tolist()), dtype=torch.int32, device=dev)
        for t in (a.d["q"], a.d["k"], a.d["v"], logits):
            t.normal_(generator=torch.Generator(device=dev).manual_seed(turn))
        got = []
        for run in (step, graph.replay):
            p.d_k.copy_(k0)
            p.d_v.copy_(v0)
            for t in results[:-2]:
                t.zero_()
            run()
            torch.cuda.synchronize()
            got.append([t.clone() for t in results])
        for x, y in zip(*got):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), turn
        assert torch.equal(new_ctx, ctx + accepted)
