"""Paged caches and batches for the tests, and the operators' definitions in 64 bits on the CPU."""
import numpy as np
import torch

from g4attn import ops

EPS = 1e-6


def normed(x, scale=1.0):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * scale


class Paged:
    """A batch of sequences: `ctx` committed rows and `new` tokens each, pages in shuffled order.
    parents: per sequence a list of parent indices (-1: the root), or None for a chain."""

    def __init__(self, dev, seed, ctx, new, hd=256, nqh=8, nkh=1, page=16, kv="f16", parents=None, masks=None,
                 positions=None, pad=0, spare_pages=3, extra_cols=0, max_tokens=None):
        self.r = r = np.random.default_rng(seed)
        self.dev, self.ctx, self.new, self.hd, self.nqh, self.nkh, self.page, self.kv = dev, list(ctx), list(new), hd, nqh, nkh, page, kv
        need = [max(1, -(-(c + t) // page)) for c, t in zip(ctx, new)]
        self.num_pages = sum(need) + spare_pages
        order = r.permutation(self.num_pages)
        self.table = np.full((len(ctx), max(need) + extra_cols), -7, np.int32)  # unused entries name no page
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.tokens = int(self.start[-1]) + pad
        self.q = normed(r.standard_normal((self.tokens, nqh, hd))).astype(np.float16)
        shape = (self.num_pages, page, nkh, hd)
        dt = torch.float8_e4m3fn if kv == "e4m3" else torch.float16
        self.k = torch.from_numpy(normed(r.standard_normal(shape), 0.125)).to(dt)
        self.v = torch.from_numpy(normed(r.standard_normal(shape))).to(dt)
        self.masks = None  # per token the set of new tokens attended
        self.positions = None
        if parents is not None:
            self.masks, pos = [], []
            for s, ps in enumerate(parents):
                seen, depth = [], []
                for j, p in enumerate(ps):
                    seen.append((seen[p] if p >= 0 else set()) | {j})
                    depth.append(depth[p] + 1 if p >= 0 else 0)
                self.masks += seen
                pos += [self.ctx[s] + d for d in depth]
            self.positions = np.array(pos + [0] * pad, np.int32)
        if masks is not None:
            self.masks = masks
        if positions is not None:
            self.positions = np.asarray(positions, np.int32)
        self.max_tokens = max(max(new), 1) if max_tokens is None else max_tokens

    def mask_words(self):
        if self.masks is None:
            return None
        words = max(1, -(-self.max_tokens // 64))
        m = np.zeros((self.tokens, words), np.uint64)
        for t, seen in enumerate(self.masks):
            for j in seen:
                m[t, j // 64] |= np.uint64(1 << (j % 64))
        return m.view(np.int64)

    def upload(self):
        dev = self.dev
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
        self.d_k, self.d_v = self.k.to(dev), self.v.to(dev)
        self.cache = ops.PagedCache(self.d_k, self.d_v)
        words = self.mask_words()
        self.d_ctx, self.d_start, self.d_table = t(np.array(self.ctx, np.int32)), t(self.start), t(self.table)
        self.batch = ops.PagedBatch(self.d_table, self.d_start, self.d_ctx, self.tokens, max_tokens=self.max_tokens,
                                    positions=None if self.positions is None else t(self.positions),
                                    tree_mask=None if words is None else t(words))
        self.d_q = t(self.q)
        return self

    def attn(self, window=0, scale=1.0, softcap=0.0, out=None, ws=None, stream=None):
        if out is None:
            out = torch.full((self.tokens, self.nqh, self.hd), -123.0, device=self.dev)
        if ws is None:
            ws = torch.empty(ops.paged_attn_workspace_bytes(self.cache, self.batch, self.nqh), dtype=torch.uint8,
                             device=self.dev)
            ws.fill_(0xff)  # NaNs: nothing may be read that the call did not write
        ops.paged_attn(self.cache, self.batch, self.d_q, out, ws, scale=scale, sliding_window=window, softcap=softcap,
                       stream=stream)
        return out

    def rows(self, s):
        """(page, row in it) of the sequence's rows; None where the table names no page."""
        got = []
        for r in range(self.ctx[s] + self.new[s]):
            p = int(self.table[s, r // self.page]) if r // self.page < self.table.shape[1] else -1
            got.append((p, r % self.page) if 0 <= p < self.num_pages else None)
        return got

    def expected(self, window=0, scale=1.0, softcap=0.0):
        """(out in 64 bits, a bound of the kernel's error per token): see the comment below."""
        k, v = self.k.double().numpy(), self.v.double().numpy()
        out = np.zeros((self.tokens, self.nqh, self.hd))
        tol = np.zeros(self.tokens)
        G = self.nqh // self.nkh
        for s in range(len(self.ctx)):
            n, t = self.ctx[s], self.new[s]
            if not t:
                continue
            place = self.rows(s)
            pos_new = [n + j for j in range(t)] if self.positions is None else \
                [int(self.positions[self.start[s] + j]) for j in range(t)]
            for j in range(t):
                tok = int(self.start[s]) + j
                see = []
                for r in range(n + t):
                    if place[r] is None:
                        continue
                    if r >= n:
                        dj = r - n
                        if self.masks is not None:
                            if dj not in self.masks[tok]:
                                continue
                        elif dj > j:
                            continue
                    rp = r if r < n else pos_new[r - n]
                    if window and not rp > pos_new[j] - window:
                        continue
                    see.append(place[r])
                if not see:
                    continue
                pg, off = np.array(see).T
                for h in range(self.nqh):
                    kk, vv, qq = k[pg, off, h // G], v[pg, off, h // G], self.q[tok, h].astype(np.float64)
                    x = kk @ qq * scale
                    if softcap:
                        x = softcap * np.tanh(x / softcap)
                    p = np.exp(x - x.max())
                    out[tok, h] = (p / p.sum()) @ vv
                    # A score is HD / 32 accumulations of 32 products each, off by at most
                    # (HD / 32 + 32) half-steps of the sum of magnitudes; scale, cap (tanh: 4) and the
                    # exponent add 8 of the score; the weights are off by twice that, relatively, and P by
                    # 2^-22; the sums over the rows by half-steps of their partial sums, at most 64 here
                    # (32-row tiles summed in turn by 4 waves, then joined).
                    mag = (np.abs(kk) @ np.abs(qq)).max() * abs(scale)
                    ds = ((self.hd / 32 + 32) * mag + 8 * (np.abs(x).max() + softcap)) * 2.0 ** -24
                    tol[tok] = max(tol[tok], (2 * ds + 2.0 ** -22 + 64 * 2.0 ** -24) * 2 * np.abs(vv).max())
        return out, tol

    def check(self, out, **kw):
        want, tol = self.expected(**kw)
        got = out.cpu().numpy()
        live = int(self.start[-1])
        assert np.isfinite(got[:live]).all()
        err = np.abs(got[:live] - want[:live]).max(axis=(1, 2))
        worst = int(np.argmax(err - tol[:live]))
        assert (err <= tol[:live]).all(), f"token {worst}: off by {err[worst]:.3e}, bound {tol[worst]:.3e}"
        assert (got[live:] == -123.0).all(), "padding tokens were written"


def random_parents(r, t):
    return [int(r.integers(-1, j)) if j else -1 for j in range(t)]
