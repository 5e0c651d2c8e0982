"""g4_paged_attn at edges of its tiles, windows and number formats: chains that run past the block table, weights far
below the largest, chunks of several windows, shares of hundreds of tiles, mixed batches, against the definition in 64 bits. Tolerances
are derived in paged_helpers.Paged.expected, or where a test stands."""
import numpy as np
import pytest
import torch

from conftest import announce
from g4attn import ops
from paged_helpers import Paged, normed

pytestmark = pytest.mark.gpu


def run(p, **kw):
    out = p.upload().attn(**kw)
    torch.cuda.synchronize()
    p.check(out, **kw)
    return out


@pytest.mark.parametrize("hd,nqh,new", [(256, 8, 1), (256, 8, 4), (256, 2, 30), (256, 8, 40), (512, 2, 30), (512, 8, 40)])
@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("window", [0, 30])
@pytest.mark.parametrize("ctx", [112, 111, 97, 80])
def test_chains_past_the_block_table(dev, hd, nqh, new, kv, window, ctx):
    """Seven pages of 16 rows: the table ends in the middle of a 32-row tile, whose second half no token attends."""
    announce(f"pagedAttn past the table hd={hd} nqh={nqh} new={new} kv={kv} window={window} ctx={ctx}")
    p = Paged(dev, ctx + new, [ctx, 20], [new, 1], hd=hd, nqh=nqh, kv=kv, page=16)
    p.table = p.table[:, :7].copy()
    run(p, window=window)


# ---- weights far below the largest ------------------------------------------------------

@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("hd,new,rows,sinks", [
    (256, 1, 32768, [0, 32, 64, 96]),  # every fourth tile a wave
    (512, 1, 32768, [0, 32, 64, 96]),
    (256, 4, 32768, [0, 32, 64, 96]),  # 32 query rows
    (256, 8, 16384, [0, 32]),          # 64, two waves a tile
    (256, 16, 16384, [0]),             # 128
    (512, 8, 16384, [0]),
])
def test_weights_far_below_the_largest_add_up(dev, hd, new, rows, sinks, kv):
    """A row 11 to 17 nats above all others, as an attention sink has it, in each wave's share, V of one sign: what
    thousands of small weights add is not lost, nor one-sided. Scores are exact (one element of q and k each), and
    a sequence a compute unit keeps all rows of one in one running state.

    The bound, in units of the largest |v| = 1. Weights: scale and log2(e) round the score twice, the difference from
    the maximum once more (it is at most 2 X + 16 ln 2 nats for scores up to X), the exponent is good to a
    step: (4 X + 14) 2^-24, in the numerator and the denominator. Eight factors of states that are joined: 16. The two
    f16 of a weight: 2^-22 of it, and a row at most 2^-32 of the largest weight (half of f16's least step, if that
    weight is 2^7 or more in f16). Sums: the numerator takes two products a tile of
    32 rows, the denominator four terms, each off by half a step of the partial sum."""
    announce(f"pagedAttn sink hd={hd} new={new} rows={rows} kv={kv}")
    r = np.random.default_rng(hd + new)
    seqs = torch.cuda.get_device_properties(dev).multi_processor_count
    page, nqh = 64, 8
    dt = torch.float8_e4m3fn if kv == "e4m3" else torch.float16
    order = r.permutation(rows // page)
    low = -6.0 if kv == "e4m3" else -5.6875  # 2^-24 times 0.7 and 0.95
    score = np.where(r.random(rows) < 0.75, low, 0.0)
    score[sinks] = 11.0
    v = np.where(r.random((rows, hd)) < 0.5, 1.0, 0.75)
    v[sinks] = 0.0
    k = torch.zeros(rows, hd)
    k[:, 0] = torch.from_numpy(score).float()
    # Row i of every sequence lies in page order[i // page].
    pool = lambda x: torch.empty(rows // page, page, 1, hd).index_copy_(  # noqa: E731
        0, torch.from_numpy(order), x.float().view(rows // page, page, 1, hd)).to(dt).to(dev)
    cache = ops.PagedCache(pool(k), pool(torch.from_numpy(v)))
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    batch = ops.PagedBatch(i32(np.tile(order, (seqs, 1))), i32(np.arange(seqs + 1) * new), i32(np.full(seqs, rows - new)),
                           seqs * new, max_tokens=new)
    factor = np.array([1.0, 1.0, 0.75, 1.0, 0.625, 1.0, 0.5, 0.875])
    q = torch.zeros(seqs * new, nqh, hd)
    q[:, :, 0] = torch.from_numpy(factor).float()
    out = torch.full((seqs * new, nqh, hd), -123.0, device=dev)
    ws = torch.empty(ops.paged_attn_workspace_bytes(cache, batch, nqh), dtype=torch.uint8, device=dev)
    ops.paged_attn(cache, batch, q.half().to(dev), out, ws)
    torch.cuda.synchronize()
    got = out.cpu().double().numpy().reshape(seqs, new, nqh, hd)
    tiles = rows // 32 // (4 if len(sinks) == 4 else len(sinks))
    bound = (2 * (4 * 11.0 + 14) + 16 + 4 + 6 * tiles) * 2.0 ** -24 + rows * 2.0 ** -32
    for j in range(new):
        n = rows - new + j + 1
        p = np.exp(factor[:, None] * (score[None, :n] - 11.0))
        want = (p / p.sum(-1, keepdims=True)) @ v[:n]
        err = np.abs(got[:, j] - want).max()
        assert err <= bound, f"token {j}: off by {err:.3e}, bound {bound:.3e}"


# ---- windows much shorter than a chunk ----------------------------------------------------

@pytest.mark.parametrize("hd,nqh,nkh", [(256, 8, 1), (256, 8, 2), (512, 8, 1)])
@pytest.mark.parametrize("form", ["chain", "mask", "positions"])
@pytest.mark.parametrize("ctx,new,window", [(0, 300, 40), (70, 300, 33), (0, 129, 1), (500, 200, 100)])
def test_chunks_of_several_windows(dev, hd, nqh, nkh, form, ctx, new, window):
    """A chain as such, as a mask of rows that are their own positions, and with positions given."""
    announce(f"pagedAttn chunk hd={hd} heads={nqh}/{nkh} {form} ctx={ctx} new={new} window={window}")
    masks = None if form == "chain" else [set(range(j + 1)) for j in range(new)] + [{0}]
    positions = [ctx + j for j in range(new)] + [9] if form == "positions" else None
    run(Paged(dev, new + window, [ctx, 9], [new, 1], hd=hd, nqh=nqh, nkh=nkh, page=16, masks=masks, positions=positions),
        window=window)


def test_work_on_a_windowed_chunk_grows_with_its_length(dev):
    """Tokens far into a chunk leave its first rows alone: four times the tokens take about four times as long, not the
    sixteen of a full chunk (a factor of 8 lies between)."""
    announce("pagedAttn windowed chunk, time by length")
    hd, nqh, page = 256, 8, 64
    took = []
    for new in (4096, 16384):
        pages = new // page
        pool = [torch.randn(pages, page, 1, hd, device=dev).half() for _ in range(2)]
        i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
        cache = ops.PagedCache(*pool)
        batch = ops.PagedBatch(torch.arange(pages, dtype=torch.int32, device=dev).view(1, -1), i32(0, new), i32(0), new)
        q = torch.randn(new, nqh, hd, device=dev).half()
        out = torch.empty(new, nqh, hd, device=dev)
        ws = torch.empty(ops.paged_attn_workspace_bytes(cache, batch, nqh), dtype=torch.uint8, device=dev)
        best = float("inf")
        for _ in range(8):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            ops.paged_attn(cache, batch, q, out, ws, scale=0.0625, sliding_window=512)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        took.append(best)
    print(f"4096 tokens {1e3 * took[0]:.0f} us, 16384 tokens {1e3 * took[1]:.0f} us", flush=True)
    assert took[1] < 8 * took[0], took


@pytest.mark.parametrize("window", [2 ** 30, 2 ** 30 + 1, 2 ** 31 - 3, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1])
def test_windows_and_positions_up_to_the_largest(dev, window):
    """A position of 2^31 - 2 leaves rows behind for every window that is shorter."""
    announce(f"pagedAttn far position window={window}")
    far = 2 ** 31 - 2
    run(Paged(dev, 5, [40, 33], [2, 20], page=16, positions=[far - 1, far] + [far - 19 + j for j in range(20)]), window=window)


def test_a_mask_of_no_words_is_refused(dev):
    """Its pointer is NULL, which stands for a chain: each token would attend those before it."""
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    for shape in ((3, 0), (3,)):
        with pytest.raises(ValueError, match="tree_mask"):
            ops.PagedBatch(i32([0]), i32(0, 3), i32(0), 3, tree_mask=torch.zeros(shape, dtype=torch.int64, device=dev))


# ---- long shares ------------------------------------------------------------------------

@pytest.mark.parametrize("hd,new,kv", [(256, 1, "f16"), (512, 1, "e4m3"), (256, 4, "e4m3"), (256, 8, "f16"), (256, 16, "f16"),
                                       (512, 8, "f16")])
def test_workgroups_that_read_page_ids_several_times(dev, hd, new, kv):
    """Five sequences of 524288 rows, 320 tiles of 32 rows a workgroup: page ids are held for 64 of a wave's tiles. All
    rows lie in 64 pages, so the definition is a sum over 1024 rows and how often a sequence names them. A page's V has
    an offset of its own, and the pages change every few tiles, so that ids of other tiles would show."""
    announce(f"pagedAttn long shares hd={hd} new={new} kv={kv}")
    r = np.random.default_rng(hd + new)
    seqs, rows, page, pages, nqh = 5, 524288, 16, 64, 8
    dt = torch.float8_e4m3fn if kv == "e4m3" else torch.float16
    k = torch.from_numpy(normed(r.standard_normal((pages, page, 1, hd)), 0.125)).to(dt)
    v = torch.from_numpy(normed(r.standard_normal((pages, page, 1, hd))) + r.choice([-1.0, 1.0], (pages, 1, 1, 1))).to(dt)
    # 11 pages of rows (176 rows, no multiple of a tile) from a page on, then from another.
    i = np.arange(rows // page)
    table = np.stack([(r.integers(0, pages, len(i))[i // 11] + i % 3) % pages for _ in range(seqs)]).astype(np.int32)
    q = normed(r.standard_normal((seqs * new, nqh, hd))).astype(np.float16)
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    cache = ops.PagedCache(k.to(dev), v.to(dev))
    batch = ops.PagedBatch(i32(table), i32(np.arange(seqs + 1) * new), i32(np.full(seqs, rows - new)), seqs * new,
                           max_tokens=new)
    out = torch.full((seqs * new, nqh, hd), -123.0, device=dev)
    ws = torch.empty(ops.paged_attn_workspace_bytes(cache, batch, nqh), dtype=torch.uint8, device=dev)
    ops.paged_attn(cache, batch, torch.from_numpy(q).to(dev), out, ws)
    torch.cuda.synchronize()
    got = out.cpu().double().numpy()
    kk, vv = k.double().numpy().reshape(-1, hd), v.double().numpy().reshape(-1, hd)
    for s in range(seqs):
        at = table[s, np.arange(rows) // page].astype(np.int64) * page + np.arange(rows) % page
        for j in range(new):
            count = np.bincount(at[:rows - new + j + 1], minlength=pages * page)
            x = q[s * new + j].astype(np.float64) @ kk.T
            p = count * np.exp(x - x.max(-1, keepdims=True))
            want = (p / p.sum(-1, keepdims=True)) @ vv
            # As in Paged.expected, with the sums of 320 tiles at most (two products and four terms a tile) and of
            # the records of 52 workgroups; the weights that two f16 leave out are below 2^-32 of the largest.
            mag = (np.abs(q[s * new + j].astype(np.float64)) @ np.abs(kk).T).max()
            ds = ((hd / 32 + 32) * mag + 8 * np.abs(x).max()) * 2.0 ** -24
            bound = (2 * ds + 2.0 ** -22 + rows * 2.0 ** -32 + (6 * 320 + 64) * 2.0 ** -24) * 2 * np.abs(vv).max()
            err = np.abs(got[s * new + j] - want).max()
            assert err <= bound, f"sequence {s} token {j}: off by {err:.3e}, bound {bound:.3e}"


@pytest.mark.parametrize("form", ["one call", "two calls"])
def test_a_chunk_beside_single_tokens(dev, form):
    """In one batch, or as two over the same token buffers: tokens of no sequence are left alone."""
    announce(f"pagedAttn chunk and single tokens, {form}")
    new = [150] + [1] * 20
    p = Paged(dev, 31, [70] + [5 * i for i in range(20)], new, page=16).upload()
    if form == "one call":
        p.check(p.attn())
        return
    out = torch.full((p.tokens, p.nqh, p.hd), -123.0, device=dev)
    whole = p.batch
    parts = [ops.PagedBatch(p.d_table[a:b].contiguous(), p.d_start[a:b + 1].contiguous(), p.d_ctx[a:b].contiguous(), p.tokens,
                            max_tokens=most) for a, b, most in ((0, 1, 150), (1, 21, 1))]
    p.batch = parts[0]
    p.attn(out=out)
    torch.cuda.synchronize()
    assert (out[150:] == -123.0).all()
    p.batch = parts[1]
    p.attn(out=out)
    p.batch = whole
    torch.cuda.synchronize()
    p.check(out)
