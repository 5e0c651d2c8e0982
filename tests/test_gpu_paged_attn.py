"""g4_paged_attn against the definition in 64 bits: lengths from one row on, page and tile edges, head layouts, trees,
windows, ragged and padded batches, pages that are none, Inf and NaN where a token does not look, captured replays,
streams and offsets past 4 GiB. Tolerances are derived in paged_helpers.Paged.expected."""
import numpy as np
import pytest
import torch

from conftest import announce
from paged_helpers import Paged, random_parents

pytestmark = pytest.mark.gpu


def run(p, **kw):
    out = p.upload().attn(**kw)
    torch.cuda.synchronize()
    p.check(out, **kw)
    return out


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("ctx", [0, 1, 15, 16, 31, 32, 33, 127, 128, 129, 300])
def test_single_token_lengths(dev, hd, kv, ctx):
    announce(f"pagedAttn one token hd={hd} kv={kv} ctx={ctx}")
    run(Paged(dev, ctx + hd, [ctx], [1], hd=hd, kv=kv, page=16 << (ctx % 3)))


@pytest.mark.parametrize("hd,nqh,nkh", [(256, 8, 1), (256, 8, 2), (256, 6, 2), (256, 4, 4), (256, 5, 1), (256, 7, 1),
                                        (512, 8, 1), (512, 8, 4), (512, 3, 1), (512, 2, 2)])
@pytest.mark.parametrize("new", [1, 3, 9, 20])
def test_head_layouts(dev, hd, nqh, nkh, new):
    announce(f"pagedAttn heads hd={hd} {nqh}/{nkh} new={new}")
    run(Paged(dev, 40 + new, [70, 5], [new, max(1, new - 2)], hd=hd, nqh=nqh, nkh=nkh, page=32))


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("ctx,new", [(0, 1), (0, 33), (0, 100), (40, 65), (257, 130), (96, 64)])
def test_chains(dev, hd, ctx, new):
    announce(f"pagedAttn chain hd={hd} ctx={ctx} new={new}")
    run(Paged(dev, ctx + new, [ctx], [new], hd=hd, page=64))


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("window", [0, 1, 20, 64])
def test_trees(dev, hd, kv, window):
    r = np.random.default_rng(window)
    new = [1, 7, 26, 64, 2]
    announce(f"pagedAttn trees hd={hd} kv={kv} window={window}")
    run(Paged(dev, 3 + window, [90, 0, 130, 33, 64], new, hd=hd, kv=kv, page=16,
              parents=[random_parents(r, t) for t in new]), window=window)


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("new", [65, 150])
def test_masks_of_several_words(dev, new, window):
    """Any mask, not only a tree's: tokens may look ahead (a prefix), and some look at nothing of the new ones."""
    r = np.random.default_rng(new)
    masks = [set(np.flatnonzero(r.random(new) < 0.3).tolist()) for _ in range(new)]
    masks[3] = set()
    announce(f"pagedAttn mask words new={new} window={window}")
    run(Paged(dev, new, [50], [new], page=32, masks=masks, positions=[50 + j // 2 for j in range(new)]), window=window)


def test_tokens_that_attend_nothing_get_zero(dev):
    announce("pagedAttn empty masks")
    p = Paged(dev, 9, [0, 0, 40], [3, 1, 2], masks=[set(), {0}, set(), set(), {0}, set()], positions=[5, 0, 100, 0, 40, 90])
    out = run(p, window=8)
    got = out.cpu().numpy()
    assert (got[[0, 2, 3]] == 0).all()
    assert (got[5] == 0).all()  # position 90: the window has left every row behind


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 5000, 1 << 31])
def test_windows_of_single_tokens_and_chains(dev, window):
    announce(f"pagedAttn window={window}")
    run(Paged(dev, 11, [200, 31, 64, 0], [1, 1, 40, 5], page=16), window=window)


@pytest.mark.parametrize("softcap,scale", [(50.0, 1.0), (2.0, 1.0), (0.0, 0.0625), (30.0, 2.0), (0.0, -0.5), (0.0, 0.0)])
def test_caps_and_scales(dev, softcap, scale):
    announce(f"pagedAttn softcap={softcap} scale={scale}")
    run(Paged(dev, 21, [100, 3], [2, 4], page=64), softcap=softcap, scale=scale)


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("page", [16, 32, 128, 1024])
def test_ragged_batches_with_padding(dev, hd, page):
    """Empty sequences, sequences of one row, more padding tokens than a tile, a block table wider than needed."""
    r = np.random.default_rng(page)
    new = [int(r.integers(0, 9)) for _ in range(11)]
    ctx = [int(r.integers(0, 200)) for _ in range(11)]
    new[0], new[-1], ctx[2] = 0, 0, 0
    announce(f"pagedAttn ragged hd={hd} page={page} new={new} ctx={ctx}")
    run(Paged(dev, page, ctx, new, hd=hd, page=page, pad=70, extra_cols=3))


@pytest.mark.parametrize("seqs", [64, 65, 200])
def test_many_sequences(dev, seqs):
    r = np.random.default_rng(seqs)
    new = [int(r.integers(0, 4)) for _ in range(seqs)]
    new[-1] = 2
    announce(f"pagedAttn {seqs} sequences")
    run(Paged(dev, seqs, [int(r.integers(0, 90)) for _ in range(seqs)], new, nqh=4, page=16))


@pytest.mark.parametrize("ctx,new,nqh,nkh,hd", [(9000, 1, 8, 1, 256), (20000, 4, 8, 2, 256), (6000, 9, 8, 1, 512)])
def test_items_cut_between_workgroups(dev, ctx, new, nqh, nkh, hd):
    announce(f"pagedAttn long ctx={ctx} new={new}")
    run(Paged(dev, ctx, [ctx, 37, ctx // 3], [new, 1, new], nqh=nqh, nkh=nkh, hd=hd, page=64))


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("bad", [-1, -2 ** 31, 2 ** 31 - 1, "num_pages"])
def test_rows_without_a_page_are_not_attended(dev, hd, bad):
    p = Paged(dev, 31, [200, 60], [3, 2], hd=hd, page=16)
    bad = p.num_pages if bad == "num_pages" else bad
    p.table[0, [0, 5]] = bad
    p.table[1, :] = bad
    announce(f"pagedAttn bad pages {bad} hd={hd}")
    out = run(p)
    assert (out.cpu().numpy()[3:5] == 0).all()


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_rows_a_token_does_not_attend_do_not_reach_it(dev, hd, kv, value):
    """Inf and NaN in drafted rows of other branches, before the window, behind the last row and in spare pages."""
    parents = [[-1, -1, 0, 1, 0, 2, -1]]
    p = Paged(dev, 77, [45], [7], hd=hd, kv=kv, page=16, parents=parents)
    p.masks[6] = set()  # the last row is attended by nobody
    window = 20
    clean = Paged(dev, 77, [45], [7], hd=hd, kv=kv, page=16, parents=parents)
    clean.masks[6] = set()
    want, tol = clean.expected(window=window)
    value = float("nan") if kv == "e4m3" else value
    flat_k, flat_v = p.k.float(), p.v.float()
    used = {(int(p.table[0, x // 16]), x % 16) for x in range(52)}
    for pg in range(p.num_pages):
        for o in range(16):
            if (pg, o) not in used:
                flat_k[pg, o], flat_v[pg, o] = value, value
    poisoned = list(range(0, 26 - 1)) + [45 + 1, 45 + 3, 45 + 6]  # before every window; the branch 1 -> 3; row 6
    for x in poisoned:
        pg, o = int(p.table[0, x // 16]), x % 16
        flat_k[pg, o, :, ::7], flat_v[pg, o, :, 1::3] = value, value
    p.k, p.v = flat_k.to(p.k.dtype), flat_v.to(p.v.dtype)
    announce(f"pagedAttn odd rows hd={hd} kv={kv} {value}")
    got = p.upload().attn(window=window).cpu().numpy()
    for tok in (0, 2, 4, 5, 6):  # tokens off the poisoned branch
        assert np.abs(got[tok] - want[tok]).max() <= tol[tok], tok
    for tok in (1, 3):  # on it: the odd elements' columns are not finite
        assert not np.isfinite(got[tok]).all()


def test_same_call_same_bits_and_other_streams(dev):
    r = np.random.default_rng(8)
    p = Paged(dev, 8, [700, 40, 3000], [8, 8, 8], page=64, parents=[random_parents(r, 8) for _ in range(3)]).upload()
    announce("pagedAttn streams")
    want = p.attn()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:  # a workspace each, at the same time
        with torch.cuda.stream(s):
            outs.append(p.attn())
    torch.cuda.synchronize()
    outs.append(p.attn(stream=streams[0]))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o.view(torch.int32), want.view(torch.int32))


def test_captured_step_replays_with_new_lengths(dev):
    """The lengths and pages are read when the kernels run: a captured call serves the steps that follow."""
    p = Paged(dev, 14, [300, 20], [4, 1], page=16, extra_cols=2)
    p.upload()
    out = torch.full((5, 8, 256), -123.0, device=dev)
    from g4attn import ops
    ws = torch.empty(ops.paged_attn_workspace_bytes(p.cache, p.batch, 8), dtype=torch.uint8, device=dev)
    announce("pagedAttn captured")
    p.attn(out=out, ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.attn(out=out, ws=ws)
    for ctx in ([300, 20], [180, 19], [0, 3], [299, 11]):
        p.ctx = ctx
        p.d_ctx.copy_(torch.tensor(ctx, dtype=torch.int32))
        out.fill_(-123.0)
        graph.replay()
        torch.cuda.synchronize()
        p.check(out)
        replayed = out.clone()
        p.attn(out=out, ws=ws)
        torch.cuda.synchronize()
        assert torch.equal(out, replayed)


def test_two_captured_graphs_share_a_workspace_in_turn(dev):
    a, b = (Paged(dev, s, [900 + s], [3], page=64).upload() for s in (1, 2))
    from g4attn import ops
    ws = torch.empty(ops.paged_attn_workspace_bytes(a.cache, a.batch, 8), dtype=torch.uint8, device=dev)
    outs, graphs = [], []
    announce("pagedAttn two graphs, one workspace")
    for p in (a, b):
        out = torch.full((3, 8, 256), -123.0, device=dev)
        p.attn(out=out, ws=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            p.attn(out=out, ws=ws)
        outs.append(out)
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.fill_(-123.0)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        a.check(outs[0])
        b.check(outs[1])


def test_rows_past_4_gib(dev):
    """Pages at the end of a pool of 5 GiB a side."""
    hd, nkh, page, pages = 512, 8, 64, 10240
    announce("pagedAttn pool of 5 GiB")
    small = Paged(dev, 3, [100], [2], hd=hd, nqh=8, nkh=nkh, page=page, spare_pages=0)
    big = [torch.empty(pages, page, nkh, hd, dtype=torch.float16, device=dev) for _ in range(2)]
    n = small.num_pages
    for b, x in zip(big, (small.k, small.v)):
        b[pages - n:] = x.to(dev)
    want, tol = small.expected()
    small.table += pages - n
    small.k, small.v = big
    out = small.upload().attn()
    got = out.cpu().numpy()
    assert (np.abs(got - want).max(axis=(1, 2)) <= tol).all()


def test_device_arrays_out_of_range_are_cut(dev):
    """Token ranges, lengths and positions beyond the buffers: defined, nothing outside is touched."""
    p = Paged(dev, 66, [100, 50], [3, 4], page=16, pad=2)
    p.upload()
    announce("pagedAttn arrays out of range")
    p.d_ctx.copy_(torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32))  # cut to the block table's rows, and to 0
    p.d_start.copy_(torch.tensor([-3, 3, 2 ** 31 - 1], dtype=torch.int32))
    out = p.attn()
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    rows = p.table.shape[1] * p.page
    q = Paged(dev, 66, [rows, 0], [3, 4], page=16, pad=2)
    q.table, q.k, q.v, q.q, q.num_pages = p.table, p.k, p.v, p.q, p.num_pages
    want, tol = q.expected()
    # max_tokens cuts the second sequence's range to its first four tokens; its rows start at 0
    assert (np.abs(got[:7] - want[:7]).max(axis=(1, 2)) <= tol[:7]).all()
    assert (got[7:] == -123.0).all()


@pytest.mark.parametrize("case", range(16))
def test_random_batches(dev, case):
    r = np.random.default_rng(4000 + case)
    hd = int(r.choice([256, 512]))
    nkh = int(r.choice([1, 1, 2, 4]))
    nqh = nkh * int(r.choice([1, 2, 3, 4, 8]))
    seqs = int(r.integers(1, 7))
    tree = bool(r.integers(2))
    most = int(r.choice([1, 4, 20, 64]))
    new = [int(r.integers(0, most + 1)) for _ in range(seqs)]
    new[0] = most
    ctx = [int(r.integers(0, r.choice([40, 700]))) for _ in range(seqs)]
    kw = dict(window=int(r.choice([0, 0, 7, 64, 300])), softcap=float(r.choice([0.0, 50.0])))
    p = Paged(dev, 5000 + case, ctx, new, hd=hd, nqh=nqh, nkh=nkh, page=int(r.choice([16, 32, 64, 256])),
              kv=str(r.choice(["f16", "e4m3"])), pad=int(r.integers(0, 5)),
              parents=[random_parents(r, t) for t in new] if tree else None)
    announce(f"pagedAttn random {case}: hd={hd} heads={nqh}/{nkh} ctx={ctx} new={new} tree={tree} kv={p.kv} {kw}")
    run(p, **kw)


@pytest.mark.parametrize("ctx,new,nqh,nkh,hd,kv", [
    ([5000, 10, 700], [40, 1, 0], 8, 2, 512, "f16"),        # three query tiles of two kv heads, some of no tokens
    ([9000, 10], [130, 1], 8, 1, 256, "f16"),               # nine query tiles, eight of them of one sequence
    ([3000, 2999, 1, 0], [33, 17, 33, 1], 8, 4, 256, "e4m3"),
    ([16000], [26], 8, 1, 512, "e4m3"),
    ([12000], [1], 1, 1, 256, "f16"),                       # more pieces than a join's group has records
    ([1500] * 60, [2] * 60, 8, 4, 256, "f16"),              # items fit one scan, their pieces do not fit the workgroups
    ([400, 300, 200], [300, 200, 100], 8, 1, 256, "f16"),   # query tiles that end at different rows
])
def test_pieces_of_items(dev, ctx, new, nqh, nkh, hd, kv):
    announce(f"pagedAttn pieces hd={hd} heads={nqh}/{nkh} {kv} ctx={ctx[:4]} new={new[:4]}")
    run(Paged(dev, 60 + len(ctx), ctx, new, nqh=nqh, nkh=nkh, hd=hd, kv=kv, page=32))


@pytest.mark.parametrize("softcap", [5.0, 50.0, 1e6])
def test_softcaps_on_both_sides_of_the_polynomial(dev, softcap):
    """Scores up to about 8: beyond half of a cap of 5 in every tile, of 50 in none, and tiny against 1e6."""
    announce(f"pagedAttn softcap={softcap} both forms")
    run(Paged(dev, 71, [700, 90], [3, 5], page=64), softcap=softcap)
    run(Paged(dev, 72, [300], [30], hd=512, page=64), softcap=softcap)
