"""g4_lora_add, and g4_linear_e4m3 with adapters, against the definition in 64 bits: ranks, segments that end inside a tile,
types, batches of one adapter, of all different ones and of none, ids out of range, non-finite adapters and tokens, streams,
graphs whose ids change."""
import pytest
import torch

from batch_rows import E, TYPES, in_8_bits, linear, lora, rounding, within
from conftest import announce
from g4attn import ops

pytestmark = pytest.mark.gpu


def adapters(dev, seed, L, rank, widths, n, kind="f16", scales=True):
    g = torch.Generator().manual_seed(seed)
    a = (torch.randn(L, len(widths) * rank, n, generator=g) * n ** -0.5).to(TYPES[kind]).to(dev)
    b = (torch.randn(L, sum(widths), rank, generator=g) * 0.3).to(TYPES[kind]).to(dev)
    s = (0.5 + torch.rand(L, generator=g)).to(dev) if scales else None
    return ops.LoraAdapters(a, b, s, widths)


def cpu(low):
    return low.a.cpu(), low.b.cpu(), None if low.scales is None else low.scales.cpu(), low.widths


def add(low, ids, x, base, xs=None, out=None, stream=None):
    out = torch.full_like(base, 7.0) if out is None else out
    space = torch.full((ops.lora_workspace_bytes(low, x.shape[0]),), 0xff, dtype=torch.uint8, device=x.device)
    ops.lora_add(low, ids, x, base, out, space, x_scales=xs, stream=stream)
    torch.cuda.synchronize()
    return out


def fused(low, ids, x, xs, w, ws, kind="f32", stream=None):
    out = torch.full((x.shape[0], w.shape[0]), 7.0, dtype=TYPES[kind], device=x.device)
    space = torch.full((ops.linear_e4m3_workspace_bytes(x.shape[0], w.shape[0], x.shape[1], low),), 0xff, dtype=torch.uint8,
                       device=x.device)
    ops.linear_e4m3(x, xs, w, ws, out, space, lora=low, adapter_ids=ids, stream=stream)
    torch.cuda.synchronize()
    return out


def batch(dev, seed, tokens, n, kind, L, runs=None):
    """x, x_scales and ids: runs of tokens with an adapter each, some of none."""
    g = torch.Generator().manual_seed(seed)
    x, xs = torch.randn(tokens, n, generator=g), None
    x, xs = in_8_bits(x) if kind == "e4m3" else (x.to(TYPES[kind]), None)
    runs = runs or tokens
    ids = torch.randint(-1, L, (runs,), generator=g, dtype=torch.int32)[torch.arange(tokens) * runs // tokens]
    return x.to(dev), None if xs is None else xs.to(dev), ids.to(dev)


def check_add(dev, seed, tokens, n, low, x_kind="f16", out_kind="f32", runs=None):
    x, xs, ids = batch(dev, seed, tokens, n, x_kind, low.n_adapters, runs)
    base = torch.randn(tokens, low.rows, generator=torch.Generator().manual_seed(seed + 1)).to(TYPES[out_kind]).to(dev)
    got = add(low, ids, x, base, xs).cpu()
    xd = x.cpu().double() * (1 if xs is None else xs.cpu().double()[:, None])
    part, tol = lora(ids.cpu(), xd, *cpu(low))
    want = base.cpu().double() + part
    # Each product's sum is added to the base in f32, as many times as there are segments in reach of a tile.
    within(got, want, tol + (want.abs() + part.abs()) * 4 * E + rounding(want, out_kind), "out")
    none = (ids < 0).cpu()
    assert torch.equal(got[none], base.cpu()[none])


def check_fused(dev, seed, tokens, n, low, kind="f32", runs=None):
    g = torch.Generator().manual_seed(seed + 2)
    x, xs, ids = batch(dev, seed, tokens, n, "e4m3", low.n_adapters, runs)
    w, ws = (t.to(dev) for t in in_8_bits(torch.randn(low.rows, n, generator=g) * n ** -0.5))
    got = fused(low, ids, x, xs, w, ws, kind).cpu()
    y, off = linear(*(t.cpu().float() for t in (x, xs, w, ws)), kind)
    part, tol = lora(ids.cpu(), x.cpu().double() * xs.cpu().double()[:, None], *cpu(low))
    want = y + part
    within(got, want, off + tol + (y.abs() + part.abs()) * 4 * E + rounding(want, kind), "out")


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 104, 128])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_ranks(dev, rank, kind):
    announce(f"lora rank={rank} {kind}")
    low = adapters(dev, rank, 5, rank, (72, 24, 40), 272, kind)
    check_add(dev, rank, 37, 272, low, kind, "f32")
    check_fused(dev, rank, 37, 272, low)
    check_fused(dev, rank + 1, 300, 272, low, runs=4)


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 48, 63, 64, 65, 200, 256, 257, 300, 1000])
@pytest.mark.parametrize("runs", [1, 3, 1000])
def test_tokens(dev, tokens, runs):
    announce(f"lora tokens={tokens} runs={runs}")
    low = adapters(dev, tokens, 9, 16, (130, 30), 160)
    check_add(dev, tokens, tokens, 160, low, "f16", "f32", min(runs, tokens))
    check_fused(dev, tokens, tokens, 160, low, "f32", min(runs, tokens))


@pytest.mark.parametrize("widths", [(1,), (7,), (16,), (1000, 24), (5, 3, 8, 1), (2048, 256, 256), (15, 1, 16), (300, 1, 1, 300)])
@pytest.mark.parametrize("tokens", [1, 40, 270])
def test_segments(dev, widths, tokens):
    announce(f"lora widths={widths} tokens={tokens}")
    low = adapters(dev, sum(widths), 4, 8, widths, 128)
    check_add(dev, tokens, tokens, 128, low)
    check_fused(dev, tokens, tokens, 128, low, "bf16")


@pytest.mark.parametrize("x_kind", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("out_kind", ["f32", "f16", "bf16"])
def test_types(dev, x_kind, kind, out_kind):
    announce(f"lora x={x_kind} adapters={kind} out={out_kind}")
    low = adapters(dev, 7, 6, 24, (100,), 336, kind, scales=out_kind == "f32")
    check_add(dev, 8, 50, 336, low, x_kind, out_kind, runs=9)
    check_add(dev, 9, 330, 336, low, x_kind, out_kind, runs=5)


@pytest.mark.parametrize("x_kind,kind", [("f16", "f16"), ("bf16", "bf16"), ("e4m3", "f16"), ("e4m3", "bf16"), ("f32", "f16"),
                                         ("bf16", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("tokens,rank,widths,n", [(530, 16, (40,), 4112), (1100, 128, (9, 20, 8, 3), 64), (2050, 24, (30, 30), 400)])
@pytest.mark.parametrize("runs", [5, 5000])
def test_down_products_by_tiles(dev, x_kind, kind, tokens, rank, widths, n, runs):
    """More than 2^25 products' worth of adapters: runs of tokens, and tiles whose every token has another adapter."""
    announce(f"lora tiles x={x_kind} adapters={kind} tokens={tokens} runs={runs}")
    low = adapters(dev, tokens, 7, rank, widths, n, kind)
    assert tokens * low.a.shape[1] * n > 1 << 25
    check_add(dev, runs, tokens, n, low, x_kind, "f32", min(runs, tokens))


@pytest.mark.parametrize("n", [16, 32, 48, 64, 80, 128, 1008, 1536, 2064, 8192])
@pytest.mark.parametrize("tokens", [1, 20, 260])
def test_inputs(dev, n, tokens):
    announce(f"lora n={n} tokens={tokens}")
    low = adapters(dev, n, 3, 16, (40, 24), n)
    check_add(dev, n, tokens, n, low, "f32" if n % 3 else "bf16")
    check_fused(dev, n, tokens, n, low)


def test_sixty_four_requests_of_forty_adapters(dev):
    announce("lora 64 requests")
    low = adapters(dev, 64, 40, 16, (2048, 256, 256), 1536)
    check_fused(dev, 64, 64, 1536, low)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_more_tiles_than_compute_units(dev, kind):
    announce(f"lora many tiles {kind}")
    low = adapters(dev, 65, 5, 24, (4000, 56, 300), 128, "bf16" if kind == "f32" else "f16")
    check_fused(dev, 66, 4360, 128, low, kind, runs=11)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_sizes_of_the_inner_sums(dev, kind):
    """Inner sums from 1e-30 to 1e30, and some far below a token's largest."""
    announce(f"lora inner sums {kind}")
    low = adapters(dev, 5, 2, 16, (64,), 64, kind)
    low.a[:, ::3] *= 2.0 ** -9
    x = torch.randn(40, 64, generator=torch.Generator().manual_seed(3))
    x *= torch.logspace(-30, 30, 40)[:, None]
    x, ids = x.to(dev), (torch.arange(40, dtype=torch.int32) % 3 - 1).to(dev)
    base = torch.zeros(40, 64, device=dev)
    got = add(low, ids, x, base).cpu()
    part, tol = lora(ids.cpu(), x.cpu(), *cpu(low))
    within(got, part, tol + part.abs() * 4 * E + rounding(part, "f32"), "out")


@pytest.mark.parametrize("tokens", [6, 300])
def test_adapters_past_32_bits(dev, tokens):
    """The last of 1100 adapters begins 4.6e9 elements after the first."""
    L, n, widths = 1100, 8192, (16, 8, 24, 16)
    announce(f"lora adapters past 32 bits, tokens={tokens}")
    small = adapters(dev, 39, 2, 128, widths, n)
    a = torch.empty(L, 512, n, dtype=torch.float16, device=dev)
    b = torch.empty(L, 64, 128, dtype=torch.float16, device=dev)
    a[0], a[L - 1], b[0], b[L - 1] = small.a[0], small.a[1], small.b[0], small.b[1]
    low = ops.LoraAdapters(a, b, None, widths)
    same = ops.LoraAdapters(small.a, small.b, None, widths)
    ids = (torch.arange(tokens, dtype=torch.int32, device=dev) % 3 - 1)
    x = torch.randn(tokens, n, generator=torch.Generator().manual_seed(4)).half().to(dev)
    base = torch.zeros(tokens, 64, device=dev)
    assert torch.equal(add(low, torch.where(ids == 1, L - 1, ids).int(), x, base), add(same, ids, x, base))


@pytest.mark.parametrize("tokens", [6, 300])
def test_ids_out_of_range_and_other_adapters_do_not_matter(dev, tokens):
    announce(f"lora ids {tokens}")
    low = adapters(dev, 31, 4, 16, (90,), 192)
    x, _, ids = batch(dev, 32, tokens, 192, "f16", 3)
    base = torch.randn(tokens, 90, device=dev)
    want = add(low, ids, x, base)
    low.a[3] = float("nan")
    low.b[3] = float("inf")
    low.scales[3] = float("nan")
    odd = ids.clone()
    odd[ids < 0] = torch.tensor([4, -1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=dev)[
        torch.arange(int((ids < 0).sum()), device=dev) % 4]
    assert torch.equal(add(low, odd, x, base), want)
    w, ws = (t.to(dev) for t in in_8_bits(torch.randn(90, 192, generator=torch.Generator().manual_seed(1))))
    x8, xs = (t.to(dev) for t in in_8_bits(x.cpu()))
    clean = fused(low, ids, x8, xs, w, ws)
    assert clean.isfinite().all()
    ids[1] = 3
    got = fused(low, ids, x8, xs, w, ws)
    keep = torch.arange(tokens) != 1
    assert torch.equal(got[keep], clean[keep]) and not got[1].isfinite().any()


@pytest.mark.parametrize("tokens", [5, 300])
def test_a_token_that_is_not_finite_stays_alone(dev, tokens):
    announce(f"lora NaN token {tokens}")
    low = adapters(dev, 33, 2, 16, (80,), 192)
    x, _, _ = batch(dev, 34, tokens, 192, "f16", 2)
    ids = torch.zeros(tokens, dtype=torch.int32, device=dev)
    base = torch.randn(tokens, 80, device=dev)
    want = add(low, ids, x, base)
    x[2, 100], x[3, 5] = float("nan"), float("inf")
    got = add(low, ids, x, base)
    keep = (torch.arange(tokens) != 2) & (torch.arange(tokens) != 3)
    assert torch.equal(got[keep], want[keep]) and not got[2:4].isfinite().any()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [1, 20, 300])
def test_strides_and_in_place(dev, kind, tokens):
    """x, base and out from larger buffers, odd offsets of the outputs; out over base."""
    announce(f"lora strides {kind} {tokens}")
    low = adapters(dev, 35, 3, 8, (50, 11), 96)
    x, _, ids = batch(dev, 36, tokens, 96, "f16", 3)
    base = torch.randn(tokens, 61, device=dev).to(TYPES[kind])
    want = add(low, ids, x, base)
    wide = torch.zeros(tokens, 120, dtype=x.dtype, device=dev)
    wide[:, 8:104] = x
    b = torch.zeros(tokens, 67, dtype=base.dtype, device=dev)
    b[:, 3:64] = base
    o = torch.full((tokens, 71), 7.0, dtype=base.dtype, device=dev)
    add(low, ids, wide[:, 8:104], b[:, 3:64], out=o[:, 5:66])
    assert torch.equal(o[:, 5:66], want) and (o[:, :5] == 7).all() and (o[:, 66:] == 7).all()
    add(low, ids, x, base, out=base)
    assert torch.equal(base, want)


@pytest.mark.parametrize("tokens", [1, 33, 400])
def test_streams_and_graphs_with_new_ids(dev, tokens):
    announce(f"lora graph {tokens}")
    low = adapters(dev, 37, 6, 16, (160, 32), 320)
    x, xs, ids = batch(dev, 38, tokens, 320, "e4m3", 6)
    w, ws = (t.to(dev) for t in in_8_bits(torch.randn(192, 320, generator=torch.Generator().manual_seed(2))))
    base = torch.randn(tokens, 192, device=dev)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert torch.equal(fused(low, ids, x, xs, w, ws, stream=s), fused(low, ids, x, xs, w, ws))
    assert torch.equal(add(low, ids, x, base, xs, stream=s), add(low, ids, x, base, xs))
    out, out2 = torch.zeros(tokens, 192, device=dev), torch.zeros(tokens, 192, device=dev)
    space = torch.empty(ops.linear_e4m3_workspace_bytes(tokens, 192, 320, low), dtype=torch.uint8, device=dev)
    space2 = torch.empty(ops.lora_workspace_bytes(low, tokens), dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.linear_e4m3(x, xs, w, ws, out, space, lora=low, adapter_ids=ids)
        ops.lora_add(low, ids, x, base, out2, space2, x_scales=xs)
    for i in range(3):
        ids.copy_(torch.randint(-1, 6, (tokens,), dtype=torch.int32, device=dev))
        space.fill_(0xff)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fused(low, ids, x, xs, w, ws)) and torch.equal(out2, add(low, ids, x, base, xs))
