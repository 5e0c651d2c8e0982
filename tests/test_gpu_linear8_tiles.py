"""g4_linear_e4m3's forms for many tokens, each at sizes that the launch rule gives it (asserted, so that a change of the rule
cannot empty these): every tile, output type and adapter type against the definition in 64 bits, over one to many stages of k, odd
numbers of outputs, strided outputs, rows that are not finite, other streams, graphs; and few tokens by many outputs."""
import pytest
import torch

from batch_rows import E, TYPES, in_8_bits, lora, rounding, within
from conftest import announce
from g4attn import ops
from test_gpu_linear8 import call, make
from test_gpu_lora import adapters, cpu, fused
from tile_rows import SIZES, cut, cut_at_most, exact, f32_sums, takes, tile

pytestmark = pytest.mark.gpu

SIDES = [64, 128, 256]
KINDS = ["f32", "f16", "bf16"]


def check(x, xs, w, ws, kind, out):
    """All outputs within what the form's unit may leave; of 24 tokens and 40 outputs, the edges among them, within what it really
    may cut off there."""
    tokens, rows, n = x.shape[0], w.shape[0], x.shape[1]
    unit8 = kind != "f32" and tile(tokens, rows, n) != 0
    x, w = x.float(), w.float()
    y, scale, size = exact(x, xs, w, ws)
    tol = f32_sums(size, y, n, unit8) + rounding(y, kind)
    within(out, y, tol + (cut_at_most(x, w) * scale.abs() if unit8 else 0), "out")
    if unit8:
        t = torch.linspace(0, tokens - 1, min(24, tokens), device=x.device).long()
        o = torch.linspace(0, rows - 1, min(40, rows), device=x.device).long()
        off = cut(x[t], w[o]) * scale[t][:, o].abs()
        within(out[t][:, o], y[t][:, o], tol[t][:, o] + off, "out, by what may be cut off")


@pytest.mark.parametrize("side", SIDES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [16, 112, 272, 1536, 4112])
def test_forms(dev, side, kind, n):
    tokens, rows = SIZES[side]
    announce(f"linearE4m3 tiles of {side} {kind} n={n}")
    takes(side, tokens, rows, n)
    x, xs, w, ws = make(dev, side + n, tokens, rows, n)
    check(x, xs, w, ws, kind, call(x, xs, w, ws, kind))


@pytest.mark.parametrize("side,rows", [(64, 832), (64, 834), (128, 1792), (128, 1810), (256, 3584), (256, 3599)])
@pytest.mark.parametrize("kind", KINDS)
def test_whole_tiles_and_other_ends(dev, side, rows, kind):
    tokens = -(-SIZES[side][0] // side) * side
    announce(f"linearE4m3 tiles of {side}, {tokens} x {rows} {kind}")
    takes(side, tokens, rows, 208)
    x, xs, w, ws = make(dev, rows, tokens, rows, 208)
    check(x, xs, w, ws, kind, call(x, xs, w, ws, kind))


@pytest.mark.parametrize("tokens,rows", [(1, 10176), (1, 10241), (16, 12288), (1, 24577), (3, 24600), (1, 49153), (16, 65536),
                                         (60000, 24), (25000, 130), (15000, 7)])
@pytest.mark.parametrize("kind", KINDS)
def test_one_side_short(dev, tokens, rows, kind):
    """A vocabulary by one token, or a few outputs of many: whatever form the rule takes."""
    announce(f"linearE4m3 {tokens} x {rows} {kind}")
    x, xs, w, ws = make(dev, tokens, tokens, rows, 144)
    check(x, xs, w, ws, kind, call(x, xs, w, ws, kind))


@pytest.mark.parametrize("side", SIDES)
@pytest.mark.parametrize("kind,offset,more", [("f32", 0, 7), ("f32", 1, 4), ("f16", 4, 3), ("f16", 1, 8), ("bf16", 3, 5), ("bf16", 8, 15)])
def test_strided_rows(dev, side, kind, offset, more):
    """Inputs and outputs whose tokens lie apart, at odd elements: the bits of contiguous ones, and nothing beside them."""
    tokens, rows = SIZES[side]
    n, stride = 176, SIZES[side][1] + more
    announce(f"linearE4m3 tiles of {side} strided {kind} {offset} {stride}")
    takes(side, tokens, rows, n + 48)
    x, xs, w, ws = make(dev, side, tokens, rows, n)
    apart = torch.full((tokens, n + 48), 0x7F, dtype=torch.uint8, device=dev)
    apart[:, :n] = x.view(torch.uint8)
    flat = torch.full((offset + tokens * stride + 8,), 7.0, dtype=TYPES[kind], device=dev)
    out = flat[offset:offset + tokens * stride].view(tokens, stride)[:, :rows]
    call(apart.view(TYPES["e4m3"])[:, :n], xs, w, ws, out=out)
    assert torch.equal(out, call(x, xs, w, ws, kind))
    out.fill_(7.0)
    assert (flat == 7.0).all()


@pytest.mark.parametrize("side", SIDES)
@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_are_not_finite_stay_alone(dev, side, kind):
    """NaN codes and scales of tokens and outputs, an infinite scale: their rows and columns, and nothing else."""
    tokens, rows = SIZES[side]
    announce(f"linearE4m3 tiles of {side} NaN {kind}")
    takes(side, tokens, rows, 336)
    x, xs, w, ws = make(dev, 10, tokens, rows, 336)
    want = call(x, xs, w, ws, kind)
    bad_t, bad_o = [1, 2, 37, tokens - 1], [0, 40, rows - 1]
    x.view(torch.uint8)[1] = 0x7F
    xs[2] = float("nan")
    x.view(torch.uint8)[37, 335] = 0xFF
    xs[tokens - 1] = float("inf")
    w.view(torch.uint8)[40, 7] = 0xFF
    ws[0] = float("nan")
    w.view(torch.uint8)[rows - 1, 200] = 0x7F
    got = call(x, xs, w, ws, kind)
    assert not got[bad_t].isfinite().any() and not got[:, bad_o].isfinite().any()
    keep_t, keep_o = torch.ones(tokens, dtype=torch.bool, device=dev), torch.ones(rows, dtype=torch.bool, device=dev)
    keep_t[bad_t], keep_o[bad_o] = False, False
    assert torch.equal(got[keep_t][:, keep_o], want[keep_t][:, keep_o])


@pytest.mark.parametrize("side", SIDES)
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_the_same_call_gives_the_same_bits(dev, side, kind):
    """Twice, on another stream, and replayed from a graph over new inputs."""
    tokens, rows = SIZES[side]
    n = 528
    announce(f"linearE4m3 tiles of {side} repeated {kind}")
    takes(side, tokens, rows, n)
    x, xs, w, ws = make(dev, 12, tokens, rows, n)
    want = call(x, xs, w, ws, kind)
    assert torch.equal(call(x, xs, w, ws, kind, spare=1000), want)
    s = torch.cuda.Stream()
    assert torch.equal(call(x, xs, w, ws, kind, stream=s), want)
    out = torch.zeros_like(want)
    space = torch.empty(ops.linear_e4m3_workspace_bytes(tokens, rows, n), dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.linear_e4m3(x, xs, w, ws, out, space)
    for i in range(3):
        x2, xs2, _, _ = make(dev, 20 + i, tokens, rows, n)
        x.copy_(x2)
        xs.copy_(xs2)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(x, xs, w, ws, kind))


@pytest.mark.parametrize("side", SIDES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("low_kind", ["f16", "bf16"])
@pytest.mark.parametrize("rank,runs", [(16, 5), (64, 10 ** 6), (72, 2), (128, 7)])
def test_adapters(dev, side, kind, low_kind, rank, runs):
    """Adapters in the tiles' epilogue: shared by a tile's tokens or one each, a second batch of a rank's steps, segments that end
    inside a tile, tokens without."""
    tokens, rows = SIZES[side]
    n = 144
    announce(f"linearE4m3 tiles of {side} {kind} adapters {low_kind} rank={rank} runs={runs}")
    takes(side, tokens, rows, n)
    low = adapters(dev, rank + side, 6, rank, (rows - 317, 250, 67), n, low_kind)
    g = torch.Generator().manual_seed(rank)
    x, xs = (t.to(dev) for t in in_8_bits(torch.randn(tokens, n, generator=g)))
    w, ws = (t.to(dev) for t in in_8_bits(torch.randn(rows, n, generator=g) * n ** -0.5))
    runs = min(runs, tokens)
    ids = torch.randint(-1, 6, (runs,), generator=g, dtype=torch.int32)[torch.arange(tokens) * runs // tokens].to(dev)
    got = fused(low, ids, x, xs, w, ws, kind)
    y, scale, size = exact(x.float(), xs, w.float(), ws)
    unit8 = kind != "f32"
    off = f32_sums(size, y, n, unit8) + (cut_at_most(x.float(), w.float()) * scale.abs() if unit8 else 0)
    part, tol = lora(ids.cpu(), x.cpu().double() * xs.cpu().double()[:, None], *cpu(low))
    want = y.cpu() + part
    within(got.cpu(), want, off.cpu() + tol + (y.cpu().abs() + part.abs()) * 4 * E + rounding(want, kind), "out")
    none = ids < 0
    assert torch.equal(got[none], call(x, xs, w, ws, kind)[none])


def test_adapters_of_tiles_in_a_graph_with_new_ids(dev):
    announce("linearE4m3 tiles, adapters in a graph")
    for side in SIDES:
        tokens, rows = SIZES[side]
        takes(side, tokens, rows, 96)
        low = adapters(dev, side, 5, 24, (rows - 40, 40), 96)
        x, xs, w, ws = make(dev, side, tokens, rows, 96)
        ids = torch.randint(-1, 5, (tokens,), dtype=torch.int32, device=dev)
        want = fused(low, ids, x, xs, w, ws, "f16")
        assert torch.equal(fused(low, ids, x, xs, w, ws, "f16", stream=torch.cuda.Stream()), want)
        out = torch.zeros_like(want)
        space = torch.empty(ops.linear_e4m3_workspace_bytes(tokens, rows, 96, low), dtype=torch.uint8, device=dev)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.linear_e4m3(x, xs, w, ws, out, space, lora=low, adapter_ids=ids)
        for i in range(3):
            ids.copy_((torch.arange(tokens, device=dev) * (i + 1) // 400 % 6 - 1).int())
            space.fill_(0xff)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, fused(low, ids, x, xs, w, ws, "f16"))
