"""How g4_linear_e4m3 adds: in f32 for f32 outputs, in small calls and where the caller asks for it; else 16-bit outputs lose what
the 8-bit matrix unit cuts off, and no more. On normal rows, rows with a few loud channels as trained models have them, and rows
whose largest products cancel."""
import pytest
import torch

from batch_rows import E, TYPES, in_8_bits, lora, rounding, within
from conftest import announce
from g4attn import ops
from test_gpu_lora import adapters, cpu
from tile_rows import SIZES, cut, cut_at_most, exact, f32_sums, takes, tile

pytestmark = pytest.mark.gpu

SIDES = [64, 128, 256]


def call(x, xs, w, ws, kind, f32, out=None, stream=None, **kw):
    tokens, rows, n = x.shape[0], w.shape[0], x.shape[1]
    out = torch.full((tokens, rows), 7.0, dtype=TYPES[kind], device=x.device) if out is None else out
    space = torch.full((ops.linear_e4m3_workspace_bytes(tokens, rows, n, kw.get("lora")),), 0xff, dtype=torch.uint8, device=x.device)
    ops.linear_e4m3(x, xs, w, ws, out, space, f32_sums=f32, stream=stream, **kw)
    torch.cuda.synchronize()
    return out


def rows_of(dev, form, seed, tokens, rows, n):
    g = torch.Generator().manual_seed(seed)
    x, w = torch.randn(tokens, n, generator=g), torch.randn(rows, n, generator=g)
    if form == "loud":
        x[:, 5::200] *= 100
    x, xs = in_8_bits(x)
    w, ws = in_8_bits(w * n ** -0.5)
    if form == "cancel":  # two products of 2^15 against each other beside six that the 8-bit unit cuts off at 4
        x, w = x.float() / 16, w.float() / 16
        x[:, 8] = x[:, 9] = 256
        w[:, 8], w[:, 9] = 128, -128
        x, w = x.to(TYPES["e4m3"]), w.to(TYPES["e4m3"])
    return [t.to(dev) for t in (x, xs, w, ws)]


def check(x, xs, w, ws, kind, f32, out, part=0.0, part_tol=0.0):
    tokens, rows, n = x.shape[0], w.shape[0], x.shape[1]
    unit8 = kind != "f32" and not f32 and tile(tokens, rows, n) != 0
    x, w = x.float(), w.float()
    y, scale, size = exact(x, xs, w, ws)
    want = y + part
    tol = f32_sums(size, y, n, unit8) + part_tol + rounding(want, kind)
    within(out, want, tol + (cut_at_most(x, w) * scale.abs() if unit8 else 0), "out")
    if unit8:
        t = torch.linspace(0, tokens - 1, min(24, tokens), device=x.device).long()
        o = torch.linspace(0, rows - 1, min(40, rows), device=x.device).long()
        within(out[t][:, o], want[t][:, o], tol[t][:, o] + cut(x[t], w[o]) * scale[t][:, o].abs(), "out, by what may be cut off")


@pytest.mark.parametrize("form", ["normal", "loud", "cancel"])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("side", SIDES)
@pytest.mark.parametrize("f32", [False, True])
def test_large_calls(dev, form, kind, side, f32):
    tokens, rows = SIZES[side]
    announce(f"linearE4m3 sums tiles of {side} {kind} {form} f32={f32}")
    takes(side, tokens, rows, 784)
    x, xs, w, ws = rows_of(dev, form, side, tokens, rows, 784)
    out = call(x, xs, w, ws, kind, f32)
    check(x, xs, w, ws, kind, f32, out)
    if kind == "f32":
        assert torch.equal(out, call(x, xs, w, ws, kind, not f32))


@pytest.mark.parametrize("form", ["normal", "loud", "cancel"])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("tokens", [1, 17, 64, 130])
def test_small_calls_have_sums_in_f32(dev, form, kind, tokens):
    announce(f"linearE4m3 sums {tokens} tokens {kind} {form}")
    takes(0, tokens, 600, 784)
    x, xs, w, ws = rows_of(dev, form, tokens, tokens, 600, 784)
    out = call(x, xs, w, ws, kind, False)
    check(x, xs, w, ws, kind, True, out)
    assert torch.equal(out, call(x, xs, w, ws, kind, True))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("side", SIDES)
@pytest.mark.parametrize("n", [16, 112, 272, 4112])
def test_sums_in_f32_over_k(dev, kind, side, n):
    tokens, rows = SIZES[side]
    announce(f"linearE4m3 f32 sums tiles of {side} {kind} n={n}")
    takes(side, tokens, rows, n)
    x, xs, w, ws = rows_of(dev, "loud", n, tokens, rows, n)
    check(x, xs, w, ws, kind, True, call(x, xs, w, ws, kind, True))


@pytest.mark.parametrize("kind,low_kind,rank", [("f16", "f16", 16), ("f16", "bf16", 72), ("bf16", "f16", 128), ("bf16", "bf16", 24)])
@pytest.mark.parametrize("side", SIDES)
@pytest.mark.parametrize("runs", [4, 10 ** 6])
def test_sums_in_f32_with_adapters(dev, kind, low_kind, rank, side, runs):
    tokens, rows = SIZES[side]
    announce(f"linearE4m3 f32 sums tiles of {side} {kind} adapters {low_kind} rank={rank}")
    takes(side, tokens, rows, 144)
    low = adapters(dev, rank, 5, rank, (rows - 50, 50), 144, low_kind)
    x, xs, w, ws = rows_of(dev, "loud", rank, tokens, rows, 144)
    runs = min(runs, tokens)
    ids = torch.randint(-1, 5, (runs,), generator=torch.Generator().manual_seed(side), dtype=torch.int32)[torch.arange(tokens) * runs // tokens].to(dev)
    out = call(x, xs, w, ws, kind, True, lora=low, adapter_ids=ids)
    part, tol = (t.to(dev) for t in lora(ids.cpu(), x.cpu().double() * xs.cpu().double()[:, None], *cpu(low)))
    y = exact(x.float(), xs, w.float(), ws)[0]
    check(x, xs, w, ws, kind, True, out, part, tol + (y.abs() + part.abs()) * 4 * E)


@pytest.mark.parametrize("kind,offset,more", [("f16", 1, 8), ("bf16", 4, 3)])
@pytest.mark.parametrize("side", SIDES)
def test_sums_in_f32_strides_streams_graphs(dev, kind, offset, more, side):
    tokens, rows = SIZES[side]
    n, stride = 176, SIZES[side][1] + more
    announce(f"linearE4m3 f32 sums tiles of {side} strided {kind}")
    takes(side, tokens, rows, n)
    x, xs, w, ws = rows_of(dev, "loud", side, tokens, rows, n)
    want = call(x, xs, w, ws, kind, True)
    flat = torch.full((offset + tokens * stride + 8,), 7.0, dtype=TYPES[kind], device=dev)
    out = flat[offset:offset + tokens * stride].view(tokens, stride)[:, :rows]
    torch.cuda.synchronize()
    assert torch.equal(call(x, xs, w, ws, kind, True, out=out, stream=torch.cuda.Stream()), want)
    out.fill_(7.0)
    assert (flat == 7.0).all()
    space = torch.empty(ops.linear_e4m3_workspace_bytes(tokens, rows, n), dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.linear_e4m3(x, xs, w, ws, out, space, f32_sums=True)
    for _ in range(3):
        xs.mul_(-2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(x, xs, w, ws, kind, True))
