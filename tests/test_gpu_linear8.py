"""g4_linear_e4m3 against the definition in 64 bits: token counts, outputs and inputs around every tile's edge, types, strides
and alignment, non-finite rows, workspaces, other streams, graphs."""
import pytest
import torch

from batch_rows import TYPES, in_8_bits, linear, rounding, within
from conftest import announce
from g4attn import ops

pytestmark = pytest.mark.gpu


def make(dev, seed, tokens, rows, n):
    g = torch.Generator().manual_seed(seed)
    x, xs = in_8_bits(torch.randn(tokens, n, generator=g))
    w, ws = in_8_bits(torch.randn(rows, n, generator=g) * n ** -0.5)
    return [t.to(dev) for t in (x, xs, w, ws)]


def call(x, xs, w, ws, kind="f32", out=None, stream=None, spare=0):
    tokens, rows = x.shape[0], w.shape[0]
    if out is None:
        out = torch.full((tokens, rows), 7.0, dtype=TYPES[kind], device=x.device)
    space = torch.full((ops.linear_e4m3_workspace_bytes(tokens + spare, rows, x.shape[1]),), 0xff, dtype=torch.uint8, device=x.device)
    ops.linear_e4m3(x, xs, w, ws, out, space, stream=stream)
    torch.cuda.synchronize()
    return out


def check(dev, seed, tokens, rows, n, kind="f32"):
    announce(f"linearE4m3 {tokens} x {rows} x {n} {kind}")
    x, xs, w, ws = make(dev, seed, tokens, rows, n)
    got = call(x, xs, w, ws, kind)
    want, tol = linear(*(t.cpu().float() for t in (x, xs, w, ws)), kind)
    within(got.cpu(), want, tol + rounding(want, kind), "out")


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 31, 33, 48, 63, 64, 65, 127, 129, 200, 255, 257, 300])
def test_tokens(dev, tokens):
    check(dev, tokens, tokens, 200, 272)


@pytest.mark.parametrize("rows", [1, 3, 15, 16, 17, 63, 64, 65, 127, 129, 250, 256, 257, 511, 1000])
@pytest.mark.parametrize("tokens", [1, 37, 260])
def test_outputs(dev, rows, tokens):
    check(dev, rows, tokens, rows, 192)


@pytest.mark.parametrize("n", [16, 32, 48, 112, 128, 144, 240, 256, 272, 384, 400, 512, 640, 1008, 1536, 4096, 8208])
@pytest.mark.parametrize("tokens", [1, 20, 70, 300])
def test_inputs(dev, n, tokens):
    check(dev, n, tokens, 136, n)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,rows,n", [(1, 2560, 1536), (64, 1537, 1536), (513, 770, 640), (1030, 1290, 256)])
def test_types(dev, kind, tokens, rows, n):
    check(dev, 3, tokens, rows, n, kind)


@pytest.mark.parametrize("tokens,rows,n", [(5, 65536, 64), (3, 8, 65536), (1, 16, 65536), (4200, 24, 128), (2049, 4112, 144)])
def test_long_sides(dev, tokens, rows, n):
    check(dev, 4, tokens, rows, n)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,rows,n", [(4500, 4100, 64), (4352, 4352, 128), (4400, 4104, 336)])
def test_more_tiles_than_compute_units(dev, kind, tokens, rows, n):
    """Workgroups that go on from tile to tile, whole ones and cut ones, over one to six stages each."""
    check(dev, 5, tokens, rows, n, kind)


@pytest.mark.parametrize("tokens", [1, 30, 260])
@pytest.mark.parametrize("kind,offset,stride", [("f32", 0, 301), ("f32", 1, 304), ("f16", 4, 304), ("f16", 1, 303), ("bf16", 2, 308)])
def test_strided_rows(dev, tokens, kind, offset, stride):
    """Inputs and outputs whose tokens lie apart; what lies between the outputs stays as it was."""
    announce(f"linearE4m3 strided {tokens} {kind} {offset} {stride}")
    x, xs, w, ws = make(dev, 9, tokens, 300, 256)
    apart = torch.full((tokens, 320), 0x7F, dtype=torch.uint8, device=dev)
    apart[:, :256] = x.view(torch.uint8)
    flat = torch.full((offset + tokens * stride + 8,), 7.0, dtype=TYPES[kind], device=dev)
    out = flat[offset:offset + tokens * stride].view(tokens, stride)[:, :300]
    call(apart.view(TYPES["e4m3"])[:, :256], xs, w, ws, out=out)
    assert torch.equal(out, call(x, xs, w, ws, kind))
    flat[offset:offset + tokens * stride].view(tokens, stride)[:, :300] = 7.0
    assert (flat == 7.0).all()


@pytest.mark.parametrize("tokens,rows,stride", [(300, 4096, (1 << 24) - 16), (270, 40, 1 << 24), (20, 24, 1 << 28)])
def test_offsets_past_32_bits(dev, tokens, rows, stride):
    """Tokens that lie far apart: by tiles, and where a tile's offsets would not fit."""
    announce(f"linearE4m3 tokens {stride} bytes apart")
    x, xs, w, ws = make(dev, 13, tokens, rows, 64)
    flat = torch.empty((tokens - 1) * stride + 64, dtype=torch.uint8, device=dev)
    far = flat.as_strided((tokens, 64), (stride, 1))
    far.copy_(x.view(torch.uint8))
    got = call(far.view(TYPES["e4m3"]), xs, w, ws, "f16")
    want, tol = linear(*(t.cpu().float() for t in (x, xs, w, ws)), "f16")
    within(got.cpu(), want, tol + rounding(want, "f16"), "out")


@pytest.mark.parametrize("tokens", [3, 50, 300])
def test_rows_that_are_not_finite_stay_alone(dev, tokens):
    """A token of NaN codes or scale, and an output's weights: its row, its column, and nothing else. NaN behind a row's
    end is not read."""
    announce(f"linearE4m3 NaN {tokens}")
    x, xs, w, ws = make(dev, 10, tokens, 100, 208)
    want = call(x, xs, w, ws)
    x.view(torch.uint8)[1] = 0x7F
    xs[2] = float("nan")
    w.view(torch.uint8)[40, 7] = 0xFF
    got = call(x, xs, w, ws)
    assert got[1:3].isnan().all() and got[:, 40].isnan().all()
    keep_t, keep_o = torch.ones(tokens, dtype=torch.bool), torch.ones(100, dtype=torch.bool)
    keep_t[1:3], keep_o[40] = False, False
    assert torch.equal(got[keep_t][:, keep_o], want[keep_t][:, keep_o])


def test_zero_tokens_and_extremes(dev):
    announce("linearE4m3 zero tokens, extreme scales")
    x, xs, w, ws = make(dev, 11, 4, 32, 64)
    assert call(x[:0], xs[:0], w, ws).shape == (0, 32)
    for f in (2.0 ** 60, 2.0 ** -60):  # powers of two: exact
        assert torch.equal(call(x, xs * f, w, ws / f), call(x, xs, w, ws))


@pytest.mark.parametrize("tokens", [1, 16, 40, 100, 300, 700])
def test_the_same_call_gives_the_same_bits(dev, tokens):
    """Twice, on another stream, in a workspace of a larger batch, and replayed from a graph over new inputs."""
    announce(f"linearE4m3 repeated {tokens}")
    x, xs, w, ws = make(dev, 12, tokens, 530, 1040)
    want = call(x, xs, w, ws)
    assert torch.equal(call(x, xs, w, ws, spare=1000), want)
    s = torch.cuda.Stream()
    assert torch.equal(call(x, xs, w, ws, stream=s), want)
    out = torch.zeros_like(want)
    space = torch.empty(ops.linear_e4m3_workspace_bytes(tokens, 530, 1040), dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.linear_e4m3(x, xs, w, ws, out, space)
    for i in range(3):
        x2, xs2, _, _ = make(dev, 20 + i, tokens, 530, 1040)
        x.copy_(x2)
        xs.copy_(xs2)
        space.fill_(0xff)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(x, xs, w, ws))
