"""g4_add_rms_norm and g4_quantize_rows against the definition in 64 bits: lengths from one element to the longest, types,
strides and alignment, both norms, rows of zeros, tiny, huge and non-finite rows, in-place sums, other streams, graphs."""
import pytest
import torch

from batch_rows import E, TYPES, rounding, unit, within
from conftest import announce
from g4attn import ops

pytestmark = pytest.mark.gpu

# Of a norm: at most 32 products a thread and then 16 partial sums in turn, all of one sign (48 half-steps, halved by the
# root), the mean, eps, root and quotient, two products.
NORM = 32 * E


def make(dev, seed, rows, n, x="f32", res=None, post=False, weight="f16"):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    d = dict(x=r(rows, n).to(TYPES[x]).to(dev))
    d["residual"] = (r(rows, n) * 3).to(TYPES[res]).to(dev) if res else None
    d["weight"] = (1 + 0.2 * r(n)).to(TYPES[weight]).to(dev) if weight else None
    d["post"] = (1 + 0.2 * r(n)).to(TYPES[weight or "f16"]).to(dev) if post else None
    return d


def codes_within(codes, scales, y, slack, what):
    """e4m3 codes of y with a scale a row: each the nearest (half the spacing at its value), the scale max |y| / 448."""
    y, codes, scales = y.double(), codes.cpu().double(), scales.cpu().double()
    want = y.abs().amax(-1).clamp(min=2.0 ** -100) / 448
    within(scales, want, want * (slack + 2 * E), what + " scale")
    v = (y / want[:, None]).abs()
    step = torch.exp2(torch.floor(torch.log2(v.clamp(min=2.0 ** -6))) - 3)
    # A value near a border of two binades may round with the upper one's spacing.
    near = torch.exp2(torch.floor(torch.log2((v * (1 + 4 * slack + 8 * E)).clamp(min=2.0 ** -6))) - 3)
    within(codes, y / want[:, None], torch.maximum(step, near) / 2 + v * 2 * (slack + 4 * E), what + " codes")


def check(d, out_type, eps=1e-6, keep=True, stream=None, like=lambda t: t):
    """like: the outputs as rows that lie apart."""
    x, res = d["x"], d["residual"]
    rows, n = x.shape
    dev = x.device
    out = like(torch.full((rows, n), 7.0, device=dev).to(TYPES[out_type]))
    scales = torch.full((rows,), 7.0, device=dev) if out_type == "e4m3" else None
    kind = next(k for k, t in TYPES.items() if t == (res if res is not None else x).dtype)
    total = like(torch.full((rows, n), 7.0, device=dev).to(TYPES[kind])) if keep else None
    ops.add_rms_norm(x, d["weight"], out, scales=scales, residual=res, residual_out=total, post_weight=d["post"], eps=eps,
                     stream=stream)
    torch.cuda.synchronize()
    b = x.cpu().double()
    off = torch.zeros_like(b)
    if d["post"] is not None:
        b = unit(b, eps) * d["post"].cpu().double()
        off = b.abs() * NORM
    r = b if res is None else res.cpu().double() + b
    if total is not None:
        within(total.cpu(), r, off + r.abs() * E + rounding(r, kind), "sum")
        r, off = total.cpu().double(), torch.zeros_like(b)  # what is normed is what is kept
    w = 1.0 if d["weight"] is None else d["weight"].cpu().double()
    y = unit(r, eps) * w
    slack = NORM if keep or (res is None and d["post"] is None) else None
    if slack is None:  # the sum was rounded to f32 only: its own error comes through both norms
        assert kind == "f32"
        slack = 3 * NORM
        off = (b.abs() * NORM + r.abs() * E) * 2 / torch.sqrt(r.square().mean(-1, keepdim=True) + eps) * torch.as_tensor(w).abs()
    if out_type == "e4m3":
        codes_within(out, scales, y, slack, "e4m3")
    else:
        within(out.cpu(), y, y.abs() * slack + off + rounding(y, out_type), "out")
    return out, scales, total


@pytest.mark.parametrize("n", [1, 2, 7, 8, 63, 64, 65, 512, 520, 1000, 1536, 2048, 2049, 2056, 4096, 4100, 8192, 8200, 16384, 16392,
                               32760, 32768])
@pytest.mark.parametrize("out_type", ["f32", "e4m3"])
def test_lengths(dev, n, out_type):
    announce(f"addRmsNorm n={n} {out_type}")
    check(make(dev, n, 3, n, "f32", "f32", post=True), out_type)


@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("res", [None, "f32", "f16", "bf16"])
@pytest.mark.parametrize("out_type", ["f32", "f16", "bf16", "e4m3"])
def test_types(dev, x, res, out_type):
    announce(f"addRmsNorm {x} + {res} -> {out_type}")
    check(make(dev, 5, 9, 1544, x, res, post=res is not None, weight="bf16" if x == "bf16" else "f16"), out_type)
    check(make(dev, 6, 2, 77, x, res, weight="f32" if res else None), out_type)


@pytest.mark.parametrize("rows", [1, 4, 5, 2047, 2048, 2051])
@pytest.mark.parametrize("n", [96, 520, 1100, 1536])
def test_rows(dev, rows, n):
    """Around the line between a wave a row and a workgroup a row."""
    announce(f"addRmsNorm rows={rows} n={n}")
    check(make(dev, rows + n, rows, n, "bf16", "f32", post=True), "e4m3")


def test_without_keeping_the_sum(dev):
    announce("addRmsNorm without residual_out")
    check(make(dev, 8, 6, 1536, "f32", "f32", post=True), "f32", keep=False)
    check(make(dev, 9, 6, 1536, "f16"), "e4m3", keep=False)


@pytest.mark.parametrize("offset,stride", [(0, 1601), (1, 1600), (8, 1608), (4, 1604), (3, 1599)])
@pytest.mark.parametrize("x,out_type", [("f32", "e4m3"), ("bf16", "bf16"), ("f16", "e4m3")])
def test_strided_and_misaligned_rows(dev, offset, stride, x, out_type):
    announce(f"addRmsNorm {x} offset={offset} stride={stride}")
    d = make(dev, stride, 5, 1536, x, x, post=True)

    def apart(t):
        bits = t.view(torch.uint8) if t.dtype == TYPES["e4m3"] else t
        flat = torch.zeros(offset + 5 * stride + 16, dtype=bits.dtype, device=dev)
        v = flat[offset:offset + 5 * stride].view(5, stride)[:, :1536]
        v.copy_(bits)
        return v.view(t.dtype)

    d["x"], d["residual"] = apart(d["x"]), apart(d["residual"])
    check(d, out_type, like=apart)


def test_sum_in_place_and_addition_alone(dev):
    d = make(dev, 11, 40, 1536, "f32", "f32", post=True)
    announce("addRmsNorm in place")
    want, ws, total = check(d, "e4m3")
    out, scales = torch.empty_like(want), torch.empty_like(ws)
    r = d["residual"].clone()
    ops.add_rms_norm(d["x"], d["weight"], out, scales=scales, residual=r, residual_out=r, post_weight=d["post"])
    assert torch.equal(r, total) and torch.equal(scales, ws) and torch.equal(out.view(torch.uint8), want.view(torch.uint8))
    r = d["residual"].clone()
    ops.add_rms_norm(d["x"], None, None, residual=r, residual_out=r, post_weight=d["post"])
    assert torch.equal(r, total)
    x = d["x"].clone()
    ops.add_rms_norm(x, d["weight"], x)
    y = unit(d["x"].cpu().double(), 1e-6) * d["weight"].cpu().double()
    within(x.cpu(), y, y.abs() * NORM + rounding(y, "f32"), "out over x")


@pytest.mark.parametrize("n", [24, 1536, 5000])
def test_rows_without_a_scale(dev, n):
    """Zeros, rows below the least scale, the largest values, Inf and NaN; the rows beside them are as always."""
    announce(f"odd rows n={n}")
    x = torch.randn(8, n, generator=torch.Generator().manual_seed(n))
    x[1] = 0
    x[2] *= 1e-36
    x[3] *= 1e30
    x[4, n // 2] = float("inf")
    x[5, n - 1] = float("nan")
    x[6] = 0
    x[6, 3] = -2.5
    x = x.to(dev)
    out, scales = torch.zeros(8, n, device=dev).to(TYPES["e4m3"]), torch.full((8,), 7.0, device=dev)
    ops.quantize_rows(x, out, scales)
    torch.cuda.synchronize()
    bad = [4, 5]
    fine = [0, 1, 2, 3, 6, 7]
    assert scales[bad].isnan().all() and out.float()[bad].isnan().all()
    codes_within(out.view(torch.uint8)[fine].view(TYPES["e4m3"]), scales[fine], x[fine].cpu(), 0.0, "quantize")
    assert (out.float()[[1, 2]].abs() < 1).all() and (out.float()[1] == 0).all()
    total = torch.empty_like(x)
    ops.add_rms_norm(x, None, out, scales=scales, residual=torch.zeros_like(x), residual_out=total)
    torch.cuda.synchronize()
    assert scales[bad].isnan().all() and out.float()[bad].isnan().all() and (out.float()[1] == 0).all()
    rest = [0, 1, 2, 6, 7]
    codes_within(out.view(torch.uint8)[rest].view(TYPES["e4m3"]), scales[rest], unit(x[rest].cpu().double(), 1e-6), NORM, "norm")


@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n", [(1, 16), (3, 2048), (2500, 256), (700, 4099)])
def test_quantize(dev, x, rows, n):
    announce(f"quantizeRows {x} {rows}x{n}")
    v = torch.randn(rows, n, generator=torch.Generator().manual_seed(rows)).to(TYPES[x]).to(dev)
    out, scales = torch.zeros(rows, n, device=dev).to(TYPES["e4m3"]), torch.zeros(rows, device=dev)
    ops.quantize_rows(v, out, scales)
    codes_within(out, scales, v.cpu(), 0.0, "quantize")


def test_every_code_and_border(dev):
    """Values on and beside the borders between codes, with a largest of 448: ties to even, subnormal codes."""
    codes = torch.arange(127, dtype=torch.uint8).view(TYPES["e4m3"]).float()
    mid = (codes[1:] + codes[:-1]) / 2
    row = torch.cat([codes, mid, torch.nextafter(mid, mid * 0), torch.nextafter(mid, mid * 2), torch.tensor([448.0])])
    x = torch.stack([row, -row]).to(dev)
    out, scales = torch.zeros_like(x).to(TYPES["e4m3"]), torch.zeros(2, device=dev)
    announce("quantizeRows borders")
    ops.quantize_rows(x, out, scales)
    assert (scales == 1).all()
    assert torch.equal(out.cpu().float(), x.cpu().to(TYPES["e4m3"]).float())


def test_another_stream_and_a_graph(dev):
    d = make(dev, 21, 33, 1536, "f32", "f32", post=True)
    announce("addRmsNorm stream and graph")
    want, ws, total = check(d, "e4m3")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        check(d, "e4m3")
    check(d, "e4m3", stream=s)
    out, scales, sums = torch.zeros_like(want), torch.zeros_like(ws), torch.zeros_like(total)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.add_rms_norm(d["x"], d["weight"], out, scales=scales, residual=d["residual"], residual_out=sums, post_weight=d["post"])
    for i in range(3):
        d["x"].mul_(-1.5)
        d["residual"].add_(1)
        graph.replay()
        torch.cuda.synchronize()
        eager = check(d, "e4m3")
        assert torch.equal(eager[0].view(torch.uint8), out.view(torch.uint8)) and torch.equal(eager[1], scales)
        assert torch.equal(eager[2], sums)
