"""Definitions in 64 bits of the operators between two attention blocks, and what their results may be off by: shared by
test_gpu_rownorm.py, test_gpu_linear8.py, test_gpu_lora.py and test_gpu_block.py."""
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative
LEAST = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half a step among subnormals
E = 2.0 ** -24


def rounding(want, kind):
    return want.abs() * HALF[kind] + LEAST[kind]


def within(got, want, tol, what):
    """got (of any type) is off by at most tol, element by element; both on the CPU."""
    off = (got.double() - want).abs()
    assert off.shape == tol.shape and got.shape == want.shape
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {(off / tol)[bad].max():.3g} of the tolerance"


def in_8_bits(x):
    """Rows as e4m3 codes with their scales (made here, apart from the kernel)."""
    scale = (x.float().abs().amax(-1) / 448).clamp(min=1e-30)
    return (x.float() / scale[:, None]).to(torch.float8_e4m3fn), scale


def unit(x, eps):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)


def linear(x, xs, w, ws, kind="f32"):
    """(sums with their scales, what they may be off by before the output's rounding). A sum of k products in f32: the
    matrix units add 16 or more products at a time to a sum, whose every rounding is at most half a step of a partial sum,
    itself at most the sum of the magnitudes; then partial sums of pieces of k are joined; two scales. 16-bit outputs may come
    from the 8-bit unit, which keeps 13 bits below a group's largest product: 2^-12.3 of it was the worst of 15000 random
    sums of 128, four times that is allowed for each 128."""
    x, w = x.double(), w.double()
    scale = xs.double()[:, None] * ws.double()[None, :]
    y, size = (x @ w.T) * scale, (x.abs() @ w.abs().T) * scale.abs()
    tol = size * (x.shape[1] / 16 + 32) * E + y.abs() * 3 * E
    if kind != "f32":
        most = (x.abs().amax(-1)[:, None] * w.abs().amax(-1)[None, :]) * scale.abs()
        tol = tol + most * 2.0 ** -10.3 * -(-x.shape[1] // 128)
    return y, tol


def lora(ids, x, a, b, alpha, widths):
    """(the adapters' part, what it may be off by): the down sums as linear's, then each as parts that leave 2^-23 of it or
    2^-39 of the token's largest, and sums of rank products."""
    L, r = a.shape[0], b.shape[2]
    out = torch.zeros(x.shape[0], b.shape[1], dtype=torch.float64)
    tol = torch.zeros_like(out)
    for ad in range(L):
        at = torch.nonzero(ids == ad)[:, 0]
        if not at.numel():
            continue
        xa, A, al = x[at].double(), a[ad].double(), 1.0 if alpha is None else float(alpha[ad])
        u = xa @ A.T
        u_off = (xa.abs() @ A.abs().T) * (x.shape[1] / 16 + 40) * E
        o = 0
        for s, w in enumerate(widths):
            B = b[ad, o:o + w].double()
            us, uo = u[:, s * r:(s + 1) * r], u_off[:, s * r:(s + 1) * r]
            out[at, o:o + w] = al * (us @ B.T)
            off = (uo + us.abs() * (2.0 ** -23 + (r / 8 + 8) * E) + 2.0 ** -38 * us.abs().amax(-1, keepdim=True)) @ B.abs().T
            tol[at, o:o + w] = abs(al) * off * 1.001 + out[at, o:o + w].abs() * 2 * E
            o += w
    return out, tol
