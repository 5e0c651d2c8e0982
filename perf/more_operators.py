"""The operators between two attention blocks of a served batch, measured one call at a time.

A case is a dict of plain values; its "op" names the operator:

  norm      residual addition and RMS norm of a batch's rows, in 8 bits with a scale a row, or in 16 (ops.add_rms_norm)
  quantize  rows in 8 bits with a scale a row (ops.quantize_rows)
  linear    projection of 8-bit rows by 8-bit weights (ops.linear_e4m3), with its requests' low-rank adapters where
            the case has some
  lora      the adapters beside a projection made elsewhere (ops.lora_add)

Where `own` is false, run() computes them in plain torch operations, in 32 bits, rounded once at the end.

The operators' definitions, as far as a reader needs them to see what the plain forms do:

* norm: b = x, or x normed and weighted by post_weight; r = residual + b, rounded to the residual's type and returned;
  y = r / sqrt(mean r^2 + eps) * weight.
* 8 bits: scale[t] = max |y[t]| / 448, the row is e4m3(y[t] / scale[t]).
* linear: out[t][o] = x_scales[t] * weight_scales[o] * sum_k x[t][k] weight[o][k].
* adapters: token t has adapter a = ids[t] (below 0: none); its down rows A[a] are [segments * rank][n], its up rows B[a]
  [outputs][rank]; output o belongs to segment s (q, k or v of a fused projection):
  out[t][o] += scales[a] * sum_j (sum_k x[t][k] A[a][s * rank + j][k]) B[a][o][j].

Inputs: branch outputs N(0, 1), residuals N(0, 3^2) with a few large channels as trained models have them, norm weights
near 1, projection weights N(0, 1 / n), adapters that change an output by about a tenth. Requests are runs of tokens;
every value and every request's adapter from the seed.
"""
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-6
E4M3 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": E4M3}
WIDTH = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}


def _ops():
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "gemma4-webgpu_amd"))
    from g4attn import ops

    return ops


# ---- the cases -----------------------------------------------------------------------

def listed():
    return [
        # One token of one chat between two blocks: the branch normed, added, normed again for the next projection.
        dict(name="norm_1", op="norm", tokens=1, n=1536, kind="f32", res="f32", post=True, out="e4m3"),
        # A decode batch of 64 in a 16-bit program.
        dict(name="norm_64", op="norm", tokens=64, n=2560, kind="bf16", res="bf16", post=False, out="bf16"),
        # Prompts' chunks: 4096 tokens, f32 residual stream.
        dict(name="norm_prompt", op="norm", tokens=4096, n=1536, kind="f32", res="f32", post=True, out="e4m3"),
        # A larger model's prompts in 16 bits, an odd number of tokens.
        dict(name="norm_wide", op="norm", tokens=8191, n=5376, kind="bf16", res="bf16", post=False, out="e4m3"),
        # The attention's outputs of 4000 tokens, before the output projection.
        dict(name="quantize_attn", op="quantize", tokens=4000, n=2048, kind="f32"),
        # One token's fused q, k, v projection.
        dict(name="linear_1", op="linear", tokens=1, rows=2560, n=1536, out="f32", adapters=0),
        # A decode batch's gate and up projection.
        dict(name="linear_64", op="linear", tokens=64, rows=12288, n=1536, out="f16", adapters=0),
        # The same of prompts' chunks.
        dict(name="linear_prompt", op="linear", tokens=4096, rows=12288, n=1536, out="f16", adapters=0),
        # A larger model's projection of prompts.
        dict(name="linear_large", op="linear", tokens=8192, rows=8192, n=8192, out="bf16", adapters=0),
        # One token's q, k, v adapters beside its projection by the f16 path.
        dict(name="lora_1", op="lora", tokens=1, runs=1, widths="2048+256+256", n=1536, kind="f32", out="f32", adapters=4,
             rank=16),
        # A decode batch of 64 requests with 40 adapters: q, k, v and the shared projection in one call.
        dict(name="lora_64", op="linear", tokens=64, runs=64, widths="2048+256+256", rows=2560, n=1536, out="f32",
             adapters=40, rank=16),
        # Four prompts with an adapter each: the output projection.
        dict(name="lora_prompts", op="linear", tokens=4003, runs=4, widths="1536", rows=1536, n=2048, out="f32", adapters=6,
             rank=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _widths(c):
    return tuple(int(w) for w in c["widths"].split("+"))


def _rows(c):
    return sum(_widths(c)) if "widths" in c else c["rows"]


def draw(rng):
    op = rng.choice(["norm", "norm", "quantize", "linear", "linear", "linear", "linear", "lora", "lora"])
    if op in ("norm", "quantize"):
        n = rng.choice([_log_int(rng, 64, 8192), 8 * _log_int(rng, 16, 1024)])
        tokens = _log_int(rng, 1, min(8192, 8191 * 5376 // n))
        kind = rng.choice(["f32", "f32", "f16", "bf16"])
        if op == "quantize":
            return dict(op=op, tokens=tokens, n=n, kind=kind)
        return dict(op=op, tokens=tokens, n=n, kind=kind, res=rng.choice([kind, "f32"]), post=rng.random() < 0.5,
                    out=rng.choice(["e4m3", "e4m3", "f32", "f16", "bf16"]))
    tokens = rng.choice([_log_int(rng, 1, 128), _log_int(rng, 1, 4096)])
    n = 16 * _log_int(rng, 16, 512)
    heads = rng.choice(["2048+256+256", "1024+512+512", "1000+24"])
    widths = heads if rng.random() < 0.5 else str(8 * _log_int(rng, 8, 1500))
    low = dict(runs=_log_int(rng, 1, min(64, tokens)), widths=widths, adapters=_log_int(rng, 1, 50),
               rank=8 * _log_int(rng, 1, 10))
    if op == "lora":
        return dict(op=op, tokens=tokens, n=n, kind=rng.choice(["f32", "f16", "bf16"]),
                    out=rng.choice(["f32", "f16", "bf16"]), **low)
    out = rng.choice(["f32", "f16", "bf16"])
    if rng.random() < 0.4:
        return dict(op=op, tokens=tokens, rows=_rows(low), n=n, out=out, **low)
    return dict(op=op, tokens=tokens, rows=_log_int(rng, 64, 16384), n=n, out=out, adapters=0)


# ---- inputs --------------------------------------------------------------------------

def _in_8_bits(x):
    """Rows as e4m3 with their scales: weights laid out once, activations as the norm leaves them."""
    scale = x.float().abs().amax(-1) / 448
    return (x.float() / scale[:, None]).to(E4M3), scale


def prepare(case, seed):
    c = case
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(1_000_003 * seed + 31)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=dev)  # noqa: E731
    st, T, n = dict(c=c), c["tokens"], c["n"]
    if c["op"] in ("norm", "quantize"):
        st["x"] = normal(T, n).to(TYPES[c["kind"]])
        st["weight"] = st["post"] = None
        if c["op"] == "norm":
            loud = torch.ones(n, device=dev)
            loud[torch.randint(n, (max(1, n // 500),), generator=gen, device=dev)] = 20
            st["residual"] = (normal(T, n) * 3 * loud).to(TYPES[c["res"]])
            st["weight"] = (1 + 0.1 * normal(n)).half()
            st["post"] = (1 + 0.1 * normal(n)).half() if c["post"] else None
        if own:
            st["ops"] = _ops()
            st["out"] = torch.empty(T, n, dtype=TYPES[c.get("out", "e4m3")], device=dev)
            st["scales"] = torch.empty(T, device=dev) if c.get("out", "e4m3") == "e4m3" else None
            st["sum"] = torch.empty_like(st["residual"]) if c["op"] == "norm" else None
        return st
    rows = _rows(c)
    st["ids"] = None
    if c["op"] == "linear":
        st["x"], st["xs"] = _in_8_bits(normal(T, n))
        st["w"], st["ws"] = _in_8_bits(normal(rows, n) * n ** -0.5)
    else:
        st["x"], st["xs"] = normal(T, n).to(TYPES[c["kind"]]), None
        st["base"] = normal(T, rows).to(TYPES[c["out"]])
    kind = torch.bfloat16 if c.get("kind") == "bf16" else torch.float16
    if c["adapters"]:
        L, r = c["adapters"], c["rank"]
        st["a"] = (normal(L, len(_widths(c)) * r, n) * n ** -0.5).to(kind)
        st["b"] = (normal(L, rows, r) * 0.1).to(kind)
        st["alpha"] = 0.5 + torch.rand(L, generator=gen, device=dev)
        # Each request's adapter, one of nine without.
        of_run = torch.randint(L, (c["runs"],), generator=gen, device=dev, dtype=torch.int32)
        of_run[4::9] = -1
        st["ids"] = of_run[torch.arange(T, device=dev) * c["runs"] // T].contiguous()
    if own:
        ops = st["ops"] = _ops()
        st["out"] = torch.empty(T, rows, dtype=TYPES[c["out"]], device=dev)
        st["low"] = ops.LoraAdapters(st["a"], st["b"], st["alpha"], _widths(c)) if c["adapters"] else None
        size = (ops.linear_e4m3_workspace_bytes(T, rows, n, st["low"]) if c["op"] == "linear" else
                ops.lora_workspace_bytes(st["low"], T))
        st["ws_buf"] = torch.empty(size, dtype=torch.uint8, device=dev)
    return st


# ---- the plain forms -----------------------------------------------------------------

def _plain_rows(st):
    c = st["c"]
    y = st["x"].float()
    if c["op"] == "norm":
        if st["post"] is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * st["post"].float()
        total = (st["residual"].float() + y).to(st["residual"].dtype)
        y = total.float()
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * st["weight"].float()
        if c["out"] != "e4m3":
            return y.to(TYPES[c["out"]]), total
    scale = y.abs().amax(-1) / 448
    y = (y / scale[:, None]).to(E4M3)
    return (y, scale, total) if c["op"] == "norm" else (y, scale)


def _plain_low(st, x):
    """Every adapter's down products at once, those of other tokens' adapters taken out, then every up product."""
    c = st["c"]
    L, r, S = c["adapters"], c["rank"], len(_widths(c))
    u = (x @ st["a"].float().view(L * S * r, -1).T).view(-1, L, S, r)
    mine = st["ids"][:, None] == torch.arange(L, device=x.device)[None, :]
    u = u * (mine * st["alpha"][None, :])[:, :, None, None]
    up = torch.split(st["b"].float(), list(_widths(c)), dim=1)
    return torch.cat([u[:, :, s].reshape(-1, L * r) @ b.transpose(1, 2).reshape(L * r, -1) for s, b in enumerate(up)], 1)


def _plain_products(st):
    c = st["c"]
    if c["op"] == "lora":
        return (st["base"].float() + _plain_low(st, st["x"].float())).to(st["base"].dtype)
    x = st["x"].float() * st["xs"][:, None]
    y = x @ (st["w"].float() * st["ws"][:, None]).T
    if c["adapters"]:
        y = y + _plain_low(st, x)
    return y.to(TYPES[c["out"]])


def run(state):
    st, c = state, state["c"]
    if not own:
        return _plain_rows(st) if c["op"] in ("norm", "quantize") else _plain_products(st)
    ops = st["ops"]
    if c["op"] == "quantize":
        ops.quantize_rows(st["x"], st["out"], st["scales"])
        return st["out"], st["scales"]
    if c["op"] == "norm":
        ops.add_rms_norm(st["x"], st["weight"], st["out"], scales=st["scales"], residual=st["residual"],
                         residual_out=st["sum"], post_weight=st["post"], eps=EPS)
        return (st["out"], st["sum"]) if st["scales"] is None else (st["out"], st["scales"], st["sum"])
    if c["op"] == "lora":
        ops.lora_add(st["low"], st["ids"], st["x"], st["base"], st["out"], st["ws_buf"])
    else:
        ops.linear_e4m3(st["x"], st["xs"], st["w"], st["ws"], st["out"], st["ws_buf"], lora=st["low"], adapter_ids=st["ids"])
    return st["out"]


# ---- what a pass cannot do without ----------------------------------------------------

def work(case):
    c = case
    T, n = c["tokens"], c["n"]
    if c["op"] == "quantize":
        return {"bytes": T * n * (WIDTH[c["kind"]] + 1) + 4 * T, "flops": 3 * T * n}
    if c["op"] == "norm":
        return {"bytes": T * n * (WIDTH[c["kind"]] + 2 * WIDTH[c["res"]] + WIDTH[c["out"]]) + n * (4 if c["post"] else 2),
                "flops": (12 if c["post"] else 8) * T * n}
    rows = _rows(c)
    need, flops = 0, 0
    if c["op"] == "linear":
        need, flops = T * n + rows * n + 4 * (T + rows) + T * rows * WIDTH[c["out"]], 2 * T * rows * n
    else:
        need = T * n * WIDTH[c["kind"]] + 2 * T * rows * WIDTH[c["out"]]
    if c["adapters"]:
        # The adapters that so many requests, each with one at random, have between them.
        live = c["adapters"] * (1 - (1 - 1 / c["adapters"]) ** (c["runs"] * 8 / 9))
        down = len(_widths(c)) * c["rank"]
        need += live * 2 * (down * n + rows * c["rank"]) + 4 * T
        flops += 2 * T * (down * n + rows * c["rank"])
    return {"bytes": int(need), "flops": int(flops)}


# ---- the definitions in 64 bits --------------------------------------------------------

def exact(case, seed):
    c = case
    st = prepare(case, seed)
    x = st["x"].double()
    if c["op"] in ("norm", "quantize"):
        unit = lambda v: v * (v.square().sum(-1, keepdim=True) / c["n"] + EPS).rsqrt()  # noqa: E731
        y, rest = x, ()
        if c["op"] == "norm":
            b = x if st["post"] is None else unit(x) * st["post"].double()
            total = st["residual"].double() + b
            y = unit(total.to(st["residual"].dtype).double()) * st["weight"].double()
            if c["out"] != "e4m3":
                return y, total
            rest = (total,)
        scale = torch.linalg.vector_norm(y, ord=float("inf"), dim=-1) / 448
        return (y / scale[:, None], scale) + rest
    if c["op"] == "linear":
        x = x * st["xs"].double()[:, None]
        out = (x @ st["w"].double().T) * st["ws"].double()[None, :]
    else:
        out = st["base"].double()
    if c["adapters"]:
        r = c["rank"]
        for a in range(c["adapters"]):
            at = torch.nonzero(st["ids"] == a)[:, 0]
            if at.numel():
                u = (st["a"][a].double() @ x[at].T).T * st["alpha"][a].double()
                o = 0
                for s, w in enumerate(_widths(c)):
                    out[at, o:o + w] += u[:, s * r:(s + 1) * r] @ st["b"][a, o:o + w].double().T
                    o += w
    return out
