"""A block of a served batch: residual norms in 8 bits, the fused projection with its requests' adapters, rows appended to the
paged cache, attention, 8-bit rows, the output projection and its adapters, the next norm. Every step is checked against the
definition in 64 bits on what the step before left; the whole as one captured graph; and through the TypeScript host (node
host/run.js block), whose calls give the same bits."""
import json
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from batch_rows import E, linear, lora, rounding, unit, within
from conftest import announce
from g4attn import ops
from paged_helpers import EPS, Paged
from test_gpu_rownorm import NORM, codes_within

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent
RUN = ROOT / "gemma4-webgpu_amd" / "host" / "run.js"
NODE = shutil.which("node")
E4M3 = torch.float8_e4m3fn


class Block:
    def __init__(self, dev, seed, ctx, new, hidden=384, nqh=4, hd=256, rank=16, adapters=3, pad=1):
        self.p = p = Paged(dev, seed, ctx, new, hd=hd, nqh=nqh, page=16, pad=pad)
        p.upload()
        self.n, self.hidden, self.nqh, self.hd, self.rank, self.adapters = p.tokens, hidden, nqh, hd, rank, adapters
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        n, width, inner = self.n, (nqh + 2) * hd, nqh * hd
        self.host = dict(
            branch=r(n, hidden), residual=r(n, hidden) * 3, post=(1 + 0.1 * r(hidden)).half(), pre=(1 + 0.1 * r(hidden)).half(),
            next=(1 + 0.1 * r(hidden)).half(), wqkv=r(width, hidden) * hidden ** -0.5, wo=r(hidden, inner) * inner ** -0.5,
            a1=(r(adapters, 3 * rank, hidden) * hidden ** -0.5).half(), b1=(r(adapters, width, rank) * 0.3).half(),
            a2=(r(adapters, rank, inner) * inner ** -0.5).half(), b2=(r(adapters, hidden, rank) * 0.3).half(),
            alpha=0.5 + torch.rand(adapters, generator=g), qw=(1 + 0.1 * r(hd)).half(), kw=((1 + 0.1 * r(hd)) / 8).half(),
            ids=torch.randint(-1, adapters, (n,), generator=g, dtype=torch.int32))
        self.d = d = {k: v.to(dev) for k, v in self.host.items()}
        self.inv = ops.rope_inv_freq(1e4, hd, False, None)
        new_t = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=dev)  # noqa: E731
        d.update(rows8=new_t(n, hidden).to(E4M3), scales=new_t(n), mid=new_t(n, hidden), w8=new_t(width, hidden).to(E4M3),
                 ws8=new_t(width), qkv=new_t(n, width), q=new_t(n, nqh, hd, dtype=torch.float16), attn=new_t(n, nqh, hd),
                 o8=new_t(n, inner).to(E4M3), os8=new_t(n), wo8=new_t(hidden, inner).to(E4M3), wos8=new_t(hidden),
                 y=new_t(n, hidden), z=new_t(n, hidden), sum=new_t(n, hidden), next8=new_t(n, hidden).to(E4M3), next_s=new_t(n))
        self.lora1 = ops.LoraAdapters(d["a1"], d["b1"], None, (inner, hd, hd))
        self.lora2 = ops.LoraAdapters(d["a2"], d["b2"], d["alpha"])
        u8 = lambda size: torch.empty(size, dtype=torch.uint8, device=dev)  # noqa: E731
        self.ws = [u8(ops.linear_e4m3_workspace_bytes(n, width, hidden, self.lora1)),
                   u8(ops.paged_attn_workspace_bytes(p.cache, p.batch, nqh)),
                   u8(ops.linear_e4m3_workspace_bytes(n, hidden, inner)), u8(ops.lora_workspace_bytes(self.lora2, n))]
        ops.quantize_rows(d["wqkv"], d["w8"], d["ws8"])  # the weights, once
        ops.quantize_rows(d["wo"], d["wo8"], d["wos8"])

    def run(self):
        d, p, nqh = self.d, self.p, self.nqh
        ops.add_rms_norm(d["branch"], d["pre"], d["rows8"], scales=d["scales"], residual=d["residual"], residual_out=d["mid"],
                         post_weight=d["post"])
        ops.linear_e4m3(d["rows8"], d["scales"], d["w8"], d["ws8"], d["qkv"], self.ws[0], lora=self.lora1, adapter_ids=d["ids"])
        qkv = d["qkv"].view(self.n, nqh + 2, self.hd)
        ops.paged_append(p.cache, p.batch, qkv[:, :nqh], qkv[:, nqh:nqh + 1], qkv[:, nqh + 1:], d["qw"], d["kw"], self.inv, d["q"],
                         eps=EPS)
        ops.paged_attn(p.cache, p.batch, d["q"], d["attn"], self.ws[1])
        ops.quantize_rows(d["attn"].view(self.n, -1), d["o8"], d["os8"])
        ops.linear_e4m3(d["o8"], d["os8"], d["wo8"], d["wos8"], d["y"], self.ws[2])
        ops.lora_add(self.lora2, d["ids"], d["o8"], d["y"], d["z"], self.ws[3], x_scales=d["os8"])
        ops.add_rms_norm(d["z"], d["next"], d["next8"], scales=d["next_s"], residual=d["mid"], residual_out=d["sum"])


STEPS = ("rows8", "scales", "mid", "qkv", "q", "attn", "o8", "os8", "y", "z", "sum", "next8", "next_s")


def bits(t):
    return t.detach().cpu().contiguous().view(torch.uint8).numpy().tobytes()


@pytest.mark.parametrize("ctx,new,pad", [([5, 0, 40], [1, 1, 1], 1), ([33, 0, 7], [20, 9, 70], 2), ([0], [300], 0)])
def test_every_step_by_its_definition(dev, ctx, new, pad):
    announce(f"block ctx={ctx} new={new}")
    b = Block(dev, 50 + len(new), ctx, new, pad=pad)
    b.run()
    torch.cuda.synchronize()
    c = {k: v.cpu() for k, v in b.d.items()}
    f = lambda k: c[k].double()  # noqa: E731
    branch = unit(f("branch"), 1e-6) * f("post")
    want = f("residual") + branch
    within(c["mid"], want, branch.abs() * NORM + want.abs() * 2 * E, "sum")
    codes_within(b.d["rows8"], b.d["scales"], unit(f("mid"), 1e-6) * f("pre"), NORM, "normed rows")
    codes_within(b.d["w8"], b.d["ws8"], f("wqkv"), 0.0, "weights")
    x = c["rows8"].double() * f("scales")[:, None]
    y, off = linear(c["rows8"].float(), c["scales"], c["w8"].float(), c["ws8"])
    part, tol = lora(c["ids"], x, c["a1"], c["b1"], None, b.lora1.widths)
    within(c["qkv"], y + part, off + tol + (y.abs() + part.abs()) * 4 * E + rounding(y + part, "f32"), "qkv")
    b.p.q = c["q"].numpy()  # the attention by its definition over what was appended
    b.p.k, b.p.v = b.p.d_k.cpu(), b.p.d_v.cpu()
    live = int(b.p.start[-1])
    want, bound = b.p.expected()
    err = np.abs(c["attn"].numpy()[:live] - want[:live]).max(axis=(1, 2))
    assert (err <= bound[:live]).all()
    codes_within(b.d["o8"], b.d["os8"], f("attn").view(b.n, -1), 0.0, "attention rows")
    y, off = linear(c["o8"].float(), c["os8"], c["wo8"].float(), c["wos8"])
    within(c["y"], y, off + rounding(y, "f32"), "output projection")
    part, tol = lora(c["ids"], c["o8"].double() * f("os8")[:, None], c["a2"], c["b2"], c["alpha"], b.lora2.widths)
    want = f("y") + part
    within(c["z"], want, tol + (want.abs() + part.abs()) * 4 * E + rounding(want, "f32"), "with adapters")
    want = f("mid") + f("z")
    within(c["sum"], want, want.abs() * 2 * E, "next sum")
    codes_within(b.d["next8"], b.d["next_s"], unit(f("sum"), 1e-6) * f("next"), NORM, "next rows")


def test_one_graph_of_the_block(dev):
    """Captured once, replayed with other inputs, lengths and adapters: as the same calls one by one."""
    announce("block graph")
    b = Block(dev, 60, [9, 30], [1, 1])
    b.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run()
    g = torch.Generator(device=dev).manual_seed(1)
    for i in range(3):
        b.d["branch"].normal_(generator=g)
        b.d["residual"].normal_(generator=g)
        b.d["ids"].random_(-1, b.adapters, generator=g)
        b.p.d_ctx.sub_(1)  # a row of the cache less
        graph.replay()
        torch.cuda.synchronize()
        got = [bits(b.d[k]) for k in STEPS]
        b.run()
        torch.cuda.synchronize()
        assert got == [bits(b.d[k]) for k in STEPS]


@pytest.mark.skipif(NODE is None, reason="node is not installed")
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 40, 110]])
def test_the_block_through_the_host(dev, tmp_path, new):
    b = Block(dev, 70 + len(new), [17, 0, 50], new, pad=0)
    p = b.p
    arrays = {k: bits(v) for k, v in b.host.items()}
    arrays.update(kPool=bits(p.d_k), vPool=bits(p.d_v), table=bits(p.d_table), start=bits(p.d_start), ctx=bits(p.d_ctx), inv=bits(b.inv))
    blob, index = bytearray(), {}
    for name, data in arrays.items():
        index[name] = [len(blob), len(data)]
        blob += data
    (tmp_path / "case.bin").write_bytes(bytes(blob))
    (tmp_path / "case.json").write_text(json.dumps(dict(
        nqh=b.nqh, hd=b.hd, hidden=b.hidden, pages=p.num_pages, pageSize=p.page, nSeqs=3, tableStride=p.table.shape[1], nTokens=b.n,
        maxTokens=max(new), rank=b.rank, adapters=b.adapters, arrays=index)))
    announce(f"TS host block new={new}")
    run = subprocess.run([NODE, str(RUN), "block", str(tmp_path)], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr
    got = (tmp_path / "out.bin").read_bytes()
    b.run()
    torch.cuda.synchronize()
    at = 0
    for name, t in (("qkv", b.d["qkv"]), ("attn", b.d["attn"]), ("sum", b.d["sum"]), ("codes", b.d["next8"]), ("scales", b.d["next_s"]),
                    ("kPool", p.d_k), ("vPool", p.d_v)):
        want = bits(t)
        assert got[at:at + len(want)] == want, name
        at += len(want)
    assert at == len(got)
