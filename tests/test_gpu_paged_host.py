"""A step of drafted trees through the TypeScript host (node host/run.js paged): append from one projection's output,
attention, the tokens' log probabilities, commit. The Python wrappers' results on the same inputs are checked against
64-bit definitions in test_gpu_paged_attn.py, test_gpu_paged_store.py and test_gpu_logprobs.py; the same calls give the
same bits, so the host's must equal them."""
import json
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from conftest import announce
from g4attn import ops
from paged_helpers import EPS, Paged

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent
RUN = ROOT / "gemma4-webgpu_amd" / "host" / "run.js"
NODE = shutil.which("node")


@pytest.mark.skipif(NODE is None, reason="node is not installed")
@pytest.mark.parametrize("hd,kv,window", [(256, "f16", 64), (512, "e4m3", 0)])
def test_a_drafted_step_through_the_host(dev, tmp_path, hd, kv, window):
    nqh, vocab, top, parents = 8, 1000, 5, [[-1, 0, 0, 1, 2], [-1], [-1, 0, 1, 1]]
    p = Paged(dev, 40 + hd, [130, 0, 37], [5, 1, 4], hd=hd, page=16, kv=kv, parents=parents, spare_pages=2, pad=1)
    p.upload()
    n = p.tokens
    r = np.random.default_rng(41)
    qkv = r.standard_normal((n, nqh + 2, hd)).astype(np.float32) * 2
    w = [(1 + 0.1 * r.standard_normal(hd)).astype(np.float16) for _ in range(2)]
    logits = (r.standard_normal((n, vocab)) * 8).astype(np.float32)
    tokens = r.integers(0, vocab, n).astype(np.int32)
    path = np.array([[0, 2, 4], [0, 0, 0], [0, 1, 3]], np.int32)
    accepted = np.array([3, 1, 2], np.int32)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    inv = ops.rope_inv_freq(1e4, hd, False, None)
    torch.cuda.synchronize()
    bits = lambda t: t.cpu().contiguous().view(torch.uint8).numpy().tobytes()  # noqa: E731
    arrays = dict(kPool=bits(p.d_k), vPool=bits(p.d_v), table=bits(p.batch.tensors[0]), start=bits(p.batch.tensors[1]),
                  ctx=bits(p.batch.tensors[2]), positions=bits(p.batch.tensors[3]), mask=bits(p.batch.tensors[4]),
                  qkv=qkv.tobytes(), qw=w[0].tobytes(), kw=w[1].tobytes(), inv=bits(inv), logits=logits.tobytes(),
                  tokens=tokens.tobytes(), path=path.tobytes(), accepted=accepted.tobytes())
    blob, index = bytearray(), {}
    for name, b in arrays.items():
        index[name] = [len(blob), len(b)]
        blob += b
    (tmp_path / "case.bin").write_bytes(bytes(blob))
    (tmp_path / "case.json").write_text(json.dumps(dict(
        nqh=nqh, nkh=1, hd=hd, pages=p.num_pages, pageSize=p.page, nSeqs=3, tableStride=p.table.shape[1], nTokens=n,
        maxTokens=5, pathStride=3, window=window, vocab=vocab, topK=top, f8=kv == "e4m3", arrays=index)))

    announce(f"TS host drafted step hd={hd} {kv}")
    run = subprocess.run([NODE, str(RUN), "paged", str(tmp_path)], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr
    got = (tmp_path / "out.bin").read_bytes()

    d_qkv = up(qkv)
    batch = ops.PagedBatch(*p.batch.tensors[:3], n, max_tokens=5, positions=p.batch.tensors[3], tree_mask=p.batch.tensors[4])
    q_out = torch.zeros(n, nqh, hd, dtype=torch.float16, device=dev)
    out = torch.zeros(n, nqh, hd, device=dev)
    ops.paged_append(p.cache, batch, d_qkv[:, :nqh], d_qkv[:, nqh:nqh + 1], d_qkv[:, nqh + 1:], up(w[0]), up(w[1]), inv,
                     q_out, eps=EPS)
    ws = torch.empty(ops.paged_attn_workspace_bytes(p.cache, batch, nqh), dtype=torch.uint8, device=dev)
    ops.paged_attn(p.cache, batch, q_out, out, ws, sliding_window=window)
    lp, ent, tops = torch.empty(n, device=dev), torch.empty(n, device=dev), torch.empty(n, top, device=dev)
    ids = torch.empty(n, top, dtype=torch.int32, device=dev)
    lws = torch.empty(ops.token_logprobs_workspace_bytes(n, vocab, top), dtype=torch.uint8, device=dev)
    ops.token_logprobs(up(logits), up(tokens), lp, ent, lws, ids, tops, cap=30.0, temperature=0.7)
    new_ctx = torch.empty(3, dtype=torch.int32, device=dev)
    ops.paged_commit([p.cache], batch, up(path), up(accepted), new_ctx)
    torch.cuda.synchronize()
    assert new_ctx.tolist() == [133, 1, 39]
    at, used = 0, sum(p.new)
    for name, t in (("out", out), ("logprobs", lp), ("entropy", ent), ("topIds", ids), ("topLogprobs", tops),
                    ("newCtxLens", new_ctx), ("kPool", p.d_k), ("vPool", p.d_v)):
        want = bits(t)
        have = got[at:at + len(want)]
        at += len(want)
        if name == "out":  # the padding's row is nobody's
            want, have = (x[:used * nqh * hd * 4] for x in (want, have))
        assert have == want, name
    assert at == len(got)
