"""g4_token_logprobs against log_softmax in 64 bits: sizes around a chunk, types, strides and alignment, ties, masks of
-inf, NaN rows, many candidates at the selection's bound."""
import numpy as np
import pytest
import torch

from conftest import announce
from g4attn import ops

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def call(logits, tokens, k, cap=0.0, temperature=1.0, stream=None):
    rows, vocab = logits.shape
    dev = logits.device
    lp, ent = torch.full((rows,), 7.0, device=dev), torch.full((rows,), 7.0, device=dev)
    ids = torch.full((rows, k), 77, dtype=torch.int32, device=dev) if k else None
    tops = torch.full((rows, k), 7.0, device=dev) if k else None
    ws = torch.full((ops.token_logprobs_workspace_bytes(rows, vocab, k),), 0xff, dtype=torch.uint8, device=dev)
    ops.token_logprobs(logits, tokens, lp, ent, ws, ids, tops, cap=cap, temperature=temperature, stream=stream)
    torch.cuda.synchronize()
    return lp, ent, ids, tops


def check(logits, tokens, k, cap=0.0, temperature=1.0):
    lp, ent, ids, tops = (None if x is None else x.cpu() for x in call(logits, tokens, k, cap, temperature))
    x, tokens = logits.cpu(), tokens.cpu().long()
    z = x.double()
    if cap:
        z = torch.where(z.isinf(), z, cap * torch.tanh(z / cap))
    z = z / temperature
    logp = torch.log_softmax(z, -1)
    p = logp.exp()
    # z is off by at most 4 half-steps (quotient, tanh, product, quotient), so is the difference to the
    # maximum, and e^d by that and 2^-22; the sums add 32 terms in turn and then 14 + a few levels.
    zmax = z.masked_fill(z.isinf(), 0).abs().max(-1).values
    eta = (10 * zmax) * 2.0 ** -24 + 2.0 ** -22
    ok = tokens >= 0
    want = torch.where(ok, logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0], torch.zeros(()).double())
    tol = eta + 64 * 2.0 ** -24 + want.abs().nan_to_num(posinf=0) * 2.0 ** -22
    fin = want.isfinite()
    assert ((lp.double() - want).abs()[fin] <= tol[fin]).all(), ((lp.double() - want).abs() / tol).max()
    assert torch.equal(lp[~fin], want[~fin].float())
    d = (z - z.max(-1, keepdim=True).values)
    mean = torch.where(p > 0, p * d.abs().nan_to_num(posinf=0), torch.zeros(()).double()).sum(-1)
    want_h = -torch.where(p > 0, p * logp, torch.zeros(()).double()).sum(-1)
    tol_h = (mean + 1) * (2 * eta + 128 * 2.0 ** -24)
    assert ((ent.double() - want_h).abs() <= tol_h).all(), ((ent.double() - want_h).abs() / tol_h).max()
    if k:
        order = torch.sort(x.float(), dim=-1, descending=True, stable=True)[1][:, :k]
        live = x.gather(1, order) > -float("inf")
        assert torch.equal(ids.long(), torch.where(live, order, torch.full((), -1)))
        want_t = logp.gather(1, order)
        assert (tops[~live] == -float("inf")).all()
        err = (tops.double() - want_t).abs()
        assert (err[live] <= (tol_of(eta, want_t))[live]).all()


def tol_of(eta, want):
    return eta[:, None] + 64 * 2.0 ** -24 + want.abs().nan_to_num(posinf=0) * 2.0 ** -22


def inputs(dev, seed, rows, vocab, dtype, spread=4.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, device=dev) * spread
    tokens = torch.randint(vocab, (rows,), generator=g, device=dev, dtype=torch.int32)
    return x.to(TYPES[dtype]), tokens


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 255, 1000, 8191, 8192, 8193, 16384, 50257, 262144])
def test_sizes(dev, dtype, vocab):
    announce(f"tokenLogprobs vocab={vocab} {dtype}")
    x, t = inputs(dev, vocab, 3, vocab, dtype)
    check(x, t, min(vocab, 20), cap=30.0 if vocab % 2 else 0.0, temperature=0.7 if vocab % 3 == 1 else 1.0)


@pytest.mark.parametrize("k", [0, 1, 2, 31, 64])
@pytest.mark.parametrize("rows", [1, 5, 130])
def test_top_counts_and_rows(dev, k, rows):
    announce(f"tokenLogprobs k={k} rows={rows}")
    x, t = inputs(dev, 10 * k + rows, rows, 20000, "bf16")
    check(x, t, k, cap=30.0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("offset,stride", [(0, 9001), (1, 9000), (8, 9008), (3, 8999)])
def test_strided_and_misaligned_rows(dev, dtype, offset, stride):
    announce(f"tokenLogprobs {dtype} offset={offset} stride={stride}")
    x, t = inputs(dev, stride, 4, stride, dtype)
    flat = torch.cat([x.flatten(), x.flatten()[:64]])
    rows = flat[offset:offset + 4 * stride].view(4, stride)[:, :8900]
    check(rows, t % 8900, 5)


@pytest.mark.parametrize("shape", ["equal", "ascending", "two values", "few", "one", "signed zeros"])
@pytest.mark.parametrize("vocab", [8192, 20001])
def test_ties_and_orders(dev, shape, vocab):
    """Equal logits rank by index; more candidates at the bound than the selection's buffer holds."""
    x = torch.zeros(2, vocab)
    if shape == "ascending":
        x = torch.arange(2 * vocab).view(2, vocab).float() / 1000
    elif shape == "two values":
        x[:, ::3] = 1.0
    elif shape == "few":  # fewer above -inf than asked for, then some thousands in few threads' hands
        x.fill_(-float("inf"))
        x[0, [5, 700, vocab - 1]] = torch.tensor([1.0, 2.0, 1.0])
        x[1, 4096:4096 + 3000] = 0.5
    elif shape == "one":
        x.fill_(-float("inf"))
        x[:, vocab // 2] = -3.0
    elif shape == "signed zeros":
        x[:, ::2] = -0.0
    announce(f"tokenLogprobs {shape} vocab={vocab}")
    check(x.to(dev), torch.tensor([5, vocab // 2], dtype=torch.int32, device=dev), 33)


@pytest.mark.parametrize("vocab", [500, 30000])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_rows_without_a_distribution(dev, vocab, cap):
    x, t = inputs(dev, 3, 5, vocab, "f32")
    x[0] = -float("inf")
    x[1, 17] = float("nan")
    x[2, vocab - 2] = float("inf")
    x[3, 1:] = -float("inf")  # one logit alone: probability 1
    t[3], t[4] = 0, -1
    announce(f"tokenLogprobs odd rows vocab={vocab} cap={cap}")
    lp, ent, ids, tops = (a.cpu() for a in call(x, t, 4, cap=cap))
    for r in (0, 1, 2):
        assert lp[r].isnan() and ent[r].isnan() and tops[r].isnan().all()
    assert (ids[0] == -1).all() and 17 not in ids[1].tolist() and ids[2, 0] == vocab - 2
    assert lp[3] == 0 and ent[3] == 0 and ids[3].tolist() == [0, -1, -1, -1] and tops[3, 0] == 0
    assert lp[4] == 0 and ent[4] > 0  # a token outside the vocabulary
    t[4] = vocab
    assert call(x, t, 4, cap=cap)[0][4] == 0


@pytest.mark.parametrize("spread,temperature", [(0.01, 1.0), (30.0, 1.0), (4.0, 0.05), (4.0, 50.0), (1e4, 1.0)])
def test_flat_and_sharp_rows(dev, spread, temperature):
    announce(f"tokenLogprobs spread={spread} temperature={temperature}")
    x, t = inputs(dev, 8, 3, 70000, "f32", spread)
    check(x, t, 8, temperature=temperature)
    check(x, t, 8, cap=30.0, temperature=temperature)


def test_parts_asked_for_alone_streams_and_replays(dev):
    x, t = inputs(dev, 9, 6, 40000, "f32")
    lp, ent, ids, tops = call(x, t, 5)
    ws = torch.empty(ops.token_logprobs_workspace_bytes(6, 40000, 5), dtype=torch.uint8, device=dev)
    only = torch.empty(6, device=dev)
    announce("tokenLogprobs parts, streams, replays")
    ops.token_logprobs(x, t, only, None, ws)
    assert torch.equal(only, lp)
    ops.token_logprobs(x, None, None, only, ws)
    assert torch.equal(only, ent)
    i2, t2 = torch.empty_like(ids), torch.empty_like(tops)
    ops.token_logprobs(x, None, None, None, ws, i2, t2)
    assert torch.equal(i2, ids) and torch.equal(t2, tops)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = call(x, t, 5)
    assert all(torch.equal(a, b) for a, b in zip(other, (lp, ent, ids, tops)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.token_logprobs(x, t, only, ent, ws, i2, t2)
    for seed in range(3):
        y, u = inputs(dev, 20 + seed, 6, 40000, "f32")
        x.copy_(y)
        t.copy_(u)
        graph.replay()
        torch.cuda.synchronize()
        want = call(y, u, 5)
        assert all(torch.equal(a, b) for a, b in zip((only, ent, i2, t2), want))


@pytest.mark.parametrize("cap", [64.0, 65.0, 1000.0, 1e6, 1e30])
def test_caps_far_above_the_logits(dev, cap):
    """A cap's rounding is the logits', not the cap's (which would leave 0.06 at 1e6): up to 64, where the sums take a
    shorter form, 4 half-steps of the cap, above it within the tolerance of every other case."""
    announce(f"tokenLogprobs cap={cap}")
    x, tokens = inputs(dev, 90, 5, 5000, "f32", spread=1.0)
    if cap > 64:
        check(x, tokens, 7, cap=cap)
        return
    lp, _, _, _ = call(x, tokens, 0, cap=cap)
    want = torch.log_softmax(cap * torch.tanh(x.double() / cap), -1).gather(1, tokens.long()[:, None])[:, 0]
    # z of the token and of the sum: two differences, each 4 half-steps of the cap.
    assert ((lp - want).abs() <= 2 * 4 * cap * 2.0 ** -24 + 64 * 2.0 ** -24 + want.abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab,most", [(262144, 16), (50257, 74), (151936, 27)])
def test_one_workspace_for_a_batch_that_shrinks(dev, dtype, vocab, most):
    """A loop sizes its workspace for its largest batch and goes on with it as sequences end."""
    announce(f"tokenLogprobs shrinking batch vocab={vocab} most={most} {dtype}")
    x, tokens = inputs(dev, vocab, most, vocab, dtype)
    ws = torch.empty(ops.token_logprobs_workspace_bytes(most, vocab, 20), dtype=torch.uint8, device=dev)
    for rows in (most, most - 1, most // 2, 1):
        want = call(x[:rows], tokens[:rows], 20)
        lp, ent, ids, tops = (torch.empty_like(a) for a in want)
        ws.fill_(0xff)
        ops.token_logprobs(x[:rows], tokens[:rows], lp, ent, ws, ids, tops)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((lp, ent, ids, tops), want)), rows
