"""The operators between two attention blocks where a row, an adapter or a call's size is out of the ordinary: rows as small as
the norm's eps, adapters of one segment that are not finite, arguments that change in place."""
import pytest
import torch

from batch_rows import TYPES, unit
from conftest import announce
from g4attn import ops
from test_gpu_rownorm import NORM, codes_within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [1e-6, 1e-12, 1e-20, 2e-38])
@pytest.mark.parametrize("n", [64, 77, 1536, 20000])
def test_zero_rows_of_a_small_eps(dev, n, eps):
    """A row of zeros, as a padded batch has it, is zeros in 8 bits whatever eps is; so is a row of zero weights, and a row whose
    norm is far below the least scale has its own codes."""
    announce(f"addRmsNorm zero rows n={n} eps={eps}")
    x = torch.randn(5, n, generator=torch.Generator().manual_seed(n))
    x[1] = 0
    x[3] *= 1e-36
    x = x.to(dev)
    out, scales = torch.full((5, n), 7.0, device=dev).to(TYPES["e4m3"]), torch.full((5,), 7.0, device=dev)
    ops.add_rms_norm(x, None, out, scales=scales, eps=eps)
    torch.cuda.synchronize()
    assert (out.float()[1] == 0).all() and scales[1].isfinite()
    some = [0, 1, 2, 4]
    codes_within(out.view(torch.uint8)[some].view(TYPES["e4m3"]), scales[some], unit(x[some].cpu().double(), eps), NORM, "beside it")
    # Squares of 1e-36 are nothing beside any of these eps.
    codes_within(out.view(torch.uint8)[3:4].view(TYPES["e4m3"]), scales[3:4], x[3:4].cpu().double() / eps ** 0.5, NORM, "a small row")
    nothing = torch.zeros(n, dtype=torch.float16, device=dev)
    ops.add_rms_norm(x, nothing, out, scales=scales, eps=eps)
    torch.cuda.synchronize()
    assert (out.float() == 0).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,runs", [(1, 1), (20, 1), (20, 20), (300, 2), (300, 300)])
@pytest.mark.parametrize("bad", ["inf", "nan"])
def test_an_inner_sum_that_is_not_finite_stays_in_its_segment(dev, kind, tokens, runs, bad):
    """Down rows of one segment that are not finite: its outputs are not, those of the segments beside it, in the same tile too,
    are what they were, whether a tile's tokens share an adapter or have one each."""
    announce(f"lora {bad} in a segment {kind} tokens={tokens} runs={runs}")
    widths, rank, n = (10, 21, 9, 60), 16, 64
    g = torch.Generator().manual_seed(tokens)
    a = (torch.randn(5, 4 * rank, n, generator=g) * 0.1).to(TYPES[kind]).to(dev)
    b = (torch.randn(5, sum(widths), rank, generator=g) + 3).to(TYPES[kind]).to(dev)
    x, base = torch.randn(tokens, n, generator=g).half().to(dev), torch.randn(tokens, sum(widths), generator=g).to(dev)
    ids = ((torch.arange(tokens) * runs // tokens) % 5).int().to(dev)
    x8, xs = x.float().to(TYPES["e4m3"]), torch.ones(tokens, device=dev)
    w, ws = torch.zeros(sum(widths), n, device=dev).to(TYPES["e4m3"]), torch.ones(sum(widths), device=dev)

    def both(a):
        low = ops.LoraAdapters(a, b, None, widths)
        out, out8 = torch.empty_like(base), torch.empty_like(base)
        ops.lora_add(low, ids, x, base, out, torch.empty(ops.lora_workspace_bytes(low, tokens), dtype=torch.uint8, device=dev))
        ops.linear_e4m3(x8, xs, w, ws, out8, torch.empty(ops.linear_e4m3_workspace_bytes(tokens, sum(widths), n, low), dtype=torch.uint8,
                                                          device=dev), lora=low, adapter_ids=ids)
        torch.cuda.synchronize()
        return out, out8

    want = both(a)
    for s in range(4):
        odd = a.clone()
        odd[:, s * rank + 3, 5] = float(bad)
        first = sum(widths[:s])
        others = [o for o in range(sum(widths)) if not first <= o < first + widths[s]]
        for got, was in zip(both(odd), want):
            assert not got[:, first:first + widths[s]].isfinite().any()
            assert torch.equal(got[:, others], was[:, others])


def test_an_eps_that_changes_in_place(dev):
    """eps as a tensor of one element: its value at the call counts, as with any number."""
    announce("addRmsNorm eps in a tensor")
    x = torch.randn(3, 64, generator=torch.Generator().manual_seed(1)).to(dev)
    eps = torch.tensor(1e-6)
    for value in (1e-6, 0.5, 1e-6):
        eps.fill_(value)
        got, want = torch.empty_like(x), torch.empty_like(x)
        ops.add_rms_norm(x, None, got, eps=eps)
        ops.add_rms_norm(x, None, want, eps=float(eps))
        assert torch.equal(got, want)


def test_the_most_rows_of_the_longest_kind(dev):
    """2^22 rows of more than 16384 elements: as many threads as a launch cannot take along one side."""
    rows, n = 2 ** 22, 16385
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < rows * n * 2 + (16 << 30):
        pytest.skip("needs 144 GB of free memory")
    announce("addRmsNorm 2^22 rows of 16385")
    x = torch.empty(rows, n, dtype=torch.float16, device=dev)
    part = rows // 16
    for i in range(16):
        x[i * part:(i + 1) * part] = 2.0 - 4.0 * (i % 2)
    ops.add_rms_norm(x, None, x)
    torch.cuda.synchronize()
    for i in range(16):  # 2 / sqrt(4 + 1e-6) is 1 in f16
        assert (x[i * part:(i + 1) * part] == 1.0 - 2.0 * (i % 2)).all()
    del x
    torch.cuda.empty_cache()
