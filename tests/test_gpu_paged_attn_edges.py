"""g4_paged_attn at edges of its tiles, windows and number formats: chains that run past the block table, against the
definition in 64 bits. Tolerances are derived in paged_helpers.Paged.expected, or where a test stands."""
import pytest
import torch

from conftest import announce
from paged_helpers import Paged

pytestmark = pytest.mark.gpu


def run(p, **kw):
    out = p.upload().attn(**kw)
    torch.cuda.synchronize()
    p.check(out, **kw)
    return out


@pytest.mark.parametrize("hd,nqh,new", [(256, 8, 1), (256, 8, 4), (256, 2, 30), (256, 8, 40), (512, 2, 30), (512, 8, 40)])
@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("window", [0, 30])
@pytest.mark.parametrize("ctx", [112, 111, 97, 80])
def test_chains_past_the_block_table(dev, hd, nqh, new, kv, window, ctx):
    """Seven pages of 16 rows: the table ends in the middle of a 32-row tile, whose second half no token attends."""
    announce(f"pagedAttn past the table hd={hd} nqh={nqh} new={new} kv={kv} window={window} ctx={ctx}")
    p = Paged(dev, ctx + new, [ctx, 20], [new, 1], hd=hd, nqh=nqh, kv=kv, page=16)
    p.table = p.table[:, :7].copy()
    run(p, window=window)
