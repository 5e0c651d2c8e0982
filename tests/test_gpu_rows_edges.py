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
