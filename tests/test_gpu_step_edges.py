"""Edges of the serving-step operators on the GPU: inputs that no kernel of the framework
wrote, refusals, orders of launches, and outputs too small for an absolute tolerance."""
import numpy as np
import pytest
import torch

from gpu_util import cuda
from test_gpu_step import BF16, F16, F32, O, fe, make_sparse

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------- scales nobody wrote
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("ctx", [900, 9000, 150001])
def test_sparse_pages_with_nan_scales_rank_as_infinite_ones(dt, ctx):
    """Far more pages with NaN scales than are chosen: the first of them, num_pages in all."""
    p = make_sparse(ctx, [ctx], 4, 1, 64, 16, dt)
    v, s = O.boxes(p["k"])
    pages = -(-ctx // 16)
    s[p["tables"][0, 3:pages - 5], 0] = np.array([0x7fffffff, 0xffffffff, 0x7fc00000],
                                                 np.uint32).view(np.float32)[
        np.arange(pages - 8) % 3]
    for first, last, num_pages in ((1, 1, 4), (2, 3, 9), (0, 1, 40)):
        out, got = fe().sparse_paged_attention(
            cuda(p["q"], dt), cuda(p["k"], dt), cuda(p["v"], dt), (cuda(v), cuda(s)),
            cuda(p["tables"]), cuda(p["lens"]), num_pages, 16, keep_first=first, keep_last=last)
        rest = num_pages - first - last
        want = list(range(first)) + list(range(3, 3 + rest)) + list(range(pages - last, pages))
        assert got[0, 0].tolist() == want
        assert torch.isfinite(out).all() and fe().device_errors() == 0
