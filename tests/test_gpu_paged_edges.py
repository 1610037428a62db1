"""GPU tier: the paged latent cache (``smla.paged``) where its inputs leave the ordinary: lengths past the table, rows and
projections that are not finite, refused slots, rows given back.  Tolerances as in ``test_gpu_paged``."""
import random

import pytest
import torch

from conftest import announce
from oracle import paged as op
from test_gpu_paged import BF16, _apply, _cache, _check_attn, _cu, _i32, _tables, _to

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("window,first", [(1, 4), (20, 4), (20, 0), (3, 1), (40, 70), (5, 64), (5, 65), (30, 1 << 29), (1 << 29, 3)])
def test_attn_window_past_the_table(dev, window, first, kv):
    """Rows past the table's columns are not there; the first rows are, also where the whole window lies past the table."""
    from smla import paged
    announce(f"paged_attn lengths past a table of 64 rows, window={window} first={first} {kv}")
    pages, scales, table = _cache(201, [64] * 5, 16, 512, kv)
    lens, cu = [64, 66, 83, 100, 84], _cu([3, 2, 3, 1, 20])
    q = torch.randn(cu[-1], 16, 512, generator=torch.Generator().manual_seed(window % 97 + first % 89)).to(torch.bfloat16)
    dq, dp, ds, dt = _to(dev, q, pages, scales, table)
    out = paged.paged_attn(dq, dp, dt, _i32(lens, dev), _i32(cu, dev), 512 ** -0.5, None, window, first, page_scales=ds)
    torch.cuda.synchronize()
    _check_attn(out, q, pages, scales, table, lens, cu, None, window, first)


@pytest.mark.parametrize("window,first,length", [(150, 1550, 1700), (10, 1 << 29, 5000), (10, 1500, 5000), (700, 900, 2000)])
def test_attn_window_past_the_table_split(dev, window, first, length):
    """The same with rows enough that tiles are split over workgroups."""
    from smla import paged
    announce(f"paged_attn a token at {length} over a table of 1600 rows, window={window} first={first}")
    pages, _, table = _cache(202, [1600], 16, 576)
    q = torch.randn(2, 64, 576, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    dq, dp, dt = _to(dev, q, pages, table)
    out = paged.paged_attn(dq, dp, dt, _i32([length], dev), _i32([0, 2], dev), 576 ** -0.5, None, window, first)
    torch.cuda.synchronize()
    _check_attn(out, q, pages, None, table, [length], [0, 2], None, window, first)
