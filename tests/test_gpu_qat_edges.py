"""GPU tier: fp4 blocks with values that are not finite: NaN in all of such a block, the others as without it."""
import math

import numpy as np
import pytest
import torch

from conftest import announce
from test_gpu_qat import _pool_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [math.nan, -math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n", [32, 128, 1024])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_blocks_that_are_not_finite(dev, n, dt, bad):
    from smla import qat as sq
    announce(f"fp4 blocks with {bad} n={n} {dt}")
    x = torch.randn(11, n, generator=torch.Generator().manual_seed(n)).to(dt)
    x[2] = 0.0
    x[3] = torch.finfo(dt).max                   # finite: the largest scale there is
    y = x.clone()
    y[0, n - 1], y[2, 7], y[10, n // 2] = bad, bad, bad
    hit = ~y.isfinite().view(11, n // 32, 32).all(-1)
    rows = hit.any(-1)
    want_codes, want_scales = [t.cpu() for t in sq.fp4_pack(x.to(dev), rotate=False)]
    codes, scales = [t.cpu() for t in sq.fp4_pack(y.to(dev), rotate=False)]
    assert hit.sum() == 3 and (scales[hit] == 255).all() and (want_scales < 255).all()
    assert torch.equal(scales[~hit], want_scales[~hit])
    assert torch.equal(codes.view(11, n // 32, 16)[~hit], want_codes.view(11, n // 32, 16)[~hit])
    trip, plain = sq.fp4_act_quant(y.to(dev)).cpu(), sq.fp4_act_quant(x.to(dev)).cpu()
    assert trip.view(11, n // 32, 32)[hit].isnan().all()
    assert torch.equal(trip.view(11, n // 32, 32)[~hit], plain.view(11, n // 32, 32)[~hit])
    # the rotation spreads it over the row (and takes the row of the largest finite values past them)
    assert (sq.fp4_pack(y.to(dev))[1].cpu()[rows] == 255).all()
    turned = sq.rotate_fp4(y.to(dev)).cpu()
    assert turned[rows].isnan().all()
    np.testing.assert_array_equal(turned[~rows].numpy(), sq.rotate_fp4(x.to(dev)).cpu()[~rows].numpy())


@pytest.mark.parametrize("d", [128, 512])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_pooled_rows_that_are_not_finite(dev, d, bad):
    """The compressor's rows with the rotate mode: a row that is NaN without it is NaN with it."""
    from smla import _lib, ops
    from smla import qat as sq
    announce(f"gated pool rotate with {bad} d={d}")
    kv, sc_, ape, nw, cis, r, rd = _pool_case(d, d)
    cos_t, sin_t = cis.real.contiguous().to(dev), cis.imag.contiguous().to(dev)
    run = lambda v, sim: ops.gated_pool_op(v.to(dev), sc_.to(dev), ape.to(dev), nw.to(dev), cos_t, sin_t, r, rd, 1e-6, sim)  # noqa: E731
    clean = run(kv, _lib.SIM_ROTATE_FP4).cpu()
    kv[1, 9, 5] = bad
    plain, fused = run(kv, _lib.SIM_NONE), run(kv, _lib.SIM_ROTATE_FP4)
    rows = plain.isnan().any(-1).cpu()
    assert rows.any() and not rows.all()
    assert fused.cpu()[rows].isnan().all() and torch.equal(fused.cpu()[~rows], clean[~rows])
    np.testing.assert_array_equal(fused.cpu().numpy(), sq.rotate_fp4(plain).cpu().numpy())
