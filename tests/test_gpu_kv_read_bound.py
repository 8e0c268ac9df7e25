"""TQ4 rows read back, held to what the products that run can be off by: for a row with scales d0, d1, 18 x 2^-24 (|d0| + |d1|) in front of the
rounding to the output type.  X and the first stage's sums are off by 2^-24 together, the value + residual split of an element of Z (below 0.17) by
2^-25 twice, each of U's outputs sums eight of those and rounds a few times more (2 x 2^-24), Y adds both halves times their scales.
Small scales are left out for fp16 outputs: there the rounding is to fixed steps, which half_step counts."""
import numpy as np
import pytest

import rows64
from rows64 import half_step, random_rows, values

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [2.0 ** -9, 1.0, 2.0 ** 7])
def test_tq4_rows_inside_the_products_bound(native_libs, dtype, scale):
    from warp34_b200 import kv
    rng, heads, pages = np.random.default_rng(7), 4, 64
    layer = kv.KvLayer(pages, heads, formats=rows64.formats("tq4"))
    rows = random_rows(rows64.TQ4, pages * heads * 16, rng, scale=scale).reshape(pages, heads, 16, 132)
    # the extremes of a transform: equal codes, alternating ones, one half without scale
    rows[3, :, :, 2:66], rows[3, :, :, 68:] = 0xff, 0x00
    rows[4, :, :, 2:66] = 0x0f
    rows[5, :, :, 66:68] = 0
    layer.k.copy_(torch.from_numpy(rows.copy()).view(-1))
    layer.v.copy_(torch.from_numpy(rows.copy()).view(-1))
    slots = rng.permutation(pages * 16).astype(np.int32)
    batch = kv.StepBatch([0, len(slots)], [0], [len(slots)], np.zeros((1, pages), np.int32), slots, pages, 0.0625)
    k, v = (torch.zeros(len(slots), heads * 256, dtype=dtype, device="cuda") for _ in range(2))
    kv.kv_cache_read(kv.Executor(1 << 12), layer, batch, k, v)
    torch.cuda.synchronize()
    taken = np.ascontiguousarray(rows[slots >> 4, :, slots & 15]).reshape(-1, 132)
    want = values(taken, rows64.TQ4)
    d = np.abs(taken.reshape(-1, 2, 66)[:, :, :2].copy().view(np.float16).astype(np.float64)).sum((1, 2))
    bound = half_step(want, dtype) * (1 + 2.0 ** -8) + 18 * 2.0 ** -24 * d[:, None]
    for got in (k, v):
        bad = ~(np.abs(got.double().cpu().numpy().reshape(want.shape) - want) <= bound)
        assert not bad.any(), f"{bad.sum()} of {bad.size}, first {np.argwhere(bad)[0]}"
