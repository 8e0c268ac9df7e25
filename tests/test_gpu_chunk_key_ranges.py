"""A chunk whose keys are cut into ranges, some of them computed in fp32 because their rows differ too much in magnitude for one power of
two (prefill_pair.cuh): the ranges' masses and rows meet on the same scale.  Against attention in 64 bits, within the library's bound."""
import numpy as np
import pytest

from rows64 import Cache, random_rows, scored_attention
from util import plain_parity

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("name", ["tq4", "q8"])
def test_ranges_of_both_kinds(native_libs, name, scored):
    from warp34_b200 import kv
    hq, hkv, new, ctx = 2, 1, 40, 6000
    cache = Cache(name, hkv, [new], [ctx], seed=3)
    rng = np.random.default_rng(4)
    # every other stretch of 256 keys holds V rows of magnitude 2^-7 and, among them, one of 2^6: larger than its tile's power of two allows
    fmt = cache.layer.layout.v_format
    for start in range(0, ctx, 512):
        pos = np.arange(start, start + 256)
        cache.rows[1][cache.table[0, pos // 16], :, pos % 16] = random_rows(fmt, 256, rng, scale=2.0 ** -7)[:, None]
        cache.rows[1][cache.table[0, (start + 100) // 16], :, (start + 100) % 16] = random_rows(fmt, 1, rng, scale=64.0)
    cache.upload()
    q = torch.randn(new, hq, 256, generator=torch.Generator().manual_seed(5)).half()
    out = torch.zeros(new, hq, 256, dtype=torch.float16, device="cuda")
    ex, batch = kv.Executor(64 << 20), cache.batch()
    if scored:
        kv.paged_attention_scored(ex, cache.layer, batch, q.cuda(), out, hq)
    else:
        kv.paged_attention(ex, cache.layer, batch, q.cuda(), out, hq)
    torch.cuda.synchronize()
    want, _ = scored_attention(cache, q.float().numpy(), hq)
    ok, msg = plain_parity(out.float().cpu().numpy(), want)
    assert ok, msg
