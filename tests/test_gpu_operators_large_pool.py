"""Scored attention and the read-back over pages more than 4 GiB from their slab's base: the bits of a small pool.

Page ids change nothing but addresses, so a layer's pages moved behind the first 4 GiB of a large one give equal outputs, through every route
(the one-launch kernel, the stream kernels, the chunk kernel, the row kernel)."""
import numpy as np
import pytest

import rows64

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FOUR_GIB = 1 << 32
HEADS, HQ = 4, 16
# lens and contexts: one token over a short context, a batch that is split over its keys, a chunk
SHAPES = {"few": ([1], [300]), "decode": ([1] * 24, [700] * 23 + [3000]), "chunk": ([130, 70], [500, 33])}


@pytest.fixture(scope="module")
def env(native_libs):
    from warp34_b200 import ffi, kv
    free, _ = torch.cuda.mem_get_info()
    assert free > (24 << 30), "these cases hold about 10 GiB of pool"
    return ffi, kv


@pytest.mark.parametrize("name", ["tq4", "fp8", "q8", "bf16"])
def test_pages_beyond_4_gib_give_the_same_bits(env, name):
    ffi, kv = env
    page = HEADS * 16 * rows64.ROW[rows64.NAMES[name][0]]
    base = FOUR_GIB // page + 5
    most = max(sum((c + n + 15) // 16 for n, c in zip(*s)) for s in SHAPES.values()) + 8
    big = kv.KvLayer(base + most, HEADS, formats=rows64.formats(name))
    dtype = torch.bfloat16 if name == "bf16" else torch.float16
    for shape, (lens, ctx) in SHAPES.items():
        cache = rows64.Cache(name, HEADS, lens, ctx, 17)
        pages = cache.rows[0].shape[0]
        for far, near in ((big.k, cache.layer.k), (big.v, cache.layer.v)):
            far.view(-1, page)[base:base + pages] = near.view(-1, page)
        n = sum(lens)
        g = torch.Generator().manual_seed(3)
        q = torch.randn(n, HQ, 256, generator=g).to(dtype).cuda()
        slopes = torch.linspace(0.001, 0.02, HQ).cuda()
        near_batch = cache.batch()
        cache.table += base
        far_batch = cache.batch()
        for flags, scratch in ((0, 64 << 20), (ffi.EXEC_FLAG_PRECISE_ATTENTION, 1 << 12)):
            ex = kv.Executor(scratch)
            ex.ex.flags = flags
            outs = []
            for layer, batch in ((cache.layer, near_batch), (big, far_batch)):
                out = torch.full((n, HQ, 256), 7.0, dtype=dtype, device="cuda")
                kv.paged_attention_scored(ex, layer, batch, q, out, HQ, softcap=30.0, slopes=slopes)
                outs.append(out)
            assert outs[0].abs().sum() > 0 and torch.equal(outs[0], outs[1]), (shape, flags)
        # read back by position and by slot
        req = np.repeat(np.arange(len(lens)), lens)
        pos = np.concatenate([np.arange(c, c + m) for c, m in zip(ctx, lens)])
        rows = []
        for layer, batch, shift in ((cache.layer, near_batch, 0), (big, far_batch, base)):
            for by_slot in (False, True):
                ids = cache.table[req, pos // 16].astype(np.int64) - base + shift
                where = torch.as_tensor((ids * 16 + pos % 16).astype(np.int32)).cuda()
                batch.desc.write_slot_mapping = where.data_ptr() if by_slot else None
                k, v = (torch.zeros(n, HEADS * 256, dtype=dtype, device="cuda") for _ in range(2))
                kv.kv_cache_read(kv.Executor(1 << 12), layer, batch, k, v)
                torch.cuda.synchronize()
                rows.append((k, v))
        for k, v in rows[1:]:
            assert torch.equal(k, rows[0][0]) and torch.equal(v, rows[0][1]), shape
        assert rows[0][0].abs().sum() > 0
