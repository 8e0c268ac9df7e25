"""Scored attention and the read-back under the bounds-checked build (see test_gpu_bounds_build.py)."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env(native_libs):
    from warp34_b200 import build, ffi, kv
    return dict(kv=kv, lib=native_libs[0], blib=ffi.bind_kernel_abi(build.build_bounds()))


def _report(blib):
    out = (C.c_int32 * 4)()
    assert blib.warp34_bounds_report(out, 1) == 0
    return dict(what=out[0] & 255, where=out[0] >> 8, value=out[1], limit=out[2], count=out[3])


@pytest.mark.parametrize("name", ["tq4", "bf16", "q8"])
def test_scored_attention_and_read_run_clean_and_catch_what_is_outside(env, name):
    """Scored attention (one launch, stream and chunk sizes) and the read-back under the checked build: nothing recorded and the regular build's
    results; pages outside a pool declared smaller than it is are recorded, with the place, and read as page 0."""
    from rows64 import Cache
    kv, lib, blib = env["kv"], env["lib"], env["blib"]
    for hq, hkv, lens, ctx in ((4, 2, [1], [100]), (16, 4, [1] * 9, [2040, 5, 64, 1000, 33, 700, 129, 300, 16]), (8, 2, [70, 5], [90, 0])):
        cache = Cache(name, hkv, lens, ctx, seed=1)
        n = sum(lens)
        q = torch.randn(n, hq, 256, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16 if name == "bf16" else torch.float16).cuda()
        batch = cache.batch()
        batch.desc.write_slot_mapping = None
        ex = kv.Executor(64 << 20)
        outs = []
        for which in (lib, blib):
            if which is blib:
                assert blib.warp34_bounds_set_pool_pages(cache.layer.num_pages) == 0
                _report(blib)
            out, rows = torch.zeros_like(q), torch.zeros(n, hkv * 256, dtype=torch.float16, device="cuda")
            kv.paged_attention_scored(ex, cache.layer, batch, q, out, hq, softcap=30.0, lib=which)
            kv.kv_cache_read(ex, cache.layer, batch, rows, None, lib=which)
            torch.cuda.synchronize()
            outs.append((out, rows))
        assert _report(blib)["count"] == 0
        assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
        assert blib.warp34_bounds_set_pool_pages(1) == 0      # page 0 only
        kv.kv_cache_read(ex, cache.layer, batch, rows, None, lib=blib)
        torch.cuda.synchronize()
        seen = _report(blib)
        assert seen["what"] == 2 and seen["where"] == 10 and seen["limit"] == 1 and seen["count"] > 0
        kv.paged_attention_scored(ex, cache.layer, batch, q, out, hq, softcap=30.0, lib=blib)
        torch.cuda.synchronize()
        seen = _report(blib)
        assert seen["what"] == 2 and seen["limit"] == 1 and seen["count"] > 0
    blib.warp34_bounds_set_pool_pages(0)
