"""Scored attention where its kernels choose by what the call or the cache holds: execution flags that change nothing."""
import pytest

from rows64 import Cache

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env(native_libs):
    from warp34_b200 import ffi, kv
    return dict(ffi=ffi, kv=kv, lib=native_libs[0])


def _queries(name, n, hq, seed, scale=4.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, hq, 256, generator=g) * scale).to(torch.bfloat16 if name == "bf16" else torch.float16).cuda()


def _attend(kv, ex, cache, batch, q, hq, **kw):
    out = torch.full_like(q, 7.0)
    kv.paged_attention_scored(ex, cache.layer, batch, q, out, hq, **kw)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("name,hq,hkv,lens,ctx", [("tq4", 24, 4, [4] * 16, [1200] * 16), ("tq4", 8, 2, [2, 1, 2], [9000, 40, 11000]), ("tq4", 24, 4, [1] * 9, [2000] * 9),
                                                  ("tq4", 8, 2, [70, 5], [90, 0]), ("fp8", 24, 4, [4] * 16, [600] * 16), ("q8", 8, 2, [70, 5], [90, 0]),
                                                  ("bf16", 24, 4, [4] * 16, [1200] * 16), ("bf16", 8, 2, [70, 5], [90, 0])])
def test_flags_of_the_plain_kernels_change_nothing(env, name, hq, hkv, lens, ctx):
    """An executor shared with plain steps that ask for the fast or the tcgen05 kernels: the same kernel, so the same bits."""
    kv, ffi = env["kv"], env["ffi"]
    cache = Cache(name, hkv, lens, ctx, seed=3, tail=0xff)
    q, batch, outs = _queries(name, sum(lens), hq, 4), cache.batch(), []
    for flags in (0, ffi.EXEC_FLAG_FAST_ATTENTION, ffi.EXEC_FLAG_TCGEN05_VERIFY, ffi.EXEC_FLAG_FAST_ATTENTION | ffi.EXEC_FLAG_TCGEN05_VERIFY):
        ex = kv.Executor(64 << 20)
        ex.ex.flags = flags
        outs.append(_attend(kv, ex, cache, batch, q, hq, softcap=30.0))
        assert ex.ex.flags == flags
    for out in outs[1:]:
        assert torch.equal(outs[0], out)
