"""Scored attention where its kernels choose by what the call or the cache holds: execution flags that change nothing, V rows of any magnitude,
NaN that a token sees and NaN that it does not."""
import numpy as np
import pytest

from rows64 import Cache, half_step, scored_attention

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


SHARE = {"tq4": 2.0 ** -11, "fp8": 2.0 ** -12, "q8": 2.0 ** -12, "bf16": 2.0 ** -12}      # of sum_k weight_k |V_k|, as test_gpu_scored_attention.py derives it


def _check(name, out, want, size, rows=None):
    got = out.double().cpu().numpy()
    tol = half_step(want, out.dtype) * (1 + 2.0 ** -8) + SHARE[name] * size
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got - want) <= tol)
    if rows is not None:
        bad = bad & rows
    assert not bad.any(), f"{name}: {bad.sum()} of {bad.size} outside, worst {np.nanmax(np.abs(got - want) / tol):.2f} x, first {np.argwhere(bad)[0]}"


def _microseconds(call):
    """The fastest of five calls, by the device's clock."""
    call()
    times = []
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return min(times)


def _scale_v(cache, powers):
    """V rows times 2^powers [pages, heads, 16] (whole numbers; never-written rows keep their pattern)."""
    rows = cache.rows[1]
    if cache.name == "fp8":
        d = rows[..., 256:]
    else:
        d = rows.reshape(*rows.shape[:3], 4, 68)[..., :4]
    f = np.ascontiguousarray(d).view(np.float32)
    f = np.where(np.isfinite(f), f * np.exp2(np.broadcast_to(powers, rows.shape[:3]))[(...,) + (None,) * (f.ndim - 3)], f).astype(np.float32)
    d[...] = f.view(np.uint8).reshape(d.shape)
    cache.upload()


STREAM = {"decode": (24, 4, [1] * 6, [255, 1, 90, 1000, 47, 48]), "verify": (16, 4, [3, 2, 4, 4, 4, 3], [40, 500, 0, 60, 100, 7])}


@pytest.mark.parametrize("power", [-14, -10, 12, "mixed"])
@pytest.mark.parametrize("shape", list(STREAM))
@pytest.mark.parametrize("name", ["fp8", "q8"])
def test_8_bit_values_of_any_magnitude(env, name, shape, power):
    """V rows far from 1, all of them or each its own way: the share of sum_k weight_k |V_k| that is off does not depend on it."""
    kv = env["kv"]
    hq, hkv, lens, ctx = STREAM[shape]
    cache = Cache(name, hkv, lens, ctx, seed=7, tail=0xff)
    _scale_v(cache, np.random.default_rng(1).integers(-12, 13, cache.rows[1].shape[:3]) if power == "mixed" else power)
    q = _queries(name, sum(lens), hq, 8)
    out = _attend(kv, kv.Executor(64 << 20), cache, cache.batch(), q, hq, softcap=20.0)
    want, size = scored_attention(cache, q.float().cpu().numpy(), hq, softcap=20.0)
    _check(name, out, want, size)


@pytest.mark.parametrize("name", ["fp8", "q8"])
def test_8_bit_values_beside_much_larger_ones(env, name):
    """Drafted tokens of two documents in one group of rows: V rows 2^40 times larger in the one take nothing from the other, and a row of
    that size with a weight near zero nothing from the rest."""
    kv = env["kv"]
    hq, hkv, lens, ctx = 16, 4, [4] * 6, [58, 59, 158, 157, 57, 56]
    cache = Cache(name, hkv, lens, ctx, seed=9, tail=0xff)
    pos = np.concatenate([c + np.arange(m) for c, m in zip(ctx, lens)])
    key_begin = (pos // 60 * 60).astype(np.int32)
    powers = np.zeros(cache.rows[1].shape[:3], np.int64)
    for r in range(len(lens)):
        for k in range(ctx[r] // 60 * 60, min((ctx[r] // 60 + 1) * 60, ctx[r] + lens[r])):      # the document of the request's first new token
            powers[cache.table[r, k // 16], :, k % 16] = 40
    _scale_v(cache, powers)
    q = _queries(name, sum(lens), hq, 10)
    out = _attend(kv, kv.Executor(64 << 20), cache, cache.batch(), q, hq, softcap=20.0, key_begin=torch.from_numpy(key_begin).cuda())
    want, size = scored_attention(cache, q.float().cpu().numpy(), hq, softcap=20.0, key_begin=key_begin)
    small = np.abs(want).max(-1, keepdims=True) < 1e3
    assert small.any() and not small.all()
    _check(name, out, want, size, rows=np.broadcast_to(small, want.shape))
    # one such row, 2000 keys away from a query whose slope leaves it exp(-200)
    cache = Cache(name, hkv, [1] * 6, [2100] * 6, seed=12, tail=0xff)
    powers = np.zeros(cache.rows[1].shape[:3], np.int64)
    powers[cache.table[:, 6], :, 4] = 40      # position 100
    _scale_v(cache, powers)
    q, slopes = _queries(name, 6, hq, 13), np.full(hq, 0.1, np.float32)
    out = _attend(kv, kv.Executor(64 << 20), cache, cache.batch(), q, hq, softcap=20.0, slopes=torch.from_numpy(slopes).cuda())
    want, size = scored_attention(cache, q.float().cpu().numpy(), hq, softcap=20.0, slopes=slopes)
    _check(name, out, want, size)


@pytest.mark.parametrize("name", ["fp8", "q8"])
def test_large_8_bit_values_take_no_longer(env, name):
    kv = env["kv"]
    hq, hkv, lens, ctx = 16, 4, [1] * 16, [8000] * 16
    ex, q, times = kv.Executor(64 << 20), _queries(name, 16, hq, 11), []
    for power in (0, 12):
        cache = Cache(name, hkv, lens, ctx, seed=10)
        _scale_v(cache, power)
        batch, out = cache.batch(), torch.zeros_like(q)
        times.append(_microseconds(lambda: kv.paged_attention_scored(ex, cache.layer, batch, q, out, hq, softcap=20.0)))
    assert times[1] < 3 * times[0], times


def _spoil_v(cache, r, pos, channels, value=np.nan):
    """V of every head at `pos` of request r: `value` in the channels (8-bit rows: NaN codes; Q8_0 and TQ4: a scale)."""
    rows = cache.rows[1][cache.table[r, pos // 16], :, pos % 16]
    if cache.name == "bf16":
        rows.view(np.uint16)[:, channels] = 0x7fc0 if np.isnan(value) else 0x7f80
    elif cache.name == "fp8":
        rows[:, channels] = 0x7f
    elif cache.name == "q8":
        rows[:, 68:72] = np.array([value], np.float32).view(np.uint8)
    else:
        rows[:, :2] = np.array([value], np.float16).view(np.uint8)


SPOILED = {"decode": (24, 4, [1] * 6, [255, 100, 90, 1000, 47, 48]), "decode_long": (8, 2, [1, 1, 1], [30000, 9000, 40]),
           "verify": (16, 4, [3, 2, 4, 4, 4, 3], [40, 500, 60, 60, 100, 37]), "chunk": (8, 2, [150, 64, 33], [90, 40, 260]), "chunk_cut": (2, 1, [40], [3000]),
           "verify_long": (4, 1, [4, 2, 4], [21900, 40, 900])}


@pytest.mark.parametrize("shape", list(SPOILED))
@pytest.mark.parametrize("name", ["tq4", "fp8", "q8", "bf16"])
def test_channels_without_a_nan_keep_their_results(env, name, shape):
    """NaN in one channel of a V row of the prefix, which every token sees, and in another channel of a row that only later tokens see: each
    token is off in the channels of its own keys and in no other (TQ4, whose channels share their scales: in no other token)."""
    kv = env["kv"]
    hq, hkv, lens, ctx = SPOILED[shape]
    cache = Cache(name, hkv, lens, ctx, seed=21, tail=0xff)
    q = _queries(name, sum(lens), hq, 22)
    for r in range(len(lens)):
        if r % 3 != 2 and not (name == "tq4" and len(lens) == 1):      # (some token stays whole)
            _spoil_v(cache, r, min(37, ctx[r] - 1), [5])
        if lens[r] > 1:
            _spoil_v(cache, r, ctx[r] + lens[r] // 2, [9, 200])
    cache.upload()
    out = _attend(kv, kv.Executor(64 << 20), cache, cache.batch(), q, hq, softcap=20.0)
    want, size = scored_attention(cache, q.float().cpu().numpy(), hq, softcap=20.0)
    finite = np.isfinite(want)
    assert finite.any() and not finite.all()
    _check(name, out, want, size, rows=finite)
    assert torch.isnan(out.cpu()[torch.from_numpy(~finite)]).all()


@pytest.mark.parametrize("where", ["prefix", "newest"])
@pytest.mark.parametrize("name,hq,hkv,lens,ctx", [("bf16", 24, 4, [700], [2048]), ("tq4", 16, 4, [700], [2048]), ("q8", 16, 4, [500, 300], [1000, 40]),
                                                  ("fp8", 16, 4, [1] * 16, [8000] * 16), ("tq4", 24, 4, [1] * 32, [8000] * 32), ("bf16", 16, 4, [4] * 16, [6000] * 16),
                                                  ("tq4", 8, 2, [100], [20000])])
def test_a_nan_that_every_row_sees_is_no_standstill(env, name, hq, hkv, lens, ctx, where):
    """One NaN in the V of a cached prefix makes every row NaN: such rows are not computed a second time, key by key (which took up to 700 times
    as long as the call).  What is left is a look at the keys."""
    kv = env["kv"]
    cache = Cache(name, hkv, lens, ctx, seed=23)
    q, batch, ex = _queries(name, sum(lens), hq, 24), cache.batch(), kv.Executor(64 << 20)
    out = torch.zeros_like(q)
    call = lambda: kv.paged_attention_scored(ex, cache.layer, batch, q, out, hq, softcap=20.0)  # noqa: E731
    clean = _microseconds(call)
    for r in range(len(lens)):
        _spoil_v(cache, r, 5 if where == "prefix" else ctx[r] - 1, [7])
    cache.upload()
    spoiled = _microseconds(call)
    assert torch.isnan(out).any(-1).all()
    assert spoiled < 20 * clean, (clean, spoiled)


@pytest.mark.parametrize("name,hq,hkv,lens,ctx,times", [("tq4", 16, 4, [2048], [2048], 110), ("tq4", 8, 2, [100], [20000], 400), ("bf16", 16, 4, [4] * 16, [6000] * 16, 60)])
def test_a_nan_among_the_new_tokens_is_bounded(env, name, hq, hkv, lens, ctx, times):
    """One NaN in the V of a token in the middle of the chunk: the rows of its tile that come before it are computed again, key by key, at most
    128 rows to a CTA.  (Keys one after the other made the first two 186 and 1100 times as long as the call without NaN, now 56 and 150.)"""
    kv = env["kv"]
    cache = Cache(name, hkv, lens, ctx, seed=25)
    q, batch, ex = _queries(name, sum(lens), hq, 26), cache.batch(), kv.Executor(64 << 20)
    out = torch.zeros_like(q)
    call = lambda: kv.paged_attention_scored(ex, cache.layer, batch, q, out, hq, softcap=20.0)  # noqa: E731
    clean = _microseconds(call)
    first = out.clone()
    at = lens[0] // 2 + (20 if lens[0] > 50 else 0)
    _spoil_v(cache, 0, ctx[0] + at, [7])
    cache.upload()
    spoiled = _microseconds(call)
    eps = torch.finfo(q.dtype).eps
    assert ((out[:at].double() - first[:at].double()).abs() <= 2 * eps * first[:at].double().abs() + 2 * SHARE[name] * 1.2).all()      # two roundings, two shares
    assert torch.isnan(out[at:lens[0]]).any(-1).all() and not torch.isnan(out[lens[0]:]).any()
    assert spoiled < times * clean, (clean, spoiled)


@pytest.mark.parametrize("shape", list(STREAM))
@pytest.mark.parametrize("name", ["fp8", "q8"])
def test_8_bit_values_behind_zero_rows(env, name, shape):
    """The newest keys, which are met first, hold V rows of zeros or next to it, the others ordinary ones; and the other way about."""
    kv = env["kv"]
    hq, hkv, lens, ctx = STREAM[shape]
    for newest, power in ((True, -2000), (True, -130), (False, -2000)):
        cache = Cache(name, hkv, lens, ctx, seed=14, tail=0xff)
        powers = np.zeros(cache.rows[1].shape[:3])
        for r, (c, m) in enumerate(zip(ctx, lens)):
            pos = np.arange(max(c + m - 37, 0), c + m) if newest else np.arange(0, max(c + m - 37, 0))
            powers[cache.table[r, pos // 16], :, pos % 16] = power
        _scale_v(cache, powers)
        q = _queries(name, sum(lens), hq, 15)
        out = _attend(kv, kv.Executor(64 << 20), cache, cache.batch(), q, hq, softcap=20.0)
        want, size = scored_attention(cache, q.float().cpu().numpy(), hq, softcap=20.0)
        _check(name, out, want, size)
