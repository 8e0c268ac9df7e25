"""Cached rows read back (warp34_kv_cache_read_f16 / _bf16) against their definition in 64 bits.

Tolerance, derived: half a step of the output type and the fp32 arithmetic in front of it: one product (2^-24) for 8-bit rows; for TQ4 rows
eight levels of sums and a product, each rounding off by 2^-24 of a partial sum of |y| / 16, twelve at most: 2^-20 sum |y| / 16."""
import ctypes as C

import numpy as np
import pytest

import rows64
from rows64 import BF16, FP8, Q8, ROW, TQ4, half_step, random_rows, stored, values

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env(native_libs):
    from warp34_b200 import ffi, kv
    return dict(ffi=ffi, kv=kv, lib=native_libs[0])


def _tolerance(rows, fmt, want, dtype):
    with np.errstate(all="ignore"):
        t = half_step(want, dtype) * (1 + 2.0 ** -8)
        return t + (2.0 ** -20 / 16 * np.abs(stored(rows, fmt)).sum(-1, keepdims=True) if fmt == TQ4 else 0)


def _check(got, rows, fmt, dtype, what):
    want = values(rows, fmt)
    got = got.double().cpu().numpy().reshape(want.shape)
    bad = ~(np.abs(got - want) <= _tolerance(rows, fmt, want, dtype))
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size}, first at {np.argwhere(bad)[0]}"


def _pool(kv, name, heads, pages, rng):
    layer = kv.KvLayer(pages, heads, formats=rows64.formats(name))
    host = []
    for slab, fmt in ((layer.k, layer.layout.k_format), (layer.v, layer.layout.v_format)):
        rows = random_rows(fmt, pages * heads * 16, rng).reshape(pages, heads, 16, ROW[fmt])
        slab.copy_(torch.from_numpy(rows.copy()).view(-1))
        host.append(rows)
    return layer, host


def _batch(kv, lens, ctx, table, slots, **kw):
    starts = np.concatenate([[0], np.cumsum(lens)])
    return kv.StepBatch(starts, ctx, np.asarray(ctx) + np.asarray(lens), table, slots, table.shape[1], 0.0625, **kw)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", ["tq4", "fp8", "q8", "q8_fp8", "bf16"])
@pytest.mark.parametrize("heads,lens,ctx", [(1, [1], [0]), (4, [37, 1, 64], [5, 16, 0]), (3, [130], [1000]), (2, [1] * 40, list(range(40)))])
def test_against_the_definition(env, name, dtype, heads, lens, ctx):
    kv, rng = env["kv"], np.random.default_rng(heads + len(lens))
    need = [(c + n + 15) // 16 for c, n in zip(ctx, lens)]
    layer, host = _pool(kv, name, heads, sum(need) + 2, rng)
    table = np.zeros((len(lens), max(need) + 1), np.int32)
    order, at = rng.permutation(sum(need) + 1) + 1, 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    pos = [c + np.arange(n) for c, n in zip(ctx, lens)]
    slots = np.concatenate([table[r, p // 16] * 16 + p % 16 for r, p in enumerate(pos)]).astype(np.int32)
    n, cols = sum(lens), heads * 256
    by_slots, by_table = _batch(kv, lens, ctx, table, slots), _batch(kv, lens, ctx, table, slots)
    by_table.desc.write_slot_mapping = None
    for batch in (by_slots, by_table):
        k, v = (torch.full((n, cols), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        kv.kv_cache_read(kv.Executor(1 << 12), layer, batch, k, v)
        torch.cuda.synchronize()
        for got, rows, fmt in ((k, host[0], layer.layout.k_format), (v, host[1], layer.layout.v_format)):
            _check(got, np.ascontiguousarray(rows[slots >> 4, :, slots & 15]).reshape(n * heads, -1), fmt, dtype, name)


@pytest.mark.parametrize("name", ["tq4", "fp8", "q8", "bf16"])
def test_what_takes_no_part_is_left_alone(env, name):
    """Masked tokens and requests, negative slots, positions outside the table, rows between strided rows; one of the outputs only."""
    kv, rng = env["kv"], np.random.default_rng(4)
    layer, host = _pool(kv, name, 2, 9, rng)
    lens, ctx = [20, 13, 30], [0, 0, 0]
    table = np.array([[1, 2], [3, 4], [5, 6]], np.int32)
    pos = [np.arange(n) for n in lens]
    slots = np.concatenate([table[r, np.minimum(p // 16, 1)] * 16 + p % 16 for r, p in enumerate(pos)]).astype(np.int32)
    slots[7] = -1
    vtm = np.ones(63, np.uint8)
    vtm[[0, 35]] = 0
    vrm = np.array([1, 0, 1], np.uint8)
    batch = _batch(kv, lens, ctx, table, slots, valid_token_mask=vtm, valid_req_mask=vrm)
    kept = [t for t in range(63) if vtm[t] and not 20 <= t < 33 and t != 7]
    for odd in (0, 1):      # 16-byte and 2-byte alignment of the output
        wide = torch.full((63, 512 + 24 + odd), 7.0, dtype=torch.float16, device="cuda")
        out = wide[:, 8 + odd:520 + odd]
        kv.kv_cache_read(kv.Executor(1 << 12), layer, batch, None, out)
        torch.cuda.synchronize()
        _check(out[kept], np.ascontiguousarray(host[1][slots[kept] >> 4, :, slots[kept] & 15]).reshape(-1, host[1].shape[-1]), layer.layout.v_format, torch.float16, name)
        rest = torch.ones(63, dtype=torch.bool, device="cuda")
        rest[kept] = False
        assert (wide[rest] == 7.0).all() and (wide[:, :8 + odd] == 7.0).all() and (wide[:, 520 + odd:] == 7.0).all()
    batch.desc.write_slot_mapping, batch.desc.max_blocks_per_req = None, 1      # the tables end after 16 tokens
    batch.bt = torch.tensor([1, 3, 5], dtype=torch.int32, device="cuda")
    batch.desc.block_tables = batch.bt.data_ptr()
    k = torch.full((63, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    kv.kv_cache_read(kv.Executor(1 << 12), layer, batch, k, None)
    inside = [t for t in range(63) if vtm[t] and (t < 16 or 33 <= t < 49)]
    rest = torch.ones(63, dtype=torch.bool, device="cuda")
    rest[inside] = False
    assert (k[rest] == 7.0).all()
    s = np.array([(16 + t) if t < 16 else 80 + t - 33 for t in inside])
    _check(k[inside], np.ascontiguousarray(host[0][s >> 4, :, s & 15]).reshape(-1, host[0].shape[-1]), layer.layout.k_format, torch.bfloat16, name)


@pytest.mark.parametrize("name", ["tq4", "fp8", "q8", "bf16"])
def test_other_strides_and_pages_beyond_4_gib(env, name):
    """Rows further apart than the canonical packing, aligned as little as the format allows, pages 2^31 bytes apart."""
    kv, ffi, rng = env["kv"], env["ffi"], np.random.default_rng(6)
    fmt = rows64.NAMES[name][0]
    pad = 4 if fmt in (FP8, Q8) else 2
    token, head = ROW[fmt] + pad, 20 * (ROW[fmt] + pad) + pad
    page = (1 << 31) + 4 * 37
    slab = torch.zeros(2 * page + 32768, dtype=torch.uint8, device="cuda")
    layer = kv.KvLayer(1, 2, formats=rows64.formats(name))
    layout = layer.layout
    layout.k_base = layout.v_base = slab.data_ptr() + pad
    layout.k_page_stride_bytes = layout.v_page_stride_bytes = page
    layout.k_head_stride_bytes = layout.v_head_stride_bytes = head
    layout.k_token_stride_bytes = layout.v_token_stride_bytes = token
    rows = random_rows(fmt, 3 * 2 * 16, rng).reshape(3, 2, 16, ROW[fmt])
    for p in range(3):
        for h in range(2):
            at = pad + p * page + h * head
            torch.as_strided(slab, (16, ROW[fmt]), (token, 1), at).copy_(torch.from_numpy(rows[p, h].copy()))
    slots = np.array([0, 15, 16, 33, 47, 40], np.int32)
    batch = _batch(kv, [6], [0], np.zeros((1, 1), np.int32), slots)
    k, v = (torch.zeros(6, 512, dtype=torch.float16, device="cuda") for _ in range(2))
    kv.kv_cache_read(kv.Executor(1 << 12), layer, batch, k, v)
    torch.cuda.synchronize()
    want = np.ascontiguousarray(rows[slots >> 4, :, slots & 15]).reshape(12, -1)
    _check(k, want, fmt, torch.float16, name)
    assert torch.equal(k, v)


def test_special_values_stay_in_their_rows(env):
    kv, rng = env["kv"], np.random.default_rng(2)
    for name in ("tq4", "fp8", "q8", "bf16"):
        layer, host = _pool(kv, name, 1, 2, rng)
        fmt, rows = layer.layout.k_format, host[0]
        if fmt == TQ4:
            rows[1, 0, 3, :2] = np.array([np.nan], np.float16).view(np.uint8)
            rows[1, 0, 5, 66:68] = np.array([0.0], np.float16).view(np.uint8)
        elif fmt == FP8:
            rows[1, 0, 3, 17] = 0x7f
        elif fmt == Q8:
            rows[1, 0, 3, 68:72] = np.array([np.inf], np.float32).view(np.uint8)
        else:
            rows[1, 0, 3, 8:10] = [0x80, 0x7f]
        layer.k.copy_(torch.from_numpy(rows.copy()).view(-1))
        batch = _batch(kv, [16], [0], np.array([[1]], np.int32), np.arange(16, 32, dtype=np.int32))
        k = torch.zeros(16, 256, dtype=torch.bfloat16, device="cuda")
        kv.kv_cache_read(kv.Executor(1 << 12), layer, batch, k, None)
        torch.cuda.synchronize()
        with np.errstate(all="ignore"):
            want = values(rows[1, 0], fmt)
        clean = np.isfinite(want).all(1)
        assert clean.sum() == 15
        _check(k[torch.from_numpy(clean).cuda()], np.ascontiguousarray(rows[1, 0][clean]), fmt, torch.bfloat16, name)
        got = k[3].double().cpu().numpy()
        assert (np.isfinite(got) == np.isfinite(want[3])).all()


@pytest.mark.parametrize("name", ["tq4", "fp8", "q8", "bf16"])
def test_append_then_read_gives_the_rows_within_the_formats_step(env, name):
    """What the append wrote comes back: exactly from BF16, within half a step of the row's scale from 8-bit rows (e4m3: 2^-4 of the value
    or half of its smallest step), and from TQ4 with the codebook's distortion, 0.0094 of the energy (test_tables.py).  That is a mean:
    a single row of 256 columns has no such bound (a coordinate beyond the outermost centroid, 2.7 standard deviations, errs by all that it
    is beyond), so it is taken over the 800 rows.  A column's squared error has a standard deviation of about 1.5 times its mean (uniform
    inside a cell, and the tails), the mean of 204 800 columns one of 0.3 %: 5 % is far outside chance."""
    kv, ffi = env["kv"], env["ffi"]
    heads, n = 4, 100
    layer = kv.KvLayer(9, heads, formats=rows64.formats(name))
    slots = (np.random.default_rng(1).permutation(9 * 16)[:n]).astype(np.int32)
    batch = _batch(kv, [n], [0], np.zeros((1, 7), np.int32), slots)
    g = torch.Generator().manual_seed(3)
    dtype = torch.bfloat16 if name == "bf16" else torch.float16
    x = [torch.randn(n, heads * 256, generator=g).to(dtype).cuda() for _ in range(2)]
    ex = kv.Executor(1 << 12)
    (kv.kv_cache_write_bf16 if name == "bf16" else kv.kv_cache_write)(ex, layer, batch, *x)
    out = [torch.zeros_like(t) for t in x]
    g = torch.cuda.CUDAGraph()
    kv.kv_cache_read(ex, layer, batch, *out)
    torch.cuda.synchronize()
    first = [t.clone() for t in out]
    with torch.cuda.graph(g):
        ex.set_stream()
        kv.kv_cache_read(ex, layer, batch, *out)
    for t in out:
        t.zero_()
    g.replay()
    torch.cuda.synchronize()
    distortion = []
    for a, b, c in zip(x, out, first):
        assert torch.equal(b, c)
        a, b = a.double().view(-1, 256), b.double().view(-1, 256)
        if name == "bf16":
            assert torch.equal(a, b)
        elif name == "tq4":
            distortion.append((((a - b) ** 2).sum(1) / (a ** 2).sum(1)).mean().item())
        elif name == "q8":
            top = a.view(-1, 4, 64).abs().amax(2, keepdim=True)
            assert ((a - b).view(-1, 4, 64).abs() <= top / 127 * 0.502 + b.view(-1, 4, 64).abs() * 2.0 ** -11).all()
        else:
            top = a.view(-1, 2, 128).abs().amax(2, keepdim=True) / 448
            assert ((a - b).view(-1, 2, 128).abs() <= torch.maximum(a.view(-1, 2, 128).abs() * 2.0 ** -4 * 1.01, top * 2.0 ** -10 * 1.01) + b.view(-1, 2, 128).abs() * 2.0 ** -11).all()
    assert name != "tq4" or abs(np.mean(distortion) / 0.009408 - 1) <= 0.05, distortion
