"""Attention with changed scores (warp34_paged_attention_scored_f16 / _bf16) against its definition in 64 bits.

Tolerance, derived: half a step of the output type at the output, and a share of sum_k weight_k |V_k| for what happens to weights and values
in front of it.  The tests' scores have sum |q k| sm_scale of about 40.
  TQ4     scores to 2.1e-6 of sum |q k|, a weight and the mass each off by 8e-5: 1.6e-4 of sum_k weight_k |V_k|; value centroids to 9.5e-5
          (residuals are left out where no key holds a quarter of the mass), an error in the rotated basis (rows64.scored_attention
          says what of): 4 x 9.5e-5.  2^-11 = 4.9e-4 of both.
  8-bit   exact operands; scores summed in fp32 (40 x 2^-20), weights carried in 22 bits: below 1e-4.  2^-12.
  BF16    exact operands; weights as bf16 value and residual, 2^-17; scores as above: below 1e-4.  2^-12.
The cap adds 1.5 x 2^-23 of itself (9e-6 at 50), the distance a rounding of a number up to 2^10 (6e-5), both in the scores; the fp32 kernel
stays inside the same."""
import ctypes as C

import numpy as np
import pytest

import rows64
from rows64 import Cache, half_step, scored_attention

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
SHARE = {"tq4": 2.0 ** -11, "fp8": 2.0 ** -12, "q8": 2.0 ** -12, "q8_fp8": 2.0 ** -12, "bf16": 2.0 ** -12}
FORMATS = ["tq4", "fp8", "q8", "bf16"]


@pytest.fixture(scope="module")
def env(native_libs):
    from warp34_b200 import ffi, kv
    return dict(ffi=ffi, kv=kv, lib=native_libs[0], ex=kv.Executor(64 << 20))


def _dtype(name):
    return torch.bfloat16 if name == "bf16" else torch.float16


def _queries(name, n, hq, seed, scale=4.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, hq, 256, generator=g) * scale).to(_dtype(name))


def _slopes(hq):
    return (2.0 ** (-8.0 * np.arange(1, hq + 1) / hq)).astype(np.float32)


def _call(kv, ex, cache, batch, q, hq, out=None, softcap=0.0, slopes=None, key_begin=None, key_end=None):
    dev = lambda a: None if a is None else torch.as_tensor(a).cuda()  # noqa: E731
    out = torch.full_like(q, 7.0).cuda() if out is None else out
    ex.set_stream()
    kv.paged_attention_scored(ex, cache.layer, batch, q.cuda(), out, hq, softcap=softcap, slopes=dev(slopes), key_begin=dev(key_begin), key_end=dev(key_end))
    torch.cuda.synchronize()
    return out


def _check(name, out, want, size, dtype, rows=None):
    got = out.double().cpu().numpy()
    tol = half_step(want, dtype) * (1 + 2.0 ** -8) + SHARE[name] * size
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got - want) <= tol)
    if rows is not None:
        bad = bad[rows]
    assert not bad.any(), f"{name}: {bad.sum()} of {bad.size} outside, worst {np.nanmax(np.abs(got - want) / tol):.2f} x, first {np.argwhere(bad)[0]}"


SHAPES = {
    "one": (24, 4, [1], [316]),
    "first_token": (4, 1, [1], [0]),
    "four_rows": (16, 4, [1, 1, 1], [0, 15, 700]),
    "gqa1": (3, 3, [1, 1, 1, 1, 1], [4, 100, 31, 32, 33]),
    "verify": (6, 1, [3, 2, 4], [40, 500, 0]),
    "verify_wide": (8, 4, [5, 5], [61, 130]),
    "chunks": (8, 2, [70, 5, 33], [90, 0, 260]),
    "chunk_alone": (6, 2, [129], [333]),
    "many": (24, 4, [1] * 9 + [30], [7 * i for i in range(9)] + [20]),
    # more than a few tokens, or long ones: the stream kernels
    "stream_four_rows": (16, 4, [1] * 9, [0, 15, 700, 33, 64, 129, 5, 16, 31]),
    "stream_six_rows": (24, 4, [1] * 6, [255, 1, 90, 1000, 47, 48]),
    "stream_gqa1": (3, 3, [1] * 9, [4, 100, 31, 32, 33, 0, 511, 62, 63]),
    "stream_verify": (6, 1, [3, 2, 4, 4, 4, 3], [40, 500, 0, 60, 100, 7]),
    "stream_long": (6, 1, [1], [33000]),
    "stream_six_rows_long": (24, 4, [1] * 5, [2047, 255, 90, 1000, 47]),
    "stream_long_batch": (16, 4, [1] * 9, [2047, 5, 64, 1000, 33, 700, 129, 300, 16]),
    "stream_long_verify": (4, 1, [4, 2, 4], [21900, 40, 900]),
    # a few tokens over short contexts: one launch
    "small_eight_rows": (8, 1, [1, 2], [1020, 100]),
    "small_five_rows": (5, 1, [2, 1], [100, 255]),
    "small_two_rows": (4, 2, [1, 1, 2], [300, 0, 77]),
}
CHANGES = ["none", "cap", "distance", "window", "ranges", "all"]


def _change(kind, hq, lens, ctx, seed):
    """Keyword arguments of the call, and the window."""
    rng = np.random.default_rng(seed)
    n = sum(lens)
    pos = np.concatenate([c + np.arange(m) for c, m in zip(ctx, lens)])
    kw, window = {}, 0
    if kind in ("cap", "all"):
        kw["softcap"] = 30.0 if kind == "cap" else 5.0
    if kind in ("distance", "all"):
        kw["slopes"] = _slopes(hq)
    if kind in ("window", "all"):
        window = 50
    if kind in ("ranges", "all"):      # documents, prefixes, and tokens without keys
        kw["key_begin"] = (pos // 37 * 37).astype(np.int32)
        kw["key_end"] = np.where(rng.random(n) < 0.3, pos + rng.integers(-40, 60, n), pos + 1).astype(np.int32)
        empty = rng.random(n) < 0.15
        kw["key_begin"][empty] = rng.choice([2 ** 31 - 1, 100000], empty.sum())
        kw["key_end"][rng.random(n) < 0.05] = -2 ** 31
        kw["key_end"][rng.random(n) < 0.05] = 2 ** 31 - 1
    return kw, window


@pytest.mark.parametrize("kind", CHANGES)
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("name", FORMATS)
def test_against_the_definition(env, name, shape, kind):
    hq, hkv, lens, ctx = SHAPES[shape]
    cache = Cache(name, hkv, lens, ctx, seed=len(shape), tail=0xff)
    kw, window = _change(kind, hq, lens, ctx, 3)
    q = _queries(name, sum(lens), hq, 11)
    out = _call(env["kv"], env["ex"], cache, cache.batch(sliding_window=window), q, hq, **kw)
    want, size = scored_attention(cache, q.float().numpy(), hq, window=window, **kw)
    _check(name, out, want, size, q.dtype)
    assert int(env["ex"].scratch[:4].view(torch.int32).item()) == 0


@pytest.mark.parametrize("name", FORMATS)
def test_symmetric_window_and_negative_scale(env, name):
    hq, hkv, lens, ctx = 4, 2, [40, 3], [70, 20]
    cache = Cache(name, hkv, lens, ctx, seed=5, tail=0xff)
    q = _queries(name, sum(lens), hq, 12)
    for kw in (dict(mask_mode=env["ffi"].ATTN_MASK_SYMMETRIC_WINDOW, sliding_window=25), dict(sm_scale=-1.0 / 32), dict(sm_scale=0.0)):
        batch = cache.batch(**kw)
        out = _call(env["kv"], env["ex"], cache, batch, q, hq, softcap=8.0, slopes=_slopes(hq))
        want, size = scored_attention(cache, q.float().numpy(), hq, sm_scale=kw.get("sm_scale", 1.0 / 16), softcap=8.0, slopes=_slopes(hq),
                                      window=kw.get("sliding_window", 0), symmetric="mask_mode" in kw)
        _check(name, out, want, size, q.dtype)


@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("shape", ["four_rows", "verify", "chunks", "stream_four_rows", "stream_verify", "stream_long_batch"])
def test_masked_rows_are_left_alone(env, name, shape):
    hq, hkv, lens, ctx = SHAPES[shape]
    cache = Cache(name, hkv, lens, ctx, seed=8, tail=0xff)
    n = sum(lens)
    vtm = np.ones(n, np.uint8)
    vtm[0] = 0
    vrm = np.ones(len(lens), np.uint8)
    vrm[1] = 0
    q = _queries(name, n, hq, 13)
    kw, _ = _change("ranges", hq, lens, ctx, 7)
    out = _call(env["kv"], env["ex"], cache, cache.batch(valid_token_mask=vtm, valid_req_mask=vrm), q, hq, softcap=20.0, **kw)
    want, size = scored_attention(cache, q.float().numpy(), hq, softcap=20.0, **kw)
    starts = np.concatenate([[0], np.cumsum(lens)])
    on = vtm.astype(bool)
    on[starts[1]:starts[2]] = False
    assert (out[torch.from_numpy(~on).cuda()] == 7.0).all()
    _check(name, out, want, size, q.dtype, rows=on)


@pytest.mark.parametrize("how", ["no_scratch", "precise", "strides"])
@pytest.mark.parametrize("name", FORMATS + ["q8_fp8"])
def test_the_row_kernel(env, name, how):
    """Calls without workspace, with the precise flag, of a packing the tensor-core kernels do not take, and mixed 8-bit formats."""
    kv, ffi = env["kv"], env["ffi"]
    hq, hkv, lens, ctx = 6, 2, [1, 30, 2], [45, 17, 0]
    cache = Cache(name, hkv, lens, ctx, seed=21, tail=0xff)
    ex = kv.Executor(64 << 20)
    if how == "no_scratch":
        ex.ex.scratch_ptr, ex.ex.scratch_size = 0, 0
    elif how == "precise":
        ex.ex.flags = ffi.EXEC_FLAG_PRECISE_ATTENTION
    else:      # rows one alignment unit further apart
        keep = []
        for side, slab in enumerate(("k", "v")):
            fmt = rows64.NAMES[name][side]
            token = rows64.ROW[fmt] + (4 if fmt in (rows64.FP8, rows64.Q8) else 2)
            head, page = 16 * token + 4, hkv * (16 * token + 4) + 8
            pages = cache.rows[side].shape[0]
            raw = torch.zeros(pages * page + 64, dtype=torch.uint8, device="cuda")
            torch.as_strided(raw, cache.rows[side].shape, (page, head, token, 1), 4).copy_(torch.from_numpy(cache.rows[side].copy()))
            keep.append(raw)
            setattr(cache.layer.layout, f"{slab}_base", raw.data_ptr() + 4)
            for what, v in (("page", page), ("head", head), ("token", token)):
                setattr(cache.layer.layout, f"{slab}_{what}_stride_bytes", v)
    q = _queries(name, sum(lens), hq, 14)
    for kind in ("cap", "all"):
        kw, window = _change(kind, hq, lens, ctx, 9)
        out = _call(kv, ex, cache, cache.batch(sliding_window=window), q, hq, **kw)
        want, size = scored_attention(cache, q.float().numpy(), hq, window=window, **kw)
        _check(name, out, want, size, q.dtype)


@pytest.mark.parametrize("name", ["tq4"])
@pytest.mark.parametrize("shape", ["one", "verify", "chunks", "stream_six_rows", "stream_six_rows_long", "stream_long_verify"])
def test_bf16_activations_over_tq4(env, name, shape):
    hq, hkv, lens, ctx = SHAPES[shape]
    cache = Cache(name, hkv, lens, ctx, seed=8, tail=0xff)
    q = _queries(name, sum(lens), hq, 15).to(torch.bfloat16)
    kw, window = _change("all", hq, lens, ctx, 5)
    out = _call(env["kv"], env["ex"], cache, cache.batch(sliding_window=window), q, hq, **kw)
    want, size = scored_attention(cache, q.float().numpy(), hq, window=window, **kw)
    _check(name, out, want, size, torch.bfloat16)


def _spoil(cache, r, pos, side, value):
    """Makes the row of every head at `pos` of request r hold NaN or infinity."""
    fmt = rows64.NAMES[cache.name][side]
    page, off = cache.table[r, pos // 16], pos % 16
    row = cache.rows[side][page, :, off]
    if fmt == rows64.TQ4:
        row[:, :2] = np.array([value], np.float16).view(np.uint8)
    elif fmt == rows64.FP8:
        if np.isnan(value):
            row[:, 5] = 0x7f
        else:
            row[:, 256:260] = np.array([value], np.float32).view(np.uint8)
    elif fmt == rows64.Q8:
        row[:, 68:72] = np.array([value], np.float32).view(np.uint8)
    else:
        row[:, 20:22] = [0x80, 0x7f] if np.isinf(value) else [0xc0, 0x7f]


@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("shape", ["decode", "verify", "chunk", "chunk_cut", "stream_verify", "stream_long_verify"])
@pytest.mark.parametrize("name", FORMATS)
def test_non_finite_rows_reach_only_the_rows_that_see_them(env, name, shape, side, value):
    """A NaN or infinity in K or V of one document: tokens of the others, in the same tile, have the results they would have without it."""
    hq, hkv, lens, ctx = {"decode": (4, 2, [1, 1], [60, 61]), "verify": (4, 1, [4, 2], [58, 60]), "chunk": (4, 2, [90, 64], [33, 0]),
                          "chunk_cut": (2, 1, [40], [2000]), "stream_verify": (4, 1, [4, 2, 4, 4, 4, 4, 4], [58, 60, 57, 58, 59, 58, 57]),
                          "stream_long_verify": (4, 1, [4, 4, 4], [21998, 19998, 30])}[shape]
    cache = Cache(name, hkv, lens, ctx, seed=31, tail=0xff)
    q = _queries(name, sum(lens), hq, 16)
    pos = np.concatenate([c + np.arange(m) for c, m in zip(ctx, lens)])
    doc = {"decode": 61, "verify": 60, "chunk": 50, "chunk_cut": 2010, "stream_verify": 60, "stream_long_verify": 2000}[shape]
    key_begin, key_end = (pos // doc * doc).astype(np.int32), (pos + 1).astype(np.int32)
    clean, size = scored_attention(cache, q.float().numpy(), hq, softcap=30.0, key_begin=key_begin, key_end=key_end)
    spoiled = {"decode": 10, "verify": 59, "chunk": 49, "chunk_cut": 2004, "stream_verify": 59, "stream_long_verify": 21999}[shape]
    for r in range(len(lens)):
        _spoil(cache, r, min(spoiled, ctx[r] + lens[r] - 1), side, value)
    cache.upload()
    want, _ = scored_attention(cache, q.float().numpy(), hq, softcap=30.0, key_begin=key_begin, key_end=key_end)
    out = _call(env["kv"], env["ex"], cache, cache.batch(), q, hq, softcap=30.0, key_begin=key_begin, key_end=key_end)
    at, unseen = 0, np.zeros(sum(lens), bool)
    for r, (c, m) in enumerate(zip(ctx, lens)):
        p = min(spoiled, c + m - 1)
        unseen[at:at + m] = ~((key_begin[at:at + m] <= p) & (p < key_end[at:at + m]))
        at += m
    assert unseen.any() and not unseen.all()
    _check(name, out, clean, size, q.dtype, rows=unseen)
    got = out.double().cpu().numpy()
    if side == 0 and np.isinf(value):
        return      # an infinite score is the cap's business: finite or not as the sign falls
    seen = ~unseen
    finite = np.isfinite(want)
    assert (np.isfinite(got[seen]) <= finite[seen]).all()      # nothing finite where the definition has NaN or infinity


@pytest.mark.parametrize("name", FORMATS)
def test_less_workspace_gives_the_same_results(env, name):
    """A workspace for part of the requests at a time, and one that holds nothing but the row kernel's needs."""
    kv = env["kv"]
    hq, hkv, lens, ctx = 24, 4, [1] * 40, [7 * i for i in range(40)]
    cache = Cache(name, hkv, lens, ctx, seed=41, tail=0xff)
    q = _queries(name, 40, hq, 17)
    kw, window = _change("all", hq, lens, ctx, 6)
    want, size = scored_attention(cache, q.float().numpy(), hq, window=window, **kw)
    for scratch in (2 << 20, 600 << 10, 1 << 12):
        out = _call(kv, kv.Executor(scratch), cache, cache.batch(sliding_window=window), q, hq, **kw)
        _check(name, out, want, size, q.dtype)
    batch = cache.batch(sliding_window=window)
    need = env["lib"].warp34_paged_attention_scored_scratch_bytes(C.byref(cache.layer.layout), C.byref(batch.desc), hq)
    assert need > 600 << 10
    out = _call(kv, kv.Executor(int(need)), cache, batch, q, hq, **kw)
    _check(name, out, want, size, q.dtype)


@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("shape", ["four_rows", "chunks", "stream_six_rows", "stream_long_batch"])
def test_capture_replay_streams_and_repeatability(env, name, shape):
    kv = env["kv"]
    hq, hkv, lens, ctx = SHAPES[shape]
    cache = Cache(name, hkv, lens, ctx, seed=51, tail=0xff)
    q = _queries(name, sum(lens), hq, 18).cuda()
    kw, window = _change("all", hq, lens, ctx, 4)
    dev = {k: torch.as_tensor(v).cuda() if not isinstance(v, float) else v for k, v in kw.items()}
    batch = cache.batch(sliding_window=window)
    ex = kv.Executor(64 << 20)
    first = _call(kv, ex, cache, batch, q, hq, **dev)
    again = _call(kv, ex, cache, batch, q, hq, **dev)
    assert torch.equal(first, again)
    side = torch.cuda.Stream()
    ex2 = kv.Executor(64 << 20, stream=side)
    out2 = torch.zeros_like(q)
    side.wait_stream(torch.cuda.current_stream())
    kv.paged_attention_scored(ex2, cache.layer, batch, q, out2, hq, **dev)
    side.synchronize()
    assert torch.equal(first, out2)
    # two captured steps with a workspace each, replayed on two streams at once
    graphs, outs = [], []
    for i in range(2):
        exg, out = kv.Executor(64 << 20), torch.zeros_like(q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            exg.set_stream()
            kv.paged_attention_scored(exg, cache.layer, batch, q, out, hq, **dev)
        graphs.append((g, exg))
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
    # the limits are read at every replay
    dev["key_end"].fill_(0)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert (outs[0] == 0).all()


@pytest.mark.parametrize("name,hq,hkv,lens,ctx", [("tq4", 16, 4, [1], [150001]), ("bf16", 24, 4, [1, 4], [40000, 20011]), ("fp8", 8, 2, [1] * 3, [9000, 70000, 31]),
                                                  ("tq4", 8, 2, [200], [30000]), ("bf16", 8, 2, [200], [30000]), ("q8", 24, 4, [300, 1, 1], [3000, 5000, 64])])
def test_long_contexts_agree_with_the_row_kernel(env, name, hq, hkv, lens, ctx):
    """Long contexts (hundreds of partials to a row, chunks cut into key ranges, both kernels of a mixed 8-bit batch): against the fp32
    kernel, which the tests above hold to the definition; its own error comes on top, hence twice the share."""
    kv, ffi = env["kv"], env["ffi"]
    cache = Cache(name, hkv, lens, ctx, seed=61)
    q = _queries(name, sum(lens), hq, 19, scale=6.0)
    pos = np.concatenate([c + np.arange(m) for c, m in zip(ctx, lens)])
    precise = kv.Executor(1 << 20)
    precise.ex.flags = ffi.EXEC_FLAG_PRECISE_ATTENTION
    for kw in (dict(softcap=50.0), dict(slopes=_slopes(hq) * 0.01, softcap=30.0), dict(key_begin=(pos // 4999 * 4999).astype(np.int32), key_end=np.maximum(pos + 1, 7000).astype(np.int32))):
        out = _call(kv, env["ex"], cache, cache.batch(), q, hq, **kw).double()
        ref = _call(kv, precise, cache, cache.batch(), q, hq, **kw).double()
        tol = torch.from_numpy(half_step(ref.cpu().numpy(), q.dtype)).cuda() * 4 + 2 * SHARE[name] * 1.2      # mean |V| is below 1.2
        bad = ~((out - ref).abs() <= tol)
        assert not bad.any(), f"{int(bad.sum())} outside, worst {float((out - ref).abs().max()):.2e}"


def test_a_layer_from_projection_to_attention(env):
    """The operators together, as a layer runs them: packed projection rows -> norm and rotation -> append -> attention with capped scores
    over documents; then the prefix read back and appended to a layer of another format, which gives the same attention up to that
    format's steps."""
    kv = env["kv"]
    hq, hkv, n, ctx = 8, 2, 24, 200
    g = torch.Generator().manual_seed(3)
    ex = kv.Executor(64 << 20)
    wl = (torch.randn(ctx + n, hq * 512 + 2 * hkv * 256, generator=g)).to(torch.bfloat16).cuda()
    q_in, k_in, v_in = wl[:, :hq * 512].view(-1, hq, 512), wl[:, hq * 512:hq * 512 + hkv * 256].view(-1, hkv, 256), wl[:, hq * 512 + hkv * 256:]
    w = [(torch.randn(256, generator=g) * 0.2).to(torch.bfloat16).cuda() for _ in range(2)]
    inv = (1e4 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)).float().cuda()
    pos = torch.arange(ctx + n, dtype=torch.int32, device="cuda")
    q, k, gate = (torch.zeros(ctx + n, h, 256, dtype=torch.bfloat16, device="cuda") for h in (hq, hkv, hq))
    kv.qk_norm_rope(ex, q_in, k_in, w[0], w[1], pos, inv, q, k, gate_out=gate)
    assert torch.equal(gate, q_in[..., 256:])
    cache = Cache("bf16", hkv, [ctx + n], [0], seed=1)
    slots = cache.table[0, np.arange(ctx + n) // 16] * 16 + np.arange(ctx + n) % 16
    fill = kv.StepBatch([0, ctx + n], [0], [ctx + n], cache.table, slots, cache.table.shape[1], 1 / 16)
    v_in = v_in.contiguous()      # (this append takes one row stride for K and V)
    kv.kv_cache_write_bf16(ex, cache.layer, fill, k.view(-1, hkv * 256), v_in)
    step = kv.StepBatch([0, n], [ctx], [ctx + n], cache.table, slots[ctx:], cache.table.shape[1], 1 / 16)
    key_begin = ((ctx + np.arange(n)) // 110 * 110).astype(np.int32)
    out = torch.zeros(n, hq, 256, dtype=torch.bfloat16, device="cuda")
    ranges = dict(key_begin=torch.from_numpy(key_begin).cuda(), softcap=30.0)
    kv.paged_attention_scored(ex, cache.layer, step, q[ctx:].contiguous(), out, hq, **ranges)
    torch.cuda.synchronize()
    for side, slab in enumerate((cache.layer.k, cache.layer.v)):
        cache.rows[side] = slab.cpu().numpy().reshape(cache.rows[side].shape)
    cache.lens, cache.ctx = [n], [ctx]
    want, size = scored_attention(cache, q[ctx:].float().cpu().numpy(), hq, softcap=30.0, key_begin=key_begin)
    _check("bf16", out, want, size, torch.bfloat16)
    # the prefix moves to an 8-bit layer
    kr, vr = (torch.zeros(ctx + n, hkv * 256, dtype=torch.float16, device="cuda") for _ in range(2))
    kv.kv_cache_read(ex, cache.layer, fill, kr, vr)
    assert torch.equal(kr, k.view(-1, hkv * 256).half()) and torch.equal(vr, v_in.half())
    other = Cache("q8", hkv, [n], [ctx], seed=2)
    slots8 = other.table[0, np.arange(ctx + n) // 16] * 16 + np.arange(ctx + n) % 16
    kv.kv_cache_write(ex, other.layer, kv.StepBatch([0, ctx + n], [0], [ctx + n], other.table, slots8, other.table.shape[1], 1 / 16), kr, vr)
    out8 = torch.zeros(n, hq, 256, dtype=torch.float16, device="cuda")
    step8 = kv.StepBatch([0, n], [ctx], [ctx + n], other.table, slots8[ctx:], other.table.shape[1], 1 / 16)
    q8 = q[ctx:].half().contiguous()
    kv.paged_attention_scored(ex, other.layer, step8, q8, out8, hq, **ranges)
    torch.cuda.synchronize()
    for side, slab in enumerate((other.layer.k, other.layer.v)):
        other.rows[side] = slab.cpu().numpy().reshape(other.rows[side].shape)
    want8, size8 = scored_attention(other, q8.float().cpu().numpy(), hq, softcap=30.0, key_begin=key_begin)
    _check("q8", out8, want8, size8, torch.float16)
