"""Scored attention on random calls: every format, head group and route, masks, windows, key ranges with empty ones among them, workspaces from
none to more than enough and full of random bytes, never-written rows that stand for NaN.  Against the definition in 64 bits (on the GPU), at
the tolerance that test_gpu_scored_attention.py derives; rows that take no part stay as they were, rows without keys are zeros."""
import random

import numpy as np
import pytest

import rows64
from rows64 import Cache

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
SHARE = {"tq4": 2.0 ** -11, "fp8": 2.0 ** -12, "q8": 2.0 ** -12, "q8_fp8": 2.0 ** -12, "bf16": 2.0 ** -12}      # of sum_k weight_k |V_k|


def _definition(cache, q, hq, softcap=0.0, slopes=None, key_begin=None, key_end=None, window=0, symmetric=False, sm_scale=1.0 / 16):
    """rows64.scored_attention with torch in float64 on the GPU: outputs, what errors are taken of, and outputs that may be NaN as well."""
    n, g = sum(cache.lens), hq // cache.heads
    q = q.double().view(n, hq, 256)
    out, size, faint = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape, dtype=torch.bool, device="cuda")
    hadamard, signs = torch.from_numpy(rows64.H).cuda() / 16, torch.from_numpy(rows64.SIGNS).cuda()
    rotated = rows64.NAMES[cache.name][1] == rows64.TQ4
    at = 0
    for r, (c, m) in enumerate(zip(cache.ctx, cache.lens)):
        pos = np.arange(c + m)
        kv = []
        for side, fmt in enumerate(rows64.NAMES[cache.name]):
            rows = cache.at(r, pos, side)
            y = torch.from_numpy(rows64.stored(rows.reshape(-1, rows.shape[-1]), fmt)).cuda().view(c + m, cache.heads, 256).transpose(0, 1)
            kv.append((y, (y @ hadamard) * signs if fmt == rows64.TQ4 else y))
        k, (stored, v) = kv[0][1], kv[1]
        if m == 0:
            continue
        p, key = torch.arange(c, c + m, device="cuda"), torch.arange(c + m, device="cuda")
        first = torch.zeros_like(p) if window <= 0 else (p - window + 1).clamp(min=0)
        last = torch.full_like(p, c + m - 1) if symmetric else p
        if key_begin is not None:
            first = torch.maximum(first, key_begin[at:at + m].long())
        if key_end is not None:
            last = key_end[at:at + m].long().clamp(0, c + m) - 1
        seen = (key >= first[:, None]) & (key <= last[:, None])
        rows = q[at:at + m].view(m, cache.heads, g, 256).permute(1, 2, 0, 3)                      # [kv head, row of the group, token]
        s = (rows @ k.unsqueeze(1).transpose(2, 3)) * sm_scale
        if softcap > 0:
            s = softcap * torch.tanh(s / softcap)
        if slopes is not None:
            s = s - slopes.double().view(cache.heads, g, 1, 1) * (p[:, None] - key).abs()
        s = s.masked_fill(~seen, -float("inf"))
        top = s.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        place = lambda x: x.permute(2, 0, 1, 3).reshape(m, hq, 256)  # noqa: E731
        # a NaN in V: in its channels, of the rows that see it (`faint`: with weights that are, or nearly, zero in fp32; what zero x NaN is is left open)
        holes = torch.isnan(v).double().unsqueeze(1)
        v, stored = torch.nan_to_num(v), torch.nan_to_num(stored)
        out[at:at + m] = place((w @ v.unsqueeze(1)).masked_fill((~(w <= 2.0 ** -120)).double() @ holes > 0, float("nan")))
        faint[at:at + m] = place((seen & (w <= 2.0 ** -120)).double() @ holes > 0)
        extra = 0.0
        if rotated:
            extra = (w @ stored.abs().unsqueeze(1)).pow(2).mean(-1, keepdim=True).sqrt()
        size[at:at + m] = place(w @ v.abs().unsqueeze(1) + extra)
        at += m
    return out, size, faint


def _spoil(cache, side, r, pos, rng):
    """NaN in a row of every head: one channel of it (BF16, FP8), the channels of a scale (Q8_0) or all (TQ4)."""
    rows = cache.rows[side][cache.table[r, pos // 16], :, pos % 16]
    fmt = rows64.NAMES[cache.name][side]
    if fmt == rows64.BF16:
        rows.view(np.uint16)[:, rng.randrange(256)] = 0x7fc0
    elif fmt == rows64.FP8:
        rows[:, rng.randrange(256)] = rng.choice([0x7f, 0xff])
    elif fmt == rows64.Q8:
        at = 68 * rng.randrange(4)
        rows[:, at:at + 4] = np.array([np.nan], np.float32).view(np.uint8)
    else:
        at = 66 * rng.randrange(2)
        rows[:, at:at + 2] = np.array([np.nan], np.float16).view(np.uint8)


def _call(seed):
    """Geometry and keyword arguments of a random call."""
    rng = random.Random(seed)
    name = rng.choice(["tq4", "tq4", "fp8", "q8", "q8_fp8", "bf16", "bf16"])
    hkv, g = rng.choice([1, 2, 3, 4]), rng.choice([1, 2, 3, 4, 6, 8, 9, 12, 16])
    kind = rng.choice(["one", "few", "decode", "verify", "chunk", "mixed"])
    b = {"one": 1, "few": rng.randint(1, 6), "decode": rng.randint(2, 40), "verify": rng.randint(1, 12), "chunk": rng.randint(1, 3), "mixed": rng.randint(1, 8)}[kind]
    lens = [{"one": 1, "few": 1, "decode": 1, "verify": rng.randint(1, 6), "chunk": rng.randint(1, 200), "mixed": rng.choice([0, 1, 2, 7, 40, 130])}[kind] for _ in range(b)]
    lens[0] = max(lens[0], 1)
    top = rng.choice([0, 5, 60, 400, 2500])
    ctx = [rng.randint(0, top) for _ in range(b)]
    n, total = sum(lens), max(x + y for x, y in zip(ctx, lens))
    gen = torch.Generator().manual_seed(seed)
    kw, batch = {}, {}
    if rng.random() < 0.7:
        kw["softcap"] = rng.choice([0.5, 15.0, 30.0, 50.0])
    if rng.random() < 0.5:
        kw["slopes"] = (torch.rand(g * hkv, generator=gen) * rng.choice([0.001, 0.1, 1.0 if total <= 700 else 0.01])).cuda()
    if rng.random() < 0.4:
        kw["key_begin"] = torch.randint(-5, total + 5, (n,), generator=gen, dtype=torch.int32).cuda()
    if rng.random() < 0.4:
        kw["key_end"] = torch.randint(-5, total + 50, (n,), generator=gen, dtype=torch.int32).cuda()
    if rng.random() < 0.4:
        batch["sliding_window"] = rng.choice([1, 3, 17, 100, 1000])
        if rng.random() < 0.4:
            batch["mask_mode"] = 1
    np_rng = np.random.default_rng(seed)
    if rng.random() < 0.3:
        batch["valid_token_mask"] = (np_rng.random(n) > 0.2).astype(np.uint8)
    if rng.random() < 0.2:
        batch["valid_req_mask"] = (np_rng.random(b) > 0.2).astype(np.uint8)
    if rng.random() < 0.2:
        batch["max_seq_len"] = 0
    scale = rng.choice([0.1, 1.0, 4.0])
    scratch = rng.choice([64 << 20, 64 << 20, 2 << 20, 300 << 10, 0])
    return name, hkv, g * hkv, lens, ctx, kw, batch, scale, scratch, gen, rng


def _run(native_libs, seed, spoiled=0):
    from warp34_b200 import ffi, kv
    name, hkv, hq, lens, ctx, kw, batch_kw, scale, scratch, gen, rng = _call(seed)
    n = sum(lens)
    dtype = torch.bfloat16 if name == "bf16" or (name == "tq4" and rng.random() < 0.3) else torch.float16
    cache = Cache(name, hkv, lens, ctx, seed, tail=0xff)
    for _ in range(spoiled):
        r = rng.choice([i for i in range(len(lens)) if ctx[i] + lens[i] > 0])
        _spoil(cache, rng.choice([0, 1, 1]), r, rng.choice([rng.randrange(ctx[r] + lens[r]), ctx[r] + rng.randrange(lens[r]) if lens[r] else 0]), rng)
    cache.upload()
    q = (torch.randn(n, hq, 256, generator=gen) * scale).to(dtype).cuda()
    batch = cache.batch(**batch_kw)
    want, size, faint = _definition(cache, q, hq, window=batch_kw.get("sliding_window", 0), symmetric="mask_mode" in batch_kw, **kw)
    on = np.ones(n, bool) if "valid_token_mask" not in batch_kw else batch_kw["valid_token_mask"].astype(bool)
    if "valid_req_mask" in batch_kw:
        on = on & np.repeat(batch_kw["valid_req_mask"].astype(bool), lens)
    on = torch.from_numpy(on).cuda()
    eps, tiny = torch.finfo(dtype).eps, torch.finfo(dtype).smallest_normal
    tol = torch.maximum(want.abs(), torch.tensor(tiny, dtype=torch.float64)) * (eps / 2 * (1 + 2.0 ** -8)) + SHARE[name] * size
    nan = torch.isnan(want)
    for flags in (0, ffi.EXEC_FLAG_PRECISE_ATTENTION):
        ex = kv.Executor(max(scratch, 1 << 12))
        ex.ex.flags = flags
        ex.scratch.random_(0, 256)
        if scratch == 0:
            ex.ex.scratch_ptr = ex.ex.scratch_size = 0
        out = torch.full_like(q, 7.0)
        kv.paged_attention_scored(ex, cache.layer, batch, q, out, hq, **kw)
        torch.cuda.synchronize()
        assert (out[~on] == 7.0).all()
        bad = ~((out.double() - want).abs() <= tol) & ~(nan | faint) & on[:, None, None]
        assert not bad.any(), f"{name} {hq}/{hkv} {lens[:4]} {ctx[:4]} {list(kw)} {list(batch_kw)} flags {flags}: {int(bad.sum())} outside, worst " \
                              f"{float(torch.nan_to_num((out.double() - want).abs() / tol)[on].max()):.2f} x"
        assert torch.isnan(out[on][nan[on]]).all()
        if not spoiled:
            assert (out[on & (size == 0).all(-1).all(-1)] == 0).all()
    return int(nan.sum())


@pytest.mark.parametrize("seed", range(150))
def test_random_calls(native_libs, seed):
    assert _run(native_libs, seed) == 0


@pytest.mark.parametrize("seed", range(1000, 1100))
def test_random_calls_over_rows_with_nan(native_libs, seed):
    """NaN in one to four random K or V rows: in the rows that see them, and there in the channels that V has it in; the rest as the definition says."""
    _run(native_libs, seed, spoiled=1 + seed % 4)
