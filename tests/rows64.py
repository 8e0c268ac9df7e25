"""Test infrastructure: cached rows and attention over them in 64 bits, on the CPU.

Random rows of every layer format as bytes, what they stand for (decode), and attention with changed scores by its definition.  The TQ4
tables are read from the generated header (tests/test_tables.py checks them against their definition)."""
import os
import re

import numpy as np
import torch

from warp34_b200 import ffi

_HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "warp34_b200", "csrc", "tq4_tables.h")
TQ4, FP8, Q8, BF16 = ffi.KV_FORMAT_TQ4, ffi.KV_FORMAT_FP8_E4M3, ffi.KV_FORMAT_Q8_0, ffi.KV_FORMAT_BF16
ROW = {TQ4: 132, FP8: 264, Q8: 272, BF16: 512}
NAMES = {"tq4": (TQ4, TQ4), "fp8": (FP8, FP8), "q8": (Q8, Q8), "q8_fp8": (Q8, FP8), "bf16": (BF16, BF16)}


def formats(name):
    """The four numbers KvLayer takes."""
    k, v = NAMES[name]
    t = ffi.KV_TRANSFORM_RADEMACHER_WHT256 if k == TQ4 else ffi.KV_TRANSFORM_IDENTITY
    return (k, v, t, t)


def _words(name):
    body = re.search(r"#define " + name + r" \{(.*?)\}", open(_HEADER).read().replace("\\\n", " "), re.S).group(1)
    return np.array([int(x.strip().rstrip("u"), 16) for x in body.split(",")], np.uint32)


CENTROIDS = _words("W34_TQ4_CENTROID_BITS").view(np.float32).astype(np.float64)
_SIGN = _words("W34_TQ4_SIGN_MASK")
SIGNS = np.array([-1.0 if (_SIGN[i >> 5] >> (i & 31)) & 1 else 1.0 for i in range(256)])
H = np.ones((1, 1))
for _ in range(8):
    H = np.block([[H, H], [H, -H]])
_E4M3 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).to(torch.float64).numpy()


def random_rows(fmt, n, rng, scale=1.0):
    """uint8 [n, row bytes]: elements of about `scale` in magnitude."""
    if fmt == BF16:
        return torch.from_numpy((rng.standard_normal((n, 256)) * scale).astype(np.float32)).to(torch.bfloat16).view(torch.uint8).numpy().reshape(n, 512)
    if fmt == TQ4:
        d = (16 * scale * np.exp(0.25 * rng.standard_normal((n, 2)))).astype(np.float16).view(np.uint8).reshape(n, 2, 2)
        return np.concatenate([d, rng.integers(0, 256, (n, 2, 64), dtype=np.uint8)], 2).reshape(n, 132)
    if fmt == FP8:
        c = torch.from_numpy((rng.standard_normal((n, 256)) * 100).clip(-448, 448)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
        return np.concatenate([c, (scale / 100 * np.exp(0.25 * rng.standard_normal((n, 2)))).astype(np.float32).view(np.uint8).reshape(n, 8)], 1)
    c = np.round(rng.standard_normal((n, 4, 64)) * 40).clip(-127, 127).astype(np.int8).view(np.uint8)
    d = (scale / 40 * np.exp(0.25 * rng.standard_normal((n, 4)))).astype(np.float32).view(np.uint8).reshape(n, 4, 4)
    return np.concatenate([d, c], 2).reshape(n, 272)


def stored(rows, fmt):
    """uint8 [n, row bytes] -> float64 [n, 256] as stored (TQ4: in the rotated basis)."""
    rows = np.ascontiguousarray(rows)
    n = rows.shape[0]
    if fmt == BF16:
        return (rows.view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    if fmt == TQ4:
        h = rows.reshape(n, 2, 66)
        d = np.ascontiguousarray(h[:, :, :2]).view(np.float16).astype(np.float64)
        codes = np.stack([h[:, :, 2:] & 15, h[:, :, 2:] >> 4], -1).reshape(n, 2, 128)
        return (CENTROIDS[codes] * d).reshape(n, 256)
    if fmt == FP8:
        d = np.ascontiguousarray(rows[:, 256:]).view(np.float32).astype(np.float64)
        return _E4M3[rows[:, :256]] * np.repeat(d, 128, 1)
    b = rows.reshape(n, 4, 68)
    d = np.ascontiguousarray(b[:, :, :4]).view(np.float32).astype(np.float64)
    return (np.ascontiguousarray(b[:, :, 4:]).view(np.int8).astype(np.float64) * d).reshape(n, 256)


def values(rows, fmt):
    """uint8 [n, row bytes] -> float64 [n, 256]."""
    y = stored(rows, fmt)
    return (y @ H) / 16 * SIGNS if fmt == TQ4 else y


def half_step(x, dtype):
    """Half a rounding step of dtype at x, as float64."""
    eps, tiny = torch.finfo(dtype).eps, torch.finfo(dtype).smallest_normal
    return np.maximum(np.abs(x) * eps / 2, tiny * eps / 2)


# ---- attention with changed scores, by its definition ----------------------------------------------------------------------
class Cache:
    """A layer's pages and their rows on the host, a page table and the metadata of one step."""

    def __init__(self, name, heads, lens, ctx, seed, device="cuda", tail=None, spare=2):
        from warp34_b200 import kv
        self.name, self.heads, self.lens, self.ctx = name, heads, list(lens), list(ctx)
        rng = np.random.default_rng(seed)
        need = [(c + n + 15) // 16 for c, n in zip(ctx, lens)]
        pages = sum(need) + spare
        self.layer = kv.KvLayer(pages, heads, formats=formats(name), device=device)
        self.table = np.zeros((len(lens), max(max(need), 1)), np.int32)
        order, at = rng.permutation(pages - 1) + 1, 0
        for r, n in enumerate(need):
            self.table[r, :n] = order[at:at + n]
            at += n
        self.rows = [random_rows(f, pages * heads * 16, rng).reshape(pages, heads, 16, ROW[f]) for f in NAMES[name]]
        if tail is not None:      # rows no sequence holds: a byte pattern that stands for NaN in every format
            held = np.zeros((pages, 16), bool)
            for r, (c, n) in enumerate(zip(ctx, lens)):
                pos = np.arange(c + n)
                held[self.table[r, pos // 16], pos % 16] = True
            for rows in self.rows:
                rows[~held[:, None, :].repeat(heads, 1)] = tail
        self.upload()

    def upload(self):
        for slab, rows in zip((self.layer.k, self.layer.v), self.rows):
            slab.copy_(torch.from_numpy(rows.copy()).view(-1))

    def batch(self, device="cuda", **kw):
        from warp34_b200 import kv
        starts = np.concatenate([[0], np.cumsum(self.lens)])
        total = np.asarray(self.ctx) + np.asarray(self.lens)
        return kv.StepBatch(starts, self.ctx, total, self.table, np.zeros(max(int(starts[-1]), 1), np.int32), self.table.shape[1],
                            kw.pop("sm_scale", 1.0 / 16.0), device=device, **kw)

    def at(self, r, pos, side):
        """Index of a row in self.rows[side]: [page, :, offset]."""
        return self.rows[side][self.table[r, pos // 16], :, pos % 16]

    def sequence(self, r):
        """K and V of request r, float64 [heads, tokens, 256]."""
        pos = np.arange(self.ctx[r] + self.lens[r])
        res = []
        for side, fmt in enumerate(NAMES[self.name]):
            rows = self.at(r, pos, side)                                    # [tokens, heads, row]
            res.append(values(rows.reshape(-1, rows.shape[-1]), fmt).reshape(len(pos), self.heads, 256).transpose(1, 0, 2))
        return res


def scored_attention(cache, q, hq, sm_scale=1.0 / 16.0, softcap=0.0, slopes=None, key_begin=None, key_end=None, window=0, symmetric=False):
    """float64 outputs [tokens, q heads, 256] and, beside them, what errors are taken of: S = sum_k weight_k |V_k| for errors of weights, which
    multiply whole rows.  On rotated layers also errors of single rotated coordinates (rounded centroids, products, sums) end in a
    channel, from all 256 coordinates with the signs of the transform: (1 / 16) sum_c +-e_c, whatever the channel's own V.  With
    |e_c| <= r A_c, A_c = sum_k weight_k |y_kc|, that is r sqrt(mean A_c^2) in the root mean square over the signs: S has
    sqrt(mean A_c^2) added there, and a tolerance of r' S holds for r up to a quarter of r' (four standard deviations and more)."""
    n, g = sum(cache.lens), hq // cache.heads
    q = np.asarray(q, np.float64).reshape(n, hq, 256)
    out, size = np.zeros((n, hq, 256)), np.zeros((n, hq, 256))
    at = 0
    with np.errstate(all="ignore"):
        for r, (c, m) in enumerate(zip(cache.ctx, cache.lens)):
            k, v = cache.sequence(r)
            rotated = NAMES[cache.name][1] == TQ4
            y = np.abs((v * SIGNS) @ H / 16) if rotated else None      # the transform is its own inverse
            key = np.arange(c + m)
            for t in range(m):
                p = c + t
                first = 0 if window <= 0 else max(0, p - window + 1)
                last = c + m - 1 if symmetric else p
                if key_begin is not None:
                    first = max(first, int(key_begin[at + t]))
                if key_end is not None:
                    last = min(max(int(key_end[at + t]), 0), c + m) - 1
                if first > last:
                    continue
                span = slice(first, last + 1)
                for h in range(hq):
                    s = k[h // g][span] @ q[at + t, h] * sm_scale
                    if softcap > 0:
                        s = softcap * np.tanh(s / softcap)
                    if slopes is not None:
                        s = s - float(slopes[h]) * np.abs(p - key[span])
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[at + t, h] = w @ v[h // g][span]
                    size[at + t, h] = w @ np.abs(v[h // g][span])
                    if rotated:
                        size[at + t, h] += np.sqrt(((w @ y[h // g][span]) ** 2).mean())
            at += m
    return out, size
