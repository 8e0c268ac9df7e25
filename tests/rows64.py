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
