"""Norm and rotary embedding of query and key heads (warp34_qk_norm_rope_f16 / _bf16) against the formula in 64 bits.

Tolerance, derived: half a step of the output type, and the fp32 arithmetic in front of it.  The sum of 256 squares is off by at most 13
roundings (8 in a lane, 5 across lanes) of 2^-24, half of that in the root; rsqrtf (2 ulp = 2^-22), its argument, the products
with weight and norm add 2^-22: below 2^-20 of the normalised value together.  Sine and cosine: 1 ulp each (2^-23) plus the angle's
rounding, 2^-24 of at most pi; two products and a sum: below 2^-20 of |a| + |b|.  2^-19 (|a| + |b|) holds both."""
import numpy as np
import pytest

from rows64 import half_step

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
F16, B16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def env(native_libs):
    from warp34_b200 import kv
    return kv


def _axes(half, planes, sections):
    i = np.arange(half)
    axis = np.zeros(half, np.int64)
    if planes == 3:
        axis[(i % 3 == 1) & (i < 3 * sections[1])] = 1
        axis[(i % 3 == 2) & (i < 3 * sections[2])] = 2
    return axis


def _reference(x, w, pos, inv_freq, sections, eps, offset):
    """float64 result and the magnitude the tolerance is taken of; x [n, heads, 256], pos [planes, n]."""
    f = x.astype(np.float64)
    y = f / np.sqrt((f * f).mean(-1, keepdims=True) + eps) * (offset + w.astype(np.float64))
    half = len(inv_freq)
    size = np.abs(y)
    if half:
        axis = _axes(half, pos.shape[0], sections)
        angle = pos[axis].T.astype(np.float64) * inv_freq.astype(np.float64)
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        a, b = y[..., :half].copy(), y[..., half:2 * half].copy()
        y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
        size[..., :half] = size[..., half:2 * half] = np.abs(a) + np.abs(b)
    return y, size


def _check(out, want, size, dtype, what):
    got = out.double().cpu().numpy()
    tol = half_step(want, dtype) * (1 + 2.0 ** -8) + 2.0 ** -19 * size
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size}, worst {np.nanmax(np.abs(got - want) / tol):.2f} x, first {np.argwhere(bad)[0]}"


def _inputs(dtype, hq, hkv, n, rotary, planes, gate, seed, shift=0):
    g = torch.Generator().manual_seed(seed)
    width = 512 if gate else 256
    row = hq * width + hkv * 256 + 256 + shift
    packed = (torch.randn(n, row, generator=g) * torch.exp(torch.randn(n, 1, generator=g))).to(dtype).cuda()
    cols = lambda a, b: packed[:, shift + a:shift + b]  # noqa: E731
    q = cols(0, hq * width).view(n, hq, width) if hq else None
    k = cols(hq * width, hq * width + hkv * 256).view(n, hkv, 256) if hkv else None
    w = [(torch.randn(256, generator=g) * 0.3).to(dtype).cuda() for _ in range(2)]
    edges = torch.tensor([0, 1, 262143, 2 ** 31 - 1, -1, -70001, 131072])
    pos = torch.cat([edges, torch.randint(0, 300000, (planes * n,), generator=g)])[:planes * n].view(planes, n).to(torch.int32)
    inv = (1e6 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / max(rotary, 1))).float()
    return q, k, w, pos, inv


CASES = [
    # dtype, query heads, kv heads, tokens, rotary, planes, gate, shift (elements by which rows miss their alignment)
    (F16, 24, 4, 1, 64, 3, True, 0),
    (B16, 16, 4, 37, 256, 1, False, 0),
    (F16, 1, 1, 7, 16, 1, False, 0),
    (B16, 6, 1, 300, 192, 3, True, 0),
    (F16, 0, 4, 64, 64, 1, False, 0),
    (B16, 5, 0, 33, 128, 3, False, 0),
    (F16, 3, 2, 29, 0, 1, True, 0),
    (F16, 6, 2, 41, 96, 1, True, 1),          # 2-byte alignment
    (B16, 24, 4, 401, 64, 3, True, 0),        # four rows a warp
    (F16, 40, 8, 260, 256, 1, False, 3),      # the same, two blocks a token, 2-byte alignment
]


@pytest.mark.parametrize("dtype,hq,hkv,n,rotary,planes,gate,shift", CASES)
def test_against_the_formula(env, dtype, hq, hkv, n, rotary, planes, gate, shift):
    kv = env
    q, k, w, pos, inv = _inputs(dtype, hq, hkv, n, rotary, planes, gate, 5 + n, shift)
    sections = (rotary // 2 - 2 * (rotary // 6), rotary // 6, rotary // 6) if planes == 3 else None
    out = lambda h: torch.full((n, h, 256), 7.0, dtype=dtype, device="cuda")  # noqa: E731
    qo, ko, go = out(hq) if hq else None, out(hkv) if hkv else None, out(hq) if gate else None
    kv.qk_norm_rope(kv.Executor(1 << 12), q, k, w[0] if hq else None, w[1] if hkv else None, pos.cuda() if planes == 3 else pos[0].cuda(), inv.cuda(),
                    qo, ko, gate_out=go, sections=sections, eps=1e-5, weight_offset=1.0 if n % 2 else 0.0)
    torch.cuda.synchronize()
    offset = 1.0 if n % 2 else 0.0
    for x, wt, o, what in ((q, w[0], qo, "q"), (k, w[1], ko, "k")):
        if x is not None:
            want, size = _reference(x[..., :256].float().cpu().numpy(), wt.float().cpu().numpy(), pos.numpy(), inv.numpy(), sections, 1e-5, offset)
            _check(o, want, size, dtype, what)
    if gate:
        assert torch.equal(go, q[..., 256:])


def test_masked_tokens_are_left_alone_and_special_rows_stay_to_themselves(env):
    kv, n, hq, hkv = env, 24, 6, 2
    q, k, w, pos, inv = _inputs(B16, hq, hkv, n, 64, 1, False, 3)
    q, k = q.clone(), k.clone()
    q[3, 1] = 0
    q[4, 2, 100] = float("nan")
    q[5, 0, 9] = float("inf")
    k[6, 1] = 3e38        # the squares overflow fp32
    mask = torch.ones(n, dtype=torch.uint8)
    mask[[0, 9]] = 0
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    kv.qk_norm_rope(kv.Executor(1 << 12), q, k, w[0], w[1], pos[0].cuda(), inv.cuda(), qo, ko, valid_token_mask=mask.cuda())
    with np.errstate(all="ignore"):
        for x, wt, o, odd in ((q, w[0], qo, [(4, 2), (5, 0)]), (k, w[1], ko, [(6, 1)])):
            want, size = _reference(x.float().cpu().numpy(), wt.float().cpu().numpy(), pos.numpy(), inv.numpy(), None, 1e-6, 1.0)
            keep = np.ones(want.shape[:2], bool)
            keep[[0, 9]] = False
            for at in odd:
                keep[at] = False
            assert (o[[0, 9]] == 7.0).all()
            _check(o[torch.from_numpy(keep).cuda()], want[keep], size[keep], B16, "rows")
    assert (qo[3, 1] == 0).all() and torch.isnan(qo[4, 2]).any()
    # inf / inf is NaN in the channel that held it, its rotated partner with it; the rest of the row is 0
    assert torch.isnan(qo[5, 0]).sum() == 2 and (qo[5, 0][~torch.isnan(qo[5, 0])] == 0).all()
    assert (ko[6, 1] == 0).all()


def test_in_place_replay_and_streams(env):
    kv, n, hq, hkv = env, 50, 24, 4
    q, k, w, pos, inv = _inputs(F16, hq, hkv, n, 64, 1, False, 8)
    pos, inv = pos[0].cuda(), inv.cuda()
    qo, ko = torch.zeros(n, hq, 256, dtype=F16, device="cuda"), torch.zeros(n, hkv, 256, dtype=F16, device="cuda")
    ex = kv.Executor(1 << 12)
    kv.qk_norm_rope(ex, q, k, w[0], w[1], pos, inv, qo, ko)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    ex_side = kv.Executor(1 << 12, stream=side)
    q2, k2 = q.clone(), k.clone()
    side.wait_stream(torch.cuda.current_stream())
    kv.qk_norm_rope(ex_side, q2, k2, w[0], w[1], pos, inv, q2, k2)          # in place, on another stream than the current one
    side.synchronize()
    assert torch.equal(q2, qo) and torch.equal(k2, ko)
    g = torch.cuda.CUDAGraph()
    q3, k3 = torch.zeros_like(qo), torch.zeros_like(ko)
    with torch.cuda.graph(g):
        ex.set_stream()
        kv.qk_norm_rope(ex, q, k, w[0], w[1], pos, inv, q3, k3)
    for _ in range(2):
        q.neg_()
        g.replay()
        torch.cuda.synchronize()
    assert torch.equal(q3, qo) and torch.equal(k3, ko)


def test_one_row_of_positions_expanded_to_three_planes(env):
    kv = env
    q, k, w, pos, inv = _inputs(F16, 4, 2, 19, 64, 1, False, 77)
    p = pos[0].cuda()
    outs = []
    for positions in (p, p.expand(3, 19), p[None].repeat(3, 1)):
        qo, ko = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty_like(k, memory_format=torch.contiguous_format)
        kv.qk_norm_rope(kv.Executor(1 << 12), q, k, w[0], w[1], positions, inv.cuda(), qo, ko, sections=(12, 10, 10))
        outs.append((qo, ko))
    for qo, ko in outs[1:]:
        assert torch.equal(qo, outs[0][0]) and torch.equal(ko, outs[0][1])
