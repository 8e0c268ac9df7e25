"""Refusals of the operators around the cache: they come from the host, before any CUDA call, so that they run without a GPU."""
import ctypes as C

import pytest
import torch

import rows64
from util import canonical_layout
from warp34_b200 import ffi, kv


@pytest.fixture(scope="module")
def lib(native_libs):
    return native_libs[0]


def _args(**kw):
    a = ffi.QkNormRopeArgs()
    p = 4096
    a.q_in = a.k_in = a.q_out = a.k_out = a.q_norm_w = a.k_norm_w = a.positions = a.inv_freq = p
    a.num_tokens, a.num_q_heads, a.num_kv_heads, a.head_dim, a.rotary_dim, a.position_planes = 3, 4, 2, 256, 64, 1
    a.q_in_stride = a.q_out_stride = a.gate_out_stride = 1024
    a.k_in_stride = a.k_out_stride = 512
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(head_dim=128), 801), (dict(rotary_dim=40), 801), (dict(rotary_dim=272), 801), (dict(rotary_dim=-16), 1), (dict(num_tokens=-1), 1),
    (dict(num_q_heads=-1), 1), (dict(num_kv_heads=-1), 1), (dict(q_in=None), 1), (dict(k_out=None), 1), (dict(q_norm_w=None), 1),
    (dict(q_in_stride=1023), 1), (dict(k_in_stride=511), 1), (dict(q_out_stride=1000), 1), (dict(gate_out=4096), 1),      # 4 x 512 with a gate
    (dict(gate_out=4096, q_in_stride=2048, gate_out_stride=1023), 1), (dict(positions=None), 1), (dict(inv_freq=None), 1),
    (dict(position_planes=2), 1), (dict(position_planes=3, position_plane_stride=2), 1), (dict(q_in=4097), 1), (dict(k_norm_w=4099), 1),
    (dict(num_tokens=0), 0), (dict(num_q_heads=0, num_kv_heads=0), 0), (dict(num_q_heads=70000, q_in_stride=1 << 25, q_out_stride=1 << 25), 1),
])
def test_qk_norm_rope(lib, change, code):
    ex = ffi.Exec()
    for fn in (lib.warp34_qk_norm_rope_f16, lib.warp34_qk_norm_rope_bf16):
        assert fn(C.byref(ex), C.byref(_args(**change))) == code
        assert fn(None, C.byref(_args())) == 1 and fn(C.byref(ex), None) == 1


def test_qk_norm_rope_wrapper_checks_what_it_is_given(lib):
    t = lambda *s, dtype=torch.float16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    ex = type("E", (), {"ex": ffi.Exec()})()
    good = dict(q=t(3, 4, 256), k=t(3, 2, 256), q_weight=t(256), k_weight=t(256), positions=torch.zeros(3, dtype=torch.int32),
                inv_freq=torch.zeros(32), q_out=t(3, 4, 256), k_out=t(3, 2, 256))
    for change in (dict(q=t(3, 4, 256, dtype=torch.float32)), dict(k=t(3, 2, 256, dtype=torch.bfloat16)), dict(q_out=t(3, 3, 256)), dict(k_out=t(2, 2, 256)),
                   dict(q=t(3, 256, 4).transpose(1, 2)), dict(q_weight=t(255)), dict(positions=torch.zeros(3, dtype=torch.int64)),
                   dict(positions=torch.zeros(3, 3, dtype=torch.int32)), dict(inv_freq=torch.zeros(32, dtype=torch.float64)), dict(gate_out=t(3, 4, 256)),
                   dict(valid_token_mask=torch.ones(2, dtype=torch.uint8)), dict(q=None, k=None)):
        with pytest.raises(ValueError):
            kv.qk_norm_rope(ex, **{**good, **change})


def _read_call(lib, layout, k=4096, v=4096, ks=1024, vs=1024, **kw):
    b = ffi.AttentionBatch()
    b.query_start_loc = b.write_slot_mapping = b.block_tables = b.seq_lens_after = 4096
    b.num_reqs, b.total_tokens, b.max_blocks_per_req = 1, 5, 2
    for name, x in kw.items():
        setattr(b, name, x)
    ex = ffi.Exec()
    codes = {fn(C.byref(ex), C.byref(layout), C.byref(b), k, v, ks, vs) for fn in (lib.warp34_kv_cache_read_f16, lib.warp34_kv_cache_read_bf16)}
    assert len(codes) == 1
    return codes.pop()


def test_kv_cache_read(lib):
    lay = canonical_layout(4)
    lay.k_base = lay.v_base = 1 << 20
    call = lambda **kw: _read_call(lib, lay, **kw)  # noqa: E731
    assert call(k=None, v=None) == 1 and call(ks=1023) == 1 and call(vs=512) == 1 and call(k=4097) == 1
    assert call(total_tokens=-1) == 1 and call(total_tokens=0) == 0 and call(num_reqs=0) == 1 and call(query_start_loc=None) == 1
    assert call(write_slot_mapping=None, block_tables=None) == 1 and call(write_slot_mapping=None, max_blocks_per_req=0) == 1
    assert call(write_slot_mapping=None, seq_lens_after=None) == 1
    ex, b = ffi.Exec(), ffi.AttentionBatch()
    assert lib.warp34_kv_cache_read_f16(None, C.byref(lay), C.byref(b), 4096, 4096, 1024, 1024) == 1
    assert lib.warp34_kv_cache_read_f16(C.byref(ex), None, C.byref(b), 4096, 4096, 1024, 1024) == 1
    for field, value, code in (("head_dim", 128, 801), ("block_size", 32, 801), ("k_format", ffi.KV_FORMAT_FP16, 801), ("k_transform", 0, 801),
                               ("v_format", ffi.KV_FORMAT_Q8_0, 801), ("k_base", 0, 1), ("v_token_stride_bytes", 133, 1), ("local_kv_heads", 0, 1)):
        lay = canonical_layout(4)
        lay.k_base = lay.v_base = 1 << 20
        setattr(lay, field, value)
        assert call() == code, field
    for name in ("fp8", "q8"):      # 8-bit rows are read a word at a time
        layer = kv.KvLayer(2, 4, formats=rows64.formats(name), device="cpu")
        layer.layout.k_token_stride_bytes += 2
        assert _read_call(lib, layer.layout) == 1


def test_kv_cache_read_wrapper_checks_what_it_is_given(lib):
    layer = kv.KvLayer(2, 2, device="cpu")
    batch = kv.StepBatch([0, 3], [0], [3], [[1]], [16, 17, 18], 1, 0.0625, device="cpu")
    ex = type("E", (), {"ex": ffi.Exec()})()
    t = lambda *s, dtype=torch.float16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    for k, v in ((None, None), (t(3, 512), t(3, 512, dtype=torch.bfloat16)), (t(3, 512, dtype=torch.float32), None), (t(2, 512), None), (None, t(3, 256)),
                 (t(512, 3).T, None)):
        with pytest.raises(ValueError):
            kv.kv_cache_read(ex, layer, batch, k, v)


def _scored_call(lib, layout, fn="f16", hq=8, cap=30.0, scratch=0, change=(), q=4096, out=4096, **kw):
    b = ffi.AttentionBatch()
    b.query_start_loc = b.block_tables = b.seq_lens_after = 4096
    b.num_reqs, b.total_tokens, b.max_blocks_per_req, b.max_q_len, b.max_seq_len, b.sm_scale = 1, 5, 2, 5, 20, 0.0625
    for name, x in kw.items():
        setattr(b, name, x)
    c = ffi.ScoreChange(None, None, None, cap, 0)
    for name, x in change:
        setattr(c, name, x)
    return getattr(lib, f"warp34_paged_attention_scored_{fn}")(C.byref(ffi.Exec()), C.byref(layout), C.byref(b), C.byref(c), q, out, hq)


def test_scored_attention(lib):
    lay = canonical_layout(4)
    lay.k_base = lay.v_base = 1 << 20
    call = lambda **kw: _scored_call(lib, lay, **kw)  # noqa: E731
    nan = float("nan")
    assert call(total_tokens=0) == 0 and call(total_tokens=-1) == 1
    assert call(cap=-1.0) == 1 and call(cap=nan) == 1 and call(cap=2000.0) == 801 and call(cap=float("inf")) == 801 and call(cap=1e-5) == 801
    assert call(hq=0) == 1 and call(hq=6) == 1 and call(num_reqs=0) == 1 and call(query_start_loc=None) == 1 and call(block_tables=None) == 1
    assert call(seq_lens_after=None) == 1 and call(max_blocks_per_req=0) == 1 and call(sliding_window=-1) == 1 and call(mask_mode=7) == 1
    assert call(q=4097) == 1 and call(out=4099) == 1 and call(change=[("key_begin", 4098)]) == 1 and call(change=[("distance_slopes", 4097)]) == 1
    ex, b, c = ffi.Exec(), ffi.AttentionBatch(), ffi.ScoreChange()
    fn = lib.warp34_paged_attention_scored_f16
    assert fn(None, C.byref(lay), C.byref(b), C.byref(c), 4096, 4096, 8) == 1 and fn(C.byref(ex), C.byref(lay), C.byref(b), None, 4096, 4096, 8) == 1
    assert fn(C.byref(ex), C.byref(lay), C.byref(b), C.byref(c), None, 4096, 8) == 1
    for field, value in (("head_dim", 128), ("block_size", 32), ("k_format", ffi.KV_FORMAT_FP16), ("k_transform", 0), ("v_format", ffi.KV_FORMAT_Q8_0)):
        lay = canonical_layout(4)
        lay.k_base = lay.v_base = 1 << 20
        setattr(lay, field, value)
        assert call() == 801 and call(fn="bf16") == 801, field
    for name, fn in (("bf16", "f16"), ("fp8", "bf16"), ("q8", "bf16")):      # activations the layer's format has no kernel for
        assert _scored_call(lib, kv.KvLayer(2, 4, formats=rows64.formats(name), device="cpu").layout, fn=fn) == 801


def test_scored_attention_wrapper_checks_what_it_is_given(lib):
    layer = kv.KvLayer(2, 2, device="cpu")
    batch = kv.StepBatch([0, 3], [0], [3], [[1]], [16, 17, 18], 1, 0.0625, device="cpu")
    ex = type("E", (), {"ex": ffi.Exec()})()
    good = dict(q=torch.zeros(3, 4, 256, dtype=torch.float16), out=torch.zeros(3, 4, 256, dtype=torch.float16), num_q_heads=4)
    for change in (dict(q=torch.zeros(3, 4, 256)), dict(out=torch.zeros(3, 4, 256, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 4, 256, dtype=torch.float16)),
                   dict(out=torch.zeros(3, 256, 4, dtype=torch.float16).transpose(1, 2)), dict(slopes=torch.zeros(3)), dict(slopes=torch.zeros(4, dtype=torch.float64)),
                   dict(key_begin=torch.zeros(2, dtype=torch.int32)), dict(key_end=torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(ValueError):
            kv.paged_attention_scored(ex, layer, batch, **{**good, **change})


def test_tensors_of_the_host_are_refused(lib):
    """Every argument checked above is right here but for where it lies."""
    layer = kv.KvLayer(2, 2, device="cpu")
    batch = kv.StepBatch([0, 3], [0], [3], [[1]], [16, 17, 18], 1, 0.0625, device="cpu")
    ex = type("E", (), {"ex": ffi.Exec()})()
    t = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    with pytest.raises(ValueError, match="GPU"):
        kv.paged_attention_scored(ex, layer, batch, t(3, 4, 256), t(3, 4, 256), 4)
    with pytest.raises(ValueError, match="GPU"):
        kv.kv_cache_read(ex, layer, batch, t(3, 512), None)
    with pytest.raises(ValueError, match="GPU"):
        kv.qk_norm_rope(ex, t(3, 4, 256), None, t(256), None, None, None, t(3, 4, 256), None)
    with pytest.raises(ValueError, match="GPU"):
        kv.qk_norm_rope(ex, None, t(3, 2, 256), None, t(256), torch.zeros(3, dtype=torch.int32), torch.zeros(32), None, t(3, 2, 256))


def test_a_stride_beyond_the_interface_is_refused(lib):
    layer = kv.KvLayer(2, 1, device="cpu")
    batch = kv.StepBatch([0, 2], [0], [2], [[1]], [16, 17], 1, 0.0625, device="cpu")
    ex = type("E", (), {"ex": ffi.Exec()})()
    far = torch.empty_strided((2, 256), ((1 << 32) + 256, 1), dtype=torch.float16, device="meta")      # its lower 32 bits are a valid stride
    with pytest.raises(ValueError, match="stride"):
        kv.kv_cache_read(ex, layer, batch, far, None)
