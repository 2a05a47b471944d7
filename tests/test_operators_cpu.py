"""Refusals of the 4-bit cache's and the rotation's entry points, and what a plan says of them; no GPU needed."""
import ctypes as C

import numpy as np
import pytest
import torch

from crispasr_b200 import abi
from tests.q4_ref import dequantize_q4_0, quantize_q4_0


def _supports(b200, q, k, v, **kw):
    from crispasr_b200.op import _dst_like, _make
    c = _make(q, k, v, None, _dst_like(q), dict(scale=1.0, kv_type=abi.Q4_0, **kw), abi.from_torch)
    why = C.c_int(0)
    return bool(b200.lib().b200_fattn_supports(*c.args(), C.byref(why))), why.value


def test_q4_0_operands(b200):
    q = torch.zeros((1, 8, 1, 128))
    k = torch.zeros((1, 2, 20, 72), dtype=torch.uint8)
    assert _supports(b200, q, k, k) == (True, 0)
    assert _supports(b200, q, k[..., :54], k[..., :54])[1] == abi.E_SHAPE                      # 96 values per row
    assert _supports(b200, q, k, torch.zeros((1, 2, 21, 72), dtype=torch.uint8))[1] == abi.E_SHAPE
    assert _supports(b200, torch.zeros((1, 8, 1, 120)), k, k)[1] == abi.E_SHAPE
    odd = torch.zeros(1 + 2 * 20 * 72, dtype=torch.uint8)[1:].view(1, 2, 20, 72)
    assert _supports(b200, q, odd, k)[1] in (abi.E_ALIGN, 0) and (odd.data_ptr() % 2 == 0 or _supports(b200, q, odd, k)[1] == abi.E_ALIGN)
    with pytest.raises(ValueError):
        abi.from_torch(torch.zeros((1, 2, 20, 72)), abi.Q4_0)
    mixed = abi.from_torch(torch.zeros((1, 2, 20, 128), dtype=torch.float16))
    tq, tk, dst = abi.from_torch(q), abi.from_torch(k, abi.Q4_0), torch.zeros((1, 1, 8, 128))
    td, p, why = abi.from_torch(dst), abi.Params(1.0, 0.0, 0.0, 0), C.c_int(0)
    assert b200.lib().b200_fattn_supports(C.byref(tq), C.byref(tk), C.byref(mixed), None, C.byref(td), C.byref(p), None, C.byref(why)) == 0
    assert why.value == abi.E_TYPE
    # a query, a mask or a result of blocks
    assert b200.lib().b200_fattn_supports(C.byref(tk), C.byref(tk), C.byref(tk), None, C.byref(td), C.byref(p), None, C.byref(why)) == 0
    assert why.value == abi.E_TYPE


def test_q4_0_plans(b200):
    k = torch.zeros((8, 8, 663, 72), dtype=torch.uint8)
    kern, ns = b200.plan(torch.zeros((8, 32, 1, 128)), k, k, scale=0.1, kv_type=abi.Q4_0)
    assert kern == abi.KERNEL_DECODE_SPLIT and ns >= 1
    kern, ns = b200.plan(torch.zeros((8, 32, 40, 128)), k, k, scale=0.1, kv_type=abi.Q4_0)
    assert kern == abi.KERNEL_PREFILL_TC5
    # the prompt's keys and values as F16 in the workspace
    assert b200.workspace_bytes(torch.zeros((8, 32, 40, 128)), k, k, scale=0.1, kv_type=abi.Q4_0) >= 2 * 8 * 8 * 663 * 256


def test_blocks_round_trip_of_the_reference():
    """The tests' own restatement: block by block, the largest value is met exactly but for the rounding of d, the others to one step."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 64)).astype(np.float32)
    y = dequantize_q4_0(quantize_q4_0(x))
    step = np.abs(x).reshape(50, 2, 32).max(-1, keepdims=True) / 8
    assert (np.abs(y - x).reshape(50, 2, 32) <= step * (1 + 2.0 ** -7)).all()
    x[0, :32] = 0
    assert quantize_q4_0(x)[0, 2:18].tolist() == [0x88] * 16


def _call(b200, q=None, k=None, q_out=None, k_out=None, q_norm=None, k_norm=None, params=None, **over):
    """b200_qk_norm_rope on host descriptors; only for calls that are refused."""
    base = dict(n_dims=64, mode=abi.ROPE_NEOX, freq_base=1e4, freq_scale=1.0, eps=1e-6)
    base.update(over)
    p = abi.RopeParams(base["n_dims"], base["mode"], base["freq_base"], base["freq_scale"], base["eps"], 0) if params is None else params

    def d(x):
        return None if x is None else C.byref(x if isinstance(x, abi.Tensor) else abi.from_torch(x))
    rc = b200.lib().b200_qk_norm_rope(d(q), d(k), d(q_norm), d(k_norm), C.byref(p) if p else None, None, 0, None, d(q_out), d(k_out), None)
    assert rc != abi.OK and rc != abi.E_CUDA, "the call was not refused"
    return rc


def test_rope_refusals(b200):
    q, k = torch.zeros((2, 4, 3, 64)), torch.zeros((2, 2, 3, 64))
    assert _call(b200) == abi.E_NULL
    assert _call(b200, q) == abi.E_NULL
    assert _call(b200, q, k, q) == abi.E_NULL                                     # k without k_out
    assert _call(b200, q, None, q, k) == abi.E_NULL
    assert _call(b200, q, k, q, k, params=False) == abi.E_NULL
    assert _call(b200, q, k.half(), q, k) == abi.E_TYPE
    assert _call(b200, q, k, q, k.half()) == abi.E_TYPE
    assert _call(b200, q, k, torch.zeros((2, 4, 3, 32)), k) == abi.E_SHAPE
    assert _call(b200, q, torch.zeros((2, 2, 4, 64)), q, torch.zeros((2, 2, 4, 64))) == abi.E_SHAPE
    assert _call(b200, q, torch.zeros((1, 2, 3, 64)), q, torch.zeros((1, 2, 3, 64))) == abi.E_SHAPE
    wide = torch.zeros((2, 4, 3, 128))
    assert _call(b200, wide[..., ::2], None, q) == abi.E_STRIDE
    big = torch.zeros((1, 1, 1, 136))
    assert _call(b200, big, None, big) == abi.E_UNSUPPORTED
    odd = torch.zeros((1, 1, 1, 60))
    assert _call(b200, odd, None, odd, n_dims=32) == abi.E_UNSUPPORTED
    assert _call(b200, q, None, q, n_dims=66) == abi.E_SHAPE
    assert _call(b200, q, None, q, n_dims=-2) == abi.E_SHAPE
    assert _call(b200, q, None, q, n_dims=31, mode=abi.ROPE_NORM) == abi.E_SHAPE
    assert _call(b200, q, None, q, n_dims=24) == abi.E_UNSUPPORTED               # NEOX: a multiple of 16
    assert _call(b200, q, None, q, mode=1) == abi.E_UNSUPPORTED
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        assert _call(b200, q, None, q, freq_base=bad) == abi.E_SHAPE
    assert _call(b200, q, None, q, freq_scale=float("nan")) == abi.E_SHAPE
    assert _call(b200, q, None, q, eps=-1e-6) == abi.E_SHAPE
    assert _call(b200, q, None, q, q_norm=torch.zeros(64, dtype=torch.float16)) == abi.E_TYPE
    assert _call(b200, q, None, q, q_norm=torch.zeros(32)) == abi.E_SHAPE
    assert _call(b200, q, k, q, k, k_norm=torch.zeros((2, 64))) == abi.E_SHAPE
    assert _call(b200, q, None, q, q_norm=torch.zeros(128)[::2]) == abi.E_STRIDE
    t = abi.from_torch(q)
    t.data += 2
    assert _call(b200, t, None, q) == abi.E_ALIGN
    t = abi.from_torch(q)
    t.ne[1] = 0
    assert _call(b200, t, None, q) == abi.E_SHAPE
    t = abi.from_torch(q)
    t.nb[2] += 2
    assert _call(b200, t, None, q) == abi.E_STRIDE
    big = abi.from_torch(q)
    big.ne[1], big.ne[3] = 1 << 20, 1 << 12
    assert _call(b200, big, None, big) == abi.E_LIMIT


def test_cache_entry_points_refuse_null(b200):
    L = b200.lib()
    x = abi.from_torch(torch.zeros((1, 1, 1, 64)))
    p = abi.RopeParams(64, abi.ROPE_NEOX, 1e4, 1.0, 1e-6, 0)
    assert L.b200_kv_read(None, 0, C.byref(x), C.byref(x), None, 0, None) == abi.E_NULL
    assert L.b200_kv_append_rope(None, 0, C.byref(x), C.byref(x), C.byref(x), None, None, C.byref(p), None, 0, None, C.byref(x), None) == abi.E_NULL
    cfg = abi.KvConfig(3, 128, 1, 1, 16, 1)   # a block type that is not kept
    h = C.c_void_p()
    assert L.b200_kv_create(C.byref(cfg), C.byref(h)) == abi.E_TYPE and not h.value


def test_python_refusals(b200):
    x = torch.zeros((1, 2, 3, 64))
    with pytest.raises(ValueError, match="CUDA"):
        b200.qk_norm_rope(x)
    with pytest.raises(TypeError, match="unexpected keyword"):
        b200.qk_norm_rope(x, rope_dim=64)
    with pytest.raises(TypeError):
        b200.qk_norm_rope()
    with pytest.raises(TypeError):
        b200.qk_norm_rope(x.numpy())


class _NoCache:
    """What the native methods see of a KvCache: its handle, here one that has been closed."""
    _h = C.c_void_p()


def test_cache_methods_refuse(b200):
    from crispasr_b200 import op
    op._load_native()
    x = torch.zeros((1, 2, 3, 64))
    assert op.KvCache.read.__doc__ and op.KvCache.append_rope.__doc__
    with pytest.raises(b200.B200Error):
        op.KvCache.read(_NoCache(), 0, 3)
    for bad in (dict(), dict(layer=0), dict(layer=0, n_rows=1, rows=2), dict(layer=0, n_rows=1, dtype="f32"), dict(layer=0, n_rows=1, dtype=torch.int8)):
        with pytest.raises((TypeError, ValueError)):
            op.KvCache.read(_NoCache(), **bad)
    with pytest.raises(TypeError, match="multiple values"):
        op.KvCache.read(_NoCache(), 0, 3, layer=1)
    with pytest.raises(ValueError, match="CUDA"):
        op.KvCache.append_rope(_NoCache(), 0, None, x, x)
    with pytest.raises(TypeError):
        op.KvCache.append_rope(_NoCache(), 0, x, x)
    with pytest.raises(TypeError, match="unexpected"):
        op.KvCache.append_rope(_NoCache(), 0, None, x, x, base=3.0)
    for layer in (1 << 32, -(1 << 32)):   # not layer 0
        with pytest.raises(OverflowError):
            op.KvCache.append_rope(_NoCache(), layer, None, x, x)
        with pytest.raises(OverflowError):
            op._kv_tensors(0, _NoCache(), layer, 1)
