"""Decode over a Q4_0 cache whose values are small, or whose blocks have scales of very different sizes.

The kernel's result is that of 32-bit arithmetic for every size of the values: the bound on the error is the one of tests/test_q4_gpu.py
(2^-17, derived there), here for each run of 32 values of the results by itself, since it is for these that a block has a scale."""
import numpy as np
import pytest

from crispasr_b200 import abi
from tests.q4_ref import attention_f64, dequantize_q4_0, quantize_q4_0
from tests.util import gpu_op, randn_f16

pytestmark = pytest.mark.gpu

EXACT_REL = 2.0 ** -17


def _check(b200, rng, kx, vx, gqa, Tq=1, splits=(0,), q=None, bound=EXACT_REL, **kw):
    B, Hkv, L, hd = kx.shape
    k, v = quantize_q4_0(kx.astype(np.float32)), quantize_q4_0(vx.astype(np.float32))
    kf, vf = dequantize_q4_0(k), dequantize_q4_0(v)
    q = randn_f16(rng, (B, Hkv * gqa, Tq, hd)) if q is None else q
    ref = attention_f64(q, kf, vf, hd ** -0.5, **kw).reshape(-1, hd // 32, 32)
    for n in splits:
        assert b200.lib().b200_set_decode_splits(n) == 0
        try:
            got = gpu_op(b200, q, k, v, scale=hd ** -0.5, kv_type=abi.Q4_0, **kw)
        finally:
            b200.lib().b200_set_decode_splits(0)
        assert b200.lib().b200_last_kernel() == abi.KERNEL_DECODE_SPLIT
        got = got.reshape(ref.shape).astype(np.float64)
        assert np.isfinite(got).all()
        rel = np.sqrt(((got - ref) ** 2).sum((0, 2)) / np.maximum((ref ** 2).sum((0, 2)), 1e-300))   # of each block of head_dim
        assert (rel <= bound).all(), f"{n} splits: {rel}"


def _normal(rng, B, Hkv, L, hd):
    return (rng.standard_normal((B, Hkv, L, hd)) for _ in "kv")


@pytest.mark.parametrize("size", [1e-2, 1e-3, 1e-4, 1e-5, 1e-6])
@pytest.mark.parametrize("gqa,Tq", [(1, 1), (4, 1), (8, 1), (4, 4)])
@pytest.mark.parametrize("hd,L", [(128, 500), (64, 130), (128, 4212)])
def test_small_values(b200, size, gqa, Tq, hd, L):
    rng = np.random.default_rng([int(-np.log10(size)), gqa, Tq, hd, L])
    kx, vx = _normal(rng, 2, 2, L, hd)
    _check(b200, rng, kx, vx * size, gqa, Tq, splits=(0, 1))


@pytest.mark.parametrize("sizes", [(1, 1e-4, 1e-6, 1e-2), (1e-6, 1, 1, 1e-5), (300, 1, 1e-3, 1e-6), (1e-5, 2000, 1, 40), (1, 1, 1, 2000)])
@pytest.mark.parametrize("gqa,Tq", [(4, 1), (8, 1), (2, 5)])
def test_blocks_of_different_sizes_in_one_row(b200, sizes, gqa, Tq):
    rng = np.random.default_rng([gqa, Tq])
    kx, vx = _normal(rng, 2, 2, 1100, 128)
    _check(b200, rng, kx, vx * np.repeat(sizes, 32), gqa, Tq, splits=(0, 1))


@pytest.mark.parametrize("case", ["zeros_first", "tiny_first", "normal_first", "growing", "shrinking", "every_other", "large_late"])
@pytest.mark.parametrize("gqa", [4, 8])
@pytest.mark.parametrize("hd", [64, 128])
def test_sizes_that_change_along_the_keys(b200, case, gqa, hd):
    """What a warp has taken for the range of its scales turns out to be another one."""
    rng = np.random.default_rng(len(case) + gqa + hd)
    L = 1000
    kx, vx = _normal(rng, 2, 2, L, hd)
    key = np.arange(L)
    size = {"zeros_first": key >= 300, "tiny_first": np.where(key < 500, 1e-6, 1e-3), "normal_first": np.where(key < 500, 1.0, 1e-5),
            "growing": 10.0 ** (key / 100 - 6), "shrinking": 10.0 ** (2 - key / 125), "every_other": np.where(key % 2, 1e-5, 1e-3),
            "large_late": np.where(key < 900, 1e-4, 500.0)}[case]
    _check(b200, rng, kx, vx * size[:, None], gqa, splits=(0, 1, 3))


@pytest.mark.parametrize("size,small", [(30.0, 1.0), (1000.0, 1.0), (10.0, 1e-3), (1.0, 1e-4)])
@pytest.mark.parametrize("at", [3, 700])
def test_a_large_value_that_no_row_attends_to(b200, size, small, at):
    """One key with large values and a weight of nothing leaves the others their bits."""
    rng = np.random.default_rng(at)
    kx, vx = _normal(rng, 1, 2, 1000, 128)
    q = np.abs(randn_f16(rng, (1, 8, 1, 128)))
    kx[:, :, at] = -8.0   # every score with it is far below the others
    vx *= small
    vx[:, :, at] *= size / small
    _check(b200, rng, kx, vx, 4, splits=(0, 1), q=q)


@pytest.mark.parametrize("gqa,Tq", [(1, 4), (2, 4), (4, 3)])
def test_small_values_causal_and_ragged(b200, gqa, Tq):
    rng = np.random.default_rng(gqa)
    kx, vx = _normal(rng, 4, 2, 300, 128)
    _check(b200, rng, kx, vx * 1e-5, gqa, Tq, kv_len=np.array([300, 1, 0, 77], np.int32), q_len=np.array([Tq, 1, 0, 2], np.int32), causal=True)
