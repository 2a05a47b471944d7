"""The Q4_0 cache: rows in, rows out, and attention over them in every operand form."""
import ctypes as C

import numpy as np
import pytest
import torch

from crispasr_b200 import abi
from tests.q4_ref import attention_f64, dequantize_q4_0, quantize_q4_0, random_q4_0
from tests.util import assert_close, cuda_view, errors, gpu_op, randn_f16

pytestmark = pytest.mark.gpu


# ---- rows into the cache and out of it ------------------------------------------------------------------------------

@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("n_new", [1, 3, 17, 65])
def test_append_row_shapes(b200, hd, n_new):
    """Every byte of the slab against the definition, the rows around the appended ones included: rows of one to four blocks,
    token-major sources, sources that are 8-byte aligned only, a stream whose rows run out of the cache."""
    rng = np.random.default_rng(40 * hd + n_new)
    S, Hkv, ctx, p0 = 2, 3, 96, 5
    kv = b200.KvCache(abi.Q4_0, hd, Hkv, n_layers=2, max_ctx=ctx, n_streams=S)
    new = rng.standard_normal((2, S, n_new, Hkv, hd)).astype(np.float32)
    new[0, 0, 0, 0, :32] = 0.0                      # a block of zeros
    new[0, 0, 0, 1, :32] = np.linspace(-1, 1, 32)   # two values of the largest magnitude: the first one counts
    new[0, 0, 0, 2, :32] = np.linspace(1, -1, 32)
    tk = torch.from_numpy(new[0]).cuda().permute(0, 2, 1, 3)
    flat = torch.zeros(new[1].size + 2, dtype=torch.float32, device="cuda")
    flat[2:] = torch.from_numpy(new[1]).cuda().reshape(-1)
    tv = flat[2:].reshape(S, n_new, Hkv, hd).permute(0, 2, 1, 3)
    assert tv.data_ptr() % 16 == 8
    pos = torch.tensor([p0, ctx - 2], dtype=torch.int32, device="cuda")
    kv.append(1, tk, tv, pos=pos)
    torch.cuda.synchronize()
    for got, x in zip(kv.tensors(1, ctx), new):
        want = np.zeros((S, Hkv, ctx, hd // 32 * 18), np.uint8)
        enc = quantize_q4_0(x.transpose(0, 2, 1, 3))
        want[0, :, p0:p0 + n_new] = enc[0]
        n1 = min(2, n_new)
        want[1, :, ctx - 2:ctx - 2 + n1] = enc[1][:, :n1]
        assert np.array_equal(got.cpu().numpy(), want)
    assert not any(x.any() for x in kv.tensors(0, ctx))   # the other layer
    kv.close()


def test_append_round_trip_bound(b200):
    """Values in [-1, 1] come back within 0.2 (tests/test-kv-quant-roundtrip.cpp:192-195)."""
    rng = np.random.default_rng(7)
    x = rng.uniform(-1, 1, (1, 2, 40, 128)).astype(np.float32)
    kv = b200.KvCache(abi.Q4_0, 128, 2, n_layers=1, max_ctx=64)
    kv.append(0, torch.from_numpy(x).cuda(), torch.from_numpy(-x).cuda(), pos0=3)
    k, v = kv.read(0, 40, pos0=3, dtype=torch.float32)
    assert (k.cpu().numpy() - x).__abs__().max() <= 0.2 and (v.cpu().numpy() + x).__abs__().max() <= 0.2
    kv.close()


@pytest.mark.parametrize("amax", [1e-38, 1e-40, 1e-44])
def test_append_blocks_of_tiny_values(b200, amax):
    """Blocks whose 1/d leaves the range of a float: d is 0 in F16, so whatever the nibbles are, the values are zeros."""
    x = np.zeros((1, 1, 2, 64), np.float32)
    x[0, 0, 0, ::3], x[0, 0, 1, ::2], x[0, 0, 1, 1::4] = amax, amax, -amax
    kv = b200.KvCache(abi.Q4_0, 64, 1, n_layers=1, max_ctx=32)
    kv.append(0, torch.from_numpy(x).cuda(), torch.from_numpy(x).cuda())
    assert not any(t.any() for t in kv.read(0, 2, dtype=torch.float32))
    kv.close()


@pytest.mark.parametrize("type_", [abi.F16, abi.Q8_0, abi.Q4_0])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_read_rows(b200, orc, type_, hd):
    """Rows of every cache type as F16 and F32, from positions of their own per stream, some outside the cache (zeros); into strided
    outputs whose other bytes stay."""
    rng = np.random.default_rng(hd + type_)
    S, Hkv, ctx = 3, 2, 64
    x = rng.standard_normal((2, S, Hkv, ctx, hd)).astype(np.float32)
    kv = b200.KvCache(type_, hd, Hkv, n_layers=1, max_ctx=ctx, n_streams=S)
    kv.append(0, *(torch.from_numpy(y).cuda() for y in x))
    values = {abi.F16: lambda y: y.astype(np.float16).astype(np.float32), abi.Q8_0: lambda y: orc.dequantize_q8_0(orc.quantize_q8_0(y)),
              abi.Q4_0: lambda y: dequantize_q4_0(quantize_q4_0(y))}[type_](x)
    start, n = [0, 41, -5], 37
    want = np.zeros((2, S, Hkv, n, hd), np.float32)
    for s, p in enumerate(start):
        lo, hi = max(0, -p), min(n, ctx - p)
        want[:, s, :, lo:hi] = values[:, s, :, p + lo:p + hi]
    pos = torch.tensor(start, dtype=torch.int32, device="cuda")
    for got, ref in zip(kv.read(0, n, pos=pos, dtype=torch.float32), want):
        assert np.array_equal(got.cpu().numpy(), ref)
    for got, ref in zip(kv.read(0, n, pos=pos), want):
        assert got.dtype == torch.float16 and np.array_equal(got.cpu().numpy(), ref.astype(np.float16))
    wide = torch.full((2, S, n, Hkv, hd + 3), 7.0, dtype=torch.float16, device="cuda")   # rows on 2-byte boundaries
    out = tuple(w[..., 1:hd + 1].permute(0, 2, 1, 3) for w in wide)
    kv.read(0, n, pos=pos, out=out)
    for got, ref in zip(out, want):
        assert np.array_equal(got.cpu().numpy(), ref.astype(np.float16))
    assert (wide[..., 0] == 7).all() and (wide[..., hd + 1:] == 7).all()
    kv.close()


def test_copy_stream_of_a_q4_cache(b200):
    rng = np.random.default_rng(3)
    kv = b200.KvCache(abi.Q4_0, 128, 2, n_layers=1, max_ctx=64, n_streams=3)
    x = torch.from_numpy(rng.standard_normal((3, 2, 50, 128)).astype(np.float32)).cuda()
    kv.append(0, x, -x)
    before = kv.tensors(0, 64)[0].clone()
    kv.copy_stream(dst_stream=2, src_stream=0, n_rows=21)
    after = kv.tensors(0, 64)[0]
    assert torch.equal(after[2, :, :21], before[0, :, :21]) and torch.equal(after[2, :, 21:], before[2, :, 21:]) and torch.equal(after[:2], before[:2])
    kv.close()


# ---- attention ------------------------------------------------------------------------------------------------------

def _caches(rng, B, Hkv, L, hd):
    k, v = (random_q4_0(rng, (B, Hkv, L, hd)) for _ in "kv")
    return k, v, dequantize_q4_0(k), dequantize_q4_0(v)


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("gqa,Tq", [(1, 1), (4, 1), (8, 1), (1, 5), (3, 2), (4, 4), (2, 8)])
@pytest.mark.parametrize("L", [1, 16, 63, 64, 65, 300])
def test_decode_forms(b200, hd, gqa, Tq, L):
    """Ragged lengths (an empty stream among them) over caches of few and many tiles, one to sixteen query rows per KV head."""
    rng = np.random.default_rng(hd + 10 * gqa + Tq + L)
    B, Hkv = 3, 2
    k, v, kf, vf = _caches(rng, B, Hkv, L, hd)
    q = randn_f16(rng, (B, Hkv * gqa, Tq, hd))
    kw = dict(scale=hd ** -0.5, kv_len=np.array([L, 0, (L + 1) // 2], np.int32))
    got = gpu_op(b200, q, k, v, kv_type=abi.Q4_0, **kw)
    assert b200.lib().b200_last_kernel() == abi.KERNEL_DECODE_SPLIT
    assert not got[1].any()
    assert_close(got, attention_f64(q, kf, vf, **kw), "decode")


@pytest.mark.parametrize("hd,gqa,Tq", [(128, 4, 2), (128, 1, 7), (64, 2, 3), (64, 5, 3), (32, 2, 2)])
def test_decode_causal_with_lengths(b200, hd, gqa, Tq):
    """New tokens at the end of their stream's keys, and fewer of them than the launch has rows for."""
    rng = np.random.default_rng(hd + gqa + Tq)
    B, Hkv, L = 5, 2, 150
    k, v, kf, vf = _caches(rng, B, Hkv, L, hd)
    q = randn_f16(rng, (B, Hkv * gqa, Tq, hd))
    kw = dict(scale=hd ** -0.5, kv_len=np.array([150, 64, 0, Tq, 129], np.int32), q_len=np.array([Tq, Tq - 1, 0, Tq, 1], np.int32), causal=True)
    assert_close(gpu_op(b200, q, k, v, kv_type=abi.Q4_0, **kw), attention_f64(q, kf, vf, **kw), "causal decode")


@pytest.mark.parametrize("form", ["mask", "mask_rows_empty", "softcap", "alibi", "causal_scalar", "batch_broadcast", "f32_query"])
@pytest.mark.parametrize("kernel", [abi.KERNEL_NONE, abi.KERNEL_TILE_MMA])
def test_decode_other_forms(b200, orc, form, kernel):
    rng = np.random.default_rng(len(form))
    B, H, Hkv, Tq, L, hd = 2, 8, 2, 2, 200, 128
    Bk = 1 if form == "batch_broadcast" else B
    k, v, kf, vf = _caches(rng, Bk, Hkv, L, hd)
    q = randn_f16(rng, (B, H, Tq, hd))
    mask, kw = None, dict(scale=hd ** -0.5)
    if form.startswith("mask"):
        mask = np.where(rng.random((1, 1, Tq, L)) < 0.3, -np.inf, rng.standard_normal((1, 1, Tq, L)) * 0.5).astype(np.float16)
        if form == "mask_rows_empty":
            mask[0, 0, 1] = -np.inf
    elif form == "softcap":
        kw["softcap"] = 5.0
    elif form == "alibi":
        kw["max_bias"] = 4.0
        mask = -np.abs(np.arange(L)[None, None, None] - np.arange(Tq)[None, None, :, None]).astype(np.float16) * np.float16(0.1)
    elif form == "causal_scalar":
        kw.update(causal=True, n_past=L - Tq)
    elif form == "f32_query":
        q = q.astype(np.float32)
    b200.lib().b200_set_kernel_override(kernel)
    try:
        got = gpu_op(b200, q, k, v, mask, kv_type=abi.Q4_0, **kw)
    finally:
        b200.lib().b200_set_kernel_override(abi.KERNEL_NONE)
    assert_close(got, orc.flash_attn_ext(q, kf, vf, mask, gold=True, **kw), form)


def test_decode_index_lists(b200, orc):
    """Keys gathered through a list per batch entry equal the gathered rows."""
    rng = np.random.default_rng(5)
    B, Hkv, pool, stride, hd = 3, 2, 90, 64, 128
    k, v, kf, vf = _caches(rng, 1, Hkv, pool, hd)
    q = randn_f16(rng, (B, 4, 1, hd))
    index = np.stack([rng.permutation(pool)[:stride] for _ in range(B)]).astype(np.int32)
    lens = np.array([64, 1, 33], np.int32)
    got = gpu_op(b200, q, k, v, scale=0.1, kv_type=abi.Q4_0, kv_index=index, kv_len=lens)
    for b in range(B):
        rows = index[b, :lens[b]]
        assert_close(got[b:b + 1], attention_f64(q[b:b + 1], kf[:, :, rows], vf[:, :, rows], 0.1), f"list {b}")


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T,L,kw", [(40, 40, dict(causal=True)), (130, 300, dict(causal=True, n_past=170)), (257, 70, {})])
def test_prefill(b200, hd, T, L, kw):
    rng = np.random.default_rng(T + hd)
    k, v, kf, vf = _caches(rng, 2, 2, L, hd)
    q = randn_f16(rng, (2, 8, T, hd))
    got = gpu_op(b200, q, k, v, scale=hd ** -0.5, kv_type=abi.Q4_0, **kw)
    assert b200.lib().b200_last_kernel() == abi.KERNEL_PREFILL_TC5
    assert_close(got, attention_f64(q, kf, vf, hd ** -0.5, **kw), "prefill")


@pytest.mark.parametrize("shift", [0, 2, 8])
@pytest.mark.parametrize("T", [1, 33])
def test_strided_and_unaligned_caches(b200, shift, T):
    """A token-major cache whose rows do not follow one another, and bases off the 16-byte grid."""
    rng = np.random.default_rng(shift + T)
    B, Hkv, L, hd = 2, 3, 100, 128
    k, v, kf, vf = _caches(rng, B, Hkv, L, hd)
    views = []
    for x in (k, v):
        base = np.zeros(shift + B * L * Hkv * 72, np.uint8)
        view = base[shift:].reshape(B, L, Hkv, 72).transpose(0, 2, 1, 3)
        view[:] = x
        views.append(cuda_view(view, base))
    q = randn_f16(rng, (B, 6, T, hd))
    assert_close(gpu_op(b200, q, *views, scale=0.09, kv_type=abi.Q4_0), attention_f64(q, kf, vf, 0.09), "strided")


def test_host_buffers_and_static_scratch(b200):
    rng = np.random.default_rng(12)
    B, H, Hkv, L, hd = 4, 8, 2, 700, 128
    k, v, kf, vf = _caches(rng, B, Hkv, L, hd)
    q = randn_f16(rng, (B, H, 1, hd))
    ref = attention_f64(q, kf, vf, 0.1)
    host = b200.flash_attn_ext_host(*(torch.from_numpy(x) for x in (q, k, v)), scale=0.1, kv_type=abi.Q4_0)
    assert_close(host.numpy(), ref, "host buffers")
    tq, tk, tv = (torch.from_numpy(x).cuda() for x in (q, k, v))
    out = torch.empty((B, 1, H, hd), device="cuda")
    desc = [abi.from_torch(tq), abi.from_torch(tk, abi.Q4_0), abi.from_torch(tv, abi.Q4_0), abi.from_torch(out)]
    p = abi.Params(0.1, 0.0, 0.0, 0)
    assert b200.lib().b200_set_decode_splits(11) == 0
    try:
        rc = b200.lib().b200_fattn_launch_static(*(C.byref(d) for d in desc[:3]), None, C.byref(desc[3]), C.byref(p), None, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
    finally:
        b200.lib().b200_set_decode_splits(0)
    assert rc == 0
    assert_close(out.cpu().numpy(), ref, "static scratch")


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("splits", [1, 2, 3, 8, 12, 40])
def test_decode_split_counts(b200, hd, splits):
    """Splits that merge in clusters and through the workspace, ragged lengths that leave some of them without a tile."""
    rng = np.random.default_rng(splits)
    B, Hkv, L = 3, 2, 2600
    k, v, kf, vf = _caches(rng, B, Hkv, L, hd)
    q = randn_f16(rng, (B, Hkv * 4, 1, hd))
    kw = dict(scale=hd ** -0.5, kv_len=np.array([2600, 70, 1999], np.int32))
    assert b200.lib().b200_set_decode_splits(splits) == 0
    try:
        got = gpu_op(b200, q, k, v, kv_type=abi.Q4_0, **kw)
    finally:
        b200.lib().b200_set_decode_splits(0)
    assert_close(got, attention_f64(q, kf, vf, **kw), "splits")


def test_rows_behind_the_length_may_hold_anything(b200):
    """Bytes of rows at or beyond a stream's length do not reach its result: scales that are infinities and NaN, any nibbles."""
    rng = np.random.default_rng(99)
    B, Hkv, L, hd = 3, 2, 100, 128
    k, v, kf, vf = _caches(rng, B, Hkv, L, hd)
    lens = np.array([100, 37, 64], np.int32)
    for x in (k, v):
        for b in range(B):
            x[b, :, lens[b]:] = 0xFF                                         # NaN scales
            x[b, :, lens[b] + 1::2] = rng.integers(0, 256, x[b, :, lens[b] + 1::2].shape)
            x[b, 0, lens[b] + 2::3, :2] = np.array([0x00, 0x7C], np.uint8)   # infinite ones
    q = randn_f16(rng, (B, 8, 1, hd))
    got = gpu_op(b200, q, k, v, scale=0.1, kv_type=abi.Q4_0, kv_len=lens)
    assert_close(got, attention_f64(q, kf, vf, 0.1, kv_len=lens), "garbage behind the length")


def test_decode_loop_on_one_slab(b200):
    """Append and attend, step after step, on one cache: prompts, then tokens of every stream at positions and lengths that live on the
    device; compared with the definition at three steps."""
    rng = np.random.default_rng(31)
    S, H, Hkv, hd, T0, steps = 3, 8, 2, 128, 70, 40
    kv = b200.KvCache(abi.Q4_0, hd, Hkv, n_layers=1, max_ctx=T0 + steps, n_streams=S)
    pre = rng.standard_normal((2, S, Hkv, T0, hd)).astype(np.float32)
    kv.append(0, *(torch.from_numpy(x).cuda() for x in pre))
    len0 = np.array([T0, T0 - 9, 1], np.int32)
    pos = torch.from_numpy(len0.copy()).cuda()
    kv_len = pos + 1
    new = rng.standard_normal((2, steps, S, Hkv, 1, hd)).astype(np.float32)
    q = randn_f16(rng, (steps, S, H, 1, hd))
    dn, dq = torch.from_numpy(new).cuda(), torch.from_numpy(q).cuda()
    k, v = kv.tensors(0, T0 + steps)
    outs = []
    for t in range(steps):
        kv.append(0, dn[0, t], dn[1, t], pos=pos)
        outs.append(b200.flash_attn_ext(dq[t], k, v, scale=hd ** -0.5, kv_type=abi.Q4_0, kv_len=kv_len))
        pos += 1
        kv_len += 1
    torch.cuda.synchronize()
    for t in (0, 17, steps - 1):
        rows = np.zeros((2, S, Hkv, T0 + steps, hd), np.float32)
        for s in range(S):
            n = int(len0[s])
            rows[:, s, :, :n] = pre[:, s, :, :n]
            rows[:, s, :, n:n + t + 1] = new[:, :t + 1, s, :, 0].transpose(0, 2, 1, 3)
        kf, vf = dequantize_q4_0(quantize_q4_0(rows))
        assert_close(outs[t].cpu().numpy(), attention_f64(q[t], kf, vf, hd ** -0.5, kv_len=len0 + t + 1), f"step {t}")
    assert b200.lib().b200_device_status() == 0
    kv.close()


def test_captured_step_follows_lengths(b200):
    """A step captured into a graph and replayed: positions and lengths are read on the device."""
    rng = np.random.default_rng(8)
    S, H, Hkv, hd, ctx = 2, 8, 2, 128, 96
    kv = b200.KvCache(abi.Q4_0, hd, Hkv, n_layers=1, max_ctx=ctx, n_streams=S)
    rows = rng.standard_normal((2, S, Hkv, ctx, hd)).astype(np.float32)
    pos = torch.zeros(S, dtype=torch.int32, device="cuda")
    kv_len = torch.zeros(S, dtype=torch.int32, device="cuda")
    new = torch.zeros((2, S, Hkv, 1, hd), device="cuda")
    q = torch.from_numpy(randn_f16(rng, (S, H, 1, hd))).cuda()
    k, v = kv.tensors(0, ctx)

    def step():
        kv.append(0, new[0], new[1], pos=pos)
        return b200.flash_attn_ext(q, k, v, scale=0.1, kv_type=abi.Q4_0, kv_len=kv_len)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t in range(70):
        new.copy_(torch.from_numpy(rows[:, :, :, t:t + 1]))
        pos.fill_(t)
        kv_len.copy_(torch.tensor([t + 1, max(0, t - 3)], dtype=torch.int32))
        graph.replay()
    torch.cuda.synchronize()
    kf, vf = dequantize_q4_0(quantize_q4_0(rows))
    assert_close(out.cpu().numpy(), attention_f64(q.cpu().numpy(), kf, vf, 0.1, kv_len=[70, 66]), "replayed step")
    kv.close()


def test_tensors_keep_the_cache_alive(b200):
    kv = b200.KvCache(abi.Q4_0, 64, 1, n_layers=1, max_ctx=32)
    x = torch.randn((1, 1, 4, 64), device="cuda")
    kv.append(0, x, x)
    k, _ = kv.tensors(0, 4)
    want = quantize_q4_0(x.cpu().numpy())
    del kv
    import gc
    gc.collect()
    junk = [torch.zeros(1 << 16, device="cuda") for _ in range(8)]
    assert np.array_equal(k.cpu().numpy(), want) and junk


# ---- the kernel of the serving form: at most 8 query rows per KV head, head_dim 64 / 128 -----------------------------

# Its result is that of 32-bit arithmetic.  A score is a sum of hd products of exact operands, accumulated in fp32: off by some 2^-22 of
# the sum of their magnitudes, which for N(0,1) operands is up to 2^3 in log2 units: 2^-19, and so is P.  Weights and the values' sums add
# 2^-21 each.  An output is a weighted mean in which these errors are independent: relative L2 2^-18 and less.  2^-17 is allowed.
EXACT_REL = 2.0 ** -17


def _exact(got, ref, what):
    assert np.isfinite(got).all(), what
    assert errors(got, ref)[1] <= EXACT_REL, f"{what}: {errors(got, ref)}"


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("gqa,Tq", [(1, 1), (3, 1), (4, 1), (1, 5), (8, 1), (2, 3)])
@pytest.mark.parametrize("B,L", [(1, 97), (3, 700), (40, 333), (2, 9001)])
def test_serving_form_is_exact(b200, hd, gqa, Tq, B, L):
    rng = np.random.default_rng(hd + gqa + Tq + L)
    Hkv = 5
    k, v, kf, vf = _caches(rng, B, Hkv, L, hd)
    q = randn_f16(rng, (B, Hkv * gqa, Tq, hd))
    kw = dict(scale=hd ** -0.5, kv_len=rng.integers(0, L + 1, B).astype(np.int32))
    kw["kv_len"][0] = L
    _exact(gpu_op(b200, q, k, v, kv_type=abi.Q4_0, **kw), attention_f64(q, kf, vf, **kw), "plain")
    if Tq > 1:
        kw.update(causal=True, q_len=np.minimum(kw["kv_len"], rng.integers(1, Tq + 1, B)).astype(np.int32))
        _exact(gpu_op(b200, q, k, v, kv_type=abi.Q4_0, **kw), attention_f64(q, kf, vf, **kw), "causal")


@pytest.mark.parametrize("case", ["tiny_q", "huge_q", "mixed_q", "tiny_v", "huge_v", "mixed_v", "one_key_wins", "growing_scores", "f32_q", "negative_scale"])
@pytest.mark.parametrize("gqa", [4, 8])
def test_serving_form_keeps_its_bits(b200, case, gqa):
    """Query rows and value blocks of any magnitude, maxima that keep growing, scales that force the weights' range down."""
    rng = np.random.default_rng(len(case) + gqa)
    B, Hkv, L, hd, scale = 2, 2, 500, 128, 128 ** -0.5
    kx, vx = (rng.standard_normal((B, Hkv, L, hd)).astype(np.float32) for _ in "kv")
    q = rng.standard_normal((B, Hkv * gqa, 1, hd)).astype(np.float32)
    if case == "tiny_q":
        q, scale = q * 1e-5, scale * 1e5
    elif case == "huge_q":
        q, scale = q * 5000, scale / 5000
    elif case == "mixed_q":
        q *= 10.0 ** rng.integers(-4, 1, q.shape)
    elif case == "tiny_v":
        vx *= 1e-3
    elif case == "huge_v":
        vx *= 9000
    elif case == "mixed_v":
        vx[:, :, ::37] *= 400
    elif case == "one_key_wins":
        kx[:, 0, 333] = 6 * np.sign(q[:, 0, 0])
    elif case == "growing_scores":
        kx = (0.02 * np.arange(L)[:, None] * np.sign(q[:, ::gqa]) * rng.uniform(0.5, 1, kx.shape)).astype(np.float32)
    elif case == "negative_scale":
        scale = -scale
    k, v = quantize_q4_0(kx), quantize_q4_0(vx)
    kf, vf = dequantize_q4_0(k), dequantize_q4_0(v)
    q = q if case == "f32_q" else q.astype(np.float16)
    got = gpu_op(b200, q, k, v, scale=scale, kv_type=abi.Q4_0)
    ref = attention_f64(q, kf, vf, scale)
    # scores of 2^8 (growing) or 2^5 (one key) in log2 units: 2^-24 of them more; a Q of 1e-5 has 8 bits below F16's smallest value, all of them kept
    bound = EXACT_REL * {"growing_scores": 16, "one_key_wins": 4, "mixed_v": 2}.get(case, 1)
    assert np.isfinite(got).all() and errors(got, ref)[1] <= bound, errors(got, ref)


@pytest.mark.parametrize("shift", [0, 4, 8, 12])
def test_serving_form_on_word_boundaries(b200, shift):
    """Heads that start anywhere on a 4-byte boundary: rows of 36 bytes, odd row counts, shifted bases of K alone."""
    rng = np.random.default_rng(shift)
    for hd, L in ((64, 101), (128, 101), (128, 64)):
        k, v, kf, vf = _caches(rng, 2, 3, L, hd)
        base = np.zeros(shift + k.size, np.uint8)
        base[shift:] = k.reshape(-1)
        q = randn_f16(rng, (2, 6, 1, hd))
        got = gpu_op(b200, q, cuda_view(base[shift:].reshape(k.shape), base), v, scale=0.1, kv_type=abi.Q4_0)
        _exact(got, attention_f64(q, kf, vf, 0.1), f"{hd} {L}")


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("gqa,Tq", [(4, 4), (1, 9), (2, 8), (3, 5), (13, 1)])
@pytest.mark.parametrize("splits", [0, 2, 7, 20])
def test_nine_to_sixteen_rows(b200, hd, gqa, Tq, splits):
    """A KV head's rows in two CTAs: plain, causal with ragged row counts, a scalar bound, every form of the merge."""
    rng = np.random.default_rng(hd + gqa + Tq + splits)
    B, Hkv, L = 3, 2, 1700
    k, v, kf, vf = _caches(rng, B, Hkv, L, hd)
    q = randn_f16(rng, (B, Hkv * gqa, Tq, hd))
    lens = np.array([L, 0, 777], np.int32)
    forms = [dict(kv_len=lens), dict(kv_len=lens, q_len=np.array([Tq, 0, max(1, Tq - 2)], np.int32), causal=True), dict(causal=True, n_past=L - Tq - 5)]
    assert b200.lib().b200_set_decode_splits(splits) == 0
    try:
        for kw in forms:
            got = gpu_op(b200, q, k, v, scale=hd ** -0.5, kv_type=abi.Q4_0, **kw)
            assert b200.lib().b200_last_kernel() == abi.KERNEL_DECODE_SPLIT
            _exact(got, attention_f64(q, kf, vf, hd ** -0.5, **kw), str(kw.keys()))
    finally:
        b200.lib().b200_set_decode_splits(0)


@pytest.mark.parametrize("gqa,Tq", [(1, 4), (2, 4), (4, 4)])
def test_query_rows_behind_their_count_may_hold_anything(b200, gqa, Tq):
    """NaN and infinities in padding rows of Q: zeros there, and nothing of them in the other rows."""
    rng = np.random.default_rng(gqa)
    B, Hkv, L, hd = 3, 2, 140, 128
    k, v, kf, vf = _caches(rng, B, Hkv, L, hd)
    q = randn_f16(rng, (B, Hkv * gqa, Tq, hd))
    q_len, kv_len = np.array([1, 0, 3], np.int32), np.array([140, 9, 77], np.int32)
    for b in range(B):
        q[b, :, q_len[b]:] = np.nan
        q[b, ::2, q_len[b]:] = np.inf
    for causal in (False, True):
        kw = dict(scale=0.1, kv_len=kv_len, q_len=q_len, causal=causal)
        got = gpu_op(b200, q, k, v, kv_type=abi.Q4_0, **kw)
        for b in range(B):
            assert not got[b, q_len[b]:].any()
        _exact(got, attention_f64(q, kf, vf, **kw), "padding rows")


def test_a_query_that_is_no_number_stays_by_itself(b200):
    """A row of NaN gives NaN, the rows that share its keys and its CTA do not change."""
    rng = np.random.default_rng(77)
    k, v, kf, vf = _caches(rng, 1, 2, 300, 128)
    q = randn_f16(rng, (1, 8, 1, 128))
    want = gpu_op(b200, q, k, v, scale=0.1, kv_type=abi.Q4_0)
    q[0, 2, 0, 5] = np.nan
    got = gpu_op(b200, q, k, v, scale=0.1, kv_type=abi.Q4_0)
    assert np.isnan(got[0, 0, 2]).all()
    keep = [h for h in range(8) if h != 2]
    assert np.array_equal(got[0, 0, keep], want[0, 0, keep])


def test_two_streams_and_two_graphs_at_once(b200):
    """Launches with splits of their own on two streams, and two graphs of different lengths over one cache replayed in turn."""
    rng = np.random.default_rng(5)
    k, v, kf, vf = _caches(rng, 1, 8, 5000, 128)
    dk, dv = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
    qs = [torch.from_numpy(randn_f16(rng, (1, 32, 1, 128))).cuda() for _ in range(2)]
    lens = [torch.tensor([n], dtype=torch.int32, device="cuda") for n in (5000, 1234)]
    streams, outs, graphs = [torch.cuda.Stream() for _ in range(2)], [None, None], []
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i] = b200.flash_attn_ext(qs[i], dk, dv, scale=0.1, kv_type=abi.Q4_0, kv_len=lens[i])
    torch.cuda.synchronize()
    for i in range(2):
        ref = attention_f64(qs[i].cpu().numpy(), kf, vf, 0.1, kv_len=lens[i].cpu().numpy())
        _exact(outs[i].cpu().numpy(), ref, f"stream {i}")
    held = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(b200.flash_attn_ext(qs[i], dk, dv, scale=0.1, kv_type=abi.Q4_0, kv_len=lens[i]))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(held[i], outs[i])
    assert b200.lib().b200_device_status() == 0


@pytest.mark.parametrize("size", [2.5, 40.0, 5000.0])
@pytest.mark.parametrize("gqa,Tq", [(4, 1), (4, 3)])
def test_serving_form_with_large_values(b200, size, gqa, Tq):
    """Block scales of 2 and more: the range of the weights goes down by as much as they need, and not by more."""
    rng = np.random.default_rng(int(size) + Tq)
    kx, vx = (rng.standard_normal((1, 2, 4212, 128)).astype(np.float32) for _ in "kv")
    vx *= size * rng.choice([0.05, 1.0], (1, 2, 4212, 1)).astype(np.float32)
    k, v = quantize_q4_0(kx), quantize_q4_0(vx)
    kf, vf = dequantize_q4_0(k), dequantize_q4_0(v)
    q = randn_f16(rng, (1, 2 * gqa, Tq, 128))
    for splits in (1, 0):
        assert b200.lib().b200_set_decode_splits(splits) == 0
        try:
            got = gpu_op(b200, q, k, v, scale=0.1, kv_type=abi.Q4_0)
        finally:
            b200.lib().b200_set_decode_splits(0)
        _exact(got, attention_f64(q, kf, vf, 0.1), f"{splits} splits")
