"""Norm, rotation and append in one pass against the definition in 64 bits.

Tolerances: a row's values are computed in fp32 - the norm's sum (relative error below hd * 2^-24 at worst, a few 2^-24 in
practice), two products and a sum per value, cosine and sine to 2^-22 of one - so a rotated value is within
  8 * 2^-22 * |row|_inf * |w|_inf-ish  of the exact one: 4e-6 of the largest value of its row is used (2^-18).  An F16 result adds half
a step, 2^-11 of its value; a quantised row may in addition land on the other side of a border, one step of its block."""
import numpy as np
import pytest
import torch

from crispasr_b200 import abi
from tests.q4_ref import dequantize_q4_0, norm_rope_f64, quantize_q4_0
from tests.util import randn_f16

pytestmark = pytest.mark.gpu

FP32_ROW = 2.0 ** -18


def assert_rows(got, ref, f16, what):
    top = np.abs(ref).max(-1, keepdims=True)
    bound = FP32_ROW * top + (2.0 ** -11 * np.abs(ref) + 2.0 ** -25 if f16 else 1e-30)
    assert (np.abs(got.astype(np.float64) - ref) <= bound).all(), f"{what}: {np.abs(got - ref).max():.3e}"


def _rows(rng, shape, dtype):
    """Token-major rows as a projection leaves them, (S, heads, n, hd)."""
    S, H, n, hd = shape
    x = rng.standard_normal((S, n, H, hd)).astype(np.float32)
    t = torch.from_numpy(x).cuda().to(dtype)
    return t.permute(0, 2, 1, 3)


@pytest.mark.parametrize("hd,dims,neox", [(128, 128, True), (128, 128, False), (64, 64, True), (64, 32, True), (64, 30, False), (128, 96, True), (128, 2, False),
                                          (96, 96, True), (80, 64, True), (32, 32, False), (16, 16, True), (8, 8, False), (128, 0, True)])
@pytest.mark.parametrize("io", [torch.float32, torch.float16])
@pytest.mark.parametrize("norm", [False, True])
def test_qk_norm_rope_forms(b200, hd, dims, neox, io, norm):
    rng = np.random.default_rng(hd + dims + norm)
    S, n, H, Hkv = 3, 5, 7, 3
    q, k = _rows(rng, (S, H, n, hd), io), _rows(rng, (S, Hkv, n, hd), io)
    w = [rng.uniform(0.5, 1.5, hd).astype(np.float32) for _ in "qk"] if norm else [None, None]
    pos = np.array([0, 1234, 131071], np.int32)
    kw = dict(eps=1e-5, rope_dims=dims, rope_base=1e6, rope_scale=0.25, neox=neox, pos=torch.from_numpy(pos).cuda())
    if norm:
        kw.update(q_norm=torch.from_numpy(w[0]).cuda(), k_norm=torch.from_numpy(w[1]).cuda())
    for out_type in (torch.float32, torch.float16):
        got = b200.qk_norm_rope(q, k, out=torch.empty(q.shape, dtype=out_type, device="cuda"), k_out=torch.empty(k.shape, dtype=out_type, device="cuda"), **kw)
        for x, g, wx in zip((q, k), got, w):
            ref = norm_rope_f64(x.cpu().numpy(), wx, pos, n_dims=dims, base=1e6, scale=0.25, neox=neox, eps=1e-5)
            assert_rows(g.cpu().numpy(), ref, out_type == torch.float16, f"{x.shape}")


@pytest.mark.parametrize("p", [0, 1, 4095, 100000, 16777217, 2147483000, -77])
def test_far_positions(b200, p):
    """The angle's reduction is exact at every position."""
    rng = np.random.default_rng(abs(p) % 1000)
    x = _rows(rng, (1, 2, 3, 128), torch.float32)
    got, none = b200.qk_norm_rope(x, pos0=p)
    assert none is None
    y, pos = x.cpu().numpy(), [p]
    # the definition's own frequencies are doubles: at a position near 2^31 their 2^-53 is 2e-7 of a turn at most
    assert_rows(got.cpu().numpy(), norm_rope_f64(y, None, pos, n_dims=128), False, f"position {p}")


@pytest.mark.parametrize("scale", [-1.0, -0.25, -1e-30, 1e-30])
def test_negative_and_tiny_frequencies(b200, scale):
    """A negative turn is one less than a whole one; one too small to differ from it is none."""
    rng = np.random.default_rng(5)
    x = _rows(rng, (1, 2, 5, 64), torch.float32)
    got, _ = b200.qk_norm_rope(x, pos0=321, rope_scale=scale)
    assert_rows(got.cpu().numpy(), norm_rope_f64(x.cpu().numpy(), None, [321], n_dims=64, scale=scale), False, f"scale {scale}")


def test_norm_of_small_and_zero_rows(b200):
    x = torch.zeros((1, 1, 4, 64), device="cuda")
    x[0, 0, 1], x[0, 0, 2, 5], x[0, 0, 3] = 1e-4, 1e-3, 1e18
    w = torch.linspace(0.5, 2, 64, device="cuda")
    got, _ = b200.qk_norm_rope(x, q_norm=w, eps=1e-6, pos0=9)
    ref = norm_rope_f64(x.cpu().numpy(), w.cpu().numpy(), [9], n_dims=64)
    assert not got[0, 0, 0].any()
    assert_rows(got.cpu().numpy(), ref, False, "small rows")


def test_infinities_stay_where_they_are_not_rotated(b200):
    x = torch.ones((1, 1, 1, 64), device="cuda")
    x[..., 40], x[..., 50] = float("inf"), float("nan")
    for neox in (True, False):
        got, _ = b200.qk_norm_rope(x, rope_dims=32, neox=neox, pos0=3)
        assert torch.isfinite(got[..., :40]).all() and got[0, 0, 0, 40] == float("inf") and got[0, 0, 0, 50].isnan() and (got[..., 51:] == 1).all()


def test_in_place_strides_and_rows_behind_the_count(b200):
    """Rows of a fused projection rotated where they lie; rows at or beyond n_rows become zeros, what lies between the rows
    stays; rows off the 16-byte grid."""
    rng = np.random.default_rng(4)
    S, n, H, Hkv, hd = 3, 6, 4, 2, 64
    for dtype, pad in ((torch.float32, 0), (torch.float32, 1), (torch.float16, 4), (torch.float16, 3)):
        x = rng.standard_normal((S, n, H + Hkv + 1, hd + pad)).astype(np.float32)
        fused = torch.from_numpy(x).cuda().to(dtype)
        before = fused.cpu().numpy().copy()
        q, k = (fused[:, :, a:b, pad:].permute(0, 2, 1, 3) for a, b in ((0, H), (H, H + Hkv)))
        counts = torch.tensor([6, 0, 2], dtype=torch.int32, device="cuda")
        got = b200.qk_norm_rope(q, k, out=q, k_out=k, n_rows=counts, pos0=50)
        assert got[0].data_ptr() == q.data_ptr()
        after = fused.cpu().numpy()
        for a, b in ((0, H), (H, H + Hkv)):
            src = before[:, :, a:b, pad:].transpose(0, 2, 1, 3)
            ref = norm_rope_f64(src, None, [50] * S, n_dims=hd)
            for s, c in enumerate(counts.tolist()):
                ref[s, :, c:] = 0
            assert_rows(after[:, :, a:b, pad:].transpose(0, 2, 1, 3), ref, dtype == torch.float16, f"{dtype} {pad}")
        assert np.array_equal(after[:, :, -1], before[:, :, -1]) and np.array_equal(after[..., :pad], before[..., :pad])


def _cache_error_bound(ref, type_):
    """Half a step of the cache's type (and one more where the fp32 row lands on the other side of a border)."""
    if type_ == abi.F16:
        return 2.0 ** -11 * np.abs(ref) + 2.0 ** -25
    b = np.abs(ref).reshape(ref.shape[:-1] + (ref.shape[-1] // 32, 32)).max(-1, keepdims=True)
    step = b / (127 if type_ == abi.Q8_0 else 8)
    # d in F16 is off by 2^-11, times up to 127 or 8 steps; a Q4_0 value may in addition be cut at nibble 15, a step more
    extra = 127 * 2.0 ** -11 if type_ == abi.Q8_0 else 8 * 2.0 ** -11 + 0.5
    return np.broadcast_to(step * (0.5 + extra + 1e-3) + 1e-7, ref.shape[:-1] + (ref.shape[-1] // 32, 32)).reshape(ref.shape)


@pytest.mark.parametrize("type_", [abi.F16, abi.Q8_0, abi.Q4_0])
@pytest.mark.parametrize("hd,dims,neox", [(128, 128, True), (64, 64, False), (96, 48, True), (32, 32, True)])
@pytest.mark.parametrize("n", [1, 9, 130])
@pytest.mark.parametrize("io", [torch.float32, torch.float16])
def test_append_rope(b200, orc, type_, hd, dims, neox, n, io):
    """Rotated q, and the cache rows of K and V: near the definition, and V's the same bits as append's.  Streams at
    positions of their own, one of them running out of the cache, rows behind a count not stored."""
    rng = np.random.default_rng(hd + n + type_)
    S, H, Hkv, ctx = 3, 5, 2, 192
    q, k, v = (_rows(rng, (S, h, n, hd), io) for h in (H, Hkv, Hkv))
    w = [torch.from_numpy(rng.uniform(0.5, 1.5, hd).astype(np.float32)).cuda() for _ in "qk"]
    start, counts = [7, ctx - 2, 40], [n, n, max(0, n - 3)]
    pos, n_rows = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (start, counts))
    kv, plain = (b200.KvCache(type_, hd, Hkv, n_layers=2, max_ctx=ctx, n_streams=S) for _ in "ab")
    fill = torch.from_numpy(rng.standard_normal((S, Hkv, ctx, hd)).astype(np.float32)).cuda()
    for c in (kv, plain):
        c.append(1, fill, fill)
    got = kv.append_rope(1, q, k, v, q_norm=w[0], k_norm=w[1], rope_dims=dims, neox=neox, pos=pos, n_rows=n_rows)
    assert got.dtype == torch.float16 and got.shape == q.shape
    ref_q, ref_k = (norm_rope_f64(x.cpu().numpy(), y.cpu().numpy(), start, n_dims=dims, neox=neox) for x, y in zip((q, k), w))
    for s, c in enumerate(counts):
        ref_q[s, :, c:] = 0
    assert_rows(got.cpu().numpy(), ref_q, True, "q")
    before = plain.read(1, ctx, dtype=torch.float32)
    after = kv.read(1, ctx, dtype=torch.float32)
    plain.append(1, k.float(), v.float(), pos=pos)
    v_rows = plain.tensors(1, ctx)[1].cpu().numpy()
    for s, c in enumerate(counts):
        p, m = start[s], min(counts[s], ctx - start[s])
        gk = after[0][s, :, p:p + m].cpu().numpy()
        assert (np.abs(gk - ref_k[s, :, :m]) <= _cache_error_bound(ref_k[s, :, :m], type_) + FP32_ROW * np.abs(ref_k).max()).all()
        assert np.array_equal(kv.tensors(1, ctx)[1].cpu().numpy()[s, :, p:p + m], v_rows[s, :, p:p + m])
        for x, y in zip(before, after):   # the rows around
            assert torch.equal(x[s, :, :p], y[s, :, :p]) and torch.equal(x[s, :, p + m:], y[s, :, p + m:])
    kv.close(), plain.close()


def test_append_rope_without_q(b200):
    rng = np.random.default_rng(2)
    k, v = _rows(rng, (2, 3, 4, 64), torch.float32), _rows(rng, (2, 3, 4, 64), torch.float32)
    kv = b200.KvCache(abi.F16, 64, 3, n_layers=1, max_ctx=32, n_streams=2)
    assert kv.append_rope(0, None, k, v, pos0=11) is None
    got, got_v = kv.read(0, 4, pos0=11)
    assert_rows(got.cpu().numpy(), norm_rope_f64(k.cpu().numpy(), None, [11, 11], n_dims=64), True, "k")
    assert torch.equal(got_v, v.half())
    kv.close()


@pytest.mark.parametrize("type_", [abi.F16, abi.Q8_0, abi.Q4_0])
def test_decoder_loop(b200, type_):
    """A layer of a Qwen3-ASR-sized decoder as a runtime runs it: a ragged batch of prompts, causal attention over them, then single
    tokens - norm, rotation and append in one call, attention in the other, on a stream of its own.  The result is compared with the
    definition on the rows that the cache holds."""
    rng = np.random.default_rng(13)
    S, H, Hkv, hd, T, steps = 3, 8, 4, 128, 50, 12
    kv_type = None if type_ == abi.F16 else type_
    kv = b200.KvCache(type_, hd, Hkv, n_layers=1, max_ctx=T + steps, n_streams=S)
    w = [torch.from_numpy(rng.uniform(0.8, 1.2, hd).astype(np.float32)).cuda() for _ in "qk"]
    lens = np.array([T, 17, 33], np.int32)
    counts = torch.from_numpy(lens).cuda()
    prompt = [_rows(rng, (S, h, T, hd), torch.float32) for h in (H, Hkv, Hkv)]
    tokens = [[_rows(rng, (S, h, 1, hd), torch.float32) for h in (H, Hkv, Hkv)] for _ in range(steps)]
    zero = torch.zeros(S, dtype=torch.int32, device="cuda")
    turn = dict(q_norm=w[0], k_norm=w[1], rope_base=1e6)
    k, v = kv.tensors(0, T + steps)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        qr = kv.append_rope(0, *prompt, pos=zero, n_rows=counts, **turn)
        first = b200.flash_attn_ext(qr, k, v, scale=hd ** -0.5, kv_type=kv_type, kv_len=counts, q_len=counts, causal=True)
        pos, outs, queries = counts.clone(), [], []
        for new in tokens:
            queries.append(kv.append_rope(0, *new, pos=pos, **turn))
            pos = pos + 1
            outs.append(b200.flash_attn_ext(queries[-1], k, v, scale=hd ** -0.5, kv_type=kv_type, kv_len=pos))
    stream.synchronize()
    from tests.q4_ref import attention_f64
    from tests.util import assert_close
    kf, vf = (x.cpu().numpy() for x in kv.read(0, T + steps, dtype=torch.float32))
    ref_q = norm_rope_f64(prompt[0].cpu().numpy(), w[0].cpu().numpy(), [0] * S, n_dims=hd, base=1e6)
    for s, c in enumerate(lens):
        ref_q[s, :, c:] = 0
    assert_rows(qr.cpu().numpy(), ref_q, True, "prompt q")
    assert_close(first.cpu().numpy(), attention_f64(qr.cpu().numpy(), kf, vf, hd ** -0.5, kv_len=lens, q_len=lens, causal=True), "prompt")
    for t in (0, steps - 1):
        assert_close(outs[t].cpu().numpy(), attention_f64(queries[t].cpu().numpy(), kf, vf, hd ** -0.5, kv_len=lens + t + 1), f"token {t}")
    assert b200.lib().b200_device_status() == 0
    kv.close()
