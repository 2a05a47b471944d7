"""The 4-bit cache and the pass that fills it where they can go wrong without the sizes of a tolerance showing it: bits of rows that were not turned,
values that are no numbers, bounds ahead of the first key, offsets past 32 bits."""
import numpy as np
import pytest
import torch

from crispasr_b200 import abi
from tests.q4_ref import attention_f64, dequantize_q4_0, quantize_q4_0, random_q4_0
from tests.util import gpu_op, randn_f16

pytestmark = pytest.mark.gpu

EXACT_REL = 2.0 ** -17   # tests/test_q4_gpu.py


def _awkward_rows(rng, shape):
    """Rows whose blocks have zeros only, largest values of both signs in every order and distance, one value, equal values, tiny ones."""
    x = rng.standard_normal(shape).astype(np.float32)
    b = x.reshape(-1, 32)
    for i in range(0, len(b)):
        kind = i % 9
        if kind == 0:
            b[i] = 0
        elif kind == 1:
            j, k = rng.choice(32, 2, replace=False)   # two of the largest magnitude, either sign first
            b[i, j], b[i, k] = 5.0, -5.0
        elif kind == 2:
            b[i, rng.integers(32)] = -7.0
        elif kind == 3:
            b[i, rng.integers(32)] = 7.0
        elif kind == 4:
            b[i] = np.where(rng.random(32) < 0.5, 2.0, -2.0)
        elif kind == 5:
            b[i] = 0
            b[i, rng.integers(32)] = rng.choice([-3.0, 3.0])
        elif kind == 6:
            j = 4 * rng.integers(8) + np.array([0, 3])   # the two of them in one lane
            b[i, j] = rng.permutation([6.0, -6.0])
    return x


@pytest.mark.parametrize("type_", [abi.F16, abi.Q8_0, abi.Q4_0])
@pytest.mark.parametrize("hd,neox", [(128, True), (64, True), (128, False), (64, False), (96, True), (32, True)])
@pytest.mark.parametrize("io", [torch.float32, torch.float16])
@pytest.mark.parametrize("Hkv,n,shift", [(1, 1, 0), (3, 7, 0), (5, 40, 0), (3, 7, 1)])
def test_rows_that_are_not_turned_are_appended_bit_for_bit(b200, type_, hd, neox, io, Hkv, n, shift):
    """With a frequency of zero and no norm, append_rope stores what append stores: K, whose lanes hold other values of a row than V's, too.  `shift`: rows off the
    16-byte grid."""
    rng = np.random.default_rng([type_, hd, Hkv, n])
    S = 2
    rows = []
    for x in (_awkward_rows(rng, (S, n, Hkv, hd)) for _ in "kv"):
        t = torch.from_numpy(x).cuda().to(io)
        if shift:
            wide = torch.zeros((S, n, Hkv, hd + shift), dtype=io, device="cuda")
            wide[..., shift:] = t
            t = wide[..., shift:]
        rows.append(t.permute(0, 2, 1, 3))
    kv, plain = (b200.KvCache(type_, hd, Hkv, n_layers=1, max_ctx=n + 40, n_streams=S) for _ in "ab")
    q = rows[0][:, :1]
    pos = torch.tensor([3, 31], dtype=torch.int32, device="cuda")
    got = kv.append_rope(0, q, *rows, neox=neox, rope_scale=0.0, pos=pos)
    assert torch.equal(got.float(), q.half().float())
    plain.append(0, *(x.float().contiguous() for x in rows), pos=pos)
    for which, (x, y) in enumerate(zip(kv.tensors(0, n + 40), plain.tensors(0, n + 40))):
        assert torch.equal(x, y), "KV"[which]   # (F16: as numbers, a zero may have either sign)
    if type_ == abi.Q4_0:
        want = quantize_q4_0(rows[0].float().cpu().numpy())
        have = kv.tensors(0, n + 40)[0].cpu().numpy()
        for s, p in enumerate((3, 31)):
            assert np.array_equal(have[s, :, p:p + n], want[s])
    kv.close(), plain.close()


@pytest.mark.parametrize("type_", [abi.Q8_0, abi.Q4_0])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("how", ["append", "append_rope"])
def test_values_that_are_no_numbers_stay_in_their_block(b200, type_, hd, how):
    """A NaN does not count for its block's scale and becomes some number of the block's range; the block's other values, and other
    blocks, are stored as if it were a zero.  A block of Q4_0 with an infinity reads as no numbers at all."""
    rng = np.random.default_rng(hd + type_)
    x = rng.standard_normal((1, 2, 40, hd)).astype(np.float32)
    bad = x.copy()
    where = rng.integers(0, hd, (2, 40))
    for h in range(2):
        for i in range(40):
            bad[0, h, i, where[h, i]] = np.nan
            x[0, h, i, where[h, i]] = 0
    bad[0, 1, 5, 8:16] = np.nan    # all values of a lane
    x[0, 1, 5, 8:16] = 0
    out = []
    for rows in (x, bad):
        kv = b200.KvCache(type_, hd, 2, n_layers=1, max_ctx=64)
        t = torch.from_numpy(rows).cuda()
        if how == "append":
            kv.append(0, t, t)
        else:   # (a rotation by nothing, of which only V has none: NaN times the sine's zero would reach the partner in K)
            kv.append_rope(0, None, t, t, rope_dims=0)
        out.append([y.cpu().numpy() for y in kv.read(0, 40, dtype=torch.float32)])
        kv.close()
    top = np.abs(x).reshape(1, 2, 40, hd // 32, 32).max(-1)
    for want, got in zip(*out):
        keep = ~np.isnan(bad)
        assert np.array_equal(got[keep], want[keep])
        assert np.isfinite(got).all()
        bound = np.repeat(top, 32, -1) * (1 + 2.0 ** -10)
        assert (np.abs(got) <= bound).all()
    if type_ != abi.Q4_0:
        return
    bad = x.copy()
    bad[0, 0, 3, 5], bad[0, 1, 7, 40] = np.inf, -np.inf
    kv = b200.KvCache(type_, hd, 2, n_layers=1, max_ctx=64)
    t = torch.from_numpy(bad).cuda()
    kv.append(0, t, t) if how == "append" else kv.append_rope(0, None, t, t, rope_dims=0)
    hit = np.zeros((1, 2, 40, hd), bool)
    hit[0, 0, 3, :32] = hit[0, 1, 7, 32:64] = True
    for want, got in zip(out[0], kv.read(0, 40, dtype=torch.float32)):
        got = got.cpu().numpy()
        assert not np.isfinite(got[hit]).any() and np.array_equal(got[~hit], want[~hit])
    kv.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("gqa,Tq", [(1, 3), (4, 1), (2, 4), (4, 4)])
@pytest.mark.parametrize("n_past", [-100, -4, -3, -2, -1, 0])
def test_causal_bounds_ahead_of_the_first_key(b200, hd, gqa, Tq, n_past):
    """Rows whose bound lies ahead of the first key see none and are zeros, the others what is left."""
    rng = np.random.default_rng(hd + gqa + Tq)
    B, Hkv, L = 2, 3, 200
    k, v = (random_q4_0(rng, (B, Hkv, L, hd)) for _ in "kv")
    q = randn_f16(rng, (B, Hkv * gqa, Tq, hd))
    for kw in (dict(), dict(kv_len=np.array([200, 1], np.int32))):
        kw.update(scale=0.1, causal=True, n_past=n_past)
        got = gpu_op(b200, q, k, v, kv_type=abi.Q4_0, **kw)
        assert b200.lib().b200_last_kernel() == abi.KERNEL_DECODE_SPLIT
        ref = attention_f64(q, dequantize_q4_0(k), dequantize_q4_0(v), **kw)
        empty = [i for i in range(Tq) if n_past + i < 0]
        assert not got[:, empty].any()
        assert np.isfinite(got).all() and np.linalg.norm(got - ref) <= EXACT_REL * np.linalg.norm(ref)


def test_bounds_ahead_of_the_first_key_by_lengths(b200):
    """More new rows than keys: the first ones' bounds lie ahead of the first key."""
    rng = np.random.default_rng(3)
    k, v = (random_q4_0(rng, (3, 2, 90, 128)) for _ in "kv")
    q = randn_f16(rng, (3, 8, 3, 128))
    kw = dict(scale=0.1, causal=True, kv_len=np.array([1, 2, 0], np.int32), q_len=np.array([3, 3, 2], np.int32))
    got = gpu_op(b200, q, k, v, kv_type=abi.Q4_0, **kw)
    ref = attention_f64(q, dequantize_q4_0(k), dequantize_q4_0(v), **kw)
    assert not got[0, :2].any() and not got[1, 0].any() and not got[2].any()
    assert np.isfinite(got).all() and np.linalg.norm(got - ref) <= EXACT_REL * np.linalg.norm(ref)


def test_offsets_past_32_bits(b200):
    """A cache of two streams of 31 million keys, 2.2 GB each per slab: rows appended, read and attended to at its far end, by bytes and by keys."""
    rng = np.random.default_rng(9)
    ctx, hd, n = 31_000_000, 128, 70
    kv = b200.KvCache(abi.Q4_0, hd, 1, n_layers=1, max_ctx=ctx, n_streams=2)
    assert ctx * 72 > 2 ** 31
    x = rng.standard_normal((2, 2, 1, n, hd)).astype(np.float32)
    q = np.abs(randn_f16(rng, (2, 4, 1, hd)))
    x[0] = np.abs(x[0]) + 0.5          # scores well above those of the zeros everywhere else
    at = np.array([ctx - n, ctx - n - 5], np.int32)
    pos = torch.from_numpy(at).cuda()
    tx = torch.from_numpy(x).cuda()
    kv.append(0, tx[0], tx[1], pos=pos)
    enc = [quantize_q4_0(y) for y in x]
    values = [dequantize_q4_0(e) for e in enc]
    for got, want in zip(kv.read(0, n, pos=pos, dtype=torch.float32), values):
        assert np.array_equal(got.cpu().numpy(), want)
    k, v = kv.tensors(0, ctx)
    assert np.array_equal(k[1, :, at[1]:at[1] + n].cpu().numpy(), enc[0][1])
    lens = torch.from_numpy(at + n).cuda()
    got = b200.flash_attn_ext(torch.from_numpy(q).cuda(), k, v, scale=1.0, kv_type=abi.Q4_0, kv_len=lens).cpu().numpy()
    # the zeros' keys: a score of 0 against more than 30 (2^-43 each, 2^25 of them: less than 2^-17 of a result)
    s = np.einsum("shtd,sgnd->shtn", q.astype(np.float64), values[0].astype(np.float64))
    assert s.max(-1).min() > 45
    ref = attention_f64(q, *values, 1.0)
    assert np.isfinite(got).all() and np.linalg.norm(got - ref) <= EXACT_REL * np.linalg.norm(ref) * (1 + np.abs(s).max() / 16)
    # one token at the far end by append_rope, its position that of its place
    kv.append_rope(0, None, tx[0][:, :, :1], tx[1][:, :, :1], pos=torch.tensor([ctx - 1, 0], dtype=torch.int32, device="cuda"), rope_scale=0.0)
    assert np.array_equal(k[0, :, ctx - 1].cpu().numpy(), enc[0][0, :, 0]) and np.array_equal(v[1, :, 0].cpu().numpy(), enc[1][1, :, 0])
    kv.close()
