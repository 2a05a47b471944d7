"""The decoder's attention block around a quantised KV cache, as measurable cases: attention over a cache of 4-bit blocks
(Q4_0), rows entering such a cache and being read back, and the pass ahead of it - the norm of each query and key head, the
rotation by position, and the new rows' way into the cache.

A case is a dict of plain values.  `prepare` makes what a runtime holds before the call, `run` is one pass: in plain torch
operations where `own` is false, through the library's entry points where it is true.  `work` is what a pass cannot do without,
`exact` its result from the definition in 64 bits.

A Q4_0 block holds 32 values in 18 bytes, {f16 d; 16 bytes}: value i (i < 16) is d * (low nibble of byte i - 8), value 16 + i is
d * (high nibble of byte i - 8).  A Q8_0 block holds them in 34 bytes, {f16 d; int8 q[32]}: value i is d * q[i].
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK_BYTES = {"q4_0": 18, "q8_0": 34}
DTYPE = {"f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # ---- attention over a Q4_0 cache, one new token per stream unless `rows` says more ----
        # One short dictation on a Canary-sized decoder (8 heads, no grouping): the smallest call, all latency.
        dict(name="q4_decode_1x8_97", kind="attend", streams=1, heads=8, kv_heads=8, hd=128, rows=1, keys=97, ragged=False, causal=False),
        # Eight resident streams of a Voxtral-mini-sized decoder: 375 audio, 32 prompt and 256 generated tokens.
        dict(name="q4_decode_8x32_663", kind="attend", streams=8, heads=32, kv_heads=8, hd=128, rows=1, keys=663, ragged=False, causal=False),
        # A server's batch of a Qwen3-ASR-sized decoder, two drafted tokens beside each stream's own, streams of every
        # length, some of them just freed.
        dict(name="q4_decode_64x16_ragged", kind="attend", streams=64, heads=16, kv_heads=8, hd=128, rows=3, keys=1501, ragged=True, causal=True),
        # One long recording: few heads, many keys.
        dict(name="q4_decode_1x32_65535", kind="attend", streams=1, heads=32, kv_heads=8, hd=128, rows=1, keys=65535, ragged=False, causal=False),
        # A full server: the largest call.
        dict(name="q4_decode_256x32_4096", kind="attend", streams=256, heads=32, kv_heads=8, hd=128, rows=1, keys=4096, ragged=True, causal=False),
        # Five beams over the encoder's rows of 16 windows of 30 s, kept in 4 bits (20 heads of 64).
        dict(name="q4_cross_16x20_1500", kind="attend", streams=16, heads=20, kv_heads=20, hd=64, rows=5, keys=1500, ragged=False, causal=False),
        # ---- rows into a Q4_0 cache ----
        # One token of 32 streams, and the attention of the step over it.
        dict(name="q4_step_32x32_535", kind="step", streams=32, heads=32, kv_heads=8, hd=128, keys=535),
        # The prompts of 16 streams enter, and are read back as F16 rows.
        dict(name="q4_prompt_16x407", kind="append", streams=16, kv_heads=8, hd=128, rows=407, past=0),
        # ---- norm, rotation and append in one pass ----
        # One token of one stream of a Qwen3-ASR-sized decoder, into an F16 cache.
        dict(name="rope_step_1x16", kind="rope_append", streams=1, heads=16, kv_heads=8, hd=128, rows=1, past=600, cache="f16", norm=True, neox=True, dims=128,
             base=1000000.0, io="f32", ragged=False),
        # The prompts of eight streams of a Voxtral-sized decoder (no norm), into a Q8_0 cache.
        dict(name="rope_prompt_8x1500", kind="rope_append", streams=8, heads=32, kv_heads=8, hd=128, rows=1500, past=0, cache="q8_0", norm=False, neox=True,
             dims=128, base=100000000.0, io="f32", ragged=True),
        # ---- norm and rotation alone, for callers with caches of their own ----
        # One token of 48 streams far into a session, adjacent pairs, half of each head rotated.
        dict(name="rope_qk_48x12", kind="rope", streams=48, heads=12, kv_heads=4, hd=64, rows=1, past=100000, norm=True, neox=False, dims=32, base=10000.0, io="f16"),
        # Long prompts of a few streams.
        dict(name="rope_qk_3x2777", kind="rope", streams=3, heads=32, kv_heads=8, hd=128, rows=2777, past=11, norm=True, neox=True, dims=128, base=10000.0, io="f32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "step", "append", "rope_append", "rope_append", "rope"])
    hd = rng.choice([64, 128, 128])
    if kind in ("attend", "step"):
        kv_heads, group = rng.choice([(8, 4), (8, 2), (8, 1), (4, 4), (20, 1), (2, 8), (5, 3)])
        streams = _log_int(rng, 1, 256)
        keys = _log_int(rng, 2, 65536)
        while streams * keys * kv_heads * hd > 256 * 4096 * 8 * 128 // 2:
            keys = max(2, keys // 2 + rng.randint(0, 1))
        if kind == "step":
            return dict(kind=kind, streams=streams, heads=kv_heads * group, kv_heads=kv_heads, hd=hd, keys=keys)
        rows = rng.randint(1, 8 // group)
        return dict(kind=kind, streams=streams, heads=kv_heads * group, kv_heads=kv_heads, hd=hd, rows=rows, keys=max(keys, rows),
                    ragged=rng.random() < 0.5, causal=rng.random() < 0.5)
    kv_heads, group = rng.choice([(8, 4), (8, 2), (8, 1), (4, 3), (1, 8)])
    streams, rows = _log_int(rng, 1, 64), _log_int(rng, 1, 3000)
    while streams * rows * kv_heads * group > 8 * 1500 * 32:
        rows = max(1, rows // 2)
    past = _log_int(rng, 1, 4000) - 1
    if kind == "append":
        return dict(kind=kind, streams=streams, kv_heads=kv_heads, hd=rng.choice([32, 64, 96, 128]), rows=rows, past=past)
    c = dict(kind=kind, streams=streams, heads=kv_heads * group, kv_heads=kv_heads, hd=hd, rows=rows, past=past, norm=rng.random() < 0.5,
             neox=rng.random() < 0.7, dims=rng.choice([hd, hd, hd // 2, hd - 16]), base=rng.choice([10000.0, 1000000.0]), io=rng.choice(["f32", "f16"]))
    if kind == "rope":
        return dict(c, past=rng.choice([0, 77, 40000, 1000000]))
    return dict(c, cache=rng.choice(["f16", "q8_0"] if rows * streams > 32 else ["f16", "q8_0", "q4_0"]), ragged=rng.random() < 0.5)


# ---- lengths of a case ----------------------------------------------------------------------------------------------

def _key_counts(c):
    """Valid keys of each stream (attend, step)."""
    n, S = c["keys"], c["streams"]
    if not c.get("ragged"):
        return [n] * S
    # every length up to the longest; each ninth stream has just been freed
    return [0 if s % 9 == 4 else n - s * n // (2 * S) for s in range(S)]


def _row_counts(c):
    """Valid new rows of each stream, or None where all are."""
    return [c["rows"] - s * c["rows"] // (2 * c["streams"]) for s in range(c["streams"])] if c.get("ragged") else None


def _row_bytes(kind, hd):
    return 2 * hd if kind == "f16" else hd // 32 * BLOCK_BYTES[kind]


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(c):
    hd, S = c["hd"], c["streams"]
    if c["kind"] in ("attend", "step"):
        keys, rows = sum(_key_counts(c)), c.get("rows", 1)
        nbytes = keys * c["kv_heads"] * 2 * _row_bytes("q4_0", hd) + S * rows * c["heads"] * hd * (2 + 4)
        if c["kind"] == "step":   # the new rows in F32; they are read as cache rows too, and counted above
            nbytes += S * c["kv_heads"] * 2 * (4 * hd + _row_bytes("q4_0", hd))
        return {"bytes": nbytes, "flops": 4.0 * keys * c["heads"] * hd * rows}
    counts = _row_counts(c)
    rows = sum(counts) if counts else S * c["rows"]
    if c["kind"] == "append":   # F32 in, blocks out; blocks in, F16 out
        n = rows * c["kv_heads"] * 2
        return {"bytes": n * (4 * hd + 2 * _row_bytes("q4_0", hd) + 2 * hd), "flops": 4.0 * n * hd}
    es, heads = 2 if c["io"] == "f16" else 4, c["heads"] + c["kv_heads"]
    flops = rows * heads * (6.0 * c["dims"] // 2 + (4.0 * hd if c["norm"] else 0.0))
    if c["kind"] == "rope":
        return {"bytes": rows * heads * hd * 2 * es, "flops": flops}
    nbytes = rows * (c["heads"] * hd * (es + 2) + c["kv_heads"] * 2 * (es * hd + _row_bytes(c["cache"], hd)))
    if c["cache"] != "f16":   # the new rows are read back as F16
        nbytes += S * c["rows"] * c["kv_heads"] * 2 * (_row_bytes(c["cache"], hd) + 2 * hd)
    return {"bytes": nbytes, "flops": flops}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _randn(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _random_blocks(g, shape, hd):
    """Rows of Q4_0 blocks as quantising N(0,1) rows leaves them: the value of largest magnitude has nibble 0, the others follow
    the normal distribution, d = that value / -8."""
    n = hd // 32
    out = torch.empty(shape + (n, 18), dtype=torch.uint8, device="cuda")
    for part in out.view(-1, n, 18).split(1 << 22):   # a part of the rows at a time: the largest caches are made in place
        x = torch.randn((part.shape[0], n, 32), generator=g, device="cuda", dtype=torch.float16)
        m = torch.gather(x, -1, x.abs().argmax(-1, keepdim=True))
        d = m / -8
        q = (x / torch.where(d == 0, torch.ones_like(d), d) + 8.5).clamp(0, 15).to(torch.uint8)
        part[..., :2] = d.view(torch.uint8)
        part[..., 2:] = q[..., :16] | (q[..., 16:] << 4)
    return out.view(shape + (n * 18,))


def _cache(c, kind, rows, g=None):
    """What a runtime keeps of its cache: the K and V rows of one layer, and the handle that appends to them."""
    shape = (c["streams"], c["kv_heads"], rows)
    if own:
        import crispasr_b200 as b200
        from crispasr_b200 import abi
        handle = b200.KvCache({"f16": abi.F16, "q8_0": abi.Q8_0, "q4_0": abi.Q4_0}[kind], c["hd"], c["kv_heads"], 1, rows, c["streams"])
        k, v = handle.tensors(0, rows)
    else:
        handle = None
        k, v = (torch.zeros(shape + ((c["hd"],) if kind == "f16" else (_row_bytes(kind, c["hd"]),)), dtype=torch.float16 if kind == "f16" else torch.uint8,
                            device="cuda") for _ in "kv")
    if g is not None:
        for x in (k, v):
            x.copy_(_random_blocks(g, shape, c["hd"]))
    return handle, k, v


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    S, hd, rows = c["streams"], c["hd"], c.get("rows", 1)
    st = dict(case=c)

    def lengths(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    # the projections leave token-major rows
    def projected(heads, dtype=torch.float32):
        return _randn(g, (S, rows, heads, hd), dtype).permute(0, 2, 1, 3)

    if c["kind"] in ("attend", "step"):
        counts = _key_counts(c)
        st["kv_len"] = lengths(counts)
        st["q"] = projected(c["heads"], torch.float16)
        if c["kind"] == "attend":
            st["k"], st["v"] = (_random_blocks(g, (S, c["kv_heads"], c["keys"]), hd) for _ in "kv")
            if c["causal"]:   # all the new tokens of a stream, or as many as it has keys
                st["q_len"] = lengths([min(rows, n) for n in counts])
        else:
            st["handle"], st["k"], st["v"] = _cache(c, "q4_0", c["keys"], g)
            st["pos"] = st["kv_len"] - 1
            st["new"] = [projected(c["kv_heads"]) for _ in "kv"]
        return st
    # new rows start anywhere in the last rows of the past
    st["pos"] = lengths([max(0, c["past"] - s % 7) for s in range(S)])
    if c["kind"] == "append":
        st["handle"], st["k"], st["v"] = _cache(c, "q4_0", c["past"] + rows)
        st["new"] = [projected(c["kv_heads"]) for _ in "kv"]
        return st
    st["q"], k_new, v_new = (projected(n, DTYPE[c["io"]]) for n in (c["heads"], c["kv_heads"], c["kv_heads"]))
    st["norms"] = [1.0 + 0.1 * _randn(g, (hd,)) for _ in "qk"] if c["norm"] else [None, None]
    st["new"] = [k_new, v_new]
    if c["kind"] == "rope_append":
        st["handle"], st["k"], st["v"] = _cache(c, c["cache"], c["past"] + rows)
        if c["ragged"]:
            st["n_rows"] = lengths(_row_counts(c))
    return st


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _values(rows, kind):
    """Cache rows as the F32 values they stand for."""
    if kind == "f16":
        return rows.float()
    n = rows.shape[-1] // BLOCK_BYTES[kind]
    b = rows.reshape(rows.shape[:-1] + (n, BLOCK_BYTES[kind]))
    d = b[..., :2].contiguous().view(torch.float16).float()
    q = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).float() - 8.0 if kind == "q4_0" else b[..., 2:].contiguous().view(torch.int8).float()
    return (d * q).reshape(rows.shape[:-1] + (n * 32,))


def _blocks(x, kind):
    """F32 rows as cache rows.  A Q4_0 block's d is its value of largest magnitude / -8 and a nibble trunc(x / d + 8.5), at most 15;
    a Q8_0 block's d is the largest magnitude / 127 and q = x / d rounded half away from zero.  1 / d is formed in 32 bits, the
    products in 64: they may lie next to the border of two nibbles."""
    if kind == "f16":
        return x.half()
    b = x.reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    if kind == "q4_0":
        d = torch.gather(b, -1, b.abs().argmax(-1, keepdim=True)) / -8.0
        inv = torch.where(d == 0, torch.zeros_like(d), 1.0 / d)
        q = torch.trunc(b.double() * inv.double() + 8.5).clamp(0, 15).to(torch.uint8)
        q = q[..., :16] | (q[..., 16:] << 4)
    else:
        d = b.abs().amax(-1, keepdim=True) / 127.0
        inv = torch.where(d == 0, torch.zeros_like(d), 1.0 / d)
        t = b * inv
        q = (torch.trunc(t.abs().double() + 0.5) * t.sign()).to(torch.int8).view(torch.uint8)
    out = torch.cat([d.half().view(torch.uint8), q], -1)
    return out.reshape(x.shape[:-1] + (-1,))


def _store(cache, rows, pos, counts=None):
    """rows (S, Hkv, n, w) -> cache rows pos[s] .. of each stream; rows at or beyond counts[s] stay out."""
    S, n = rows.shape[0], rows.shape[2]
    i = torch.arange(n, device="cuda")
    at = (pos.long()[:, None] + i).unsqueeze(1).unsqueeze(-1)
    at = at.expand(rows.shape)
    if counts is not None:
        live = (i < counts.long()[:, None]).view(S, 1, n, 1)
        rows = torch.where(live, rows, torch.gather(cache, 2, at))
    cache.scatter_(2, at, rows)


def _rows_at(cache, pos, n):
    at = (pos.long()[:, None] + torch.arange(n, device="cuda")).view(pos.shape[0], 1, n, 1)
    return torch.gather(cache, 2, at.expand(cache.shape[:2] + (n, cache.shape[-1])))


def _attention(st, hd):
    q = st["q"].float()
    S, H, T, _ = q.shape
    k, v = _values(st["k"], "q4_0"), _values(st["v"], "q4_0")
    Hkv, L = k.shape[1], k.shape[2]
    s = torch.matmul(q.reshape(S, Hkv, H // Hkv * T, hd), k.transpose(2, 3)).view(S, H, T, L) * (hd ** -0.5)
    key = torch.arange(L, device="cuda")
    kv_len = st["kv_len"].long().view(S, 1, 1, 1)
    seen = key < kv_len
    if "q_len" in st:   # new token i of a stream sees the keys up to its own, the last q_len of kv_len
        q_len = st["q_len"].long().view(S, 1, 1, 1)
        i = torch.arange(T, device="cuda").view(1, 1, T, 1)
        seen = seen & (key <= kv_len - q_len + i) & (i < q_len)
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, Hkv, H // Hkv * T, L), v).view(S, H, T, hd) / torch.where(total == 0, torch.ones_like(total), total)
    return o.transpose(1, 2).contiguous()


def _normed_rotated(x, weight, c, pos, counts=None):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight
    n, half = c["dims"], c["dims"] // 2
    freq = c["base"] ** (-2.0 * torch.arange(half, device="cuda", dtype=torch.float64) / n)
    at = pos.double()[:, None] + torch.arange(x.shape[2], device="cuda")
    angle = (at[..., None] * freq).unsqueeze(1)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if c["neox"]:
        a, b = y[..., :half], y[..., half:n]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = y[..., 0:n:2], y[..., 1:n:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    y = torch.cat([turned, y[..., n:]], -1)
    if counts is not None:
        live = torch.arange(x.shape[2], device="cuda") < counts.long()[:, None]
        y = torch.where(live[:, None, :, None], y, torch.zeros_like(y))
    return y


def _run_plain(st):
    c = st["case"]
    kind, rows = c["kind"], c.get("rows", 1)
    if kind == "attend":
        return _attention(st, c["hd"])
    if kind in ("step", "append"):
        for cache, new in zip((st["k"], st["v"]), st["new"]):
            _store(cache, _blocks(new, "q4_0"), st["pos"])
        if kind == "step":
            return _attention(st, c["hd"])
        return [_values(_rows_at(x, st["pos"], rows), "q4_0").half() for x in (st["k"], st["v"])]
    counts = st.get("n_rows")
    q = _normed_rotated(st["q"], st["norms"][0], c, st["pos"], counts)
    k = _normed_rotated(st["new"][0], st["norms"][1], c, st["pos"])
    if kind == "rope":
        return [q.to(st["q"].dtype), k.to(st["q"].dtype)]
    for cache, new in zip((st["k"], st["v"]), (k, st["new"][1].float())):
        _store(cache, _blocks(new, c["cache"]), st["pos"], counts)
    if c["cache"] == "f16":
        return [q.half(), st["k"], st["v"]]
    return [q.half()] + [_values(_rows_at(x, st["pos"], rows), c["cache"]).half() for x in (st["k"], st["v"])]


# ---- the library's calls --------------------------------------------------------------------------------------------

def _run_own(st):
    import crispasr_b200 as b200
    from crispasr_b200 import abi
    c = st["case"]
    kind = c["kind"]
    if kind == "attend":
        return b200.flash_attn_ext(st["q"], st["k"], st["v"], scale=c["hd"] ** -0.5, kv_type=abi.Q4_0, kv_len=st["kv_len"], q_len=st.get("q_len"), causal=c["causal"])
    if kind == "step":
        st["handle"].append(0, *st["new"], pos=st["pos"])
        return b200.flash_attn_ext(st["q"], st["k"], st["v"], scale=c["hd"] ** -0.5, kv_type=abi.Q4_0, kv_len=st["kv_len"])
    if kind == "append":
        st["handle"].append(0, *st["new"], pos=st["pos"])
        return list(st["handle"].read(0, c["rows"], pos=st["pos"]))
    turn = dict(q_norm=st["norms"][0], k_norm=st["norms"][1], eps=EPS, rope_dims=c["dims"], rope_base=c["base"], neox=c["neox"], pos=st["pos"])
    if kind == "rope":
        return list(b200.qk_norm_rope(st["q"], st["new"][0], **turn))
    q = st["handle"].append_rope(0, st["q"], *st["new"], n_rows=st.get("n_rows"), **turn)
    if c["cache"] == "f16":
        return [q, st["k"], st["v"]]
    return [q, *st["handle"].read(0, c["rows"], pos=st["pos"])]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _exact_rows(raw):
    """(n, hd / 32 * 18) bytes -> (n, hd) F64 values, byte by byte as the block is laid out."""
    n, nb = raw.shape[0], raw.shape[1] // 18
    out = torch.empty((n, nb, 2, 16), dtype=torch.float64, device=raw.device)
    for j in range(nb):
        block = raw[:, 18 * j:18 * j + 18]
        d = block[:, :2].contiguous().view(torch.float16).double()
        out[:, j, 0] = d * ((block[:, 2:] % 16).double() - 8)
        out[:, j, 1] = d * (torch.div(block[:, 2:], 16, rounding_mode="floor").double() - 8)
    return out.view(n, nb * 32)


def _exact_attention(q, k_rows, v_rows, kv_len, q_len, causal):
    """`k_rows(s, h)` and `v_rows(s, h)`: the F64 rows of one head of one stream."""
    S, H, T, hd = q.shape
    Hkv = H // q.group
    out = torch.zeros((S, T, H, hd), dtype=torch.float64, device="cuda")
    for s in range(S):
        n = int(kv_len[s])
        live = int(q_len[s]) if causal else T
        if n == 0 or live == 0:
            continue
        for h in range(Hkv):
            k, v = k_rows(s, h)[:n], v_rows(s, h)[:n]
            x = q.rows[s, h * q.group:(h + 1) * q.group, :live].double() @ k.T / math.sqrt(hd)
            if causal:
                last = n - live + torch.arange(live, device="cuda")
                x = x.masked_fill(torch.arange(n, device="cuda")[None, :] > last[:, None], -math.inf)
            out[s, :live, h * q.group:(h + 1) * q.group] = (torch.softmax(x, -1) @ v).transpose(0, 1)
    return out


class _Queries:
    def __init__(self, rows, kv_heads):
        self.rows, self.shape, self.group = rows, rows.shape, rows.shape[1] // kv_heads


def _exact_stored(x, kind):
    """F64 rows -> the F64 values that a cache row of them stands for (an F16 row: the values themselves, which it is a rounding of)."""
    if kind == "f16":
        return x.clone()
    b = x.reshape(-1, 32)
    top = b.abs().max(-1)
    if kind == "q4_0":
        d = b[torch.arange(b.shape[0], device=b.device), top.indices] / -8
        q = torch.floor(b / torch.where(d == 0, 1.0, d)[:, None] + 8.5).clamp(max=15) - 8
    else:
        d = top.values / 127
        t = b / torch.where(d == 0, 1.0, d)[:, None]
        q = torch.sign(t) * torch.floor(t.abs() + 0.5)
    return (d.half().double()[:, None] * q).view(x.shape)


def _exact_turned(x, weight, c, pos):
    """Norm and rotation of (S, heads, n, hd) rows, as a product of complex numbers."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + EPS) * weight.double()
    n = c["dims"]
    i = torch.arange(n // 2, dtype=torch.float64, device="cuda")
    at = pos.double().view(-1, 1, 1, 1) + torch.arange(x.shape[2], device="cuda").double().view(1, 1, -1, 1)
    angle = at * torch.exp(-2.0 * i / n * math.log(c["base"]))
    first, second = (i.long(), i.long() + n // 2) if c["neox"] else (2 * i.long(), 2 * i.long() + 1)
    z = torch.complex(y[..., first], y[..., second]) * torch.polar(torch.ones_like(angle), angle)
    out = y.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


def exact(case, seed):
    st = prepare(case, seed)
    c = st["case"]
    kind, rows = c["kind"], c.get("rows", 1)
    if kind in ("attend", "step"):
        new = [_exact_stored(x.double(), "q4_0") for x in st["new"]] if kind == "step" else None
        lens = st["kv_len"].tolist()

        def of(cache, which):
            def one(s, h):
                x = _exact_rows(cache[s, h])
                if new is not None:
                    x[lens[s] - 1] = new[which][s, h, 0]
                return x
            return one
        q_len = st["q_len"].tolist() if "q_len" in st else None
        return _exact_attention(_Queries(st["q"], c["kv_heads"]), of(st["k"], 0), of(st["v"], 1), lens, q_len, q_len is not None)
    if kind == "append":
        return [_exact_stored(x.double(), "q4_0") for x in st["new"]]
    counts = _row_counts(c) or [rows] * c["streams"]
    q = _exact_turned(st["q"], st["norms"][0], c, st["pos"])
    k = _exact_turned(st["new"][0], st["norms"][1], c, st["pos"])
    if kind == "rope":
        return [q, k]
    kv = [_exact_stored(k, c["cache"]), _exact_stored(st["new"][1].double(), c["cache"])]
    for s, n in enumerate(counts):
        for x in (q, *kv):
            x[s, :, n:] = 0
    if c["cache"] != "f16":
        return [q, *kv]
    whole = [torch.zeros(st["k"].shape, dtype=torch.float64, device="cuda") for _ in "kv"]
    for s, n in enumerate(counts):
        p = int(st["pos"][s])
        for x, y in zip(whole, kv):
            x[s, :, p:p + n] = y[s, :, :n]
    return [q, *whole]
