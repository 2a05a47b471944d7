"""The KV cache and streams of the caller's own: what is ordered by the library, and what by the caller."""
import pytest
import torch

from crispasr_b200 import abi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", ["append", "append_rope", "copy"])
@pytest.mark.parametrize("type_", [abi.F16, abi.Q4_0])
def test_first_rows_of_a_new_cache_on_a_non_blocking_stream(b200, type_, how):
    """Rows written right after construction, on a stream that is ordered behind no other: nothing clears them afterwards.  The arena
    is large (gigabytes, whose clearing takes a millisecond) and the rows are its last ones."""
    S, Hkv, hd, ctx, layers = 4, 8, 128, 65536, 4 if type_ == abi.F16 else 8
    g = torch.Generator(device="cuda")
    g.manual_seed(type_)
    x = torch.randn((2, S, Hkv, 5, hd), generator=g, device="cuda")
    small = b200.KvCache(type_, hd, Hkv, n_layers=1, max_ctx=32, n_streams=S)
    small.append(0, x[0], x[1])
    want = [t.clone() for t in small.tensors(0, 5)]
    side = torch.cuda.Stream()   # (torch's are non-blocking)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            kv = b200.KvCache(type_, hd, Hkv, n_layers=layers, max_ctx=ctx, n_streams=S)
            if how == "append":
                kv.append(layers - 1, x[0], x[1], pos0=ctx - 5)
            elif how == "append_rope":   # a scale of zero turns nothing
                kv.append_rope(layers - 1, None, x[0], x[1], pos0=ctx - 5, rope_scale=0.0)
            else:
                for to, rows in zip(kv.tensors(layers - 1, ctx), want):
                    to[:, :, ctx - 5:].copy_(rows)
        torch.cuda.synchronize()
        for got, rows in zip(kv.tensors(layers - 1, ctx), want):
            assert torch.equal(got[:, :, ctx - 5:], rows)
            assert not got[:, :, :ctx - 5].any()
        kv.close()
        torch.cuda.synchronize()
    small.close()


def _calls(b200, side):
    """Each call that makes its results, on `side`: (results, all of one shape and type)."""
    S, H, n, hd = 2, 5, 8191, 128
    q = torch.randn((S, H, n, hd), device="cuda", dtype=torch.float16)
    kv = b200.KvCache(abi.Q8_0, hd, H, n_layers=1, max_ctx=n, n_streams=S)
    return {"qk_norm_rope": lambda: b200.qk_norm_rope(q, q, stream=side), "append_rope": lambda: (kv.append_rope(0, q, q, q, stream=side),),
            "read": lambda: kv.read(0, n, stream=side)}, q


@pytest.mark.parametrize("call", ["qk_norm_rope", "append_rope", "read"])
@pytest.mark.parametrize("handle", ["stream", "integer", "current"])
def test_results_come_from_the_pool_of_the_launch_stream(b200, call, handle):
    """A block that the current stream has given back, and may still be working on, is not handed to a launch on another stream."""
    side = torch.cuda.Stream()
    calls, like = _calls(b200, None if handle == "current" else side if handle == "stream" else side.cuda_stream)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    back = [torch.empty_like(like) for _ in range(2)]
    freed = {x.data_ptr() for x in back}
    del back
    results = calls[call]()
    at = {x.data_ptr() for x in results}
    assert (at <= freed) if handle == "current" else not at & freed
    torch.cuda.synchronize()
    del results
    with torch.cuda.stream(side):   # ... and goes back to that pool
        again = {torch.empty_like(like).data_ptr() for _ in range(1)}
    assert handle == "current" or again <= at
