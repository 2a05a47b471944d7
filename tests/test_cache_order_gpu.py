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
