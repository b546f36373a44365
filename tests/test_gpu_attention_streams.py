"""The streams that the attention and cache calls are given: those of the tensors' device
take the native route, those of another device are refused."""
import pytest

pytestmark = pytest.mark.gpu


def _cache(pkg, dev, B=2):
    import torch
    gen = torch.Generator(device=dev).manual_seed(0)
    k, v = (torch.randn(2, B, 2, 64, 64, generator=gen, device=dev).half() for _ in range(2))
    counts = torch.tensor([[10, 20], [12, 20]], dtype=torch.int32, device=dev)[:, :B].contiguous()
    return pkg.KVCache.from_tensors(k, v, counts)


def test_streams_of_another_device(pkg, dev):
    import torch

    class Elsewhere:
        device = torch.device("cuda", 1)
        cuda_stream = torch.cuda.current_stream(dev).cuda_stream

    q = torch.randn(2, 3, 4, 64, device=dev).half()
    k = q[:, :, :2]
    out, cache, s = torch.empty_like(q), _cache(pkg, dev), Elsewhere()
    tracked = pkg.KVCache(1, 1, 2, 16, 64, track_weights=True, device=dev)
    pkg.kv_evict(tracked, 8, sinks=1, recent=1)      # scratch is there
    pkg.attention_cached(q, cache, 0, 0.1)
    torch.cuda.synchronize()
    for call in (lambda: pkg.attention(q, k, k, 0.1, out=out, stream=s),
                 lambda: pkg.attention(q, k, k, 0.1, stream=s),
                 lambda: pkg.kv_append(q, k, k, cache, 0, q_out=out, stream=s),
                 lambda: pkg.attention_cached(q, cache, 0, 0.1, out=out, stream=s),
                 lambda: pkg.kv_accept(cache, 2, stream=s),
                 lambda: pkg.kv_evict(tracked, 8, sinks=1, recent=1, stream=s)):
        with pytest.raises(ValueError, match="stream of cuda:1"):
            call()
    torch.cuda.synchronize()
    assert cache.length.tolist() == [10, 20]


def test_streams_of_the_same_device(pkg, dev):
    """A stream object and its number make the call in native code."""
    import torch
    if not pkg._native_tried:
        pkg._load_binding()
    q = torch.randn(2, 3, 4, 64, device=dev).half()
    k, out, cache = q[:, :, :2], torch.empty_like(q), _cache(pkg, dev)
    want = pkg.attention(q, k, k, 0.1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (s, s.cuda_stream, torch.cuda.ExternalStream(s.cuda_stream)):
        out.zero_()
        torch.cuda.synchronize()
        got = pkg._native.attention(q, k, k, 0.1, 0.0, None, 0, False, None, None, None, None, None, out, stream)
        assert got is out
        assert pkg._native.kv_accept(*cache._handle, 1, None, None, stream) is True
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert cache.length.tolist() == [13, 23]
