"""PagedKVCache against RawKVCache (the same codes, so the same attention to rounding) and against itself
after eviction, release and reuse of pages."""

import threading

import pytest
import torch

from prismkv_b200 import _lib
from prismkv_b200.cache import PagedKVCache, PrismKVBackend, PrismKVConfig, RawKVCache

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = 1e-4          # two fp32-grade kernels over the same codes: a few 1e-6 each at these sizes


def _kv(B, H, s, d, seed):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(B, H, s, d, generator=g).to(DEV) for _ in range(2))


@pytest.mark.parametrize("d,bits", [(64, (4, 4, 4)), (96, (3, 3, 2)), (128, (4, 4, 4))])
def test_matches_raw_cache(cuda_ready, d, bits):
    backend = PrismKVBackend(PrismKVConfig(*bits), head_dim=d)
    raw = RawKVCache(backend)
    cache = PagedKVCache(backend, 2, 2, num_pages=24, page_size=16, page_summaries=True, track_weights=True)
    q = torch.randn(2, 4, d, generator=torch.Generator().manual_seed(1)).to(DEV)
    for i, s in enumerate((37, 1, 1, 30, 16)):
        k, v = _kv(2, 2, s, d, i)
        raw.append(0, k, v)
        assert cache.append(0, k, v) == [raw.get_seq_length(0)] * 2
        want = raw.attention(0, q)
        got = cache.attention(0, q)
        assert (got - want).abs().max() <= TOL
        assert (cache.attention(0, q, top_pages=100) - want).abs().max() <= TOL
        assert cache.attention(0, q, top_pages=3, out_dtype=torch.bfloat16).shape == (2, 4, d)
    assert _lib.device_error() == 0
    # every call's weights sum to one per query head
    total = cache.get_weights(0).sum(-1)
    assert torch.allclose(total, torch.full_like(total, 2 * 15.0), atol=1e-3)
    fp = cache.memory_footprint()
    assert fp["codes_bytes"] == raw.memory_footprint()["codes_bytes"] and fp["pool_bytes"] > fp["codes_bytes"]
    with pytest.raises(ValueError, match="pages"):
        cache.append(0, *_kv(2, 2, 400, d, 9)[:2])


def test_ragged_append_release_and_reuse(cuda_ready):
    d = 96
    backend = PrismKVBackend(PrismKVConfig(), head_dim=d)
    cache = PagedKVCache(backend, 3, 2, num_pages=12, page_size=16, max_tokens=64)
    k, v = _kv(3, 2, 40, d, 0)
    assert cache.append(0, k, v, lengths=[40, 0, 17]) == [40, 0, 17]
    assert cache.free_pages(0) == 12 - 3 - 2
    q = torch.randn(3, 2, d, generator=torch.Generator().manual_seed(2)).to(DEV)
    out = cache.attention(0, q)
    assert (out[1] == 0).all()
    for b, n in ((0, 40), (2, 17)):
        raw = RawKVCache(backend)
        raw.append(0, k[b:b + 1, :, :n], v[b:b + 1, :, :n])
        assert (out[b] - raw.attention(0, q[b:b + 1])[0]).abs().max() <= TOL
    cache.release(0, 0)
    assert cache.get_seq_lengths(0) == [0, 0, 17] and cache.free_pages(0) == 10
    assert cache.append(0, k, v, lengths=[1, 40, 0]) == [1, 40, 17]
    again = cache.attention(0, q)
    assert torch.equal(again[2], out[2])
    raw = RawKVCache(backend)
    raw.append(0, k[1:2], v[1:2])
    assert (again[1] - raw.attention(0, q[1:2])[0]).abs().max() <= TOL
    for bad in (lambda: cache.append(0, k, v), lambda: cache.append(0, k[:2], v[:2]), lambda: cache.append(0, k, v, [1, 2]),
                lambda: cache.append(0, k, v, [41, 0, 0])):
        with pytest.raises(ValueError):
            bad()
    assert cache.get_seq_lengths(0) == [1, 40, 17]
    with pytest.raises(RuntimeError):
        cache.attention(0, q, top_pages=1)
    with pytest.raises(RuntimeError):
        cache.evict(0, 8)
    with pytest.raises(KeyError):
        cache.attention(1, q)
    assert _lib.device_error() == 0


def test_eviction_keeps_what_was_attended_to(cuda_ready):
    d = 96
    backend = PrismKVBackend(PrismKVConfig(), head_dim=d)
    cache = PagedKVCache(backend, 2, 2, num_pages=40, page_size=16, page_summaries=True, track_weights=True)
    k, v = _kv(2, 2, 200, d, 3)
    q = torch.randn(2, 4, d, generator=torch.Generator().manual_seed(4)).to(DEV)
    hot = [60, 61, 99, 130]
    for h in range(2):
        k[:, h, hot] = 3.0 * q[:, 2 * h:2 * h + 1] / q[:, 2 * h:2 * h + 1].norm(dim=-1, keepdim=True) * d ** 0.5 / 3
    cache.append(0, k, v, lengths=[200, 30])
    for _ in range(3):
        before = cache.attention(0, q)
    w = cache.get_weights(0).clone()
    assert cache.evict(0, 64, sinks=2, recent=20) == [64, 30]
    assert cache.free_pages(0) == 40 - 4 - 2
    w2 = cache.get_weights(0).clone()
    assert torch.equal(w2[1], w[1]) and (w2[0, :, 64:] == 0).all()
    for h in range(2):
        order = sorted(range(2, 180), key=lambda t: (-w[0, h, t].item(), t))[:42]
        kept = sorted([0, 1] + order + list(range(180, 200)))
        assert set(hot) <= set(kept)
        assert torch.equal(w2[0, h, :64], w[0, h, kept])
        raw = RawKVCache(backend)
        raw.append(0, k[:1, h:h + 1, kept], v[:1, h:h + 1, kept])
        got = cache.attention(0, q)[0, 2 * h:2 * h + 2]
        assert (got - raw.attention(0, q[:1, 2 * h:2 * h + 2])[0]).abs().max() <= TOL
    after = cache.attention(0, q)
    assert torch.equal(after[1], before[1])
    assert cache.evict(0, 64, sinks=2, recent=20) == [64, 30]           # nothing to do
    # the cache goes on growing
    cache.append(0, *_kv(2, 2, 10, d, 5))
    assert cache.get_seq_lengths(0) == [74, 40]
    full = cache.attention(0, q)
    assert (cache.attention(0, q, top_pages=5) - full).abs().max() <= TOL
    assert torch.isfinite(cache.attention(0, q, top_pages=3)).all()
    assert _lib.device_error() == 0


def test_calls_at_the_edges(cuda_ready):
    d = 96
    backend = PrismKVBackend(PrismKVConfig(), head_dim=d)
    cache = PagedKVCache(backend, 2, 2, num_pages=8, page_size=16, page_summaries=True, track_weights=True)
    k, v = _kv(2, 2, 5, d, 0)
    assert cache.append(0, k[:, :, :0], v[:, :, :0]) == [0, 0]            # no token yet
    q = torch.randn(2, 4, d, generator=torch.Generator().manual_seed(1)).to(DEV)
    assert (cache.attention(0, q) == 0).all()
    # a page count that cannot hold the first and last pages is refused at every length
    for top in (0, 1, -1):
        with pytest.raises(ValueError, match="top_pages"):
            cache.attention(0, q, top_pages=top)
    assert cache.append(0, k.cpu(), v.cpu()) == [5, 5]
    out = cache.attention(0, q)
    assert cache.append(0, k[:, :, :0], v[:, :, :0]) == [5, 5]
    assert torch.equal(cache.attention(0, q.cpu()), out)
    assert cache.evict(0, 5, sinks=0, recent=0) == [5, 5]
    assert cache.evict(0, 1, sinks=0, recent=1) == [1, 1]
    raw = RawKVCache(backend)
    raw.append(0, k[:, :, 4:], v[:, :, 4:])
    assert (cache.attention(0, q) - raw.attention(0, q)).abs().max() <= TOL
    assert _lib.device_error() == 0


def test_threads_share_a_cache(cuda_ready):
    """Attention waits while another thread moves the tokens (an eviction changes table, lengths and weights)."""
    d = 96
    backend = PrismKVBackend(PrismKVConfig(), head_dim=d)
    cache = PagedKVCache(backend, 1, 2, num_pages=8, page_size=16, track_weights=True)
    cache.append(0, *_kv(1, 2, 40, d, 0))
    q = torch.randn(1, 2, d, generator=torch.Generator().manual_seed(1)).to(DEV)
    want, got = cache.attention(0, q), []
    t = threading.Thread(target=lambda: got.append(cache.attention(0, q)))
    with cache._lock:
        t.start()
        t.join(0.5)
        assert t.is_alive()
    t.join(60)
    assert not t.is_alive() and torch.equal(got[0], want)


def test_a_codec_stays_on_its_device(cuda_ready):
    from prismkv_b200.codec import DeviceCodec

    codec = PrismKVBackend(PrismKVConfig(), head_dim=96).codec(torch.device(DEV))
    assert DeviceCodec(codec.host, torch.device("cuda")).device == codec._R.device
