"""PagedKVCache's pages and buffers on the GPU: eviction with few or no free pages, buffers in proportion to the
tokens, attention captured into a graph."""

import pytest
import torch

from prismkv_b200 import _lib
from prismkv_b200.cache import PagedKVCache, PrismKVBackend, PrismKVConfig, RawKVCache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _kv(B, H, s, d, seed):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(B, H, s, d, generator=g).to(DEV) for _ in range(2))


def _q(B, H, d, seed=1):
    return torch.randn(B, H, d, generator=torch.Generator().manual_seed(seed)).to(DEV)


def _filled(num_pages, lengths, seed=3):
    """A cache of 2 KV heads that has attended once, and what it holds."""
    backend = PrismKVBackend(PrismKVConfig(), head_dim=96)
    cache = PagedKVCache(backend, len(lengths), 2, num_pages=num_pages, page_size=16, page_summaries=True, track_weights=True)
    k, v = _kv(len(lengths), 2, max(lengths), 96, seed)
    q = _q(len(lengths), 4, 96)
    cache.append(0, k, v, lengths=lengths)
    cache.attention(0, q)
    return cache, q


@pytest.mark.parametrize("lengths,keep", [([100, 90, 20], 40), ([64, 64, 64], 48), ([33, 64, 17], 32), ([40, 40, 1], 1)])
def test_eviction_needs_no_free_pages(cuda_ready, lengths, keep):
    """The same tokens stay whether the pool has room for every move, for some or for none."""
    used = sum(-(-n // 16) for n in lengths)
    per = -(-keep // 16)
    roomy, q = _filled(used + 100, lengths)
    want_n = roomy.evict(0, keep, sinks=0, recent=1)
    want = roomy.attention(0, q)
    for spare in (0, 1, per, 2 * per):
        cache, _ = _filled(used + spare, lengths)
        assert cache.free_pages(0) == spare
        assert cache.evict(0, keep, sinks=0, recent=1) == want_n == [min(n, keep) for n in lengths]
        left = used + spare - sum(-(-n // 16) for n in want_n)
        assert cache.free_pages(0) == left
        owned = [p for row in cache._layers[0].rows for p in row]
        assert sorted(owned + cache._layers[0].free) == list(range(used + spare))
        assert torch.equal(cache.attention(0, q), want)
        n = max(want_n)
        assert torch.equal(cache.get_weights(0)[..., :n], roomy.get_weights(0)[..., :n])
        assert (cache.attention(0, q, top_pages=max(2, per)) - cache.attention(0, q)).abs().max() <= 1e-4
        if left:                                        # the freed pages serve again
            more = [1 if n % 16 else 0 for n in want_n]
            cache.append(0, *_kv(3, 2, 1, 96, 5), lengths=more)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("track", [False, True])
def test_captured_attention_follows_the_cache(cuda_ready, track):
    """Attention captured while the sequences are short, replayed as they grow and after an eviction."""
    backend = PrismKVBackend(PrismKVConfig(), head_dim=96)
    make = lambda: PagedKVCache(backend, 2, 2, num_pages=40, page_size=16, max_tokens=320, page_summaries=True,  # noqa: E731
                                track_weights=track)
    caches, q = [make(), make()], _q(2, 4, 96)
    for c in caches:
        c.append(0, *_kv(2, 2, 20, 96, 0))
        c.attention(0, q), c.attention(0, q, top_pages=3)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = caches[0].attention(0, q), caches[0].attention(0, q, top_pages=3)
    for step in range(3):
        g.replay()
        want = caches[1].attention(0, q), caches[1].attention(0, q, top_pages=3)
        torch.cuda.synchronize()
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1]), step
        if track:
            w = [c.get_weights(0) for c in caches]
            assert torch.equal(*w)
        for c in caches:
            if step == 0:
                c.append(0, *_kv(2, 2, 150, 96, 1), lengths=[150, 60])
            elif track:
                c.evict(0, 50)
    assert _lib.device_error() == 0



def test_buffers_follow_the_tokens_not_the_pool(cuda_ready):
    """Running weights and an attention call's scratch grow with the longest sequence, not with the pool."""
    B, H, Hq, d = 16, 2, 8, 96
    backend = PrismKVBackend(PrismKVConfig(), head_dim=d)
    cache = PagedKVCache(backend, B, H, num_pages=B * 256, page_size=16, page_summaries=True, track_weights=True)
    q = _q(B, Hq, d)
    k, v = _kv(B, H, 40, d, 0)
    cache.append(0, k, v)
    slots = 48
    cache.attention(0, q)
    assert cache.get_weights(0).shape[:2] == (B, H) and slots <= cache.get_weights(0).shape[2] <= 4 * slots
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = cache.attention(0, q)
    used = torch.cuda.max_memory_allocated() - before
    # scores of 48 slots (16 x 8 rows), and what does not depend on lengths: partial states and query fragments
    fixed = 4 * (160 + B * H) * 2 * 4 * (d + 2) + 4 * B * H * 2 * (48 * 32 + 8) + out.numel() * 4
    assert used <= 4 * B * Hq * slots + fixed + (1 << 16)
    # growth keeps what was there
    before = cache.get_weights(0)[..., :slots].clone()
    cache.append(0, *_kv(B, H, 300, d, 1))
    assert torch.equal(cache.get_weights(0)[..., :slots], before) and not cache.get_weights(0)[..., slots:].any()
    wide = PagedKVCache(backend, B, H, num_pages=B * 256, page_size=16, max_tokens=4096, track_weights=True)
    for s, seed in ((40, 0), (300, 1)):
        wide.append(0, *_kv(B, H, s, d, seed))
        if s == 40:
            wide.attention(0, q), wide.attention(0, q)
    assert wide.get_weights(0).shape == (B, H, 4096)
    assert torch.equal(wide.attention(0, q), cache.attention(0, q))
    n = cache.get_weights(0).shape[2]
    assert torch.equal(wide.get_weights(0)[..., :n], cache.get_weights(0)) and not wide.get_weights(0)[..., n:].any()
    assert cache.evict(0, 64) == wide.evict(0, 64) == [64] * B
    assert torch.equal(wide.attention(0, q), cache.attention(0, q))
    assert _lib.device_error() == 0


def test_capture_with_buffers_that_may_grow_is_refused(cuda_ready):
    """Without max_tokens the weights' buffer is replaced when a sequence outgrows it; a graph would hold the old one."""
    backend = PrismKVBackend(PrismKVConfig(), head_dim=96)
    cache = PagedKVCache(backend, 12, 2, num_pages=240, page_size=16, track_weights=True)
    cache.append(0, *_kv(12, 2, 20, 96, 0))
    q = _q(12, 4, 96)
    want = cache.attention(0, q)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="max_tokens"):
        with torch.cuda.graph(g):
            cache.attention(0, q)
    assert torch.equal(cache.attention(0, q), want)


def test_a_growing_cache_without_tokens(cuda_ready):
    backend = PrismKVBackend(PrismKVConfig(), head_dim=96)
    cache = PagedKVCache(backend, 12, 2, num_pages=240, page_size=16, page_summaries=True, track_weights=True)
    none = torch.empty(12, 2, 0, 96, device=DEV)
    assert cache.append(0, none, none) == [0] * 12
    q = _q(12, 4, 96)
    assert not cache.attention(0, q).any() and not cache.attention(0, q, top_pages=2).any()
    assert cache.evict(0, 1, sinks=0, recent=0) == [0] * 12
    k, v = _kv(12, 2, 3, 96, 0)
    assert cache.append(0, k, v, lengths=[3] + [0] * 11) == [3] + [0] * 11
    raw = RawKVCache(backend)
    raw.append(0, k[:1], v[:1])
    out = cache.attention(0, q)
    assert (out[0] - raw.attention(0, q[:1])[0]).abs().max() <= 1e-4 and not out[1:].any()
    assert (cache.get_weights(0)[0, :, :3].sum(-1) - 2).abs().max() <= 1e-5 and not cache.get_weights(0)[1:].any()
    assert _lib.device_error() == 0
