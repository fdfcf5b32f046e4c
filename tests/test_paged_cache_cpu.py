"""PagedKVCache's bookkeeping against plain lists, on a codec of torch operations (no GPU needed)."""

import random
import threading

import pytest
import torch

from prismkv_b200.cache import PagedKVCache
from prismkv_b200.cache.dim_aligner import DimAligner


class PlainCodec:
    """The paged calls in torch on the CPU: a token's code is its first channel."""

    m = 1

    def encode(self, x):
        return x[:, :1].to(torch.int16)

    def empty_pages(self, num_pages, kv_heads, page_size, code_dtype=None):
        return torch.full((num_pages, kv_heads, page_size, 8), -9, dtype=torch.int16)[..., :1]

    def empty_summaries(self, num_pages, kv_heads):
        return torch.zeros(num_pages, kv_heads, 2, 16, dtype=torch.int8)

    def store_pages(self, codes, pages, table, start, counts=None):
        ps = pages.shape[2]
        for b in range(codes.shape[0]):
            for i in range(codes.shape[2] if counts is None else int(counts[b])):
                t = int(start[b]) + i
                pages[int(table[b, t // ps]), :, t % ps] = codes[b, :, i]

    def summarize_pages(self, k, table, lens, out, start=None):
        ps = k.shape[2]
        for b, n in enumerate(lens.tolist()):
            for j in range((0 if start is None else int(start[b])) // ps, -(-n // ps)):
                if start is None or int(start[b]) < n:
                    x = k[int(table[b, j]), :, :min(ps, n - j * ps), 0]
                    out[int(table[b, j]), :, 0, 0], out[int(table[b, j]), :, 1, 0] = x.amin(1) // 256, x.amax(1) // 256
        return out

    def select_pages(self, q, sums, table, lens, ps, top, sinks=1, recent=1):
        return torch.zeros(len(lens), sums.shape[1], top, dtype=torch.int32)

    def paged_attention(self, q, k, v, table, lens, scale=None, pages=None, weights=None, out_dtype=torch.float32):
        """Adds (token's code + 1) to its weight; the output is the sum of the V codes."""
        self.seen = (tuple(table.shape), None if weights is None else tuple(weights.shape), pages is not None)
        ps, out = k.shape[2], torch.zeros(q.shape)
        for b, n in enumerate(lens.tolist()):
            for t in range(n):
                page = int(table[b, t // ps])
                if weights is not None:
                    weights[b, :, t] += k[page, :, t % ps, 0] + 1
                out[b] += v[page, :, t % ps].float().repeat_interleave(q.shape[1] // k.shape[1], 0)
        return out

    def select_tokens(self, w, lens, keep, sinks=0, recent=0):
        kept = torch.full((*w.shape[:2], keep), -1, dtype=torch.int32)
        kw = torch.zeros(kept.shape)
        for b, n in enumerate(lens.tolist()):
            for h in range(w.shape[1]):
                ids = sorted(sorted(range(n), key=lambda i: (not (i < sinks or i >= n - recent), -float(w[b, h, i]), i))[:keep])
                kept[b, h, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
                kw[b, h, :len(ids)] = w[b, h, ids]
        return kept, kw

    def gather_tokens(self, k, v, table, kept, ko, vo, table_out):
        ps, moved = k.shape[2], []
        for b in range(kept.shape[0]):
            for h in range(kept.shape[1]):
                for i, t in enumerate(kept[b, h].tolist()):
                    if t >= 0:
                        src, dst = int(table[b, t // ps]), int(table_out[b, i // ps])
                        assert src >= 0 and dst >= 0
                        moved.append((dst, h, i % ps, k[src, h, t % ps].clone(), v[src, h, t % ps].clone()))
                        assert ko is not k or dst not in table[b, :].tolist()[:-(-max(kept[b, h].tolist()) // ps) or 1], "source page"
        for dst, h, r, a, c in moved:
            ko[dst, h, r], vo[dst, h, r] = a, c


class PlainBackend:
    head_dim = 3
    aligner = DimAligner(3)

    class quantizer:
        code_dtype = torch.int16

    def __init__(self):
        self._codec = PlainCodec()

    def codec(self, device=None):
        return self._codec


def _cache(batch=3, num_pages=12, **kw):
    kw = dict(dict(page_summaries=True, track_weights=True), **kw)
    return PagedKVCache(PlainBackend(), batch, 2, num_pages=num_pages, page_size=16, device=torch.device("cpu"), **kw)


def _tokens(batch, s, first):
    """K codes count up from `first` (KV head 1: 100 more), V codes are 7 more than K's."""
    k = torch.zeros(batch, 2, s, 3)
    k[..., 0] = first + torch.arange(s) + 1000 * torch.arange(batch)[:, None, None] + 100 * torch.arange(2)[None, :, None]
    return k, k + 7


def _content(cache, b):
    """(K codes, V codes, weights) of a sequence, per KV head, read through the table and lengths that the calls get."""
    k, v, table, lens = cache.get_pages(0)
    t = range(int(lens[b]))
    at = [(int(table[b, i // 16]), i % 16) for i in t]
    w = cache.get_weights(0)
    return [([int(k[p, h, r, 0]) for p, r in at], [int(v[p, h, r, 0]) for p, r in at],
             None if w is None else [float(w[b, h, i]) for i in t]) for h in range(2)]


def _whole(cache):
    """Every page is free or belongs to one sequence, and host and device agree."""
    st = cache._layers[0]
    assert sorted(st.free + [p for r in st.rows for p in r]) == list(range(cache.num_pages))
    assert st.lens.tolist() == st.lengths == cache.get_seq_lengths(0)
    for b, (r, n) in enumerate(zip(st.rows, st.lengths)):
        assert len(r) == -(-n // 16) and st.table[b, :len(r)].tolist() == r
        if st.weights is not None:
            assert not st.weights[b, :, n:].any()


class _Broken(RuntimeError):
    pass


@pytest.mark.parametrize("call", ["store_pages", "summarize_pages", "encode", "empty_summaries"])
@pytest.mark.parametrize("nth", [1, 2])
def test_a_failed_append_changes_nothing(monkeypatch, call, nth):
    for before in (0, 20):
        cache = _cache()
        codec = cache._backend(0)._codec
        if before:
            cache.append(0, *_tokens(3, before, 0))
            cache.attention(0, torch.zeros(3, 2, 3))
        state = (cache.free_pages(0), cache.get_seq_lengths(0), [_content(cache, b) for b in range(3)] if before else None)
        real, count = getattr(codec, call), [0]

        def fail(*a, **k):
            count[0] += 1
            if count[0] == nth:
                raise _Broken
            return real(*a, **k)

        with monkeypatch.context() as mp:
            mp.setattr(codec, call, fail)
            try:
                cache.append(0, *_tokens(3, 30, 500), lengths=[30, 0, 13])
                failed = False
            except _Broken:
                failed = True
        if not failed:                                                   # the call is not made that often
            continue
        assert (cache.free_pages(0), cache.get_seq_lengths(0)) == state[:2]
        if before:
            _whole(cache)
            assert [_content(cache, b) for b in range(3)] == state[2]
        else:
            assert cache.cached_layers == []
        cache.append(0, *_tokens(3, 30, 500), lengths=[30, 0, 13])
        _whole(cache)
        assert [len(c[0][0]) for c in (_content(cache, b) for b in range(3))] == [before + 30, before, before + 13]


@pytest.mark.parametrize("call", ["select_tokens", "gather_tokens", "summarize_pages"])
def test_a_failed_eviction_changes_nothing(monkeypatch, call):
    cache = _cache(num_pages=20)
    codec = cache._backend(0)._codec
    cache.append(0, *_tokens(3, 60, 0), lengths=[60, 10, 45])
    cache.attention(0, torch.zeros(3, 2, 3))
    state = cache.free_pages(0), cache.get_seq_lengths(0), [_content(cache, b) for b in range(3)]

    def fail(*a, **k):
        raise _Broken

    with monkeypatch.context() as mp:
        mp.setattr(codec, call, fail)
        with pytest.raises(_Broken):
            cache.evict(0, 20, sinks=1, recent=2)
    _whole(cache)
    assert (cache.free_pages(0), cache.get_seq_lengths(0), [_content(cache, b) for b in range(3)]) == state
    assert cache.evict(0, 20, sinks=1, recent=2) == [20, 10, 20]
    _whole(cache)


@pytest.mark.parametrize("seed", range(12))
def test_appends_evictions_and_releases_against_lists(seed):
    """A run of calls on a pool that is nearly always full: tokens, weights and pages as plain lists have them."""
    rng = random.Random(seed)
    batch, num_pages = rng.choice([1, 2, 3, 5]), rng.randint(4, 14)
    cache = _cache(batch, num_pages, max_tokens=rng.choice([None, num_pages * 16]))
    model = [[([], [], []) for _ in range(2)] for _ in range(batch)]     # per sequence and head: K, V, weights
    at = 0
    for _ in range(25):
        act = rng.choice(["append", "append", "append", "evict", "attend", "release"])
        used = lambda: sum(-(-len(m[0][0]) // 16) for m in model)  # noqa: E731
        if act == "append":
            s = rng.choice([1, 5, 16, 33])
            n = [rng.randint(0, s) for _ in range(batch)]
            k, v = _tokens(batch, s, at % 800)
            at += s
            fits = sum(-(-(len(m[0][0]) + x) // 16) for m, x in zip(model, n)) <= num_pages
            if not fits:
                with pytest.raises((RuntimeError, ValueError)):
                    cache.append(0, k, v, lengths=n)
                continue
            cache.append(0, k, v, lengths=n)
            for b in range(batch):
                for h in range(2):
                    for x, src in ((0, k), (1, v)):
                        model[b][h][x].extend(src[b, h, :n[b], 0].int().tolist())
                    model[b][h][2].extend([0.0] * n[b])
        elif 0 not in cache.cached_layers:
            continue
        elif act == "attend":
            cache.attention(0, torch.zeros(batch, 2, 3))
            for m in model:
                for kk, _, ww in m:
                    ww[:] = [w + x + 1 for w, x in zip(ww, kk)]
        elif act == "release":
            b = rng.randrange(batch)
            cache.release(0, b)
            model[b] = [([], [], []) for _ in range(2)]
        else:
            keep = rng.choice([1, 7, 16, 30])
            sinks, recent = rng.choice([(0, 0), (0, 1), (min(2, keep - 1), 1), (0, keep)])
            cache.evict(0, keep, sinks=sinks, recent=recent)             # never refused, however full the pool
            for m in model:
                n = len(m[0][0])
                if n > keep:
                    for h in range(2):
                        w = m[h][2]
                        order = sorted(range(n), key=lambda i: (not (i < sinks or i >= n - recent), -w[i], i))
                        ids = sorted(order[:keep])
                        m[h] = tuple([x[i] for i in ids] for x in m[h])
        if 0 in cache.cached_layers:
            _whole(cache)
            assert cache.free_pages(0) == num_pages - used()
            for b in range(batch):
                assert _content(cache, b) == [tuple(x) for x in model[b]], (act, b)


@pytest.mark.parametrize("call,nth", [("select_tokens", 1), ("gather_tokens", 1), ("gather_tokens", 2), ("summarize_pages", 1),
                                      ("empty_pages", 1), ("empty_pages", 2), ("empty_summaries", 1)])
def test_a_failed_eviction_of_a_full_pool_changes_nothing(monkeypatch, call, nth):
    cache = _cache(num_pages=8)
    codec = cache._backend(0)._codec
    cache.append(0, *_tokens(3, 60, 0), lengths=[60, 10, 45])
    assert cache.free_pages(0) == 0
    cache.attention(0, torch.zeros(3, 2, 3))
    state = cache.get_seq_lengths(0), [_content(cache, b) for b in range(3)], cache._layers[0].summaries.clone()
    real, count = getattr(codec, call), [0]

    def fail(*a, **k):
        count[0] += 1
        if count[0] == nth:
            raise RuntimeError("broken")
        return real(*a, **k)

    with monkeypatch.context() as mp:
        mp.setattr(codec, call, fail)
        with pytest.raises(RuntimeError, match="broken"):
            cache.evict(0, 20, sinks=1, recent=2)
    _whole(cache)
    assert (cache.get_seq_lengths(0), [_content(cache, b) for b in range(3)]) == state[:2]
    assert torch.equal(cache._layers[0].summaries, state[2])
    assert cache.evict(0, 20, sinks=1, recent=2) == [20, 10, 20]
    _whole(cache)
    # the summaries are those of the pages as they are
    k, _, table, lens = cache.get_pages(0)
    want = codec.summarize_pages(k, table, lens, codec.empty_summaries(8, 2))
    for r in cache._layers[0].rows:
        assert torch.equal(cache._layers[0].summaries[r], want[r])


def test_buffers_and_tables_follow_the_tokens():
    cache = _cache(batch=8, num_pages=8 * 64)
    codec = cache._backend(0)._codec
    cache.append(0, *_tokens(8, 20, 0))
    assert cache.get_weights(0).shape == (8, 2, 32)
    cache.attention(0, torch.zeros(8, 2, 3))
    assert codec.seen == ((8, 2), (8, 2, 32), False)
    cache.attention(0, torch.zeros(8, 2, 3), top_pages=2)
    assert codec.seen == ((8, 2), (8, 2, 32), False)                     # no sequence has more than two pages
    seen = [_content(cache, b) for b in range(8)]
    cache.append(0, *_tokens(8, 30, 100), lengths=[30] + [0] * 7)
    assert 64 <= cache.get_weights(0).shape[2] <= 96
    assert [_content(cache, b) for b in range(1, 8)] == seen[1:]
    cache.attention(0, torch.zeros(8, 2, 3), top_pages=2)
    assert codec.seen[0] == (8, 4) and codec.seen[2]
    _whole(cache)
    # given a longest sequence, or where whole rows cost little beside the codes, there is one buffer for good
    fixed = _cache(batch=8, num_pages=8 * 64, max_tokens=200)
    fixed.append(0, *_tokens(8, 20, 0))
    assert fixed.get_weights(0).shape == (8, 2, 13 * 16)
    few = _cache(batch=2, num_pages=30)
    few.append(0, *_tokens(2, 20, 0))
    assert few.get_weights(0).shape == (2, 2, 480)


@pytest.mark.parametrize("read", [lambda c: c.get_weights(0), lambda c: c.get_pages(0), lambda c: c.memory_footprint(),
                                  lambda c: c.get_seq_lengths(0), lambda c: c.free_pages(0), lambda c: c.cached_layers])
def test_readers_wait_for_a_change_in_another_thread(read):
    """What a reader gets belongs together: not a table from before an eviction beside lengths from after it."""
    cache = _cache()
    cache.append(0, *_tokens(3, 5, 0))
    got = []
    t = threading.Thread(target=lambda: got.append(read(cache)))
    with cache._lock:
        t.start()
        t.join(0.2)
        assert t.is_alive()
    t.join(60)
    assert not t.is_alive() and len(got) == 1
