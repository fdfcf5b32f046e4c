"""Paged calls beside the tables of test_gpu_paged.py: what one output's type, an earlier call or a value's size must
not change.  Tolerances are that file's; weights below 2^-15 of the largest are off by 2^-37 of it instead of 2^-22 of
themselves, n 2^-37 for n tokens, which its n/16 u covers."""

import pytest
import torch

from prismkv_b200 import StackedPlaneQuantizer, _lib
from test_gpu_paged import BF, DEV, F16, F32, U, Cache, _close, _no_error, _quantizer, _query

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("odt", [BF, F16])
@pytest.mark.parametrize("bits,dim,Hq,Hkv,variant", [
    ((4, 4, 4), 96, 8, 2, "v1"), ((3, 3, 2), 96, 4, 4, "v1"), ((4, 4, 4), 129, 8, 2, "v1"), ((4, 4, 4), 96, 16, 2, "v1"),
    ((4, 4, 4), 96, 4, 1, "learned_bias"), ((3, 3, 2), 192, 4, 2, "lloyd")])
def test_weights_do_not_depend_on_the_output_type(cuda_ready, bits, dim, Hq, Hkv, variant, odt):
    """The running weights are float32 whatever the outputs are; a 16-bit output is the float32 one, rounded."""
    c = Cache(_quantizer(variant, bits, dim), [900, 77], Hkv, 16, seed=dim)
    q = _query(2, Hq, dim)
    _, _, w, wt = c.reference(q)
    w32, w16 = (torch.zeros(w.shape, device=DEV) for _ in range(2))
    out32 = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, weights=w32)
    out16 = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, weights=w16, out_dtype=odt)
    assert torch.equal(w16, w32) and torch.equal(out16, out32.to(odt))
    assert ((w16.double() - w).abs() <= wt + Hq // Hkv * w * 2 * U).all()
    _no_error()


def test_a_refused_call_does_not_spoil_the_next_one(cuda_ready):
    """The workspace's size is kept by the shapes; a call that is refused has none to keep."""
    c = Cache(_quantizer(), [100, 50], 2, 16)
    q = _query(2, 8, 96)
    with pytest.raises(RuntimeError, match="invalid"):
        c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, scale=float("nan"))
    ref, tol, _, _ = c.reference(q)
    _close(c.codec.paged_attention(q, c.k, c.v, c.table, c.lens), ref, tol)
    _no_error()


def _expired_wait(q):
    """A split-sequence exchange whose second rank does not exist: the wait runs out after 20 ms and sets error 4."""
    from prismkv_b200.dist import SequenceExchange

    g = torch.Generator(device=DEV).manual_seed(7)
    kc, vc = (q.encode_compact(torch.randn(2 * 4 * 3000, 96, generator=g, device=DEV)).view(2, 4, 3000, 32) for _ in range(2))
    ex = SequenceExchange.single_process(q, _query(2, 16, 96, BF), kc, world=2, wait_ms=20)
    ex.run(_query(2, 16, 96, BF), kc, vc)
    torch.cuda.synchronize()
    return ex


def _bad_page():
    c = Cache(_quantizer(), [100], 2, 16)
    c.table[0, 1] = c.k.shape[0]
    c.codec.paged_attention(_query(1, 4, 96), c.k, c.v, c.table, c.lens)
    torch.cuda.synchronize()


def test_no_device_error_hides_another(cuda_ready):
    """An expired wait and a page outside the pool are both reported, one reading after the other."""
    _no_error()
    ex = _expired_wait(_quantizer())
    try:
        _bad_page()
        assert _lib.device_error(clear=False) == 4
        assert _lib.device_error(clear=True) == 4
        assert _lib.device_error(clear=False) == 6
        assert _lib.device_error(clear=True) == 6
        assert _lib.device_error(clear=True) == 0
    finally:
        ex.close()


def test_exchange_check_leaves_page_errors_to_their_reader(cuda_ready):
    """A page error is not an expired wait: the exchange's check neither raises for it nor clears it."""
    _no_error()
    _bad_page()
    ex = _expired_wait(_quantizer())
    try:
        with pytest.raises(RuntimeError, match="device error 4"):
            ex.check()
        ex.check()
        assert _lib.device_error(clear=True) == 6
        ex.check()
    finally:
        ex.close()


def test_codec_tables_written_just_before_the_call(cuda_ready):
    """The codec's tables are inputs like any other: a kernel right before the call, of the same library or not, may
    write them."""
    c = Cache(_quantizer(), [900, 700, 64], 2, 16, seed=5)
    q, w = _query(3, 8, 96), torch.rand(3, 2, 960, generator=torch.Generator().manual_seed(3)).to(DEV)
    names = ("_R", "_dz", "_dxy", "_grid_z", "_grid_xy")
    sums = c.codec.empty_summaries(c.k.shape[0], 2).zero_()
    first = [getattr(c.codec, n).clone() for n in names]
    turned = [first[0].view(96, 96).flip(0).reshape(first[0].shape).contiguous(), first[1] * 0.5, first[2] * 0.25, first[3] // 2,
              first[4] // 4]

    def use(tables, settle):
        wait = torch.cuda.synchronize if settle else (lambda: None)

        def put():
            for n, t in zip(names, tables):
                getattr(c.codec, n).copy_(t)
            wait()

        put()
        s = c.codec.summarize_pages(c.k, c.table, c.lens, sums).clone()
        put()
        pages = c.codec.select_pages(q, s, c.table, c.lens, 16, 9)
        put()
        a = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens)
        put()
        w2 = w.clone()
        b = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, pages=pages, weights=w2, out_dtype=BF)
        return s, pages, a, b, w2

    want = [use(t, True) for t in (first, turned)]
    assert not torch.equal(want[0][2], want[1][2]) and not torch.equal(want[0][0], want[1][0])
    for i in (1, 0) * 5:
        got = use((first, turned)[i], False)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want[i]))
    _no_error()


@pytest.mark.parametrize("size", [2.0 ** -40, 2.0 ** -30, 2.0 ** 40])
@pytest.mark.parametrize("bits", [(4, 4, 4), (3, 3, 2), (2, 5, 5)])
def test_codecs_of_any_size(cuda_ready, size, bits):
    """Codecs calibrated to values far from one, queries the other way round: the same softmax, outputs in proportion."""
    quant = StackedPlaneQuantizer(96, *bits, seed=42, z_min=-7.0 * size, z_max=9.0 * size, r_max=8.0 * size)
    c = Cache(quant, [300, 21], 2, 16, seed=2, spread=size)
    q = _query(2, 8, 96) / size
    ref, tol, w, wt = c.reference(q)
    for odt in (F32, BF):
        _close(c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, out_dtype=odt), ref, tol)
    got = torch.zeros(w.shape, device=DEV)
    c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, weights=got)
    assert ((got.double() - w).abs() <= wt + 8 * U * w).all()


@pytest.mark.parametrize("size", [2.0 ** 100, 2.0 ** 112])
@pytest.mark.parametrize("bits", [(4, 4, 4), (3, 3, 2), (2, 5, 5)])
def test_queries_as_large_as_float32_holds(cuda_ready, size, bits):
    """Scores of 2^100 and more are finite: the largest takes all the weight."""
    c = Cache(_quantizer(bits=bits), [300, 21], 2, 16, seed=2)
    q = _query(2, 8, 96) * size
    out = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens)
    for b in range(2):
        for h in range(8):
            _, k, v = c.slots(b, h // 4)
            s = (q[b, h].double() @ c.R.T) @ k.T
            best = s.topk(2)
            # only where the two best are further apart than the operands' 2^-22 can bring them together
            if best.values[0] - best.values[1] > 2.0 ** -16 * ((q[b, h].double() @ c.R.T).abs() @ k.abs().T).max():
                want = v[best.indices[0]] @ c.R
                assert (out[b, h].double() - want).abs().max() <= 2.0 ** -18 * v[best.indices[0]].norm()
            else:
                assert torch.isfinite(out[b, h]).all()
    _no_error()


def test_strides_of_single_pages_and_heads_do_not_count(cuda_ready):
    """A dimension of one element has no stride of its own: pools that differ there alone are the same."""
    c = Cache(_quantizer(), [14], 1, 16, seed=4)
    page = int(c.table[0, 0])
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    k = c.k[page:page + 1].clone(memory_format=torch.contiguous_format)
    wide = torch.zeros(3, 5, 16, 32, dtype=c.v.dtype, device=DEV)
    wide[1, 2] = c.v[page, 0]
    v = wide[1:2, 2:3]
    assert v.stride() != k.stride()
    q = _query(1, 4, 96)
    ref, tol, _, _ = c.reference(q)
    _close(c.codec.paged_attention(q, k, v, table, c.lens), ref, tol)
    _no_error()


def test_page_selection_at_the_widest_table(cuda_ready):
    """The limit itself is served: the keys of a row's slices fill the shared memory that the cluster has."""
    c = Cache(_quantizer(dim=192), [900, 30], 1, 16, seed=6)
    sums = c.codec.summarize_pages(c.k, c.table, c.lens, c.codec.empty_summaries(c.k.shape[0], 1))
    q = _query(2, 16, 192)
    want = c.codec.select_pages(q, sums, c.table, c.lens, 16, 9)
    table = torch.full((2, 303104), -1, dtype=torch.int32, device=DEV)
    table[:, :c.table.shape[1]] = c.table
    assert torch.equal(c.codec.select_pages(q, sums, table, c.lens, 16, 9), want)
    # every page of the row in use: the first sequence's pages over and over
    long = c.table[:1, :56].repeat(1, 303104 // 56 + 1)[:, :303104].contiguous()
    lens = torch.full((1,), 303104 * 16, dtype=torch.int32, device=DEV)
    got = c.codec.select_pages(q[:1], sums, long, lens, 16, 40, sinks=0, recent=0)
    one = c.codec.select_pages(q[:1], sums, c.table[:1, :56].contiguous(), c.lens[:1] * 0 + 56 * 16, 16, 1, sinks=0, recent=0)
    assert torch.equal(got[0, 0], one[0, 0] + 56 * torch.arange(40, dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="unsupported"):
        c.codec.select_pages(q, sums, torch.full((2, 303105), -1, dtype=torch.int32, device=DEV), c.lens, 16, 9)
    _no_error()


@pytest.mark.parametrize("lens,Hq,Hkv", [([100, 50], 8, 2), ([90], 4, 4), ([70, 33, 5], 4, 1), ([60], 2, 1)])
def test_weights_may_be_the_first_slots_of_wider_rows(cuda_ready, lens, Hq, Hkv):
    """The columns of a table and the slots of the weights as far as the tokens go: the same, and nothing behind them."""
    c = Cache(_quantizer(), lens, Hkv, 16, seed=8)
    B, n = len(lens), -(-max(lens) // 16)
    q = _query(B, Hq, 96)
    w = torch.rand(B, Hkv, c.table.shape[1] * 16, generator=torch.Generator().manual_seed(3)).to(DEV)
    want_w = w.clone()
    want = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, weights=want_w)
    kept, kw = c.codec.select_tokens(want_w, c.lens, 30, recent=2)
    wide = torch.full((B, Hkv, w.shape[2] + 7), -5.0, device=DEV)
    wide[..., :w.shape[2]] = w
    view = wide[..., :n * 16]
    assert torch.equal(c.codec.paged_attention(q, c.k, c.v, c.table[:, :n], c.lens, weights=view), want)
    assert torch.equal(wide[..., :w.shape[2]], want_w) and (wide[..., w.shape[2]:] == -5.0).all()
    got = c.codec.select_tokens(view, c.lens, 30, recent=2)
    assert torch.equal(got[0], kept) and torch.equal(got[1], kw)
    to = torch.full_like(wide, -6.0)[..., :n * 16]
    wide[..., :w.shape[2]] = w
    c.codec.paged_attention(q, c.k, c.v, c.table[:, :n], c.lens, weights=view, weights_out=to)
    for b, t in enumerate(lens):
        assert torch.equal(to[b, :, :t], want_w[b, :, :t]) and (to[b, :, t:] == -6.0).all()
    _no_error()


def test_weights_in_other_strides_are_refused(cuda_ready):
    c = Cache(_quantizer(), [100, 50], 2, 16)
    q, full = _query(2, 8, 96), torch.zeros(2, 2, 256, device=DEV)
    good = full[..., :128]
    for bad in (full[..., ::2], torch.zeros(1, 1, 128, device=DEV).expand(2, 2, 128), torch.zeros(2, 128, 2, device=DEV).transpose(1, 2),
                torch.zeros(2, 3, 128, device=DEV)[:, :2], torch.zeros(2, 2, 128, device=DEV).transpose(0, 1), good.double(), good[0],
                good[:, :1]):
        with pytest.raises(ValueError, match="weights"):
            c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, weights=bad)
        if bad.dim() == 3 and bad.shape[1] == 2 and bad.dtype == F32:
            with pytest.raises(ValueError, match="weights"):
                c.codec.select_tokens(bad, c.lens, 8)
    for bad in (torch.zeros(2, 2, 128, device=DEV), full[..., :127]):
        with pytest.raises(ValueError, match="weights"):
            c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, weights=good, weights_out=bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, weights=good.cpu())
    assert not full.any()
    _no_error()


@pytest.mark.parametrize("dim,bits,ps", [(96, (4, 4, 4), 16), (129, (3, 3, 2), 32), (66, (2, 5, 5), 64)])
def test_page_score_bounds_the_rounded_query_with_every_token(cuda_ready, dim, bits, ps):
    """A page's score is at least every token's product with the int8 query, in grid steps, but for the 1/256 of a step
    per channel that a summary may leave out -- and the pages chosen are those of the largest scores."""
    c = Cache(_quantizer(bits=bits, dim=dim), [700], 2, ps, seed=8)
    sums = c.codec.summarize_pages(c.k, c.table, c.lens, c.codec.empty_summaries(c.k.shape[0], 2))
    q = _query(1, 8, dim)
    grid = 127 / max(c.dz.abs().max().item(), c.dxy.abs().max().item())
    n = -(-700 // ps)
    got = c.codec.select_pages(q, sums, c.table, c.lens, ps, 3, sinks=0, recent=0)
    for h in range(2):
        qr = q[0, 4 * h:4 * h + 4].double() @ c.R.T
        qi = torch.round(qr * 127 / qr.abs().max())
        s = sums[c.table[0, :n].long(), h].double()[..., :dim]
        score = qi.clamp(min=0) @ s[:, 1].T + qi.clamp(max=0) @ s[:, 0].T            # (heads, pages)
        t, k, _ = c.slots(0, h)
        own = qi @ (k * grid).T                                                      # (heads, tokens)
        assert (own <= score[:, t // ps] + qi.abs().sum(1, keepdim=True) / 256 * (1 + 1e-9)).all()
        best = score.amax(0)
        assert best[got[0, h].long()].min() == best.topk(3).values.min()
    _no_error()


def test_workspace_size_is_checked(cuda_ready):
    import ctypes

    from test_paged_cpu import ALIGNMENT, WORKSPACE, _args, _codec

    lib, a, c = _lib.load(), _args(), _codec()
    need = lib.pkv_paged_attn_workspace_size(ctypes.byref(c), ctypes.byref(a))
    assert need > 0
    call = lambda ws, n: lib.pkv_paged_attn(ctypes.byref(c), ctypes.byref(a), ws, n, None)  # noqa: E731
    assert call(None, 0) == WORKSPACE and call(None, need) == WORKSPACE and call(256, need - 1) == WORKSPACE
    assert call(256 + 16, need) == ALIGNMENT


def test_weights_of_no_slots_do_not_size_the_next_workspace(cuda_ready):
    c = Cache(_quantizer(), [9, 0], 2, 16)
    q = _query(2, 8, 96)
    want = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens)
    assert torch.equal(c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, weights=torch.empty(2, 2, 0, device=DEV)), want)
    w = torch.zeros(2, 2, 48, device=DEV)
    assert torch.equal(c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, weights=w), want)
    assert (w.sum(-1) - torch.tensor([[4.0], [0.0]], device=DEV)).abs().max() <= 1e-5
    _no_error()
