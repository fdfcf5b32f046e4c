"""GPU parity of the paged-cache calls against plain implementations in 64 bits.

Tolerances (u = 2^-24).  Decoded values and rotated queries are held to a relative 2^-22 or better, so a
score, a sum of dim products of magnitude A = scale * sum |q' k| in all, is off by at most
ds = A (2^-21 + 6 sqrt(dim) u) (rounding errors of a sum grow as the root of its length; 6 standard
deviations).  A weight is off by 2 ds relative, and the weighted sum of n tokens by a further
2^-20 + n/16 u (tiles of 16 tokens are summed one after the other, each truncated).  So a channel o_k in
the rotated space is off by c P_k, P_k = sum_t p |V_k|, c = 2 ds + 2^-20 + n/16 u, and an output
component, a product with a unit column of R, by c |P| (Euclidean).  16-bit outputs add half a step.
"""

import numpy as np
import pytest
import torch

from prismkv_b200 import BiasTable, LearnedSliceCodebook, StackedPlaneQuantizer, _lib
from prismkv_b200.synthetic import synthetic_bias, synthetic_codebook

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _quantizer(variant="v1", bits=(4, 4, 4), dim=96):
    q = StackedPlaneQuantizer(dim, *bits, seed=42)
    Cz, K = 1 << bits[0], 1 << (bits[1] + bits[2])
    if "learned" in variant:
        q._codebooks = LearnedSliceCodebook(synthetic_codebook(Cz, K, q.r_max, 11), Cz, K, q.z_min, q.z_max, q.r_max)
    if "bias" in variant:
        q._bias = BiasTable(synthetic_bias(Cz, 12), delta_z=(q.z_max - q.z_min) / Cz)
    if "lloyd" in variant:
        q.calibrate_lloyd_max_z(torch.randn(2048, dim, generator=torch.Generator().manual_seed(5)).to(DEV))
    return q


class Cache:
    """A paged cache with scattered pages, table entries behind the end that must not be followed, and the
    same tokens in 64 bits."""

    def __init__(self, q, lens, Hkv, ps, seed=0, layout="hnd", spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.q, self.codec, self.ps, self.lens_host, self.Hkv = q, q.codec(torch.device(DEV)), ps, lens, Hkv
        m, B = q.m, len(lens)
        need = [-(-n // ps) for n in lens]
        P = sum(need) + 2
        per = 16 // (1 if q.code_dtype == torch.uint8 else 2)
        pitch = -(-m // per) * per
        shape = (P, Hkv, ps, pitch) if layout == "hnd" else (P, ps, Hkv, pitch)
        self.pools = []
        for _ in range(2):
            vec = torch.randn(P * Hkv * ps, q.dim, generator=g) * spread
            codes = torch.zeros(shape, dtype=q.code_dtype, device=DEV)
            view = codes[..., :m] if layout == "hnd" else codes.transpose(1, 2)[..., :m]
            view.copy_(q.encode_compact(vec.to(DEV)).view(P, Hkv, ps, m))
            self.pools.append(view)
        self.k, self.v = self.pools
        perm = torch.randperm(P, generator=g).tolist()
        width = max(need + [1]) + 2
        table = torch.full((B, width), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor(perm[at:at + n], dtype=torch.int32)
            table[b, n:] = 1 << 30 if b % 2 else -1
            at += n
        self.table = table.to(DEV)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        h = self.codec.host
        self.fb = q.bits_r + q.bits_theta
        self.R = torch.from_numpy(h.R).to(DEV).double()
        self.dz = torch.from_numpy(np.asarray(h.dec_z)).to(DEV).double()
        xy = np.asarray(h.dec_xy).reshape(-1, 2)
        self.dxy = torch.from_numpy(np.tile(xy, ((1 << sum(h.bits)) // xy.shape[0], 1))).to(DEV).double()

    def slots(self, b, hk, pages=None):
        """Token indexes and (K, V) of one sequence and KV head in 64 bits."""
        n = self.lens_host[b]
        if pages is None:
            t = torch.arange(n, device=DEV)
        else:
            pg = pages[pages >= 0].long()
            t = (pg[:, None] * self.ps + torch.arange(self.ps, device=DEV)).reshape(-1)
            t = t[t < n]
        page = self.table[b].long()[t // self.ps]
        kv = []
        for pool in (self.k, self.v):
            c = pool[page, hk, t % self.ps].long() & ((1 << sum(self.codec.host.bits)) - 1)
            kv.append(torch.cat([self.dz[c >> self.fb].unsqueeze(-1), self.dxy[c]], -1).flatten(-2))
        return t, kv[0], kv[1]

    def reference(self, query, scale=None, pages=None):
        """(out, per-component bound, weights, bound) in 64 bits; weights (B, Hkv, slots)."""
        B, Hq, dim = query.shape
        G = Hq // self.Hkv
        scale = dim ** -0.5 if scale is None else scale
        T = self.table.shape[1] * self.ps
        out = torch.zeros(B, Hq, dim, dtype=torch.float64, device=DEV)
        tol = torch.zeros(B, Hq, 1, dtype=torch.float64, device=DEV)
        w = torch.zeros(B, self.Hkv, T, dtype=torch.float64, device=DEV)
        wt = torch.zeros_like(w)
        for b in range(B):
            for h in range(self.Hkv):
                t, k, v = self.slots(b, h, None if pages is None else pages[b, h])
                if t.numel() == 0:
                    continue
                qr = query[b, h * G:(h + 1) * G].double() @ self.R.T
                p = torch.softmax(qr @ k.T * scale, -1)
                out[b, h * G:(h + 1) * G] = p @ v @ self.R
                A = (qr.abs() @ k.abs().T).amax(-1) * abs(scale)
                ds = A * (2.0 ** -21 + 6 * dim ** 0.5 * U)
                c = 2 * ds + 2.0 ** -20 + t.numel() / 16 * U
                tol[b, h * G:(h + 1) * G, 0] = c * (p @ v.abs()).norm(dim=-1)
                w[b, h, t] = p.sum(0)
                wt[b, h, t] = ((2 * ds + 2.0 ** -20)[:, None] * p).sum(0)
        return out, tol, w, wt


def _query(B, Hq, dim, dt=torch.float32, seed=7):
    return torch.randn(B, Hq, dim, generator=torch.Generator().manual_seed(seed)).to(DEV).to(dt)


def _close(got, ref, tol, what=""):
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - ref).abs()
    bound = tol + half * ref.abs() + 1e-30
    assert torch.isfinite(got).all(), what
    assert (err <= bound).all(), f"{what}: worst {(err / bound).max().item():.3f} of the bound, error {err.max().item():.3e}"


def _no_error():
    torch.cuda.synchronize()
    assert _lib.device_error(clear=True) == 0


F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16
CASES = [
    # lens, Hq, Hkv, dim, variant, bits, q dtype, page size, layout
    ([1], 1, 1, 96, "v1", (4, 4, 4), F32, 16, "hnd"),
    ([15, 16, 17, 31, 33], 4, 2, 96, "v1", (4, 4, 4), BF, 16, "hnd"),
    ([0, 5, 0, 200], 8, 8, 96, "v1", (4, 4, 4), F32, 32, "hnd"),          # sequences without tokens
    ([0, 0], 4, 1, 96, "v1", (4, 4, 4), F32, 16, "hnd"),
    ([700, 64, 129], 12, 4, 96, "v1", (4, 4, 4), F16, 64, "hnd"),         # group 3
    ([1000, 3], 10, 2, 96, "v1", (4, 4, 4), BF, 128, "hnd"),              # group 5
    ([513, 1, 77], 16, 2, 96, "v1", (4, 4, 4), F32, 16, "nhd"),           # group 8, heads inside tokens
    ([300], 32, 2, 96, "v1", (4, 4, 4), BF, 1024, "hnd"),                 # group 16, one page
    ([2100, 900], 8, 2, 96, "learned_bias", (4, 4, 4), BF, 32, "hnd"),
    ([333, 44], 4, 4, 96, "learned", (4, 4, 4), F32, 16, "hnd"),
    ([450], 4, 2, 96, "bias", (4, 4, 4), F32, 16, "hnd"),
    ([450, 20], 4, 2, 96, "lloyd", (4, 4, 4), F32, 16, "hnd"),
    ([257, 100], 4, 4, 96, "v1", (3, 3, 2), F32, 16, "hnd"),              # one-byte codes
    ([600], 8, 2, 96, "learned", (3, 3, 2), BF, 64, "hnd"),
    ([600, 31], 4, 1, 96, "lloyd_bias", (3, 3, 2), F16, 16, "nhd"),
    ([300], 4, 2, 96, "v1", (2, 5, 5), F32, 16, "hnd"),                   # 1024 (r, theta) cells
    ([300, 2], 4, 2, 96, "v1", (1, 1, 1), F32, 16, "hnd"),
    ([300, 2], 4, 2, 96, "v1", (8, 2, 2), BF, 16, "hnd"),
    ([300], 2, 1, 96, "v1", (2, 4, 4), F32, 16, "hnd"),
    ([260, 40], 8, 2, 66, "v1", (4, 4, 4), BF, 16, "hnd"),
    ([260, 40], 4, 2, 66, "v1", (3, 3, 2), F32, 16, "hnd"),
    ([260, 40], 8, 2, 129, "v1", (4, 4, 4), F16, 16, "hnd"),
    ([260], 4, 4, 129, "learned", (3, 3, 2), F32, 32, "nhd"),
    ([260, 70], 8, 2, 192, "v1", (4, 4, 4), F32, 16, "hnd"),
    ([130], 16, 2, 192, "learned_bias", (4, 4, 4), BF, 16, "hnd"),
    ([130], 4, 4, 192, "v1", (3, 3, 2), BF, 16, "hnd"),
    ([100, 17], 4, 2, 3, "v1", (4, 4, 4), F32, 16, "hnd"),                # one triplet
    ([100], 4, 2, 51, "v1", (4, 4, 4), F32, 16, "hnd"),
    ([9000, 4000, 100, 1], 4, 1, 96, "v1", (4, 4, 4), BF, 16, "hnd"),     # ragged
    ([40] * 70, 4, 1, 96, "v1", (4, 4, 4), F32, 16, "hnd"),               # more sequences than a warp's lanes
    ([20000], 4, 1, 96, "v1", (4, 4, 4), F32, 16, "hnd"),
    # more than four query heads per KV head: two blocks of heads to a unit (up to head size 144)
    ([700, 33, 0], 64, 8, 129, "v1", (4, 4, 4), BF, 16, "hnd"),
    ([300], 12, 2, 129, "learned_bias", (4, 4, 4), F32, 32, "nhd"),
    ([300, 65], 16, 2, 96, "learned", (3, 3, 2), BF, 16, "hnd"),
    ([300, 1], 10, 1, 66, "v1", (3, 3, 2), F16, 16, "hnd"),
    ([513], 18, 2, 96, "lloyd_bias", (4, 4, 4), BF, 64, "hnd"),           # group 9: three blocks, the last one alone
    ([200], 14, 2, 192, "v1", (4, 4, 4), F32, 16, "hnd"),                 # one block to a unit
    ([200, 90], 16, 1, 144, "learned", (3, 3, 2), F32, 16, "nhd"),
]


@pytest.mark.parametrize("lens,Hq,Hkv,dim,variant,bits,qdt,ps,layout", CASES)
def test_attention_and_weights(cuda_ready, lens, Hq, Hkv, dim, variant, bits, qdt, ps, layout):
    c = Cache(_quantizer(variant, bits, dim), lens, Hkv, ps, seed=len(lens) + dim, layout=layout)
    q = _query(len(lens), Hq, dim, qdt)
    ref, tol, w, wt = c.reference(q)
    out = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens)
    assert out.dtype == F32
    _close(out, ref, tol, "out")
    out16 = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, out_dtype=BF)
    _close(out16, ref, tol, "bf16 out")
    w_in = torch.rand(w.shape, generator=torch.Generator().manual_seed(3)).to(DEV)
    w_out = torch.full_like(w_in, -5.0)
    again = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, weights=w_in, weights_out=w_out)
    assert torch.equal(again, out)
    for b, n in enumerate(lens):
        assert (w_out[b, :, n:] == -5.0).all()                       # behind the last token: untouched
        err = (w_out[b, :, :n].double() - w_in[b, :, :n].double() - w[b, :, :n]).abs()
        # the sum is rounded once per head and once into the running weight
        bound = wt[b, :, :n] + (w_in[b, :, :n].double() + Hq // Hkv * w[b, :, :n]) * 2 * U + 1e-30
        assert (err <= bound).all(), (err / bound).max().item()
    c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, weights=w_in)
    for b, n in enumerate(lens):
        assert torch.equal(w_in[b, :, :n], w_out[b, :, :n])          # in place
    _no_error()


@pytest.mark.parametrize("lens,Hq,Hkv,dim", [([3100, 0, 1, 40], 8, 8, 96), ([1700, 20], 18, 2, 96), ([900, 33], 8, 2, 192)])
def test_weights_under_a_wide_table(cuda_ready, lens, Hq, Hkv, dim):
    """Room for many more tokens than there are: the same results, whichever form of the weight pass that takes."""
    c = Cache(_quantizer("v1", (4, 4, 4), dim), lens, Hkv, 16, seed=dim)
    q = _query(len(lens), Hq, dim)
    T = c.table.shape[1] * 16
    w = torch.rand((len(lens), Hkv, T), generator=torch.Generator().manual_seed(3)).to(DEV)
    want_w = w.clone()
    want = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, weights=want_w)
    ref, tol, _, _ = c.reference(q)
    _close(want, ref, tol, "out")
    rows = len(lens) * Hkv
    for tokens in (T + 1536, 1536 * (1200 // rows + 1)):             # one beside it, and past a thousand tiles of 1536
        n = -(-tokens // 16)
        table = torch.full((len(lens), n), -1, dtype=torch.int32, device=DEV)
        table[:, :c.table.shape[1]] = c.table
        wide = torch.full((len(lens), Hkv, n * 16), -5.0, device=DEV)
        wide[..., :T] = w
        got = c.codec.paged_attention(q, c.k, c.v, table, c.lens, weights=wide)
        assert torch.equal(got, want) and torch.equal(wide[..., :T], want_w) and (wide[..., T:] == -5.0).all()
    _no_error()


@pytest.mark.parametrize("spread,scale", [(6.0, None), (1.0, 0.0), (1.0, -0.3), (20.0, 1.0)])
def test_attention_scales(cuda_ready, spread, scale):
    """Peaked, flat, negated and one-token softmaxes; values at the ends of the grid."""
    c = Cache(_quantizer(), [700, 90], 2, 16, seed=3, spread=spread)
    q = _query(2, 8, 96)
    ref, tol, _, _ = c.reference(q, scale)
    _close(c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, scale=scale), ref, tol)


def test_attention_strided_query_and_output(cuda_ready):
    c = Cache(_quantizer(), [100, 50], 2, 16)
    wide = _query(2, 12, 96, BF)
    q = wide[:, 2:10]
    ref, tol, _, _ = c.reference(q)
    buf = torch.full((2, 20, 96), 9.0, dtype=BF, device=DEV)
    out = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, out=buf[:, 5:13])
    _close(out, ref, tol)
    assert (buf[:, :5] == 9).all() and (buf[:, 13:] == 9).all()
    odd = torch.empty(2, 8, 97, device=DEV)[..., 1:].copy_(q)           # rows off 16-byte boundaries
    _close(c.codec.paged_attention(odd, c.k, c.v, c.table, c.lens), ref, tol)
    q4 = q.float().unsqueeze(2)
    _close(c.codec.paged_attention(q4, c.k, c.v, c.table, c.lens), ref, tol)
    _close(c.codec.paged_attention(q.double(), c.k, c.v, c.table, c.lens), ref, tol)


def test_attention_listed_pages(cuda_ready):
    c = Cache(_quantizer(), [500, 40, 0, 16], 2, 16, seed=9)
    q = _query(4, 8, 96)
    lists = torch.full((4, 2, 5), -1, dtype=torch.int32)
    lists[0, 0] = torch.tensor([0, 3, 4, 9, 31])
    lists[0, 1, :2] = torch.tensor([7, 30])
    lists[1, 0, :3] = torch.tensor([0, 1, 2])
    lists[1, 1, :1] = torch.tensor([2])
    lists[3, :, 0] = 0
    lists = lists.to(DEV)
    ref, tol, w, wt = c.reference(q, pages=lists)
    w_in = torch.zeros(w.shape, device=DEV)
    out = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, pages=lists, weights=w_in)
    _close(out, ref, tol)
    assert (out[2] == 0).all()
    assert ((w_in.double() - w).abs() <= wt + 8 * U * w).all()
    assert (w_in[w == 0] == 0).all()
    _no_error()
    every = torch.arange(32, device=DEV, dtype=torch.int32).expand(4, 2, 32).contiguous()
    every[1, :, 3:], every[2], every[3, :, 1:] = -1, -1, -1
    ref, tol, _, _ = c.reference(q)
    _close(c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, pages=every), ref, tol)
    _no_error()


def test_pages_outside_the_pool_are_masked_and_reported(cuda_ready):
    c = Cache(_quantizer(), [100, 100], 2, 16, seed=2)
    q = _query(2, 4, 96)
    ref, tol, _, _ = c.reference(q)
    bad = c.table.clone()
    bad[1, 2] = c.k.shape[0]                                            # one past the pool
    out = c.codec.paged_attention(q, c.k, c.v, bad, c.lens)
    torch.cuda.synchronize()
    assert _lib.device_error(clear=True) == 6
    _close(out[:1], ref[:1], tol[:1])
    lists = torch.tensor([0, 1, 3, 4, 5, 6], dtype=torch.int32, device=DEV).expand(2, 2, 6).contiguous()
    ref2, tol2, _, _ = c.reference(q, pages=lists)
    _close(out[1:], ref2[1:], tol2[1:])                                 # the others' softmax
    # lengths past the table: clamped
    long = torch.tensor([1 << 30, -3], dtype=torch.int32, device=DEV)
    full = torch.arange(9, dtype=torch.int32, device=DEV).view(1, 9).expand(2, 9) % c.k.shape[0]
    out = c.codec.paged_attention(q, c.k, c.v, full.contiguous(), long)
    c.table, c.lens_host = full, [9 * 16, 0]
    ref, tol, _, _ = c.reference(q)
    _close(out, ref, tol)
    # lists that repeat, fall or leave the sequence
    for bad_list in ([3, 3], [5, 2], [-1, 2], [100, 101]):
        pg = torch.tensor(bad_list, dtype=torch.int32, device=DEV).expand(2, 2, 2).contiguous()
        c.codec.paged_attention(q, c.k, c.v, c.table, torch.tensor([100, 100], dtype=torch.int32, device=DEV), pages=pg)
        torch.cuda.synchronize()
        assert _lib.device_error(clear=True) == 6, bad_list


def test_non_finite_queries_stay_in_their_rows(cuda_ready):
    c = Cache(_quantizer(), [70, 70], 2, 16)
    q = _query(2, 8, 96)
    ref, tol, _, _ = c.reference(q)
    q[0, 1, 5] = float("nan")
    q[1, 6, 0] = float("inf")
    for dt in (F32, BF):
        out = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, out_dtype=dt)
        assert torch.isnan(out[0, 1]).all() and torch.isnan(out[1, 6]).all()
        for b, h in ((0, 1), (1, 6)):
            out[b, h], ref[b, h] = 0, 0
        _close(out, ref, tol)


def test_shared_prefix_pages(cuda_ready):
    c = Cache(_quantizer(), [64, 80], 2, 16, seed=4)
    c.table[1, :4] = c.table[0, :4]
    q = _query(2, 4, 96)
    ref, tol, _, _ = c.reference(q)
    _close(c.codec.paged_attention(q, c.k, c.v, c.table, c.lens), ref, tol)


def test_attention_long_pool_offsets(cuda_ready):
    """A pool whose byte offsets pass 32 bits: the last pages are the ones attended to."""
    q = _quantizer("v1", (3, 3, 2))
    codec = q.codec(torch.device(DEV))
    P = (1 << 32) // (4 * 1024 * 32) + 8
    k = codec.empty_pages(P, 4, 1024)
    assert k.numel() > 1 << 32
    small = Cache(q, [1500], 4, 1024, seed=1)
    last = torch.arange(P - small.k.shape[0], P, device=DEV)
    k[last] = small.k
    v = codec.empty_pages(P, 4, 1024)
    v[last] = small.v
    query = _query(1, 8, 96)
    ref, tol, _, _ = small.reference(query)
    n = -(-1500 // 1024)
    table = small.table.clone()
    table[:, :n] += P - small.k.shape[0]
    out = codec.paged_attention(query, k, v, table, small.lens)
    del k, v
    _close(out, ref, tol)
    _no_error()


@pytest.mark.parametrize("qdt,odt,ps", [(BF, BF, 16), (F32, F32, 64)])
def test_attention_long_ranges(cuda_ready, qdt, odt, ps):
    """Ranges of more pages than a CTA's list holds at a time, cut evenly: most CTAs serve parts of two units."""
    c = Cache(_quantizer("v1", (3, 3, 2)), [43210], 32, ps, seed=11)
    q = _query(1, 32, 96, qdt)
    ref, tol, w, wt = c.reference(q)
    w_in = torch.zeros(w.shape, device=DEV)
    _close(c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, weights=w_in, out_dtype=odt), ref, tol)
    assert ((w_in.double() - w).abs() <= wt + 4 * U * w).all()
    lists = torch.arange(0, -(-43210 // ps), 1, dtype=torch.int32, device=DEV)
    lists = lists[lists % 7 != 3].expand(1, 32, -1).contiguous()
    ref, tol, _, _ = c.reference(q, pages=lists)
    _close(c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, pages=lists, out_dtype=odt), ref, tol)
    _no_error()


@pytest.mark.parametrize("size", [2.0 ** -20, 3e-3, 1e3, 2.0 ** 20])
@pytest.mark.parametrize("bits", [(4, 4, 4), (3, 3, 2), (2, 5, 5)])
def test_attention_other_ranges(cuda_ready, size, bits):
    """Codecs calibrated to small and large values, queries the other way round: the operands are rescaled."""
    quant = StackedPlaneQuantizer(96, *bits, seed=42, z_min=-7.0 * size, z_max=9.0 * size, r_max=8.0 * size)
    c = Cache(quant, [300, 21], 2, 16, seed=2, spread=size)
    q = _query(2, 8, 96) / size
    ref, tol, _, _ = c.reference(q)
    _close(c.codec.paged_attention(q, c.k, c.v, c.table, c.lens), ref, tol)
    small = q * 2.0 ** -30                                               # scores of almost nothing
    ref, tol, _, _ = c.reference(small)
    _close(c.codec.paged_attention(small, c.k, c.v, c.table, c.lens), ref, tol)
    sums = c.codec.summarize_pages(c.k, c.table, c.lens, c.codec.empty_summaries(c.k.shape[0], 2))
    got = c.codec.select_pages(q, sums, c.table, c.lens, 16, 5)
    assert torch.equal(got, _ref_select(c, q, sums, 5, 1, 1))


def test_inputs_written_just_before_the_call(cuda_ready):
    """Every input of every call is rewritten by the kernel right before it (launches may come up while it runs)."""
    c = Cache(_quantizer(), [900, 700, 64], 2, 16, seed=5)
    sums = c.codec.summarize_pages(c.k, c.table, c.lens, c.codec.empty_summaries(c.k.shape[0], 2))
    g = torch.Generator(device=DEV).manual_seed(3)
    rounds = []
    for _ in range(20):
        lens = torch.stack([torch.randint(1, n + 1, (), generator=g, device=DEV) for n in c.lens_host]).to(torch.int32)
        rounds.append((torch.randn(3, 8, 96, generator=g, device=DEV), lens, torch.rand(3, 2, 960, generator=g, device=DEV)))

    def calls(q, lens, w, settle):
        wait = torch.cuda.synchronize if settle else (lambda: None)
        wait()
        pages = c.codec.select_pages(q, sums, c.table, lens, 16, 9)
        wait()
        a = c.codec.paged_attention(q, c.k, c.v, c.table, lens, pages=pages)
        wait()
        b = c.codec.paged_attention(q, c.k, c.v, c.table, lens, weights=w)
        wait()
        kept, kw = c.codec.select_tokens(w, lens, 50, recent=3)
        return pages, a, b, w.clone(), kept, kw

    want = [calls(q, lens.clone(), w.clone(), True) for q, lens, w in rounds]
    bufs = [torch.empty_like(t) for t in rounds[0]]
    got = []
    for q, lens, w in rounds:
        bufs[0].copy_(q * 1.0), torch.add(lens, 0, out=bufs[1]), torch.mul(w, 1.0, out=bufs[2])
        bufs[0].mul_(1.0)
        got.append(calls(*bufs, False))
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(x, y))
    # the same, captured once and replayed on new contents
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        bufs[0].mul_(1.0)
        held = calls(*bufs, False)
    for (q, lens, w), y in zip(rounds, want):
        for b, t in zip(bufs, (q, lens, w)):
            b.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, y))
    _no_error()


# ---- summaries, page selection ---------------------------------------------------------------------
def _ref_summaries(c, out, start=None):
    top = max(c.dz.abs().max().item(), c.dxy.abs().max().item())
    for b, n in enumerate(c.lens_host):
        for j in range(-(-n // c.ps)):
            if start is not None and min(n, (j + 1) * c.ps) <= start[b]:
                continue
            for h in range(c.Hkv):
                pg = torch.tensor([j], device=DEV)
                _, k, _ = c.slots(b, h, pg)
                s = torch.round(k * (127 * 128 / top)).long()
                page = int(c.table[b, j])
                out[page, h, 0, :c.q.dim] = (s.amin(0) >> 7).to(torch.int8)
                out[page, h, 1, :c.q.dim] = ((s.amax(0) + 127) >> 7).to(torch.int8)
                out[page, h, :, c.q.dim:] = 0
    return out


@pytest.mark.parametrize("lens,Hkv,dim,variant,bits,ps,layout", [
    ([1, 16, 40, 0], 2, 96, "v1", (4, 4, 4), 16, "hnd"), ([200, 65], 3, 96, "learned_bias", (4, 4, 4), 64, "nhd"),
    ([90], 2, 66, "v1", (3, 3, 2), 32, "hnd"), ([130, 7], 1, 129, "lloyd", (4, 4, 4), 16, "hnd"),
    ([1030], 2, 192, "v1", (2, 5, 5), 1024, "hnd"), ([40], 2, 3, "v1", (1, 1, 1), 16, "hnd")])
def test_summaries(cuda_ready, lens, Hkv, dim, variant, bits, ps, layout):
    c = Cache(_quantizer(variant, bits, dim), lens, Hkv, ps, seed=5, layout=layout)
    got = c.codec.empty_summaries(c.k.shape[0], Hkv).fill_(55)
    want = _ref_summaries(c, got.clone())
    assert c.codec.summarize_pages(c.k, c.table, c.lens, got) is got
    assert torch.equal(got, want)
    start = [max(0, n - 3) for n in lens]
    got.fill_(44)
    want = _ref_summaries(c, got.clone(), start)
    c.codec.summarize_pages(c.k, c.table, c.lens, got, start=torch.tensor(start, dtype=torch.int32, device=DEV))
    assert torch.equal(got, want)
    _no_error()


def _ref_select(c, q, sums, top, sinks, recent):
    B, Hq, dim = q.shape
    qr = (q.double() @ c.R.T).view(B, c.Hkv, -1, dim)
    a = qr.abs().amax((2, 3), keepdim=True)
    qi = torch.where(a > 0, torch.round(qr * 127 / a), 0.0).nan_to_num(0, 0, 0).cpu()
    out = torch.full((B, c.Hkv, top), -1, dtype=torch.int32)
    for b, n in enumerate(c.lens_host):
        npg = -(-n // c.ps)
        s = sums[c.table[b, :npg].long()][..., :dim].double().cpu()
        for h in range(c.Hkv):
            score = (qi[b, h].clamp(min=0) @ s[:, h, 1].T + qi[b, h].clamp(max=0) @ s[:, h, 0].T).amax(0).tolist()
            order = sorted(range(npg), key=lambda j: (not (j < sinks or j >= npg - recent), -score[j], j))
            pick = sorted(order[:top])
            out[b, h, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
    return out.to(DEV)


@pytest.mark.parametrize("lens,Hq,Hkv,dim,ps,top,sinks,recent,qdt", [
    ([1000, 33, 0, 16], 8, 2, 96, 16, 8, 1, 1, BF), ([1000, 500], 4, 4, 96, 16, 1, 0, 0, F32),
    ([900], 16, 1, 66, 16, 20, 2, 3, F16), ([700, 650, 1], 6, 2, 129, 32, 5, 0, 5, BF), ([640], 4, 2, 192, 16, 40, 1, 1, F32),
    ([640], 4, 2, 192, 16, 64, 40, 24, F32), ([33000], 4, 1, 96, 16, 100, 1, 1, BF)])
def test_select_pages(cuda_ready, lens, Hq, Hkv, dim, ps, top, sinks, recent, qdt):
    c = Cache(_quantizer(dim=dim), lens, Hkv, ps, seed=6)
    sums = c.codec.summarize_pages(c.k, c.table, c.lens, c.codec.empty_summaries(c.k.shape[0], Hkv))
    q = _query(len(lens), Hq, dim, qdt)
    got = c.codec.select_pages(q, sums, c.table, c.lens, ps, top, sinks=sinks, recent=recent)
    assert torch.equal(got, _ref_select(c, q, sums, top, sinks, recent))
    ref, tol, _, _ = c.reference(q, pages=got)
    _close(c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, pages=got), ref, tol)
    _no_error()


def test_select_pages_ties_and_dead_queries(cuda_ready):
    c = Cache(_quantizer(), [800, 800], 2, 16, seed=6)
    sums = torch.zeros_like(c.codec.empty_summaries(c.k.shape[0], 2))
    q = _query(2, 8, 96)
    got = c.codec.select_pages(q, sums, c.table, c.lens, 16, 7, sinks=1, recent=1)      # every page alike
    assert got[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 49]
    sums = c.codec.summarize_pages(c.k, c.table, c.lens, sums)
    q[0] = 0
    q[1, 0, 0] = float("nan")
    got = c.codec.select_pages(q, sums, c.table, c.lens, 16, 7, sinks=0, recent=1)
    assert got[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 49] and got[1, 0].tolist() == [0, 1, 2, 3, 4, 5, 49]
    assert torch.equal(got[1, 1:], _ref_select(c, q, sums, 7, 0, 1)[1, 1:])


def test_summary_bounds_every_score(cuda_ready):
    """The score of a page is an upper bound of its tokens' (with the rounded query, in grid steps)."""
    c = Cache(_quantizer(), [600], 2, 16, seed=8)
    sums = c.codec.summarize_pages(c.k, c.table, c.lens, c.codec.empty_summaries(c.k.shape[0], 2))
    top = max(c.dz.abs().max().item(), c.dxy.abs().max().item())
    for h in range(2):
        t, k, _ = c.slots(0, h)
        s = sums[c.table[0].long()[t // 16], h].double()[..., :96]
        k = k * (127 / top)
        assert (s[:, 0] <= k + 1 / 256).all() and (s[:, 1] >= k - 1 / 256).all()


# ---- token selection and gather --------------------------------------------------------------------
def _ref_keep(w, n, keep, sinks, recent):
    def rank(i):
        x = w[i]
        return (not (i < sinks or i >= n - recent), x != x, -x if x == x else 0, i)
    return sorted(sorted(range(n), key=rank)[:keep])


@pytest.mark.parametrize("lens,H,T,keep,sinks,recent,kind", [
    ([1], 1, 1, 1, 0, 0, "exp"), ([100, 0, 7, 64], 3, 100, 20, 2, 5, "exp"), ([300, 299], 2, 321, 300, 0, 0, "exp"),
    ([1000, 513], 2, 1000, 1, 0, 0, "ties"), ([1000, 513], 2, 1024, 130, 4, 64, "ties"), ([700], 2, 700, 300, 0, 10, "odd"),
    ([5000, 4097], 1, 5000, 2500, 4, 100, "exp"), ([40000, 20000], 2, 40000, 1000, 0, 0, "exp"),
    ([40000], 1, 40000, 39999, 0, 0, "ties"), ([400000], 1, 400000, 777, 3, 33, "exp")])
def test_select_tokens(cuda_ready, lens, H, T, keep, sinks, recent, kind):
    g = torch.Generator().manual_seed(T + keep)
    w = torch.empty(len(lens), H, T).exponential_(generator=g)
    if kind == "ties":
        w = torch.floor(w)
    if kind == "odd":
        special = torch.tensor([float("nan"), float("inf"), -float("inf"), -0.0, 0.0, -1.0, 1e-42])
        pick = torch.randint(0, 14, w.shape, generator=g)
        w = torch.where(pick < 7, special[pick.clamp(max=6)], w)
    codec = _quantizer().codec(torch.device(DEV))
    kept, kw = codec.select_tokens(w.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), keep, sinks=sinks, recent=recent)
    kept, kw = kept.cpu(), kw.cpu()
    for b, n in enumerate(lens):
        for h in range(H):
            want = _ref_keep(w[b, h].tolist(), n, keep, sinks, recent)
            assert kept[b, h, :len(want)].tolist() == want
            assert (kept[b, h, len(want):] == -1).all() and (kw[b, h, len(want):] == 0).all()
            assert torch.equal(kw[b, h, :len(want)].view(torch.int32), w[b, h][want].view(torch.int32))
    _no_error()


@pytest.mark.parametrize("dim,bits,ps,ps2,layout", [(96, (4, 4, 4), 16, 16, "hnd"), (129, (4, 4, 4), 32, 16, "nhd"),
                                                   (66, (3, 3, 2), 16, 64, "hnd"), (3, (3, 3, 2), 16, 16, "hnd")])
def test_gather_tokens(cuda_ready, dim, bits, ps, ps2, layout):
    c = Cache(_quantizer(bits=bits, dim=dim), [150, 20, 0], 2, ps, seed=3, layout=layout)
    keep = 37
    w = torch.rand(3, 2, c.table.shape[1] * ps, generator=torch.Generator().manual_seed(1)).to(DEV)
    kept, _ = c.codec.select_tokens(w, c.lens, keep, sinks=1, recent=4)
    n = -(-keep // ps2)
    table = torch.randperm(3 * n + 1, generator=torch.Generator().manual_seed(2))[:3 * n].view(3, n).to(torch.int32).to(DEV)
    ko, vo = (c.codec.empty_pages(3 * n + 1, 2, ps2).fill_(9) for _ in range(2))
    c.codec.gather_tokens(c.k, c.v, c.table, kept, ko, vo, table)
    for b in range(3):
        for h in range(2):
            ids = kept[b, h][kept[b, h] >= 0].long()
            src = c.table[b].long()[ids // ps]
            i = torch.arange(n * ps2, device=DEV)
            for a, o in ((c.k, ko), (c.v, vo)):
                row = o[table[b].long()[i // ps2], h, i % ps2]
                assert torch.equal(row[:ids.numel()], a[src, h, ids % ps])
                assert (row[ids.numel():] == 9).all()
    _no_error()


def test_store_pages(cuda_ready):
    for bits, dim in (((4, 4, 4), 96), ((3, 3, 2), 129)):
        c = Cache(_quantizer(bits=bits, dim=dim), [100, 40, 16], 2, 16, seed=3)
        before = c.k.clone()
        new = torch.randint(0, 200, (3, 2, 9, c.q.m), generator=torch.Generator().manual_seed(4)).to(c.k.dtype).to(DEV)
        start = torch.tensor([91, 3, 7], dtype=torch.int32, device=DEV)
        c.codec.store_pages(new, c.k, c.table, start, counts=torch.tensor([9, 0, 5], dtype=torch.int32, device=DEV))
        for b, n in enumerate((9, 0, 5)):
            for i in range(n):
                t = int(start[b]) + i
                before[int(c.table[b, t // 16]), :, t % 16] = new[b, :, i]
        assert torch.equal(c.k, before)
        _no_error()
        c.codec.store_pages(new, c.k, c.table, torch.full((3,), 16 * c.table.shape[1] - 2, dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
        assert _lib.device_error(clear=True) == 6


# ---- how they are called ---------------------------------------------------------------------------
def test_a_run_of_them_in_a_graph_and_on_two_streams(cuda_ready):
    """Summaries, selection, attention with weights, eviction and attention over what is left, captured; the
    same eagerly on two streams at once, each with its own cache."""
    def step(c, q, w, bufs):
        sums, ko, vo, table2, lens2 = bufs
        c.codec.summarize_pages(c.k, c.table, c.lens, sums)
        pages = c.codec.select_pages(q, sums, c.table, c.lens, c.ps, 12)
        a = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, pages=pages)
        w2 = torch.empty_like(w).copy_(w)
        d = c.codec.paged_attention(q, c.k, c.v, c.table, c.lens, weights=w2)
        kept, kw = c.codec.select_tokens(w2, c.lens, 100, sinks=1, recent=16)
        c.codec.gather_tokens(c.k, c.v, c.table, kept, ko, vo, table2)
        e = c.codec.paged_attention(q, ko, vo, table2, lens2)
        return pages, a, d, w2, kept, kw, e

    def make(seed):
        c = Cache(_quantizer(), [900, 400], 2, 16, seed=seed)
        w = torch.zeros(2, 2, c.table.shape[1] * 16, device=DEV)
        table2 = torch.arange(14, dtype=torch.int32, device=DEV).view(2, 7)
        bufs = (c.codec.empty_summaries(c.k.shape[0], 2).zero_(), c.codec.empty_pages(14, 2, 16), c.codec.empty_pages(14, 2, 16),
                table2, torch.full((2,), 100, dtype=torch.int32, device=DEV))
        return c, _query(2, 8, 96, BF, seed), w, bufs

    sets = [make(1), make(2)]
    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    c, q, w, bufs = sets[0]
    kept = want[0][4]
    lens = c.lens_host
    for b in range(2):
        assert (kept[b, :, 0] == 0).all() and (kept[b, :, -1] == lens[b] - 1).all()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for st, s in zip(streams, sets):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(step(*s))
        torch.cuda.synchronize()
        for g, x in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, x))
    graphs, outs = [], []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(*s))
        graphs.append(gr)
    for _ in range(3):
        for st, gr in zip(streams, graphs):                             # replayed side by side
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for g, x in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(g, x))
    _no_error()


def test_refusals(cuda_ready):
    c = Cache(_quantizer(), [100, 50], 2, 16)
    q = _query(2, 8, 96)
    call = lambda **k: c.codec.paged_attention(  # noqa: E731
        k.get("q", q), k.get("k", c.k), k.get("v", c.v), k.get("table", c.table), k.get("lens", c.lens), **k.get("kw", {}))
    for bad in (dict(q=q[:, :7]), dict(q=q[:1]), dict(q=q[..., :93]), dict(q=q.unsqueeze(2).expand(2, 8, 2, 96)),
                dict(k=c.k.long()), dict(k=c.k[:, :1]), dict(v=c.v[:, :, :8]), dict(table=c.table.long()),
                dict(table=c.table[0]), dict(lens=c.lens.long()), dict(lens=c.lens[:1]),
                dict(k=c.k[:, :, :8], v=c.v[:, :, :8]), dict(kw=dict(out_dtype=torch.float64)),
                dict(kw=dict(out=torch.empty(2, 8, 95, device=DEV))),
                dict(kw=dict(pages=torch.zeros(2, 2, 0, dtype=torch.int32, device=DEV))),
                dict(kw=dict(pages=torch.zeros(2, 2, dtype=torch.int32, device=DEV))),
                dict(kw=dict(pages=torch.zeros(2, 1, 3, dtype=torch.int32, device=DEV))),
                dict(kw=dict(weights=torch.zeros(2, 2, 128, dtype=BF, device=DEV))),
                dict(kw=dict(weights_out=torch.zeros(2, 2, 128, device=DEV))),
                dict(kw=dict(weights=torch.zeros(2, 2, 128, device=DEV), weights_out=torch.zeros(2, 2, 127, device=DEV)))):
        with pytest.raises((ValueError, RuntimeError)):
            call(**bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        call(lens=c.lens.cpu())
    with pytest.raises(RuntimeError, match="misaligned"):
        m = torch.zeros(4, 2, 16, 35, dtype=torch.int16, device=DEV)[..., :32]
        call(k=m, v=m)
    with pytest.raises(RuntimeError, match="misaligned"):
        m = torch.zeros(4 * 2 * 16 * 32 + 1, dtype=torch.int16, device=DEV)[1:].view(4, 2, 16, 32)
        call(k=m, v=m)
    sums = c.codec.empty_summaries(c.k.shape[0], 2)
    for bad in (dict(top=0), dict(top=2, sinks=2, recent=1), dict(top=3, sinks=-1), dict(top=2, page_size=20)):
        with pytest.raises(ValueError):
            c.codec.select_pages(q, sums, c.table, c.lens, bad.pop("page_size", 16), **bad)
    with pytest.raises(ValueError):
        c.codec.summarize_pages(c.k, c.table, c.lens, sums[1:])
    w = torch.zeros(2, 2, 128, device=DEV)
    for bad in (dict(keep=0), dict(keep=3, sinks=2, recent=2), dict(keep=3, recent=-1)):
        with pytest.raises(ValueError):
            c.codec.select_tokens(w, c.lens, **bad)
    kept, _ = c.codec.select_tokens(w, c.lens, 40)
    with pytest.raises(ValueError):
        c.codec.gather_tokens(c.k, c.v, c.table, kept, c.k, c.v, c.table[:, :2])
    _no_error()
