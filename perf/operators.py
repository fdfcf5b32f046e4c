"""Measured cases of the paged-cache operators: attention of one new token over pages of packed codes, the
same with page selection, the same with accumulated attention weights, eviction by those weights, and the page
summaries that the selection reads.

A cache is a pool of pages, K and V apart: (pages, kv_heads, page_size, m) packed codes, m = dim / 3, each code
(z bin, flat (x, y) bin); row b of `table` lists sequence b's pages.  Everything happens in the space rotated
by R, where a code stands for one (z, x, y) triplet of its token's vector.

``run`` computes either the plain form (torch, 32 bits) or, with ``own`` set, the calls a user makes.
"""

import functools
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# code formats: bits of z, r, theta; learned: (x, y) centroids per z bin and a per-bin bias instead of the polar grid
FORMATS = {"444": ((4, 4, 4), False), "332": ((3, 3, 2), False), "learned": ((4, 4, 4), True)}


def _case(op, name=None, **kw):
    c = dict(op=op, batch=1, q_heads=8, kv_heads=8, seq=1024, ragged=0.0, dim=96, fmt="444", q="bf16",
             page=16, top=0, keep=0, recent=0, sinks=0, fresh=0)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the first steps of one chat: a handful of tokens, where the call's latency is all there is
        _case("attend", "attend-start", seq=37, q="f32"),
        # batched decode with ragged sequences, one KV head per query head, mid-sized contexts
        _case("attend", "attend-batch", batch=8, q_heads=32, kv_heads=32, seq=4096, ragged=0.5),
        # learned codebooks, grouped heads, long ragged contexts, large pages
        _case("attend", "attend-learned", batch=16, q_heads=32, kv_heads=8, seq=32768, ragged=0.75, fmt="learned", page=64),
        # the long-context decode, the largest call
        _case("attend", "attend-long", batch=4, q_heads=32, kv_heads=8, seq=131072, page=32),
        # block-sparse decode of one sequence of ordinary length
        _case("sparse", "sparse-one", q_heads=32, kv_heads=8, seq=8000, top=64, sinks=1, recent=2),
        # block-sparse decode over the long contexts: 1/32 of the pages read
        _case("sparse", "sparse-long", batch=4, q_heads=32, kv_heads=8, seq=131072, page=32, top=128, sinks=1, recent=2),
        # decode with running attention weights, head size 128 (129 with padding)
        _case("weigh", "weigh-128", batch=4, q_heads=32, kv_heads=8, seq=16384, ragged=0.3, dim=129, q="f16"),
        # the same over one-byte codes, one query head per KV head
        _case("weigh", "weigh-bytes", batch=4, q_heads=32, kv_heads=32, seq=16384, fmt="332"),
        # eviction on a small cache: one sequence down to half
        _case("evict", "evict-half", kv_heads=8, seq=1024, keep=512, recent=64, sinks=4),
        # eviction of long contexts to an eighth
        _case("evict", "evict-long", batch=4, kv_heads=8, seq=131072, keep=16384, recent=1024, sinks=4, page=32),
        # summaries after one appended token per sequence: only each last page
        _case("summarise", "summarise-step", batch=8, q_heads=32, kv_heads=32, seq=4096, ragged=0.5, fresh=1),
        # summaries of whole prompts
        _case("summarise", "summarise-prompt", batch=4, q_heads=32, kv_heads=8, seq=131072, page=32, fresh=131072),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "sparse", "weigh", "evict", "summarise"])
    fmt = rng.choice(["444", "444", "332", "learned"])
    dim = rng.choice([96, 96, 96, 66, 129, 192])
    kv = rng.choice([1, 2, 4, 8, 8, 32])
    group = rng.choice([1, 2, 3, 4, 4, 5, 8, 16]) if kv < 32 else rng.choice([1, 2])
    page = rng.choice([16, 32, 64, 128])
    batch = _log(rng, 1, 32)
    seq = _log(rng, 1, 131072)
    cap = 4 * 8 * 131072 * 96 // 2                       # half of the largest listed case's channels, at most
    seq = max(1, min(seq, cap // (batch * kv * dim)))
    c = _case(op, batch=batch, q_heads=kv * group, kv_heads=kv, seq=seq, ragged=round(rng.uniform(0, 0.95), 3),
              dim=dim, fmt=fmt, q=rng.choice(["f32", "bf16", "f16"]), page=page)
    if op == "sparse":
        c["sinks"], c["recent"] = rng.choice([0, 1, 2]), rng.choice([0, 1, 2])
        c["top"] = max(c["sinks"] + c["recent"], _log(rng, 1, max(1, -(-seq // page))), 1)
    if op == "evict":
        c["keep"] = _log(rng, 1, seq)
        c["sinks"] = rng.randint(0, min(8, c["keep"] // 2))
        c["recent"] = rng.randint(0, c["keep"] // 2)
    if op == "summarise":
        c["fresh"] = rng.choice([1, _log(rng, 1, seq), seq])
    return c


# ---- sizes that follow from a case ----------------------------------------------------------------
def _lens(c):
    """Tokens of each sequence: the longest has `seq`, the shortest (1 - ragged) of it."""
    B, S = c["batch"], c["seq"]
    return [max(1, S - int(S * c["ragged"] * b / max(1, B - 1))) for b in range(B)]


def _pages(c):
    return [-(-n // c["page"]) for n in _lens(c)]


def _code_bytes(c):
    return 1 if sum(FORMATS[c["fmt"]][0]) <= 8 else 2


def work(c):
    m, cb, dim, kv, hq = c["dim"] // 3, _code_bytes(c), c["dim"], c["kv_heads"], c["q_heads"]
    lens, pages = _lens(c), _pages(c)
    qb = 4 if c["q"] == "f32" else 2
    io = c["batch"] * hq * dim * 2 * qb
    if c["op"] in ("attend", "weigh"):
        toks = sum(lens)
        extra = 8 * kv * toks if c["op"] == "weigh" else 0
        return {"bytes": 2 * m * cb * kv * toks + io + extra, "flops": 4 * dim * hq * toks}
    if c["op"] == "sparse":
        toks = sum(min(n, c["top"] * c["page"]) for n in lens)
        return {"bytes": 2 * m * cb * kv * toks + io + sum(pages) * kv * 2 * dim + 4 * c["batch"] * kv * c["top"],
                "flops": 4 * dim * hq * toks + 2 * dim * hq * sum(pages)}
    if c["op"] == "evict":
        kept = sum(min(n, c["keep"]) for n in lens)
        return {"bytes": kv * (4 * sum(lens) + kept * (8 + 4 * m * cb)), "flops": kv * sum(lens)}
    toks = sum(min(n, n - max(0, n - c["fresh"]) // c["page"] * c["page"]) for n in lens)
    npg = sum(p - max(0, n - c["fresh"]) // c["page"] for n, p in zip(lens, pages))
    return {"bytes": kv * (m * cb * toks + 2 * dim * npg), "flops": 2 * dim * kv * toks}


# ---- the quantizer: fixed by format and size, as a model's is --------------------------------------
@functools.lru_cache(maxsize=None)
def _quantizer(fmt, dim):
    """(R, z of each z bin, (x, y) of each code, codebook, bias, ranges) as float32 arrays."""
    (bz, br, bt), learned = FORMATS[fmt]
    g = np.random.default_rng([bz, br, bt, dim])
    R = np.linalg.qr(g.standard_normal((dim, dim)))[0].astype(np.float32)
    span = math.sqrt(dim)
    nz, nr, nt = 1 << bz, 1 << br, 1 << bt
    f = np.float32                                       # the tables are built in 32 bits, step by step
    z = f(-span) + (np.arange(nz, dtype=f) + f(0.5)) * f(2 * span / nz)
    book = bias = None
    if learned:
        ang = g.uniform(-math.pi, math.pi, (nz, nr * nt))
        rad = np.sqrt(g.uniform(0, 1, (nz, nr * nt))) * span * 0.4
        book = np.stack([rad * np.cos(ang), rad * np.sin(ang)], -1).astype(np.float32)
        bias = (g.standard_normal((nz, 3)) * 0.05).astype(np.float32)
        z = z - bias[:, 0]
        xy = (book - bias[:, None, 1:]).reshape(-1, 2)
    else:
        flat = np.arange(nr * nt)
        rad = (flat // nt).astype(f) / f(nr - 1) * f(span)
        ang = torch.from_numpy((flat % nt).astype(f) / f(nt - 1) * f(2) * f(math.pi) - f(math.pi)).repeat(256)
        cos, sin = torch.cos(ang).numpy()[:flat.size], torch.sin(ang).numpy()[:flat.size]
        xy = np.tile(np.stack([rad * cos, rad * sin], -1), (nz, 1))
    return R, z.astype(np.float32), xy.astype(np.float32), book, bias, span


@functools.lru_cache(maxsize=None)
def _handle(fmt, dim):
    """The framework's codec of that quantizer on the current device."""
    from prismkv_b200 import BiasTable, LearnedSliceCodebook, StackedPlaneQuantizer
    R, _, _, book, bias, span = _quantizer(fmt, dim)
    (bz, br, bt), learned = FORMATS[fmt]
    q = StackedPlaneQuantizer.from_rotation(torch.from_numpy(R), bz, br, bt, z_min=-span, z_max=span, r_max=span)
    if learned:
        q._codebooks = LearnedSliceCodebook(torch.from_numpy(book), 1 << bz, 1 << (br + bt), -span, span, span)
        q._bias = BiasTable(torch.from_numpy(bias), delta_z=2 * span / (1 << bz))
    return q.codec(torch.device("cuda"))


# ---- inputs ----------------------------------------------------------------------------------------
def _encode(x, fmt, span, g):
    """Codes of rotated (..., m, 3) vectors: z floored into its bin, (x, y) to the nearest radius and angle.
    Learned centroids are used about evenly: their index is drawn."""
    (bz, br, bt), learned = FORMATS[fmt]
    nz, nr, nt = 1 << bz, 1 << br, 1 << bt
    iz = torch.floor((x[..., 0] + span) * (nz / (2 * span))).clamp_(0, nz - 1).to(torch.int32)
    if learned:
        flat = torch.randint(0, nr * nt, iz.shape, generator=g, device=x.device, dtype=torch.int32)
    else:
        r = torch.round(torch.hypot(x[..., 1], x[..., 2]) * ((nr - 1) / span)).clamp_(0, nr - 1).to(torch.int32)
        th = torch.round((torch.atan2(x[..., 2], x[..., 1]) + math.pi) * ((nt - 1) / (2 * math.pi))).clamp_(0, nt - 1)
        flat = r * nt + th.to(torch.int32)
    return (iz << (br + bt)) | flat


def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    fmt, dim, ps, kv, B = c["fmt"], c["dim"], c["page"], c["kv_heads"], c["batch"]
    m, cb = dim // 3, _code_bytes(c)
    R, z, xy, _, _, span = _quantizer(fmt, dim)
    lens, pages = _lens(c), _pages(c)
    s = {"case": c, "lens": torch.tensor(lens, dtype=torch.int32, device=dev), "lens_host": lens,
         "R": torch.from_numpy(R).to(dev), "z": torch.from_numpy(z).to(dev), "xy": torch.from_numpy(xy).to(dev)}
    # a pool a little larger than the sequences need, its pages handed out in no order
    total = sum(pages) + 3
    perm = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.full((B, max(pages) + 1), -1, dtype=torch.int32, device=dev)
    # rows of codes start on 16-byte boundaries
    pitch = -(-m * cb // 16) * 16 // cb
    dt = torch.uint8 if cb == 1 else torch.int16
    pools = [torch.zeros((total, kv, ps, pitch), dtype=dt, device=dev)[..., :m] for _ in range(2)]
    topics = torch.randn(B, kv, 16, dim, generator=g, device=dev) * 0.5
    at = 0
    for b in range(B):
        ids = perm[at:at + pages[b]]
        at += pages[b]
        table[b, :pages[b]] = ids
        for i, pool in enumerate(pools):
            n = pages[b] * ps
            x = torch.randn(kv, n, dim, generator=g, device=dev)
            if i == 0:                                   # keys: runs of tokens share a direction
                x += topics[b][:, (torch.arange(n, device=dev) // 97) * 7 % 16]
            codes = _encode(x.view(kv, n, m, 3), fmt, span, g).to(dt)
            pool[ids.long()] = codes.view(kv, pages[b], ps, m).transpose(0, 1)
    s.update(k=pools[0], v=pools[1], table=table)
    op = c["op"]
    if op in ("attend", "sparse", "weigh"):
        hq = c["q_heads"]
        qr = torch.randn(B, kv, hq // kv, dim, generator=g, device=dev) + 2.0 * topics[:, :, 3:4]
        s["q"] = (qr.reshape(B, hq, dim) @ s["R"]).to(DTYPES[c["q"]])
    T = max(pages) * ps
    if op == "weigh":
        s["w"] = torch.rand(B, kv, T, generator=g, device=dev)
        s["w_out"] = torch.zeros_like(s["w"])
    if op == "evict":                                    # a few tokens hold most of the weight, many hold none
        w = torch.rand(B, kv, T, generator=g, device=dev)
        s["w"] = torch.where(w < 0.2, torch.zeros_like(w), -torch.log(w) * 0.01 / (1e-3 + torch.rand(B, kv, T, generator=g, device=dev)))
        kp = -(-c["keep"] // ps)
        fresh = torch.randperm(B * kp + 2, generator=g, device=dev).to(torch.int32)[:B * kp].view(B, kp)
        s["table_out"] = fresh.contiguous()
        s["k_out"], s["v_out"] = (torch.zeros((B * kp + 2, kv, ps, pitch), dtype=dt, device=dev)[..., :m] for _ in range(2))
    if op in ("sparse", "summarise"):
        s["summaries"] = torch.zeros((total, kv, 2, -(-dim // 16) * 16), dtype=torch.int8, device=dev)
        start = 0 if op == "sparse" else None
        s["start_host"] = [0 if start == 0 else max(0, n - c["fresh"]) for n in lens]
        s["start"] = torch.tensor(s["start_host"], dtype=torch.int32, device=dev)
        if op == "sparse":
            _summarise(s, s["summaries"])
    if own:
        s["codec"] = _handle(fmt, dim)
    return s


# ---- the plain forms -------------------------------------------------------------------------------
def _flat_bits(c):
    bz, br, bt = FORMATS[c["fmt"]][0]
    return br + bt


def _decode(s, codes):
    """(..., m) codes -> (..., 3 m) rotated vectors, 32 bits."""
    i = codes.to(torch.int64)
    z, xy = s["z"][i >> _flat_bits(s["case"])], s["xy"][i]
    return torch.cat([z.unsqueeze(-1), xy], -1).flatten(-2)


def _tokens(s, pool, b, pages=None):
    """Sequence b's codes as (kv_heads, tokens, m); `pages` (kv_heads, n): those logical pages only."""
    ps = s["case"]["page"]
    if pages is None:
        n = -(-s["lens_host"][b] // ps)
        x = pool[s["table"][b, :n].long()].transpose(0, 1)
    else:
        ids = s["table"][b].long()[pages]
        x = pool[ids, torch.arange(pool.shape[1], device=ids.device)[:, None]]
    return x.flatten(1, 2)


def _attend(s, b, pages=None):
    """(out (q_heads, dim) in 32 bits, weights (q_heads, tokens)) of sequence b."""
    c = s["case"]
    kv, dim, ps, n = c["kv_heads"], c["dim"], c["page"], s["lens_host"][b]
    q = (s["q"][b].float() @ s["R"].T).view(kv, -1, dim)
    k = _decode(s, _tokens(s, s["k"], b, pages))
    if pages is None:
        live = torch.arange(k.shape[1], device=k.device).expand(kv, -1) < n
    else:
        live = (pages.unsqueeze(-1) * ps + torch.arange(ps, device=k.device)).flatten(1) < n
    x = torch.matmul(q, k.transpose(1, 2)) * (dim ** -0.5)
    del k
    x = x.masked_fill(~live.unsqueeze(1), float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p, _decode(s, _tokens(s, s["v"], b, pages)))
    return out.view(-1, dim) @ s["R"], p


def _grid(s):
    """Decoded values on the summaries' grid of 1/128 steps, the largest magnitude at 127 steps."""
    top = max(s["z"].abs().max().item(), s["xy"].abs().max().item())
    f = 127.0 * 128.0 / top
    return torch.round(s["z"].double() * f).to(torch.int32), torch.round(s["xy"].double() * f).to(torch.int32)


def _summarise(s, out):
    """Per page, KV head and channel: floor of the least and ceiling of the greatest decoded key, in steps."""
    c = s["case"]
    ps, dim = c["page"], c["dim"]
    gz, gxy = _grid(s)
    for b, n in enumerate(s["lens_host"]):
        first = s["start_host"][b] // ps
        ids = s["table"][b, first:-(-n // ps)].long()
        if ids.numel() == 0:
            continue
        i = s["k"][ids].to(torch.int64)
        v = torch.cat([gz[i >> _flat_bits(c)].unsqueeze(-1), gxy[i]], -1).flatten(-2)
        t = (first * ps + torch.arange(ids.numel() * ps, device=ids.device)).view(-1, 1, ps, 1)
        lo = v.masked_fill(t >= n, 1 << 20).amin(2) >> 7
        hi = (v.masked_fill(t >= n, -(1 << 20)).amax(2) + 127) >> 7
        out[ids, :, 0, :dim] = lo.to(torch.int8)
        out[ids, :, 1, :dim] = hi.to(torch.int8)
    return out


def _select(s):
    """Logical pages of each sequence and KV head, ascending, -1 behind the last."""
    c = s["case"]
    kv, dim, ps, B, top = c["kv_heads"], c["dim"], c["page"], c["batch"], c["top"]
    out = torch.full((B, kv, top), -1, dtype=torch.int32, device=s["q"].device)
    q = (s["q"].double() @ s["R"].double().T).view(B, kv, -1, dim)        # 64 bits: values next to a rounding border
    qi = torch.round(q * 127.0 / q.abs().amax((2, 3), keepdim=True))
    for b, n in enumerate(s["lens_host"]):
        npg = -(-n // ps)
        sm = s["summaries"][s["table"][b, :npg].long()][..., :dim].double()  # (pages, kv, 2, dim)
        lo, hi = sm[:, :, 0].permute(1, 2, 0), sm[:, :, 1].permute(1, 2, 0)
        score = (torch.matmul(qi[b].clamp(min=0), hi) + torch.matmul(qi[b].clamp(max=0), lo)).amax(1)
        j = torch.arange(npg, device=score.device)
        score[:, (j < c["sinks"]) | (j >= npg - c["recent"])] = 1e9
        k = min(top, npg)
        pick = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :k]
        out[b, :, :k] = pick.sort(-1).values.to(torch.int32)
    return out


def _evict(s):
    c = s["case"]
    kv, ps, B, keep = c["kv_heads"], c["page"], c["batch"], c["keep"]
    kept = torch.full((B, kv, keep), -1, dtype=torch.int32, device=s["w"].device)
    w_out = torch.zeros((B, kv, keep), device=s["w"].device)
    for b, n in enumerate(s["lens_host"]):
        w = s["w"][b, :, :n].clone()
        t = torch.arange(n, device=w.device)
        w[:, (t < c["sinks"]) | (t >= n - c["recent"])] = float("inf")
        k = min(keep, n)
        pick = torch.sort(w, dim=-1, descending=True, stable=True).indices[:, :k].sort(-1).values
        kept[b, :, :k] = pick.to(torch.int32)
        w_out[b, :, :k] = s["w"][b].gather(1, pick)
        src, dst = s["table"][b].long()[pick // ps], s["table_out"][b].long()[torch.arange(k, device=w.device) // ps]
        h = torch.arange(kv, device=w.device).unsqueeze(1)
        for pool, to in (("k", "k_out"), ("v", "v_out")):
            s[to][dst.expand(kv, k), h, torch.arange(k, device=w.device) % ps] = s[pool][src, h, pick % ps]
    return {"kept": kept, "weights": w_out, "k": s["k_out"], "v": s["v_out"]}


def _plain(s):
    c = s["case"]
    op, B = c["op"], c["batch"]
    if op == "summarise":
        return _summarise(s, s["summaries"])
    if op == "evict":
        return _evict(s)
    dt = s["q"].dtype
    if op == "sparse":
        sel = _select(s)
        outs = []
        for b, n in enumerate(s["lens_host"]):
            k = min(c["top"], -(-n // c["page"]))
            outs.append(_attend(s, b, sel[b, :, :k].long())[0])
        return {"pages": sel, "out": torch.stack(outs).to(dt)}
    outs = []
    for b, n in enumerate(s["lens_host"]):
        o, p = _attend(s, b)
        outs.append(o)
        if op == "weigh":
            s["w_out"][b, :, :n] = s["w"][b, :, :n] + p.view(c["kv_heads"], -1, p.shape[-1]).sum(1)[:, :n]
    out = torch.stack(outs).to(dt)
    return {"out": out, "weights": s["w_out"]} if op == "weigh" else out


def run(s):
    if not own:
        return _plain(s)
    c, codec = s["case"], s["codec"]
    op, dt = c["op"], DTYPES[c["q"]]
    if op == "attend":
        return codec.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], out_dtype=dt)
    if op == "weigh":
        out = codec.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], weights=s["w"],
                                    weights_out=s["w_out"], out_dtype=dt)
        return {"out": out, "weights": s["w_out"]}
    if op == "sparse":
        sel = codec.select_pages(s["q"], s["summaries"], s["table"], s["lens"], c["page"], c["top"],
                                 sinks=c["sinks"], recent=c["recent"])
        out = codec.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], pages=sel, out_dtype=dt)
        return {"pages": sel, "out": out}
    if op == "summarise":
        return codec.summarize_pages(s["k"], s["table"], s["lens"], s["summaries"], start=s["start"])
    kept, w = codec.select_tokens(s["w"], s["lens"], c["keep"], sinks=c["sinks"], recent=c["recent"])
    codec.gather_tokens(s["k"], s["v"], s["table"], kept, s["k_out"], s["v_out"], s["table_out"])
    return {"kept": kept, "weights": w, "k": s["k_out"], "v": s["v_out"]}


# ---- the definition in 64 bits ---------------------------------------------------------------------
def exact(c, seed):
    """What ``run`` returns, from the definition, one (sequence, KV head) at a time in 64 bits."""
    if c["op"] in ("evict", "summarise"):
        return None                                      # copies and whole numbers: the plain form is the definition
    s = prepare(c, seed)
    dim, kv, hq, ps, B = c["dim"], c["kv_heads"], c["q_heads"], c["page"], c["batch"]
    G = hq // kv
    R, z, xy = s["R"].double(), s["z"].double(), s["xy"].double()
    fb = _flat_bits(c)
    out = torch.zeros(B, hq, dim, dtype=torch.float64, device=R.device)
    w = s["w_out"].double() if c["op"] == "weigh" else None
    sel = _select(s) if c["op"] == "sparse" else None
    for b, n in enumerate(s["lens_host"]):
        for h in range(kv):
            if sel is None:
                slots = torch.arange(n, device=R.device)
            else:
                pg = sel[b, h][sel[b, h] >= 0].long()
                slots = (pg[:, None] * ps + torch.arange(ps, device=R.device)).reshape(-1)
                slots = slots[slots < n]
            at = s["table"][b].long()[slots // ps]
            kc, vc = s["k"][at, h, slots % ps].long(), s["v"][at, h, slots % ps].long()
            qr = s["q"][b, h * G:(h + 1) * G].double() @ R.T
            x = (qr[:, 0::3] @ z[kc >> fb].T + qr[:, 1::3] @ xy[kc][..., 0].T + qr[:, 2::3] @ xy[kc][..., 1].T) / math.sqrt(dim)
            p = torch.softmax(x, -1)
            o = torch.stack([p @ z[vc >> fb], p @ xy[vc][..., 0], p @ xy[vc][..., 1]], -1).reshape(G, dim)
            out[b, h * G:(h + 1) * G] = o @ R
            if w is not None:
                w[b, h, :n] = s["w"][b, h, :n].double() + p.sum(0)
    if c["op"] == "weigh":
        return {"out": out, "weights": w}
    return {"pages": None, "out": out} if c["op"] == "sparse" else out
