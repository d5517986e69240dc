"""The operators of the 4-bit paged KV cache and of the cache's pages, measured as a serving program calls them.

``own = False``: each operator in elementary torch operations, in 32 bits, rounded once at the end. ``own = True``: the same
pass through the library (tessel_b200.gpu.Gpu).

Four kinds of case:

* ``write``: one layer's step of a model that keeps its cache in 4 bits: rotate Q and K, store the dense Q, K, V, quantise K
  and V into their cache slots (``rope_kv_q4``), and read the written slots back as f16 (``kv_unpack_q4``).
* ``decode``: paged grouped-query decode attention over the 4-bit cache (``decode_attention_q4``).
* ``chunk``: causal attention of pieces of prompts against the 4-bit cache (``chunk_attention_q4``).
* ``pages``: pages of all layers' K and V caches copied (``page_copy``): forks of a shared prefix, compaction.

The 4-bit cache: u8 [pages, kv heads, 16, D/2 + 2 D/64]. A (page, head) record is 16 rows of D/2 bytes of codes followed by 16
rows of D/64 16-bit headers, one for each 64 elements of a token's row: an f16 scale whose low four mantissa bits hold the zero
point instead. value = scale * (code - zero point), which an f16 holds exactly. Each 8 elements e0..e7 take four bytes: e0|e2<<4,
e4|e6<<4, e1|e3<<4, e5|e7<<4.
"""
import math
import random

import torch

own = False

PAGE = 16
DEV = "cuda"


# ---- the cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # The smallest serving step: 16 rows (the engine's least) of a TinyLlama-shaped layer, 3 of them padding.
        dict(name="write, 16 rows, 32/4/64", op="write", T=16, live=13, H=32, G=4, D=64),
        # The benchmark's decode step: 256 sequences, Llama-3-8B heads.
        dict(name="write, 256 rows, 32/8/128", op="write", T=256, live=256, H=32, G=8, D=128),
        # A packed prefill step of odd length, padded to a multiple of 256 rows.
        dict(name="write, 4352 rows, 32/8/128", op="write", T=4352, live=4173, H=32, G=8, D=128),
        # One user, short context: latency.
        dict(name="decode, 1 x 700, 32/4/64", op="decode", B=1, pad=0, H=32, G=4, D=64, lo=700, hi=700),
        # A batch that does not fill its step: 37 sequences of mixed lengths, 27 padding rows.
        dict(name="decode, 37 of 64, 32/8/128", op="decode", B=37, pad=27, H=32, G=8, D=128, lo=1, hi=3001),
        # The benchmark's decode step.
        dict(name="decode, 256 x 512-2304, 32/8/128", op="decode", B=256, pad=0, H=32, G=8, D=128, lo=512, hi=2304),
        # Few users with long documents.
        dict(name="decode, 4 x 131072, 32/8/128", op="decode", B=4, pad=0, H=32, G=8, D=128, lo=100000, hi=131072),
        # Short ends of prompts (or a handful of rows to score) for many sequences.
        dict(name="chunk, 8 x 1-8 rows, 32/8/128", op="chunk", C=8, rlo=1, rhi=8, H=32, G=8, D=128, lo=700, hi=6000),
        # Two prompts fed 512 rows at a time beside each other.
        dict(name="chunk, 2 x 512 at 3000-4000", op="chunk", C=2, rlo=500, rhi=512, H=32, G=8, D=128, lo=3000, hi=4000),
        # A long document fed in large pieces.
        dict(name="chunk, 2048 at 30000, 32/8/128", op="chunk", C=1, rlo=2048, rhi=2048, H=32, G=8, D=128, lo=30000, hi=30000),
        # Forking a prefix: the last, partly filled page for 7 new sequences, 32 layers of K and V, f16 pages.
        dict(name="pages, fork 7 x 64 of 32 KB", op="pages", A=64, NP=96, N=7, words=16 * 8 * 128),
        # Compacting a cache.
        dict(name="pages, move 190 x 64 of 32 KB", op="pages", A=64, NP=400, N=190, words=16 * 8 * 128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "decode", "chunk", "pages"])
    G = rng.choice([1, 2, 3, 4, 5, 8])
    H = G * rng.choice([1, 2, 3, 4, 7, 8])
    D = rng.choice([64, 128])
    if op == "write":
        T = _log(rng, 1, 4352)
        return dict(op=op, T=T, live=rng.randint(max(1, T // 2), T), H=min(H, 40), G=G, D=D)
    if op == "decode":
        B = _log(rng, 1, 256)
        hi = _log(rng, 1, max(2, min(131072, 550000 // B)))
        return dict(op=op, B=B, pad=rng.choice([0, 0, 1, rng.randint(0, 16)]), H=min(H, 40) // G * G, G=G, D=D,
                    lo=rng.randint(1, hi), hi=hi)
    if op == "chunk":
        C = rng.choice([1, 1, 2, 3, 5, 8])
        rhi = _log(rng, 1, 2048 // C)
        hi = _log(rng, 1, 30000 if rhi * C <= 512 else 12000)
        return dict(op=op, C=C, rlo=rng.randint(1, rhi), rhi=rhi, H=min(H, 32) // G * G, G=G, D=D, lo=rng.randint(0, hi), hi=hi)
    NP = _log(rng, 8, 400)
    return dict(op=op, A=rng.choice([2, 6, 32, 44, 64]), NP=NP, N=_log(rng, 1, NP // 2 - 1),
                words=16 * G * rng.choice([34, 64, 68, 128]))


def _lengths(c):
    """The tokens each decode row attends to (0: a padding row)."""
    r = random.Random("%s %s %s" % (c["B"], c["lo"], c["hi"]))
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["B"])] + [0] * c["pad"]


def _pieces(c):
    """(row0, nrows, pos0) of each piece, and the rows of the step: a row belongs to no piece between the pieces."""
    r = random.Random("%s %s %s %s %s" % (c["C"], c["rlo"], c["rhi"], c["lo"], c["hi"]))
    out, row = [], 0
    for _ in range(c["C"]):
        n = r.randint(c["rlo"], c["rhi"])
        out.append((row, n, r.randint(c["lo"], c["hi"])))
        row += n + 1
    return out, row


def _row_bytes(D):
    return D // 2 + 2 * (D // 64)


def work(c):
    if c["op"] == "pages":
        return {"bytes": 2.0 * 2 * c["A"] * c["N"] * c["words"], "flops": 0}
    H, G, D = c["H"], c["G"], c["D"]
    if c["op"] == "write":
        T, live = c["T"], c["live"]
        step = T * (H + 2 * G) * D * 2
        # QKV and the rotations in, the dense Q, K, V and the cache rows out, and the cache rows in and out again as f16.
        return {"bytes": 2.0 * step + T * (D * 4 + 8) + 2 * live * G * (2 * _row_bytes(D) + 2 * D), "flops": 6.0 * T * (H + G) * D}
    if c["op"] == "decode":
        n = _lengths(c)
        return {"bytes": sum(n) * G * 2.0 * _row_bytes(D) + len(n) * H * D * 4 + sum(-(-x // PAGE) for x in n) * 4 + 4 * len(n),
                "flops": 4.0 * H * D * sum(n)}
    p, T = _pieces(c)
    rows = sum(n for _, n, _ in p)
    seen = sum(n * pos + n * (n + 1) // 2 for _, n, pos in p)
    return {"bytes": sum(n + pos for _, n, pos in p) * G * 2.0 * _row_bytes(D) + rows * H * D * 4, "flops": 4.0 * H * D * seen}


# ---- the 4-bit format in torch -----------------------------------------------------------------------------------------
def _quantise(x):
    """f16 rows [..., D] -> codes u8 [..., D/64, 64], scale and zero point f64 [..., D/64]. In 64 bits: a range that divides to
    the edge of the scale's grid must not be pushed over it."""
    g = x.double().unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
    r = (hi - lo) / 15
    # Rounded up to seven significant bits (f16 subnormals: to a multiple of 2^-20).
    step = torch.exp2((torch.frexp(r).exponent.clamp(min=-13) - 7).double())
    scale = torch.ceil(r / step) * step
    div = torch.where(scale > 0, scale, 1.0)
    zero = torch.round(-lo / div).clamp(0, 15)
    codes = (torch.round(g / div.unsqueeze(-1)) + zero.unsqueeze(-1)).clamp(0, 15)
    return codes.to(torch.uint8), scale, zero


def _pack(codes, scale, zero):
    """Byte rows [..., D/2] and header rows [..., D/64] (int16)."""
    c = codes.flatten(-2).unflatten(-1, (-1, 8))
    b = torch.stack([c[..., 0] | c[..., 2] << 4, c[..., 4] | c[..., 6] << 4, c[..., 1] | c[..., 3] << 4, c[..., 5] | c[..., 7] << 4], -1)
    return b.flatten(-2), scale.half().view(torch.int16) | zero.to(torch.int16)


def _unpack(rows, heads):
    """The f32 values [..., D] that byte rows [..., D/2] and header rows [..., D/64] stand for."""
    b = rows.unflatten(-1, (-1, 4))
    lo, hi = b & 15, b >> 4
    c = torch.stack([lo[..., 0], lo[..., 2], hi[..., 0], hi[..., 2], lo[..., 1], lo[..., 3], hi[..., 1], hi[..., 3]], -1)
    scale, zero = (heads & -16).view(torch.float16).float(), (heads & 15).float()
    return ((c.flatten(-2).unflatten(-1, (-1, 64)).float() - zero.unsqueeze(-1)) * scale.unsqueeze(-1)).flatten(-2)


def _parts(cache, D):
    """A cache's codes [NP, G, 16, D/2] and headers [NP, G, 16, D/64], as views."""
    flat = cache.flatten(2)
    n = PAGE * D // 2
    return flat[..., :n].unflatten(-1, (PAGE, D // 2)), flat.view(torch.int16)[..., n // 2:].unflatten(-1, (PAGE, D // 64))


def _pages_of(cache, table, D):
    """f32 [rows, G, tokens, D]: the values of the pages that `table` [rows, MP] names."""
    rows, heads = _parts(cache, D)
    v = _unpack(rows[table], heads[table])  # [rows, MP, G, 16, D]
    return v.transpose(1, 2).flatten(2, 3)


# ---- inputs ------------------------------------------------------------------------------------------------------------
def prepare(c, seed):
    r = torch.Generator(DEV)
    r.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=r, device=DEV)
    s = {"case": c}
    if c["op"] == "pages":
        s["caches"] = torch.randint(-30000, 30000, (c["A"], c["NP"], c["words"]), generator=r, device=DEV, dtype=torch.int16).half()
        order = torch.randperm(c["NP"], generator=r, device=DEV)
        # Sources may repeat (a fork), destinations do not, and no page is both.
        src = order[: c["N"]][torch.randint(0, c["N"], (c["N"],), generator=r, device=DEV)]
        s["pairs"] = torch.stack([src, order[c["N"]: 2 * c["N"]]], 1).int().contiguous()
        # The caches' addresses, which a program writes once.
        s["bases"] = s["caches"].data_ptr() + torch.arange(c["A"], dtype=torch.int64, device=DEV) * (c["NP"] * c["words"] * 2)
        return s
    H, G, D = c["H"], c["G"], c["D"]
    if c["op"] == "write":
        T = c["T"]
        s["qkv"] = normal(T, (H + 2 * G) * D).half()
        npos = 8192
        ang = torch.arange(npos, dtype=torch.float64, device=DEV)[:, None] * (
            10000.0 ** (-torch.arange(D // 2, dtype=torch.float64, device=DEV) / (D // 2)))
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        s["pos"] = torch.randint(0, npos, (T,), generator=r, device=DEV, dtype=torch.int32)
        s["np"] = -(-T // PAGE) + 3
        slot = torch.randperm(s["np"] * PAGE, generator=r, device=DEV)[:T].int()
        slot[c["live"]:] = s["np"] * PAGE  # padding rows write to no slot
        s["slot"] = slot
        for k in ("kc", "vc"):
            s[k] = torch.zeros(s["np"], G, PAGE, _row_bytes(D), dtype=torch.uint8, device=DEV)
        return s
    if c["op"] == "decode":
        lens = _lengths(c)
        T = len(lens)
        pages = [-(-n // PAGE) for n in lens]
    else:
        pieces, T = _pieces(c)
        pages = [0] * T
        for row0, n, pos in pieces:
            pages[row0] = -(-(pos + n) // PAGE)
    mp, total = max(max(pages), 1), sum(pages)
    order = torch.randperm(total + 2, generator=r, device=DEV).int()
    table = torch.zeros(T, mp, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at: at + n]
        at += n
    s["table"] = table
    s["q"] = normal(T, H, D).half()
    for k in ("kc", "vc"):
        cache = torch.empty(total + 2, G, PAGE, _row_bytes(D), dtype=torch.uint8, device=DEV)
        rows, heads = _parts(cache, D)
        for a in range(0, total + 2, 4096):
            b = min(a + 4096, total + 2)
            rows[a:b], heads[a:b] = _pack(*_quantise(normal(b - a, G, PAGE, D).half()))
        s[k] = cache
    if c["op"] == "decode":
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    else:
        s["meta"] = torch.tensor([[a, n, p, 0] for a, n, p in pieces], dtype=torch.int32, device=DEV)
        s["o"] = torch.zeros(T, H, D, dtype=torch.float16, device=DEV)
        # Where each piece's rows lie in the step (a row beyond the piece: beyond the step), for the plain form.
        most = max(n for _, n, _ in pieces)
        i = torch.arange(most, device=DEV)
        m = s["meta"].long()
        s["rows"] = torch.where(i[None] < m[:, 1:2], m[:, :1] + i[None], T)
    s["scale"] = 1.0 / math.sqrt(D)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------
def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_write(s):
    c = s["case"]
    H, G, D = c["H"], c["G"], c["D"]
    x = s["qkv"].float().unflatten(-1, (H + 2 * G, D))
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    q, k = _rotate(x[:, :H], cos, sin).half(), _rotate(x[:, H: H + G], cos, sin).half()
    v = x[:, H + G:].half()
    slot = s["slot"].long()
    keep = (slot >= 0) & (slot < s["np"] * PAGE)
    live = slot[keep]
    page, at = slot.clamp(max=s["np"] * PAGE - 1) // PAGE, slot % PAGE
    out = {"q": q, "k": k, "v": v}
    kr, kh = _parts(s["kc"], D)
    vr, vh = _parts(s["vc"], D)
    kr[live // PAGE, :, live % PAGE], kh[live // PAGE, :, live % PAGE] = _pack(*_quantise(k[keep]))
    vr[live // PAGE, :, live % PAGE], vh[live // PAGE, :, live % PAGE] = _pack(*_quantise(v[keep]))
    drop = keep[:, None, None]
    out["kc"] = torch.where(drop, _unpack(kr[page, :, at], kh[page, :, at]), 0.0).half()
    out["vc"] = torch.where(drop, _unpack(vr[page, :, at], vh[page, :, at]), 0.0).half()
    return out


def _plain_decode(s):
    c = s["case"]
    H, G, D = c["H"], c["G"], c["D"]
    k, v = _pages_of(s["kc"], s["table"].long(), D), _pages_of(s["vc"], s["table"].long(), D)
    q = s["q"].float().unflatten(1, (G, H // G))
    x = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]  # [B, G, H/G, tokens]
    seen = torch.arange(x.shape[-1], device=DEV)[None] < s["lens"][:, None]
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))  # an empty row is 0/0: NaN
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).flatten(1, 2).half()


def _plain_chunk(s):
    c = s["case"]
    H, G, D = c["H"], c["G"], c["D"]
    m = s["meta"].long()
    table = s["table"][m[:, 0]].long()
    k, v = _pages_of(s["kc"], table, D), _pages_of(s["vc"], table, D)
    q = torch.cat([s["q"], s["q"][:1]])[s["rows"]].float()  # [C, R, H, D]
    C, R = q.shape[:2]
    q = q.unflatten(2, (G, H // G)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [C, G, H/G * R, D]
    x = torch.matmul(q, k.transpose(-1, -2)).unflatten(2, (H // G, R)).mul_(s["scale"])
    last = m[:, 2:3] + torch.arange(R, device=DEV)[None]  # the position of each row
    x.masked_fill_((torch.arange(x.shape[-1], device=DEV) > last[..., None])[:, None, None], -math.inf)
    p = x.sub_(x.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p.flatten(2, 3), v) / p.sum(-1).flatten(2, 3)[..., None]
    o = o.unflatten(2, (H // G, R)).permute(0, 3, 1, 2, 4).flatten(2, 3).half()
    live = s["rows"] < s["o"].shape[0]
    s["o"][s["rows"][live]] = o[live]
    return s["o"]


def _plain_pages(s):
    x, p = s["caches"], s["pairs"].long()
    x[:, p[:, 1]] = x[:, p[:, 0]]
    return x


# ---- the library's calls -----------------------------------------------------------------------------------------------
_gpu = None


def _plan(s):
    """What a program makes once for these buffers: the kernels and their arguments, in the order of their launches."""
    global _gpu
    from tessel_b200.gpu import F32, I32, Gpu
    if _gpu is None:
        _gpu = Gpu(0)
    c, g = s["case"], _gpu
    buf = lambda t: g.wrap(t.data_ptr(), t.numel() * t.element_size())
    made = lambda name, ts, *scalars: (g.kernel(name, [list(t.shape) for t in ts]), [buf(t) for t in ts] + list(scalars))
    if c["op"] == "pages":
        s["out"] = s["caches"]
        return [made("page_copy", [s["bases"], s["pairs"]], I32(c["N"]), I32(c["NP"]), I32(c["words"] * 2))]
    H, G, D = c["H"], c["G"], c["D"]
    if c["op"] == "write":
        T = c["T"]
        new = lambda heads: torch.empty(T, heads, D, dtype=torch.float16, device=DEV)
        o = s["out"] = {"q": new(H), "k": new(G), "v": new(G), "kc": new(G), "vc": new(G)}
        return [made("rope_kv_q4", [s["qkv"], s["pos"], s["slot"], s["cos"], s["sin"], o["q"], s["kc"], s["vc"], o["k"], o["v"]]),
                made("kv_unpack_q4", [s["kc"], s["vc"], s["slot"], o["kc"], o["vc"]])]
    if c["op"] == "decode":
        s["out"] = torch.empty_like(s["q"])
        return [made("decode_attention_q4", [s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["out"]], F32(s["scale"]))]
    s["out"] = s["o"]
    return [made("chunk_attention_q4", [s["q"], s["kc"], s["vc"], s["table"], s["meta"], s["o"]], F32(s["scale"]))]


def run(s):
    if not own:
        return {"write": _plain_write, "decode": _plain_decode, "chunk": _plain_chunk, "pages": _plain_pages}[s["case"]["op"]](s)
    if "plan" not in s:
        s["plan"] = _plan(s)
    for kernel, args in s["plan"]:
        _gpu.launch(kernel, args)
    return s["out"]


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
_ORDER = [0, 4, 1, 5, 2, 6, 3, 7]  # the nibble of a 32-bit word that holds element 0..7


def _exact_values(record, D):
    """f64 [n, 16, D] of records [n, 16 * row bytes]: nibble by nibble, header by header."""
    n, cut = record.shape[0], PAGE * D // 2
    by = record[:, :cut].reshape(n, PAGE, D // 8, 4).long()
    word = by[..., 0] + (by[..., 1] << 8) + (by[..., 2] << 16) + (by[..., 3] << 24)
    code = torch.stack([(word >> (4 * k)) & 15 for k in _ORDER], -1).reshape(n, PAGE, D).double()
    hb = record[:, cut:].reshape(n, PAGE, D // 64, 2).long()
    head = hb[..., 0] + (hb[..., 1] << 8)
    e, m = (head >> 10) & 31, (head >> 4) & 63
    scale = torch.where(e > 0, (64 + m).double() * torch.exp2((e - 15 - 6).double()), m.double() * 2.0 ** -20)
    return (code - (head & 15).double().repeat_interleave(64, -1)) * scale.repeat_interleave(64, -1)


def _exact_quantised(x):
    """f64 rows [n, D] (of f16 numbers) as the cache holds them."""
    g = x.reshape(-1, 64)
    lo, hi = torch.clamp(g.min(1).values, max=0.0), torch.clamp(g.max(1).values, min=0.0)
    r = (hi - lo) / 15.0
    e = torch.floor(torch.log2(torch.clamp(r, min=2.0 ** -14)))
    e = torch.where(torch.exp2(e + 1) <= r, e + 1, e)
    grid = torch.exp2(e - 6)
    scale = torch.ceil(r / grid) * grid
    d = torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]
    zero = torch.clamp(torch.round(-lo[:, None] / d), 0, 15)
    return ((torch.clamp(torch.round(g / d) + zero, 0, 15) - zero) * scale[:, None]).reshape(x.shape)


def _exact_attention(q, k, v, scale, first):
    """q [H, R, D], k and v [G, N, D] in f64; row i sees keys 0 .. first + i."""
    H, R, D = q.shape
    out = torch.empty_like(q)
    hidden = torch.arange(k.shape[1], device=DEV)[None] > first + torch.arange(R, device=DEV)[:, None]
    for h in range(H):
        kh, vh = k[h * k.shape[0] // H], v[h * k.shape[0] // H]
        for a in range(0, R, 512):
            x = (q[h, a: a + 512] @ kh.T) * scale
            out[h, a: a + 512] = torch.softmax(x.masked_fill(hidden[a: a + 512], -math.inf), -1) @ vh
    return out


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "pages":
        x = s["caches"].clone()
        for a, b in s["pairs"].tolist():
            x[:, b] = s["caches"][:, a]
        return x
    H, G, D = c["H"], c["G"], c["D"]
    if c["op"] == "write":
        T = c["T"]
        x = s["qkv"].double().reshape(T, H + 2 * G, D)
        cos, sin = s["cos"].double()[s["pos"].long()][:, None], s["sin"].double()[s["pos"].long()][:, None]
        a, b = x[..., : D // 2], x[..., D // 2:]
        rot = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        k16 = rot[:, H: H + G].half().double()  # the cache is made from K as f16 holds it
        live = ((s["slot"] >= 0) & (s["slot"] < s["np"] * PAGE)).double()[:, None, None]
        held = lambda y: _exact_quantised(y.reshape(-1, D)).reshape(T, G, D) * live
        return {"q": rot[:, :H], "k": rot[:, H: H + G], "v": x[:, H + G:], "kc": held(k16), "vc": held(x[:, H + G:])}
    q = s["q"].double()
    fetch = lambda name, row, n: torch.stack([
        _exact_values(s[name][s["table"][row, : -(-n // PAGE)].long(), g].reshape(-(-n // PAGE), -1), D).reshape(-1, D)[:n]
        for g in range(G)])
    if c["op"] == "decode":
        out = torch.full((len(q), H, D), math.nan, dtype=torch.float64, device=DEV)
        for b, n in enumerate(_lengths(c)):
            if n:
                out[b] = _exact_attention(q[b][:, None], fetch("kc", b, n), fetch("vc", b, n), s["scale"], n - 1)[:, 0]
        return out
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for row0, n, pos in _pieces(c)[0]:
        o = _exact_attention(q[row0: row0 + n].transpose(0, 1), fetch("kc", row0, pos + n), fetch("vc", row0, pos + n), s["scale"], pos)
        out[row0: row0 + n] = o.transpose(0, 1)
    return out
