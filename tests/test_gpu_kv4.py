"""The 4-bit KV cache and page copies on the GPU, through the C ABI: the cache's bytes against the host quantiser
(tessel_b200/kv4.py), attention against the definition in 64 bits on the values the cache stands for, and the engine and the
scheduler on them.

Attention's tolerance, per element: the f16 result is off by half a step, 2^-11 |want|, and by what the f32 arithmetic in front
of it loses. A score is a sum of D products code * q, |code - zero| <= 15, in f32 (2^-24 a step, at most 32 steps deep on any
path, zero point's part of the same size): off by at most ds = 2 * 32 * 2^-24 * scale * 15 * max header scale * sum |q|. An
error ds of every score moves a weight by a factor within exp(+-ds), so the mean of the v by at most 2 ds max |v|; the weights'
own arithmetic (exp2 to 2 ulp, products split in two f16, the sums of both, some hundred roundings of 2^-24) by 2^-16 max |v|.
Where the weights are rounded to f16 before they weigh V (chunk_attention_q4) 2^-11 max |v| more.
"""
import numpy as np
import pytest

import oracle
from emu import EmuGpu
from refs import rel_err
from tessel_b200 import kv4
from tessel_b200.engine import Decode, Engine, Limits, Mixed, Packed, Prefill
from tessel_b200.gpu import F32, GpuError, I32
from tessel_b200.model import Config, Weights, argmax, rope_tables
from tessel_b200.sched import Request, Scheduler, generate_with

pytestmark = pytest.mark.gpu
h, f, i32, u8, f64 = np.float16, np.float32, np.int32, np.uint8, np.float64


def run(gpu, name, arrays, outs, scalars=()):
    bufs = [gpu.tensor(a) for a in arrays]
    gpu.launch(gpu.kernel(name, [a.shape for a in arrays]), bufs + list(scalars))
    gpu.sync()
    res = [gpu.fetch(bufs[i], arrays[i].dtype, arrays[i].shape) for i in outs]
    for b in bufs:
        gpu.free(b)
    return res


def new_cache(NP, G, P, D, fill=0xA5):
    return np.full((NP, G, P, kv4.row_bytes(D)), fill, u8)


# ---- the cache write and its inverse -----------------------------------------------------------------------------------
def write_case(seed, T, H, G, D, P, NP):
    r = np.random.default_rng(seed)
    W = (H + 2 * G) * D
    qkv = r.standard_normal((T, W)).astype(h)
    kv = qkv[:, H * D:].reshape(T, 2 * G, D)
    if T >= 8:
        kv[1] = 0                                     # scale 0
        kv[2, 0, 3] = np.inf                          # a spoilt group of K (the rotation spreads it to its partner) ...
        kv[2, G, 5] = np.nan                          # ... and of V
        kv[3, G:] = np.abs(kv[3, G:])                 # zero point 0
        kv[4, G:] = -np.abs(kv[4, G:])                # zero point 15
        kv[5] = (kv[5].astype(f64) * 2.0 ** -19).astype(h)   # subnormal numbers and scales
        kv[6, G:, ::2], kv[6, G:, 1::2] = 65504, -65504
        kv[7, G:, 0] = 65504
    npos = 4 * T + 9
    c, s = rope_tables(Config(dim=64, layers=1, heads=1, kv_heads=1, head_dim=D, ffn=64, vocab=8, max_pos=npos, eos=-1))
    pos = r.integers(0, npos, T).astype(i32)
    slot = r.permutation(NP * P)[:T].astype(i32) if T <= NP * P else np.arange(T, dtype=i32)
    if T >= 8:
        pos[0], slot[T // 2], slot[T - 1] = npos, NP * P, -1   # a position and slots that do not exist
    return qkv, pos, slot, np.asarray(c, f), np.asarray(s, f)


@pytest.mark.parametrize("T,H,G,D,P,NP", [(1, 1, 1, 16, 2, 1), (16, 32, 4, 64, 16, 4), (77, 6, 3, 96, 16, 9), (33, 2, 1, 256, 4, 11),
                                          (256, 32, 8, 128, 16, 40), (40, 5, 5, 48, 6, 7), (300, 4, 1, 128, 16, 16)])
def test_rope_kv_q4_writes_the_host_quantisers_bytes(gpu, T, H, G, D, P, NP):
    qkv, pos, slot, c, s = write_case(T + D, T, H, G, D, P, NP)
    z = lambda n: np.full((T, n, D), 7, h)
    kc, vc = new_cache(NP, G, P, D), new_cache(NP, G, P, D)
    q, kq, vq, k, v = run(gpu, "rope_kv_q4", [qkv, pos, slot, c, s, z(H), kc, vc, z(G), z(G)], [5, 6, 7, 8, 9])
    flat = np.zeros((1, G, D), h)
    wq, wk, wv = run(gpu, "rope_kv", [qkv, pos, np.full(T, 1, i32), c, s, z(H), flat, flat, z(G), z(G)], [5, 8, 9])
    assert q.tobytes() == wq.tobytes() and k.tobytes() == wk.tobytes() and v.tobytes() == wv.tobytes()
    wantk, wantv = new_cache(NP, G, P, D), new_cache(NP, G, P, D)
    kv4.write(wantk, slot, k)
    kv4.write(wantv, slot, v)
    assert kq.tobytes() == wantk.tobytes(), "K"
    assert vq.tobytes() == wantv.tobytes(), "V"
    # Back again: what the cache stands for, exactly, and zeros for slots that do not exist.
    at = np.concatenate([slot, [NP * P, -5, 0]]).astype(i32)
    n = len(at)
    y = np.full((n, G, D), 7, h)
    uk, uv = run(gpu, "kv_unpack_q4", [kq, vq, at, y, y.copy()], [3, 4])
    ok = (at >= 0) & (at < NP * P)
    for got, cache in ((uk, kq), (uv, vq)):
        want = np.where(ok[:, None, None], kv4.read(cache, D).reshape(NP * P, G, D)[np.where(ok, at, 0)], h(0))
        assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("D", [64, 128])
def test_rope_kv_q4_rounds_the_scale_up_from_the_exact_range(gpu, D):
    from test_kv4 import far_bounds
    x = far_bounds()
    T, G, H = len(x), 2, 1
    x = np.stack([x, -x], 1)                                   # [T, G, 64]
    kv = np.concatenate([x, x[::-1]], -1)[..., :D]
    qkv = np.zeros((T, (H + 2 * G) * D), h)
    qkv[:, H * D:(H + G) * D], qkv[:, (H + G) * D:] = kv.reshape(T, -1), kv[::-1].reshape(T, -1)
    c, s = np.ones((1, D // 2), f), np.zeros((1, D // 2), f)   # the rotation leaves K as it is
    NP = -(-T // 16)
    z = lambda n: np.zeros((T, n, D), h)
    kc, vc = new_cache(NP, G, 16, D), new_cache(NP, G, 16, D)
    slot = np.arange(T, dtype=i32)
    kq, vq, k, v = run(gpu, "rope_kv_q4", [qkv, np.zeros(T, i32), slot, c, s, z(H), kc, vc, z(G), z(G)], [6, 7, 8, 9])
    assert np.array_equal(k, kv) and np.array_equal(v, kv[::-1])
    for got, rows in ((kq, kv), (vq, kv[::-1])):
        want = new_cache(NP, G, 16, D)
        kv4.write(want, slot, rows)
        assert got.tobytes() == want.tobytes()


# ---- attention ---------------------------------------------------------------------------------------------------------
def attention_case(seed, B, H, G, D, P, pages):
    """Queries, caches of quantised rows in scrambled pages, and a block table of `pages[b]` pages for row b."""
    r = np.random.default_rng(seed)
    NP = sum(pages) + 2
    cache = []
    for _ in range(2):
        c = np.zeros((NP, G, P, kv4.row_bytes(D)), u8)
        code, head = kv4.parts(c, D)
        # Rows of different sizes and offsets, so that scales and zero points vary over tokens, heads and groups.
        x = r.standard_normal((NP, G, P, D)) * np.exp(0.5 * r.standard_normal((NP, G, P, 1))) + 0.5 * r.standard_normal((NP, G, 1, D))
        cd, hd = kv4.quantize(x.astype(h))
        code[:], head[:] = kv4.pack(cd), hd
        cache.append(c)
    order, at = r.permutation(NP), 0
    table = np.zeros((B, max(max(pages), 1)), i32)
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    q = r.standard_normal((B, H, D)).astype(h)
    return q, cache[0], cache[1], table


def attend(q, kc, vc, row, first, scale, f16_weights=False):
    """f64: q [R, H, D]; row i sees keys 0 .. first + i of block table `row`. The result and its tolerance."""
    R, H, D = q.shape
    NP, G, P, _ = kc.shape
    n = first + R
    col = np.arange(-(-n // P))
    page = np.where(col < len(row), row[np.minimum(col, len(row) - 1)], 0)
    inside = (page >= 0) & (page < NP)
    fetch = lambda c: np.where(inside[:, None, None, None], kv4.read(c[np.where(inside, page, 0)], D),
                               0).reshape(-1, G, D)[:n].astype(f64)
    k, v = fetch(kc), fetch(vc)
    heads = (kv4.parts(kc, D)[1] & np.uint16(0xFFF0)).view(h).astype(f64).max()
    out, tol = np.zeros((R, H, D)), np.zeros((R, H, 1))
    for hh in range(H):
        g = hh // (H // G)
        x = q[:, hh].astype(f64) @ k[:, g].T * f64(f(scale))
        x[np.arange(n)[None] > first + np.arange(R)[:, None]] = -np.inf
        p = np.exp(x - x.max(1, keepdims=True))
        out[:, hh] = p @ v[:, g] / p.sum(1, keepdims=True)
        ds = 2 * 32 * 2.0 ** -24 * abs(scale) * 15 * heads * np.abs(q[:, hh].astype(f64)).sum(1, keepdims=True)
        tol[:, hh] = (2 * ds + 2.0 ** -16 + (2.0 ** -11 if f16_weights else 0)) * np.abs(v[:, g]).max()
    return out, 2.0 ** -11 * np.abs(out) + tol + 2.0 ** -25


def near(got, want, tol):
    d = np.abs(got.astype(f64) - want)
    assert np.isfinite(got.astype(f64)).all()
    assert (d <= tol).all(), f"off by {d.max()}, {(d / tol).max()} of the tolerance"


def decode_q4(gpu, q, kc, vc, table, lens, scale):
    return run(gpu, "decode_attention_q4", [q, kc, vc, table, np.asarray(lens, i32), np.full(q.shape, 3, h)], [5], [F32(scale)])[0]


DECODES = [
    (1, 1, 16, 2, [1, 2, 3, 9]),                          # generic shapes
    (6, 3, 96, 16, [37, 1, 64, 0, 15]),
    (4, 2, 256, 8, [5, 64, 0, 41]),
    (2, 2, 48, 6, [100, 7]),
    (32, 4, 64, 16, [700]),
    (8, 1, 64, 16, [1, 15, 16, 17, 31, 32, 33, 500, 0]),
    (32, 8, 128, 16, [1, 15, 16, 17, 1000, 2303, 0, 512, 255, 257]),
    (8, 8, 128, 16, [63, 64, 65, 4000]),                  # one query head per KV head
    (24, 8, 128, 16, [130, 3000]),                        # three
    (14, 2, 128, 16, [333, 40]),                          # seven
    (20, 2, 64, 16, [100, 260, 1]),                       # ten: two groups of heads
    (16, 1, 128, 16, [100, 9000]),                        # multi-query
    (40, 5, 64, 16, [2000, 0, 5]),
]


@pytest.mark.parametrize("H,G,D,P,lens", DECODES)
def test_decode_attention_q4(gpu, H, G, D, P, lens):
    q, kc, vc, table = attention_case(len(lens) + D, len(lens), H, G, D, P, [-(-n // P) for n in lens])
    scale = D ** -0.5
    got = decode_q4(gpu, q, kc, vc, table, lens, scale)
    for b, n in enumerate(lens):
        if n == 0:
            assert np.isnan(got[b].astype(f)).all(), "an empty row is 0/0, as in decode_attention"
            continue
        near(got[b][None], *attend(q[b][None], kc, vc, table[b], n - 1, scale))


@pytest.mark.parametrize("H,G,D,P", [(32, 8, 128, 16), (8, 2, 64, 16), (4, 2, 32, 8)])
def test_decode_attention_q4_ignores_what_it_must_not_see(gpu, H, G, D, P):
    """Stale rows behind the last token (NaN headers among them), pages that no table names, a length beyond the table (page 0,
    as decode_attention) and pages outside the cache (zeros)."""
    lens = [5, 3 * P + 1, 2 * P]
    q, kc, vc, table = attention_case(7, 3, H, G, D, P, [1, 4, 2])
    scale = D ** -0.5
    a = decode_q4(gpu, q, kc, vc, table, lens, scale)
    bk, bv = kc.copy(), vc.copy()
    for c in (bk, bv):
        code, head = kv4.parts(c, D)
        for b, n in enumerate(lens):
            if n % P:
                page = table[b, n // P]
                head[page, :, n % P:] = 0x7E00
                code[page, :, n % P:] = 0xFF
        for page in set(range(c.shape[0])) - set(table[0, :1]) - set(table[1]) - set(table[2, :2]):
            head[page] = 0x7E00
    assert a.tobytes() == decode_q4(gpu, q, bk, bv, table, lens, scale).tobytes()
    # Past the table, and outside the cache.
    lens = [4 * P + 3, 3 * P + 1, 2 * P]
    table[1, 1], table[1, 2] = kc.shape[0], -1
    got = decode_q4(gpu, q, kc, vc, table, lens, scale)
    for b, n in enumerate(lens):
        near(got[b][None], *attend(q[b][None], kc, vc, table[b], n - 1, scale))


def test_decode_attention_q4_spreads_nans_to_their_sequence_only(gpu):
    q, kc, vc, table = attention_case(8, 3, 8, 2, 128, 16, [3, 3, 3])
    kv4.parts(kc, 128)[1][table[1, 1], 0, 4, 0] = 0x7E00
    kv4.parts(vc, 128)[1][table[2, 0], 1, 2, 1] = 0x7E00
    got = decode_q4(gpu, q, kc, vc, table, [48, 40, 41], 0.1).astype(f)
    assert np.isfinite(got[0]).all()
    assert np.isnan(got[1, :4]).all() and np.isfinite(got[1, 4:]).all()
    assert np.isnan(got[2, 4:, 64:]).all() and np.isfinite(got[2, 4:, :64]).all() and np.isfinite(got[2, :4]).all()


@pytest.mark.parametrize("scale,size", [(8.0, 1.0), (-0.3, 1.0), (0.0, 1.0), (0.088, 300.0)])
def test_decode_attention_q4_at_peaked_and_flat_scores(gpu, scale, size):
    lens = [2000, 33]
    q, kc, vc, table = attention_case(9, 2, 8, 2, 128, 16, [125, 3])
    q = (q * h(size)).astype(h) if size != 1.0 else q
    got = decode_q4(gpu, q, kc, vc, table, lens, scale)
    for b, n in enumerate(lens):
        near(got[b][None], *attend(q[b][None], kc, vc, table[b], n - 1, scale))


def test_decode_attention_q4_long_context_is_split_and_joined(gpu):
    n = 70001
    q, kc, vc, table = attention_case(10, 2, 8, 2, 64, 16, [-(-n // 16), 3])
    got = decode_q4(gpu, q, kc, vc, table, [n, 40], 0.125)
    near(got[0][None], *attend(q[0][None], kc, vc, table[0], n - 1, 0.125))
    near(got[1][None], *attend(q[1][None], kc, vc, table[1], 39, 0.125))


def chunk_q4(gpu, q, kc, vc, table, meta, scale, fill=3):
    return run(gpu, "chunk_attention_q4", [q, kc, vc, table, np.asarray(meta, i32), np.full(q.shape, fill, h)], [5], [F32(scale)])[0]


CHUNKS = [  # heads, kv heads, D, page, pieces (row0, rows, pos0), rows of the step
    (1, 1, 16, 2, [(0, 3, 0)], 3),
    (6, 3, 96, 16, [(2, 9, 30), (12, 1, 0)], 14),
    (4, 2, 256, 8, [(0, 17, 5)], 20),
    (8, 2, 64, 16, [(0, 1, 0)], 1),
    (8, 2, 64, 16, [(1, 1, 700), (3, 5, 0), (9, 8, 1000)], 20),
    (32, 8, 128, 16, [(0, 7, 333), (8, 64, 0), (72, 65, 191)], 160),
    (32, 8, 128, 16, [(5, 300, 1000)], 310),
    (8, 8, 128, 16, [(0, 129, 127), (130, 257, 0)], 400),
    (14, 2, 128, 16, [(0, 40, 50)], 40),                   # seven query heads per KV head
    (20, 2, 64, 16, [(0, 70, 3)], 71),                     # ten
    (24, 1, 64, 16, [(0, 33, 3), (33, 31, 64)], 64),
    (3, 1, 128, 16, [(0, 512, 0)], 512),
    (4, 1, 128, 16, [(1, 6, 20000)], 8),                   # few rows, many keys
]


@pytest.mark.parametrize("H,G,D,P,pieces,T", CHUNKS)
def test_chunk_attention_q4(gpu, H, G, D, P, pieces, T):
    pages = [0] * T
    for row0, n, pos in pieces:
        pages[row0] = -(-(pos + n) // P)
    q, kc, vc, table = attention_case(T + D, T, H, G, D, P, pages)
    scale = D ** -0.5
    # Pieces outside the step, an empty one, and the padding descriptors of an engine's step are skipped.
    meta = [(a, n, p, 0) for a, n, p in pieces] + [(0, 0, 0, 0), (T - 1, 2, 0, 0), (-1, 1, 0, 0), (0, 1, -1, 0), (T, 1, 0, 0)]
    got = chunk_q4(gpu, q, kc, vc, table, meta, scale)
    rest = np.ones(T, bool)
    for row0, n, pos in pieces:
        near(got[row0:row0 + n], *attend(q[row0:row0 + n], kc, vc, table[row0], pos, scale, True))
        rest[row0:row0 + n] = False
    assert (got[rest] == 3).all(), "rows outside every piece were written"


@pytest.mark.parametrize("H,G,D,P", [(8, 2, 128, 16), (8, 2, 64, 16), (4, 2, 32, 8)])
def test_chunk_attention_q4_ignores_what_it_must_not_see(gpu, H, G, D, P):
    n, pos = 21, 3 * P + 5
    pages = -(-(pos + n) // P)
    q, kc, vc, table = attention_case(11, n + 1, H, G, D, P, [pages] + [0] * n)
    meta, scale = [(0, n, pos, 0)], D ** -0.5
    a = chunk_q4(gpu, q, kc, vc, table, meta, scale)
    bk, bv = kc.copy(), vc.copy()
    for c in (bk, bv):
        code, head = kv4.parts(c, D)
        end = (pos + n) % P
        if end:
            head[table[0, pages - 1], :, end:] = 0x7E00
            code[table[0, pages - 1], :, end:] = 0xFF
        for page in set(range(c.shape[0])) - set(table[0]):
            head[page] = 0x7E00
    assert a.tobytes() == chunk_q4(gpu, q, bk, bv, table, meta, scale).tobytes()
    # A later row's key must not reach an earlier row.
    code, head = kv4.parts(bk, D)
    at = pos + n - 1
    head[table[0, at // P], :, at % P] = 0x7E00
    b = chunk_q4(gpu, q, bk, bv, table, meta, scale)
    assert b[:n - 1].tobytes() == a[:n - 1].tobytes() and np.isnan(b[n - 1].astype(f)).all()
    # A position beyond the table lies on page 0, a page outside the cache reads as zeros.
    short = table[:, :2].copy()
    short[0, 1] = kc.shape[0] + 3
    got = chunk_q4(gpu, q, kc, vc, short, meta, scale)
    near(got[:n], *attend(q[:n], kc, vc, short[0], pos, scale, True))


def test_attention_agrees_between_a_decode_row_and_a_piece_of_one_row(gpu):
    q, kc, vc, table = attention_case(12, 4, 32, 8, 128, 16, [20, 70, 1, 9])
    lens = [311, 1111, 1, 144]
    a = decode_q4(gpu, q, kc, vc, table, lens, 0.088)
    b = chunk_q4(gpu, q, kc, vc, table, [(r, 1, n - 1, 0) for r, n in enumerate(lens)], 0.088)
    for r, n in enumerate(lens):
        want, tol = attend(q[r][None], kc, vc, table[r], n - 1, 0.088, True)
        near(a[r][None], want, tol)
        near(b[r][None], want, tol)


def spoil(rng, cache, table, rows, D, share):
    """Marks a share of the groups of the tokens that `rows` (table row, tokens) name as NaN."""
    head = kv4.parts(cache, D)[1]
    for b, n in rows:
        for t in np.nonzero(rng.random(n) < share)[0]:
            head[table[b, t // 16], rng.integers(0, head.shape[1]), t % 16, rng.integers(0, head.shape[3])] = 0x7E00


@pytest.mark.parametrize("H,G,D", [(32, 8, 128), (8, 8, 128), (16, 2, 64), (3, 1, 128), (10, 5, 64)])
def test_decode_attention_q4_many_short_rows(gpu, H, G, D):
    """Shares that run over many sequences and heads: units that lie whole in a share, cut ones, empty rows between them, and
    spoilt values that must stay in their head, group and sequence."""
    r = np.random.default_rng(D + H)
    lens = np.where(r.random(300) < 0.2, 0, r.integers(1, 90, 300)).astype(i32)
    q, kc, vc, table = attention_case(21 + H, 300, H, G, D, 16, [-(-n // 16) for n in lens])
    spoil(r, vc, table, [(b, lens[b]) for b in range(0, 300, 3)], D, 0.02)
    spoil(r, kc, table, [(b, lens[b]) for b in range(1, 300, 7)], D, 0.01)
    clean = without_nans(kc, D), without_nans(vc, D)
    got = decode_q4(gpu, q, kc, vc, table, lens, D ** -0.5)
    for b, n in enumerate(lens):
        if n == 0:
            assert np.isnan(got[b].astype(f)).all()
            continue
        check_with_nans(got[b][None], q[b][None], (kc, vc), clean, table[b], n - 1, D ** -0.5, False)


@pytest.mark.parametrize("H,G,D,P", [(32, 8, 128, 16), (8, 1, 128, 16), (16, 2, 64, 16), (4, 2, 32, 8)])
def test_attention_q4_keeps_bad_queries_to_themselves(gpu, H, G, D, P):
    """A query with an infinity or a NaN has NaN as its result (an infinite score less an infinite maximum), and no other
    head, row or sequence changes: bit for bit the result without it."""
    lens = np.array([1, 40, 700, 33, 300], i32)
    q, kc, vc, table = attention_case(31, 5, H, G, D, P, [-(-int(n) // P) for n in lens])
    dirty = q.copy()
    dirty[1, 1, 3], dirty[2, H - 1, D - 1], dirty[4, 0, 0] = np.inf, -np.inf, np.nan
    bad = [(1, 1), (2, H - 1), (4, 0)]
    clean, got = (decode_q4(gpu, x, kc, vc, table, lens, D ** -0.5) for x in (q, dirty))
    keep = np.ones((5, H), bool)
    for b, hh in bad:
        assert np.isnan(got[b, hh].astype(f)).all()
        keep[b, hh] = False
    assert np.array_equal(got[keep].view(np.uint16), clean[keep].view(np.uint16))
    pieces = [(0, 2, 50, 0), (2, 3, 200, 0)]
    q, kc, vc, table = attention_case(32, 5, H, G, D, P, [-(-60 // P), 0, -(-210 // P), 0, 0])
    dirty = q.copy()
    dirty[1, 1, 3], dirty[2, H - 1, D - 1], dirty[4, 0, 0] = np.inf, -np.inf, np.nan
    clean, got = (chunk_q4(gpu, x, kc, vc, table, pieces, D ** -0.5) for x in (q, dirty))
    for b, hh in bad:
        assert np.isnan(got[b, hh].astype(f)).all()
    assert np.array_equal(got[keep].view(np.uint16), clean[keep].view(np.uint16))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 3, 4])
def test_attention_q4_of_every_head_layout(gpu, D, G):
    """One to seventeen query heads per KV head on one to four KV heads: every way warps and tiles are laid out, with
    sequences that end in a page, at its end, and are cut among many shares."""
    for hq in (1, 2, 3, 4, 5, 7, 8, 9, 16, 17):
        lens = np.array([1, 16, 0, 333, 1500], i32)
        q, kc, vc, table = attention_case(100 * D + 10 * G + hq, 5, hq * G, G, D, 16, [-(-int(n) // 16) for n in lens])
        got = decode_q4(gpu, q, kc, vc, table, lens, D ** -0.5)
        for b, n in enumerate(lens):
            if n:
                near(got[b][None], *attend(q[b][None], kc, vc, table[b], n - 1, D ** -0.5))
            else:
                assert np.isnan(got[b].astype(f)).all()
        pieces = [(0, 1, 200), (2, 40, 100), (43, 2, 1400)]
        q, kc, vc, table = attention_case(100 * D + 10 * G + hq, 46, hq * G, G, D, 16, [13] + [0] + [9] + [0] * 40 + [88, 0, 0])
        got = chunk_q4(gpu, q, kc, vc, table, [(a, n, at, 0) for a, n, at in pieces], D ** -0.5)
        for a, n, at in pieces:
            near(got[a:a + n], *attend(q[a:a + n], kc, vc, table[a], at, D ** -0.5, True))
        assert (got[[1, 42, 45]] == 3).all()


@pytest.mark.parametrize("H,G,D,P", [(32, 8, 128, 16), (8, 1, 64, 16), (4, 2, 32, 8)])
def test_attention_q4_values_of_very_different_sizes(gpu, H, G, D, P):
    """Values between 2^-20 and the largest f16, groups of zeros among them, growing and shrinking along the sequence:
    the error stays a rounding of the largest."""
    r = np.random.default_rng(5)
    lens = np.array([700, 33, 1, 260], i32)
    q, kc, vc, table = attention_case(77, 4, H, G, D, P, [-(-int(n) // P) for n in lens])
    code, head = kv4.parts(vc, D)
    size = 2.0 ** np.sort(r.uniform(-20, 13, (vc.shape[0], 1, P, 1)), axis=2)
    size[::2] = size[::2, :, ::-1]                       # up along one page, down along the next
    x = (r.standard_normal((vc.shape[0], G, P, D)) * size).clip(-65504, 65504)
    x[r.random((vc.shape[0], G, P)) < 0.1] = 0
    cd, hd = kv4.quantize(x.astype(h))
    code[:], head[:] = kv4.pack(cd), hd
    got = decode_q4(gpu, q, kc, vc, table, lens, D ** -0.5)
    for b, n in enumerate(lens):
        near(got[b][None], *attend(q[b][None], kc, vc, table[b], n - 1, D ** -0.5))
    got = chunk_q4(gpu, q, kc, vc, table, [(0, 1, 600, 0), (1, 1, 32, 0), (3, 1, 255, 0)], D ** -0.5)
    for b, n in ((0, 600), (1, 32), (3, 255)):
        near(got[b][None], *attend(q[b][None], kc, vc, table[b], n, D ** -0.5, True))


@pytest.mark.parametrize("H,G,D,P", [(32, 8, 128, 16), (16, 2, 64, 16), (5, 5, 128, 16), (4, 2, 32, 8)])
def test_attention_q4_of_a_single_token_is_its_value(gpu, H, G, D, P):
    q, kc, vc, table = attention_case(8, 40, H, G, D, P, [1] * 40)
    want = np.repeat(kv4.read(vc, D)[table[:, 0], 0], H // G, axis=1)
    assert np.array_equal(decode_q4(gpu, q, kc, vc, table, [1] * 40, D ** -0.5), want)
    assert np.array_equal(chunk_q4(gpu, q, kc, vc, table, [(b, 1, 0, 0) for b in range(40)], D ** -0.5), want)


def without_nans(c, D):
    """`c` with its spoilt groups as zeros."""
    c = c.copy()
    head = kv4.parts(c, D)[1]
    head[head == 0x7E00] = 0
    return c


def check_with_nans(got, q, caches, clean, row, first, scale, f16_weights):
    """As `near`, where spoilt keys and values make NaNs: exactly the NaNs of the definition, and the rest near it."""
    D, (kc, vc) = q.shape[2], caches
    want, tol = attend(q, clean[0], clean[1], row, first, scale, f16_weights)
    bad = np.zeros(got.shape, bool)
    G = kc.shape[1]
    for i in range(q.shape[0]):
        t = np.arange(first + i + 1)
        for g in range(G):
            heads = slice(g * (q.shape[1] // G), (g + 1) * (q.shape[1] // G))
            if (kv4.parts(kc, D)[1][row[t // 16], g, t % 16] == 0x7E00).any():
                bad[i, heads] = True
            spoilt = (kv4.parts(vc, D)[1][row[t // 16], g, t % 16] == 0x7E00).any(0)
            bad[i, heads] |= np.repeat(spoilt, 64)
    assert np.array_equal(np.isnan(got.astype(f)), bad)
    ok = ~bad
    assert (np.abs(got.astype(f64) - want)[ok] <= np.broadcast_to(tol, want.shape)[ok]).all()


@pytest.mark.parametrize("H,G,D,most", [(32, 8, 128, 6), (8, 8, 128, 150), (16, 2, 64, 70), (128, 1, 64, 3), (100, 1, 128, 4)])
def test_chunk_attention_q4_many_pieces(gpu, H, G, D, most):
    """Shares that run over many pieces, heads and blocks: blocks of one tile's rows and of two, of a single key and of several
    tiles, cut or whole, with spoilt values that later rows see and earlier ones do not."""
    r = np.random.default_rng(D + H)
    pieces, row = [], 0
    for _ in range(70):
        n = int(r.integers(1, most + 1))
        pieces.append((row, n, int(r.choice([0, 1, 30, 63, 64, 127, 128, 300]))))
        row += n + int(r.integers(0, 2))
    T = row + 2
    pages = [0] * T
    for row0, n, pos in pieces:
        pages[row0] = -(-(pos + n) // 16)
    q, kc, vc, table = attention_case(T + H, T, H, G, D, 16, pages)
    spoil(r, vc, table, [(a, n + p) for a, n, p in pieces[::2]], D, 0.01)
    spoil(r, kc, table, [(a, n + p) for a, n, p in pieces[1::5]], D, 0.005)
    got = chunk_q4(gpu, q, kc, vc, table, [(a, n, p, 0) for a, n, p in pieces], D ** -0.5)
    clean = without_nans(kc, D), without_nans(vc, D)
    rest = np.ones(T, bool)
    for row0, n, pos in pieces:
        check_with_nans(got[row0:row0 + n], q[row0:row0 + n], (kc, vc), clean, table[row0], pos, D ** -0.5, True)
        rest[row0:row0 + n] = False
    assert (got[rest] == 3).all()


# ---- pages -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("A,NP,words,n", [(1, 2, 1, 1), (2, 9, 34, 4), (64, 40, 2048, 13), (7, 300, 68, 149), (3, 8, 5000, 3)])
def test_page_copy(gpu, A, NP, words, n):
    r = np.random.default_rng(A + NP)
    caches = [r.integers(0, 256, (NP, words * 16)).astype(u8) for _ in range(A)]
    order = r.permutation(NP)
    pairs = np.stack([order[r.integers(0, NP - n, n + 3)], np.concatenate([order[NP - n:], [0, 1, 0]])], 1).astype(i32)
    if n >= 3:
        pairs[0, 0], pairs[1, 1] = NP, -1      # pages that do not exist: the pair is skipped
        pairs[2, 0] = pairs[2, 1]              # a page onto itself
    bufs = [gpu.tensor(c) for c in caches]
    bases = gpu.tensor(np.array([b.ptr for b in bufs], np.uint64))
    pb = gpu.tensor(pairs)
    k = gpu.kernel("page_copy", [[A], [n + 3, 2]])
    gpu.launch(k, [bases, pb, I32(n), I32(NP), I32(words * 16)])   # the last three pairs lie behind n
    gpu.sync()
    for c, b in zip(caches, bufs):
        want = c.copy()
        for s, d in pairs[:n]:
            if 0 <= s < NP and 0 <= d < NP:
                want[d] = c[s]
        assert np.array_equal(gpu.fetch(b, u8, c.shape), want)
    gpu.launch(k, [bases, pb, I32(0), I32(NP), I32(words * 16)])
    gpu.sync()
    for b in bufs + [bases, pb]:
        gpu.free(b)


def test_page_copy_skips_caches_without_an_aligned_address(gpu):
    r = np.random.default_rng(9)
    c = r.integers(0, 256, (4, 64)).astype(u8)
    b = gpu.tensor(c)
    bases = gpu.tensor(np.array([0, b.ptr + 8, b.ptr], np.uint64))
    pairs = gpu.tensor(np.array([[0, 2], [1, 3]], i32))
    gpu.launch(gpu.kernel("page_copy", [[3], [2, 2]]), [bases, pairs, I32(2), I32(4), I32(64)])
    gpu.sync()
    assert np.array_equal(gpu.fetch(b, u8, c.shape), c[[0, 1, 0, 1]])
    for x in (b, bases, pairs):
        gpu.free(x)


@pytest.mark.parametrize("H,G,D,P", [(32, 8, 128, 16), (8, 4, 256, 16)])
def test_caches_beyond_four_gigabytes(gpu, H, G, D, P):
    """The last pages of a cache of more than 2^32 bytes: every kernel gives what it gives in a small cache, to the bit."""
    small, pages = 70, [40, 20]
    lens = np.array([39 * P + 3, 20 * P], i32)
    q, kc, vc, table = attention_case(3, 2, H, G, D, P, pages)
    kc, vc = (np.concatenate([c, np.zeros((small - len(c),) + c.shape[1:], u8)]) for c in (kc, vc))
    size = kc[0].nbytes
    NP = (2 ** 32 + 2 ** 28) // size
    off = NP - small
    big = [gpu.alloc(NP * size) for _ in range(2)]
    for b, c in zip(big, (kc, vc)):
        gpu.write(b, off * size, c)
    shape = [NP] + list(kc.shape[1:])
    T, W = 5, (H + 2 * G) * D
    r = np.random.default_rng(4)
    qkv, pos = r.standard_normal((T, W)).astype(h), np.arange(T, dtype=i32)
    slot = (r.permutation(2 * P)[:T] + (small - 2) * P).astype(i32)
    cs = [r.standard_normal((T, D // 2)).astype(f) for _ in range(2)]
    meta = np.array([[0, 1, 38 * P, 0], [1, 1, 5, 0]], i32)
    res = []
    for big_one in (False, True):
        o = off if big_one else 0
        caches = big if big_one else [gpu.tensor(kc), gpu.tensor(vc)]
        cshape = shape if big_one else list(kc.shape)
        t = lambda a: gpu.tensor(a)
        out = []
        def call(name, arrays, shapes, scalars, outs):
            bufs = [a if not isinstance(a, np.ndarray) else t(a) for a in arrays]
            gpu.launch(gpu.kernel(name, shapes), bufs + scalars)
            gpu.sync()
            out.extend(gpu.fetch(bufs[i], h, shapes[i]).view(np.uint16) for i in outs)
            for a, b in zip(arrays, bufs):
                if isinstance(a, np.ndarray):
                    gpu.free(b)
        at = (table + o).astype(i32)
        qs = [2, H, D]
        call("decode_attention_q4", [q, *caches, at, lens, np.zeros(qs, h)], [qs, cshape, cshape, at.shape, [2], qs],
             [F32(D ** -0.5)], [5])
        call("chunk_attention_q4", [q, *caches, at, meta, np.zeros(qs, h)], [qs, cshape, cshape, at.shape, [2, 4], qs],
             [F32(D ** -0.5)], [5])
        kv = [T, G, D]
        call("rope_kv_q4", [qkv, pos, (slot + o * P).astype(i32), *cs, np.zeros((T, H, D), h), *caches, np.zeros(kv, h), np.zeros(kv, h)],
             [qkv.shape, [T], [T], cs[0].shape, cs[1].shape, [T, H, D], cshape, cshape, kv, kv], [], [5, 8, 9])
        call("kv_unpack_q4", [*caches, (slot + o * P).astype(i32), np.zeros(kv, h), np.zeros(kv, h)], [cshape, cshape, [T], kv, kv],
             [], [3, 4])
        bases, pair = t(np.array([b.ptr for b in caches], np.uint64)), t(np.array([[o + small - 1, o + 1], [o, o + 2]], i32))
        gpu.launch(gpu.kernel("page_copy", [[2], [2, 2]]), [bases, pair, I32(2), I32(cshape[0]), I32(size)])
        gpu.sync()
        for b in caches:
            raw = np.empty(kc.shape, u8)
            gpu.read(b, o * size, raw)
            out.append(raw)
            gpu.free(b)
        for b in (bases, pair):
            gpu.free(b)
        res.append(out)
    for a, b in zip(*res):
        assert np.array_equal(a, b)


# ---- refusals ----------------------------------------------------------------------------------------------------------
def test_refusals(gpu):
    kc = lambda NP=4, G=2, P=16, D=128: [NP, G, P, kv4.row_bytes(D)]
    dec = lambda **c: [[3, 4, 128], kc(**c), kc(**c), [3, 5], [3], [3, 4, 128]]
    for shapes, what in [
        (dec()[:1] + [kc(), kc(NP=5)] + dec()[3:], "two arrays"),
        (dec()[:1] + [kc()[:3], kc()[:3]] + dec()[3:], "two arrays"),
        (dec(D=64), "a cache row has"),
        (dec(P=15), "must be even"),
        (dec(G=3), "multiple of kv heads"),
        (dec(G=0), "kv head"),
        (dec()[:4] + [[4], [3, 4, 128]], "shapes are"),
        (dec()[:5] + [[3, 4, 64]], "shapes are"),
        ([[3, 4, 24]] + [kc(D=24)] * 2 + [[3, 5], [3], [3, 4, 24]], "head_dim"),
        ([[3, 4, 272]] + [kc(D=272)] * 2 + [[3, 5], [3], [3, 4, 272]], "head_dim"),
        (dec(NP=1 << 30), "too many pages"),
        (dec(NP=(1 << 30) + 1), "beyond"),
    ]:
        with pytest.raises(GpuError, match=what):
            gpu.kernel("decode_attention_q4", shapes)
    with pytest.raises(GpuError, match="shapes are"):
        gpu.kernel("chunk_attention_q4", dec())
    with pytest.raises(GpuError, match="W must be"):
        gpu.kernel("rope_kv_q4", [[3, 1000], [3], [3], [9, 64], [9, 64], [3, 4, 128], kc(), kc(), [3, 2, 128], [3, 2, 128]])
    with pytest.raises(GpuError, match="T rows"):
        gpu.kernel("rope_kv_q4", [[3, 1024], [4], [3], [9, 64], [9, 64], [3, 4, 128], kc(), kc(), [3, 2, 128], [3, 2, 128]])
    with pytest.raises(GpuError, match="tables"):
        gpu.kernel("rope_kv_q4", [[3, 1024], [3], [3], [9, 63], [9, 63], [3, 4, 128], kc(), kc(), [3, 2, 128], [3, 2, 128]])
    with pytest.raises(GpuError, match="shapes are"):
        gpu.kernel("kv_unpack_q4", [kc(), kc(), [3], [4, 2, 128], [4, 2, 128]])
    with pytest.raises(GpuError, match="caches i64"):
        gpu.kernel("page_copy", [[3], [4, 3]])
    b = gpu.alloc(1 << 16)
    pc = gpu.kernel("page_copy", [[3], [4, 2]])
    for n, pages, size, what in [(5, 4, 64, "pairs"), (-1, 4, 64, "pairs"), (1, 4, 24, "multiple of 16"), (1, 4, 0, "multiple of 16"),
                                 (1, -4, 64, "multiple of 16")]:
        with pytest.raises(GpuError, match=what):
            gpu.launch(pc, [b, b, I32(n), I32(pages), I32(size)])
    k = gpu.kernel("decode_attention_q4", dec())
    with pytest.raises(GpuError, match="aligned"):
        gpu.launch(k, [gpu.wrap(b.ptr + 8, 64), b, b, b, b, b, F32(1.0)])
    with pytest.raises(GpuError, match="arguments"):
        gpu.launch(k, [b, b])
    k = gpu.kernel("chunk_attention_q4", dec()[:4] + [[2, 4], [3, 4, 128]])
    with pytest.raises(GpuError, match="4-byte"):
        gpu.launch(k, [b, b, b, gpu.wrap(b.ptr + 2, 64), b, b, F32(1.0)])
    with pytest.raises(GpuError, match="meta must be"):
        gpu.launch(k, [b, b, b, b, gpu.wrap(b.ptr + 4, 64), b, F32(1.0)])
    with pytest.raises(GpuError, match="too large"):
        gpu.kernel("decode_attention_q4", [[1, 1 << 21, 128], kc(NP=1, G=1 << 21), kc(NP=1, G=1 << 21), [1, 1], [1],
                                                                     [1, 1 << 21, 128]])
    gpu.free(b)


def test_empty_calls_do_nothing(gpu):
    b = gpu.alloc(1 << 12)
    c = [4, 2, 16, kv4.row_bytes(64)]
    gpu.launch(gpu.kernel("decode_attention_q4", [[0, 4, 64], c, c, [0, 5], [0], [0, 4, 64]]), [b] * 6 + [F32(1.0)])
    gpu.launch(gpu.kernel("chunk_attention_q4", [[0, 4, 64], c, c, [0, 5], [0, 4], [0, 4, 64]]), [b] * 6 + [F32(1.0)])
    gpu.launch(gpu.kernel("chunk_attention_q4", [[2, 4, 64], c, c, [2, 5], [0, 4], [2, 4, 64]]), [b] * 6 + [F32(1.0)])
    gpu.launch(gpu.kernel("kv_unpack_q4", [c, c, [0], [0, 2, 64], [0, 2, 64]]), [b] * 5)
    gpu.launch(gpu.kernel("rope_kv_q4", [[0, 512], [0], [0], [9, 32], [9, 32], [0, 4, 64], c, c, [0, 2, 64], [0, 2, 64]]), [b] * 10)
    gpu.launch(gpu.kernel("page_copy", [[0], [4, 2]]), [b, b, I32(4), I32(4), I32(16)])
    gpu.sync()
    assert not gpu.fetch(b, u8, (1 << 12,)).any()
    gpu.free(b)
    # An empty cache: every length is beyond it, every page outside it, and reads as zeros.
    none = np.zeros((0, 2, 16, kv4.row_bytes(64)), u8)
    q = np.ones((1, 4, 64), h)
    got = decode_q4(gpu, q, none, none, np.zeros((1, 1), i32), [5], 0.1)
    assert (got == 0).all()


# ---- captured, replayed, on another stream -----------------------------------------------------------------------------
def test_captured_and_replayed_with_new_inputs(gpu):
    """One step's chain (write, decode attention, a piece, a page copy) recorded once and replayed on other inputs: the bits of
    plain launches."""
    H, G, D, P, T = 8, 2, 128, 16, 16
    NP = 24
    r = np.random.default_rng(3)

    def inputs(seed):
        r = np.random.default_rng(seed)
        qkv, _, _, c, s = write_case(seed, T, H, G, D, P, NP)
        qkv = r.standard_normal(qkv.shape).astype(h)
        pos = r.integers(0, 60, T).astype(i32)
        slot = r.permutation(NP * P)[:T].astype(i32)
        table = np.stack([r.permutation(NP)[:4] for _ in range(T)]).astype(i32)
        lens = r.integers(1, 64, T).astype(i32)
        return [qkv, pos, slot, table, lens], c, s

    _, c, s = inputs(1)
    z = lambda *sh: np.zeros(sh, h)
    cache = lambda: np.zeros((NP, G, P, kv4.row_bytes(D)), u8)
    meta = np.array([[2, 6, 30, 0]], i32)
    host = [*inputs(1)[0], c, s, z(T, H, D), cache(), cache(), z(T, G, D), z(T, G, D), z(T, H, D), z(T, H, D), meta]
    names = "qkv pos slot table lens c s q kc vc k v o o2 meta".split()
    pairs = np.array([[3, 1], [5, 2]], i32)

    def chain(b):
        sh = dict(zip(names, (a.shape for a in host)))
        go = lambda name, on, *sc: gpu.launch(gpu.kernel(name, [sh[n] for n in on.split()]), [b[n] for n in on.split()] + list(sc))
        go("rope_kv_q4", "qkv pos slot c s q kc vc k v")
        go("decode_attention_q4", "q kc vc table lens o", F32(0.09))
        go("chunk_attention_q4", "q kc vc table meta o2", F32(0.09))
        gpu.launch(gpu.kernel("page_copy", [[2], [2, 2]]), [b["bases"], b["pairs"], I32(2), I32(NP), I32(G * P * kv4.row_bytes(D))])

    def buffers():
        b = {n: gpu.tensor(a) for n, a in zip(names, host)}
        b["bases"] = gpu.tensor(np.array([b["kc"].ptr, b["vc"].ptr], np.uint64))
        b["pairs"] = gpu.tensor(pairs)
        return b

    def feed(b, seed):
        for n, a in zip(names, inputs(seed)[0]):
            gpu.write(b[n], 0, a)

    def results(b):
        return [gpu.fetch(b[n], a.dtype, a.shape).tobytes() for n, a in zip(names, host) if n in "q kc vc k v o o2".split()]

    eager, graph = buffers(), buffers()
    chain(eager)
    want = [results(eager)]
    chain(graph)                       # the kernels are made before the capture
    gpu.sync()
    gpu.capture_begin()
    chain(graph)
    g = gpu.capture_end()
    for n in ("kc", "vc", "o", "o2"):
        gpu.fill(graph[n], 0)
    gpu.replay(g)
    assert results(graph) == want[0]
    for seed in (2, 3, 2):
        feed(eager, seed), feed(graph, seed)
        chain(eager)
        gpu.replay(g)
        gpu.replay(g)
        chain(eager)
        assert results(graph) == results(eager)
    for b in list(eager.values()) + list(graph.values()):
        gpu.free(b)


def test_two_contexts_at_once_and_a_foreign_stream(gpu):
    """Two contexts' launches overlap on the device (each on its own stream, with its own scratch), one of them on a stream
    that torch owns, over buffers that torch allocated."""
    import torch
    from tessel_b200.gpu import Gpu
    other = Gpu(0)
    stream = torch.cuda.Stream()
    other.set_stream(stream.cuda_stream)
    H, G, D, n = 32, 8, 128, 30000
    q, kc, vc, table = attention_case(13, 1, H, G, D, 16, [-(-n // 16)])
    q2 = np.flip(q, 1).copy()
    lens = np.array([n], i32)
    want = [decode_q4(gpu, x, kc, vc, table, lens, 0.088).tobytes() for x in (q, q2)]
    dev = [torch.from_numpy(a).cuda() for a in (q2, kc, vc, table, lens)]
    out = torch.zeros(q.shape, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    mine = [gpu.tensor(a) for a in (q, kc, vc, table, lens, np.zeros(q.shape, h))]
    shapes = [a.shape for a in (q, kc, vc, table, lens, q)]
    k1, k2 = gpu.kernel("decode_attention_q4", shapes), other.kernel("decode_attention_q4", shapes)
    theirs = [other.wrap(t.data_ptr(), t.numel() * t.element_size()) for t in dev + [out]]
    for _ in range(20):
        gpu.launch(k1, mine + [F32(0.088)])
        other.launch(k2, theirs + [F32(0.088)])
    gpu.sync(), other.sync()
    assert gpu.fetch(mine[5], h, q.shape).tobytes() == want[0]
    assert out.cpu().numpy().tobytes() == want[1]
    other.set_stream(None)
    other.close()
    for b in mine:
        gpu.free(b)


@pytest.mark.parametrize("D", [64, 128])
def test_attention_of_many_shapes_shares_one_workspace(gpu, D):
    """A handle for each of many step sizes must not hold memory of its own; and launches of different sizes and of both kinds,
    back to back without waiting, do not disturb one another."""
    import torch
    from tessel_b200.gpu import Gpu
    H, G, P = 8, 2, 16
    other = Gpu(0)                                    # a context of its own: nothing is made yet
    sizes = [(1, 40), (4, 300), (9, 33), (16, 8), (2, 700), (64, 5)]
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for T, MP in sizes + [(T, MP + i) for T, MP in sizes for i in range(1, 6)]:
        row, cache = [T, H, D], [4096, G, P, kv4.row_bytes(D)]
        other.kernel("decode_attention_q4", [row, cache, cache, [T, MP], [T], row])
        other.kernel("chunk_attention_q4", [row, cache, cache, [T, MP], [1, 4], row])
    held = free - torch.cuda.mem_get_info()[0]
    assert held < 96 << 20, f"72 handles hold {held >> 20} MB"

    cases, want = [], []
    for i, (T, MP) in enumerate(sizes):
        q, kc, vc, table = attention_case(i + D, T, H, G, D, P, [MP] * T)
        lens = np.random.default_rng(i).integers(1, MP * P + 1, T).astype(i32)
        meta = np.array([[0, T, MP * P - T, 0]], i32)
        for name, last in (("decode_attention_q4", lens), ("chunk_attention_q4", meta)):
            a = [q, kc, vc, table, last, np.zeros((T, H, D), h)]
            want.append(run(other, name, a, [5], [F32(0.1)])[0].tobytes())
            cases.append((other.kernel(name, [x.shape for x in a]), [other.tensor(x) for x in a], a[5]))
    for order in (cases, cases[::-1], cases[1::2] + cases[::2]):
        for _, b, o in cases:
            other.write(b[5], 0, o)
        for k, b, _ in order:
            other.launch(k, b + [F32(0.1)])
        other.sync()
        assert [other.fetch(b[5], h, o.shape).tobytes() for _, b, o in cases] == want
    # The same as two graphs that take turns.
    graphs = []
    for half in (cases[::2], cases[1::2]):
        other.capture_begin()
        for k, b, _ in half:
            other.launch(k, b + [F32(0.1)])
        graphs.append(other.capture_end())
    for _, b, o in cases:
        other.write(b[5], 0, o)
    for g in graphs * 3:
        other.replay(g)
    other.sync()
    assert [other.fetch(b[5], h, o.shape).tobytes() for _, b, o in cases] == want
    other.close()


# ---- the engine and the scheduler --------------------------------------------------------------------------------------
CFG = Config(dim=256, layers=2, heads=8, kv_heads=2, head_dim=64, ffn=512, vocab=1000, eps=1e-5, rope_theta=10000.0, max_pos=512,
             bos=1, eos=-1)


@pytest.mark.parametrize("fp8", [False, True])
def test_engine_with_a_4bit_cache(gpu, fp8):
    """Prefill, decode and a mixed step. What the engine leaves behind its last layer is checked against the definition: the
    step's cache slots hold the host quantiser's bytes of its dense K and V, its attention rows are attention over the cache
    (the kernels' own tolerances). Against the same engine on the CPU stand-in the logits are off by less than 1e-2 in the f16
    engine: the GPU's K differs from the CPU's by an f16 step (2^-11) here and there, one step in sixteen of those crosses a
    rounding border of a code (a fifteenth of a group's range, 0.3 of its deviation) at most every 2^-11 * 15 / 0.3, so the rows
    differ by some 1e-3 of their size. Not in the FP8 engine, whose E4M3 bytes move by an eighth of their value when a code
    moves: there only what is checked above says that a step is right."""
    w = Weights.random(CFG, 13)
    lim = Limits(page=16, pages=40, max_tokens=64, max_seq_pages=8)
    prompt = np.random.default_rng(0).integers(0, CFG.vocab, 30).tolist()
    n = len(prompt)
    G, D, H = CFG.kv_heads, CFG.head_dim, CFG.heads
    scale = float(f(1.0 / np.sqrt(D)))
    out = {}
    for name, dev in (("gpu", gpu), ("cpu", EmuGpu())):
        e = Engine(dev, w, lim, kv4=True, fp8=fp8)

        def behind(rows, slots):
            """Q, O and the caches of the last layer, and that the rows' slots hold their K and V."""
            l = e.layers[-1]
            shape = (40, G, 16, kv4.row_bytes(D))
            kc, vc = dev.fetch(l.kc, u8, shape), dev.fetch(l.vc, u8, shape)
            for c, dense in ((kc, e.k), (vc, e.v)):
                want = c.copy()
                kv4.write(want, slots, dev.fetch(dense, h, (rows, G, D)))
                assert np.array_equal(c, want)
            return dev.fetch(e.q, h, (rows, H, D)), dev.fetch(e.o, h, (rows, H, D)), kc, vc

        pre = e.step(prompt, list(range(n)), list(range(n)), Prefill(), [n - 1]).copy()
        behind(n, list(range(n)))
        dec = e.step([7], [n], [n], Decode([[0, 1]], [n + 1]), [0]).copy()
        if name == "gpu":
            q, o, kc, vc = behind(1, [n])
            near(o, *attend(q, kc, vc, np.array([0, 1]), n, scale))
        # One decode row, and eleven more rows of the same tokens on other pages, as a piece.
        toks = [9] + prompt[:11]
        mix = e.step(toks, [n + 1] + list(range(11)), [n + 1] + list(range(64, 75)),
                     Mixed(np.array([[0, 1]] + [[4, 5]] * 11, i32), [n + 2] + [1] * 11, [(1, 11, 0)]), [0, 11]).copy()
        if name == "gpu":
            q, o, kc, vc = behind(12, [n + 1] + list(range(64, 75)))
            near(o[:1], *attend(q[:1], kc, vc, np.array([0, 1]), n + 1, scale))
            near(o[1:], *attend(q[1:], kc, vc, np.array([4, 5]), 0, scale, True))
        out[name] = (pre, dec, mix, e.read_cache(1))
    if not fp8:
        for i in range(3):
            assert rel_err(out["gpu"][i], out["cpu"][i]) <= 1e-2
    for a, b in zip(out["gpu"][3], out["cpu"][3]):
        assert a.shape == b.shape == (40, 16, 2, 64)


def test_decode_resident_with_a_4bit_cache_is_the_steps_one_by_one(gpu):
    w = Weights.random(CFG, 14)
    lim = Limits(page=16, pages=40, max_tokens=64, max_seq_pages=8)

    def start():
        e = Engine(gpu, w, lim, kv4=True)
        toks, pos, slots, starts = [], [], [], []
        for s in range(3):
            n = 20 + s
            starts += [len(toks)] * n
            toks += [(7 * s + 3 * i) % CFG.vocab for i in range(n)]
            pos += list(range(n))
            slots += [(8 * s + i // 16) * 16 + i % 16 for i in range(n)]
        last = e.step_greedy(toks, pos, slots, Packed(starts), [19, 40, 62])
        return e, [int(t) for t in last]

    def one(e, toks, at):
        tables = [[8 * s + p for p in range(8)] for s in range(3)]
        slots = [(8 * s + a // 16) * 16 + a % 16 for s, a in enumerate(at)]
        return [int(t) for t in e.step_greedy(toks, at, slots, Decode(tables, [a + 1 for a in at]), [0, 1, 2])]

    e, toks = start()
    at, want = [20, 21, 22], []
    for _ in range(13):
        toks = one(e, toks, at)
        at = [a + 1 for a in at]
        want.append(toks)
    e, toks = start()
    first = one(e, toks, [20, 21, 22])
    got = e.decode_resident(3, 12)
    assert [first] + got.tolist() == want


@pytest.mark.parametrize("quantised", [False, True])
def test_shared_prefix_and_compaction(gpu, quantised):
    """Sequences behind a shared prefix that ends inside a page, with and without the pages being moved after every step: the
    same tokens bit for bit; and (f16 cache) the tokens of whole prompts fed the same way."""
    w = Weights.random(CFG, 15)
    lim = Limits(page=16, pages=64, max_tokens=64, max_seq_pages=16)
    prefix = [(5 * i + 1) % CFG.vocab for i in range(75)]
    reqs = [Request([(11 * s + 3 * i) % CFG.vocab for i in range(3 + 9 * s)], 5 + 4 * s) for s in range(5)]

    def go(compact, dev=gpu):
        s = Scheduler(Engine(dev, w, lim, kv4=quantised), reqs, 4, chunk=24, prefix=prefix)
        while not s.done():
            s.step()
            if compact:
                used = s.compact()
                assert len(s.free) == lim.pages - used
        assert sorted(s.free + s.prefix_pages) == list(range(lim.pages))
        return [o.tokens for o in s.finish()[0]]

    plain = go(False)
    assert plain == go(True)
    assert [len(t) for t in plain] == [r.max_new for r in reqs]
    if not quantised:
        cpu = [o.tokens for o in generate_with(Engine(EmuGpu(), w, lim), [Request(prefix + list(r.prompt), r.max_new) for r in reqs],
                                               4, True, chunk=63)[0]]
        # A near-tie may be broken the other way by the f16 rounding of the weights; most sequences agree throughout.
        assert sum(a == b for a, b in zip(plain, cpu)) >= 4


# ---- what little weights and small groups lose -------------------------------------------------------------------------
# The tolerance of an element here is from its own group's values and weights, not from the largest of the head. The kernel
# sums P = p * scale times codes of 0..15, so an error of P's own size e gives at most 15 e: with A = sum(15 p scale) / sum(p) over
# the group's tokens, a result is off by half a step of f16, by 2 ds A (ds: the scores' error, as above), by the f32 sums,
# 2^-16 A, and by the weights that the two f16 parts cannot hold: less than 2^-34 of the largest P for each of n tokens,
# and so n 2^-34 A at most.
def group_mean(q, kc, vc, row, n, scale):
    """As `attend` for one row q [H, D] and n keys: the result and that tolerance, each [H, D]."""
    H, D = q.shape
    G, P = kc.shape[1:3]
    pages = row[:-(-n // P)]
    k = kv4.read(kc[pages], D).reshape(-1, G, D)[:n].astype(f64)
    v = kv4.read(vc[pages], D).reshape(-1, G, D)[:n].astype(f64)
    ks, vs = ((kv4.parts(c[pages], D)[1] & np.uint16(0xFFF0)).view(h).astype(f64).transpose(0, 2, 1, 3).reshape(-1, G, kv4.groups(D))[:n]
              for c in (kc, vc))
    out, tol = np.zeros((H, D)), np.zeros((H, D))
    for hh in range(H):
        g = hh // (H // G)
        x = k[:, g] @ q[hh].astype(f64) * f64(f(scale))
        p = np.exp(x - x.max())
        p /= p.sum()
        out[hh] = p @ v[:, g]
        A = np.repeat(15 * (p @ vs[:, g]), 64)[:D]
        ds = 2 * 32 * 2.0 ** -24 * abs(scale) * 15 * ks[:, g].max() * np.abs(q[hh].astype(f64)).sum()
        tol[hh] = 2.0 ** -11 * np.abs(out[hh]) + (2 * ds + 2.0 ** -16 + n * 2.0 ** -34) * A + 2.0 ** -25
    return out, tol


def sink_case(seed, n, H, G, D, at, above, ratio):
    """n keys of which `at` scores `above` more than the rest's typical one and has no value; the values' last group of 64 is
    2^-ratio of the first."""
    r = np.random.default_rng(seed)
    NP = -(-n // 16) + 1
    scale = 1 / np.sqrt(D)
    q = r.standard_normal((H, D)).astype(h)
    q[:, 0] = 4                                       # every head sees the sink's key alike
    k, v = r.standard_normal((2, NP, G, 16, D))
    k[..., 0] = 0
    v *= 2.0 ** 12
    v[..., 64:] *= 2.0 ** -ratio
    page = r.permutation(NP).astype(i32)
    for t in at:
        k[page[t // 16], :, t % 16], v[page[t // 16], :, t % 16] = 0, 0
        k[page[t // 16], :, t % 16, 0] = above / (4 * scale)
    cache = []
    for x in (k, v):
        c = np.zeros((NP, G, 16, kv4.row_bytes(D)), u8)
        code, head = kv4.parts(c, D)
        cd, hd = kv4.quantize(x.astype(h))
        code[:], head[:] = kv4.pack(cd), hd
        cache.append(c)
    return q, cache[0], cache[1], page[None], scale


@pytest.mark.parametrize("H,G,D", [(8, 2, 128), (12, 2, 128), (4, 1, 64), (40, 5, 64)])
@pytest.mark.parametrize("at,above,ratio", [((0,), 14, 10), ((2000,), 14, 0), ((3999,), 14, 20), ((0,), 20, 0), ((5, 900, 3500), 20, 16),
                                            ((3999,), 24, 10), ((), 0, 20)])
def test_decode_weights_next_to_a_sink_without_value(gpu, H, G, D, at, above, ratio):
    n = 4000
    q, kc, vc, table, scale = sink_case(n + H + ratio, n, H, G, D, at, above, ratio if D == 128 else 0)
    want, tol = group_mean(q, kc, vc, table[0], n, scale)
    o, = run(gpu, "decode_attention_q4", [q[None], kc, vc, table, np.array([n], i32), np.zeros((1, H, D), h)], [5], [F32(scale)])
    near(o[0], want, tol)


@pytest.mark.parametrize("H,G,D", [(8, 2, 128), (12, 2, 64)])
def test_decode_scores_that_grow_all_along(gpu, H, G, D):
    # Every page's scores outgrow the ones before (the running maximum is renewed again and again), and most of the weight's
    # tokens have no value: what counts lies behind, 2^-12 and less of the maximum.
    n = 640
    q, kc, vc, table, scale = sink_case(H + D, n, H, G, D, (), 0, 10 if D == 128 else 0)
    kc, vc = kc.copy(), vc.copy()
    for i, page in enumerate(table[0][:n // 16]):
        x = np.zeros((G, 16, D), h)
        x[..., 0] = (9.0 * i) / (4 * scale)
        cd, hd = kv4.quantize(x)
        code, head = kv4.parts(kc, D)
        code[page], head[page] = kv4.pack(cd), hd
        if i % 3 == 2 or i == n // 16 - 1:
            kv4.parts(vc, D)[1][page] = 0             # scale 0: no value
    want, tol = group_mean(q, kc, vc, table[0], n, scale)
    o, = run(gpu, "decode_attention_q4", [q[None], kc, vc, table, np.array([n], i32), np.zeros((1, H, D), h)], [5], [F32(scale)])
    near(o[0], want, tol)


@pytest.mark.parametrize("H,G,D", [(8, 2, 128), (12, 2, 128), (16, 4, 64)])
def test_decode_of_a_long_context_has_no_bias(gpu, H, G, D):
    # The tensor cores cut products and sums off towards zero. Cuts of one sign do not average out: they stay the same share of
    # A (see above) at every length, while the result becomes smaller with it. Here a result is about A 2^-11 (64 normal numbers
    # span some fifteen steps of 0.35, and 131072 of them average to 1 / 362), half a step of f16 2^-22 A. The mean error must
    # not pass a quarter of that, 2^-24 A; rounding to f16, 2^-23 A each over 1024 elements or more, leaves 2^-28 A.
    n = 131072
    q, kc, vc, table, scale = sink_case(H, n, H, G, D, (), 0, 0)
    want, _ = group_mean(q, kc, vc, table[0], n, scale)
    o, = run(gpu, "decode_attention_q4", [q[None], kc, vc, table, np.array([n], i32), np.zeros((1, H, D), h)], [5], [F32(scale)])
    A = 15 * 2.0 ** 12 * 0.35
    assert abs((o[0].astype(f64) - want).mean()) <= 2.0 ** -24 * A


@pytest.mark.parametrize("H,G,D", [(8, 2, 128), (12, 2, 128), (5, 5, 64)])
@pytest.mark.parametrize("q_size,k_size", [(2.0 ** -18, 2e4), (2.0 ** -12, 300.0), (1000.0, 0.01), (1.2e4, 2e-3)])
def test_decode_scores_of_small_and_large_queries(gpu, H, G, D, q_size, k_size):
    n = 40
    _, _, vc, table, _ = sink_case(D + H, n, H, G, D, (), 0, 0)
    r = np.random.default_rng(H)
    q = (q_size * r.standard_normal((H, D)).clip(-3, 3)).astype(h)
    kc = np.zeros(vc.shape, u8)
    code, head = kv4.parts(kc, D)
    cd, hd = kv4.quantize((k_size * r.standard_normal(code.shape[:3] + (D,)).clip(-3, 3)).astype(h))
    code[:], head[:] = kv4.pack(cd), hd
    scale = 2 / (q_size * k_size * np.sqrt(D))
    want, tol = group_mean(q, kc, vc, table[0], n, scale)
    o, = run(gpu, "decode_attention_q4", [q[None], kc, vc, table, np.array([n], i32), np.zeros((1, H, D), h)], [5], [F32(scale)])
    near(o[0], want, tol)


@pytest.mark.parametrize("H,G,D", [(8, 2, 128), (5, 5, 64)])
@pytest.mark.parametrize("rows", [1, 3, 200])
@pytest.mark.parametrize("at,above", [((0,), 14), ((299,), 14), ((100,), 12), ((), 0)])
def test_chunk_weights_next_to_a_sink_without_value(gpu, H, G, D, rows, at, above):
    # Per element: half a step of f16; the weights' rounding to f16, 2^-11 of each, or half the spacing of the smallest f16
    # numbers, 2^-25 where the row's largest weight is 2^7 or more: 2^-32 of that one; the scores' errors, each 64 roundings of
    # 2^-24 of its products' sum, which move a weight's share of v and of the weights' sum; the f32 sums, 2^-16.
    n = 300
    _, kc, vc, table, scale = sink_case(n + H, n + rows, H, G, D, at, above, 0)
    q = np.random.default_rng(rows).standard_normal((rows, H, D)).astype(h)
    q[..., 0] = 4
    meta = np.array([[0, rows, n, 0]], i32)
    tables = np.zeros((rows, table.shape[1]), i32)
    tables[0] = table[0]
    o, = run(gpu, "chunk_attention_q4", [q, kc, vc, tables, meta, np.zeros((rows, H, D), h)], [5], [F32(scale)])
    k, v = (kv4.read(c[table[0]], D).reshape(-1, G, D).astype(f64) for c in (kc, vc))
    for i in range(rows):
        for hh in range(H):
            kk, vv = (x[:n + i + 1, hh // (H // G)] for x in (k, v))
            qq = q[i, hh].astype(f64)
            p = np.exp(kk @ qq * scale)
            p /= p.sum()
            want = p @ vv
            ds = 64 * 2.0 ** -24 * scale * (np.abs(kk) @ np.abs(qq))
            tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + (2.0 ** -11 + 2.0 ** -16) * (p @ np.abs(vv)) \
                + 2.0 ** -32 * p.max() * np.abs(vv).sum(0) + (p * ds) @ (np.abs(vv) + np.abs(want))
            near(o[i, hh], want, tol)
