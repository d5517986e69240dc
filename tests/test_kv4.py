"""The 4-bit KV cache's host side (tessel_b200/kv4.py): the quantiser's rule, the layout, and the order of page copies."""
import numpy as np
import pytest

from tessel_b200 import kv4

f16, f64 = np.float16, np.float64


def rows_of(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(f16)


@pytest.mark.parametrize("D", [16, 48, 64, 96, 128, 256])
def test_every_value_is_within_half_a_step_and_exact_in_f16(D):
    x = rows_of(D, 50, 3, D)
    x[0] = 0
    x[1, 0] = np.abs(x[1, 0])                  # zero point 0
    x[2, 1] = -np.abs(x[2, 1])                 # zero point 15
    x[3, 2, 0] = f16(65504)
    x[4] = (x[4].astype(f64) * 2.0 ** -20).astype(f16)   # subnormal f16 numbers
    codes, heads = kv4.quantize(x)
    scale = (heads & np.uint16(0xFFF0)).view(f16).astype(f64)
    zero = (heads & np.uint16(15)).astype(f64)
    wide = lambda a: np.repeat(a, kv4.GROUP, -1)[..., :D]
    exact = (codes.astype(f64) - wide(zero)) * wide(scale)
    assert np.array_equal(kv4.values(codes, heads).astype(f64), exact), "an f16 does not hold a value exactly"
    # Rounding both the zero point and x / scale to nearest: half a step, and half a step more where the sum is clamped.
    assert (np.abs(exact - x.astype(f64)) <= wide(scale) * 0.5 * (1 + 2.0 ** -20)).mean() > 0.99
    assert (np.abs(exact - x.astype(f64)) <= wide(scale) * (1 + 2.0 ** -20)).all()
    # Fifteen steps reach across the group, and the scale is no more than one part in 64 larger than that needs.
    for g in range(kv4.groups(D)):
        y = x[..., g * 64:(g + 1) * 64].astype(f64)
        span = np.maximum(y.max(-1), 0) - np.minimum(y.min(-1), 0)
        assert (scale[..., g] * 15 >= span * (1 - 2.0 ** -22)).all()
        assert (scale[..., g] <= np.maximum(span / 15 * (1 + 1 / 64), span / 15 + 2.0 ** -20)).all()


def test_infinities_and_nans_spoil_their_group_only():
    x = rows_of(1, 4, 128)
    x[0, 3], x[1, 70], x[2, 127] = np.inf, np.nan, -np.inf
    v = kv4.values(*kv4.quantize(x)).astype(f64)
    assert np.isnan(v[0, :64]).all() and np.isnan(v[1, 64:]).all() and np.isnan(v[2, 64:]).all()
    assert np.isfinite(v[0, 64:]).all() and np.isfinite(v[1, :64]).all() and np.isfinite(v[3]).all()


def test_words_hold_neighbours_in_their_halves():
    c = np.arange(8, dtype=np.uint8)[None]
    w = int(kv4.pack(c).view("<u4")[0, 0])
    for k in range(4):
        assert ((w >> (4 * k)) & 15, (w >> (16 + 4 * k)) & 15) == (2 * k, 2 * k + 1)
    r = np.random.default_rng(2).integers(0, 16, (5, 3, 64)).astype(np.uint8)
    assert np.array_equal(kv4.unpack(kv4.pack(r)), r)


@pytest.mark.parametrize("D,P", [(16, 2), (64, 16), (96, 8), (128, 16)])
def test_write_then_read(D, P):
    G, NP, T = 3, 5, 9
    cache = np.zeros((NP, G, P, kv4.row_bytes(D)), np.uint8)
    x = rows_of(3, T, G, D)
    slots = np.random.default_rng(4).permutation(NP * P)[:T].tolist()
    slots[2], slots[5] = NP * P, -1
    kv4.write(cache, slots, x)
    got = kv4.read(cache, D).reshape(NP * P, G, D)
    want = np.zeros_like(got)
    for t, s in enumerate(slots):
        if 0 <= s < NP * P:
            want[s] = kv4.values(*kv4.quantize(x[t]))
    assert np.array_equal(got, want)


def test_page_copies_read_what_was_there_before():
    rng = np.random.default_rng(5)
    for _ in range(200):
        pages = int(rng.integers(2, 30))
        n = int(rng.integers(0, pages + 1))
        pairs = list(zip(rng.integers(0, pages, n).tolist(), rng.permutation(pages)[:n].tolist()))
        try:
            waves = kv4.copy_waves(pairs, pages)
        except ValueError as e:
            assert "circle" in str(e)
            continue
        x = np.arange(pages)
        want = x.copy()
        for s, d in pairs:
            want[d] = x[s]
        for w in waves:
            assert not {s for s, _ in w} & {d for _, d in w}, "a wave reads a page it writes"
            x[[d for _, d in w]] = x[[s for s, _ in w]]
        assert np.array_equal(x, want)


def test_page_copies_that_are_refused():
    with pytest.raises(ValueError, match="written twice"):
        kv4.copy_waves([(0, 2), (1, 2)], 4)
    with pytest.raises(ValueError, match="has 4 pages"):
        kv4.copy_waves([(0, 4)], 4)
    with pytest.raises(ValueError, match="circle"):
        kv4.copy_waves([(0, 1), (1, 2), (2, 0)], 4)
    assert kv4.copy_waves([(3, 3)], 4) == []


# ---- the engine and the scheduler on the CPU stand-in ------------------------------------------------------------------
def tiny(**lim):
    from emu import EmuGpu
    from tessel_b200.engine import Engine, Limits
    from tessel_b200.model import Config, Weights
    w = Weights.random(Config.tiny(), 9)
    lim = Limits(**{**dict(page=8, pages=64, max_tokens=32, max_seq_pages=16), **lim})
    return lambda **kw: Engine(EmuGpu(), w, lim, **kw)


def test_a_step_quantises_the_keys_it_attends_to():
    from tessel_b200.engine import Decode, Prefill
    make = tiny()
    e4, e16 = make(kv4=True), make()
    prompt = [3, 1, 4, 1, 5, 9, 2, 6, 5, 3]
    n = len(prompt)
    slots = [3 * 8 + i for i in range(8)] + [5 * 8, 5 * 8 + 1]
    a = e4.step(prompt, list(range(n)), slots, Prefill(), [n - 1]).copy()
    b = e16.step(prompt, list(range(n)), slots, Prefill(), [n - 1]).copy()
    assert np.array_equal(a, b), "a prompt's own step attends to its rows in f16"
    for l in range(len(e4.layers)):
        k4, v4 = e4.read_cache(l)
        k, v = e16.read_cache(l)
        assert np.array_equal(k4, kv4.values(*kv4.quantize(k))) and np.array_equal(v4, kv4.values(*kv4.quantize(v)))
        # The f16 engine with the values the 4-bit cache stands for: the next step's logits are the same but for its own key.
        e16.gpu.write(e16.layers[l].kc, 0, k4)
        e16.gpu.write(e16.layers[l].vc, 0, v4)
    dec = Decode([[3, 5]], [n + 1])
    a = e4.step([7], [n], [5 * 8 + 2], dec, [0]).copy()
    b = e16.step([7], [n], [5 * 8 + 2], dec, [0]).copy()
    # One of eleven keys differs, by at most a step of its group's fifteen: far below the logits' own size, not nothing.
    assert 0 < np.abs(a - b).max() < 0.2 * np.abs(b).max()
    assert e4.page_bytes * 4 < e16.page_bytes * 2


def test_modes_and_limits_that_are_refused():
    with pytest.raises(ValueError, match="4-bit cache"):
        tiny(page=7)(kv4=True)
    with pytest.raises(ValueError, match="written twice"):
        tiny()().copy_pages([(0, 2), (1, 2)])


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n", [1, 8, 13, 32, 45])
def test_a_shared_prefix_gives_the_tokens_of_whole_prompts(n, quantised):
    from tessel_b200.sched import Request, Scheduler, generate_with
    prefix = [1 + (i * 37 % 250) for i in range(n)]
    own = [[5, 6, 7], [200], [9] * 20, [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11]]
    make = tiny()
    whole = [Request(prefix + p, 6) for p in own]
    rest = [Request(p, 6) for p in own]
    e = make(kv4=quantised)
    s = Scheduler(e, rest, 3, prefix=prefix)
    while not s.done():
        assert s.step() != "idle"
    assert len(s.free) == e.lim.pages - len(s.prefix_pages), "pages were lost or freed twice"
    assert sorted(s.free + s.prefix_pages) == list(range(e.lim.pages))
    got, st = s.finish()
    assert st.prompt_tokens == n + sum(map(len, own)), "the prefix is computed once"
    if quantised:
        # A whole prompt's own step attends to f16 rows, a prompt behind a prefix to quantised ones: other tokens are right.
        assert [len(o.tokens) for o in got] == [6] * len(own)
        return
    want, _ = generate_with(make(), whole, 3, True, chunk=31)
    for a, b in zip(got, want):
        assert a.tokens == b.tokens


@pytest.mark.parametrize("quantised", [False, True])
def test_compacting_changes_no_token(quantised):
    from tessel_b200.sched import Request, Scheduler
    reqs = [Request([1 + (i * 7 + j) % 250 for j in range(5 + 3 * i)], 4 + 3 * i) for i in range(5)]

    def run(compact):
        s = Scheduler(tiny()(kv4=quantised), reqs, 3, chunk=8, prefix=[11, 12, 13])
        used = []
        while not s.done():
            s.step()
            if compact:
                used.append(s.compact())
                live = set(s.prefix_pages).union(*(q.pages for q in s.running + s.feeding)) if s.running + s.feeding else set(s.prefix_pages)
                assert live == set(range(used[-1])) and len(s.free) == 64 - used[-1]
        return [o.tokens for o in s.finish()[0]]

    assert run(True) == run(False)


def test_a_prefix_that_does_not_fit_is_refused():
    from tessel_b200.sched import Request, generate_with
    with pytest.raises(ValueError, match="shared prefix"):
        generate_with(tiny()(), [Request([1], 2)], 1, True, prefix=[1] * 129)
    with pytest.raises(ValueError, match="does not fit"):
        generate_with(tiny()(), [Request([1] * 100, 2)], 1, True, prefix=[1] * 40)


@pytest.mark.parametrize("quantised", [False, True])
def test_resident_decoding_does_not_go_on_from_pages_that_moved(quantised):
    from tessel_b200.sched import Request, Scheduler
    reqs = [Request([1 + (i * 7 + j) % 250 for j in range(p)], n) for i, (p, n) in enumerate([(30, 3), (8, 20), (11, 21), (14, 22)])]

    def run(compact):
        s = Scheduler(tiny()(kv4=quantised), reqs, 4, device_argmax=True)
        moved = False
        while not s.done():
            rows = [q.id for q in s.running]
            if s.step() != "decode" or [q.id for q in s.running] != rows:
                continue                             # (a sequence has ended: the step's rows are not the running ones)
            before = [q.pages for q in s.running]
            if compact:
                s.compact()
            n = len(s.running)
            if [q.pages for q in s.running] != before:
                moved = True
                with pytest.raises(ValueError, match="moved"):
                    s.e.decode_resident(n, 2)
            elif min(q.left for q in s.running) > 2:
                for picks in s.e.decode_resident(n, 2):
                    s.absorb(picks)
        return [o.tokens for o in s.finish()[0]], moved

    (got, moved), (want, _) = run(True), run(False)
    assert moved, "no page was moved: the test shows nothing"
    assert got == want


def test_resident_decoding_after_a_copy_of_pages_needs_a_step_with_its_tables():
    from tessel_b200.engine import Decode, Prefill
    e = tiny()()
    e.step_greedy([3, 1, 4], [0, 1, 2], [24, 25, 26], Prefill(), [2])
    e.step_greedy([7], [3], [27], Decode([[3]], [4]), [0])
    e.copy_pages([(3, 5)])
    assert e.decode_resident(1, 0).shape == (0, 1)
    with pytest.raises(ValueError, match="moved"):
        e.decode_resident(1, 1)
    e.copy_pages([])                                  # copies nothing
    e.step_greedy([8], [4], [44], Decode([[5]], [5]), [0])
    assert e.decode_resident(1, 2).shape == (2, 1)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n", [8, 13, 0])
def test_a_request_that_does_not_fit_leaves_those_before_it_whole(n, quantised):
    from tessel_b200.sched import Request, Scheduler
    prefix = [1 + (i * 37 % 250) for i in range(n)]
    good = [Request([5, 6, 7], 6), Request([9] * 12, 6)]
    bad = Request([3] * 20, 16 * 8)

    def run(reqs, drop):
        s = Scheduler(tiny()(kv4=quantised), reqs, 4, prefix=prefix)
        s.e.gpu.write(s.e.layers[0].kc, 0, np.full(s.e.page_bytes * s.e.lim.pages, 0x55, np.uint8))   # no page is zeros to begin with
        refused = 0
        while not s.done():
            try:
                s.step()
            except ValueError:
                refused += 1
                assert s.waiting.popleft() == drop   # the caller drops the request at the head and goes on
        assert refused == (drop is not None)
        assert sorted(s.free + s.prefix_pages) == list(range(s.e.lim.pages)), "pages were lost"
        return [o.tokens for o in s.finish()[0]]

    want = run(good, None)
    assert run([good[0], bad, good[1]], 1)[::2] == want
    assert run(good + [bad], 2)[:2] == want


def far_bounds():
    """Groups of 64 whose two bounds need more than 24 bits side by side: an end of the range 15 * 2^e or 15 * scale next to a
    much smaller number of the other sign; and, for comparison, the end alone. The ranges, and the rows f16 [n, 64]."""
    rows = []
    for e in (-8, 0, 5, 11):
        for top in (15 * 2.0 ** e, 15 * 127 / 64 * 2.0 ** e, 15 * 65 / 64 * 2.0 ** e):
            for small in (0.0, 2.0 ** -24, 2.0 ** -23, 3 * 2.0 ** -24, 2.0 ** -14, 2.0 ** -10):
                for sign in (1, -1):
                    rows.append([sign * top, -sign * small] + [sign * top * i / 70 for i in range(62)])
    x = np.asarray(rows, f16)
    assert (x[:, 0].astype(f64) == [r[0] for r in rows]).all()   # both ends are f16 numbers
    return x


def test_the_scale_is_rounded_up_from_the_exact_range():
    from fractions import Fraction as F
    x = far_bounds()
    codes, heads = kv4.quantize(x)
    got = (heads[:, 0] & np.uint16(0xFFF0)).view(f16).astype(f64)
    for row, scale in zip(x.astype(f64), got):
        r = (F(max(row.max(), 0)) - F(min(row.min(), 0))) / 15
        step = F(2) ** (int(np.frexp(float(r))[1]) - 7)
        want = -(-r // step) * step
        assert F(scale) == want, (row[:2], scale, float(want))


def test_the_attention_kernels_workspace_is_asked_for_with_the_cache():
    # On a device the library allocates it with the first handle; here the handles are looked at.
    make = tiny()
    assert "decode_attention_q4" in [name for name, _ in make(kv4=True).gpu._kernels]
    assert "decode_attention_q4" not in [name for name, _ in make().gpu._kernels]


def test_copying_pages_does_not_wait_for_the_device():
    """On a stand-in whose device is behind the host: copies to it and launches happen when somebody waits for it, and an array
    handed to `write_async` is read only then."""
    from emu import EmuGpu
    from tessel_b200.engine import Decode, Engine, Limits, Prefill
    from tessel_b200.model import Config, Weights

    class Late(EmuGpu):
        def __init__(self):
            super().__init__()
            self.queue, self.waits = [], 0

        def sync(self):
            self.waits += bool(self.queue)
            queue, self.queue = self.queue, []
            for call in queue:
                call()

        def write(self, b, offset, data):
            self.sync()
            super().write(b, offset, data)

        def read(self, b, offset, out):
            self.sync()
            return super().read(b, offset, out)

        def write_async(self, b, offset, a):
            assert offset + a.nbytes <= b.bytes
            self.queue.append(lambda: EmuGpu.write(self, b, offset, a))

        def launch(self, k, args):
            args = list(args)
            self.queue.append(lambda: EmuGpu.launch(self, k, args))

    w = Weights.random(Config.tiny(), 9)
    e = Engine(Late(), w, Limits(page=4, pages=40, max_tokens=16, max_seq_pages=8))
    e.graphs = False
    e.copy_pages([(0, 1)])                            # (the first call makes its tables)
    e.gpu.sync()
    rng = np.random.default_rng(1)
    shape = (40, e.page_bytes // 2)
    want = []
    for l in e.layers:
        for b in (l.kc, l.vc):
            x = rng.standard_normal(shape).astype(f16)
            e.gpu.write(b, 0, x)
            want.append(x)
    e.step_greedy([3, 1], [0, 1], [0, 1], Prefill(), [1])
    want = [e.gpu.fetch(b, f16, shape) for l in e.layers for b in (l.kc, l.vc)]
    before = e.gpu.waits
    calls = [[(0, 9), (0, 10), (3, 11)], [(9, 20)], [(20, 30), (11, 20)], [(i, i + 1) for i in range(39)], [(5, 6)]]
    for pairs in calls[:3]:
        e.copy_pages(pairs)
    assert e.gpu.waits == before and e.gpu.queue, "the host waited for the device"
    for i in range(60):                               # many more than fit side by side, whatever that takes
        e.copy_pages(calls[3 + i % 2])
    e.gpu.sync()
    for x, b in zip(want, (b for l in e.layers for b in (l.kc, l.vc))):
        for pairs in calls[:3] + [calls[3 + i % 2] for i in range(60)]:
            old = x.copy()
            for s, d in pairs:
                x[d] = old[s]
        assert np.array_equal(e.gpu.fetch(b, f16, shape), x)
    # A step's end has waited for the device in any case: from there on the room is free again.
    for i in range(100):
        e.step_greedy([7], [2 + i % 4], [2 + i % 4], Decode([[0]], [3 + i % 4]), [0])
        before = e.gpu.waits
        e.copy_pages([(i % 40, (i + 1) % 40), ((i + 2) % 40, (i + 3) % 40)])
        assert e.gpu.waits == before


def test_pages_that_cannot_be_copied_are_refused_before_anything_is_admitted():
    # head_dim 16 in 4 bits: 10 bytes a row and head, so two tokens of two heads are a page of 40 bytes.
    from tessel_b200.sched import Request, Scheduler
    e = tiny(page=2)(kv4=True)
    assert e.page_bytes % 16
    with pytest.raises(ValueError, match="multiple of 16"):
        e.copy_pages([(0, 1)])
    with pytest.raises(ValueError, match="multiple of 16"):
        Scheduler(e, [Request([1], 2)], 1, prefix=[1, 2, 3])
    s = Scheduler(e, [Request([1], 2), Request([7, 8], 2)], 2, prefix=[1, 2])   # ends with a page: nothing is forked
    while not s.done():
        assert s.step() != "idle"
    with pytest.raises(ValueError, match="multiple of 16"):
        s = Scheduler(e, [Request([1, 2, 3], 2), Request([7, 8], 6)], 2)
        while not s.done():
            s.step()
            s.compact()
    assert s.running and [q.pages for q in s.running] == [[3, 4, 5, 6]], "the tables are as they were"
